"""The ways a program may write the calls of the attention over a serving cache, and what their argument
checks refuse beyond tests/test_cache_refusals.py. No GPU: every call ends in the argument checks."""
import pytest

from ctranslate2_amd import _lib
from test_cache_refusals import A, B, C, D, E, S, evict, refused


def test_eviction_takes_the_tail_of_the_attention_calls():
    """(.., d_scratch, scratch_bytes, stream) as well as (.., stream): the workspace is not the stream."""
    L = _lib.lib()
    name, own = evict(batch=0)
    assert L.ct2x_cache_evict(*own) == 0
    assert L.ct2x_cache_evict(*own[:-1], S + 65536, 1 << 20, None) == 0
    assert L.ct2x_cache_evict(*own[:-1], None, 0, None) == 0
    name, own = evict(budget=0)
    assert "budget" in refused(name, own)
    assert "budget" in refused(name, own[:-1] + [S + 65536, 1 << 20, None])


def test_the_stream_stays_the_last_argument():
    given = []

    def call(*args):
        given.append(args)
        return 0

    call.argtypes = [None] * 3
    either = _lib._without_workspace(call)
    assert either(1, 2, "stream") == 0 and either(1, 2, "workspace", 16, "stream") == 0
    assert given == [(1, 2, "stream")] * 2


@pytest.mark.parametrize("change", (-1, 1, 3))
def test_eviction_refuses_other_numbers_of_arguments(change):
    own = evict(batch=0)[1]
    with pytest.raises(TypeError, match="arguments"):
        _lib.lib().ct2x_cache_evict(*(own[:change] if change < 0 else own + [None] * change))


# the arguments of `evict` by where they lie: k A, v B, weights C, k_out D, v_out E, weights_out S,
# positions S + 4096, lengths_out S + 8192; keys and values in are 4096 bytes, out 1024, weights in 128, out 32,
# positions 32, lengths 4
@pytest.mark.parametrize("change", [
    dict(weights_out=A), dict(weights_out=B + 4064), dict(weights_out=D + 512), dict(weights_out=E),
    dict(weights_out=C + 64), dict(weights_out=C), dict(positions=A + 4092), dict(positions=B), dict(positions=C),
    dict(positions=C + 124), dict(positions=D), dict(positions=E + 1020), dict(positions=S), dict(positions=S + 28),
    dict(lengths_out=A), dict(lengths_out=B + 4092), dict(lengths_out=C + 4), dict(lengths_out=D), dict(lengths_out=E),
    dict(lengths_out=S + 28), dict(lengths_out=S + 4096 + 28),
    dict(k_out=C - 1008), dict(v_out=C + 112), dict(k_out=B), dict(k_out=A, t_max_out=8), dict(v_out=B, t_max_out=8),
    # two entries' lengths on the device: one entry apart is an overlap, the same pointer is in place
    dict(batch=2, lengths=S + 16384, lengths_out=S + 16388), dict(batch=2, lengths=S + 16388, lengths_out=S + 16384),
    dict(lengths=S + 16384, positions=S + 16380), dict(lengths=S + 16384, weights_out=S + 16384),
    dict(lengths=D + 64), dict(lengths=E + 1020),
], ids=str)
def test_eviction_refuses_every_other_overlap(change):
    assert "overlap" in refused(*evict(**change))


def test_eviction_in_place_passes_the_overlap_checks():
    """What follows the overlap checks is a launch: the checks are passed where the error is not theirs (no GPU) or
    there is none to be had without one."""
    import torch
    if torch.cuda.is_available():
        pytest.skip("the pointers are numbers")
    for change in (dict(), dict(k_out=A, v_out=B, weights_out=C, t_max_out=16), dict(v_out=B, t_max_out=16),
                   dict(lengths=S + 8192), dict(lengths=S + 16384, positions=S + 16384 - 32), dict(k_out=A + 4096),
                   dict(lengths_out=C + 128), dict(positions=S + 32)):
        assert "overlap" not in refused(*evict(**change)), change
