"""The ways a program may write the calls of the attention over a serving cache, and what their argument
checks refuse beyond tests/test_cache_refusals.py. No GPU: every call ends in the argument checks."""
import pytest

from ctranslate2_amd import _lib
from test_cache_refusals import S, evict, refused


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
