"""What the attention over a serving cache refuses (include/ct2_mi355.h): every call here ends in the
argument checks, before a stream or a kernel is touched, so it needs no GPU. Pointers are numbers."""
import pytest

from ctranslate2_amd import _lib

F32, I8, F16, BF16 = 0, 1, 4, 5
A, B, C, D, E, S = (0x10000000 * i for i in range(1, 7))  # far apart, aligned


def refused(name, args):
    L = _lib.lib()
    assert getattr(L, name)(*args) != 0
    return L.ct2x_last_error().decode()


def tree(**kw):
    a = dict(q=A, k=B, v=C, kv_dtype=F16, lengths=None, length=5, mask=None, batch=1, tokens=2, heads=4, heads_kv=2,
             dhead=64, t_max=16, scale=1.0, out=D, scratch=S, scratch_bytes=1 << 30, stream=None)
    a.update(kw)
    return "ct2x_attention_tree", list(a.values())


def accumulate(**kw):
    a = dict(q=A, k=B, v=C, kv_dtype=F16, lengths=None, length=5, batch=1, heads=4, heads_kv=2, dhead=64, t_max=16,
             scale=1.0, weights=E, out=D, scratch=S, scratch_bytes=1 << 30, stream=None)
    a.update(kw)
    return "ct2x_attention_accumulate", list(a.values())


def evict(**kw):
    a = dict(k=A, v=B, kv_dtype=F16, weights=C, lengths=None, length=9, batch=1, heads_kv=2, dhead=64, t_max=16,
             budget=4, recent=1, t_max_out=4, k_out=D, v_out=E, weights_out=S, positions=S + 4096,
             lengths_out=S + 8192, stream=None)
    a.update(kw)
    return "ct2x_cache_evict", list(a.values())


def bounds(**kw):
    a = dict(k=A, kv_dtype=F16, first=None, lengths=None, length=9, batch=1, heads_kv=2, dhead=64, t_max=16, block=16,
             bounds=B, stream=None)
    a.update(kw)
    return "ct2x_cache_block_bounds", list(a.values())


def blocks(**kw):
    a = dict(q=A, k=B, v=C, kv_dtype=F16, bounds=E, lengths=None, length=5, batch=1, heads=4, heads_kv=2, dhead=64,
             t_max=64, block=16, top=2, sink=1, local=1, scale=1.0, out=D, selected=None, scratch=S,
             scratch_bytes=1 << 30, stream=None)
    a.update(kw)
    return "ct2x_attention_blocks", list(a.values())


COMMON = [
    (dict(batch=-1), "batch"), (dict(heads_kv=0), "heads_kv"), (dict(dhead=4), "dhead"), (dict(dhead=60), "dhead"),
    (dict(dhead=264), "dhead"), (dict(t_max=0), "t_max"), (dict(t_max=1 << 40), "t_max"), (dict(kv_dtype=I8), "type"),
    (dict(kv_dtype=7), "type"), (dict(length=-1), "length"), (dict(length=1000), "length"), (dict(batch=1 << 40), "2^22"),
    (dict(k=None), "NULL"), (dict(k=A + 8), "aligned"),
]
HEADS = [(dict(heads=5), "multiple"), (dict(heads=0), "multiple"), (dict(heads=4096), "1024"),
         (dict(batch=1 << 20, heads=256), "2^26"), (dict(q=None), "NULL"), (dict(out=None), "NULL"),
         (dict(out=D + 4), "aligned"), (dict(scratch=None), "scratch"), (dict(scratch_bytes=8), "scratch"),
         (dict(scratch=S + 8), "aligned")]


@pytest.mark.parametrize("entry", (tree, accumulate, evict, bounds, blocks), ids=lambda f: f.__name__)
@pytest.mark.parametrize("change, word", COMMON, ids=lambda c: str(c)[:30])
def test_common_refusals(entry, change, word):
    assert word in refused(*entry(**change))


@pytest.mark.parametrize("entry", (accumulate, blocks), ids=lambda f: f.__name__)
@pytest.mark.parametrize("change, word", HEADS, ids=lambda c: str(c)[:30])
def test_attention_refusals(entry, change, word):
    assert word in refused(*entry(**change))


@pytest.mark.parametrize("call, word", [
    (tree(tokens=-1), "tokens"), (tree(tokens=1025, t_max=4096), "tokens"), (tree(tokens=17), "tokens"),
    (tree(length=15), "length"), (tree(heads=5), "multiple"), (tree(v=None), "NULL"), (tree(q=A + 4), "aligned"),
    (accumulate(weights=None), "NULL"),
    (evict(budget=0), "budget"), (evict(recent=5), "recent"), (evict(recent=-1), "recent"),
    (evict(t_max_out=3), "t_max_out"), (evict(k_out=A), "overlap"), (evict(k_out=A, t_max_out=16), None),
    (evict(k_out=A + 256), "overlap"), (evict(v_out=A), "overlap"), (evict(v_out=D), "overlap"),
    (evict(weights_out=C), "overlap"), (evict(positions=None), "NULL"), (evict(lengths_out=None), "NULL"),
    (bounds(block=8), "block"), (bounds(block=24), "block"), (bounds(block=272), "block"), (bounds(bounds=None), "NULL"),
    (blocks(top=0), "top"), (blocks(sink=-1), "sink"), (blocks(sink=2), "sink"), (blocks(local=3), "sink"),
    (blocks(scale=0.0), "scale"), (blocks(scale=-1.0), "scale"), (blocks(scale=float("nan")), "scale"),
    (blocks(block=20), "block"), (blocks(bounds=None), "NULL"),
], ids=str)
def test_refusals(call, word):
    if word is None:  # the same output as an input is in place, which is legal: refused for its weights only
        call[1][15] = call[1][3]  # weights_out = weights
        call[1][14] = call[1][0]  # v_out = k
        word = "overlap"
    assert word in refused(*call)


def test_scratch_sizes_and_empty_calls():
    L = _lib.lib()
    assert L.ct2x_attention_tree_scratch_bytes(2, 8, 8, 2, 64, 1000) >= 0
    assert L.ct2x_attention_accumulate_scratch_bytes(2, 8, 2, 64, 1000) > 0
    assert L.ct2x_attention_blocks_scratch_bytes(2, 8, 2, 64, 1000, 32, 4) > 0
    assert L.ct2x_attention_tree_scratch_bytes(2, 8, 7, 2, 64, 1000) == -1
    assert L.ct2x_attention_accumulate_scratch_bytes(2, 8, 2, 65, 1000) == -1
    assert L.ct2x_attention_blocks_scratch_bytes(2, 8, 2, 64, 1000, 31, 4) == -1
    for name, args in (tree(batch=0), tree(tokens=0), accumulate(batch=0), evict(batch=0), bounds(batch=0),
                       blocks(batch=0)):
        assert getattr(L, name)(*args) == 0, name
