"""Attention over a serving cache at the edges of its documentation (include/ct2_mi355.h): values that are not
finite among the committed positions, sizes at the limits. Oracles and tolerances of
tests/test_cache_ops_gpu.py."""
import math

import numpy as np
import pytest
import torch

import test_cache_ops_gpu as C
from ctranslate2_amd import _lib

pytestmark = pytest.mark.gpu


# one case for each kernel of a tree: every wave loads for itself; tiles shared, 16 and 32 rows a wave (the long
# trees of float16 and float32); heads beyond 128 channels
@pytest.mark.parametrize("dtype", C.TYPES)
@pytest.mark.parametrize("tokens, heads, dhead, n, t_max", [
    (3, 2, 64, 50, 60), (20, 4, 64, 50, 80), (20, 4, 128, 77, 100), (40, 4, 128, 1900, 384000),
    (40, 4, 64, 1900, 384000), (5, 4, 200, 45, 60)], ids=str)
@pytest.mark.parametrize("value", (math.inf, -math.inf, math.nan), ids=str)
def test_tree_committed_values_that_are_not_finite(gpu, dtype, tokens, heads, dhead, n, t_max, value):
    """A committed position's infinite or NaN value leaves infinities or NaN in its channel of every row, wherever
    it stands: before the step that the drafted tokens begin in, first in it, and last of the committed ones."""
    gen, rng = C.generator(41), np.random.default_rng(41)
    k, v = C.make_cache(gen, dtype, 1, 1, t_max, dhead)
    q = torch.randn((1, tokens, heads, dhead), device="cuda", generator=gen)
    seen = C.tree_mask(rng, 1, tokens)
    scale = 1 / math.sqrt(dhead)
    for at, channel in ((3, 0), (n - n % 32, 5), (n - 1, dhead - 1)):
        held = v[0, 0, at, channel].clone()
        v[0, 0, at, channel] = value
        got = C.run_tree(q, k, v, dtype, None, n, C.to_words(seen), scale)
        finite = torch.isfinite(got[0]).all(dim=0).all(dim=0)
        assert not bool(torch.isfinite(got[0, :, :, channel]).any()), at
        assert int(finite.sum()) == dhead - 1, at
        v[0, 0, at, channel] = held
    got = C.run_tree(q, k, v, dtype, None, n, C.to_words(seen), scale)
    C.check_tree(got, q, k, v, dtype, [n], seen, scale)


ROWS = 2 ** 22  # the most (entry, head of the cache) pairs of a call


def test_evict_of_the_most_rows(gpu):
    """A launch holds less than 2^32 threads: this many rows take several."""
    gen = C.generator(42)
    shape = (ROWS // 2, 2, 2, 8)
    k = torch.randn(shape, device="cuda", generator=gen).half()
    v = torch.randn(shape, device="cuda", generator=gen).half()
    w = torch.rand(shape[:3], device="cuda", generator=gen)
    k_out, v_out, w_out = k[:, :, :1].clone(), v[:, :, :1].clone(), w[:, :, :1].clone()
    n_out = torch.full((shape[0],), -7, dtype=torch.int32, device="cuda")
    positions = C.run_evict(k, v, w, "f16", None, 2, 1, 0, k_out, v_out, w_out, n_out)
    heavier = (w[:, :, 1] > w[:, :, 0]).int()
    assert torch.equal(positions[:, :, 0], heavier)
    at = heavier.long()[:, :, None]
    assert torch.equal(w_out, torch.gather(w, 2, at))
    for out, old in ((k_out, k), (v_out, v)):
        assert torch.equal(out, torch.gather(old, 2, at[..., None].expand(-1, -1, -1, 8)))
    assert bool((n_out == 1).all())


def test_blocks_of_the_most_rows(gpu):
    gen = C.generator(43)
    batch, t_max = ROWS // 2, 17
    shape = (batch, 2, t_max, 8)
    k = torch.randn(shape, device="cuda", generator=gen).half()
    v = torch.randn(shape, device="cuda", generator=gen).half()
    q = torch.randn((batch, 2, 8), device="cuda", generator=gen)
    out, selected = torch.full_like(q, 7.0), torch.full((batch, 2, 1), 7, dtype=torch.int32, device="cuda")
    bounds = torch.zeros((batch, 2, 2, 2, 8), dtype=k.dtype, device="cuda")
    L = _lib.lib()
    need = L.ct2x_attention_blocks_scratch_bytes(batch, 2, 2, 8, t_max, 16, 1)
    scratch = torch.empty((need,), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    _lib.check(L.ct2x_cache_block_bounds(_lib.ptr(k), 4, None, None, t_max, batch, 2, 8, t_max, 16, _lib.ptr(bounds),
                                         None))
    _lib.check(L.ct2x_attention_blocks(
        _lib.ptr(q), _lib.ptr(k), _lib.ptr(v), 4, _lib.ptr(bounds), None, t_max, batch, 2, 2, 8, t_max, 16, 1, 0, 1,
        0.3, _lib.ptr(out), _lib.ptr(selected), _lib.ptr(scratch), need, None))
    C.sync()
    assert bool((selected == 1).all())  # the last block, of one position: its value
    assert torch.equal(bounds[:, :, 1, 0], k[:, :, 16]) and torch.equal(bounds[:, :, 0, 1], k[:, :, :16].amax(2))
    # One probability p, whatever its reference: out = (y0 v + y1 v) (1 / p) with y0 + y1 within 2^-23 of p; the sum,
    # the reciprocal (2^-23 allowed) and the last product round by 2^-24 each: 2^-21 in all.
    want = v[:, :, 16].double()
    assert bool(((out.double() - want).abs() <= 2.0 ** -21 * want.abs()).all())


# What the terms of a 16-bit type leave of a query and of a probability, at worst: of the value itself, and of the
# row's largest (include/ct2_mi355.h).
QUERY_LEFT = {"f32": (0, 0), "f16": (2.0 ** -23, 2.0 ** -36), "bf16": (2.0 ** -26, 0)}
PROBABILITY_LEFT = {"f32": (0, 0), "f16": (2.0 ** -23, 2.0 ** -38), "bf16": (2.0 ** -26, 0)}
SPANS = [(4, 2, 64, None), (20, 8, 64, None), (20, 8, 128, None), (40, 4, 64, 380000),
         (40, 4, 128, 380000), (2, 2, 256, None)]


@pytest.mark.parametrize("dtype", C.TYPES)
@pytest.mark.parametrize("tokens, heads, dhead, room", SPANS, ids=str)
@pytest.mark.parametrize("size", (1024.0, 16384.0))
def test_tree_one_large_query_channel(gpu, dtype, tokens, heads, dhead, room, size):
    """A query channel far above the others, on key channels of zero: the others' products decide, and each is to be
    as good as its own size allows.

    The scores are off by ds as in tests/test_cache_ops_gpu.py, its split term among them (that formula counts terms
    relative to each element), and by what is left of the largest element's size times the keys' 1-norm."""
    gen, rng = C.generator(44), np.random.default_rng(44)
    n = 300
    k, v = C.make_cache(gen, dtype, 1, 1, room or n + tokens, dhead)
    k[..., 5] = 0
    q = torch.randn((1, tokens, heads, dhead), device="cuda", generator=gen) * 2
    q[..., 5] = size
    seen = C.tree_mask(rng, 1, tokens)
    scale = 1 / math.sqrt(dhead)
    got = C.run_tree(q, k, v, dtype, None, n, C.to_words(seen), scale)
    visible = torch.ones((tokens, n + tokens), dtype=torch.bool, device="cuda")
    visible[:, n:] = torch.from_numpy(seen[0]).cuda()
    for h in range(heads):
        kk, vv = k[0, 0, :n + tokens], v[0, 0, :n + tokens]
        want, tol, _ = C.reference(q[0, :, h], kk, vv, visible, scale, dtype)
        left = QUERY_LEFT[dtype][1] * size * scale * float(kk.double().abs().sum(1).max())
        C.within(got[0, :, h], want, tol + 2 * left * float(vv.double().abs().max()), "head %d" % h)


@pytest.mark.parametrize("dtype", C.TYPES)
@pytest.mark.parametrize("tokens, heads, dhead, room", SPANS, ids=str)
@pytest.mark.parametrize("depth", (15.3, 18.7, 20.6))
def test_tree_a_long_tail_of_small_probabilities(gpu, dtype, tokens, heads, dhead, room, depth):
    """Every sixteenth position takes nearly all of the probability and has values of zero: the output is the sum over
    thousands of positions with probabilities 2^-depth of those, all alike, whose errors add up. Each is off by what
    is left of it and of the row's largest, on top of the tolerance of tests/test_cache_ops_gpu.py."""
    gen = C.generator(45)
    n = 4000
    k = torch.zeros((1, 1, room or n + tokens, dhead), dtype=C.TYPES[dtype][1], device="cuda")
    v = torch.zeros_like(k)
    v[0, 0, :n] = 1 + torch.rand((n, dhead), device="cuda", generator=gen)
    k[0, 0, :n:16, 0] = 1
    v[0, 0, :n:16] = 0
    q = torch.zeros((1, tokens, heads, dhead), device="cuda")
    q[..., 0] = depth * math.log(2)  # the score of those positions; the others' are zero
    seen = np.zeros((1, tokens, tokens), dtype=bool)
    got = C.run_tree(q, k, v, dtype, None, n, C.to_words(seen), 1.0)
    visible = torch.ones((tokens, n), dtype=torch.bool, device="cuda")
    for h in range(heads):
        want, tol, p = C.reference(q[0, :, h], k[0, 0, :n], v[0, 0, :n], visible, 1.0, dtype)
        off = PROBABILITY_LEFT[dtype][1] * float(p[0][0].max()) * v[0, 0, :n].double().sum(0)
        C.within(got[0, :, h], want, tol + off, "head %d" % h)
