"""How precise the attention over a serving cache is as a whole (include/ct2_mi355.h): the relative 2-norm of an
output's error against float64, per kernel and type. The tolerances element by element of
tests/test_cache_ops_gpu.py hold for the worst of all roundings; they would not notice a term less.

The bound for 16-bit caches, 25 x 2^-24 = 1.5e-6, for queries of twice a normal distribution's size: scores are of size 2, their
exponents' arguments up to about 12 x log2(e) and rounded at 2^-24 of that, twice; the matrix cores' partial sums of
up to 256 products round at 2^-24 of what they hold, some ten times; the exponential, the terms and the last sums add
a few times 2^-24. All of them have independent signs, so that their squares add up: between 5 and 15 x 2^-24 for a
probability, and a sum over many of them is off by no more, relatively. Two terms of bfloat16 instead of three leave
2^-17 of every query element and probability at worst, a quarter of that in the square's mean: 2^-19 x (2 of the
score's size, 1) = 71 x 2^-24, which the bound tells apart (the last test, in float64).

float32 caches have no terms to tell apart, and a rounding for every product instead of one for 32: a rounding is off
by 0.41 x 2^-24 of the partial sum in the square's mean (half a step, evenly spread over a step and over the step's
octave), the partial sums of a score s grow to it about evenly, so that d of them leave 0.41 sqrt(d / 3) |s| x 2^-24:
3.8 |s| for d = 256. Positions that carry the weight have scores of about 4 (the variance of a score, by which
exp(s) shifts its mean) and up to 8: 30 x 2^-24 where those decide. Twice that for the spread of a few rows: 64."""
import math

import numpy as np
import pytest
import torch

import test_cache_ops_gpu as C
from ctranslate2_amd import _lib

BOUND = {"f32": 64 * 2.0 ** -24, "f16": 25 * 2.0 ** -24, "bf16": 25 * 2.0 ** -24}


def attention(q, k, v, visible, scale):
    """float64, all rows at once: q [.., r, d], k, v [.., n, d], visible [.., r, n] -> (out, probabilities)"""
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()) * scale
    p = torch.softmax(torch.where(visible, s, torch.full_like(s, -math.inf)), -1)
    return torch.matmul(p, v), p


def error(got, want):
    return float((got.double() - want).norm() / want.norm())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", C.TYPES)
@pytest.mark.parametrize("tokens, heads, dhead, room", [
    (4, 2, 64, 0), (4, 2, 128, 0), (4, 2, 256, 0),  # every wave loads for itself
    (20, 8, 64, 0), (20, 8, 128, 0), (40, 4, 256, 0),  # tiles shared, 16 rows a wave (but heads of 256)
    (40, 4, 64, 380000), (40, 4, 128, 380000)], ids=str)  # and 32
def test_tree_precision(gpu, dtype, tokens, heads, dhead, room):
    gen, rng = C.generator(51), np.random.default_rng(51)
    n = 2000
    k, v = C.make_cache(gen, dtype, 1, 1, room or n + tokens, dhead)
    q = torch.randn((1, tokens, heads, dhead), device="cuda", generator=gen) * 2
    seen = C.tree_mask(rng, 1, tokens)
    scale = 1 / math.sqrt(dhead)
    got = C.run_tree(q, k, v, dtype, None, n, C.to_words(seen), scale)
    visible = torch.ones((tokens, n + tokens), dtype=torch.bool, device="cuda")
    visible[:, n:] = torch.from_numpy(seen[0]).cuda()
    want, _ = attention(q[0].double().transpose(0, 1), k[0, 0, :n + tokens].double(), v[0, 0, :n + tokens].double(),
                        visible, scale)
    off = error(got[0], want.transpose(0, 1))
    print("error %.2g" % off)
    assert off <= BOUND[dtype]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", C.TYPES)
@pytest.mark.parametrize("heads, dhead", [(4, 64), (4, 128), (40, 128), (2, 256)])
def test_accumulate_precision(gpu, dtype, heads, dhead):
    gen = C.generator(52)
    n = 3000
    k, v = C.make_cache(gen, dtype, 2, 1, n, dhead)
    q = torch.randn((2, heads, dhead), device="cuda", generator=gen) * 2
    weights = torch.zeros((2, 1, n), device="cuda")
    got = C.run_accumulate(q, k, v, dtype, None, n, 1 / math.sqrt(dhead), weights)
    seen = torch.ones((2, heads, n), dtype=torch.bool, device="cuda")
    want, p = attention(q.double(), k[:, 0].double(), v[:, 0].double(), seen, 1 / math.sqrt(dhead))
    off = error(got, want), error(weights[:, 0], p.sum(1))
    print("error %.2g, weights %.2g" % off)
    assert max(off) <= BOUND[dtype]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", C.TYPES)
@pytest.mark.parametrize("heads, dhead", [(4, 64), (4, 128), (2, 256)])
def test_blocks_precision(gpu, dtype, heads, dhead):
    gen = C.generator(53)
    n, block, top = 4096, 64, 16
    k, v = C.make_cache(gen, dtype, 2, 1, n, dhead)
    q = torch.randn((2, heads, dhead), device="cuda", generator=gen) * 2
    L = _lib.lib()
    bounds = torch.zeros((2, 1, n // block, 2, dhead), dtype=k.dtype, device="cuda")
    out, selected = torch.full_like(q, 7.0), torch.zeros((2, 1, top), dtype=torch.int32, device="cuda")
    need = L.ct2x_attention_blocks_scratch_bytes(2, heads, 1, dhead, n, block, top)
    scratch = torch.full((need,), 0xA5, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    kind = C.TYPES[dtype][0]
    _lib.check(L.ct2x_cache_block_bounds(_lib.ptr(k), kind, None, None, n, 2, 1, dhead, n, block, _lib.ptr(bounds), None))
    _lib.check(L.ct2x_attention_blocks(
        _lib.ptr(q), _lib.ptr(k), _lib.ptr(v), kind, _lib.ptr(bounds), None, n, 2, heads, 1, dhead, n, block, top, 1, 2,
        1 / math.sqrt(dhead), _lib.ptr(out), _lib.ptr(selected), _lib.ptr(scratch), need, None))
    C.sync()
    seen = torch.zeros((2, n // block, block), dtype=torch.bool, device="cuda")
    seen[torch.arange(2, device="cuda")[:, None], selected[:, 0].long()] = True
    seen = seen.reshape(2, 1, n).expand(2, heads, n)
    want, _ = attention(q.double(), k[:, 0].double(), v[:, 0].double(), seen, 1 / math.sqrt(dhead))
    off = error(out, want)
    print("error %.2g" % off)
    assert off <= BOUND[dtype]


def split(x, terms):
    """x as a sum of bfloat16 values, in float64"""
    out = torch.zeros_like(x)
    for _ in range(terms):
        out += (x - out).bfloat16().double()
    return out


@pytest.mark.parametrize("rows, dhead, n", [(64, 64, 2000), (64, 128, 2000), (16, 256, 4000)])
def test_the_bound_tells_two_terms_from_three(rows, dhead, n):
    """Queries and probabilities as sums of bfloat16 terms, everything else in float64."""
    gen = torch.Generator().manual_seed(54)
    q = torch.randn((rows, dhead), generator=gen, dtype=torch.float64).float().double() * 2
    k, v = (torch.randn((n, dhead), generator=gen).bfloat16().double() for _ in range(2))
    seen = torch.ones((rows, n), dtype=torch.bool)
    want, _ = attention(q, k, v, seen, dhead ** -0.5)
    off = {}
    for terms in (2, 3):
        s = split(q, terms) @ k.T * dhead ** -0.5
        p = torch.exp(s - s.amax(1, keepdim=True))
        off[terms] = error(split(p, terms) @ v / p.sum(1, keepdim=True), want)
    print("two terms %.2g, three %.2g" % (off[2], off[3]))
    assert off[2] > BOUND["bf16"] > 8 * off[3]
