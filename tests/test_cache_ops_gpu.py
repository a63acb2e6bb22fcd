"""Attention over a serving cache and the cache's upkeep (include/ct2_mi355.h) against their formulas in
float64.

Tolerance of an attention output, per element. A score s = scale sum_d q_d k_d is off by ds: every
product and sum of fp32 rounds by at most 2^-24 relative, and the roundings are independent, so six
standard deviations of d of them are within 6 sqrt(d) 2^-24 of scale |q o k|_2 (in quadrature: each
partial sum is at most of the size of the terms' 2-norm up to sqrt(d)); a query enters the matrix cores
of a 16-bit type as three terms (bfloat16) or two (float16), each rounded to half a step, which leaves
2^-27 or 2^-22 of it; the exponent's argument s log2(e) rounds at 2^-24 |s|, twice. A probability then is off by 2 ds
relative (its own exponential and the sum's), plus the same split of the probability, plus an
exponential and n additions in fp32. So |out - exact| <= (2 ds + split + 2^-20 + 6 sqrt(n) 2^-24) sum_t p_t |v_t|.
Choices, moves and bounds are exact."""
import math

import numpy as np
import pytest
import torch

from ctranslate2_amd import _lib

pytestmark = pytest.mark.gpu

TYPES = {"f32": (0, torch.float32), "f16": (4, torch.float16), "bf16": (5, torch.bfloat16)}
SPLIT = {"f32": 0.0, "f16": 2.0 ** -22, "bf16": 2.0 ** -27}
GUARD = 64  # elements behind every output that no call may touch


def sync():
    _lib.check(_lib.lib().ct2x_stream_synchronize(None))
    torch.cuda.synchronize()


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def make_cache(gen, dtype, batch, heads_kv, t_max, dhead, behind=None):
    """behind: lengths from which the cache holds NaN"""
    out = []
    for _ in range(2):
        x = torch.randn((batch, heads_kv, t_max, dhead), device="cuda", generator=gen).to(TYPES[dtype][1])
        if behind is not None:
            for b, n in enumerate(behind):
                x[b, :, n:] = float("nan")
        out.append(x)
    return out


def to_words(seen):
    """[batch, tokens, tokens] bool -> int64 words"""
    b, t, _ = seen.shape
    n = -(-t // 64)
    bits = np.zeros((b, t, n * 64), dtype=np.uint64)
    bits[:, :, :t] = seen
    words = (bits.reshape(b, t, n, 64) << np.arange(64, dtype=np.uint64)).sum(-1, dtype=np.uint64)
    return torch.from_numpy(words.view(np.int64)).cuda()


def tree_mask(rng, batch, tokens):
    """ancestors (and self) of random trees"""
    seen = np.zeros((batch, tokens, tokens), dtype=bool)
    for b in range(batch):
        for i in range(tokens):
            parent = rng.integers(-1, i) if i else -1
            if parent >= 0:
                seen[b, i] = seen[b, parent]
            seen[b, i, i] = True
    return seen


def reference(q, k, v, visible, scale, dtype):
    """float64 softmax(scale q k^T) v of one (entry, head): q [r, d], k, v [n, d], visible [r, n]
    -> (out, tolerance, probabilities); positions that no row sees may hold anything"""
    q, k, v = q.double(), k.double(), v.double()
    n, d = k.shape
    zero = torch.zeros((), dtype=torch.float64, device="cuda")
    out, tol, probs = [], [], []
    for r in range(q.shape[0]):
        see = visible[r]
        kk = torch.where(see[:, None], k, zero)
        vv = torch.where(see[:, None], v, zero)
        if not bool(see.any()):
            out.append(torch.zeros(v.shape[1], dtype=torch.float64, device="cuda"))
            tol.append(torch.zeros_like(out[-1]))
            probs.append(torch.zeros(n, dtype=torch.float64, device="cuda"))
            continue
        s = (kk @ q[r]) * scale
        s = torch.where(see, s, torch.full_like(s, -math.inf))
        p = torch.softmax(s, 0)
        size = (kk * q[r]).norm(dim=1) * abs(scale)
        ds = (6 * math.sqrt(d) * 2.0 ** -24 + 6 * SPLIT[dtype]) * size + torch.where(see, s.abs(), zero) * 2.0 ** -23
        rel = 2 * ds[see].max() + 2 * SPLIT[dtype] + 2.0 ** -20 + 6 * math.sqrt(n) * 2.0 ** -24
        out.append(p @ vv)
        tol.append(rel * (p @ vv.abs()) + 1e-30)
        probs.append(torch.stack([p, rel * p + 1e-30]))
    return torch.stack(out), torch.stack(tol), probs


def within(got, want, tol, what=""):
    off = (got.double() - want).abs()
    bad = ~(off <= tol)
    assert not bool(bad.any()), "%s: %d of %d off, worst %.3g of its tolerance" % (
        what, int(bad.sum()), bad.numel(), float((off / tol)[bad].max()))


def run_tree(q, k, v, dtype, lengths, length, mask, scale, t_max=None, stream=None, out=None, scratch=None):
    L = _lib.lib()
    batch, tokens, heads, dhead = q.shape
    heads_kv, t_max = k.shape[1], t_max or k.shape[2]
    need = L.ct2x_attention_tree_scratch_bytes(batch, tokens, heads, heads_kv, dhead, t_max)
    assert need >= 0
    if scratch is None:
        scratch = torch.full((max(need, 16),), 0xA5, dtype=torch.uint8, device="cuda")
    if out is None:
        out = torch.full((q.numel() + GUARD,), 7.0, device="cuda")
    torch.cuda.synchronize()
    _lib.check(L.ct2x_attention_tree(
        _lib.ptr(q), _lib.ptr(k), _lib.ptr(v), TYPES[dtype][0], _lib.ptr(lengths), length, _lib.ptr(mask), batch,
        tokens, heads, heads_kv, dhead, t_max, scale, _lib.ptr(out), _lib.ptr(scratch), need, stream))
    if stream is None:
        sync()
    assert bool((out[q.numel():] == 7.0).all()) or stream is not None
    return out[:q.numel()].reshape(q.shape)


def check_tree(got, q, k, v, dtype, lengths, seen, scale, entries=None):
    batch, tokens, heads, dhead = q.shape
    group = heads // k.shape[1]
    for b in entries if entries is not None else range(batch):
        n = lengths[b]
        visible = torch.ones((tokens, n + tokens), dtype=torch.bool, device="cuda")
        visible[:, n:] = torch.from_numpy(np.ascontiguousarray(seen[b])).cuda()
        for h in range(heads):
            want, tol, _ = reference(q[b, :, h], k[b, h // group, :n + tokens], v[b, h // group, :n + tokens], visible,
                                     scale, dtype)
            within(got[b, :, h], want, tol, "entry %d head %d" % (b, h))


TREES = [
    # batch, tokens, heads, heads_kv, dhead, lengths, room behind
    (1, 1, 1, 1, 8, [0], 0),
    (1, 1, 4, 1, 64, [1], 3),
    (2, 5, 8, 8, 64, [150, 31], 9),
    (3, 7, 8, 2, 128, [0, 33, 257], 1),
    (2, 16, 6, 3, 80, [100, 15], 2),
    (2, 17, 8, 1, 72, [64, 63], 5),
    (1, 33, 4, 4, 200, [700], 0),
    (2, 65, 4, 2, 128, [130, 1], 7),
    (1, 130, 2, 1, 256, [40], 0),
    (1, 3, 71, 1, 64, [90], 4),
    (1, 64, 8, 2, 128, [1500], 11),
    (1, 2, 2, 1, 96, [4097], 5),
    (1, 600, 4, 1, 64, [100], 3),
    (150, 2, 2, 1, 32, [1 + 13 * (i % 7) * (i % 11) for i in range(150)], 2),  # more entries than lanes
    (300, 1, 8, 8, 16, [i % 5 for i in range(300)], 1),  # more units than the line takes
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", TREES, ids=str)
def test_tree(gpu, dtype, shape):
    batch, tokens, heads, heads_kv, dhead, lengths, room = shape
    gen, rng = generator(1), np.random.default_rng(1)
    t_max = max(lengths) + tokens + room
    k, v = make_cache(gen, dtype, batch, heads_kv, t_max, dhead, [n + tokens for n in lengths])
    q = torch.randn((batch, tokens, heads, dhead), device="cuda", generator=gen) * 2
    seen = tree_mask(rng, batch, tokens)
    scale = 1 / math.sqrt(dhead)
    got = run_tree(q, k, v, dtype, torch.tensor(lengths, dtype=torch.int32, device="cuda"), 0, to_words(seen), scale)
    check_tree(got, q, k, v, dtype, lengths, seen, scale)


@pytest.mark.parametrize("dtype", TYPES)
def test_tree_any_mask_and_empty_rows(gpu, dtype):
    """Rows that see nothing, only a later token, or everything; entries without committed positions."""
    gen, rng = generator(2), np.random.default_rng(2)
    batch, tokens, heads, heads_kv, dhead = 3, 70, 4, 2, 64
    lengths = [0, 5, 0]
    k, v = make_cache(gen, dtype, batch, heads_kv, 80, dhead, [n + tokens for n in lengths])
    q = torch.randn((batch, tokens, heads, dhead), device="cuda", generator=gen)
    seen = rng.random((batch, tokens, tokens)) < 0.1
    seen[0, 3] = seen[0, 69] = seen[1, 4] = False
    seen[0, 5] = False
    seen[0, 5, 66] = True
    seen[1, 7] = True
    seen[2] = False
    got = run_tree(q, k, v, dtype, torch.tensor(lengths, dtype=torch.int32, device="cuda"), 0, to_words(seen), 0.125)
    check_tree(got, q, k, v, dtype, lengths, seen, 0.125)
    assert bool((got[0, 3] == 0).all()) and bool((got[2] == 0).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens, heads", [(9, 2), (40, 8)])
def test_tree_masked_drafts_may_hold_anything(gpu, dtype, tokens, heads):
    """Drafted tokens with NaN and infinite keys and values: rows that do not see them are untouched."""
    gen, rng = generator(3), np.random.default_rng(3)
    n, dhead = 50, 64
    k, v = make_cache(gen, dtype, 1, 1, n + tokens, dhead)
    q = torch.randn((1, tokens, heads, dhead), device="cuda", generator=gen)
    seen = tree_mask(rng, 1, tokens)
    seen[0, :, 2] = seen[0, :, 6] = False
    k[0, 0, n + 2], v[0, 0, n + 2] = float("nan"), float("inf")
    k[0, 0, n + 6], v[0, 0, n + 6] = float("-inf"), float("nan")
    words = to_words(seen)
    got = run_tree(q, k, v, dtype, None, n, words, 0.125)
    check_tree(got, q, k, v, dtype, [n], seen, 0.125)
    # one row that does see them: it alone is not finite
    seen[0, 4, 6] = True
    got = run_tree(q, k, v, dtype, None, n, to_words(seen), 0.125)
    assert not bool(torch.isfinite(got[0, 4]).any())
    rows = [i for i in range(tokens) if i != 4]
    assert bool(torch.isfinite(got[0, rows]).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_tree_chain_and_clamped_lengths(gpu, dtype):
    """No mask: token j <= i. Lengths beyond the cache's room, and negative ones, are clamped."""
    gen = generator(4)
    batch, tokens, heads, heads_kv, dhead, t_max = 3, 20, 4, 2, 128, 90
    k, v = make_cache(gen, dtype, batch, heads_kv, t_max, dhead)
    q = torch.randn((batch, tokens, heads, dhead), device="cuda", generator=gen)
    seen = np.tril(np.ones((batch, tokens, tokens), dtype=bool))
    given = torch.tensor([1000, -3, 70], dtype=torch.int32, device="cuda")
    got = run_tree(q, k, v, dtype, given, 0, None, 0.1)
    check_tree(got, q, k, v, dtype, [70, 0, 70], seen, 0.1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", (1e-20, 1e20), ids=("small", "large"))
def test_tree_queries_of_any_size(gpu, dtype, size):
    """Queries outside float16's range: the scale brings the scores back."""
    gen = generator(5)
    k, v = make_cache(gen, dtype, 1, 1, 300, 64)
    q = torch.randn((1, 4, 2, 64), device="cuda", generator=gen) * size
    q[0, 1] = 0  # equal scores everywhere
    seen = np.tril(np.ones((1, 4, 4), dtype=bool))
    got = run_tree(q, k, v, dtype, None, 290, None, 0.125 / size)
    check_tree(got, q, k, v, dtype, [290], seen, 0.125 / size)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", (3, 40))
@pytest.mark.parametrize("scale", (0.0, -0.3))
def test_tree_scales(gpu, dtype, tokens, scale):
    """Scale zero weighs all that is seen alike, a negative one turns the order round."""
    gen, rng = generator(8), np.random.default_rng(8)
    k, v = make_cache(gen, dtype, 1, 1, 400, 64)
    q = torch.randn((1, tokens, 2, 64), device="cuda", generator=gen)
    seen = tree_mask(rng, 1, tokens)
    got = run_tree(q, k, v, dtype, None, 333, to_words(seen), scale)
    check_tree(got, q, k, v, dtype, [333], seen, scale)


@pytest.mark.parametrize("dtype", TYPES)
def test_tree_peaked_rows(gpu, dtype):
    """One key far above the others (a sink), early or late; the rest must not be lost or doubled."""
    gen = generator(6)
    k, v = make_cache(gen, dtype, 2, 2, 2100, 128)
    q = torch.randn((2, 3, 4, 128), device="cuda", generator=gen)
    for b, at in ((0, 3), (1, 2047)):
        for g in range(2):
            k[b, g, at] = (q[b, 0, 2 * g] * 3).to(k.dtype)
    seen = np.tril(np.ones((2, 3, 3), dtype=bool))
    got = run_tree(q, k, v, dtype, None, 2090, None, 128 ** -0.5)
    check_tree(got, q, k, v, dtype, [2090, 2090], seen, 128 ** -0.5)


def test_tree_offsets_beyond_32_bits(gpu):
    """A cache of more than 2^32 bytes and 2^31 elements: the last entry's rows."""
    gen = generator(7)
    batch, heads_kv, t_max, dhead, tokens = 3, 8, 700000, 128, 3  # 2.15e9 elements, 4.3 GB each
    k = torch.zeros((batch, heads_kv, t_max, dhead), dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    lengths = [2, 0, t_max - tokens]
    for x in (k, v):
        x[2, 7].normal_(generator=gen)
        x[0, :, :8].normal_(generator=gen)
    q = torch.randn((batch, tokens, 8, dhead), device="cuda", generator=gen) * 2
    seen = np.tril(np.ones((batch, tokens, tokens), dtype=bool))
    got = run_tree(q, k, v, "bf16", torch.tensor(lengths, dtype=torch.int32, device="cuda"), 0, None, 128 ** -0.5)
    check_tree(got[:, :, 7:], q[:, :, 7:], k[:, 7:], v[:, 7:], "bf16", lengths, seen, 128 ** -0.5, entries=(0, 2))


def run_accumulate(q, k, v, dtype, lengths, length, scale, weights, stream=None, out=None, scratch=None):
    L = _lib.lib()
    batch, heads, dhead = q.shape
    heads_kv, t_max = k.shape[1:3]
    need = L.ct2x_attention_accumulate_scratch_bytes(batch, heads, heads_kv, dhead, t_max)
    if scratch is None:
        scratch = torch.full((need,), 0xA5, dtype=torch.uint8, device="cuda")
    if out is None:
        out = torch.full((q.numel() + GUARD,), 7.0, device="cuda")
    torch.cuda.synchronize()
    _lib.check(L.ct2x_attention_accumulate(
        _lib.ptr(q), _lib.ptr(k), _lib.ptr(v), TYPES[dtype][0], _lib.ptr(lengths), length, batch, heads, heads_kv,
        dhead, t_max, scale, _lib.ptr(weights), _lib.ptr(out), _lib.ptr(scratch), need, stream))
    if stream is None:
        sync()
        assert bool((out[q.numel():] == 7.0).all())
    return out[:q.numel()].reshape(q.shape)


ACCUMULATE = [
    (1, 1, 1, 8, [0]), (2, 8, 8, 64, [1, 333]), (3, 8, 2, 128, [0, 65, 1000]), (2, 20, 4, 80, [77, 500]),
    (1, 71, 1, 64, [130]), (1, 16, 16, 256, [300]), (1, 4, 2, 128, [9000]), (5, 4, 1, 96, [31, 32, 33, 64, 1]),
    (130, 2, 1, 16, [i % 9 * 40 for i in range(130)]), (260, 8, 8, 8, [i % 4 * 7 for i in range(260)]),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", ACCUMULATE, ids=str)
def test_accumulate(gpu, dtype, shape):
    batch, heads, heads_kv, dhead, lengths = shape
    gen = generator(11)
    t_max, group = max(lengths) + 13, heads // heads_kv
    k, v = make_cache(gen, dtype, batch, heads_kv, t_max, dhead, lengths)
    q = torch.randn((batch, heads, dhead), device="cuda", generator=gen) * 2
    before = torch.rand((batch, heads_kv, t_max), device="cuda", generator=gen)
    for b, n in enumerate(lengths):
        before[b, :, n:] = float("nan")
    weights = before.clone()
    given = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    scale = 1 / math.sqrt(dhead)
    want, slack = before.double(), torch.zeros_like(before, dtype=torch.float64)
    for call in range(2):
        got = run_accumulate(q, k, v, dtype, given, 0, scale, weights)
        for b, n in enumerate(lengths):
            see = torch.ones((1, n), dtype=torch.bool, device="cuda")
            for h in range(heads):
                o, tol, p = reference(q[b, h][None], k[b, h // group, :n], v[b, h // group, :n], see, scale, dtype)
                within(got[b, h][None], o, tol, "entry %d head %d" % (b, h))
                if n:
                    want[b, h // group, :n] += p[0][0]
                    slack[b, h // group, :n] += p[0][1]
        slack += want.nan_to_num() * (group + 1) * 2.0 ** -24
        for b, n in enumerate(lengths):
            within(weights[b, :, :n], want[b, :, :n], slack[b, :, :n] + 1e-30, "weights of entry %d" % b)
            assert bool(weights[b, :, n:].isnan().all())


def evict_reference(weights, n, budget, recent):
    if n <= budget:
        return list(range(n))
    old = n - recent
    w = [float(x) for x in weights[:old]]
    order = sorted(range(old), key=lambda i: (not math.isnan(w[i]), 0.0 if math.isnan(w[i]) else -w[i], i))
    return sorted(order[:budget - recent]) + list(range(old, n))


def run_evict(k, v, w, dtype, lengths, length, budget, recent, k_out, v_out, w_out, lengths_out, stream=None):
    L = _lib.lib()
    batch, heads_kv, t_max, dhead = k.shape
    positions = torch.full((batch * heads_kv * budget + GUARD,), 12345, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    _lib.check(L.ct2x_cache_evict(
        _lib.ptr(k), _lib.ptr(v), TYPES[dtype][0], _lib.ptr(w), _lib.ptr(lengths), length, batch, heads_kv, dhead,
        t_max, budget, recent, k_out.shape[2], _lib.ptr(k_out), _lib.ptr(v_out), _lib.ptr(w_out),
        _lib.ptr(positions), _lib.ptr(lengths_out), stream))
    if stream is None:
        sync()
        assert bool((positions[-GUARD:] == 12345).all())
    return positions[:-GUARD].reshape(batch, heads_kv, budget)


EVICT = [
    # batch, heads_kv, dhead, lengths, t_max, budget, recent, room behind the budget
    (1, 1, 8, [1], 1, 1, 0, 0),
    (2, 2, 64, [0, 40], 50, 16, 4, 3),
    (3, 3, 80, [500, 64, 65], 511, 64, 64, 0),
    (2, 2, 128, [1025, 3000], 3001, 1000, 0, 24),
    (1, 4, 200, [700], 700, 699, 1, 0),
    (1, 1, 256, [5000], 5003, 1, 1, 0),
    (2, 1, 128, [4096, 2000], 4100, 4096, 10, 4),
    (1, 2, 64, [70001], 70001, 33333, 333, 0),
]


def make_weights(gen, batch, heads_kv, t_max):
    w = torch.empty((batch, heads_kv, t_max), device="cuda").exponential_(generator=gen)
    w = (w * 16).round() / 16  # many equal ones
    w[torch.rand(w.shape, device="cuda", generator=gen) < 0.05] = -0.0
    w[torch.rand(w.shape, device="cuda", generator=gen) < 0.01] = float("nan")
    w[torch.rand(w.shape, device="cuda", generator=gen) < 0.01] = float("inf")
    w[torch.rand(w.shape, device="cuda", generator=gen) < 0.01] = -1.5
    return w


@pytest.mark.parametrize("in_place", (False, True), ids=("apart", "in_place"))
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", EVICT, ids=str)
def test_evict(gpu, dtype, shape, in_place):
    batch, heads_kv, dhead, lengths, t_max, budget, recent, room = shape
    gen = generator(21)
    k, v = make_cache(gen, dtype, batch, heads_kv, t_max, dhead)
    w = make_weights(gen, batch, heads_kv, t_max)
    given = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    k0, v0, w0 = k.clone(), v.clone(), w.clone()
    if in_place:
        if budget > t_max:
            pytest.skip("an output in place has the input's room")
        k_out, v_out, w_out, n_out = k, v, w, given
    else:
        k_out = torch.full((batch, heads_kv, budget + room, dhead), 3.0, dtype=k.dtype, device="cuda")
        v_out, w_out = k_out.clone(), torch.full((batch, heads_kv, budget + room), 3.0, device="cuda")
        n_out = torch.full((batch,), -7, dtype=torch.int32, device="cuda")
    k1, v1, w1 = k_out.clone(), v_out.clone(), w_out.clone()
    positions = run_evict(k, v, w, dtype, given, 0, budget, recent, k_out, v_out, w_out, n_out)
    assert n_out.tolist() == [min(n, budget) for n in lengths]
    host = w0.cpu().numpy()
    for b, n in enumerate(lengths):
        for h in range(heads_kv):
            keep = evict_reference(host[b, h], n, budget, recent)
            m = len(keep)
            assert positions[b, h].tolist() == keep + [-1] * (budget - m), (b, h)
            at = torch.tensor(keep, dtype=torch.long, device="cuda")
            for out, was, old in ((k_out, k1, k0), (v_out, v1, v0), (w_out, w1, w0)):
                same = torch.cat([old[b, h, at], was[b, h, m:]])
                assert torch.equal(out[b, h].view(torch.int16), same.view(torch.int16)), (b, h)


def run_bounds(k, dtype, first, lengths, length, block, bounds, stream=None):
    batch, heads_kv, t_max, dhead = k.shape
    torch.cuda.synchronize()
    _lib.check(_lib.lib().ct2x_cache_block_bounds(
        _lib.ptr(k), TYPES[dtype][0], _lib.ptr(first), _lib.ptr(lengths), length, batch, heads_kv, dhead, t_max, block,
        _lib.ptr(bounds), stream))
    if stream is None:
        sync()


BOUNDS = [
    # batch, heads_kv, dhead, t_max, block, first, lengths
    (1, 1, 8, 1, 16, None, [1]),
    (2, 2, 64, 100, 16, None, [0, 99]),
    (3, 2, 128, 257, 64, [0, 64, 200], [257, 65, 201]),
    (2, 3, 80, 1000, 48, [999, 5], [1000, 3]),
    (2, 1, 256, 513, 256, [-4, 512], [512, 513]),
    (1, 5, 200, 2000, 128, [100], [1777]),
    (1, 8, 128, 5000, 32, None, [5000]),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", BOUNDS, ids=str)
def test_block_bounds(gpu, dtype, shape):
    batch, heads_kv, dhead, t_max, block, first, lengths = shape
    gen = generator(31)
    k, _ = make_cache(gen, dtype, batch, heads_kv, t_max, dhead, lengths)
    hurt = torch.rand((batch, heads_kv, t_max), device="cuda", generator=gen)
    k[..., 3][hurt < 0.02] = float("nan")
    k[..., 5][hurt > 0.98] = float("-inf")
    blocks = -(-t_max // block)
    bounds = torch.full((batch, heads_kv, blocks, 2, dhead), 3.0, dtype=k.dtype, device="cuda")
    want = bounds.clone()
    for b, n in enumerate(lengths):
        for j in range(max(0, first[b] if first else 0) // block, -(-n // block)):
            rows = k[b, :, j * block:min(n, (j + 1) * block)].float()  # amin / amax hand on a NaN
            want[b, :, j, 0], want[b, :, j, 1] = rows.amin(1).to(k.dtype), rows.amax(1).to(k.dtype)
    given = [None if x is None else torch.tensor(x, dtype=torch.int32, device="cuda") for x in (first, lengths)]
    run_bounds(k, dtype, given[0], given[1], 0, block, bounds)
    assert torch.equal(torch.nan_to_num(bounds.float(), 99.0), torch.nan_to_num(want.float(), 99.0))
    if first is None:  # the scalar length
        again = torch.full_like(bounds, 3.0)
        run_bounds(k[:1], dtype, None, None, lengths[0], block, again[:1])
        assert torch.equal(torch.nan_to_num(again[:1].float(), 99.0), torch.nan_to_num(want[:1].float(), 99.0))
        assert bool((again[1:] == 3.0).all())


def run_blocks(q, k, v, dtype, bounds, lengths, length, block, top, sink, local, scale, want_selected=True,
               stream=None, out=None, scratch=None):
    L = _lib.lib()
    batch, heads, dhead = q.shape
    heads_kv, t_max = k.shape[1:3]
    need = L.ct2x_attention_blocks_scratch_bytes(batch, heads, heads_kv, dhead, t_max, block, top)
    assert need > 0
    if scratch is None:
        scratch = torch.full((need,), 0xA5, dtype=torch.uint8, device="cuda")
    if out is None:
        out = torch.full((q.numel() + GUARD,), 7.0, device="cuda")
    selected = torch.full((batch * heads_kv * top + GUARD,), 777, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    _lib.check(L.ct2x_attention_blocks(
        _lib.ptr(q), _lib.ptr(k), _lib.ptr(v), TYPES[dtype][0], _lib.ptr(bounds), _lib.ptr(lengths), length, batch,
        heads, heads_kv, dhead, t_max, block, top, sink, local, scale, _lib.ptr(out),
        _lib.ptr(selected) if want_selected else None, _lib.ptr(scratch), need, stream))
    if stream is None:
        sync()
        assert bool((out[q.numel():] == 7.0).all()) and bool((selected[-GUARD:] == 777).all())
    return out[:q.numel()].reshape(q.shape), selected[:-GUARD].reshape(batch, heads_kv, top)


def select_reference(q, bounds, n, block, top, sink, local):
    """q [group, d], bounds [blocks, 2, d] -> the blocks taken"""
    count = -(-n // block)
    low, high = bounds[:count, 0].double(), bounds[:count, 1].double()
    x = torch.stack([torch.maximum(one.double() * low, one.double() * high).sum(1) for one in q]).amax(0).tolist()
    always = [j for j in range(count) if j < sink or j >= count - local]
    others = [j for j in range(count) if j not in always]
    others.sort(key=lambda j: (not math.isnan(x[j]), 0.0 if math.isnan(x[j]) else -x[j], j))
    return sorted(always + others[:max(0, top - len(always))])


BLOCKS = [
    # batch, heads, heads_kv, dhead, t_max, block, top, sink, local, lengths
    (1, 1, 1, 8, 1, 16, 1, 0, 0, [1]),
    (2, 8, 8, 64, 400, 16, 5, 1, 2, [0, 399]),
    (3, 8, 2, 128, 1000, 64, 4, 1, 1, [1000, 250, 64]),
    (2, 20, 4, 80, 900, 48, 7, 0, 1, [900, 335]),
    (1, 71, 1, 64, 600, 32, 6, 0, 0, [555]),
    (1, 4, 2, 256, 2000, 256, 3, 1, 1, [1801]),
    (2, 4, 1, 96, 3000, 16, 40, 2, 3, [2999, 17]),
    (1, 8, 2, 128, 20000, 16, 300, 1, 2, [19999]),
    (1, 2, 2, 200, 300, 32, 64, 4, 4, [300]),
    (1, 2, 1, 8, 300000, 16, 5, 1, 1, [299990]),  # more blocks than the selection keeps in registers
    (90, 4, 1, 16, 400, 16, 6, 1, 1, [i % 10 * 40 for i in range(90)]),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", BLOCKS, ids=str)
def test_blocks(gpu, dtype, shape):
    batch, heads, heads_kv, dhead, t_max, block, top, sink, local, lengths = shape
    gen = generator(41)
    group = heads // heads_kv
    k, v = make_cache(gen, dtype, batch, heads_kv, t_max, dhead, lengths)
    q = torch.randn((batch, heads, dhead), device="cuda", generator=gen) * 2
    given = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    bounds = torch.full((batch, heads_kv, -(-t_max // block), 2, dhead), float("nan"), dtype=k.dtype, device="cuda")
    run_bounds(k, dtype, None, given, 0, block, bounds)
    scale = 1 / math.sqrt(dhead)
    got, selected = run_blocks(q, k, v, dtype, bounds, given, 0, block, top, sink, local, scale)
    for b, n in enumerate(lengths):
        for g in range(heads_kv):
            rows = q[b, g * group:(g + 1) * group]
            keep = select_reference(rows, bounds[b, g], n, block, top, sink, local)
            assert selected[b, g].tolist() == keep + [-1] * (top - len(keep)), (b, g)
            see = torch.zeros((group, n), dtype=torch.bool, device="cuda")
            for j in keep:
                see[:, j * block:(j + 1) * block] = True
            want, tol, _ = reference(rows, k[b, g, :n], v[b, g, :n], see, scale, dtype)
            within(got[b, g * group:(g + 1) * group], want, tol, "entry %d group %d" % (b, g))
    again, untouched = run_blocks(q, k, v, dtype, bounds, given, 0, block, top, sink, local, scale, False)
    assert torch.equal(got, again) and bool((untouched == 777).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_blocks_ties_and_nan_bounds(gpu, dtype):
    """Equal blocks go to the lowest; a block with a NaN bound is taken first; unselected blocks may hold anything."""
    gen = generator(42)
    block, n, dhead = 16, 16 * 40, 64
    k, v = make_cache(gen, dtype, 1, 1, n, dhead)
    k[0, 0] = k[0, 0, :block].repeat(40, 1)
    q = torch.randn((1, 2, dhead), device="cuda", generator=gen)
    bounds = torch.empty((1, 1, 40, 2, dhead), dtype=k.dtype, device="cuda")
    run_bounds(k, dtype, None, None, n, block, bounds)
    bounds[0, 0, 23, 0, 7] = float("nan")
    k[0, 0, 16 * 20:16 * 23], v[0, 0, 16 * 20:16 * 23] = float("nan"), float("inf")
    got, selected = run_blocks(q, k, v, dtype, bounds, None, n, block, 9, 1, 2, 0.125)
    assert selected[0, 0].tolist() == [0, 1, 2, 3, 4, 5, 23, 38, 39]
    see = torch.zeros((2, n), dtype=torch.bool, device="cuda")
    for j in selected[0, 0].tolist():
        see[:, j * block:(j + 1) * block] = True
    want, tol, _ = reference(q[0], k[0, 0], v[0, 0], see, 0.125, dtype)
    within(got[0], want, tol)


@pytest.mark.parametrize("dtype", TYPES)
def test_blocks_infinite_bounds(gpu, dtype):
    """Infinite keys bound by infinity: taken first where a query leans to them, last where it leans away."""
    gen = generator(44)
    block, dhead = 16, 64
    n = block * 30
    k, v = make_cache(gen, dtype, 1, 1, n, dhead)
    k[0, 0, 16 * 7 + 3, 5] = float("inf")
    k[0, 0, 16 * 11:16 * 12, 6] = float("-inf")
    q = torch.randn((1, 3, dhead), device="cuda", generator=gen)
    q[0, :, 5] = 1.0
    q[0, :, 6] = 1.0
    q[0, 2, 5] = -1.0
    bounds = torch.empty((1, 1, 30, 2, dhead), dtype=k.dtype, device="cuda")
    run_bounds(k, dtype, None, None, n, block, bounds)
    _, selected = run_blocks(q, k, v, dtype, bounds, None, n, block, 12, 0, 0, 0.125)
    keep = select_reference(q[0], bounds[0, 0], n, block, 12, 0, 0)
    assert selected[0, 0].tolist() == keep and 7 in keep and 11 not in keep


@pytest.mark.parametrize("dtype", TYPES)
def test_every_view_agrees_where_it_shows_the_same(gpu, dtype):
    """A tree of one token, the accumulating attention and enough blocks see the same positions."""
    gen = generator(43)
    n, block = 700, 32
    k, v = make_cache(gen, dtype, 2, 2, n + 1, 128)
    q = torch.randn((2, 8, 128), device="cuda", generator=gen)
    weights = torch.zeros((2, 2, n + 1), device="cuda")
    dense = run_accumulate(q, k, v, dtype, None, n, 0.09, weights)
    bounds = torch.empty((2, 2, -(-(n + 1) // block), 2, 128), dtype=k.dtype, device="cuda")
    run_bounds(k, dtype, None, None, n, block, bounds)
    sparse, _ = run_blocks(q, k, v, dtype, bounds, None, n, block, 22, 1, 1, 0.09)
    tree = run_tree(q[:, None], k, v, dtype, None, n, to_words(np.zeros((2, 1, 1), dtype=bool)), 0.09)
    see = torch.ones((4, n), dtype=torch.bool, device="cuda")
    for got in (dense, sparse, tree[:, 0]):
        for b in range(2):
            for g in range(2):
                want, tol, _ = reference(q[b, 4 * g:4 * g + 4], k[b, g, :n], v[b, g, :n], see, 0.09, dtype)
                within(got[b, 4 * g:4 * g + 4], want, tol)
    assert torch.allclose(weights[:, :, :n].sum(2), torch.full((2, 2), 4.0, device="cuda"), rtol=1e-4)


class Session:
    """A serving loop's state: cache, weights, bounds, lengths - and one step over them by every operator."""

    def __init__(self, dtype, seed):
        gen = generator(seed)
        self.dtype, self.block, self.budget = dtype, 16, 200
        self.lengths = torch.tensor([333, 90], dtype=torch.int32, device="cuda")
        self.k, self.v = make_cache(gen, dtype, 2, 2, 360, 64)
        self.weights = torch.zeros((2, 2, 360), device="cuda")
        self.bounds = torch.zeros((2, 2, 23, 2, 64), dtype=self.k.dtype, device="cuda")
        self.q = torch.randn((2, 8, 64), device="cuda", generator=gen)
        self.drafts = torch.randn((2, 5, 8, 64), device="cuda", generator=gen)
        self.mask = to_words(tree_mask(np.random.default_rng(seed), 2, 5))
        L = _lib.lib()
        self.scratch = torch.empty(max(L.ct2x_attention_tree_scratch_bytes(2, 5, 8, 2, 64, 360),
                                       L.ct2x_attention_accumulate_scratch_bytes(2, 8, 2, 64, 360),
                                       L.ct2x_attention_blocks_scratch_bytes(2, 8, 2, 64, 360, 16, 6)),
                                   dtype=torch.uint8, device="cuda")
        self.out = [torch.zeros_like(self.q), torch.zeros_like(self.drafts), torch.zeros_like(self.q)]
        self.positions = torch.zeros((2, 2, 200), dtype=torch.int32, device="cuda")
        self.selected = torch.zeros((2, 2, 6), dtype=torch.int32, device="cuda")
        self.start = [x.clone() for x in (self.k, self.v, self.weights, self.bounds, self.lengths)]

    def restore(self):
        for x, y in zip((self.k, self.v, self.weights, self.bounds, self.lengths), self.start):
            x.copy_(y)

    def step(self, stream):
        L, p, t = _lib.lib(), _lib.ptr, TYPES[self.dtype][0]
        n = self.scratch.numel()
        _lib.check(L.ct2x_attention_accumulate(p(self.q), p(self.k), p(self.v), t, p(self.lengths), 0, 2, 8, 2, 64, 360,
                                               0.125, p(self.weights), p(self.out[0]), p(self.scratch), n, stream))
        _lib.check(L.ct2x_cache_evict(p(self.k), p(self.v), t, p(self.weights), p(self.lengths), 0, 2, 2, 64, 360, 200,
                                      20, 360, p(self.k), p(self.v), p(self.weights), p(self.positions),
                                      p(self.lengths), stream))
        _lib.check(L.ct2x_cache_block_bounds(p(self.k), t, None, p(self.lengths), 0, 2, 2, 64, 360, 16, p(self.bounds),
                                             stream))
        _lib.check(L.ct2x_attention_tree(p(self.drafts), p(self.k), p(self.v), t, p(self.lengths), 0, p(self.mask), 2, 5,
                                         8, 2, 64, 360, 0.125, p(self.out[1]), p(self.scratch), n, stream))
        _lib.check(L.ct2x_attention_blocks(p(self.q), p(self.k), p(self.v), t, p(self.bounds), p(self.lengths), 0, 2, 8,
                                           2, 64, 360, 16, 6, 1, 2, 0.125, p(self.out[2]), p(self.selected),
                                           p(self.scratch), n, stream))

    def results(self):
        torch.cuda.synchronize()
        return [x.clone() for x in (*self.out, self.weights, self.bounds, self.positions, self.selected, self.lengths,
                                    self.k, self.v)]


def same(a, b):
    return all(torch.equal(x.contiguous().view(torch.uint8), y.contiguous().view(torch.uint8)) for x, y in zip(a, b))


@pytest.mark.parametrize("dtype", TYPES)
def test_a_step_of_all_operators(gpu, dtype):
    s = Session(dtype, 51)
    k0, v0 = s.start[0], s.start[1]
    torch.cuda.synchronize()
    s.step(None)
    sync()
    got = s.results()
    assert s.lengths.tolist() == [200, 90]
    # the cache after eviction, by the weights that the step itself accumulated
    kept = []
    for b, n in enumerate((333, 90)):
        for g in range(2):
            see = torch.ones((4, n), dtype=torch.bool, device="cuda")
            want, tol, probs = reference(s.q[b, 4 * g:4 * g + 4], k0[b, g, :n], v0[b, g, :n], see, 0.125, dtype)
            within(got[0][b, 4 * g:4 * g + 4], want, tol)
            keep = s.positions[b, g, :min(n, 200)].long()
            assert torch.equal(s.k[b, g, :len(keep)], k0[b, g, keep])
            w = torch.stack([x[0] for x in probs]).sum(0)
            if n > 200:  # what stayed weighs at least as much as what left, up to the weights' own error
                gone = torch.ones(n, dtype=torch.bool, device="cuda")
                gone[keep] = False
                assert float(w[keep[:180]].min()) >= float(w[gone].max()) * (1 - 1e-4)
            kept.append(keep)
    lengths = [200, 90]
    seen = tree_mask(np.random.default_rng(51), 2, 5)
    check_tree(got[1], s.drafts, s.k, s.v, dtype, lengths, seen, 0.125)
    for b, n in enumerate(lengths):
        for g in range(2):
            rows = s.q[b, 4 * g:4 * g + 4]
            keep = select_reference(rows, s.bounds[b, g], n, 16, 6, 1, 2)
            assert s.selected[b, g].tolist() == keep
            see = torch.zeros((4, n), dtype=torch.bool, device="cuda")
            for j in keep:
                see[:, j * 16:(j + 1) * 16] = True
            want, tol, _ = reference(rows, s.k[b, g, :n], s.v[b, g, :n], see, 0.125, dtype)
            within(got[2][b, 4 * g:4 * g + 4], want, tol)


@pytest.mark.parametrize("dtype", TYPES)
def test_captured_steps_and_other_streams(gpu, dtype):
    """Two sessions that share nothing but their sizes, captured into a graph each and replayed in turn with
    eager steps between; every replay gives the eager step's bits."""
    sessions = [Session(dtype, 61), Session(dtype, 62)]
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    eager = []
    for s in sessions:
        s.step(stream.cuda_stream)
        eager.append(s.results())
    graphs = []
    for s in sessions:
        s.restore()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            s.step(torch.cuda.current_stream().cuda_stream)
        graphs.append(graph)
    for turn in range(4):
        for s, graph, want in zip(sessions, graphs, eager):
            s.restore()
            for x in s.out:
                x.fill_(9.0)
            torch.cuda.synchronize()
            graph.replay()
            assert same(s.results(), want), "replay %d" % turn
        # an eager step of the first session on the library's own stream between the replays
        sessions[0].restore()
        torch.cuda.synchronize()
        sessions[0].step(None)
        sync()
        assert same(sessions[0].results(), eager[0])


@pytest.mark.parametrize("dtype", ("bf16", "f32"))
def test_two_calls_at_once(gpu, dtype):
    """Two streams, a scratch each: the results of one alone."""
    sessions = [Session(dtype, 71), Session(dtype, 72)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    want = []
    for s in sessions:
        s.step(None)
        sync()
        want.append(s.results())
    for turn in range(5):
        for s in sessions:
            s.restore()
        torch.cuda.synchronize()
        for s, stream in zip(sessions, streams):
            s.step(stream.cuda_stream)
        torch.cuda.synchronize()
        for s, w in zip(sessions, want):
            assert same(s.results(), w), "turn %d" % turn


def test_repeated_calls_give_the_same_bits(gpu):
    gen = generator(81)
    k, v = make_cache(gen, "bf16", 4, 2, 3100, 128)
    q = torch.randn((4, 30, 8, 128), device="cuda", generator=gen)
    lengths = torch.tensor([3070, 1500, 10, 2222], dtype=torch.int32, device="cuda")
    first = run_tree(q, k, v, "bf16", lengths, 0, None, 0.09).clone()
    for _ in range(5):
        assert torch.equal(first, run_tree(q, k, v, "bf16", lengths, 0, None, 0.09))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("batch", (24, 65))
def test_many_units_of_several_rounds(gpu, dtype, batch):
    """Enough (entry, head) units that a workgroup takes one from end to end, over several rounds and
    lengths that end inside them; every view, a sample of the entries."""
    gen, rng = generator(91), np.random.default_rng(91)
    heads, heads_kv, dhead, t_max, scale = 16, 8, 64, 640, 0.125
    lengths = [int(rng.integers(0, 600)) for _ in range(batch)]
    lengths[:3] = [600, 0, 1]
    sample = (0, 1, 2, batch // 2, batch - 1)
    given = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    for tokens in (3, 20):
        k, v = make_cache(gen, dtype, batch, heads_kv, t_max, dhead, [n + tokens for n in lengths])
        q = torch.randn((batch, tokens, heads, dhead), device="cuda", generator=gen) * 2
        seen = tree_mask(rng, batch, tokens)
        got = run_tree(q, k, v, dtype, given, 0, to_words(seen), scale)
        check_tree(got, q, k, v, dtype, lengths, seen, scale, sample)
    k, v = make_cache(gen, dtype, batch, heads_kv, 270, dhead, [min(n, 270) for n in lengths])
    q = torch.randn((batch, heads, dhead), device="cuda", generator=gen) * 2
    weights = torch.zeros((batch, heads_kv, 270), device="cuda")
    got = run_accumulate(q, k, v, dtype, given, 0, scale, weights)
    block, top = 16, 12
    bounds = torch.full((batch, heads_kv, -(-270 // block), 2, dhead), float("nan"), dtype=k.dtype, device="cuda")
    run_bounds(k, dtype, None, given, 0, block, bounds)
    some, selected = run_blocks(q, k, v, dtype, bounds, given, 0, block, top, 1, 2, scale)
    for b in sample:
        n = min(lengths[b], 270)
        for g in range(heads_kv):
            rows = q[b, 2 * g:2 * g + 2]
            see = torch.ones((2, n), dtype=torch.bool, device="cuda")
            want, tol, p = reference(rows, k[b, g, :n], v[b, g, :n], see, scale, dtype)
            within(got[b, 2 * g:2 * g + 2], want, tol, "entry %d group %d" % (b, g))
            if n:
                within(weights[b, g, :n], p[0][0] + p[1][0], p[0][1] + p[1][1] + (p[0][0] + p[1][0]) * 3 * 2.0 ** -24,
                       "weights of entry %d group %d" % (b, g))
            keep = select_reference(rows, bounds[b, g], n, block, top, 1, 2)
            assert selected[b, g].tolist() == keep + [-1] * (top - len(keep))
            see[:] = False
            for j in keep:
                see[:, j * block:(j + 1) * block] = True
            want, tol, _ = reference(rows, k[b, g, :n], v[b, g, :n], see, scale, dtype)
            within(some[b, 2 * g:2 * g + 2], want, tol, "blocks of entry %d group %d" % (b, g))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dhead, tokens, heads, lengths, t_max", [
    (64, 40, 16, [900, 33, 0], 31500), (128, 33, 8, [65, 4000], 114000), (80, 130, 4, [511], 116000),
], ids=str)
def test_tree_in_a_large_cache(gpu, dtype, dhead, tokens, heads, lengths, t_max):
    """Many rows in a cache with room for many positions: 32 rows a wave. Any mask, rows that see nothing,
    drafted tokens that no row sees hold anything."""
    gen, rng = generator(93), np.random.default_rng(93)
    batch, heads_kv = len(lengths), 2
    k, v = make_cache(gen, dtype, batch, heads_kv, t_max, dhead, [n + tokens for n in lengths])
    q = torch.randn((batch, tokens, heads, dhead), device="cuda", generator=gen) * 2
    seen = tree_mask(rng, batch, tokens)
    seen[0, 3] = rng.random(tokens) < 0.3
    seen[-1, 1] = seen[-1, 32] = False
    seen[:, :, 5] = False
    for b, n in enumerate(lengths):
        k[b, :, n + 5], v[b, :, n + 5] = float("nan"), float("inf")
    given = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    got = run_tree(q, k, v, dtype, given, 0, to_words(seen), dhead ** -0.5)
    check_tree(got, q, k, v, dtype, lengths, seen, dhead ** -0.5)
