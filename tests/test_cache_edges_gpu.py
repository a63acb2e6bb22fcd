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
