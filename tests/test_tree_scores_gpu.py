"""Scores of tree attention (mynah_hip_tree_attention_dev) that its other tests do
not hold: far apart, of a negative scale, of -inf, much weight in many small
probabilities."""
from __future__ import annotations

import numpy as np
import pytest

import elem_lib as E
from tree_lib import Tree

pytestmark = pytest.mark.gpu
TYPES = [E.F32, E.F16, E.BF16]
U = E.U


@pytest.fixture(scope="module")
def M():
    import mynah_amd
    mynah_amd.check(mynah_amd.lib.mynah_hip_init(0), "init")
    return mynah_amd


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("scale", [2.0 ** 20, 2.0 ** 28, 2.0 ** 33, 1e30, 3e38, -2.0 ** 33, -3e38])
@pytest.mark.parametrize("lens", [[(300, 4)], [(5000, 20)], [(40, 3)] * 3], ids=str)
def test_scores_far_apart(M, t, scale, lens):
    """Small whole numbers in q and k: scores are exact, and another than the
    largest is smaller by 2^20 at least, its weight 0. The output is the mean of
    the values at the largest: m ties, each weighted by one power of two, add up
    within (m + 2) u of their sizes, then the result's own rounding."""
    print("[case] far apart", t, scale, lens, flush=True)
    c = Tree(M, lens, 4, 2, 128, t, mask="chain", seed=3, scale=scale)
    c.q = E.encode(c.rng.integers(-2, 3, c.q.shape), t)
    c.k = E.encode(c.rng.integers(-2, 3, c.k.shape), t)
    got = E.decode(c.call(), t).reshape(c.rows, 4, 128)
    q, k, v = (E.decode(a, t).reshape(len(a), -1, 128) for a in (c.q, c.k, c.v))
    for b, (past, nodes) in enumerate(lens):
        at = c.cache_rows(b, past + nodes)
        for i in range(nodes):
            row = int(c.start[b]) + i
            for h in range(4):
                s = np.sign(scale) * (k[at[:past + i + 1], h // 2] @ q[row, h])
                best = v[at[:past + i + 1]][s == s.max(), h // 2]
                want = best.mean(0)
                tol = (len(best) + 2) * U * np.abs(best).mean(0) + E.rounded(want, t)
                assert np.all(np.abs(got[row, h] - want) <= tol), (row, h, len(best))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_negative_scale(M, t, hd):
    c = Tree(M, [(333, 9), (20, 2)], 6, 2, hd, t, seed=hd, scale=-hd ** -0.5)
    c.check(c.call())
