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


@pytest.mark.parametrize("below", [12.0, 15.0, 17.4, 20.0])
@pytest.mark.parametrize("t", TYPES)
def test_much_weight_in_small_probabilities(M, t, below):
    """One position `below` nats above 130,000 others, and values of one sign: each
    other's probability is small, their sum is not. The bound is that of
    tree_lib.Tree.expected but for two terms. One key head's positions go to 128
    workgroups at least, so that no sum is a chain of more than n / 128 additions and
    those that join 512 waves' and workgroups': n / 128 + 512 in place of n. And an f16
    probability below the type's smallest normal number is off by up to 2^-25
    where the row's largest is at least 2^11: n 2^-36 of it at most."""
    print("[case] small probabilities", t, below, flush=True)
    hd, n = 64, 130_003
    c = Tree(M, [(n - 3, 3)], 2, 1, hd, t, mask="chain", seed=5)
    q = np.zeros(c.q.shape)
    q[:, ::hd] = 8.0
    k = 0.01 * c.rng.standard_normal(c.k.shape)
    k[:, 0] = 0.0
    k[7, 0] = below                                      # 8 below * 64^-0.5
    c.q, c.k = E.encode(q, t), E.encode(k, t)
    c.v = E.encode(1.0 + 0.25 * c.rng.random(c.v.shape), t)
    raw = c.call()
    assert c.ws.nbytes > 128 * 16 * (hd + 2) * 4
    want = c.expected()[0]
    got = E.decode(raw, t).reshape(want.shape)
    dm = (hd + 4) * U * below
    tol = want * (2 * dm + (6 + n / 128 + 512) * U + (0 if t == E.F32 else E.HALF[t]))
    tol += E.rounded(want, t) + (n * 2.0 ** -36 * 1.25 if t == E.F16 else 0)
    off = np.abs(got - want) / tol
    print(f"largest error {float(off.max()):.2f} of its bound", flush=True)
    assert off.max() <= 1


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_committed_keys_of_minus_infinity(M, t, hd):
    """A committed key whose score is -inf is unseen in effect: the bound is that
    of the call in which its page is no page."""
    c = Tree(M, [(200, 6), (90, 2)], 4, 2, hd, t, page=16, seed=2)
    for h in range(4):                                   # so that -inf times it is -inf
        c.q[:, h * hd] = E.encode(np.abs(E.decode(c.q[:, h * hd], t)) + 0.5, t)
    gone = [(0, 0), (0, 3), (0, 11), (1, 4)]
    for b, p in gone:
        rows = slice(int(c.pages[b, p]) * 16, int(c.pages[b, p]) * 16 + 16)
        for h in range(2):
            c.k[rows, h * hd] = E.encode(np.full(16, -np.inf), t)
    raw = c.call()
    for b, p in gone:
        c.pages[b, p] = -1
    c.check(raw)
