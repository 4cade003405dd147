"""Attention over an 8-bit cache at the ends of what it takes: factors of scores from
f32's largest to below its smallest, scales that count as 0 beside them, weights' bits."""
from __future__ import annotations

import numpy as np
import pytest

import elem_lib as E
from kv8_lib import E4M3, I8, Kv8, values

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def M():
    import mynah_amd
    mynah_amd.check(mynah_amd.lib.mynah_hip_init(0), "init")
    return mynah_amd


TYPES, FORMATS = [E.F32, E.F16, E.BF16], [I8, E4M3]
LARGE = {E.F32: 2.0 ** 108, E.F16: 2.0 ** 12, E.BF16: 2.0 ** 108}


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("f", FORMATS)
@pytest.mark.parametrize("nodes", [2, 12, 60])
def test_large_queries(M, t, f, nodes):
    """Large queries under a small scale: scores of a few units."""
    print("[case] kv8 large queries", t, f, nodes, flush=True)
    c = Kv8(M, [(100, nodes)], 4, 2, 64, t, f, seed=15, scale=0.2 / LARGE[t], mask="tree")
    c.q = E.encode(E.decode(c.q, t) * LARGE[t], t)
    c.check(c.attend())


@pytest.mark.parametrize("t", [E.F32, E.BF16])
@pytest.mark.parametrize("f", FORMATS)
@pytest.mark.parametrize("nodes", [2, 12, 60])
def test_small_key_scales(M, t, f, nodes):
    """Key scales at the least that the store makes (2^-100 over the largest code), and
    queries that make scores of a few units of them."""
    c = Kv8(M, [(100, nodes)], 4, 2, 64, t, f, seed=16, scale=0.5, mask="tree")
    c.ks[:] = np.float32(2.0 ** -107)
    c.q = E.encode(E.decode(c.q, t) * 2.0 ** 100, t)
    c.check(c.attend())


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("f", FORMATS)
@pytest.mark.parametrize("nodes", [2, 12, 60])
@pytest.mark.parametrize("scale", [0.2, 0.0])
def test_scales_of_nothing_beside_large_queries(M, t, f, nodes, scale):
    """A key scale that is not positive and finite makes scores of 0 whatever the
    queries' size, and so does a scale of 0."""
    c = Kv8(M, [(100, nodes)], 4, 2, 64, t, f, seed=17, scale=scale / LARGE[t], mask="tree")
    c.ks[1], c.ks[3, 0], c.ks[3, 1], c.ks[5], c.ks[6] = 0, np.nan, np.inf, -1, 1e-45
    c.q = E.encode(E.decode(c.q, t) * LARGE[t], t)
    c.check(c.attend(), scale)


@pytest.mark.parametrize("t", [E.F16, E.BF16])
@pytest.mark.parametrize("f", FORMATS)
@pytest.mark.parametrize("hd,nodes", [(64, 1), (64, 7), (64, 16), (128, 3), (128, 8), (128, 13),
                                      (256, 4), (256, 8)])
def test_weights_of_few_rows(M, t, f, hd, nodes):
    """Up to 64 rows a key head, 32 of 256 values, a weight keeps 16 bits: outputs are off by the result's
    own rounding and 2^-16 of A = sum p |v|, besides what kv8_lib.Kv8.expected gives
    scores, exponentials and sums (2 d A, 6 u A, and 2 n u A of two products a position)."""
    past, heads, kvh = 57, 8, 2
    c = Kv8(M, [(past, nodes)], heads, kvh, hd, t, f, 64, seed=hd + nodes)
    got = E.decode(c.attend(), t)[:, :heads * hd].reshape(nodes, heads, hd)
    k, v = ((values(x, f).reshape(-1, kvh, hd) * np.repeat(s.astype(np.float64), 64, 0)[..., None])
            for x, s in ((c.k, c.ks), (c.v, c.vs)))
    q = E.decode(c.q, t).reshape(nodes, heads, hd)
    for i in range(nodes):
        n = past + i + 1
        for h in range(heads):
            kk, vv = k[:n, h // 4], v[:n, h // 4]
            x = c.scale * (kk @ q[i, h])
            p = np.exp(x - x.max())
            p /= p.sum()
            d = (hd + 8) * E.U * c.scale * (np.abs(kk) @ np.abs(q[i, h])).max()
            want, size = p @ vv, p @ np.abs(vv)
            tol = (2 * d + (6 + 2 * n) * E.U + 2.0 ** -16) * size + E.rounded(want, t)
            assert (np.abs(got[i, h] - want) <= tol).all(), (i, h)


@pytest.mark.parametrize("t", [E.F32, E.BF16])
@pytest.mark.parametrize("f", FORMATS)
@pytest.mark.parametrize("past,nodes", [(100, 2), (5003, 12), (100, 60)])
@pytest.mark.parametrize("size", [2.0 ** 90, 2.0 ** -100])
def test_sizes_of_values(M, t, f, past, nodes, size):
    """Values near the largest that are taken, and of the least scale that the store makes."""
    c = Kv8(M, [(past, nodes)], 4, 2, 128, t, f, 64, seed=18, mask="tree")
    c.vs = (c.vs * np.float32(size)).astype(np.float32)
    c.check(c.attend(), size)
