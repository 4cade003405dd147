"""Attention over an 8-bit cache at the ends of what it takes: factors of scores from
f32's largest to below its smallest, and scales that count as 0 beside them."""
from __future__ import annotations

import numpy as np
import pytest

import elem_lib as E
from kv8_lib import E4M3, I8, Kv8

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
