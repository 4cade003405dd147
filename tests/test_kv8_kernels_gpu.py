"""What either kernel of the attention over an 8-bit cache has of its own, few rows a
key head (one and two column tiles, one and two groups of rows, whole sequences and
pieces) and many: e4m3's NaN,
bad scales, offsets past 32 bits, cache rows that sequences share."""
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


TYPES = [E.F32, E.F16, E.BF16]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("nodes", [5, 14, 25, 40])
@pytest.mark.parametrize("past", [37, 5003])
def test_nan(M, t, hd, nodes, past):
    """Behind the last position and in unseen nodes NaN reaches nobody; a seen node's
    NaN value is 0, its NaN key is seen; a committed one's value reaches all."""
    print("[case] kv8 nan", t, hd, nodes, past, flush=True)
    c = Kv8(M, [(past, nodes)], 4, 2, hd, t, E4M3, mask="tree", seed=4, max_kv=past + 400)
    c.k[past + nodes:], c.v[past + nodes:] = 127, 255
    last = -(-(past + nodes) // 16)
    c.ks[last:], c.vs[last:] = np.nan, np.inf
    c.v[past, 5], c.v[past + 3, hd + 1], c.v[past + 4], c.v[past + nodes - 1, 7] = 127, 255, 127, 255
    c.check(c.attend())
    # A node that some see, not all.
    seen = (c.mask[:, :, None] >> np.arange(32, dtype=np.uint32) & 1).reshape(nodes, -1).sum(0)
    node = int(np.flatnonzero((seen > 1) & (seen < nodes))[-1])
    c.k[past + node, 3] = 127                           # its head 0 only, for those who see it
    sees = (c.mask[:, node // 32] >> np.uint32(node % 32) & 1).astype(bool)
    got = E.decode(c.attend(), t)[:, :4 * hd].reshape(-1, 4, hd)
    assert np.isnan(got[sees][:, :2]).all() and sees.any() and not sees.all()
    assert np.isfinite(got[~sees]).all() and np.isfinite(got[:, 2:]).all()
    c.k[past + node, 3] = 0
    c.v[past - 30, hd + 2] = 255                        # a committed value of head 1
    got = E.decode(c.attend(), t)[:, :4 * hd].reshape(-1, 4, hd)
    assert np.isnan(got[:, 2:, 2]).all()
    got[:, 2:, 2] = 0
    assert np.isfinite(got).all()


@pytest.mark.parametrize("f,nodes", [(I8, 40), (E4M3, 1), (E4M3, 40)])
def test_offsets_past_32_bits(M, f, nodes):
    """Pages far into a cache of over 4 GiB, for either kernel."""
    kvh, hd, page = 8, 256, 256
    c = Kv8(M, [(700, nodes)], 8, kvh, hd, E.BF16, f, 64, page=page, seed=12)
    rows = (1 << 32) // (kvh * hd) + 4096
    first = rows - c.slots
    c.upload()
    big = {n: M.DeviceBuffer(rows * kvh * hd) for n in ("k", "v")}
    scales = {n: M.DeviceBuffer(rows // 64 * kvh * 4) for n in ("ks", "vs")}
    for n, b in big.items():
        M.check(M.lib.mynah_hip_h2d(b.ptr + first * kvh * hd, M.ptr(getattr(c, n)),
                                    c.slots * kvh * hd), "h2d")
    for n, b in scales.items():
        M.check(M.lib.mynah_hip_h2d(b.ptr + first // 64 * kvh * 4, M.ptr(getattr(c, n)),
                                    getattr(c, n).nbytes), "h2d")
    c.d["pages"].upload((c.pages + first // page).astype(np.int32))
    a = c.attn_args()
    a.cache.k, a.cache.v, a.cache.n_slots = big["k"].ptr, big["v"].ptr, rows
    a.cache.k_scale, a.cache.v_scale = scales["ks"].ptr, scales["vs"].ptr
    n = M.kv8_attention_workspace(a)
    ws = M.DeviceBuffer(n)
    M.kv8_attention_dev(a, ws.ptr, n)
    M.sync()
    c.check(c.raw())


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("nodes", [2, 50])
@pytest.mark.parametrize("seq_slots", [0, 32])
def test_shared_rows(M, t, nodes, seq_slots):
    """Sequences over one run of rows, from one place or a block or two apart."""
    c = Kv8(M, [(100, nodes), (90, 1), (100, nodes)], 4, 2, 64, t, I8, seed=5)
    c.seq_slots = seq_slots
    c.check(c.attend())
