"""Attention over an 8-bit cache (mynah_hip_kv8_attention_dev) against the formula in
64 bits (kv8_lib.Kv8.expected has the bound): types, formats, head sizes and groups,
lengths from nothing to several pieces, blocks and pages that end inside a tile, masks
that leave a row empty, NaN in unseen places, bad pages, counts that lie, streams and
captured graphs."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import elem_lib as E
from kv8_lib import E4M3, I8, Kv8
from test_tree_attention_gpu import LENGTHS, RAGGED, Hip

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def M():
    import mynah_amd
    mynah_amd.check(mynah_amd.lib.mynah_hip_init(0), "init")
    return mynah_amd


TYPES, FORMATS = [E.F32, E.F16, E.BF16], [I8, E4M3]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("f", FORMATS)
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("heads,kvh", [(2, 2), (6, 2), (14, 2), (8, 1)])
def test_heads(M, t, f, hd, heads, kvh):
    print("[case] kv8 heads", t, f, hd, heads, kvh, flush=True)
    c = Kv8(M, [(77, 5)], heads, kvh, hd, t, f, mask="tree", seed=hd + heads)
    c.check(c.attend())


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("f", FORMATS)
@pytest.mark.parametrize("lens", LENGTHS + [[(700, 150)], [(64, 64), (0, 64), (130, 60)]], ids=str)
def test_lengths(M, t, f, lens):
    print("[case] kv8 lengths", t, f, lens, flush=True)
    c = Kv8(M, lens, 8, 2, 128, t, f, 32, mask="tree", seed=len(lens))
    c.check(c.attend())


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("f", FORMATS)
@pytest.mark.parametrize("page,block", [(16, 16), (32, 16), (64, 64), (256, 128), (256, 256)])
def test_pages(M, t, f, page, block):
    c = Kv8(M, [(1003, 20), (15, 4), (0, 2), (256, 33)], 6, 2, 128, t, f, block, page=page, seed=page)
    c.check(c.attend())


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("f", FORMATS)
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_prompts(M, t, f, hd):
    # Many rows: a prompt's chunk behind a prefix, and prompts side by side.
    c = Kv8(M, [(90, 200)], 6, 2, hd, t, f, 64, seed=hd)
    c.check(c.attend())
    c = Kv8(M, [(0, 129), (33, 1), (5, 97), (0, 0)], 4, 1, hd, t, f, 16, page=16, seed=hd,
            extra_rows=3, pad=16)
    c.check(c.attend())


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_strides_and_rows_of_no_sequence(M, t, hd):
    c = Kv8(M, [(50, 6), (20, 3)], 4, 2, hd, t, I8, extra_rows=5, pad=16, max_nodes=40, max_kv=600)
    c.check(c.attend())


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("past", [0, 40])
def test_rows_that_see_little(M, t, past):
    # Node 1 sees no node (with no committed position: nothing), node 3 only node 0.
    mask = np.array([[1], [0], [0b101], [1], [0b11111]], np.uint32)
    c = Kv8(M, [(past, 5)], 4, 2, 128, t, E4M3, mask=mask)
    raw = c.attend()
    c.check(raw)
    if past == 0:
        assert np.all(E.decode(raw, t)[1] == 0)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("nodes", [40, 150])
def test_nan_where_nobody_looks(M, t, hd, nodes):
    """e4m3's NaN and bad scales behind the last position reach nobody, nor does an
    unseen node's NaN; as a seen node's value it is 0."""
    past = 37
    c = Kv8(M, [(past, nodes)], 4, 2, hd, t, E4M3, mask="tree", seed=4, max_kv=400)
    c.k[past + nodes:], c.v[past + nodes:] = 127, 255
    last = -(-(past + nodes) // 16)
    c.ks[last:], c.vs[last:] = np.nan, np.inf
    c.v[past + 3, 5], c.v[past + 9, hd + 1], c.v[past + 35] = 127, 255, 127
    c.check(c.attend())
    c.k[past + 20, 3] = 127                             # its head 0 only, for those who see it
    sees = (c.mask[:, 0] >> np.uint32(20) & 1).astype(bool)
    got = E.decode(c.attend(), t)[:, :4 * hd].reshape(-1, 4, hd)
    assert np.isnan(got[sees][:, :2]).all() and sees.any() and not sees.all()
    assert np.isfinite(got[~sees]).all() and np.isfinite(got[:, 2:]).all()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("f", FORMATS)
@pytest.mark.parametrize("nodes", [2, 80])
def test_scales(M, t, f, nodes):
    """Scales far apart, zeros, negative and not finite: the last four count as 0."""
    c = Kv8(M, [(200, nodes)], 4, 2, 128, t, f, seed=6)
    # A block of large values that is far from the query, and small values near it.
    c.vs[2] = np.float32(1e6)
    c.vs[5], c.ks[6], c.vs[7] = np.float32(1e-9), np.float32(1e-9), np.float32(0)
    c.ks[8], c.ks[9, 0], c.ks[9, 1], c.ks[10] = 0, np.nan, np.inf, -1
    c.vs[9, 0], c.vs[9, 1], c.vs[10] = np.inf, np.nan, -2
    c.check(c.attend())
    c.vs[:] = 0
    raw = c.attend()
    assert np.all(E.decode(raw, t)[:, :512] == 0)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("nodes", [3, 70])
def test_a_small_value_block_that_takes_all(M, t, nodes):
    """The block that the queries attend to holds values 2^30 smaller than the one
    before it, whose probabilities are next to nothing."""
    c = Kv8(M, [(64, nodes)], 2, 1, 64, t, I8, seed=8, mask="chain")
    q = np.zeros((nodes, 64))
    q[:, 0] = 8.0
    c.q = E.encode(np.tile(q, 2), t)
    c.k[:, 0] = np.where(np.arange(c.slots) // 16 == 2, 100, 156)         # +-100
    c.ks[:] = np.float32(0.5)
    c.vs[:] = np.float32(1.0)
    c.vs[2] = np.float32(2.0 ** -30)
    c.check(c.attend())


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("nodes", [4, 90])
def test_large_scores(M, t, nodes):
    for scale in (3.0, -0.3, 0.0):
        c = Kv8(M, [(300, nodes)], 4, 2, 128, t, I8, scale=scale, seed=9)
        c.check(c.attend(), scale)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("nodes", [6, 100])
def test_bad_pages_are_unseen(M, t, nodes):
    c = Kv8(M, [(200, nodes), (90, 2)], 4, 2, 128, t, I8, page=16, seed=2)
    c.pages[0, 2], c.pages[0, 7], c.pages[1, 0] = -1, 1 << 30, c.slots // 16
    c.check(c.attend())
    c.pages[1, :] = -7                                  # a sequence with no page at all
    raw = c.attend()
    c.check(raw)
    assert np.all(E.decode(raw, t)[nodes:] == 0)


def test_counts_that_lie(M):
    c = Kv8(M, [(50, 9), (200, 3)], 4, 2, 128, E.F32, I8, max_nodes=4, max_kv=120)
    c.check(c.attend())
    c = Kv8(M, [(-5, 3), (10, 2)], 4, 2, 128, E.F32, I8)
    c.check(c.attend())
    c = Kv8(M, [(20, 3), (10, 2)], 4, 2, 128, E.F32, I8)
    c.start = np.array([-2, 1, 400], np.int32)          # rows -2 .. 0 and 1 .. 399 of 5
    raw = c.attend(max_nodes=3)
    assert np.isfinite(raw).all()
    assert np.array_equal(raw[4:], c.out0[4:])
    for start in ([3, 3, 1], [-2147483648, 2147483647, -2147483648]):
        c.start = np.array(start, np.int32)
        assert np.array_equal(c.attend(), c.out0)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("f", FORMATS)
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_long_context_and_equal_bits(M, t, f, hd):
    # One key head: its positions go to every CU, and more than 64 sums meet in a wave.
    c = Kv8(M, [(40_989, 3)], 4, 1, hd, t, f, 64, seed=1)
    a = c.attend()
    c.check(a)
    assert np.array_equal(a.view(np.uint8), c.attend().view(np.uint8))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("lens", RAGGED, ids=lambda v: f"{len(v)}-{max(v)[0]}")
def test_ragged_batches(M, t, lens):
    c = Kv8(M, lens, 2, 1, 64, t, I8, page=16, seed=7, extra_rows=1)
    raw = c.attend()
    c.check(raw)
    assert np.array_equal(raw, c.attend())


def test_one_workspace_byte_short(M):
    c = Kv8(M, [(9000, 2)], 4, 1, 128, E.F32, I8)
    c.upload()
    a = c.attn_args()
    n = M.kv8_attention_workspace(a)
    ws = M.DeviceBuffer(n)
    assert M.lib.mynah_hip_kv8_attention_dev(C.byref(a), ws.ptr, n - 1, None) == -1
    assert b"workspace" in M.lib.mynah_hip_last_error()
    assert np.array_equal(c.raw(), c.out0)


def test_two_streams_with_workspaces_of_their_own(M):
    h = Hip()
    c = [Kv8(M, [(2000 + 50 * i, 5)], 8, 2, 128, E.BF16, E4M3, seed=i) for i in range(2)]
    for x in c:
        x.upload()
    a = [x.attn_args() for x in c]
    ws = [M.DeviceBuffer(M.kv8_attention_workspace(x)) for x in a]
    st = [h.stream() for _ in c]
    for _ in range(5):
        for x, w, s in zip(a, ws, st):
            M.kv8_attention_dev(x, w.ptr, w.nbytes, s)
    for s in st:
        M.check(M.lib.mynah_hip_sync(s), "sync")
    for x in c:
        x.check(x.raw())
    for s in st:
        h.lib.hipStreamDestroy(C.c_void_p(s))


@pytest.mark.parametrize("t", [E.F32, E.BF16])
@pytest.mark.parametrize("f", FORMATS)
def test_captured_store_and_attention(M, t, f):
    """One captured step, replayed while lengths and inputs on the device move on,
    against the definition and the eager calls."""
    h = Hip()
    c = Kv8(M, [(500, 1)], 8, 2, 128, t, f, 32, page=64, max_kv=600, seed=6)
    c.upload()
    st, a = c.store_args(), c.attn_args()
    n = M.kv8_attention_workspace(a)
    ws = M.DeviceBuffer(n)
    s = h.stream()

    def step(stream):
        M.kv8_store_dev(st, stream)
        M.kv8_attention_dev(a, ws.ptr, n, stream)

    g, e = h.capture(s, lambda: step(s))
    for past in (500, 3, 501, 599, 64):
        for name in ("kx", "vx"):
            x = E.encode(c.rng.standard_normal(c.kx.shape) * 2, t)
            setattr(c, name, x)
            c.d[name].upload(x)
        c.lens, c.past = [(past, 1)], np.array([past], np.int32)
        c.d["past"].upload(c.past)
        assert h.lib.hipGraphLaunch(e, C.c_void_p(s)) == 0
        M.check(M.lib.mynah_hip_sync(s), "sync")
        got, cache = c.raw(), c.stored()
        c.check_store(cache, past)
        for name, x in cache.items():
            setattr(c, name, x)
        c.check(got, past)
        c.d["out"].upload(c.out0)
        step(None)                                      # the same rows again, eagerly
        M.sync()
        assert np.array_equal(got, c.raw()), past
        assert all(np.array_equal(x, c.stored()[name]) for name, x in cache.items())
    h.lib.hipGraphExecDestroy(e)
    h.lib.hipGraphDestroy(g)
    h.lib.hipStreamDestroy(C.c_void_p(s))


def test_offsets_past_32_bits(M):
    """Pages far into a cache of over 4 GiB: byte offsets need 64 bits."""
    kvh, hd, page = 8, 256, 256
    c = Kv8(M, [(700, 4)], 8, kvh, hd, E.BF16, I8, 64, page=page, seed=12)
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
@pytest.mark.parametrize("nodes", [1, 6, 20])
def test_long_sequences_beside_short_ones(M, t, nodes):
    """More pieces than CUs: sequences are cut by their lengths, pieces of 16 turns."""
    lens = [(20_011, nodes), (3, 1), (9000, nodes), (0, 0), (14_500, 2)]
    c = Kv8(M, lens, 4, 1, 128, t, E4M3, 64, page=64, seed=11)
    raw = c.attend()
    assert M.kv8_attention_workspace(c.attn_args()) > 12 * 130 * 4 * 16
    c.check(raw)
    assert np.array_equal(raw, c.attend())


@pytest.mark.parametrize("t", TYPES)
def test_a_prompt_cut_into_pieces(M, t):
    # 96 tokens of one sequence over a long context: few workgroups of rows, so its
    # positions are cut too.
    c = Kv8(M, [(6000, 96)], 8, 2, 128, t, I8, 32, page=32, seed=12)
    c.check(c.attend())
    c = Kv8(M, [(3000, 40), (100, 96), (0, 3)], 4, 1, 64, t, E4M3, 16, mask="tree", seed=13)
    c.check(c.attend())


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("f", FORMATS)
@pytest.mark.parametrize("nodes", [2, 60])
def test_small_queries(M, t, f, nodes):
    # f16 subnormals, and sizes at which the parts of an f32 are still normal bf16 numbers
    size = {E.F32: 2.0 ** -90, E.F16: 2.0 ** -16, E.BF16: 2.0 ** -90}[t]
    c = Kv8(M, [(100, nodes)], 4, 2, 64, t, f, seed=15, scale=0.2 / size)
    c.q = E.encode(E.decode(c.q, t) * size, t)
    c.check(c.attend())


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("nodes", [2, 60])
@pytest.mark.parametrize("size", [2.0 ** 20, -2.0 ** 20, 2.0 ** 28])
def test_equal_scores_of_any_size(M, t, hd, nodes, size):
    """Every position scores the same: the mean of the values that a row sees, whatever
    the size."""
    c = Kv8(M, [(48, nodes)], 2, 1, hd, t, I8, seed=16)
    c.k[:] = 3
    c.ks[:] = np.float32(1 / 3)
    c.q = E.encode(np.ones((nodes, 2 * hd)), t)
    c.scale = size / hd
    got = E.decode(c.attend(), t)
    v = c.v.view(np.int8).astype(np.float64) * np.repeat(c.vs, 16, 0)
    half = {E.F32: 0.0, E.F16: 2.0 ** -16, E.BF16: 2.0 ** -8}[t]
    for i in range(nodes):
        n = 48 + i + 1
        want, big = v[:n].mean(0), np.abs(v[:n]).mean(0)
        tol = (half + 4 * n * E.U) * big + E.rounded(want, t)
        assert (np.abs(got[i].reshape(2, hd) - want) <= tol).all(), i
