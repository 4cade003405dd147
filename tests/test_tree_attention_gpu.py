"""Attention of drafted tokens over a cache (mynah_hip_tree_attention_dev)
against the formula in 64 bits (tree_lib.Tree.expected has the bound): types,
head sizes and groups, lengths from nothing to several splits, pages that end
inside a tile, masks that leave a row empty, values that are not finite in
unseen places, bad pages, counts that lie, streams and captured graphs."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import elem_lib as E
from tree_lib import Tree

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def M():
    import mynah_amd
    mynah_amd.check(mynah_amd.lib.mynah_hip_init(0), "init")
    return mynah_amd


TYPES = [E.F32, E.F16, E.BF16]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("heads,kvh", [(2, 2), (6, 2), (14, 2), (8, 1)])
def test_heads(M, t, hd, heads, kvh):
    print("[case] tree heads", t, hd, heads, kvh, flush=True)
    c = Tree(M, [(77, 5)], heads, kvh, hd, t, seed=hd + heads)
    c.check(c.call())


LENGTHS = [[(0, 1)], [(1, 1)], [(15, 1)], [(16, 1)], [(31, 2)], [(128, 1)], [(513, 1)], [(0, 9)],
           [(0, 40)], [(3, 70)], [(1000, 33)], [(4099, 3)], [(200, 130)],
           [(0, 1), (300, 7), (0, 0), (65, 12), (128, 1)], [(0, 0), (5, 2)]]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("lens", LENGTHS, ids=str)
def test_lengths(M, t, lens):
    print("[case] tree lengths", t, lens, flush=True)
    c = Tree(M, lens, 8, 2, 128, t, seed=len(lens))
    c.check(c.call())


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("page", [16, 32, 256])
def test_pages(M, t, page):
    print("[case] tree pages", t, page, flush=True)
    c = Tree(M, [(1003, 20), (15, 4), (0, 2), (256, 33)], 6, 2, 128, t, page=page, seed=page)
    c.check(c.call())


@pytest.mark.parametrize("t", TYPES)
def test_chain(M, t):
    c = Tree(M, [(100, 37), (0, 5), (64, 1)], 4, 2, 64, t, mask="chain")
    c.check(c.call())


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_strides_and_rows_of_no_sequence(M, t, hd):
    c = Tree(M, [(50, 6), (20, 3)], 4, 2, hd, t, extra_rows=5, pad=16, max_nodes=40, max_kv=600)
    c.check(c.call())


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("past", [0, 40])
def test_rows_that_see_little(M, t, past):
    # Node 1 sees no node (with no committed position: nothing), node 3 only node 0.
    mask = np.array([[1], [0], [0b101], [1], [0b11111]], np.uint32)
    c = Tree(M, [(past, 5)], 4, 2, 128, t, mask=mask)
    raw = c.call()
    c.check(raw)
    if past == 0:
        assert np.all(E.decode(raw, t)[1] == 0)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
def test_not_finite_where_nobody_looks(M, t, hd):
    """NaN and infinities in the keys and values of nodes reach exactly the rows
    that see them, and those past the end nobody."""
    past, nodes = 37, 40
    c = Tree(M, [(past, nodes)], 4, 2, hd, t, seed=4, max_kv=200)
    nan, inf = E.encode(np.nan, t), E.encode(np.inf, t)
    c.v[past + 3, 5], c.v[past + 9, hd + 1] = nan, inf
    c.v[past + 35, :] = nan
    c.k[past + 20, :hd] = nan
    c.k[past + nodes:], c.v[past + nodes:] = nan, nan           # behind the last position
    want, tol, _ = c.expected()
    got = E.decode(c.call(), t)[:, :c.heads * hd].reshape(want.shape)
    assert np.isnan(want).any() and np.isinf(want).any() and np.isfinite(want).any()
    assert np.array_equal(np.isnan(want), np.isnan(got))
    odd = ~np.isfinite(want)
    assert np.array_equal(want[odd & ~np.isnan(want)], got[odd & ~np.isnan(want)])
    assert np.all(np.abs(got - want)[~odd] <= tol[~odd])


def test_not_finite_committed(M):
    # A committed key of -inf scores is unseen in effect; one value of inf reaches all.
    c = Tree(M, [(70, 3)], 2, 1, 128, E.F32, mask="chain")
    c.v[11, 4] = np.inf
    got = c.call().reshape(3, 2, 128)
    assert np.all(np.isinf(got[..., 4])) and np.isfinite(np.delete(got, 4, 2)).all()


@pytest.mark.parametrize("t", TYPES)
def test_large_scores(M, t):
    # Scores of +-200 and above: the maximum keeps exp in range; one position takes all.
    c = Tree(M, [(300, 4)], 4, 2, 128, t, scale=3.0, seed=9)
    c.check(c.call())
    c = Tree(M, [(300, 4)], 4, 2, 128, t, scale=0.0)
    c.check(c.call())


@pytest.mark.parametrize("t", TYPES)
def test_bad_pages_are_unseen(M, t):
    c = Tree(M, [(200, 6), (90, 2)], 4, 2, 128, t, page=16, seed=2)
    c.pages[0, 2], c.pages[0, 7], c.pages[1, 0] = -1, 1 << 30, c.slots // 16
    c.check(c.call())
    c.pages[1, :] = -7                                  # a sequence with no page at all
    raw = c.call()
    c.check(raw)
    assert np.all(E.decode(raw, t)[6:8] == 0)


def test_fewer_slots_than_said(M):
    # n_slots cuts the cache inside a tile: the rest is unseen and not read.
    c = Tree(M, [(90, 4)], 4, 2, 128, E.BF16, seed=3)
    full, c.slots = c.slots, 75
    raw = c.call()
    c.check(raw)
    assert full > 75


def test_counts_that_lie(M):
    """Nodes past max_nodes are left out, positions past max_kv unseen, row starts
    outside the rows untouched, a negative n_past none."""
    c = Tree(M, [(50, 9), (200, 3)], 4, 2, 128, E.F32, mask="chain", max_nodes=4, max_kv=120)
    c.check(c.call())
    c = Tree(M, [(-5, 3), (10, 2)], 4, 2, 128, E.F32, mask="chain")
    c.check(c.call())
    c = Tree(M, [(20, 3), (10, 2)], 4, 2, 128, E.F32, mask="chain")
    c.start = np.array([-2, 1, 400], np.int32)          # rows -2 .. 0 and 1 .. 399 of 5
    raw = c.call(max_nodes=3)
    assert np.isfinite(raw).all()
    assert np.array_equal(raw[4:], c.out0[4:])
    c.start = np.array([3, 3, 1], np.int32)             # empty, and less than empty
    assert np.array_equal(c.call(), c.out0)
    c.start = np.array([-2147483648, 2147483647, -2147483648], np.int32)
    assert np.array_equal(c.call(), c.out0)


@pytest.mark.parametrize("t", TYPES)
def test_long_context_and_equal_bits(M, t):
    c = Tree(M, [(9000, 2)], 4, 1, 128, t, seed=1)
    a = c.call()
    c.check(a)
    assert np.array_equal(a.view(np.uint8), c.call().view(np.uint8))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_more_splits_than_lanes(M, t, hd):
    # One key head: its positions go to every CU, and more than 64 sums meet in a wave.
    c = Tree(M, [(29_989, 3)], 4, 1, hd, t, seed=5)
    assert M.tree_attention_workspace(c.args()) > 65 * 12 * (hd + 2) * 4
    c.check(c.call())


RAGGED = [[(9000, 4)] + [(20, 2)] * 15, [(0, 0)] * 3 + [(5000, 3), (0, 0), (1, 1)], [(0, 0)] * 4,
          [(40 * i % 1201, i % 4) for i in range(70)], [(i % 3, i % 2) for i in range(200)]]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("lens", RAGGED, ids=lambda v: f"{len(v)}-{max(v)[0]}")
def test_ragged_batches(M, t, lens):
    # Sequences of very different lengths are cut into pieces by theirs.
    print("[case] tree ragged", t, len(lens), flush=True)
    c = Tree(M, lens, 2, 1, 64, t, page=16, seed=7, extra_rows=1)
    raw = c.call()
    c.check(raw)
    assert np.array_equal(raw, c.call())


def test_one_workspace_byte_short(M):
    c = Tree(M, [(900, 2)], 4, 1, 128, E.F32)
    a = c.args()
    n = M.tree_attention_workspace(a)
    ws = M.DeviceBuffer(n)
    assert M.lib.mynah_hip_tree_attention_dev(C.byref(a), ws.ptr, n - 1, None) == -1
    assert b"workspace" in M.lib.mynah_hip_last_error()
    assert np.array_equal(c.raw(), c.out0)


# ── streams and graphs ───────────────────────────────────────────────────────

class Hip:
    """The few runtime calls a caller with its own streams makes."""

    def __init__(self):
        self.lib = C.CDLL("libamdhip64.so.7")
        for name in ("hipStreamCreateWithFlags", "hipStreamBeginCapture", "hipStreamEndCapture",
                     "hipGraphInstantiate", "hipGraphLaunch", "hipGraphDestroy",
                     "hipGraphExecDestroy", "hipStreamDestroy", "hipStreamSynchronize"):
            getattr(self.lib, name).restype = C.c_int

    def stream(self):
        s = C.c_void_p()
        assert self.lib.hipStreamCreateWithFlags(C.byref(s), C.c_uint(1)) == 0
        return s.value

    def capture(self, stream, calls):
        s, g, e = C.c_void_p(stream), C.c_void_p(), C.c_void_p()
        assert self.lib.hipStreamBeginCapture(s, C.c_int(2)) == 0
        calls()
        assert self.lib.hipStreamEndCapture(s, C.byref(g)) == 0
        assert self.lib.hipGraphInstantiate(C.byref(e), g, None, None, C.c_size_t(0)) == 0
        return g, e


def test_two_streams_with_workspaces_of_their_own(M):
    h = Hip()
    c = [Tree(M, [(2000 + 50 * i, 5)], 8, 2, 128, E.BF16, seed=i) for i in range(2)]
    a = [x.args() for x in c]
    ws = [M.DeviceBuffer(M.tree_attention_workspace(x)) for x in a]
    st = [h.stream() for _ in c]
    for _ in range(5):
        for x, w, s in zip(a, ws, st):
            M.tree_attention_dev(x, w.ptr, w.nbytes, s)
    for s in st:
        M.check(M.lib.mynah_hip_sync(s), "sync")
    for x in c:
        x.check(x.raw())
    for s in st:
        h.lib.hipStreamDestroy(C.c_void_p(s))


def test_captured_call_follows_its_inputs(M):
    """One captured norm + rotation + attention step, replayed while the positions,
    slots and lengths on the device move on, against the eager calls."""
    h = Hip()
    heads, kvh, hd, cap, t = 8, 2, 128, 600, E.F32
    c = Tree(M, [(500, 1)], heads, kvh, hd, t, mask="chain", max_kv=cap, seed=6)
    a = c.args()
    freqs, _ = M.rope_freqs(hd, 1e6)
    B = M.DeviceBuffer.from_array
    row = (heads + 2 * kvh) * hd
    rng = np.random.default_rng(8)
    w = B(np.ones(hd, np.float32))
    f, x = B(freqs), M.DeviceBuffer(4 * row)
    pos = M.DeviceBuffer(4)
    p = M.QkNormRope(type=t, out_type=t, layout=0, n_heads=heads, n_kv_heads=kvh, head_dim=hd,
                     rot_dim=hd, tokens=1, q=x.ptr, k=x.ptr + 4 * heads * hd,
                     v=x.ptr + 4 * (heads + kvh) * hd, q_stride=row, k_stride=row, v_stride=row,
                     q_norm=w.ptr, k_norm=w.ptr, eps=1e-6, mscale=1.0, freqs=f.ptr, pos=pos.ptr,
                     slots=pos.ptr, n_slots=c.slots, q_out=c.d["q"].ptr, q_out_stride=heads * hd,
                     k_cache=c.d["k"].ptr, v_cache=c.d["v"].ptr, slot_stride=kvh * hd)
    n = M.tree_attention_workspace(a)
    ws = M.DeviceBuffer(n)
    s = h.stream()

    def step(stream):
        M.qk_norm_rope_dev(p, stream)
        M.tree_attention_dev(a, ws.ptr, n, stream)

    g, e = h.capture(s, lambda: step(s))
    for past in (500, 3, 501, 599, 64):
        x.upload(rng.standard_normal(row).astype(np.float32))
        pos.upload(np.array([past], np.int32))
        c.d["past"].upload(np.array([past], np.int32))
        assert h.lib.hipGraphLaunch(e, C.c_void_p(s)) == 0
        M.check(M.lib.mynah_hip_sync(s), "sync")
        got = c.raw()
        c.d["out"].upload(c.out0)
        step(None)
        M.sync()
        assert np.array_equal(got, c.raw()), past
        c.q = c.d["q"].download(np.float32, c.q.size).reshape(c.q.shape)
        c.k = c.d["k"].download(np.float32, c.k.size).reshape(c.k.shape)
        c.v = c.d["v"].download(np.float32, c.v.size).reshape(c.v.shape)
        c.lens, c.past = [(past, 1)], np.array([past], np.int32)
        c.check(got, past)
    h.lib.hipGraphExecDestroy(e)
    h.lib.hipGraphDestroy(g)
    h.lib.hipStreamDestroy(C.c_void_p(s))


def test_offsets_past_32_bits(M):
    """Pages far into a cache of over 4 GiB: byte offsets need 64 bits."""
    t, kvh, hd, page = E.BF16, 8, 256, 256
    c = Tree(M, [(700, 4)], 8, kvh, hd, t, page=page, seed=12)
    rows = (1 << 32) // (kvh * hd * 2) + 2048           # cache rows: 4 GiB and 8 MiB
    first = rows - c.slots
    a = c.args()
    size = kvh * hd * 2
    k, v = M.DeviceBuffer(rows * size), M.DeviceBuffer(rows * size)
    for big, small in ((k, c.k), (v, c.v)):
        M.check(M.lib.mynah_hip_h2d(big.ptr + first * size, M.ptr(small), small.nbytes), "h2d")
    c.d["pages"].upload((c.pages + first // page).astype(np.int32))
    assert first % page == 0
    a.k_cache, a.v_cache, a.n_slots = k.ptr, v.ptr, rows
    n = M.tree_attention_workspace(a)
    ws = M.DeviceBuffer(n)
    M.tree_attention_dev(a, ws.ptr, n)
    M.sync()
    c.check(c.raw())
