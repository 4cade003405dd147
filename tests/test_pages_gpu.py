"""The pages of a cache (mynah_hip_pages_*) against their definition done one
sequence after the other (pages_lib): tables, counts, lengths, status and every byte
of the content."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from pages_lib import Pool
from test_tree_attention_gpu import Hip

pytestmark = pytest.mark.gpu

# Parts of 16-, 4- and 1-byte runs, with and without a gap, below and above 16 KiB.
PARTS = ((4096, 4096), (32, 48), (20, 20), (7, 9), (40_000, 40_000), (16_400, 16_416))


@pytest.fixture(scope="module")
def M():
    import mynah_amd
    mynah_amd.check(mynah_amd.lib.mynah_hip_init(0), "init")
    return mynah_amd


def start(M, past, n_pages, max_pages, page=16, parts=((64, 64),), seed=0):
    """A pool whose sequences hold the given positions, pages anywhere."""
    p = Pool(M, n_pages, len(past), max_pages, page, parts, seed)
    ids = iter(p.rng.permutation(n_pages))
    for b, n in enumerate(past):
        for j in range(-(-n // page)):
            p.pages[b, j] = next(ids)
    p.n_past[:] = past
    p.count()
    return p


def test_beams(M):
    print("[case] pages beams", flush=True)
    p = start(M, [37, 64, 0, 5, 0, 0], 40, 8, parts=PARTS)
    for step in range(6):
        p.both("fork", [0, 1, 0, 3, 1, 0] if step % 2 == 0 else [2, 4, 2, 3, 1, 0], what=step)
        p.both("reserve", [1, 20, 1, 0, 1, 3], what=step)
        p.n_past += np.array([1, 2, 1, 0, 1, 3], np.int32)
        p.d["n_past"].upload(p.n_past)


def test_first_holder_keeps(M):
    # Page held by 1, 3, 4: all ask, so 1 keeps it; then only 3 asks, and copies it.
    for ask in ([0, 1, 0, 1, 1], [0, 0, 0, 1, 0], [0, 0, 0, 1, 1]):
        p = start(M, [8, 20, 3, 0, 0], 24, 4, parts=PARTS[:4])
        p.both("fork", [0, 1, 2, 1, 1])
        p.both("reserve", ask)
        # asked for again: nothing more is needed
        before = p.pages.copy()
        p.both("reserve", ask)
        assert np.array_equal(before, p.pages)


def test_whole_pages_and_nothing_to_copy(M):
    # Positions that end with their page: the next page is new, none is copied.
    p = start(M, [32, 0, 16], 16, 6)
    p.both("fork", [0, 0, 2])
    p.both("reserve", [1, 1, 17])
    assert p.refs[p.pages[0, 0]] == 2 and p.refs[p.pages[0, 2]] == 1


def test_permuted_emptied_and_odd_sources(M):
    p = start(M, [10, 20, 30, 40], 12, 4)
    p.both("fork", [3, 2, 1, 0])
    p.both("fork", [1, -1, 7, 3])
    p.both("fork", [-2147483648, 2147483647, 0, 0])
    assert p.n_past.tolist() == [0, 0, 30, 30] and sorted(p.refs)[-3:] == [0, 2, 2]


def test_too_few_pages_and_too_long(M):
    """Nothing changes, and the status says how many were missing."""
    p = start(M, [30, 47, 16], 8, 4, parts=PARTS[:2])
    for ask in ([3, 18, 1], [100, 1, 1], [1000, 2000, 3000], [2147483647, 0, 2147483647]):
        before = p.pages.copy()
        p.both("reserve", ask, what=ask)
        assert np.array_equal(before, p.pages) == bool(p.status.any())
        p.both("release", p.n_past)
    p.both("reserve", [0, -5, 0])
    assert not p.status.any()


def test_release(M):
    p = start(M, [70, 33, 16, 0], 24, 6)
    p.both("reserve", [20, 30, 1, 5])
    p.both("release", [64, -1, 16, 0])
    p.both("release", [65, 1000, 0, 2147483647])
    p.both("release", [0, 0, 0, 0])
    assert not p.refs.any() and (p.pages == -1).all()


@pytest.mark.parametrize("live", [0, 1, 7, 30, 63, 64])
def test_compact(M, live):
    p = Pool(M, 64, 5, 16, 16, PARTS, seed=live)
    ids = p.rng.permutation(64)[:live]
    for i, pg in enumerate(ids):
        p.pages[i % 5, i // 5] = pg
    if live > 10:
        p.pages[4, 14:16] = p.pages[0, :2]              # shared
    p.count()
    p.both("compact")
    p.both("compact", what="again")
    assert p.status[1] == 0


def test_copy(M):
    p = Pool(M, 50, 1, 4, 16, PARTS, seed=3)
    p.both("copy", [3, 7, 50, 9, -1], [4, 0, 2, 49, 5])


def test_entries_that_are_no_pages(M):
    p = start(M, [40, 20, 5], 16, 4, parts=PARTS[:3])
    p.pages[0, 1], p.pages[1, 1], p.pages[2, 0] = 1 << 30, -2147483648, 16
    p.count()
    p.both("fork", [0, 1, 0])
    p.both("reserve", [5, 20, 5])
    p.both("compact")
    p.both("release", [17, 0, 0])


def test_negative_lengths(M):
    p = start(M, [10, 20], 8, 4)
    p.n_past[:] = [-3, -2147483648]
    p.both("reserve", [17, 1])
    p.both("fork", [1, 0])


@pytest.mark.parametrize("seed", range(4))
def test_any_order_of_calls(M, seed):
    rng = np.random.default_rng(seed)
    n, mp = int(rng.integers(2, 12)), int(rng.integers(3, 9))
    p = Pool(M, int(rng.integers(n, n * mp)), n, mp, 16, PARTS[:4], seed)
    for step in range(25):
        op = rng.choice(["fork", "reserve", "reserve", "reserve", "release", "compact"])
        if op == "fork":
            f = np.arange(n)
            some = rng.random(n) < 0.4
            f[some] = rng.integers(-1, n, some.sum())
            p.both("fork", f, what=step)
        elif op == "reserve":
            ask = rng.integers(0, 24, n) * (rng.random(n) < 0.6)
            p.both("reserve", ask, what=step)
            if not p.status.any():
                p.n_past += ask.astype(np.int32)
                p.d["n_past"].upload(p.n_past)
        elif op == "release":
            p.both("release", np.where(rng.random(n) < 0.5, -1, rng.integers(0, 60, n)), what=step)
        else:
            p.both("compact", what=step)


def test_many_sequences_and_pages(M):
    """More of each than the one workgroup's threads take at a time."""
    rng = np.random.default_rng(5)
    past = rng.integers(0, 90, 1500)
    p = start(M, past, 13_001, 12, parts=((4, 4),), seed=5)
    p.both("fork", np.where(rng.random(1500) < 0.3, rng.integers(-1, 1500, 1500), np.arange(1500)))
    p.both("reserve", rng.integers(-1, 80, 1500))
    p.both("release", rng.integers(-20, 90, 1500))
    p.both("compact")
    p.both("reserve", np.full(1500, 40))


def test_a_long_prompt(M):
    p = start(M, [100, 0, 7], 3000, 2500, parts=((16, 16),))
    p.both("fork", [0, 0, 0])
    p.both("reserve", [37_000, 1, 3])


def test_workspace_refused(M):
    p = start(M, [10], 8, 4)
    p.upload()
    for ws, n in ((None, p.need), (p.ws.ptr + 16, p.need), (p.ws.ptr, p.need - 1)):
        for f in ("fork", "reserve"):
            call = getattr(M.lib, f"mynah_hip_pages_{f}_dev")
            assert call(C.byref(p.args), p.ask[0].ptr, ws, n, None) == -1
            assert b"workspace" in M.lib.mynah_hip_last_error()
        assert M.lib.mynah_hip_pages_compact_dev(C.byref(p.args), ws, n, None) == -1
    p.check(("", "reserve"))


def test_captured_step(M):
    """fork, reserve and compact in one captured graph, replayed while what they ask for
    moves on, against the definition."""
    h = Hip()
    p = start(M, [37, 12, 0, 0], 30, 8, parts=PARTS[:4])
    p.upload()
    s = h.stream()
    new = M.DeviceBuffer.from_array(np.zeros(4, np.int32))

    def step():
        M.pages_fork_dev(p.args, p.ask[0].ptr, p.ws.ptr, p.need, s)
        M.pages_reserve_dev(p.args, new.ptr, p.ws.ptr, p.need, s)
        M.pages_compact_dev(p.args, p.ws.ptr, p.need, s)

    g, e = h.capture(s, step)
    for source, ask in (([0, 1, 0, 1], [1, 1, 1, 1]), ([1, 0, 3, 2], [0, 9, 20, 0]),
                        ([0, -1, 0, 0], [3, 3, 3, 3]), ([3, 3, 3, 3], [1, 0, 0, 40])):
        p.ask[0].upload(np.array(source, np.int32))
        new.upload(np.array(ask, np.int32))
        assert h.lib.hipGraphLaunch(e, C.c_void_p(s)) == 0
        M.check(M.lib.mynah_hip_sync(s), "sync")
        p.fork(source)
        p.reserve(ask)
        p.compact()
        p.check((ask, "compact"))
    h.lib.hipGraphExecDestroy(e)
    h.lib.hipGraphDestroy(g)
    h.lib.hipStreamDestroy(C.c_void_p(s))


def test_content_past_32_bits(M):
    """Pages far into a pool of over 4 GiB."""
    size, n = 1 << 20, 4200
    mem = M.DeviceBuffer(size * n)
    p = Pool(M, n, 1, 4, 16, ((8, 8),))
    p.upload()
    rows = np.array([[mem.ptr, size, size]], np.uint64)
    p.d["parts"].upload(rows)
    x = p.rng.integers(0, 256, size).astype(np.uint8)
    mem.upload(x, 4199 * size)
    p.call("copy", [4199, 4198], [3, 4197])
    M.sync()
    assert np.array_equal(mem.download(np.uint8, size, 3 * size), x)
    p.call("copy", [3], [4196])
    M.sync()
    assert np.array_equal(mem.download(np.uint8, size, 4196 * size), x)
