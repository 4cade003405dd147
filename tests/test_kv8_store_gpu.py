"""New rows into an 8-bit cache (mynah_hip_kv8_store_dev): every code and scale, and
every byte beside them, against the definition in 32 bits (kv8_lib)."""
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


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("f", FORMATS)
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("block", [16, 64, 256])
def test_blocks(M, t, f, hd, block):
    print("[case] kv8 store", t, f, hd, block, flush=True)
    c = Kv8(M, [(0, 1), (block - 1, 2), (5, 3 * block), (block, block)], 4, 2, hd, t, f, block,
            seed=block, pad=16)
    c.check_store(c.store())


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("f", FORMATS)
@pytest.mark.parametrize("lens", [[(0, 1)], [(1, 1)], [(63, 1)], [(64, 1)], [(513, 1)], [(0, 700)],
                                  [(300, 7), (0, 0), (65, 12), (15, 1), (16, 1)]], ids=str)
@pytest.mark.parametrize("page", [0, 32])
def test_lengths(M, t, f, lens, page):
    c = Kv8(M, lens, 4, 3, 128, t, f, 16 if page else 64, page, seed=len(lens), extra_rows=2)
    c.check_store(c.store())


@pytest.mark.parametrize("f", FORMATS)
@pytest.mark.parametrize("n,where", [(70, 0), (70, 69), (300, 150), (5000, 3000)])
def test_a_prompt_among_single_tokens(M, f, n, where):
    """So many sequences, one of them long, that blocks are numbered by rows."""
    rng = np.random.default_rng(n)
    lens = [(int(a), int(b)) for a, b in zip(rng.integers(0, 20, n), rng.integers(0, 3, n))]
    lens[where] = (13, 2400 if n < 1000 else 300)
    c = Kv8(M, lens, 2, 1, 64, E.BF16, f, 16, seed=n, max_kv=2413, page=16 if n < 100 else 0,
            extra_rows=3) if n < 1000 else \
        Kv8(M, lens, 2, 1, 64, E.BF16, f, 16, seed=n, extra_rows=3)
    c.check_store(c.store())


@pytest.mark.parametrize("f", FORMATS)
def test_scales_that_grow(M, f):
    # Small committed values under large new ones, and the other way round.
    for size in (1e-3, 1.0, 4.0, 1e4, 1e30):
        c = Kv8(M, [(37, 3), (50, 20), (64, 1)], 2, 2, 64, E.F32, f, 32, seed=3)
        c.kx, c.vx = (c.kx * size).astype(np.float32), (c.vx / size).astype(np.float32)
        c.check_store(c.store(), size)


@pytest.mark.parametrize("f", FORMATS)
def test_token_by_token(M, f):
    """One call a token. Of e4m3 the scales are the one call's over all tokens; of i8 too,
    the earlier codes within half a step of each growth."""
    n = 40
    c = Kv8(M, [(0, n)], 2, 1, 64, E.F32, f, 16, seed=9)
    c.kx *= np.exp(np.linspace(0, 3, n, dtype=np.float32))[:, None]
    whole = c.store()
    one = Kv8(M, [(0, n)], 2, 1, 64, E.F32, f, 16, seed=9)
    one.kx = c.kx
    for i in range(n):
        one.lens, one.past, one.nodes = [(i, 1)], np.array([i], np.int32), np.array([1], np.int32)
        one.start = np.array([i, i + 1], np.int32)
        got = one.store()
        one.check_store(got, i)
        for name in ("k", "v", "ks", "vs"):
            setattr(one, name, got[name])
    used = -(-n // 16)
    for name in ("ks", "vs"):
        assert np.array_equal(got[name][:used], whole[name][:used])


@pytest.mark.parametrize("f", FORMATS)
def test_values_at_the_borders(M, f):
    """Ties, the largest code, zeros, blocks of nothing but zeros, infinities and NaN."""
    c = Kv8(M, [(0, 64)], 2, 1, 64, E.F32, f, 16, seed=1)
    c.kx[:16] = np.float32(0)
    c.kx[16] = np.arange(64, dtype=np.float32) * 0.5 - 16 if f == I8 else np.float32(2.0 ** -9)
    c.kx[17, 0] = 127 if f == I8 else 448
    c.kx[18] = (np.arange(64) + 0.5) / 16
    c.kx[32, 3], c.kx[33, 4], c.kx[34, 5] = np.inf, -np.inf, np.nan
    c.kx[48:] = np.nan
    c.vx[:16] = np.float32(1e-38)
    c.vx[16:32, 7] = np.float32(3e38)
    got = c.store()
    c.check_store(got)
    assert np.isfinite(got["ks"]).all() and (got["ks"] > 0).all()


@pytest.mark.parametrize("f", FORMATS)
def test_old_scales_that_are_none(M, f):
    c = Kv8(M, [(20, 2)] * 5, 2, 1, 64, E.F32, f, 32, seed=2)
    c.ks[:, 0] = [np.nan, np.inf, -1.0, 0.0, 1e-45]
    c.check_store(c.store())


@pytest.mark.parametrize("f", FORMATS)
def test_pages_that_are_none(M, f):
    c = Kv8(M, [(20, 60), (3, 5), (90, 2)], 2, 2, 64, E.BF16, f, 16, page=16, seed=4)
    c.pages[0, 2], c.pages[0, 4], c.pages[1, 0] = -1, 1 << 30, c.slots // 16
    c.check_store(c.store())


def test_counts_that_lie(M):
    c = Kv8(M, [(50, 9), (100, 30)], 2, 1, 64, E.F32, I8, max_nodes=4, max_kv=102)
    c.check_store(c.store())
    c = Kv8(M, [(-5, 3), (10, 2)], 2, 1, 64, E.F32, I8)
    c.check_store(c.store())
    c = Kv8(M, [(20, 3), (10, 2)], 2, 1, 64, E.F32, I8)
    c.start = np.array([-2, 1, 3], np.int32)            # rows -2 .. 0, then 1 and 2
    c.check_store(c.store())
    for start in ([3, 3, 1], [-2147483648, 2147483647, -2147483648]):
        c.start = np.array(start, np.int32)
        got = c.store()
        for n in ("k", "v", "ks", "vs"):
            assert np.array_equal(got[n], getattr(c, n)), (start, n)


def test_rows_past_32_bits(M):
    """Pages far into a cache of over 4 GiB."""
    kvh, hd, page = 8, 256, 256
    c = Kv8(M, [(700, 40)], 8, kvh, hd, E.BF16, I8, 64, page=page, seed=12)
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
    a = c.store_args()
    a.cache.k, a.cache.v, a.cache.n_slots = big["k"].ptr, big["v"].ptr, rows
    a.cache.k_scale, a.cache.v_scale = scales["ks"].ptr, scales["vs"].ptr
    M.kv8_store_dev(a)
    M.sync()
    got = {n: b.download(np.uint8, c.slots * kvh * hd, first * kvh * hd).reshape(c.k.shape)
           for n, b in big.items()}
    got |= {n: b.download(np.float32, c.ks.size, first // 64 * kvh * 4).reshape(c.ks.shape)
            for n, b in scales.items()}
    c.check_store(got)
