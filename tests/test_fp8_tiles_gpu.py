"""The tile kernels of the e4m3 product, each forced in turn (MYNAH_FP8_TILE), over
rows, columns and tokens that end inside a tile and inside a block. Bounds as in
test_fp8_gpu.py."""
from __future__ import annotations

import numpy as np
import pytest

import elem_lib as E
import test_fp8_gpu as F

pytestmark = pytest.mark.gpu
U = E.U


@pytest.fixture(scope="module")
def M():
    import mynah_amd
    mynah_amd.check(mynah_amd.lib.mynah_hip_init(0), "init")
    return mynah_amd


def product(M, w, ws, xq, xs, out):
    """The product, behind which 64 values stay as they were."""
    rows, cols, tokens = w.shape[0], w.shape[1], xq.shape[0]
    d = [M.DeviceBuffer.from_array(a) for a in (w, ws, xq, xs)]
    y0 = E.encode(np.full(tokens * rows + 64, 5.0), out)
    y = M.DeviceBuffer.from_array(y0)
    M.fp8_matmat_dev(d[0].ptr, d[1].ptr, rows, cols, d[2].ptr, d[3].ptr, out, y.ptr, tokens)
    M.sync()
    raw = y.download(E.NP[out], y0.size)
    assert np.all(E.decode(raw[tokens * rows:], out) == 5.0)
    return E.decode(raw[:tokens * rows], out).reshape(tokens, rows)


# Fewer blocks than a tile has buffers, one row of scales, one token in the last
# tile: the copies past the last block find nothing to read.
SHORT = [(1, 16, 65), (1, 128, 129), (130, 272, 257), (64, 400, 17), (257, 1040, 33)]


@pytest.mark.parametrize("tile", range(4))
@pytest.mark.parametrize("rows,cols,tokens", SHORT)
def test_few_blocks(M, monkeypatch, tile, rows, cols, tokens):
    print("[case] fp8 tile", tile, rows, cols, tokens, flush=True)
    monkeypatch.setenv("MYNAH_FP8_TILE", str(tile))
    rng = np.random.default_rng(rows + cols + tokens)
    w, ws, xq, xs = F.operands(rng, rows, cols, tokens)
    got = product(M, w, ws, xq, xs, E.F32)
    want, s, _ = F.expected(w, ws, xq, xs)
    nb = ws.shape[1]
    assert np.all(np.abs(got - want) <= (128 + nb + 4) * U * s + E.rounded(want, E.F32))


RAGGED = [(64, 128, 64), (129, 272, 65), (100, 1168, 130), (513, 912, 127), (1000, 640, 257),
          (257, 2048, 300), (130, 144, 513)]


@pytest.mark.parametrize("out", [E.F32, E.F16, E.BF16])
@pytest.mark.parametrize("tile", range(4))
@pytest.mark.parametrize("rows,cols,tokens", RAGGED)
def test_tiles(M, monkeypatch, out, tile, rows, cols, tokens):
    print("[case] fp8 tile", tile, out, rows, cols, tokens, flush=True)
    monkeypatch.setenv("MYNAH_FP8_TILE", str(tile))
    rng = np.random.default_rng(rows + 3 * cols + tokens)
    w, ws, xq, xs = F.operands(rng, rows, cols, tokens)
    got = product(M, w, ws, xq, xs, out)
    want, s, _ = F.expected(w, ws, xq, xs)
    sums = (128 + ws.shape[1] + 4) * U * s           # then one rounding to the type
    assert np.all(np.abs(got - want) <= sums * (1 + E.HALF[out]) + E.rounded(want, out))


def cancelling(rng, rows, cols, tokens):
    """Whole numbers up to 8 beside two products of 448 x 448 and its negative in each
    block: every sum in f32 is exact (below 2^24), scales are powers of two."""
    nr, nb = -(-rows // 128), -(-cols // 128)
    w = rng.integers(-8, 9, (rows, cols)).astype(np.float64)
    x = rng.integers(-8, 9, (tokens, cols)).astype(np.float64)
    for b in range(nb):
        i, j = b * 128 + rng.choice(min(128, cols - b * 128), 2, replace=False)
        x[:, i] = x[:, j] = 448
        w[:, i] = 448
        w[:, j] = -448
    ws = np.full((nr, nb), 2.0 ** -3, np.float32)
    xs = (2.0 ** rng.integers(-2, 3, (tokens, nb))).astype(np.float32)
    return E.to_e4m3(w), ws, E.to_e4m3(x), xs


@pytest.mark.parametrize("out", [E.F32, E.F16, E.BF16])
@pytest.mark.parametrize("tile", [None, 0, 1, 2, 3])
@pytest.mark.parametrize("tokens", [1, 16, 17, 64, 65, 300])
def test_sums_that_cancel(M, monkeypatch, out, tile, tokens):
    # Sums in 32 bits, whatever the type and the number of tokens.
    rows, cols = 400, 400
    print("[case] fp8 cancelling", tile, out, tokens, flush=True)
    if tile is not None:
        monkeypatch.setenv("MYNAH_FP8_TILE", str(tile))
    w, ws, xq, xs = cancelling(np.random.default_rng(tokens), rows, cols, tokens)
    want, s, _ = F.expected(w, ws, xq, xs)
    assert np.abs(want).max() < 1e-2 * s.max()
    got = product(M, w, ws, xq, xs, out)
    assert np.all(np.abs(got - want) <= (0 if out == E.F32 else E.rounded(want, out)))


@pytest.mark.parametrize("long_side", ["rows", "tokens"])
@pytest.mark.parametrize("tile", [None, 0, 2, 3])
def test_offsets_past_32_bits(M, monkeypatch, long_side, tile):
    """Weights, or activations, of over 4 GiB: the last rows, or tokens, are held to
    their values; what lies before them is whatever the memory held."""
    many, few, cols, tail = 1_050_000, 17 if tile is None else 70, 4112, 300
    print("[case] fp8 offsets", long_side, tile, flush=True)
    if tile is not None:
        monkeypatch.setenv("MYNAH_FP8_TILE", str(tile))
    nb, rng = -(-cols // 128), np.random.default_rng(4)
    rows, tokens = (many, few) if long_side == "rows" else (few, many)
    first = (many - tail) // 128 * 128                   # where a block of scales starts
    tail = many - first
    w, ws, xq, xs = F.operands(rng, tail if rows == many else rows, cols,
                               tail if tokens == many else tokens)
    nr = -(-rows // 128)
    d = [M.DeviceBuffer(n) for n in (rows * cols, 4 * nr * nb, tokens * cols, 4 * tokens * nb)]
    at = [first * cols, first // 128 * nb * 4, 0, 0] if rows == many else \
        [0, 0, first * cols, first * nb * 4]
    assert max(at) > 1 << 32
    for b, o, a in zip(d, at, (w, ws, xq, xs)):
        M.check(M.lib.mynah_hip_h2d(b.ptr + o, M.ptr(a), a.nbytes), "h2d")
    y = M.DeviceBuffer(2 * rows * tokens)
    M.fp8_matmat_dev(d[0].ptr, d[1].ptr, rows, cols, d[2].ptr, d[3].ptr, E.F16, y.ptr, tokens)
    M.sync()
    got = E.decode(y.download(np.float16, rows * tokens), E.F16).reshape(tokens, rows)
    got = got[:, first:] if rows == many else got[first:]
    want, s, _ = F.expected(w, ws, xq, xs)
    ok = np.abs(want) + s < 60_000                       # f16 holds them
    tol = (128 + nb + 4) * U * s * (1 + E.HALF[E.F16]) + E.rounded(want, E.F16)
    assert ok.mean() > 0.9 and np.all(np.abs(got - want)[ok] <= tol[ok])


@pytest.mark.parametrize("out", [E.F32, E.F16, E.BF16])
@pytest.mark.parametrize("tokens", [3, 40, 200])
def test_result_aligned_to_its_type_alone(M, out, tokens):
    rows, cols = 256, 272
    w, ws, xq, xs = F.operands(np.random.default_rng(6), rows, cols, tokens)
    d = [M.DeviceBuffer.from_array(a) for a in (w, ws, xq, xs)]
    y0 = E.encode(np.full(tokens * rows + 8, 5.0), out)
    y, size = M.DeviceBuffer.from_array(y0), E.SIZE[out]
    got = []
    for at in (0, 1):
        y.upload(y0)
        M.fp8_matmat_dev(d[0].ptr, d[1].ptr, rows, cols, d[2].ptr, d[3].ptr, out,
                         y.ptr + at * size, tokens)
        M.sync()
        raw = y.download(E.NP[out], y0.size)
        got.append(raw[at:at + tokens * rows])
        assert np.array_equal(np.delete(raw, np.s_[at:at + tokens * rows]), y0[:8])
    assert np.array_equal(got[0].view(np.uint8), got[1].view(np.uint8))
