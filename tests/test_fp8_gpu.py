"""The 8-bit floating point quantiser and product (mynah_hip_fp8_quantize_dev,
mynah_hip_fp8_matmat_dev).

The quantiser is held to its definition bit for bit. The product against 64 bits:
with S = sum_b xs ws sum |xq| |w|, an f32 output sums 128 exact products in f32
(each addition within u = 2^-24 of its partial sum), then nb blocks with two
scales: (128 + nb + 4) u S. For 16-bit outputs the inner sums may come from the
8-bit matrix instructions, which drop what lies more than 16 bits under the
largest of a block's products: at most 2^-16 of it for each of 128 products;
the output's own rounding is half a step."""
from __future__ import annotations

import numpy as np
import pytest

import elem_lib as E

pytestmark = pytest.mark.gpu
U = E.U


@pytest.fixture(scope="module")
def M():
    import mynah_amd
    mynah_amd.check(mynah_amd.lib.mynah_hip_init(0), "init")
    return mynah_amd


def blocks(x, cols):
    nb = -(-cols // 128)
    return np.pad(x, ((0, 0), (0, nb * 128 - cols))).reshape(x.shape[0], nb, 128)


def quantized(x):
    """The definition: every operation rounded to f32."""
    n, cols = x.shape
    b = blocks(x, cols)
    with np.errstate(invalid="ignore", over="ignore"):
        amax = np.maximum(np.nanmax(np.abs(b), -1), np.float32(2.0 ** -100)).astype(np.float32)
        inv = (np.float32(448.0) * (np.float32(1.0) / amax)).astype(np.float32)
        codes = E.to_e4m3(b * inv[..., None]).reshape(n, -1)[:, :cols]
        return codes, amax * (np.float32(1.0) / np.float32(448.0))


@pytest.mark.parametrize("t", [E.F32, E.F16, E.BF16])
@pytest.mark.parametrize("tokens,cols,pad", [(1, 128, 0), (3, 16, 16), (37, 2560, 0), (5, 1040, 8),
                                             (700, 272, 0)])
def test_quantize(M, t, tokens, cols, pad):
    print("[case] quantize", t, tokens, cols, pad, flush=True)
    rng = np.random.default_rng(tokens * cols)
    x = rng.standard_normal((tokens, cols + pad)) * np.exp(rng.standard_normal(cols + pad))
    x[0, :16] = 0
    if tokens > 2:
        x[1, :min(cols, 128)] = 0                        # a block of zeros
        x[2, :cols] *= 1e-6
    x = E.encode(x, t)
    d = M.DeviceBuffer.from_array(x)
    nb = -(-cols // 128)
    q, s = M.DeviceBuffer(tokens * cols), M.DeviceBuffer(4 * tokens * nb)
    M.fp8_quantize_dev(t, d.ptr, cols + pad, tokens, cols, q.ptr, s.ptr)
    M.sync()
    codes, scales = quantized(E.decode(x, t)[:, :cols].astype(np.float32))
    assert np.array_equal(s.download(np.float32, tokens * nb).reshape(tokens, nb), scales)
    got = q.download(np.uint8, tokens * cols).reshape(tokens, cols)
    assert np.array_equal(E.E4M3[got], E.E4M3[codes])


def test_quantize_not_finite(M):
    x = np.ones((3, 256), np.float32)
    x[0, 5], x[1, 130], x[2, 0] = np.nan, np.inf, 3e38
    d, q, s = M.DeviceBuffer.from_array(x), M.DeviceBuffer(3 * 256), M.DeviceBuffer(24)
    M.fp8_quantize_dev(0, d.ptr, 256, 3, 256, q.ptr, s.ptr)
    M.sync()
    v = E.E4M3[q.download(np.uint8, 768).reshape(3, 256)]
    sc = s.download(np.float32, 6).reshape(3, 2)
    assert np.isnan(v[0, 5]) and np.isnan(v[0]).sum() == 1 and sc[0, 0] == np.float32(1 / 448)
    assert np.isinf(sc[1, 1]) and np.isnan(v[1, 130]) and np.all(v[1, :128] == 448)
    assert v[2, 0] == 448 and np.all(v[2, 1:128] == 0)


def operands(rng, rows, cols, tokens):
    nr, nb = -(-rows // 128), -(-cols // 128)
    w = E.to_e4m3(np.clip(rng.standard_normal((rows, cols)) * 90, -448, 448))
    xq = E.to_e4m3(np.clip(rng.standard_normal((tokens, cols)) * 110, -448, 448))
    ws = (2.0 ** rng.uniform(-1, 1, (nr, nb)) / 4000).astype(np.float32)
    xs = np.exp(rng.standard_normal((tokens, nb)) - 3).astype(np.float32)
    return w, ws, xq, xs


def expected(w, ws, xq, xs):
    """(y, S, T): S as in the module's note, T the same of each block's largest
    product, 128 times."""
    rows, cols = w.shape
    y = np.zeros((xq.shape[0], rows))
    s, t = np.zeros_like(y), np.zeros_like(y)
    wd, xd = blocks(E.E4M3[w], cols), blocks(E.E4M3[xq], cols)
    for b in range(ws.shape[1]):
        scale = xs[:, b, None].astype(np.float64) * np.repeat(ws[:, b], 128)[None, :rows]
        a, x = wd[:, b], xd[:, b]
        y += (x @ a.T) * scale
        s += (np.abs(x) @ np.abs(a).T) * scale
        t += 128 * np.outer(np.abs(x).max(1), np.abs(a).max(1)) * scale
    return y, s, t


def tolerance(y, s, t, nb, out):
    tol = (128 + nb + 4) * U * s + E.rounded(y, out)
    return tol if out == E.F32 else tol + 2.0 ** -16 * t


SHAPES = [  # rows, cols, tokens
    (1, 16, 1), (16, 128, 1), (130, 256, 1), (100, 144, 2), (257, 640, 5), (64, 2560, 16),
    (48, 1040, 17), (300, 384, 32), (129, 1168, 33), (1024, 512, 64), (200, 256, 65),
    (384, 128, 130), (513, 912, 127), (256, 1024, 300), (1000, 2048, 257), (640, 272, 1000),
    (9000, 272, 17), (9000, 144, 40), (4128, 1040, 64), (8208, 400, 33),   # few, in tiles
]


@pytest.mark.parametrize("out", [E.F32, E.F16, E.BF16])
@pytest.mark.parametrize("rows,cols,tokens", SHAPES)
def test_product(M, out, rows, cols, tokens):
    print("[case] fp8", out, rows, cols, tokens, flush=True)
    rng = np.random.default_rng(rows * 7 + cols + tokens)
    w, ws, xq, xs = operands(rng, rows, cols, tokens)
    B = M.DeviceBuffer.from_array
    d = [B(a) for a in (w, ws, xq, xs)]
    y0 = E.encode(np.full(tokens * rows + 64, 5.0), out)
    y = B(y0)
    M.fp8_matmat_dev(d[0].ptr, d[1].ptr, rows, cols, d[2].ptr, d[3].ptr, out, y.ptr, tokens)
    M.sync()
    raw = y.download(E.NP[out], y0.size)
    assert np.all(E.decode(raw[tokens * rows:], out) == 5.0)
    got = E.decode(raw[:tokens * rows], out).reshape(tokens, rows)
    want, s, t = expected(w, ws, xq, xs)
    bad = ~(np.abs(got - want) <= tolerance(want, s, t, ws.shape[1], out))
    assert not bad.any(), (int(bad.sum()), float(np.max(np.abs(got - want))))
    M.fp8_matmat_dev(d[0].ptr, d[1].ptr, rows, cols, d[2].ptr, d[3].ptr, out, y.ptr, tokens)
    M.sync()
    assert np.array_equal(raw.view(np.uint8), y.download(E.NP[out], y0.size).view(np.uint8))


@pytest.mark.parametrize("tokens", [1, 40, 200])
def test_product_not_finite(M, tokens):
    # A NaN weight or activation stays in its own rows and tokens.
    rows, cols = 150, 272
    w, ws, xq, xs = operands(np.random.default_rng(3), rows, cols, tokens)
    w[17, 200] = 0x7F
    xs[tokens - 1, 0] = np.inf
    B = M.DeviceBuffer.from_array
    d = [B(a) for a in (w, ws, xq, xs)]
    for out in (E.F32, E.BF16):
        y = M.DeviceBuffer(tokens * rows * E.SIZE[out])
        M.fp8_matmat_dev(d[0].ptr, d[1].ptr, rows, cols, d[2].ptr, d[3].ptr, out, y.ptr, tokens)
        M.sync()
        v = E.decode(y.download(E.NP[out], tokens * rows), out).reshape(tokens, rows)
        odd = np.zeros(v.shape, bool)
        odd[:, 17] = odd[tokens - 1] = True
        assert np.array_equal(~np.isfinite(v), odd)
