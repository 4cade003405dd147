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
