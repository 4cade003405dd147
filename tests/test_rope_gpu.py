"""Rotary positions and the q/k norms with the rotation and the cache store
(mynah_hip_rope_dev, mynah_hip_qk_norm_rope_dev) against the formulas in 64
bits.

Tolerances, u = 2^-24: cos and sin come within 4 u of theirs (the reduced
angle's rounding 0.8 u, the sums' two last roundings, mscale), their products
and the sum add 2 u each: 6 u (|x0| + |x1|) mscale; the angle's product with
1 / (2 pi) may turn it by its size times 2^-52. A norm before that: the sum of
squares of at most 512 values is a tree of 14 roundings, halved by the root, plus
those of the mean, the root, the quotient and the two products: 12 u more. The
store adds half a step of its type."""
from __future__ import annotations

import ctypes as C

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


def turned(x, layout, rot, freqs, mscale, pos):
    """(x [tokens][heads][hd] rotated, the bound of the rotation's own error in u,
    and in what the angle may be off)."""
    a = np.asarray(pos, np.float64)[:, None, None] * freqs
    c, s = np.cos(a) * mscale, np.sin(a) * mscale
    y, size, far = x.copy(), np.abs(x), np.zeros_like(x)
    lo = (slice(0, rot // 2), slice(rot // 2, rot)) if layout == 0 else \
        (slice(0, rot, 2), slice(1, rot, 2))
    x0, x1 = x[..., lo[0]], x[..., lo[1]]
    y[..., lo[0]], y[..., lo[1]] = x0 * c - x1 * s, x1 * c + x0 * s
    for i in lo:
        size[..., i] = (np.abs(x0) + np.abs(x1)) * mscale
        far[..., i] = size[..., i] * np.abs(a) * 2.0 ** -52
    return y, size, far


def close(got, want, tol, what):
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (what, int(bad.sum()), float(np.max(np.abs(got - want) / tol)))


CASES = [  # type, layout, tokens, heads, hd, rot, first position, strides padded by
    (E.F32, 0, 1, 1, 8, 8, 0, 0), (E.F32, 0, 1, 32, 128, 128, 40959, 0),
    (E.BF16, 1, 7, 3, 64, 32, 5, 0), (E.F16, 0, 5, 2, 80, 40, 1000, 8),
    (E.F32, 1, 3, 5, 96, 96, 70000, 4), (E.BF16, 0, 33, 4, 256, 256, 1 << 20, 0),
    (E.F16, 1, 2, 7, 512, 504, 3, 0), (E.BF16, 0, 9, 2, 72, 8, 11, 1),
    (E.F32, 1, 4, 3, 128, 64, 2000, 3), (E.F16, 0, 2, 1, 24, 16, (1 << 31) - 2, 0),
    (E.F32, 0, 700, 40, 64, 64, 17, 0), (E.BF16, 1, 2100, 33, 128, 128, 0, 0),
]


@pytest.mark.parametrize("case", CASES)
def test_rope(M, case):
    t, layout, n, heads, hd, rot, first, pad = case
    print("[case] rope", case, flush=True)
    freqs, mscale = M.rope_freqs(rot, 1e6, M.ROPE_YARN if rot >= 64 else M.ROPE_NONE, 4.0,
                                 32768.0, 32.0, 1.0)
    freqs = freqs[:rot // 2]
    rng = np.random.default_rng(hash(case) % 1000)
    xh, xt = hd + pad, (hd + pad) * heads + 2 * pad
    yh, yt = hd + 2 * pad, (hd + 2 * pad) * heads
    x = E.encode(rng.standard_normal((n, xt)), t)
    pos = np.minimum(first + np.arange(n), (1 << 31) - 1).astype(np.int32)
    rng.shuffle(pos)
    y0 = E.encode(np.full((n, yt), 7.5), t)
    xd, yd = M.DeviceBuffer.from_array(x), M.DeviceBuffer.from_array(y0)
    fd, pd = M.DeviceBuffer.from_array(freqs), M.DeviceBuffer.from_array(pos)
    M.rope_dev(t, layout, xd.ptr, xt, xh, yd.ptr, yt, yh, n, heads, hd, rot, fd.ptr, mscale,
               pd.ptr)
    M.sync()
    y = yd.download(E.NP[t], n * yt).reshape(n, yt)
    rows = E.decode(x, t)[:, :heads * xh].reshape(n, heads, xh)[..., :hd]
    want, size, far = turned(rows, layout, rot, freqs, mscale, pos)
    got = E.decode(y, t).reshape(n, heads, yh)
    close(got[..., :hd], want, 6 * U * size + far + E.rounded(want, t), "rope")
    assert np.all(got[..., hd:] == 7.5)                  # between the rows nothing is written
    # values past rot_dim are the same bits
    raw = x[:, :heads * xh].reshape(n, heads, xh)[..., rot:hd]
    assert np.array_equal(y.reshape(n, heads, yh)[..., rot:hd], raw)


def test_rope_in_place_back_and_without_positions(M):
    n, heads, hd = 37, 6, 128
    freqs, _ = M.rope_freqs(hd, 1e6)
    x = np.random.default_rng(1).standard_normal((n, heads, hd)).astype(np.float32)
    d, f = M.DeviceBuffer.from_array(x), M.DeviceBuffer.from_array(freqs)
    M.rope_dev(0, 0, d.ptr, heads * hd, hd, d.ptr, heads * hd, hd, n, heads, hd, hd, f.ptr, 1.0,
               None)
    M.sync()
    want, size, far = turned(x.astype(np.float64), 0, hd, freqs, 1.0, np.arange(n))
    got = d.download(np.float32, x.size).reshape(x.shape)
    close(got.astype(np.float64), want, 6 * U * size + far + E.rounded(want, 0), "in place")
    back = M.DeviceBuffer.from_array(-np.arange(n, dtype=np.int32))
    M.rope_dev(0, 0, d.ptr, heads * hd, hd, d.ptr, heads * hd, hd, n, heads, hd, hd, f.ptr, 1.0,
               back.ptr)
    M.sync()
    two, size, _ = turned(got.astype(np.float64), 0, hd, freqs, 1.0, -np.arange(n))
    got = d.download(np.float32, x.size).reshape(x.shape)
    close(got.astype(np.float64), two, 6 * U * size + E.rounded(two, 0), "back")
    # there and back: each rotation's own error, the first one's turned
    close(got.astype(np.float64), x, 2 * (6 + 1) * U * 2 * size, "there and back")


def test_rope_not_finite(M):
    # A NaN or an infinity stays in its own pair.
    hd = 64
    x = np.ones((1, 2, hd), np.float32)
    x[0, 0, 3], x[0, 1, 40] = np.nan, np.inf
    freqs, _ = M.rope_freqs(hd, 1e4)
    d, f = M.DeviceBuffer.from_array(x), M.DeviceBuffer.from_array(freqs)
    p = M.DeviceBuffer.from_array(np.array([5], np.int32))
    M.rope_dev(0, 0, d.ptr, 2 * hd, hd, d.ptr, 2 * hd, hd, 1, 2, hd, hd, f.ptr, 1.0, p.ptr)
    M.sync()
    y = d.download(np.float32, x.size).reshape(2, hd)
    odd = np.zeros((2, hd), bool)
    odd[0, [3, 35]] = odd[1, [8, 40]] = True
    assert np.array_equal(~np.isfinite(y), odd)


QK_CASES = [  # type, out, layout, tokens, heads, kv heads, hd, rot, slots, pad
    (E.F32, E.F32, 0, 1, 16, 8, 128, 128, 4, 0), (E.BF16, E.BF16, 0, 5, 8, 2, 128, 128, 9, 0),
    (E.F32, E.BF16, 0, 33, 32, 8, 128, 128, 64, 0), (E.F32, E.F16, 1, 3, 4, 1, 64, 32, 7, 1),
    (E.F16, E.F32, 1, 2, 3, 3, 80, 40, 2, 4), (E.BF16, E.F16, 0, 4, 7, 1, 256, 128, 5, 8),
    (E.F16, E.BF16, 0, 2, 2, 1, 96, 96, 3, 0), (E.BF16, E.F32, 1, 6, 5, 5, 8, 8, 11, 0),
    (E.F16, E.F16, 0, 700, 40, 8, 64, 64, 800, 0), (E.F32, E.F32, 1, 3, 2, 2, 512, 512, 5, 0),
]


def run_qk(M, case, norms=True, slots=None, with_v=True):
    t, ot, layout, n, heads, kvh, hd, rot, n_slots, pad = case
    rng = np.random.default_rng(hash(case) % 997)
    row = (heads + 2 * kvh) * hd + pad
    x = E.encode(rng.standard_normal((n, row)) * 3, t)
    qw, kw = (1 + 0.2 * rng.standard_normal((2, hd))).astype(np.float32)
    freqs, mscale = M.rope_freqs(rot, 1e6, M.ROPE_LINEAR, 2.0, mscale=1.1)
    freqs = freqs[:rot // 2]
    pos = rng.integers(0, 5000, n).astype(np.int32)
    if slots is None:
        slots = rng.permutation(n_slots)[:n].astype(np.int32)
        if n > 3:
            slots[1], slots[2] = -1, n_slots           # padding rows
    ss = kvh * hd + pad
    kc = E.encode(rng.standard_normal((n_slots, ss)), ot)
    vc = E.encode(rng.standard_normal((n_slots, ss)), ot)
    B = M.DeviceBuffer.from_array
    d = [B(a) for a in (x, qw, kw, freqs, pos, slots, kc, vc)]
    q = B(E.encode(np.full((n, heads * hd + pad), -3.0), ot))
    size = E.SIZE[t]
    a = M.QkNormRope(type=t, out_type=ot, layout=layout, n_heads=heads, n_kv_heads=kvh,
                     head_dim=hd, rot_dim=rot, tokens=n, q=d[0].ptr,
                     k=d[0].ptr + heads * hd * size,
                     v=d[0].ptr + (heads + kvh) * hd * size if with_v else None, q_stride=row,
                     k_stride=row, v_stride=row, q_norm=d[1].ptr if norms else None,
                     k_norm=d[2].ptr if norms else None, eps=1e-5, mscale=mscale, freqs=d[3].ptr,
                     pos=d[4].ptr, slots=d[5].ptr, n_slots=n_slots, q_out=q.ptr,
                     q_out_stride=heads * hd + pad, k_cache=d[6].ptr, v_cache=d[7].ptr,
                     slot_stride=ss)
    M.qk_norm_rope_dev(a)
    M.sync()
    get = lambda b, r, c: b.download(E.NP[ot], r * c).reshape(r, c)  # noqa: E731
    qo, ko, vo = get(q, n, heads * hd + pad), get(d[6], n_slots, ss), get(d[7], n_slots, ss)
    v = E.decode(x, t)[:, :(heads + 2 * kvh) * hd].reshape(n, heads + 2 * kvh, hd)

    def expect(y, w):
        size0 = y
        if norms:
            y = y / np.sqrt((y * y).mean(-1, keepdims=True) + 1e-5) * w.astype(np.float64)
        del size0
        return turned(y, layout, rot, freqs, mscale, pos)

    want, size, far = expect(v[:, :heads], qw)
    got = E.decode(qo, ot)[:, :heads * hd].reshape(n, heads, hd)
    close(got, want, 18 * U * size + far + E.rounded(want, ot), "q")
    if pad:
        assert np.all(E.decode(qo, ot)[:, heads * hd:] == -3.0)
    want, size, far = expect(v[:, heads:heads + kvh], kw)
    kept_k, kept_v = kc.copy(), vc.copy()
    for i, s in enumerate(slots):
        if not 0 <= s < n_slots:
            continue
        got = E.decode(ko[s, :kvh * hd], ot).reshape(kvh, hd)
        close(got, want[i], 18 * U * size[i] + far[i] + E.rounded(want[i], ot), "k")
        kept_k[s, :kvh * hd] = ko[s, :kvh * hd]
        if with_v:
            kept_v[s, :kvh * hd] = E.encode(v[i, heads + kvh:], ot).reshape(-1)
    assert np.array_equal(kept_k.view(np.uint8), ko.view(np.uint8))   # other slots untouched
    assert np.array_equal(kept_v.view(np.uint8), vo.view(np.uint8))   # values: one rounding


@pytest.mark.parametrize("case", QK_CASES)
def test_qk_norm_rope(M, case):
    print("[case] qk", case, flush=True)
    run_qk(M, case)


def test_qk_without_norms_or_values(M):
    run_qk(M, QK_CASES[1], norms=False)
    run_qk(M, QK_CASES[2], with_v=False)


def test_qk_all_padding(M):
    run_qk(M, QK_CASES[1], slots=np.full(5, -1, np.int32))


def test_qk_queries_only_and_keys_only(M):
    hd, n = 128, 3
    rng = np.random.default_rng(5)
    x = rng.standard_normal((n, 2 * hd)).astype(np.float32)
    freqs, _ = M.rope_freqs(hd, 1e4)
    d, f = M.DeviceBuffer.from_array(x), M.DeviceBuffer.from_array(freqs)
    out = M.DeviceBuffer.from_array(np.zeros((n, 2 * hd), np.float32))
    want, size, far = turned(x.astype(np.float64).reshape(n, 2, hd), 0, hd, freqs, 1.0,
                             np.arange(n))
    tol = 6 * U * size + far + E.rounded(want, 0)
    base = dict(type=0, out_type=0, layout=0, head_dim=hd, rot_dim=hd, tokens=n, eps=0.0,
                mscale=1.0, freqs=f.ptr)
    for a in (M.QkNormRope(n_heads=2, q=d.ptr, q_stride=2 * hd, q_out=out.ptr,
                           q_out_stride=2 * hd, **base),
              # slots NULL: token t to slot t
              M.QkNormRope(n_kv_heads=2, k=d.ptr, k_stride=2 * hd, k_cache=out.ptr, n_slots=n,
                           slot_stride=2 * hd, **base)):
        M.check(M.lib.mynah_hip_memset(out.ptr, 0, out.nbytes))
        M.check(M.lib.mynah_hip_qk_norm_rope_dev(C.byref(a), None))
        M.sync()
        close(out.download(np.float32, x.size).reshape(want.shape).astype(np.float64), want, tol,
              "one side")


def test_qk_zero_row_and_nan(M):
    # A zero head normalises to zero (eps), a NaN stays in its own head.
    hd = 64
    x = np.zeros((1, 3, hd), np.float32)
    x[0, 1], x[0, 2] = 1.0, 2.0
    x[0, 1, 7] = np.nan
    freqs, _ = M.rope_freqs(hd, 1e4)
    B = M.DeviceBuffer.from_array
    d, f, w, out = B(x), B(freqs), B(np.ones(hd, np.float32)), B(np.full_like(x, 9.0))
    a = M.QkNormRope(type=0, out_type=0, layout=0, n_heads=3, head_dim=hd, rot_dim=hd, tokens=1,
                     q=d.ptr, q_stride=3 * hd, q_out=out.ptr, q_out_stride=3 * hd, q_norm=w.ptr,
                     eps=1e-6, mscale=1.0, freqs=f.ptr)
    M.qk_norm_rope_dev(a)
    M.sync()
    y = out.download(np.float32, x.size).reshape(3, hd)
    assert np.all(y[0] == 0) and np.all(np.isnan(y[1])) and np.all(np.isfinite(y[2]))
