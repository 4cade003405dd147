"""Element types of the operator tests in numpy: f32, f16, bf16 (as uint16) and
e4m3 (as uint8), rounding to nearest, ties to even, and how far a rounding may
be off."""
from __future__ import annotations

import numpy as np

F32, F16, BF16 = 0, 1, 30
NAME = {F32: "f32", F16: "f16", BF16: "bf16"}
NP = {F32: np.float32, F16: np.float16, BF16: np.uint16}
SIZE = {F32: 4, F16: 2, BF16: 2}
# Half a step relative to the value, and below the smallest normal absolutely.
HALF = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}
TINY = {F32: 2.0 ** -149, F16: 2.0 ** -25, BF16: 2.0 ** -133}
U = 2.0 ** -24


def encode(x, t):
    """Values as the stored type's array."""
    x = np.asarray(x, np.float32)
    if t == F32:
        return x
    if t == F16:
        with np.errstate(over="ignore"):
            return x.astype(np.float16)
    b = x.view(np.uint32).astype(np.uint64)
    r = ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def decode(a, t):
    """The stored values in 64 bits."""
    if t == BF16:
        return (a.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return a.astype(np.float64)


def rounded(x, t):
    """Bound of one rounding to t of values x."""
    return HALF[t] * np.abs(x) + TINY[t]


# e4m3: sign, four exponent bits (bias 7), three mantissa bits; 0x7f is NaN.
_c = np.arange(256)
_e, _m = (_c >> 3) & 15, _c & 7
E4M3 = np.where(_e > 0, (8.0 + _m) * 2.0 ** (_e - 10.0), _m * 2.0 ** -9.0)
E4M3 = np.where(_c & 128, -E4M3, E4M3)
E4M3[[127, 255]] = np.nan
_pos = E4M3[:127]
_mid = (_pos[1:] + _pos[:-1]) / 2


def to_e4m3(x):
    """Codes of values up to 448 (464 and beyond are not asked for)."""
    a = np.abs(np.asarray(x, np.float64))
    k = np.searchsorted(_mid, a, side="left")         # at a midpoint: the lower code
    tie = (k < 126) & (a == _mid[np.minimum(k, 125)]) & (k % 2 == 1)
    k = np.where(tie, k + 1, k)
    k = np.where(np.isnan(a), 127, k)
    return (k | np.where(np.signbit(x), 128, 0)).astype(np.uint8)
