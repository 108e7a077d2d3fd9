"""numpy restatement of the 8-bit cache format and of attention over it, in 64 bits, for the tests only.

A row x[0 .. D) of one token and KV head: the scale s is the smallest power of two >= 2^-126 with
max|x| <= 448 s over the finite elements (a row of zeros: 2^-126), kept as the E8M0 byte log2(s) + 127; the
codes are the OCP e4m3 values nearest to x / s, ties to even; what is not finite becomes NaN.

``E4M3`` lists the 256 codes' values from the format's definition: sign, 4 exponent bits of bias 7, 3 mantissa
bits, subnormals m * 2^-9, and 0x7F / 0xFF NaN.
"""
from __future__ import annotations

import numpy as np


def _e4m3_table() -> np.ndarray:
    out = np.empty(256)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        v = np.nan if (e, m) == (15, 7) else (m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10))
        out[c] = -v if c & 128 else v
    return out


E4M3 = _e4m3_table()


def quantise(x: np.ndarray) -> tuple:
    """x [..., D] (float64 values) -> (codes uint8 [..., D], scale bytes uint8 [...])."""
    x = np.asarray(x, dtype=np.float64)
    fine = np.isfinite(x)
    amax = np.max(np.where(fine, np.abs(x), 0.0), axis=-1)
    m, e = np.frexp(amax / 448.0)          # amax / 448 = m 2^e, 1/2 <= m < 1 (0: 0, 0); exact but for the / 7
    e = np.where(np.ldexp(448.0, e - 1) >= amax, e - 1, e)
    e = np.where(amax > 0, np.maximum(e, -126), -126)
    y = np.abs(np.ldexp(np.where(fine, x, 0.0), -e[..., None]))
    mags = E4M3[:127]                      # 0 .. 448, increasing: a code is its value's rank
    hi = np.clip(np.searchsorted(mags, y), 0, 126)
    lo = np.maximum(hi - 1, 0)
    up = (mags[hi] - y < y - mags[lo]) | ((mags[hi] - y == y - mags[lo]) & (hi % 2 == 0))
    code = np.where(mags[hi] == y, hi, np.where(up, hi, lo)).astype(np.uint8)
    code = np.where(np.signbit(x), code | 128, code).astype(np.uint8)
    return np.where(fine, code, np.where(np.signbit(x), 0xFF, 0x7F)).astype(np.uint8), (e + 127).astype(np.uint8)


def values(codes: np.ndarray, scales: np.ndarray) -> np.ndarray:
    """codes [pages, ..., ps, H, D], scales [pages, ..., H, ps] (bytes) -> float64 values."""
    s = np.ldexp(1.0, scales.astype(np.int64) - 127)
    return E4M3[codes] * np.swapaxes(s, -1, -2)[..., None]


def norm_rotate(x, w, cos, sin, eps):
    """x [n, H, D] normalised by its rows' root mean square (w None: not), then rotated; cos / sin [n, D]."""
    x = np.asarray(x, dtype=np.float64)
    if w is not None:
        x = x / np.sqrt(np.mean(x * x, axis=-1, keepdims=True) + eps) * w
    h = x.shape[-1] // 2
    return x * cos[:, None] + np.concatenate([-x[..., h:], x[..., :h]], axis=-1) * sin[:, None]


def attend(q, k, v, sm_scale):
    """One query token: q [Hq, D], k / v [L, Hkv, D] -> (out [Hq, D], sum p |v| [Hq, D], the largest sum |q k| a head)."""
    hq, d = q.shape
    L, hkv, _ = k.shape
    if L == 0:
        return np.zeros((hq, d)), np.zeros((hq, d)), np.zeros((hq, 1))
    g = hq // hkv
    out, mag, big = np.empty((hq, d)), np.empty((hq, d)), np.empty((hq, 1))
    for a in range(hq):
        h = a // g
        s = k[:, h] @ q[a] * sm_scale
        p = np.exp(s - s.max())
        p /= p.sum()
        out[a], mag[a] = p @ v[:, h], p @ np.abs(v[:, h])
        big[a] = np.max(np.abs(k[:, h]) @ np.abs(q[a])) * sm_scale
    return out, mag, big
