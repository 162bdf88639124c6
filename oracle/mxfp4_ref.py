"""numpy restatement of the MXFP4 codec and products in 64 bits — test infrastructure.

E2M1 values with one E8M0 scale per 32 columns.  Written from the format: the scale is found by
comparing powers of two, the code by counting the midpoints below a magnitude.
"""
from __future__ import annotations

import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def quantize(x: np.ndarray, rounding: str) -> tuple[np.ndarray, np.ndarray]:
    """(codes uint8 [..., cols], scale bytes uint8 [..., ceil(cols/32)]) of x [..., cols]."""
    x = np.asarray(x, np.float64)
    cols = x.shape[-1]
    b = np.concatenate([x, np.zeros((*x.shape[:-1], -cols % 32))], -1).reshape(*x.shape[:-1], -1, 32)
    bad = ~np.isfinite(b).all(-1)
    a = np.abs(np.where(bad[..., None], 0, b)).max(-1)
    mant, exp = np.frexp(a)                               # a = mant * 2^exp, mant in [0.5, 1)
    e = exp - 3
    if rounding == "ceil":
        e = e + (mant > 0.75)
    e = np.where(a == 0, -127, np.clip(e, -127, 127))
    m = np.abs(b) * np.exp2(-e.astype(np.float64))[..., None]
    code = np.zeros(m.shape, np.uint8)
    with np.errstate(invalid="ignore"):
        for i in range(7):
            mid = (GRID[i] + GRID[i + 1]) / 2
            code += (m > mid) if i % 2 == 0 else (m >= mid)
    code |= np.signbit(b).astype(np.uint8) << 3
    code[bad] = 0
    s = np.where(bad, 255, e + 127).astype(np.uint8)
    return code.reshape(*x.shape[:-1], -1)[..., :cols], s


def values(codes: np.ndarray, scales: np.ndarray) -> np.ndarray:
    v = GRID[codes & 7] * np.where(codes & 8, -1.0, 1.0)
    s = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    return v * np.repeat(s, 32, -1)[..., : codes.shape[-1]]


def pack(codes: np.ndarray) -> np.ndarray:
    """Row-major bytes, low nibble = even column."""
    c = np.concatenate([codes, np.zeros((*codes.shape[:-1], codes.shape[-1] % 2), np.uint8)], -1)
    return c[..., 0::2] | (c[..., 1::2] << 4)


def swiglu7(z: np.ndarray) -> np.ndarray:
    g = np.minimum(z[..., 0::2], 7.0)
    u = np.clip(z[..., 1::2], -7.0, 7.0)
    return g / (1 + np.exp(-1.702 * g)) * (u + 1)


def product(xv: np.ndarray, wv: np.ndarray, bias=None, activation=None, row_weights=None):
    """(y, bound): act(x w^T + bias) * row_weights in 64 bits and a bound of the error of fp32 sums.

    The terms are exact in fp32.  A sum of K terms takes K/64 accumulation steps of 64 terms,
    each off by at most four units of 2^-23 of the terms' absolute sum; the bias and the weight
    add a rounding each.  SwiGLU7 scales an error in z by at most 1.13 * 8 (gate) and 7 (linear
    part), and adds 2^-18 of |y| for its exponential and quotient."""
    K = xv.shape[-1]
    z = xv @ wv.T
    mag = np.abs(xv) @ np.abs(wv).T
    if bias is not None:
        z = z + bias
        mag = mag + np.abs(bias)
    err = (K / 16 + 8) * 2.0 ** -23 * mag
    if activation == "swiglu7":
        y = swiglu7(z)
        err = 9.04 * err[..., 0::2] + 7 * err[..., 1::2] + 2.0 ** -18 * np.abs(y)
    else:
        y = z
    if row_weights is not None:
        y = y * row_weights[:, None]
        err = err * np.abs(row_weights)[:, None] + 2.0 ** -23 * np.abs(y)
    return y, err
