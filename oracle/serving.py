"""The serving operators (include/hc_b200_kernels.h) in NumPy, in 64 bits.

Test infrastructure: written from the formulas alone, element by element where
that is clearest.  8-bit outputs are returned as the real numbers before
rounding, with their scales, so that a test can say how far a stored value may
lie from them.
"""

from __future__ import annotations

import numpy as np

PEAK = {"int8": 127.0, "e4m3": 448.0}


def add_rms_norm(x, residual, gain, eps):
    """(y, s) of rows x + residual; all float64."""
    s = x if residual is None else x + residual
    return s / np.sqrt((s * s).mean(axis=1, keepdims=True) + eps) * gain, s


def group_scales(y, group, store):
    """Scale of each row and group of columns, [rows, groups]."""
    rows, cols = y.shape
    width = group if 0 < group < cols else cols
    starts = range(0, cols, width)
    return np.stack([np.abs(y[:, c:c + width]).max(axis=1) for c in starts], axis=1) / PEAK[store]


def widen(scale, group, cols):
    """A scale per row and group -> one per element."""
    width = group if 0 < group < cols else cols
    return np.repeat(scale, width, axis=1)[:, :cols]


def e4m3_values():
    """The value of each of the 256 bit patterns of the 8-bit float."""
    out = np.empty(256)
    for b in range(256):
        sign = -1.0 if b & 128 else 1.0
        exp, frac = (b >> 3) & 15, b & 7
        if exp == 15 and frac == 7:
            out[b] = np.nan
        else:
            out[b] = sign * (frac / 8 * 2.0 ** -6 if exp == 0 else (1 + frac / 8) * 2.0 ** (exp - 7))
    return out


def stored_values(raw, store):
    """Bytes (any integer view) -> the numbers they stand for, before the scale."""
    if store == "int8":
        return raw.view(np.int8).astype(np.float64)
    return e4m3_values()[raw.view(np.uint8)]


def unpack_w4(w, scale, zero, k, group):
    """Weights [N, K] in float64 of the packed bytes w [N, ceil(K / 2)]."""
    n = w.shape[0]
    u = np.empty((n, 2 * w.shape[1]))
    u[:, 0::2] = w & 15
    u[:, 1::2] = w >> 4
    u = u[:, :k]
    z = np.full(scale.shape, 8.0) if zero is None else zero.astype(np.float64)
    return (u - np.repeat(z, group, axis=1)[:, :k]) * np.repeat(scale, group, axis=1)[:, :k]
