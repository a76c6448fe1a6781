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


def to_e4m3(x):
    """Nearest 8-bit floats (ties to even, saturating, NaN kept) as bit patterns."""
    x = np.asarray(x, dtype=np.float64)
    mag = np.minimum(np.abs(np.nan_to_num(x, nan=0.0, posinf=448.0, neginf=-448.0)), 448.0)
    expo = np.maximum(np.floor(np.log2(np.where(mag > 0, mag, 1.0))), -6)
    step = 2.0 ** (expo - 3)
    value = np.minimum(np.rint(mag / step) * step, 448.0)
    code = np.searchsorted(e4m3_values()[:127], value).astype(np.uint8)
    code |= np.where(np.signbit(x), 128, 0).astype(np.uint8)
    return np.where(np.isnan(x), np.uint8(127) | (np.signbit(x) * 128).astype(np.uint8), code)


def _quantise(x, store):
    if store == "e4m3":
        return to_e4m3(x)
    q = np.clip(np.rint(np.nan_to_num(x, nan=0.0, posinf=127.0, neginf=-127.0)), -127, 127)
    return q.astype(np.int8).view(np.uint8)


def place(lengths, starts, tokens, width, block, max_new):
    """(row, first position, count) of each sequence's new tokens that have a place."""
    spans = []
    for s, length in enumerate(lengths):
        begin = min(max(starts[s], 0), tokens)
        end = min(max(starts[s + 1], begin), tokens)
        rows = range(begin, end)
        pos = [max(length, 0) - (end - begin) + i for i in range(end - begin)]
        kept = [(r, p) for r, p in zip(rows, pos) if p >= 0][:max_new]
        kept = [(r, p) for r, p in kept if p < width * block]
        spans.append((kept[0][0], kept[0][1], len(kept)) if kept else (begin, 0, 0))
    return spans


def kv_append(cache, scale, new, table, spans, store):
    """Bytes `cache` [pages, heads, block, dim] and `scale` float32 after appending
    `new` float64 [tokens, heads, dim]; every step one float32 operation."""
    cache, scale = cache.copy(), scale.copy()
    pages, heads, block, dim = cache.shape
    one = np.float32
    for s, (row, first, count) in enumerate(spans):
        for b in range(first // block, (first + count - 1) // block + 1 if count else 0):
            lo, hi = max(first, b * block), min(first + count, (b + 1) * block)
            page = table[s][b]
            if not 0 <= page < pages:
                continue
            for h in range(heads):
                x = new[row + lo - first: row + hi - first, h].astype(one)
                top = np.abs(np.where(np.isfinite(x), x, 0)).max(initial=one(0))
                need = one(top) * (one(1) / one(PEAK[store]))
                if store == "e4m3" and need > 0:
                    frac, expo = np.frexp(need)
                    need = np.ldexp(one(1), int(expo) - (1 if frac == 0.5 else 0))
                old = scale[page, h] if lo > b * block and scale[page, h] > 0 else one(0)
                now = max(old, one(need))
                held = slice(0, lo - b * block)
                if lo > b * block and now > old:
                    q = stored_values(cache[page, h, held], store).astype(one)
                    cache[page, h, held] = _quantise(q * (old / now), store)
                with np.errstate(invalid="ignore"):
                    q = x / now if now > 0 else x * one(0)
                cache[page, h, lo - b * block: hi - b * block] = _quantise(q, store)
                scale[page, h] = now
    return cache, scale


def kv_attention(values, scales, q, table, spans, share, softmax_scale, window):
    """(out, lse) in float64; `values` the pair (keys, values) [pages, heads, block, dim]
    as stored numbers, `scales` theirs.  Rows without a place: zeros and -inf."""
    (k, v), (ks, vs) = values, scales
    pages, heads, block, dim = k.shape
    out = np.zeros(q.shape)
    lse = np.full(q.shape[:2], -np.inf)
    for s, (row, first, count) in enumerate(spans):
        for i in range(count):
            pos = first + i
            seen = [j for j in range(max(0, pos - window + 1) if window else 0, pos + 1)
                    if 0 <= table[s][j // block] < pages]
            if not seen:
                continue
            page = np.array([table[s][j // block] for j in seen])
            at = np.array(seen) % block
            for h in range(q.shape[1]):
                kv = h // share
                keys = k[page, kv, at] * ks[page, kv, None]
                vals = v[page, kv, at] * vs[page, kv, None]
                x = keys @ q[row + i, h] * softmax_scale
                top = x.max()
                e = np.exp(x - top)
                out[row + i, h] = e @ vals / e.sum()
                lse[row + i, h] = top + np.log(e.sum())
    return out, lse
