"""Microscaled (MX) formats and the expert path over them, in numpy and 64
bits: the plain statement the GPU tests compare with."""

from __future__ import annotations

import numpy as np

FP8, FP4 = 0, 1
EMAX = {FP8: 8, FP4: 2}


def table(fmt) -> np.ndarray:
    """The value of every element code (e4m3 / e2m1), from the definition."""
    if fmt == FP4:
        mag = [(1 + (c & 1) / 2) * 2.0 ** ((c >> 1) - 1) if c >> 1 else (c & 1) / 2 for c in range(8)]
    else:
        mag = [(1 + (c & 7) / 8) * 2.0 ** ((c >> 3) - 7) if c >> 3 else (c & 7) / 8 * 2.0**-6 for c in range(127)]
        mag.append(np.nan)
    return np.array(mag + [-m for m in mag])


def pack4(codes) -> np.ndarray:
    return (codes[..., 0::2] | (codes[..., 1::2] << 4)).astype(np.uint8)


def unpack4(q) -> np.ndarray:
    return np.stack([q & 15, q >> 4], -1).reshape(*q.shape[:-1], -1)


def scale_values(scales) -> np.ndarray:
    v = np.ldexp(1.0, scales.astype(np.int64) - 127)
    return np.where(scales == 255, np.nan, v)


def decode(q, scales, fmt) -> np.ndarray:
    """float64 values of MX rows."""
    codes = unpack4(q) if fmt == FP4 else q
    v = table(fmt)[codes].reshape(*scales.shape, 32)
    return (v * scale_values(scales)[..., None]).reshape(codes.shape)


def block_scales(amax, fmt) -> np.ndarray:
    """Scale bytes of blocks with largest magnitudes `amax` (float64)."""
    with np.errstate(invalid="ignore", divide="ignore"):
        e = np.frexp(np.where(np.isfinite(amax), amax, 1.0))[1] - 1
    s = np.maximum(0, e + 127 - EMAX[fmt])
    s = np.where(amax == 0, 0, s)
    return np.where(np.isfinite(amax), s, 255).astype(np.uint8)


def encode(x, fmt):
    """Values (fp32-representable) -> (q bytes, scale bytes); ties to the even code."""
    x = np.asarray(x, np.float64)
    b = x.reshape(*x.shape[:-1], -1, 32)
    with np.errstate(invalid="ignore"):
        amax = np.abs(b).max(-1)
    scales = block_scales(amax, fmt)
    bad = scales == 255
    with np.errstate(invalid="ignore"):
        v = np.where(bad[..., None], 0.0, b) * np.ldexp(1.0, 127 - scales.astype(np.int64))[..., None]
    mags = table(fmt)[: 8 if fmt == FP4 else 127]
    a = np.minimum(np.abs(v), mags[-1])
    hi = np.minimum(np.searchsorted(mags, a), len(mags) - 1)
    lo = np.maximum(hi - 1, 0)
    down, up = a - mags[lo], mags[hi] - a
    code = np.where((down < up) | ((down == up) & (lo % 2 == 0)), lo, hi)
    code = (code | np.where(np.signbit(v), 8 if fmt == FP4 else 128, 0)).astype(np.uint8).reshape(x.shape)
    return (pack4(code) if fmt == FP4 else code), scales


def add_norm(x, r, w, eps):
    """(fp32 sum, float64 norm of it)."""
    s = x if r is None else (x + r).astype(np.float32)
    d = s.astype(np.float64)
    with np.errstate(all="ignore"):
        inv = 1.0 / np.sqrt((d * d).mean(-1, keepdims=True) + float(np.float32(eps)))
        return s, d * inv * w.astype(np.float64)


def expert_rows(idx, n_expert):
    """(offsets, entries, row_of), ids out of range left out with row_of -1."""
    flat = idx.reshape(-1)
    ok = (flat >= 0) & (flat < n_expert)
    order = np.argsort(np.where(ok, flat, n_expert), kind="stable")[: ok.sum()].astype(np.int32)
    offsets = np.concatenate([[0], np.cumsum(np.bincount(flat[ok], minlength=n_expert))]).astype(np.int32)
    row_of = np.full(flat.size, -1, np.int32)
    row_of[order] = np.arange(order.size)
    return offsets, order, row_of


def grouped(x, w, offsets, rows):
    """float64 [n_sorted, n_out]: row r of group e times w[e]^T; x row rows[r]."""
    out = np.zeros((len(rows), w.shape[1]))
    for e in range(len(offsets) - 1):
        lo, hi = offsets[e], offsets[e + 1]
        if lo < hi:
            out[lo:hi] = x[rows[lo:hi]] @ w[e].T
    return out


def silu(g):
    with np.errstate(over="ignore"):
        return g / (1.0 + np.exp(-g))
