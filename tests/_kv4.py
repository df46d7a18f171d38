"""Plain numpy form of the 4-bit KV cache: quantisation in f32, decoding and attention in f64."""
from __future__ import annotations

import numpy as np


def quantise(x):
    """f32 [..., d] -> (codes uint8 [..., d / 2], scales int16 [..., d / 32]) by the format's definition."""
    x = np.asarray(x, np.float32)
    nb = x.shape[-1] // 32
    y = x.reshape(*x.shape[:-1], nb, 32)
    bad = ~np.isfinite(y).all(-1)
    y = np.where(bad[..., None], np.float32(0), y)
    lo, hi = np.minimum(y.min(-1), np.float32(0)), np.maximum(y.max(-1), np.float32(0))
    with np.errstate(over="ignore"):
        s = np.minimum((hi - lo) / np.float32(15), np.float32(4352)).astype(np.float32)
    h = s.astype(np.float16)
    bits = h.view(np.uint16).astype(np.uint32) + (h.astype(np.float32) < s)
    bits = (bits + 15) // 16 * 16
    step = bits.astype(np.uint16).view(np.float16).astype(np.float32)
    div = np.where(step > 0, step, np.float32(1))
    with np.errstate(over="ignore"):
        z = np.clip(np.rint(-lo / div), 0, 15)
        c = np.clip(np.rint(y / div[..., None]) + z[..., None], 0, 15).astype(np.uint32)
    c = np.where((bad | (step == 0))[..., None], 0, c)
    scales = np.where(bad, 0x7E00, bits + z.astype(np.uint32)).astype(np.uint16).view(np.int16)
    words = np.zeros((*x.shape[:-1], 4 * nb), np.uint32)
    for b in range(nb):
        for t in range(4):
            for n in range(8):
                words[..., t * nb + b] |= c[..., b, 8 * t + n].astype(np.uint32) << np.uint32(4 * n)
    return words.astype("<u4").view(np.uint8), scales


def values(codes, scales):
    """f64 values of 4-bit rows."""
    nb = scales.shape[-1]
    words = np.ascontiguousarray(codes).view("<u4")
    h = np.asarray(scales).view(np.uint16)
    step = (h & 0xFFF0).astype(np.uint16).view(np.float16).astype(np.float64)
    z = (h & 15).astype(np.float64)
    out = np.empty((*codes.shape[:-1], 32 * nb))
    for b in range(nb):
        for t in range(4):
            for n in range(8):
                c = (words[..., t * nb + b] >> np.uint32(4 * n)) & 15
                out[..., 32 * b + 8 * t + n] = (c - z[..., b]) * step[..., b]
    return out


def attention(q, k, v, ctx, scale=None):
    """q [T, H, d], k / v [Hkv, rows, d] (rows past ctx ignored) -> f64 [T, H, d]; a token that sees no row gives zeros."""
    T, H, d = q.shape
    G = H // k.shape[0]
    scale = 1 / np.sqrt(d) if scale is None else scale
    out = np.zeros((T, H, d))
    for t in range(T):
        n = ctx - T + 1 + t
        if n <= 0:
            continue
        for h in range(H):
            s = k[h // G, :n] @ q[t, h].astype(np.float64) * scale
            p = np.exp(s - s.max())
            out[t, h] = (p / p.sum()) @ v[h // G, :n]
    return out


def random_cache(rng, units, heads, rows, d, scale=1.0):
    """Random N(0, scale) rows as 4-bit codes and scales [units, heads, rows, ..] for K and V."""
    parts = []
    for _ in range(2):
        parts += quantise(rng.standard_normal((units, heads, rows, d)).astype(np.float32) * np.float32(scale))
    return parts  # k_codes, k_scales, v_codes, v_scales
