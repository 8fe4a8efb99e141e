"""64-bit restatements of the operators around the quantized cache, apart from the kernels' code."""
from __future__ import annotations

import numpy as np

GROUP = 64


def bf16(x: np.ndarray) -> np.ndarray:
    """Rounded to bf16 (nearest even), as float64.  Finite inputs that are binary32 values."""
    u = np.ascontiguousarray(x, dtype=np.float32).view(np.uint32).astype(np.uint64)
    u = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16) << 16
    return u.astype(np.uint32).view(np.float32).astype(np.float64)


def quantize(x: np.ndarray, bits: int):
    """(codes, scale, bias) of the rows x [..., dim], the weights' rule with 2^bits - 1 steps; its quotients
    are binary32 by definition (double quotients rounded once to binary32 are the correctly rounded ones)."""
    w = bf16(x).reshape(*x.shape[:-1], -1, GROUP)
    top = 2**bits - 1

    def f32(v):
        return v.astype(np.float32).astype(np.float64)

    def away(v):
        return np.trunc(v + 0.5 * np.sign(v))

    hi, lo = np.maximum(w.max(-1), 0.0), w.min(-1)
    s = np.maximum(f32(f32(hi - lo) / top), float(np.float32(1e-7)))
    side = np.abs(lo) > np.abs(hi)
    s, edge = np.where(side, s, -s), np.where(side, lo, hi)
    n = away(f32(edge / s))
    s = np.where(n != 0, f32(edge / np.where(n != 0, n, 1)), s)
    b = np.where(n != 0, edge, 0.0)
    c = np.clip(away(f32(f32(w - b[..., None]) / s[..., None])), 0, top)
    return c.astype(np.int64).reshape(x.shape), bf16(s), bf16(b)


def dequantize(codes: np.ndarray, s: np.ndarray, b: np.ndarray) -> np.ndarray:
    c = codes.reshape(*codes.shape[:-1], codes.shape[-1] // GROUP, GROUP)
    return (c * s[..., None] + b[..., None]).reshape(codes.shape)


def norm_rope(x, w, positions, freqs, eps, interleaved, axes=None):
    """x [tokens, heads, dim] -> normalised and turned, all float64.  positions [axes, tokens]."""
    x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * (1.0 + w)
    n = len(freqs)
    ax = np.zeros(n, int) if axes is None else np.asarray(axes)
    ang = positions[ax].T.astype(np.float64) * freqs.astype(np.float64)
    c, s = np.cos(ang)[:, None], np.sin(ang)[:, None]
    y = x.copy()
    i, j = (2 * np.arange(n), 2 * np.arange(n) + 1) if interleaved else (np.arange(n), np.arange(n) + n)
    y[..., i] = x[..., i] * c - x[..., j] * s
    y[..., j] = x[..., j] * c + x[..., i] * s
    return y


def attention(q, ks, vs, lens, starts, scale):
    """q [tokens, heads, dim]; ks, vs: per sequence [len, kv_heads, dim].  Returns (out, mix, top, spread): the
    attention; sum p |v|; the same with each |v| raised to the largest of its 64-feature group; and the
    largest scale * sum |q| |k| over the row's positions (what errors scale with)."""
    out, mix, top = np.zeros_like(q), np.zeros_like(q), np.zeros_like(q)
    spread = np.zeros(q.shape[:2])
    for b, n_pos in enumerate(lens):
        n = starts[b + 1] - starts[b]
        group = q.shape[1] // ks[b].shape[1]
        raised = np.abs(vs[b]).reshape(n_pos, ks[b].shape[1], q.shape[2] // GROUP, GROUP).max(-1).repeat(GROUP, -1)
        for i in range(n):
            seen = n_pos - n + i + 1
            if seen <= 0:
                continue
            t = starts[b] + i
            for h in range(q.shape[1]):
                k, v = ks[b][:seen, h // group], vs[b][:seen, h // group]
                x = scale * (k @ q[t, h])
                p = np.exp(x - x.max())
                p /= p.sum()
                out[t, h], mix[t, h], top[t, h] = p @ v, p @ np.abs(v), p @ raised[:seen, h // group]
                spread[t, h] = scale * (np.abs(k) @ np.abs(q[t, h])).max()
    return out, mix, top, spread
