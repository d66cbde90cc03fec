"""MXFP4 in numpy: rows of 17-byte blocks (exponent byte, then 16 bytes of 4-bit
codes, value j low and j + 16 high in byte j), and the experts' products in 64
bits with a given routing."""
from __future__ import annotations

import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def quantise(x: np.ndarray) -> np.ndarray:
    """float32 [..., cols] -> uint8 [..., cols / 32 * 17]: nearest grid value, ties
    to the even code, by distances in float64"""
    v = np.ascontiguousarray(x, np.float32).astype(np.float64).reshape(-1, 32)
    out = np.zeros((len(v), 17), np.uint8)
    for b, row in enumerate(v):
        if not np.isfinite(row).all():
            out[b, 0] = 255
            continue
        amax = np.abs(row).max()
        e = int(np.floor(np.log2(amax))) - 2 if amax > 0 else -127
        e = max(e, -127)
        a = np.abs(row) / 2.0 ** e
        d = np.abs(np.minimum(a, 6.0)[:, None] - GRID)
        near = d == d.min(axis=1, keepdims=True)
        # among equals the even code
        code = np.where(near, np.arange(8) % 2 * 8 + np.arange(8), 99).argmin(axis=1).astype(np.uint8)
        code |= np.signbit(row).astype(np.uint8) << 3
        out[b, 0] = e + 127
        out[b, 1:] = code[:16] | (code[16:] << 4)
    return out.reshape(*x.shape[:-1], -1)


def values(q: np.ndarray) -> np.ndarray:
    """uint8 [..., row bytes] -> float64 [..., cols]"""
    b = q.reshape(*q.shape[:-1], -1, 17)
    codes = np.concatenate([b[..., 1:] & 15, b[..., 1:] >> 4], axis=-1)
    s = b[..., :1].astype(np.float64)
    scale = np.where(s == 255, np.nan, 2.0 ** (s - 127))
    v = GRID[codes & 7] * np.where(codes & 8, -1.0, 1.0) * scale
    return v.reshape(*q.shape[:-1], -1)


def swiglu(x, gate, up, down):
    g, u = x @ gate.T, x @ up.T
    return (g / (1.0 + np.exp(-g)) * u) @ down.T


def experts(x, idx, w, gate, up, down, shared=None, shared_w=None):
    """float64 y [T, H] of float64 weights [E, ...]; an idx outside 0 .. E - 1 is no expert"""
    x = x.astype(np.float64)
    y = np.zeros_like(x)
    for e in range(len(gate)):
        t, j = np.nonzero(idx == e)
        if len(t):
            np.add.at(y, t, w[t, j].astype(np.float64)[:, None] * swiglu(x[t], gate[e], up[e], down[e]))
    if shared is not None and shared_w is not None:
        y += shared_w.astype(np.float64)[:, None] * swiglu(x, *shared)
    return y
