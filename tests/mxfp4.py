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


def block(seed, H, E, I, Is, std=0.05, device="cuda"):
    """a seeded block: {name: uint8 rows} of the projections and their float64 values"""
    rng = np.random.default_rng(seed)
    shapes = dict(gate=(E, I, H), up=(E, I, H), down=(E, H, I))
    if Is:
        shapes.update(sgate=(Is, H), sup=(Is, H), sdown=(H, Is))
    rows, vals = {}, {}
    for n, s in shapes.items():
        # rows of several magnitudes, packed directly: scale bytes around 2^-5, random codes
        q = rng.integers(0, 256, s[:-1] + (s[-1] // 32, 17), dtype=np.uint8)
        q[..., 0] = 127 + np.round(np.log2(std)).astype(int) - rng.integers(1, 4, s[:-1] + (s[-1] // 32,))
        rows[n] = q.reshape(s[:-1] + (-1,))
        vals[n] = values(rows[n])
    return rows, vals


def load(rows, H, E, k, I, Is, act, router=None, seg=None):
    """the block on the GPU; router: float32 [E, H] (zeros if None)"""
    import torch
    from helexa_amd import moe as hx
    cfg = hx.TextConfig(hidden_size=H, num_experts=E, num_experts_per_tok=k, moe_intermediate_size=I,
                        shared_expert_intermediate_size=Is, norm_topk_prob=True)
    w = {n: (hx.MXFP4, torch.from_numpy(r)) for n, r in rows.items()}
    dt, tt = (hx.BF16, torch.bfloat16) if act == hx.BF16 else (hx.F32, torch.float32)
    w["router"] = (dt, torch.zeros((E, H), dtype=tt) if router is None else torch.from_numpy(router).to(tt))
    if Is:
        w["seg"] = (dt, torch.zeros((1, H), dtype=tt) if seg is None else torch.from_numpy(seg).to(tt))
    return hx.Qwen3_5MoeBlock.load(cfg, w, act_dtype=act)


def _blockmax(x):
    return np.repeat(np.abs(x).reshape(x.shape[0], -1, 32).max(axis=2), 32, axis=1)


def _swiglu_bound(x, gate, up, down, rec, planes):
    """(d, bound of the kernels' error in d) in float64. rec: what a record may leave
    of a value, relative to its block's largest magnitude. A product over K columns is
    K / 64 x planes MFMAs of 64 products each, every one taken to add at most 2^-23 of
    the sum of magnitudes, then at most 16 partial sums in f32; exp and the division
    to (|g| + 8) 2^-23."""
    def product(a, da, w):
        steps = a.shape[1] / 64 + 1
        return a @ w.T, da @ np.abs(w).T + (steps * planes + 16) * 2.0 ** -23 * ((np.abs(a) + da) @ np.abs(w).T)
    dx = rec * _blockmax(x)
    g, dg = product(x, dx, gate)
    u, du = product(x, dx, up)
    s = 1.0 / (1.0 + np.exp(-g))
    h = g * s * u
    # |silu'| <= 1.1
    dh = 1.1 * dg * (np.abs(u) + du) + np.abs(g * s) * du + np.abs(h) * (np.abs(g) + 8) * 2.0 ** -23
    dh = dh + rec * (_blockmax(h) + _blockmax(dh))
    return product(h, dh, down)


def experts_bound(x, idx, w, vals, shared_w, act_bf16, few):
    """(y, bound) float64 of the experts' outputs. Roundings to bf16 are off by at most
    2^-8 of the value: the result's, and above the few-token kernels each row's."""
    rec, planes = (2.0 ** -13, 3) if act_bf16 else (2.0 ** -23, 5)
    rnd = 2.0 ** -8 if act_bf16 else 2.0 ** -24
    x = x.astype(np.float64)
    y, b = np.zeros_like(x), np.zeros_like(x)
    mag = np.zeros_like(x)
    parts = [(e, *np.nonzero(idx == e)) for e in range(len(vals["gate"]))]
    jobs = [(t, w[t, j], vals["gate"][e], vals["up"][e], vals["down"][e]) for e, t, j in parts if len(t)]
    if shared_w is not None:
        jobs.append((np.arange(len(x)), shared_w, vals["sgate"], vals["sup"], vals["sdown"]))
    for t, wt, gate, up, down in jobs:
        d, dd = _swiglu_bound(x[t], gate, up, down, rec, planes)
        if not few:
            dd = dd + rnd * (np.abs(d) + dd)
        wt = wt.astype(np.float64)[:, None]
        np.add.at(y, t, wt * d)
        np.add.at(b, t, np.abs(wt) * dd)
        np.add.at(mag, t, np.abs(wt) * (np.abs(d) + dd))
    b += 80 * 2.0 ** -24 * mag                    # at most 65 + 16 additions and as many products in f32
    return y, b + rnd * (np.abs(y) + b) + 1e-37
