"""hx_moe_experts on MXFP4 blocks over the range of its types: activations and h whose
blocks lie near the smallest normal float, weights at both ends of the scale byte,
against 64-bit products of the stored weights within the bound that the formats and the
sums allow."""
import numpy as np
import pytest

import mxfp4 as M

pytestmark = pytest.mark.gpu

BF16, F32 = 30, 0
H, E, K, I = 256, 3, 2, 128
LEAST = 2.0 ** -130   # what a record may leave of a value, however small its block


def cuda(a, act=None):
    import torch
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t.to(torch.bfloat16) if act == BF16 else t


def to_act(x, act):
    import torch
    x = np.ascontiguousarray(x, np.float32)
    return torch.from_numpy(x).to(torch.bfloat16).float().numpy() if act == BF16 else x


def weights(seed, gate, up, down):
    """random codes; a projection's scale bytes drawn from the ones given"""
    rng = np.random.default_rng(seed)
    rows = {}
    for n, (r, c), scales in (("gate", (I, H), gate), ("up", (I, H), up), ("down", (H, I), down)):
        q = rng.integers(0, 256, (E, r, c // 32, 17), dtype=np.uint8)
        q[..., 0] = rng.choice(np.asarray(scales), (E, r, c // 32))
        rows[n] = q.reshape(E, r, -1)
    return rows, {n: M.values(q) for n, q in rows.items()}


def routing(seed, T):
    rng = np.random.default_rng(seed)
    idx = np.stack([rng.permutation(E)[:K] for _ in range(T)]).astype(np.int32)
    return idx, rng.random((T, K)).astype(np.float32)


def reference(x, idx, w, vals, act):
    """(y, bound): as mxfp4.experts_bound, a record leaving at most 2^-13 (f32: 2^-23) of
    its block's largest or LEAST; rows rounded to bf16 as above the few tokens"""
    rec, planes, rnd = (2.0 ** -13, 3, 2.0 ** -8) if act == BF16 else (2.0 ** -23, 5, 2.0 ** -24)
    x = x.astype(np.float64)

    def product(a, da, m):
        return a @ m.T, da @ np.abs(m).T + ((a.shape[1] / 64 + 1) * planes + 16) * 2.0 ** -23 * ((np.abs(a) + da) @ np.abs(m).T)
    y, b, mag = np.zeros_like(x), np.zeros_like(x), np.zeros_like(x)
    for e in range(E):
        t, j = np.nonzero(idx == e)
        if not len(t):
            continue
        xs = x[t]
        g, dg = product(xs, np.maximum(rec * M._blockmax(xs), LEAST), vals["gate"][e])
        u, du = product(xs, np.maximum(rec * M._blockmax(xs), LEAST), vals["up"][e])
        with np.errstate(over="ignore"):
            s = 1.0 / (1.0 + np.exp(-g))
        h = g * s * u
        # |silu'| <= 1.1; exp and the division to (|g| + 8) 2^-23; a quotient below 2^-126 may be 0
        dh = (1.1 * dg * (np.abs(u) + du) + np.abs(g * s) * du + np.abs(h) * (np.abs(g) + 8) * 2.0 ** -23
              + np.abs(g) * 2.0 ** -126 * np.abs(u))
        dh = dh + np.maximum(rec * (M._blockmax(h) + M._blockmax(dh)), LEAST)
        d, dd = product(h, dh, vals["down"][e])
        dd = dd + rnd * (np.abs(d) + dd)
        wt = w[t, j].astype(np.float64)[:, None]
        np.add.at(y, t, wt * d)
        np.add.at(b, t, np.abs(wt) * dd)
        np.add.at(mag, t, np.abs(wt) * (np.abs(d) + dd))
    b += 80 * 2.0 ** -24 * mag
    return y, b + rnd * (np.abs(y) + b) + 2.0 ** -126


def check(blk, x, idx, w, vals, act, what):
    y = blk.experts(cuda(x, act), cuda(idx), cuda(w)).float().cpu().numpy().astype(np.float64)
    ref, bound = reference(x, idx, w, vals, act)
    off = np.abs(y - ref) / bound
    print(f"[err] {what}: worst {off.max():.3f} of the bound, bound {np.median(bound / np.maximum(np.abs(ref), 1e-300)):.1e} "
          f"of the value", flush=True)
    assert np.isfinite(ref).all() and np.abs(ref).max() < 3e38
    assert off.max() <= 1.0, (what, np.unravel_index(off.argmax(), off.shape))


@pytest.mark.parametrize("act", [BF16, F32])
@pytest.mark.parametrize("T", [1, 4, 24, 300])
def test_blocks_of_small_activations(T, act):
    """blocks whose largest value is 2^-100 .. 2^-124, each of values over 10 binades, met by weights that
    bring the sums to ordinary size"""
    for top in (-100, -108, -112, -115, -118, -121, -124):
        rows, vals = weights(-top, [127 - top - 4, 127 - top - 3], [127 - top - 3], [122, 123])
        blk = M.load(rows, H, E, K, I, 0, act)
        rng = np.random.default_rng(T)
        x = rng.standard_normal((T, H)) * np.exp2(top - rng.integers(0, 10, (T, H)))
        x[:, ::32] = np.exp2(top)
        idx, w = routing(T - top, T)
        check(blk, to_act(x, act), idx, w, vals, act, f"largest 2^{top}, {T} tokens")
        blk.close()


@pytest.mark.parametrize("act", [BF16, F32])
@pytest.mark.parametrize("T", [1, 4, 24, 300])
def test_blocks_of_small_h(T, act):
    """ordinary tokens, h about 2^-100 .. 2^-120 by its factor u, down weights that bring it back"""
    for top in (-100, -108, -114, -120):
        rows, vals = weights(-top, [122], [127 + top - 6, 127 + top - 3], [127 - top - 6])
        blk = M.load(rows, H, E, K, I, 0, act)
        x = np.random.default_rng(T).standard_normal((T, H))
        idx, w = routing(T - top, T)
        check(blk, to_act(x, act), idx, w, vals, act, f"h about 2^{top}, {T} tokens")
        blk.close()


@pytest.mark.parametrize("act", [BF16, F32])
@pytest.mark.parametrize("T", [1, 4, 24, 300])
@pytest.mark.parametrize("size,gate,up,down", [
    (60, [62, 64], [0, 1, 2, 40], [252, 253, 254]),        # up at the lower end, down at the upper
    (-60, [182, 184], [253, 254, 200], [0, 1, 2, 60]),     # up at the upper end, down at the lower
    (117, [0, 1, 2], [5, 10], [122, 127]),                 # gate at the lower end
    (-121, [253, 254, 240], [243, 244], [120])])           # gate at the upper end
def test_weights_at_both_ends_of_the_scale(size, gate, up, down, T, act):
    rows, vals = weights(abs(size), gate, up, down)
    blk = M.load(rows, H, E, K, I, 0, act)
    x = np.random.default_rng(T).standard_normal((T, H)) * 2.0 ** size
    idx, w = routing(T, T)
    check(blk, to_act(x, act), idx, w, vals, act, f"scales {gate} {up} {down}, {T} tokens")
    blk.close()


@pytest.mark.parametrize("act", [BF16, F32])
@pytest.mark.parametrize("T", [1, 4, 12, 300])
def test_blocks_of_zeros_tiny_and_large_values(T, act):
    """each element of tokens of zeros, of about 1e-30, and with one block a million times
    the others"""
    rows, vals = M.block(4, H, E, I, 0)
    blk = M.load(rows, H, E, K, I, 0, act)
    x = np.random.default_rng(T).standard_normal((T, H))
    idx, w = routing(T, T)
    for first in range(3):   # one token: each of the three in turn
        z = x.copy()
        kind = (np.arange(T) + first) % 3
        z[kind == 0] = 0.0
        z[kind == 1] *= 1e-30
        z[kind == 2, 32:64] *= 1e6
        check(blk, to_act(z, act), idx, w, vals, act, f"kind {first}, {T} tokens")


@pytest.mark.parametrize("act", [BF16, F32])
@pytest.mark.parametrize("T", [1, 4, 12, 300])
def test_a_token_whose_h_overflows(T, act):
    """a token of 2^100 has an h past the largest float with every expert: NaN for that token,
    the others' bits as they were"""
    import torch
    rows, vals = M.block(4, H, E, I, 0)
    blk = M.load(rows, H, E, K, I, 0, act)
    x = to_act(np.random.default_rng(T).standard_normal((T, H)), act)
    idx, w = routing(T, T)
    y = blk.experts(cuda(x, act), cuda(idx), cuda(w))
    big = x.copy()
    big[T // 2] = 2.0 ** 100
    for e in idx[T // 2]:
        g, u = vals["gate"][e] @ big[T // 2].astype(np.float64), vals["up"][e] @ big[T // 2].astype(np.float64)
        assert (np.maximum(g, 0) * np.abs(u)).max() > 1e39 and np.abs(g).max() < 3e38 and np.abs(u).max() < 3e38
    yb = blk.experts(cuda(big, act), cuda(idx), cuda(w))
    others = [t for t in range(T) if t != T // 2]
    assert yb[T // 2].isnan().all()
    assert torch.equal(yb[others], y[others])
