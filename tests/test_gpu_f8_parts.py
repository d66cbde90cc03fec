"""E4M3 experts: how many bits an expert's outputs keep until the weighted sum, in both forms of the sum."""
import numpy as np
import pytest

import f8 as F

pytestmark = pytest.mark.gpu
BF16, F32 = 30, 0


def cuda(a, bf=False):
    import torch
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t.to(torch.bfloat16) if bf else t


def thrice(seed, H, E, I):
    """experts in pairs: the second's down scales are three times the first's. A row of h is one block, so that
    an output is one product of an instruction's sum with the scales"""
    d = F.block(seed, H, E, I, 0)
    for n in ("gate", "up", "down"):
        c, s = d[n]
        c[1::2], s[1::2] = c[::2], s[::2]
    d["down"][1][1::2] *= 3
    return d


def parts(blk, x, first, k, act):
    """-> 3 p - 3 p of outputs p rounded apart, and p"""
    import torch
    T = x.shape[0]
    idx = torch.full((T, k), -1, dtype=torch.int32, device="cuda")
    idx[:, 0], idx[:, k - 1] = first, first + 1
    w = torch.zeros((T, k), device="cuda")
    w[:, 0], w[:, k - 1] = 3.0, -1.0
    left = blk.experts(x, idx, w)
    one = torch.zeros_like(w)
    one[:, 0] = 1.0
    return left, blk.experts(x, idx, one), idx, w


@pytest.mark.parametrize("act", [F32, BF16])
@pytest.mark.parametrize("T", [1, 2, 5, 16, 17, 60, 300, 2000])
def test_a_parts_bits(T, act):
    """what is left of 3 p - p3, p3 = 3 p but for roundings: with 24 bits two products' and the sums' half steps;
    with 11 (bf16 activations, above 16 tokens) 2^-11 of each part, or 2^-39 of the largest in its 32"""
    import torch
    H, E, k, I = 160, 6, 3, 96
    d = thrice(T, H, E, I)
    blk = F.load(d, H, E, k, I, 0, act)
    x = np.random.default_rng(T).standard_normal((T, H), dtype=np.float32)
    xt = cuda(F.bf16(x) if act == BF16 else x, act == BF16)
    first = cuda(np.random.default_rng(T + 1).integers(0, 3, T).astype(np.int32) * 2)
    left, p, _, _ = parts(blk, xt, first, k, act)
    left, p = left.double().abs(), p.double().abs()
    half = 2.0 ** -11 if act == BF16 and T > 16 else 0.0
    tol = 3 * (2 * half + 12 * F.U) * p * (1 + 2.0 ** -7) + (2.0 ** -37 if half else 2.0 ** -140) * p.max(dim=1, keepdim=True).values
    print(f"[err] worst {float((left / tol).max()):.3f} of the bound", flush=True)
    assert (left <= tol).all() and (p > 0).any()
    if half:   # and the test sees a rounding to 11 bits
        assert float((left / (3 * p + 1e-30)).max()) > 2.0 ** -13
    blk.close()


def test_many_rows_of_parts():
    """more than 256 MB of them, which the sum reads past the caches: bit by bit what two halves of the tokens
    give, which it reads through them; a sample against 64 bits"""
    import torch
    H, E, k, I, T = 2048, 4, 2, 128, 33000
    d = thrice(9, H, E, I)
    blk = F.load(d, H, E, k, I, 0, BF16)
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn((T, H), generator=g, device="cuda").to(torch.bfloat16)
    first = (torch.randint(0, 2, (T,), generator=g, device="cuda") * 2).int()
    left, p, idx, w = parts(blk, x, first, k, BF16)
    assert T * k * H * 2 > 256 << 20 and T // 2 * k * H * 2 < 256 << 20
    half = T // 2
    for a, b in ((0, half), (half, T)):
        assert torch.equal(blk.experts(x[a:b], idx[a:b].contiguous(), w[a:b].contiguous()), left[a:b])
    left, p = left.double().abs(), p.double().abs()
    tol = 3 * (2 * 2.0 ** -11 + 12 * F.U) * p * (1 + 2.0 ** -7) + 2.0 ** -37 * p.max(dim=1, keepdim=True).values
    assert (left <= tol).all()
    rows = torch.tensor([0, 1, half - 1, half, T - 2, T - 1] + list(range(1000, T, 3001)), device="cuda")
    one = torch.zeros_like(w)
    one[:, 0], one[:, 1] = 0.75, 0.25
    y = blk.experts(x, idx, one)[rows]
    ref, bound = F.experts(x[rows].float().cpu().numpy(), idx[rows].cpu().numpy(), one[rows].cpu().numpy(), d, None, True)
    assert (np.abs(y.double().cpu().numpy() - ref) <= bound).all()
    blk.close()
