"""E4M3: rows whose places pass 32 bits: codes, activations, results."""
import numpy as np
import pytest

import f8 as F

pytestmark = pytest.mark.gpu


def cuda(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def some(T, seed=1):
    """the first, the last, those around 2^31 and 2^32 elements of 4096, others"""
    at = [0, 1, T - 2, T - 1] + [b + d for b in (1 << 19, 1 << 20) for d in (-1, 0, 1)]
    return np.unique(np.concatenate([np.array([a for a in at if a < T]), np.random.default_rng(seed).integers(0, T, 30)]))


def made(T, H, seed):
    """bf16 rows [T, H], a different one each: a base of 1000 rows, a column that grows with the row"""
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    base = torch.randn((1000, H), generator=g, device="cuda").to(torch.bfloat16)
    x = base.repeat(T // 1000 + 1, 1)[:T]
    x[:, 7] = (torch.arange(T, device="cuda") % 251).to(torch.bfloat16) / 64
    return x


def test_quantise():
    """more than 2^32 elements, by rows and by blocks"""
    import helexa_amd as hx
    import torch
    T, H = (1 << 20) + 70, 4100
    x = made(T, H, 1)
    for block_rows in (1, 128):
        codes, scales = hx.quantize_f8(x, block_rows)
        for r in some(T // block_rows):
            a, n = r * block_rows, min(block_rows, T - r * block_rows)
            c, s = F.quantise(x[a:a + n].float().cpu().numpy(), block_rows)
            assert np.array_equal(codes[a:a + n].view(torch.uint8).cpu().numpy(), c), r
            assert np.array_equal(scales[r:r + 1].cpu().numpy(), s), r
        del codes, scales


def test_layer():
    """more than 2^32 codes of rows, and more than 2^32 results"""
    import helexa_amd as hx
    import torch
    for T, N, K in (((1 << 20) + 70, 24, 4096), ((1 << 20) + 70, 4104, 130)):
        codes, scales = F.make_weights(N, N, K)
        x = made(T, K, 2)
        y = hx.F8Linear.load(cuda(codes), cuda(scales))(x)
        rows = some(T)
        at = torch.from_numpy(rows).cuda()
        ref, mag, fixed = F.linear(x[at].float().cpu().numpy(), codes, scales)
        bound = (F.sum_steps(K) * F.U * mag + fixed) * (1 + 2.0 ** -8) + 2.0 ** -8 * np.abs(ref) + 2.0 ** -140
        assert (np.abs(y[at].double().cpu().numpy() - ref) <= bound).all()
        del x, y


@pytest.mark.parametrize("act", [30, 0])
def test_experts(act):
    """more than 2^32 codes of tokens (tiles of 64 in bf16, whatever the experts' rows) and as many results"""
    import helexa_amd as hx
    import torch
    T, H, E, k, I = (1 << 20) + 70, 4096, 3, 2, 32
    d = F.block(3, H, E, I, 0)
    blk = F.load(d, H, E, k, I, 0, act)
    x = made(T, H, 3)
    if act == 0:
        x = x.float()
    g = torch.Generator(device="cuda").manual_seed(4)
    idx = torch.randint(-1, E, (T, k), generator=g, device="cuda", dtype=torch.int32)
    w = torch.rand((T, k), generator=g, device="cuda")
    y = blk.experts(x, idx, w)
    rows = some(T)
    at = torch.from_numpy(rows).cuda()
    ref, bound = F.experts(x[at].float().cpu().numpy(), idx[at].cpu().numpy(), w[at].cpu().numpy(), d, None, act == 30)
    assert (np.abs(y[at].double().cpu().numpy() - ref) <= bound).all()
    blk.close()
