"""E4M3: errors against 64 bits relative to the results' norm, as the header states them.

A result's rounding to bf16 is at most half a step, 2^-8 of the power of two below it, evenly spread: 2^-8 / sqrt(3) of
the norm if all results were powers of two, less for others. What comes before it adds by squares:
 - the 8-bit instruction's fixed point, at most 5.5e-5 of a sum's norm;
 - codes of h that become a neighbour, a step of at most 2^-3 of the value: where gate's and up's sums are float32's they
   are off by some 20 half steps, about 2^-20, of the codes' distance of 2^-4, so that one in 2^14 does: 2^-3 2^-7;
 - in calls of more than 16 tokens and 18 entries an expert 1.3e-3 instead, taken as 1.5e-3;
 - above 16 tokens a part's 11 bits, 2^-11 / sqrt(3) at most."""
import numpy as np
import pytest

import f8 as F

pytestmark = pytest.mark.gpu
BF16, F32 = 30, 0
ROUND = 2.0 ** -8 / 3 ** 0.5


def cuda(a, bf=False):
    import torch
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t.to(torch.bfloat16) if bf else t


def rows_of(seed, M, K, act):
    """normal values, a few columns much larger"""
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((M, K), dtype=np.float32)
    x[:, rng.random(K) < 0.01] *= 16
    return F.bf16(x) if act == BF16 else x


def norm_of(y, ref):
    n = np.linalg.norm(y.double().cpu().numpy() - ref) / np.linalg.norm(ref)
    print(f"[err] norm {n:.2e}", flush=True)
    return n


@pytest.mark.parametrize("act", [F32, BF16])
def test_experts(act):
    H, E, k, I, Is = 1024, 24, 10, 512, 512
    d = F.block(1, H, E, I, Is)
    blk = F.load(d, H, E, k, I, Is, act)
    for T in (1, 4, 16, 17, 43, 44, 120, 300):
        print("case", act, T, flush=True)
        x = rows_of(T, T, H, act)
        idx, w, sw = F.routing(T, T, E, k)
        n = norm_of(blk.experts(cuda(x, act == BF16), cuda(idx), cuda(w), shared_w=cuda(sw)), F.experts(x, idx, w, d, sw, act == BF16)[0])
        codes = 1.5e-3 if act == BF16 and T > 16 and T * k > 18 * E else 2.0 ** -10
        if act == F32:
            assert n <= codes
        else:
            assert n <= (ROUND ** 2 + codes ** 2 + (2.0 ** -11 / 3 ** 0.5 if T > 16 else 0.0) ** 2 + 5.5e-5 ** 2) ** 0.5
    blk.close()


@pytest.mark.parametrize("N,K", [(1031, 2080), (4104, 384), (512, 4096)])
def test_layers(N, K):
    import helexa_amd as hx
    import torch
    codes, scales = F.make_weights(N, N, K)
    layer = hx.F8Linear.load(cuda(codes), cuda(scales))
    for M in (1, 5, 16, 48, 64, 300, 1500):
        for act in (F32, BF16):
            print("case", N, K, M, act, flush=True)
            x = rows_of(M, M, K, act)
            ref = F.linear(x, codes, scales)[0]
            t = cuda(x, act == BF16)
            # float32: a multiply-add a block and the sums of 16 waves, half a step of what there is so far each
            assert norm_of(layer(t, out_dtype=torch.float32), ref) <= (F.blocks(K) + 16) * F.U
            assert norm_of(layer(t, out_dtype=torch.bfloat16), ref) <= (ROUND ** 2 + 5.5e-5 ** 2) ** 0.5
    layer.close()
