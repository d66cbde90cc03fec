"""E4M3 experts: gate/up's small products beside large ones that cancel. An instruction on 8-bit codes drops what lies
13 bits below the largest of a lane's products; where the sums are documented as float32's, that product is the result."""
import numpy as np
import pytest

import f8 as F

pytestmark = pytest.mark.gpu
BF16, F32 = 30, 0
CODE = {0.25: 0x28, 0.5: 0x30, 1.0: 0x38, 2.0: 0x40, 64.0: 0x68, -64.0: 0xe8}


def cuda(a, bf=False):
    import torch
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t.to(torch.bfloat16) if bf else t


def block(H, E, I, Is, at):
    """Columns at .. at + 2 of gate and up hold 64, -64 and the value that counts: 1 in gate, v in up; row n
    of down is column n % I of h. -> the block, v [E, I], v of the shared expert"""
    rng = np.random.default_rng(H + I)
    v = rng.choice([0.25, 0.5, 1.0, 2.0], (E, I))
    vs = rng.choice([0.25, 0.5, 1.0, 2.0], (Is,))
    one = lambda *s: np.ones(s[:-2] + (F.blocks(s[-2]), F.blocks(s[-1])), np.float32)

    def up(values):
        c = np.zeros(values.shape + (H,), np.uint8)
        c[..., at], c[..., at + 1] = CODE[64.0], CODE[-64.0]
        c[..., at + 2] = np.vectorize(CODE.get)(values)
        return c, one(*c.shape)

    def down(*s):
        c = np.zeros(s, np.uint8)
        c[..., np.arange(H), np.arange(H) % s[-1]] = CODE[1.0]
        return c, one(*s)
    d = dict(gate=up(np.ones((E, I))), up=up(v), down=down(E, H, I))
    if Is:
        d.update(sgate=up(np.ones(Is)), sup=up(vs), sdown=down(H, Is))
    return d, v, vs


@pytest.mark.parametrize("act", [F32, BF16])
@pytest.mark.parametrize("H,E,k,I,Is,at", [(256, 16, 2, 128, 128, 3), (384, 16, 3, 512, 0, 301), (160, 40, 2, 96, 64, 144)])
def test_gate_and_up_keep_them(H, E, k, I, Is, at, act):
    """up to 16 tokens, and above while an expert has 18 entries at most"""
    d, v, vs = block(H, E, I, Is, at)
    blk = F.load(d, H, E, k, I, Is, act)
    silu = 1 / (1 + np.exp(-1.0))
    h, hs = F.quantised(silu * v), F.quantised(silu * vs[None])[0] if Is else None
    n = np.arange(H)
    for T in (1, 2, 3, 4, 5, 8, 16, 17, 33, 18 * E // k):
        print("case", H, E, k, I, Is, act, T, flush=True)
        x = np.zeros((T, H), np.float32)
        x[:, at:at + 2], x[:, at + 2] = 448.0, 1.0   # a scale of 1: the products are 28672, -28672 and v
        idx, w, sw = F.routing(T, T, E, k)
        w = w + 0.5
        y = blk.experts(cuda(x, act == BF16), cuda(idx), cuda(w), shared_w=cuda(sw) if Is else None).float().cpu().numpy()
        ref = (w.astype(np.float64)[:, :, None] * h[idx][:, :, n % I]).sum(axis=1)
        if Is:
            ref += sw.astype(np.float64)[:, None] * hs[n % Is]
        # silu's exponential and reciprocal 20 half steps of float32, the scale 3, the weighted sum 2 (k + 2);
        # the codes are powers of two of the block's largest, in the middle of their range; bf16: above 16 tokens a part's
        # 11 bits, and the result's rounding
        tol = 64 * F.U if act == F32 else 2.0 ** -8 + 2.0 ** -11 + 2.0 ** -16
        off = np.abs(y - ref) / ref
        print(f"[err] worst {off.max():.2e}", flush=True)
        assert (off <= tol).all(), np.argwhere(~(off <= tol))[:5]
    blk.close()
