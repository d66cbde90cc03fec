"""E4M3 layers of many rows: every size of tile, filled in part, with both ways that results leave; all elements
against 64 bits."""
import numpy as np
import pytest

import f8 as F

pytestmark = pytest.mark.gpu

# (tile, rows, features, columns): the last tiles with one row or one feature, features that are multiples of 8
# (whole rows leave) and not (element by element), one block of columns, an even and an odd number of them
CASES = [(256, 3841, 3848, 100), (256, 4000, 4008, 260), (256, 3850, 3841, 130), (256, 4096, 4090, 384), (256, 7900, 4000, 640),
         (128, 1100, 4104, 130), (128, 2049, 2049, 300), (128, 5000, 3304, 100),
         (64, 500, 4100, 260), (64, 577, 2056, 128), (0, 65, 1032, 520), (0, 300, 1001, 130), (0, 49, 8, 2048)]


def tile(M, N, exact):
    import ctypes as C
    import helexa_amd as hx
    f = hx.lib()._ZN2hx14f8_linear_tileEllb   # the library's own choice
    f.restype, f.argtypes = C.c_int, [C.c_int64, C.c_int64, C.c_bool]
    return f(M, N, exact)


@pytest.mark.parametrize("t,M,N,K", CASES)
def test_tiles(t, M, N, K):
    import helexa_amd as hx
    import torch
    assert tile(M, N, False) == t
    codes, scales = F.make_weights(M, N, K)
    layer = hx.F8Linear.load(torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda())
    x = F.bf16(np.random.default_rng(M).standard_normal((M, K)).astype(np.float32))
    ref, mag, fixed = F.linear(x, codes, scales)
    sums = F.sum_steps(K) * F.U * mag + 2.0 ** -140
    xt = torch.from_numpy(x).cuda().to(torch.bfloat16)

    def check(y, bound, tag):
        off = np.abs(y.float().cpu().numpy().astype(np.float64) - ref)
        print(f"[err] {tag} worst {np.max(off / bound):.3f} of the bound", flush=True)
        assert (off <= bound).all(), (tag, np.argwhere(off > bound)[:5])
    bf = (sums + fixed) * (1 + 2.0 ** -8) + 2.0 ** -8 * np.abs(ref)
    place = torch.full(((M + 2) * N + 16,), 5.0, dtype=torch.bfloat16, device="cuda")
    for at in (N + (-N) % 8, N + (-N) % 8 + 1):   # on 16 bytes, and an element behind
        place.fill_(5.0)
        out = place[at:at + M * N].view(M, N)
        layer(xt, out=out)
        check(out, bf, f"at {at}")
        assert (place[:at] == 5).all() and (place[at + M * N:] == 5).all()
        for _ in range(2):
            assert torch.equal(layer(xt), out)
    y = layer(xt, out_dtype=torch.float32)
    assert tile(M, N, True) in (128, 64)
    check(y, sums + F.U * np.abs(ref), "f32")
    bad = xt.clone()
    bad[M - 1, K - 1] = np.nan
    z = layer(bad)
    assert torch.isnan(z[M - 1]).all() and torch.equal(z[:M - 1], out[:M - 1])
    layer.close()


def test_the_rule_reaches_every_tile():
    assert {tile(M, N, False) for _, M, N, _ in CASES} == {256, 128, 64, 0}
    assert {tile(M, N, True) for _, M, N, _ in CASES} == {128, 64}
