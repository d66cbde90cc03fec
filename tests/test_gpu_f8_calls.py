"""E4M3 layers and their quantiser: calls whose memory overlaps, types and sizes at the edges of what they take."""
import numpy as np
import pytest

import f8 as F

pytestmark = pytest.mark.gpu


def cuda(a, bf=False):
    import torch
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t.to(torch.bfloat16) if bf else t


@pytest.mark.parametrize("bf", [False, True])
@pytest.mark.parametrize("M", [1, 4, 16, 17, 60, 300])
def test_a_result_in_its_inputs_place_is_refused(M, bf):
    """a square layer: in place, and with a row or an element in common on either side; neighbours are fine"""
    import helexa_amd as hx
    import torch
    n = 256
    layer = hx.F8Linear.load(*(cuda(a) for a in F.make_weights(M, n, n)))
    x = cuda(np.random.default_rng(M).standard_normal((M, n)).astype(np.float32), bf)
    want = layer(x)
    place = torch.zeros(3 * M * n + 16, dtype=x.dtype, device="cuda")
    mid = place[M * n:2 * M * n].view(M, n)
    mid.copy_(x)
    at = lambda i: place[i:i + M * n].view(M, n)
    for i in (M * n, M * n - 8, M * n + 8, 1, 2 * M * n - 1):
        with pytest.raises(hx.HxError, match="overlap"):
            layer(mid, out=at(i))
    assert torch.equal(mid, x)
    for i in (0, 2 * M * n):
        layer(mid, out=at(i))
        assert torch.equal(at(i), want) and torch.equal(mid, x)
    wide = torch.zeros(M * n + 2 * M * n, dtype=torch.float32, device="cuda")   # y's bytes are as many as its type says
    if not bf:
        wide[:M * n].view(M, n).copy_(x)
        y = wide.view(torch.bfloat16)
        with pytest.raises(hx.HxError, match="overlap"):
            layer(wide[:M * n].view(M, n), out=y[2 * M * n - 1:3 * M * n - 1].view(M, n))
        layer(wide[:M * n].view(M, n), out=y[2 * M * n:3 * M * n].view(M, n))
    layer.close()


@pytest.mark.parametrize("M", [1, 5, 17, 48, 100, 700])
def test_scales_whose_product_is_subnormal(M):
    """a product of scales keeps what float32 has there: a block is off by 2^-150 times its codes' products,
    128 of 448^2 at most, on top of what it is off elsewhere"""
    import helexa_amd as hx
    import torch
    N, K = 300, 520
    codes, scales = F.make_weights(M, N, K)
    x = np.random.default_rng(M).standard_normal((M, K)).astype(np.float32)
    rows = np.arange(M) % 3
    x *= np.exp2(np.choose(rows, [-100, -114, -125])).astype(np.float32)[:, None]
    small = (scales * np.float32(2.0 ** -12)).astype(np.float32)
    assert 0 < F.quantise(x, 1)[1].min() * float(small.max()) < 2.0 ** -126
    ref, mag, fixed = F.linear(x, codes, small)
    y = hx.F8Linear.load(cuda(codes), cuda(small))(cuda(x), out_dtype=torch.float32).cpu().numpy().astype(np.float64)
    off, bound = np.abs(y - ref), F.sum_steps(K) * F.U * mag + F.blocks(K) * 2.0 ** -125
    print(f"[err] worst {np.max(off / bound):.3f} of the bound", flush=True)
    assert (off <= bound).all() and np.abs(ref).max() > 2.0 ** -110


@pytest.mark.parametrize("key", ["router", "seg", "gate", "sdown"])
def test_weights_of_two_places_are_refused(key):
    """one tensor on the CPU among those on the GPU: a host address is none that a kernel may read"""
    import helexa_amd as hx
    import torch
    H, E, k, I, Is = 96, 4, 2, 64, 32
    cfg = hx.TextConfig(hidden_size=H, num_experts=E, num_experts_per_tok=k, moe_intermediate_size=I, shared_expert_intermediate_size=Is)
    w = {n: (hx.F8_E4M3, cuda(c), cuda(s)) for n, (c, s) in F.block(1, H, E, I, Is).items()}
    w["router"], w["seg"] = (hx.F32, torch.zeros((E, H), device="cuda")), (hx.F32, torch.zeros((1, H), device="cuda"))
    mixed = {**w, key: (w[key][0],) + tuple(t.cpu() for t in w[key][1:])}
    with pytest.raises(ValueError, match="all on"):
        hx.Qwen3_5MoeBlock.load(cfg, mixed, act_dtype=hx.F32)
    with pytest.raises(ValueError, match="all on"):
        hx.Qwen3_5MoeBlock.load(cfg, w, act_dtype=hx.F32, device=1)
    for good in (w, {n: (e[0],) + tuple(t.cpu() for t in e[1:]) for n, e in w.items()}):
        hx.Qwen3_5MoeBlock.load(cfg, good, act_dtype=hx.F32).close()


@pytest.mark.parametrize("M", [4, 16, 30, 400])
def test_two_calls_at_once(M):
    """a layer and a block from two streams, a workspace each; then the same as two graphs replayed together"""
    import helexa_amd as hx
    import torch
    n, E, k, I = 256, 8, 2, 128
    layer = hx.F8Linear.load(*(cuda(a) for a in F.make_weights(M, n, n)))
    blk = F.load(F.block(M, n, E, I, 0), n, E, k, I, 0, hx.BF16)
    idx, w, _ = F.routing(M, M, E, k)
    idx, w = cuda(idx), cuda(w)
    xs = [cuda(np.random.default_rng(i).standard_normal((M, n)).astype(np.float32), True) for i in range(2)]
    want = [(layer(x), blk.experts(x, idx, w)) for x in xs]
    ws = [[torch.empty(max(s, 16), dtype=torch.uint8, device="cuda") for s in (layer.workspace_size(M), blk.workspace_size(M))] for _ in xs]
    streams, graphs, outs = [torch.cuda.Stream() for _ in xs], [], []
    torch.cuda.synchronize()
    got = []
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append((i, layer(xs[i], workspace=ws[i][0]), blk.experts(xs[i], idx, w, workspace=ws[i][1])))
    torch.cuda.synchronize()
    assert all(torch.equal(a, want[i][0]) and torch.equal(b, want[i][1]) for i, a, b in got)
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append((layer(xs[i], workspace=ws[i][0]), blk.experts(xs[i], idx, w, workspace=ws[i][1])))
        graphs.append(g)
    for _ in range(5):
        for a, b in outs:
            a.zero_(), b.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) and torch.equal(b, d) for (a, b), (c, d) in zip(outs, want))
    blk.close(), layer.close()


def test_a_captured_call_without_the_memory_that_it_needs():
    """refused while it is captured, the graph's other work stays; few rows need none"""
    import helexa_amd as hx
    import torch
    layer = hx.F8Linear.load(*(cuda(a) for a in F.make_weights(1, 128, 256)))
    x = cuda(np.random.default_rng(1).standard_normal((40, 256)).astype(np.float32))
    want = layer(x[:16])
    assert layer.workspace_size(16) == 0 and layer.workspace_size(40) > 0
    out = torch.zeros((16, 128), device="cuda")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(hx.HxError, match="captured"):
            layer(x)
        layer(x[:16], out=out)
    for _ in range(3):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
