"""The MXFP4 operators together, as a program uses them: float weights quantised on
the device, a block loaded from them, its router and its experts called apart and as
one forward, the decoder half around it, the entries without an allocation and for
host buffers, graphs of a layer stack."""
import ctypes as C

import numpy as np
import pytest

import mxfp4 as M

pytestmark = pytest.mark.gpu

BF16, F32 = 30, 0


def make(seed, H, E, k, I, Is, act, seg_zero=True):
    """(block, float32 weights on the device, quantised rows): a float checkpoint through hx_quantize"""
    import torch
    from helexa_amd import moe as hx
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(s, generator=g, device="cuda") * 0.05
    w = dict(gate=rnd(E, I, H), up=rnd(E, I, H), down=rnd(E, H, I))
    if Is:
        w.update(sgate=rnd(Is, H), sup=rnd(Is, H), sdown=rnd(H, Is))
    q = {n: hx.quantize(hx.MXFP4, v) for n, v in w.items()}
    tt = torch.bfloat16 if act == BF16 else torch.float32
    weights = {n: (hx.MXFP4, v) for n, v in q.items()}
    weights["router"] = (act, rnd(E, H).to(tt))
    if Is:
        weights["seg"] = (act, torch.zeros(1, H, device="cuda", dtype=tt))   # a gate of sigmoid(0) = 0.5
    cfg = hx.TextConfig(hidden_size=H, num_experts=E, num_experts_per_tok=k, moe_intermediate_size=I,
                        shared_expert_intermediate_size=Is, norm_topk_prob=True)
    torch.cuda.synchronize()
    return hx.Qwen3_5MoeBlock.load(cfg, weights, act_dtype=act), w, q


def tokens(seed, T, H, act):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((T, H), generator=g, device="cuda")
    return x.to(torch.bfloat16) if act == BF16 else x


@pytest.mark.parametrize("act", [BF16, F32])
@pytest.mark.parametrize("shape", [(256, 16, 4, 128, 128), (160, 40, 6, 96, 0), (2048, 32, 10, 512, 512)])
def test_forward_is_route_then_experts(shape, act):
    import torch
    H, E, k, I, Is = shape
    blk, _, q = make(H, H, E, k, I, Is, act)
    vals = {n: M.values(v.cpu().numpy()) for n, v in q.items()}
    for T in (1, 2, 6, 8, 9, 33, 130):
        x = tokens(T, T, H, act)
        y = blk.forward(x)
        r = blk.route(x)
        sw = torch.full((T,), 0.5, device="cuda") if Is else None
        assert torch.equal(y, blk.experts(x, r["topk_idx"], r["topk_w"], shared_w=sw)), T
        few = T <= (8 if act == BF16 else 6) and T * ((H + 127) // 128 * 4) * (80 if act == BF16 else 128) <= 60 * 1024
        ref, bound = M.experts_bound(x.float().cpu().numpy(), r["topk_idx"].cpu().numpy(), r["topk_w"].cpu().numpy(),
                                     vals, sw.cpu().numpy() if Is else None, act == BF16, few)
        assert (np.abs(y.float().cpu().numpy() - ref) <= bound).all(), T
        assert torch.equal(blk.forward(x.view(1, T, H)).view(T, H), y)
        out = torch.empty_like(x)
        assert torch.equal(blk.forward_noalloc(x, out), y)


def test_forward_host_equals_forward():
    import torch
    from helexa_amd import moe as hx
    H, E, k, I, Is = 256, 8, 2, 64, 64
    blk, _, _ = make(3, H, E, k, I, Is, F32)
    for T in (1, 40):
        x = tokens(T, T, H, F32)
        y = blk.forward(x).cpu().numpy()
        xh, yh = x.cpu().numpy(), np.zeros((T, H), np.float32)
        hx.check(hx.lib().hx_moe_forward_host(blk.handle, xh.ctypes.data_as(C.c_void_p), T,
                                              yh.ctypes.data_as(C.c_void_p), None), "hx_moe_forward_host")
        assert np.array_equal(yh, y)
    torch.cuda.synchronize()


@pytest.mark.parametrize("act", [BF16, F32])
@pytest.mark.parametrize("T", [1, 7, 20, 100])
def test_decoder_half(T, act):
    """rows of +-1 with eps 0 and norm_w 0 are their own RMSNorm, so that the stream
    becomes x + forward(x), forward(x) rounded to the activations' type first; also
    where the stream is off 16 bytes"""
    import torch
    H, E, k, I, Is = 256, 16, 4, 128, 128
    blk, _, _ = make(8, H, E, k, I, Is, act)
    x = tokens(T, T, H, act).sign()
    x[x == 0] = 1
    want = x + blk.forward(x)
    nw = torch.zeros(H, device="cuda")
    assert torch.equal(blk.decoder_mlp_(x.clone(), nw, 0.0), want)
    base = torch.zeros(T * H + 1, dtype=x.dtype, device="cuda")
    base[1:] = x.view(-1)
    assert torch.equal(blk.decoder_mlp_(base[1:].view(T, H), nw, 0.0), want)
    # an ordinary norm: finite, and the stream moved
    y = blk.decoder_mlp_(tokens(5, T, H, act), torch.randn(H, device="cuda"), 1e-6)
    assert torch.isfinite(y).all()


@pytest.mark.parametrize("T", [1, 8, 30])
def test_stack_of_layers_in_a_graph(T):
    """three layers on one stream of tokens and one workspace, captured; replays between
    eager calls give the eager bits"""
    import torch
    H, E, k, I, Is = 256, 16, 4, 128, 128
    blks = [make(s, H, E, k, I, Is, BF16)[0] for s in (1, 2, 3)]
    nw = torch.randn(H, device="cuda") * 0.1
    ws = torch.empty(max(b.workspace_size(T) for b in blks), dtype=torch.uint8, device="cuda")

    def stack(x):
        for b in blks:
            b.decoder_mlp_(x, nw, 1e-6, workspace=ws)
        return x
    ins = [tokens(s, T, H, BF16) for s in range(3)]
    refs = [stack(x.clone()).clone() for x in ins]
    x = ins[0].clone()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        stack(x)
    for r in range(4):
        x.copy_(ins[r % 3])
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(x, refs[r % 3]), r
        assert torch.equal(stack(ins[(r + 1) % 3].clone()), refs[(r + 1) % 3])


def test_workspace_sizes():
    """a buffer sized for T tokens serves every smaller call; the handle's own grows with the calls"""
    import torch
    H, E, k, I, Is = 256, 16, 4, 128, 128
    for act in (BF16, F32):
        blk, _, _ = make(4, H, E, k, I, Is, act)
        sizes = [blk.workspace_size(T) for T in range(0, 600)] + [blk.workspace_size(T) for T in (5000, 70000, 70001, 300000)]
        assert all(a <= b for a, b in zip(sizes, sizes[1:]))
        ws = torch.empty(blk.workspace_size(50), dtype=torch.uint8, device="cuda")
        for T in (50, 1, 9, 8, 33):
            x = tokens(T, T, H, act)
            assert torch.equal(blk.forward(x, workspace=ws), blk.forward(x))


def test_many_tokens_one_call():
    """a routing of several dispatch chunks: 20,000 tokens, compared with the same tokens in calls of 500"""
    import torch
    H, E, k, I = 64, 32, 8, 32
    blk, _, _ = make(6, H, E, k, I, 0, BF16)
    x = tokens(2, 20000, H, BF16)
    g = torch.Generator(device="cuda").manual_seed(3)
    idx = torch.randint(-1, E, (20000, k), generator=g, device="cuda", dtype=torch.int32)
    w = torch.rand((20000, k), generator=g, device="cuda")
    y = blk.experts(x, idx, w)
    for a in range(0, 20000, 500):
        assert torch.equal(blk.experts(x[a:a + 500], idx[a:a + 500], w[a:a + 500]), y[a:a + 500]), a


@pytest.mark.parametrize("act", [BF16, F32])
def test_more_rows_than_the_last_cache(act):
    """experts' rows of more than 256 MB, compared with the same tokens in calls of 300"""
    import torch
    H, E, k, I, Is, T = 2048, 8, 8, 32, 32, 8000 if act == BF16 else 4000
    blk, _, _ = make(7, H, E, k, I, Is, act)
    x = tokens(3, T, H, act)
    g = torch.Generator(device="cuda").manual_seed(4)
    idx = torch.randint(-1, E, (T, k), generator=g, device="cuda", dtype=torch.int32)
    w = torch.rand((T, k), generator=g, device="cuda")
    sw = torch.rand(T, generator=g, device="cuda")
    y = blk.experts(x, idx, w, shared_w=sw)
    for a in (0, 100, T // 2, T - 300):
        b = slice(a, a + 300)
        assert torch.equal(blk.experts(x[b], idx[b], w[b], shared_w=sw[b]), y[b]), a
    blk.close()


def test_a_routing_without_dimensions_is_refused():
    import torch
    blk, _, _ = make(8, 64, 4, 1, 32, 0, BF16)
    x, i, w = tokens(1, 1, 64, BF16), torch.tensor(1, device="cuda", dtype=torch.int32), torch.tensor(0.5, device="cuda")
    with pytest.raises(ValueError, match="topk_idx"):
        blk.experts(x, i, w.view(1, 1))
    with pytest.raises(ValueError, match="topk_w"):
        blk.experts(x, i.view(1, 1), w)


def test_timing_slots():
    H, E, k, I, Is = 256, 16, 4, 128, 128
    blk, _, _ = make(4, H, E, k, I, Is, BF16)
    for T, slots in ((1, {"gate_up", "down"}), (40, {"x_f16", "gate_up", "down", "combine"})):
        x = tokens(1, T, H, BF16)
        blk.forward(x)
        blk.timing_begin(2)
        blk.forward(x)
        blk.forward(x)
        t = {n for n, (ms, c) in blk.timing_end().items() if c == 2 and ms > 0}
        assert slots <= t, t


def test_quantised_weights_lose_what_the_format_loses():
    """the device's rows against numpy's, for a checkpoint's distribution"""
    _, w, q = make(9, 96, 3, 2, 64, 0, F32)
    for n in w:
        assert np.array_equal(q[n].cpu().numpy(), M.quantise(w[n].cpu().numpy())), n
