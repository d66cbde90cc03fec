"""Blocks of E4M3 experts: experts() with a routing of the caller's against 64 bits, the block's other calls."""
import numpy as np
import pytest

import f8 as F

pytestmark = pytest.mark.gpu
BF16, F32 = 30, 0


def cuda(a, bf=False):
    import torch
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t.to(torch.bfloat16) if bf else t


def acts(seed, T, H, act):
    x = np.random.default_rng(seed).standard_normal((T, H), dtype=np.float32)
    return F.bf16(x) if act == BF16 else x


def check(y, x, idx, w, d, sw, act):
    import torch
    ref, bound = F.experts(x, idx, w, d, sw, act == BF16)
    got = y.float().cpu().numpy().astype(np.float64).reshape(ref.shape)
    off = np.abs(got - ref)
    norm = np.linalg.norm(off) / max(np.linalg.norm(ref), 1e-300)
    print(f"[err] worst {np.max(off / bound, initial=0):.3f} of the bound, norm {norm:.2e}", flush=True)
    assert (off <= bound).all(), np.argwhere(~(off <= bound))[:5]
    # two roundings to bf16, each of at most 2^-8 of what it rounds; f32: what a few values of h
    # lose that fall to the neighbouring code, 2^-3 of each at most
    assert norm <= (2.0 ** -7 if act == BF16 else 2.0 ** -8)


TOKENS = [1, 2, 5, 16, 17, 40, 130, 600]
BLOCKS = [(256, 16, 4, 128, 128), (96, 5, 2, 160, 0), (160, 40, 3, 32, 288), (32, 3, 3, 64, 32), (544, 8, 2, 416, 96), (2048, 24, 10, 512, 512)]


@pytest.mark.parametrize("act", [F32, BF16])
@pytest.mark.parametrize("H,E,k,I,Is", BLOCKS)
def test_experts(H, E, k, I, Is, act):
    d = F.block(H + I, H, E, I, Is)
    blk = F.load(d, H, E, k, I, Is, act)
    for T in TOKENS if H < 2048 else [1, 9, 40, 200]:
        for padded in sorted({0, T // 3}):
            print("case", H, E, k, I, Is, act, T, padded, flush=True)
            x = acts(T, T, H, act)
            idx, w, sw = F.routing(T + padded, T, E, k, padded)
            y = blk.experts(cuda(x, act == BF16), cuda(idx), cuda(w), shared_w=cuda(sw) if Is else None)
            check(y, x, idx, w, d, sw if Is else None, act)
    blk.close()


@pytest.mark.parametrize("act", [F32, BF16])
@pytest.mark.parametrize("T", [1, 3, 16, 50, 300])
def test_routings_at_the_edges(T, act):
    """one expert for all, the same index twice, indices outside on either side, no shared expert
    in the call, nothing at all"""
    H, E, k, I, Is = 160, 6, 4, 96, 64
    d = F.block(3, H, E, I, Is)
    blk = F.load(d, H, E, k, I, Is, act)
    x = acts(T, T, H, act)
    _, w, sw = F.routing(T, T, E, k)
    xt, wt = cuda(x, act == BF16), cuda(w)
    for idx in (np.full((T, k), 5), np.tile([2, 2, 2, 0], (T, 1)), np.tile([6, -1, 3, 2 ** 31 - 1], (T, 1)), np.tile([-2 ** 31, 1, 1, 6], (T, 1)),
                np.full((T, k), -1)):
        idx = idx.astype(np.int32)
        check(blk.experts(xt, cuda(idx), wt, shared_w=cuda(sw)), x, idx, w, d, sw, act)
        y = blk.experts(xt, cuda(idx), wt)
        check(y, x, idx, w, d, None, act)
    assert not y.any()
    blk.close()


@pytest.mark.parametrize("T", [1, 7, 33, 200])
def test_many_choices_and_weights_of_any_size(T):
    """64 entries a token; weights negative, zero, far apart"""
    H, E, k, I = 64, 80, 64, 32
    d = F.block(4, H, E, I, 0)
    blk = F.load(d, H, E, k, I, 0, F32)
    x = acts(T, T, H, F32)
    idx, w, _ = F.routing(T, T, E, k)
    w = (w - 0.5) * np.exp2(np.random.default_rng(T).integers(-20, 20, w.shape)).astype(np.float32)
    w[:, 3] = 0
    ref, bound = F.experts(x, idx, w, d, None, False)
    y = blk.experts(cuda(x), cuda(idx), cuda(w)).cpu().numpy()
    assert (np.abs(y - ref) <= bound).all()
    blk.close()


@pytest.mark.parametrize("act", [F32, BF16])
@pytest.mark.parametrize("T", [2, 16, 40, 300])
def test_tokens_without_numbers_stay_by_themselves(T, act):
    H, E, k, I, Is = 256, 8, 3, 128, 128
    d = F.block(5, H, E, I, Is)
    blk = F.load(d, H, E, k, I, Is, act)
    x = acts(T, T, H, act)
    idx, w, sw = F.routing(T, T, E, k)
    call = lambda a: blk.experts(cuda(a, act == BF16), cuda(idx), cuda(w), shared_w=cuda(sw)).float().cpu().numpy()
    plain = call(x)
    x[1, 130] = np.nan
    x[0, 5] = np.inf if T > 2 else x[0, 5]
    y = call(x)
    bad = [0, 1] if T > 2 else [1]
    assert np.isnan(y[bad]).all()
    keep = np.setdiff1d(np.arange(T), bad)
    assert np.array_equal(y[keep], plain[keep])
    blk.close()


@pytest.mark.parametrize("act", [F32, BF16])
@pytest.mark.parametrize("T", [1, 2, 8, 12, 16, 17, 100, 520])
def test_the_blocks_other_calls(T, act):
    """forward() is experts() with its own routing (bit by bit without a shared expert), in every
    form; decoder_mlp_() is x + forward(rmsnorm(x))"""
    import helexa_amd as hx
    import torch
    H, E, k, I = 256, 32, 4, 128
    rng = np.random.default_rng(T)
    router = rng.standard_normal((E, H)).astype(np.float32)
    seg = rng.standard_normal((1, H)).astype(np.float32) * 0.1
    x = acts(T, T, H, act)
    xt = cuda(x, act == BF16)
    for Is in (0, 96):
        d = F.block(6, H, E, I, Is)
        blk = F.load(d, H, E, k, I, Is, act, router, seg if Is else None)
        y = blk.forward(xt)
        r = blk.route(xt)
        sw = torch.sigmoid((xt.double() @ cuda(seg).double().t())[:, 0]).float() if Is else None
        z = blk.experts(xt, r["topk_idx"], r["topk_w"], shared_w=sw)
        if not Is:
            assert torch.equal(y, z)
        else:
            # the shared expert's gate has the activations' rounding
            assert (y.double() - z.double()).norm() <= (2.0 ** -6 if act == BF16 else 2.0 ** -18) * z.double().norm()
        ws = torch.empty(blk.workspace_size(T), dtype=torch.uint8, device="cuda")
        assert torch.equal(blk.forward(xt, workspace=ws), y) and torch.equal(blk.forward(xt.view(1, T, H)), y.view(1, T, H))
        assert torch.equal(blk.forward_noalloc(xt, torch.empty_like(xt)), y)
        host, xh = torch.empty((T, H), dtype=xt.dtype), xt.cpu()
        hx.moe.check(hx.lib().hx_moe_forward_host(blk.handle, xh.data_ptr(), T, host.data_ptr(), None), "forward_host")
        assert torch.equal(host.cuda(), y)
        nw = cuda(rng.standard_normal(H).astype(np.float32) * 0.1)
        n = xt.double()
        n = (n * torch.rsqrt((n * n).mean(dim=1, keepdim=True) + 1e-6) * (1 + nw.double())).to(xt.dtype)
        want = xt.double() + blk.forward(n).double()
        got = blk.decoder_mlp_(xt.clone(), nw, 1e-6).double()
        # the norm in 32 bits may move a token's values by a step, which may move codes: a share of the block's part
        assert (got - want).norm() <= 2.0 ** -6 * want.norm()
        out = torch.full((T + 2, H), 3.0, dtype=xt.dtype, device="cuda")
        blk.experts(xt, r["topk_idx"], r["topk_w"], shared_w=sw, out=out[1:T + 1])
        assert torch.equal(out[1:T + 1], z) and (out[0] == 3).all() and (out[T + 1] == 3).all()
        both = xt.clone()
        blk.experts(both, r["topk_idx"], r["topk_w"], shared_w=sw, out=both)
        assert torch.equal(both, z)
        blk.close()


@pytest.mark.parametrize("T", [1, 9, 16, 17, 60, 300])
def test_workspaces_and_smaller_calls(T):
    """a workspace of exactly workspace_size() bytes serves every smaller call, its neighbours stay;
    one off 16 bytes or too small is refused; the handle's own grows"""
    import helexa_amd as hx
    import torch
    H, E, k, I, Is = 160, 12, 5, 96, 64
    d = F.block(7, H, E, I, Is)
    blk = F.load(d, H, E, k, I, Is, BF16)
    n = blk.workspace_size(T)
    big = torch.full((n + 512,), 9, dtype=torch.uint8, device="cuda")
    ws = big[256:256 + n]
    for t in sorted({1, 2, 9, 16, 17, T // 2 + 1, T}):
        if t > T:
            continue
        assert blk.workspace_size(t) <= n
        x = cuda(acts(t, t, H, BF16), True)
        idx, w, sw = (cuda(a) for a in F.routing(t, t, E, k))
        y = blk.experts(x, idx, w, shared_w=sw, workspace=ws)
        assert torch.equal(y, blk.experts(x, idx, w, shared_w=sw)) and blk.forward(x, workspace=ws).shape == x.shape
    torch.cuda.synchronize()
    assert (big[:256] == 9).all() and (big[256 + n:] == 9).all()
    with pytest.raises(hx.HxError):
        blk.experts(x, idx, w, workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))
    with pytest.raises(hx.HxError):
        blk.experts(x, idx, w, workspace=big[8:])
    blk.close()


@pytest.mark.parametrize("T", [1, 7, 30, 250])
def test_captured_replayed_and_on_another_stream(T):
    import torch
    H, E, k, I, Is = 256, 16, 4, 128, 128
    d = F.block(8, H, E, I, Is)
    blk = F.load(d, H, E, k, I, Is, BF16)
    sets = []
    for i in range(3):
        idx, w, sw = F.routing(T + i, T, E, k, padded=i if T > 3 else 0)
        sets.append([cuda(acts(T + i, T, H, BF16), True), cuda(idx), cuda(w), cuda(sw)])
    want = [blk.experts(a, b, c, shared_w=e) for a, b, c, e in sets]
    ws = torch.empty(blk.workspace_size(T), dtype=torch.uint8, device="cuda")
    s = torch.cuda.Stream()
    mine = [t.clone() for t in sets[0]]
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        torch.cuda._sleep(20_000_000)
    y = blk.experts(*mine[:3], shared_w=mine[3], stream=s, workspace=ws)
    del mine
    junk = [torch.zeros_like(t) for t in sets[0] for _ in range(3)]
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(y, want[0])
    held = [t.clone() for t in sets[0]]
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = blk.experts(*held[:3], shared_w=held[3], workspace=ws)
    for i in (1, 2, 0, 1):
        for h, t in zip(held, sets[i]):
            h.copy_(t)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i]) and torch.equal(blk.experts(*sets[i][:3], shared_w=sets[i][3]), want[i])
    del junk
    blk.close()


def test_host_weights_and_refusals():
    import helexa_amd as hx
    import torch
    H, E, k, I, Is = 96, 4, 2, 64, 32
    d = F.block(9, H, E, I, Is)
    a, b = F.load(d, H, E, k, I, Is, F32), F.load(d, H, E, k, I, Is, F32, host=True)
    x = cuda(acts(1, 20, H, F32))
    idx, w, sw = (cuda(t) for t in F.routing(1, 20, E, k))
    assert torch.equal(a.experts(x, idx, w, shared_w=sw), b.experts(x, idx, w, shared_w=sw))
    cfg = a.cfg
    good = {n: (hx.F8_E4M3, cuda(c), cuda(s)) for n, (c, s) in d.items()}
    good["router"] = (hx.F32, torch.zeros((E, H), device="cuda"))
    good["seg"] = (hx.F32, torch.zeros((1, H), device="cuda"))
    hx.Qwen3_5MoeBlock.load(cfg, good, act_dtype=hx.F32)
    for key, entry, err in (("gate", (hx.F8_E4M3, good["gate"][1]), ValueError), ("gate", good["gate"][:2] + (good["gate"][2][:1],), ValueError),
                            ("down", (hx.F8_E4M3, good["down"][1].transpose(1, 2), good["down"][2]), ValueError),
                            ("sup", (hx.F8_E4M3, good["sup"][1].float(), good["sup"][2]), ValueError),
                            ("up", good["up"][:2] + (good["up"][2].cpu(),), ValueError),
                            ("down", (hx.BF16, torch.zeros((E, H, I), dtype=torch.bfloat16, device="cuda")), hx.HxError),
                            ("sdown", (hx.F32, torch.zeros((H, Is), device="cuda")), hx.HxError)):
        with pytest.raises(err):
            hx.Qwen3_5MoeBlock.load(cfg, {**good, key: entry}, act_dtype=hx.F32)


def test_a_model_is_quantised_routed_run_and_balanced():
    """float weights through quantize_f8 into a block, its forward, then the balance loss of its
    routing; a linear layer on the block's outputs"""
    import helexa_amd as hx
    import torch
    H, E, k, I, T = 256, 16, 4, 128, 70
    g = torch.Generator(device="cuda").manual_seed(1)
    draw = lambda *s: torch.randn(s, generator=g, device="cuda") * 0.05
    flt = dict(gate=draw(E, I, H), up=draw(E, I, H), down=draw(E, H, I), sgate=draw(I, H), sup=draw(I, H), sdown=draw(H, I))
    w = {n: (hx.F8_E4M3,) + hx.quantize_f8(t, block_rows=128) for n, t in flt.items()}
    w["router"], w["seg"] = (hx.F32, draw(E, H) * 10), (hx.F32, draw(1, H))
    cfg = hx.TextConfig(hidden_size=H, num_experts=E, num_experts_per_tok=k, moe_intermediate_size=I, shared_expert_intermediate_size=I, norm_topk_prob=True)
    blk = hx.Qwen3_5MoeBlock.load(cfg, w, act_dtype=hx.F32)
    ref = hx.Qwen3_5MoeBlock.load(cfg, {n: (hx.F32, flt[n]) if n in flt else w[n] for n in w}, act_dtype=hx.F32)
    x = torch.randn((T, H), generator=g, device="cuda")
    y, z = blk.forward(x), ref.forward(x)
    # four roundings to E4M3 on the way of a product, each of at most 2^-4 of the value
    assert (y - z).norm() <= 4 * 2.0 ** -4 * z.norm()
    r = blk.route(x)
    out = hx.balance_loss(blk.router_logits(x), r["topk_idx"])
    assert torch.equal(out["counts"], r["offsets"][1:] - r["offsets"][:-1]) and float(out["loss"]) > 0
    layer = hx.F8Linear.load(*hx.quantize_f8(draw(192, H), block_rows=128))
    assert layer(y).shape == (T, 192)
    blk.close(), ref.close(), layer.close()


@pytest.mark.parametrize("T,E,k,skew", [(90, 4, 3, 0), (250, 3, 3, 0), (333, 6, 4, 3), (129, 1, 1, 0), (700, 5, 2, 3)])
def test_many_rows_an_expert(T, E, k, skew):
    """tiles of 128 rows: their halves full, in part and empty, sizes that are no whole blocks, the same
    token twice with an expert, padded tokens"""
    for H, I, Is in ((256, 128, 128), (160, 96, 64), (544, 416, 0), (128, 32, 288)):
        d = F.block(T + H, H, E, I, Is)
        blk = F.load(d, H, E, k, I, Is, BF16)
        print("case", T, E, k, H, I, Is, flush=True)
        x = acts(T, T, H, BF16)
        idx, w, sw = F.routing(T, T, E, k, padded=T // 7)
        rng = np.random.default_rng(T)
        if skew:
            idx = np.where((rng.random(idx.shape) < 0.5) & (idx >= 0), 0, idx).astype(np.int32)
        check(blk.experts(cuda(x, True), cuda(idx), cuda(w), shared_w=cuda(sw) if Is else None), x, idx, w, d, sw if Is else None, BF16)
        x[1, 3] = np.nan
        y = blk.experts(cuda(x, True), cuda(idx), cuda(w), shared_w=cuda(sw) if Is else None)
        import torch
        assert torch.isnan(y[1]).all() and torch.isfinite(y[2:]).all() and torch.isfinite(y[0]).all()
        blk.close()


@pytest.mark.parametrize("M,N,K", [(300, 9000, 260), (1100, 4100, 130), (5000, 3300, 100), (257, 16640, 384)])
def test_a_layers_large_tiles(M, N, K):
    """rows and features that fill tiles of 256 and 128 in part"""
    import helexa_amd as hx
    import torch
    codes, scales = F.make_weights(M, N, K)
    x = F.bf16(np.random.default_rng(M).standard_normal((M, K)).astype(np.float32))
    y = hx.F8Linear.load(cuda(codes), cuda(scales))(cuda(x, True))
    rows = np.unique(np.concatenate([np.arange(3), np.arange(M - 3, M), np.random.default_rng(1).integers(0, M, 40)]))
    ref, mag, fixed = F.linear(x[rows], codes, scales)
    bound = (F.sum_steps(K) * F.U * mag + fixed) * (1 + 2.0 ** -8) + 2.0 ** -8 * np.abs(ref) + 2.0 ** -140
    off = np.abs(y[torch.from_numpy(rows).cuda()].float().cpu().numpy().astype(np.float64) - ref)
    assert (off <= bound).all()
    # every element, against the same product in bf16 operands and float32 sums by another path of the layer
    z = hx.F8Linear.load(cuda(codes), cuda(scales))(cuda(x, True), out_dtype=torch.float32)
    assert (y.float() - z).norm() <= 2.0 ** -8 * z.norm() and ((y.float() - z).abs() <= 2.0 ** -7 * z.abs() + 2.0 ** -7 * z.std()).all()


@pytest.mark.parametrize("act", [F32, BF16])
def test_the_widest_tokens(act):
    """the codes of one fit where the few-token kernel quantises them, those of two do not"""
    H, E, k, I, Is = 16384, 3, 2, 64, 32
    d = F.block(5, H, E, I, Is)
    blk = F.load(d, H, E, k, I, Is, act)
    for T in (1, 2, 5, 20):
        print("case", act, T, flush=True)
        x = acts(T, T, H, act)
        idx, w, sw = F.routing(T, T, E, k, 0)
        y = blk.experts(cuda(x, act == BF16), cuda(idx), cuda(w), shared_w=cuda(sw))
        check(y, x, idx, w, d, sw, act)
    blk.close()
