"""Per-expert counts and the balance loss against 64 bits: sizes, types, masks, strides, streams, graphs."""
import numpy as np
import pytest

import balance as B

pytestmark = pytest.mark.gpu


def cuda(a, bf=False):
    import torch
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t.to(torch.bfloat16) if bf else t


def check(out, x, idx, coef, counts=None, bf=False):
    """x as the kernel has it, float32"""
    r = B.reference(x, idx, coef, counts)
    b = B.bounds(x, r, x.shape[0], 2.0 ** -8 if bf else 2.0 ** -24)
    assert np.array_equal(out["counts"].cpu().numpy(), r["counts"])
    for name in ("loss", "probs", "dlogits"):
        if out[name] is None:
            continue
        got = out[name].float().cpu().numpy().astype(np.float64).reshape(np.shape(r[name]))
        off = np.abs(got - r[name])
        worst = float(np.max(off / np.maximum(b[name], 1e-300), initial=0.0))
        print(f"[err] {name}: worst {worst:.3f} of the bound", flush=True)
        assert (off <= b[name]).all(), (name, worst)
    return r


SIZES = [(1, 1, 1), (1, 4, 2), (7, 5, 3), (33, 16, 4), (64, 512, 10), (65, 512, 10), (300, 130, 8), (1000, 1024, 64),
         (257, 1000, 7), (1, 1024, 64), (5000, 48, 6), (1024, 8, 2), (1025, 8, 2), (20001, 512, 10), (3001, 772, 5)]


@pytest.mark.parametrize("bf", [False, True])
@pytest.mark.parametrize("T,E,k", SIZES)
def test_loss_counts_and_gradient(T, E, k, bf):
    import helexa_amd as hx
    for padded in sorted({0, T // 3}):
        print("case", T, E, k, bf, padded, flush=True)
        x, idx = B.inputs(T + E, T, E, k, padded)
        t = cuda(x, bf)
        out = hx.balance_loss(t, cuda(idx), coef=0.01)
        check(out, t.float().cpu().numpy(), idx, 0.01, bf=bf)
        assert np.array_equal(hx.expert_counts(cuda(idx), E).cpu().numpy(), B.counts_of(idx, E))
        again = hx.balance_loss(t, cuda(idx), coef=0.01)
        assert all((out[n].view(-1) == again[n].view(-1)).all() for n in out)


@pytest.mark.parametrize("T", [40, 3000])
def test_masks_and_far_logits(T):
    """-inf for experts that a token may not choose, logits far apart and far from zero, the
    same index several times in a token, tokens with some entries outside"""
    import helexa_amd as hx
    E, k = 64, 6
    x, idx = B.inputs(T, T, E, k, 4)
    rng = np.random.default_rng(T)
    x[:T - 4][rng.random((T - 4, E)) < 0.3] = -np.inf
    x[:T - 4, 0] = 1.0
    x[5] = np.where(np.arange(E) == 9, 3.0e38, -3.0e38)
    x[6] += 80.0 * rng.standard_normal(E).astype(np.float32)
    x[7] = 5e4
    idx[8] = 3
    idx[9, 1:] = -1
    idx[10, :5] = E
    check(hx.balance_loss(cuda(x), cuda(idx), coef=1.0), x, idx, 1.0)


@pytest.mark.parametrize("T", [40, 3000])
def test_a_live_row_without_a_number_shows(T):
    import helexa_amd as hx
    import torch
    for v in (np.nan, np.inf):
        x, idx = B.inputs(T, T, 64, 6)
        x[3, 7] = v
        out = hx.balance_loss(cuda(x), cuda(idx))
        assert torch.isnan(out["loss"]) and torch.isnan(out["probs"]).all() and torch.isnan(out["dlogits"][3]).all()
        assert torch.isfinite(out["dlogits"][4:]).all() and torch.isfinite(out["dlogits"][:3]).all()


@pytest.mark.parametrize("T", [0, 9, 2000])
def test_without_live_tokens_or_counts(T):
    import helexa_amd as hx
    import torch
    E, k = 32, 4
    x, idx = B.inputs(T + 1, T, E, k, T)
    out = hx.balance_loss(cuda(x), cuda(idx))
    assert float(out["loss"]) == 0.0 and not out["probs"].any() and not out["counts"].any()
    assert out["dlogits"].shape == (T, E) and not out["dlogits"].any()
    assert not hx.expert_counts(cuda(idx), E).any()
    if T:
        x, idx = B.inputs(T + 1, T, E, k)
        out = hx.balance_loss(cuda(x), cuda(idx), counts=torch.zeros(E, dtype=torch.int32, device="cuda"))
        assert float(out["loss"]) == 0.0 and not out["dlogits"].any() and out["probs"].any() and out["counts"].sum() == T * k


@pytest.mark.parametrize("T", [100, 4000])
def test_counts_of_several_calls(T):
    """counts added up over two batches, near the end of their 32 bits too"""
    import helexa_amd as hx
    x, idx = B.inputs(T, T, 96, 8, 5)
    _, other = B.inputs(T + 1, T, 96, 8)
    both = hx.expert_counts(cuda(idx), 96) + hx.expert_counts(cuda(other), 96)
    check(hx.balance_loss(cuda(x), cuda(idx), coef=2.0, counts=both), x, idx, 2.0, both.cpu().numpy())
    far = np.full(96, 2 ** 31 - 1, np.int32)
    far[3] = 5
    check(hx.balance_loss(cuda(x), cuda(idx), coef=2.0, counts=cuda(far)), x, idx, 2.0, far)


@pytest.mark.parametrize("bf", [False, True])
@pytest.mark.parametrize("T,E", [(50, 64), (700, 520)])
def test_layouts(T, E, bf):
    """logits off 16 bytes, strided logits and indices, leading dimensions, no gradient, the gradient in the logits' place"""
    import helexa_amd as hx
    import torch
    from helexa_amd import moe
    x, idx = B.inputs(T, T, E, 5)
    t, i = cuda(x, bf), cuda(idx)
    want = hx.balance_loss(t, i)
    off = torch.empty(T * E + 1, dtype=t.dtype, device="cuda")[1:].view(T, E)
    off.copy_(t)
    check(hx.balance_loss(off, i), t.float().cpu().numpy(), idx, 1.0, bf=bf)
    wide = torch.zeros((T, E + 7), dtype=t.dtype, device="cuda")
    wide[:, 3:E + 3] = t
    iw = torch.zeros((T, 9), dtype=torch.int32, device="cuda")
    iw[:, ::2] = i
    got = hx.balance_loss(wide[:, 3:E + 3], iw[:, ::2])
    assert all(torch.equal(got[n], want[n]) for n in want)
    got = hx.balance_loss(t.view(2, T // 2, E), i.view(2, T // 2, 5), grad=False)
    assert got["dlogits"] is None and torch.equal(got["loss"], want["loss"]) and torch.equal(got["probs"], want["probs"])
    ws = torch.empty(hx.balance_workspace_size(T, E), dtype=torch.uint8, device="cuda")
    both = t.clone()
    loss, probs = torch.empty((), device="cuda"), torch.empty(E, device="cuda")
    moe.check(moe.lib().hx_moe_balance_loss(both.data_ptr(), hx.BF16 if bf else hx.F32, T, E, i.data_ptr(), 5, None, 1.0,
                                            loss.data_ptr(), None, probs.data_ptr(), both.data_ptr(), ws.data_ptr(), ws.nbytes,
                                            torch.cuda.current_stream().cuda_stream), "hx_moe_balance_loss")
    assert torch.equal(both, want["dlogits"]) and torch.equal(loss, want["loss"])


def test_the_gradient_is_the_losss():
    """differences of the kernel's own loss along a direction: each loss is off by its bound, the
    quotient besides by what 64 bits' quotient is off their derivative"""
    import helexa_amd as hx
    T, E, k, h = 24, 20, 3, 0.05
    x, idx = B.inputs(3, T, E, k)
    rng = np.random.default_rng(4)
    r = B.reference(x, idx, 1.0)
    b = B.bounds(x, r, T, 2.0 ** -24)
    grad = hx.balance_loss(cuda(x), cuda(idx))["dlogits"].cpu().numpy().astype(np.float64)
    for _ in range(4):
        v = rng.standard_normal(x.shape).astype(np.float32)
        hi, lo = (x + np.float32(s * h) * v for s in (1, -1))
        step = hi.astype(np.float64) - lo   # what was added, after rounding
        ours = float(hx.balance_loss(cuda(hi), cuda(idx))["loss"]) - float(hx.balance_loss(cuda(lo), cuda(idx))["loss"])
        rh, rl = (B.reference(a, idx, 1.0) for a in (hi, lo))
        exact = rh["loss"] - rl["loss"]
        far = abs(exact - float((r["dlogits"] * step).sum()))
        tol = 2 * max(B.bounds(hi, rh, T, 0)["loss"], B.bounds(lo, rl, T, 0)["loss"]) + far + float((b["dlogits"] * abs(step)).sum())
        assert far < 0.2 * abs(exact) and abs(ours - float((grad * step).sum())) <= tol


@pytest.mark.parametrize("T", [20, 3000])
def test_another_stream_and_dropped_tensors(T):
    import helexa_amd as hx
    import torch
    x, idx = B.inputs(T, T, 128, 8, 3)
    want = hx.balance_loss(cuda(x), cuda(idx))
    s = torch.cuda.Stream()
    a, i = cuda(x), cuda(idx)
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        torch.cuda._sleep(20_000_000)
    got = hx.balance_loss(a, i, stream=s)
    c = hx.expert_counts(i, 128, stream=s)
    del a, i
    junk = [torch.full((T, 128), 7.0, device="cuda") for _ in range(4)]   # takes what was freed
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(got[n], want[n]) for n in want) and torch.equal(c, want["counts"])
    del junk


@pytest.mark.parametrize("T", [20, 3000])
def test_captured_and_replayed(T):
    """new logits and indices before each replay, eager work between"""
    import helexa_amd as hx
    import torch
    E, k = 128, 8
    sets = [B.inputs(T + i, T, E, k, i) for i in range(4)]
    a, i = cuda(sets[0][0]), cuda(sets[0][1])
    ws = torch.empty(hx.balance_workspace_size(T, E), dtype=torch.uint8, device="cuda")
    hx.balance_loss(a, i, workspace=ws)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = hx.balance_loss(a, i, workspace=ws)
    for x, idx in sets[1:] + sets[:2]:
        a.copy_(cuda(x))
        i.copy_(cuda(idx))
        g.replay()
        torch.cuda.synchronize()
        want = hx.balance_loss(cuda(x), cuda(idx))
        assert all(torch.equal(out[n], want[n]) for n in want)


def test_with_the_block_it_balances():
    """router_logits() and route() of a block, then the loss: the counts are the dispatch's"""
    import helexa_amd as hx
    import torch
    from helexa_amd import synth
    cfg = synth.C1
    blk = hx.Qwen3_5MoeBlock.load(cfg, synth.make_weights(cfg, synth.FMT_F32, 7), act_dtype=hx.F32)
    x = synth.make_x(cfg, 200, 3, hx.F32)
    logits, r = blk.router_logits(x), blk.route(x)
    out = hx.balance_loss(logits, r["topk_idx"])
    check(out, logits.cpu().numpy(), r["topk_idx"].cpu().numpy(), 1.0)
    assert torch.equal(out["counts"], r["offsets"][1:] - r["offsets"][:-1])
    blk.close()


def test_refusals():
    import helexa_amd as hx
    import torch
    x, idx = B.inputs(1, 10, 16, 4)
    t, i = cuda(x), cuda(idx)
    ws = torch.empty(hx.balance_workspace_size(10, 16) - 1, dtype=torch.uint8, device="cuda")
    for bad, err in ((lambda: hx.balance_loss(t.half(), i), TypeError), (lambda: hx.balance_loss(t.cpu(), i), ValueError),
                     (lambda: hx.balance_loss(t, i.long()), ValueError), (lambda: hx.balance_loss(t, i.cpu()), ValueError),
                     (lambda: hx.balance_loss(t[:9], i), ValueError), (lambda: hx.balance_loss(t, i, workspace=ws), hx.HxError),
                     (lambda: hx.balance_loss(t, i, counts=torch.zeros(15, dtype=torch.int32, device="cuda")), ValueError),
                     (lambda: hx.balance_loss(t, i, counts=torch.zeros(16, device="cuda")), ValueError),
                     (lambda: hx.expert_counts(i, 0), hx.HxError), (lambda: hx.expert_counts(i, 1025), hx.HxError),
                     (lambda: hx.expert_counts(i[:, :0], 16), ValueError),
                     (lambda: hx.balance_loss(torch.zeros((4, 1025), device="cuda"), i[:4]), hx.HxError)):
        with pytest.raises(err):
            bad()
