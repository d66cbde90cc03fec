"""hx_moe_experts on MXFP4 blocks against 64-bit products of the stored weights,
element by element within the bound that the formats and the sums allow
(mxfp4.experts_bound), and what the call promises about routings, special values,
alignment, streams and graphs."""
import numpy as np
import pytest

import mxfp4 as M

pytestmark = pytest.mark.gpu

BF16, F32 = 30, 0


def bf16(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a, np.float32)).to(torch.bfloat16).float().numpy()


def inputs(seed, T, H, E, k, act, distinct=True):
    rng = np.random.default_rng(seed + 1000)
    x = rng.standard_normal((T, H)).astype(np.float32)
    x *= np.exp2(rng.integers(-3, 4, (T, 1))).astype(np.float32)
    if act == BF16:
        x = bf16(x)
    idx = np.stack([rng.permutation(E)[:k] if distinct else rng.integers(0, E, k) for _ in range(T)]).astype(np.int32)
    w = rng.random((T, k)).astype(np.float32)
    return x, idx, w, rng.random(T).astype(np.float32)


def cuda(a, act=None):
    import torch
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t.to(torch.bfloat16) if act == BF16 else t


def few(T, H, act):
    """whether the few-token kernels take the call: their records in 60 KiB"""
    blocks = (H + 127) // 128 * 4
    return T <= (8 if act == BF16 else 6) and T * blocks * (80 if act == BF16 else 128) <= 60 * 1024


def check(y, x, idx, w, vals, sw, act):
    y = y.float().cpu().numpy().astype(np.float64)
    ref, bound = M.experts_bound(x, idx, w, vals, sw, act == BF16, few(*x.shape, act))
    off = np.abs(y - ref) / bound
    print(f"[err] worst {off.max():.3f} of the bound, rel {np.linalg.norm(y - ref) / np.linalg.norm(ref):.2e}", flush=True)
    assert off.max() <= 1.0, np.unravel_index(off.argmax(), off.shape)


SHAPES = [  # H, E, k, I, Is
    (32, 1, 1, 32, 0), (256, 16, 4, 128, 128), (160, 5, 3, 96, 224), (288, 7, 7, 320, 32), (64, 1024, 10, 32, 0),
    (2048, 24, 10, 512, 512), (4096, 4, 2, 64, 64)]


@pytest.mark.parametrize("act", [BF16, F32])
@pytest.mark.parametrize("shape", SHAPES)
def test_experts_against_64_bits(shape, act):
    H, E, k, I, Is = shape
    rows, vals = M.block(H + E, H, E, I, Is)
    blk = M.load(rows, H, E, k, I, Is, act)
    for T in (1, 2, 3, 5, 8, 9, 16, 33, 64, 65, 130):
        print("case", shape, act, T, flush=True)
        x, idx, w, sw = inputs(T, T, H, E, k, act)
        y = blk.experts(cuda(x, act), cuda(idx), cuda(w), shared_w=cuda(sw) if Is else None)
        check(y, x, idx, w, vals, sw if Is else None, act)
    blk.close()


@pytest.mark.parametrize("act", [BF16, F32])
@pytest.mark.parametrize("H", [32, 96, 544])
def test_many_features_of_few_tokens(H, act):
    """few tokens with many groups of features: K by one wave, or shared by two"""
    E, k, I, Is = 64, 10, 1056, 1024
    rows, vals = M.block(H, H, E, I, Is, std=0.02)
    blk = M.load(rows, H, E, k, I, Is, act)
    for T in (1, 2, 6, 8):
        x, idx, w, sw = inputs(T, T, H, E, k, act)
        check(blk.experts(cuda(x, act), cuda(idx), cuda(w), shared_w=cuda(sw)), x, idx, w, vals, sw, act)
    blk.close()


@pytest.mark.parametrize("act", [BF16, F32])
def test_many_rows_an_expert(act):
    """tiles of 64 rows, several an expert, their last rows short; experts without rows"""
    H, E, k, I, Is = 192, 6, 2, 96, 64
    rows, vals = M.block(11, H, E, I, Is)
    blk = M.load(rows, H, E, k, I, Is, act)
    T = 700
    x, idx, w, sw = inputs(3, T, H, E, k, act)
    idx[idx == 4] = 3
    idx[:, 1][idx[:, 1] == idx[:, 0]] = -1
    check(blk.experts(cuda(x, act), cuda(idx), cuda(w), shared_w=cuda(sw)), x, idx, w, vals, sw, act)
    check(blk.experts(cuda(x, act), cuda(idx), cuda(w)), x, idx, w, vals, None, act)


@pytest.mark.parametrize("T", [1, 2, 8, 9, 40, 300])
def test_entries_that_are_no_expert(T):
    """indices outside the experts, weights of NaN at them, whole tokens and whole
    calls of them, the same index twice"""
    import torch
    H, E, k, I, Is = 128, 8, 4, 64, 64
    rows, vals = M.block(2, H, E, I, Is)
    blk = M.load(rows, H, E, k, I, Is, BF16)
    x, idx, w, sw = inputs(7, T, H, E, k, BF16, distinct=False)
    rng = np.random.default_rng(T)
    gone = rng.random((T, k)) < 0.4
    gone[T // 2] = True
    idx[gone] = rng.choice([-1, E, E + 1, 1 << 30, -(1 << 31), 2147483647], gone.sum()).astype(np.int32)
    wn = w.copy()
    wn[gone] = np.nan
    y = blk.experts(cuda(x, BF16), cuda(idx), cuda(wn))
    check(y, x, idx, w, vals, None, BF16)
    assert not y[T // 2].any()
    check(blk.experts(cuda(x, BF16), cuda(idx), cuda(wn), shared_w=cuda(sw)), x, idx, w, vals, sw, BF16)
    none = np.full_like(idx, -1)
    assert not blk.experts(cuda(x, BF16), cuda(none), cuda(wn)).any()
    check(blk.experts(cuda(x, BF16), cuda(none), cuda(wn), shared_w=cuda(sw)), x, none, w, vals, sw, BF16)
    y0 = blk.experts(cuda(x[:0], BF16), cuda(idx[:0]), cuda(w[:0]))
    assert y0.shape == (0, H)
    torch.cuda.synchronize()


@pytest.mark.parametrize("act", [BF16, F32])
@pytest.mark.parametrize("T", [4, 20])
def test_special_values_stay_in_their_rows(T, act):
    """a token of NaN or infinity gives NaN, an expert with NaN scales gives NaN to
    its tokens; every other token's bits stay as they are"""
    import torch
    H, E, k, I, Is = 256, 8, 2, 64, 0
    rows, vals = M.block(9, H, E, I, Is)
    x, idx, w, _ = inputs(5, T, H, E, k, act)
    idx %= E - 1
    clean = M.load(rows, H, E, k, I, Is, act)
    y = clean.experts(cuda(x, act), cuda(idx), cuda(w))
    bad = x.copy()
    bad[1, 3] = np.nan
    bad[2, 250] = np.inf
    yb = clean.experts(cuda(bad, act), cuda(idx), cuda(w))
    assert yb[1:3].isnan().all()
    keep = [t for t in range(T) if t not in (1, 2)]
    assert torch.equal(yb[keep], y[keep])
    for name in ("gate", "up", "down"):
        r = {n: v.copy() for n, v in rows.items()}
        r[name][E - 1, :, 0] = 255
        blk = M.load(r, H, E, k, I, Is, act)
        i2 = idx.copy()
        i2[T - 1, 1] = E - 1
        yb = blk.experts(cuda(x, act), cuda(i2), cuda(w))
        assert yb[T - 1].isnan().all()
        assert torch.equal(yb[:T - 1], y[:T - 1])
        blk.close()


def test_tiny_and_huge_values():
    """blocks of zeros, of denormals, of values near the largest bf16; weights at both
    ends of the scale"""
    import torch
    H, E, k, I = 128, 2, 1, 64
    rows, vals = M.block(4, H, E, I, 0)
    blk = M.load(rows, H, E, k, I, 0, BF16)
    for T in (4, 12):
        x, idx, w, _ = inputs(1, T, H, E, k, BF16)
        x[0] = 0.0
        x[1] = 1e-40
        x[2] *= 1e-30
        x[3, :32] *= 1e6
        x = bf16(x)
        y = blk.experts(cuda(x, BF16), cuda(idx), cuda(w))
        assert not y[0].any()
        live = np.r_[2:T]
        check(y[2:], x[live], idx[live], w[live], vals, None, BF16) if T > 10 else None
        assert y[1].abs().max() < 1e-37
        big = np.full((T, H), 2.0 ** 100, np.float32)
        yb = blk.experts(cuda(big, BF16), cuda(idx), cuda(w))
        torch.cuda.synchronize()
        assert yb.shape == (T, H)


@pytest.mark.parametrize("act", [BF16, F32])
@pytest.mark.parametrize("T", [1, 5, 9, 70])
def test_pointers_off_alignment_and_guards(T, act):
    """x and y on the smallest alignment of their type, nothing written around y or
    behind the workspace"""
    import torch
    from helexa_amd import moe as hx
    H, E, k, I, Is = 160, 6, 3, 96, 32
    rows, vals = M.block(21, H, E, I, Is)
    blk = M.load(rows, H, E, k, I, Is, act)
    x, idx, w, sw = inputs(2, T, H, E, k, act)
    xt = cuda(x, act)
    ref = blk.experts(xt, cuda(idx), cuda(w), shared_w=cuda(sw))
    es = xt.element_size()
    xs = torch.zeros(T * H + 8, dtype=xt.dtype, device="cuda")
    xs[1:1 + T * H] = xt.view(-1)
    ys = torch.full((T * H + 8,), 3.0, dtype=xt.dtype, device="cuda")
    n = blk.workspace_size(T)
    ws = torch.full((n + 256,), 7, dtype=torch.uint8, device="cuda")
    it, wt, st = cuda(idx), cuda(w), cuda(sw)
    s = torch.cuda.current_stream().cuda_stream
    args = (blk.handle, xs.data_ptr() + es, T, it.data_ptr(), wt.data_ptr(), st.data_ptr(), ys.data_ptr() + es)
    hx.check(hx.lib().hx_moe_experts(*args, ws.data_ptr(), n, s), "hx_moe_experts")
    assert torch.equal(ys[1:1 + T * H].view(T, H), ref)
    assert (ys[0] == 3).all() and (ys[1 + T * H:] == 3).all() and (ws[n:] == 7).all()
    # a workspace off 16 bytes or too small is refused, y untouched
    before = ys.clone()
    assert hx.lib().hx_moe_experts(*args, ws.data_ptr() + 4, n, s) == 1
    assert hx.lib().hx_moe_experts(*args, ws.data_ptr(), 1024, s) == 4
    torch.cuda.synchronize()
    assert torch.equal(before, ys)
    # in place
    y = blk.experts(xt, it, wt, shared_w=st, out=xt)
    assert y is xt and torch.equal(xt, ref)


@pytest.mark.parametrize("T", [1, 6, 24, 90])
def test_streams_and_graphs(T):
    """another stream than the current one; a captured call replayed between eager
    calls on other inputs, two graphs in turn on one workspace; a capture without a
    workspace of the caller's is refused"""
    import torch
    from helexa_amd import moe as hx
    H, E, k, I, Is = 256, 16, 4, 128, 128
    rows, _ = M.block(5, H, E, I, Is)
    blk = M.load(rows, H, E, k, I, Is, BF16)
    ins = []
    for i in range(4):
        x, idx, w, sw = inputs(50 + i, T, H, E, k, BF16)
        ins.append([cuda(x, BF16), cuda(idx), cuda(w), cuda(sw)])
    refs = [blk.experts(a, b, c, shared_w=d).clone() for a, b, c, d in ins]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    out = blk.experts(*ins[1][:3], shared_w=ins[1][3], stream=s)
    s.synchronize()
    assert torch.equal(out, refs[1])
    ws = torch.empty(blk.workspace_size(T), dtype=torch.uint8, device="cuda")
    graphs = []
    for i in range(2):
        a = [t.clone() for t in ins[i]]
        y = torch.empty_like(a[0])
        blk.experts(*a[:3], shared_w=a[3], workspace=ws, out=y)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            blk.experts(*a[:3], shared_w=a[3], workspace=ws, out=y)
        graphs.append((g, a, y))
    for r in range(3):
        for i, (g, a, y) in enumerate(graphs):
            j = (i + r) % 4
            for t, v in zip(a, ins[j]):
                t.copy_(v)
            y.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, refs[j]), (r, i)
            assert torch.equal(blk.experts(*ins[3][:3], shared_w=ins[3][3]), refs[3])
    g = torch.cuda.CUDAGraph()
    y = torch.empty_like(ins[0][0])
    with torch.cuda.graph(g):
        with pytest.raises(hx.HxError, match="workspace"):
            blk.experts(*ins[0][:3], out=y)
        y.zero_()


def test_same_bits_each_time_and_in_any_batch():
    """the order in which rows get their places does not show: calls repeat bit for bit, and a
    token's row does not depend on the others"""
    import torch
    H, E, k, I, Is = 256, 4, 3, 128, 32
    rows, _ = M.block(6, H, E, I, Is)
    blk = M.load(rows, H, E, k, I, Is, BF16)
    x, idx, w, sw = inputs(8, 3000, H, E, k, BF16)
    a = [cuda(x, BF16), cuda(idx), cuda(w), cuda(sw)]
    y = blk.experts(*a[:3], shared_w=a[3])
    for _ in range(3):
        assert torch.equal(blk.experts(*a[:3], shared_w=a[3]), y)
    p = torch.randperm(3000, device="cuda")
    assert torch.equal(blk.experts(a[0][p], a[1][p], a[2][p], shared_w=a[3][p]), y[p])
    assert torch.equal(blk.experts(a[0][:40], a[1][:40], a[2][:40], shared_w=a[3][:40]), y[:40])


def test_python_refusals():
    import torch
    from helexa_amd import moe as hx
    H, E, k, I, Is = 64, 4, 2, 32, 0
    rows, _ = M.block(1, H, E, I, Is)
    blk = M.load(rows, H, E, k, I, Is, BF16)
    x, idx, w, sw = inputs(1, 6, H, E, k, BF16)
    a, i, v, s = cuda(x, BF16), cuda(idx), cuda(w), cuda(sw)
    for bad in (dict(topk_idx=i.long()), dict(topk_idx=i[:5]), dict(topk_w=v.double()), dict(topk_w=v.t().contiguous()),
                dict(topk_idx=cuda(np.repeat(idx, 2, 1))[:, ::2]), dict(topk_idx=i.cpu()), dict(xs=a[:, :32]),
                dict(out=torch.empty(6, H, device="cuda")), dict(shared_w=s[:3])):
        with pytest.raises((ValueError, TypeError)):
            blk.experts(**{**dict(xs=a, topk_idx=i, topk_w=v), **bad})
    with pytest.raises(hx.HxError, match="shared expert"):
        blk.experts(a, i, v, shared_w=s)
    # a block of other experts
    cfg = hx.TextConfig(hidden_size=H, num_experts=E, num_experts_per_tok=k, moe_intermediate_size=I)
    f = lambda *sh: (hx.F32, torch.zeros(sh))
    other = hx.Qwen3_5MoeBlock.load(cfg, dict(router=f(E, H), gate=f(E, I, H), up=f(E, I, H), down=f(E, H, I)), act_dtype=hx.F32)
    with pytest.raises(hx.HxError, match="HX_MXFP4"):
        other.experts(a.float(), i, v)


@pytest.mark.parametrize("act", [BF16, F32])
@pytest.mark.parametrize("T", [1, 8, 9, 70])
def test_each_plane_of_a_record_counts(T, act):
    """Tokens whose blocks hold one large value, at a column of zero weights, next to
    values that only the record's second, third (.. fifth) plane can hold, exactly: the
    block's scale is 1, the planes step by 2^-3, 2^-6, 2^-11, 2^-16, 2^-21. The outputs then are
    within the roundings of the sums and of h and the result alone."""
    H, E, k, I = 256, 3, 1, 64
    rows, _ = M.block(31, H, E, I, 0)
    for n in ("gate", "up"):
        b = rows[n].reshape(E, I, H // 32, 17)
        b[..., 1] &= 0xF0            # column 0 of each block
        b[..., 0] = 127
    vals = {n: M.values(r) for n, r in rows.items()}
    blk = M.load(rows, H, E, k, I, 0, act)
    rng = np.random.default_rng(T)
    # plane p: whole multiples of twice its step, below half of the step of the plane before
    for step, top in ([(2.0 ** -5, 2.0 ** -4), (2.0 ** -10, 2.0 ** -7)] +
                      ([(2.0 ** -15, 2.0 ** -12), (2.0 ** -20, 2.0 ** -17)] if act == F32 else [])):
        n = int(top / step)
        x = (rng.integers(-n + 1, n, (T, H)) * step if n > 2 else rng.choice([-1, 0, 1], (T, H)) * step).astype(np.float32)
        x[:, ::32] = 4.0
        idx = rng.integers(0, E, (T, k)).astype(np.int32)
        w = np.ones((T, k), np.float32)
        xs = x.copy()
        xs[:, ::32] = 0.0            # what the products see
        y = blk.experts(cuda(x, act), cuda(idx), cuda(w)).float().cpu().numpy().astype(np.float64)
        ref, bound = M.experts_bound(xs, idx, w, vals, None, act == BF16, few(T, H, act))
        assert np.abs(ref).max() > 0
        # xs has records of its own scale: the bound of its planes is far below these values
        assert (np.abs(y - ref) <= bound).all(), (step, (np.abs(y - ref) / bound).max())
