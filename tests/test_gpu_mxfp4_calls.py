"""Calls of the MXFP4 experts whose sizes or arguments meet an edge of a kernel or of an
entry point: rows that fill only some lanes of the combine, workspaces off 16 bytes,
tensors dropped while another stream uses them, the border between the few-token kernels
and the others, and their instance for many features in f32, rows and results on another
stream."""
import numpy as np
import pytest

import mxfp4 as M
from test_gpu_mxfp4_experts import BF16, F32, cuda, inputs

pytestmark = pytest.mark.gpu


def few(T, H, act):
    """whether the few-token kernels take the call: at most 8 tokens, whose records with one of
    zeros, and whose sums (8 waves, gate and up, 32 features, a column a plane and token; then
    h), fit 60 KiB"""
    planes, rec = (3, 80) if act == BF16 else (5, 128)
    records, sums = (T * ((H + 127) // 128 * 4) + 1) * rec, (8 * 2 * 32 * planes * T + 8 * 33 * T) * 4
    return T <= 8 and max(records, sums) <= 60 * 1024


def check(y, x, idx, w, vals, sw, act):
    ref, bound = M.experts_bound(x, idx, w, vals, sw, act == BF16, few(*x.shape, act))
    off = np.abs(y.float().cpu().numpy().astype(np.float64) - ref) / bound
    print(f"[err] worst {off.max():.3f} of the bound", flush=True)
    assert off.max() <= 1.0, np.unravel_index(off.argmax(), off.shape)


@pytest.mark.parametrize("act", [BF16, F32])
@pytest.mark.parametrize("H,k,Is", [(32, 64, 32), (64, 10, 0), (64, 33, 64), (544, 64, 32), (1056, 24, 0)])
def test_more_entries_than_lanes_with_outputs(H, k, Is, act):
    """the combine's lanes hold a token's entries also where they hold none of its outputs:
    rows of 32 and 64, and rows whose last segment is 32 wide"""
    E, I = 80, 32
    rows, vals = M.block(H + k, H, E, I, Is)
    blk = M.load(rows, H, E, k, I, Is, act)
    for T in (2, 5, 9, 40):
        print("case", H, k, act, T, flush=True)
        x, idx, w, sw = inputs(T, T, H, E, k, act)
        check(blk.experts(cuda(x, act), cuda(idx), cuda(w), shared_w=cuda(sw) if Is else None), x, idx, w, vals,
              sw if Is else None, act)
    blk.close()


@pytest.mark.parametrize("T", [1, 6, 9, 70])
def test_a_workspace_off_16_bytes_is_refused_before_any_launch(T):
    """hx_moe_forward, hx_moe_decoder_mlp and hx_moe_experts: the error, and workspace, y and
    the stream of tokens as they were"""
    import torch
    from helexa_amd import moe as hx
    H, E, k, I, Is = 256, 16, 4, 128, 128
    rows, _ = M.block(3, H, E, I, Is)
    blk = M.load(rows, H, E, k, I, Is, BF16)
    x, idx, w, sw = inputs(T, T, H, E, k, BF16)
    xt, it, wt, st = cuda(x, BF16), cuda(idx), cuda(w), cuda(sw)
    nw = torch.zeros(H, device="cuda")
    n = blk.workspace_size(T)
    ws = torch.full((n + 16,), 7, dtype=torch.uint8, device="cuda")
    y = torch.full_like(xt, 3.0)
    was = xt.clone()
    s = torch.cuda.current_stream().cuda_stream
    for off in (4, 8):
        p = ws.data_ptr() + off
        assert hx.lib().hx_moe_forward(blk.handle, xt.data_ptr(), T, y.data_ptr(), p, n, None, s) == 1
        assert "16 bytes" in hx.last_error()
        assert hx.lib().hx_moe_decoder_mlp(blk.handle, xt.data_ptr(), T, nw.data_ptr(), 1e-6, p, n, s) == 1
        assert hx.lib().hx_moe_experts(blk.handle, xt.data_ptr(), T, it.data_ptr(), wt.data_ptr(), st.data_ptr(),
                                       y.data_ptr(), p, n, s) == 1
    torch.cuda.synchronize()
    assert (ws == 7).all() and (y == 3).all() and torch.equal(xt, was)
    # 16 bytes are enough
    want = blk.forward(xt)
    assert torch.equal(blk.forward(xt, workspace=ws[16:]), want)


@pytest.mark.parametrize("T", [1, 6, 30])
def test_tensors_dropped_while_another_stream_uses_them(T):
    """a call on a busy stream whose tensors the caller drops at once: their memory goes to
    nobody else before that stream has read and written it"""
    import torch
    H, E, k, I, Is = 256, 16, 4, 128, 128
    rows, _ = M.block(3, H, E, I, Is)
    blk = M.load(rows, H, E, k, I, Is, BF16)
    x, idx, w, sw = inputs(T, T, H, E, k, BF16)
    ref = blk.experts(cuda(x, BF16), cuda(idx), cuda(w), shared_w=cuda(sw))
    n = blk.workspace_size(T)
    # sizes of their own, so that the memory of each comes back for a tensor of its size
    torch.cuda.empty_cache()
    s = torch.cuda.Stream()
    ts = [cuda(x, BF16), cuda(idx), cuda(w), cuda(sw), torch.empty(n, dtype=torch.uint8, device="cuda")]
    torch.cuda.synchronize()
    shapes = [(t.shape, t.dtype) for t in ts]
    places = {t.data_ptr() for t in ts}
    with torch.cuda.stream(s):
        torch.cuda._sleep(200_000_000)
    y = blk.experts(*ts[:3], shared_w=ts[3], workspace=ts[4], stream=s)
    del ts
    again = [torch.zeros(sh, dtype=dt, device="cuda") for sh, dt in shapes for _ in range(2)]
    assert not s.query(), "the stream was done too early to show anything"
    assert not places & {t.data_ptr() for t in again}
    s.synchronize()
    assert torch.equal(y, ref)


@pytest.mark.parametrize("act,H,most", [(BF16, 64, 8), (F32, 64, 5), (BF16, 2944, 8), (BF16, 2976, 7), (F32, 2944, 5),
                                        (F32, 2976, 4), (BF16, 4864, 5), (BF16, 4896, 4)])
def test_which_calls_take_the_few_token_kernels(act, H, most):
    """up to `most` tokens no records are made ahead of gate/up (the x_f16 slot), from there on they are"""
    assert few(most, H, act) and not few(most + 1, H, act)
    E, k, I = 4, 2, 32
    rows, vals = M.block(1, H, E, I, 0)
    blk = M.load(rows, H, E, k, I, 0, act)
    for T in (most, most + 1):
        x, idx, w, _ = inputs(T, T, H, E, k, act)
        blk.experts(cuda(x, act), cuda(idx), cuda(w))
        blk.timing_begin(1)
        y = blk.experts(cuda(x, act), cuda(idx), cuda(w))
        slots = {n for n, (ms, c) in blk.timing_end().items() if c}
        assert ("x_f16" in slots) == (T > most), (T, slots)
        check(y, x, idx, w, vals, None, act)
    blk.close()


@pytest.mark.parametrize("T,H,I,Is", [(5, 256, 736, 768), (5, 96, 800, 0), (4, 1024, 928, 928), (5, 2048, 736, 64)])
def test_many_features_of_few_f32_tokens(T, H, I, Is):
    """at least 1200 groups of 32 features in all: K by one wave, with five planes"""
    E, k = 64, 10
    groups = (T * k + (Is > 0)) * ((max(I, Is) + 127) // 128 * 4)
    assert groups >= 1200
    rows, vals = M.block(H, H, E, I, Is, std=0.02)
    blk = M.load(rows, H, E, k, I, Is, F32)
    x, idx, w, sw = inputs(T, T, H, E, k, F32)
    # every token its own experts, so that no two entries share a slot
    idx[:] = np.random.default_rng(H).permutation(E)[:T * k].reshape(T, k)
    check(blk.experts(cuda(x), cuda(idx), cuda(w), shared_w=cuda(sw) if Is else None), x, idx, w, vals,
          sw if Is else None, F32)
    blk.close()


@pytest.mark.parametrize("fn", ["quantize", "dequantize"])
def test_rows_on_another_stream(fn):
    """a call on another stream: rows that are no contiguous tensor are copied on that stream, not
    on the busy current one, and memory that the caller drops while the stream is busy
    goes to nobody else"""
    import torch
    import helexa_amd as hx
    rows, cols = 300, 96
    g = torch.Generator(device="cuda").manual_seed(1)
    w = torch.randn((rows, cols), generator=g, device="cuda")
    q = hx.quantize(hx.MXFP4, w)
    if fn == "quantize":
        call, src, want = lambda t, **kw: hx.quantize(hx.MXFP4, t, **kw), w, q
    else:
        call, src, want = lambda t, **kw: hx.dequantize(hx.MXFP4, t, cols, **kw), q, hx.dequantize(hx.MXFP4, q, cols)
    s = torch.cuda.Stream()
    turned = src.t().contiguous()   # its .t() is src again, not contiguous
    torch.cuda.synchronize()
    torch.cuda._sleep(200_000_000)
    got = call(turned.t(), stream=s)
    s.synchronize()
    there = torch.empty_like(want)
    with torch.cuda.stream(s):
        there.copy_(got)
    s.synchronize()
    assert not torch.cuda.current_stream().query(), "the current stream was done too early to show anything"
    torch.cuda.synchronize()
    assert torch.equal(there, want)
    x = src.clone()
    torch.cuda.synchronize()
    place, like = x.data_ptr(), (x.shape, x.dtype)
    with torch.cuda.stream(s):
        torch.cuda._sleep(200_000_000)
    got = call(x, stream=s)
    del x
    again = [torch.zeros(like[0], dtype=like[1], device="cuda") for _ in range(2)]
    assert not s.query(), "the stream was done too early to show anything"
    assert place not in [t.data_ptr() for t in again]
    s.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("fn", ["quantize", "dequantize", "experts"])
def test_a_result_on_another_stream_keeps_off_what_the_current_one_has_to_do(fn):
    """memory of the result's size that the current stream frees but has still to write: the call
    on another stream does not take it"""
    import torch
    import helexa_amd as hx
    rows, cols = 300, 96
    w = torch.randn((rows, cols), device="cuda")
    q = hx.quantize(hx.MXFP4, w)
    if fn == "quantize":
        call = lambda **kw: hx.quantize(hx.MXFP4, w, **kw)
    elif fn == "dequantize":
        call = lambda **kw: hx.dequantize(hx.MXFP4, q, cols, **kw)
    else:
        H, E, k, I, Is = 256, 16, 4, 128, 0
        blk = M.load(M.block(3, H, E, I, Is)[0], H, E, k, I, Is, BF16)
        x, idx, wt, _ = (cuda(a, BF16 if i == 0 else None) for i, a in enumerate(inputs(1, 90, H, E, k, BF16)))
        ws = torch.empty(blk.workspace_size(90), dtype=torch.uint8, device="cuda")
        call = lambda **kw: blk.experts(x, idx, wt, workspace=ws, **kw)
    want = call()
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    torch.cuda._sleep(200_000_000)
    late = [torch.full_like(want, 5) for _ in range(4)]
    del late
    got = call(stream=s)
    s.synchronize()
    assert not torch.cuda.current_stream().query(), "the current stream was done too early to show anything"
    torch.cuda.synchronize()
    assert torch.equal(got, want)
