"""The block's calls on another stream than the current one, which is busy: tokens that are no
contiguous tensor are copied on the stream that reads them, and results lie in no
memory that the current stream has still to write."""
import pytest

pytestmark = pytest.mark.gpu


def make():
    import helexa_amd as hx
    from helexa_amd import synth
    cfg = hx.TextConfig(hidden_size=256, num_experts=16, num_experts_per_tok=4, moe_intermediate_size=128,
                        shared_expert_intermediate_size=128, norm_topk_prob=True)
    return hx.Qwen3_5MoeBlock.load(cfg, synth.make_weights(cfg, synth.FMT_Q8_0, 9), act_dtype=hx.BF16)


def calls(b):
    import helexa_amd as hx
    return {"forward": lambda x, **kw: [b.forward(x, **kw)],
            "route": lambda x, **kw: list(b.route(x, **kw).values()),
            "router_logits": lambda x, **kw: [b.router_logits(x, **kw)],
            "quantize_activations": lambda x, **kw: list(hx.quantize_activations(hx.Q8_0, x, **kw))}


@pytest.mark.parametrize("name", ["forward", "route", "router_logits", "quantize_activations"])
@pytest.mark.parametrize("T", [1, 40])
def test_calls_on_another_stream_than_a_busy_current_one(name, T):
    import torch
    b = make()
    call = calls(b)[name]
    x = torch.randn((T, 256), device="cuda").to(torch.bfloat16)
    wide = torch.zeros((T, 512), dtype=x.dtype, device="cuda")
    wide[:, ::2] = x
    want = call(x)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    torch.cuda._sleep(200_000_000)
    late = [torch.full_like(w, 5) for w in want for _ in range(4)]
    late += [torch.full_like(x, 5) for _ in range(4)]
    del late
    got = call(wide[:, ::2], stream=s)
    s.synchronize()
    assert not torch.cuda.current_stream().query(), "the current stream was done too early to show anything"
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert torch.equal(g, w)


@pytest.mark.parametrize("name", ["forward", "forward_noalloc", "decoder_mlp_"])
def test_tokens_dropped_while_another_stream_uses_them(name):
    import torch
    b = make()
    x = torch.randn((40, 256), device="cuda").to(torch.bfloat16)
    nw = torch.zeros(256, device="cuda")
    out = torch.empty_like(x)
    call = {"forward": lambda t, **kw: b.forward(t, out=out, **kw),
            "forward_noalloc": lambda t, **kw: b.forward_noalloc(t, out, **kw),
            "decoder_mlp_": lambda t, **kw: out.copy_(b.decoder_mlp_(t, nw, 1e-6, **kw))}[name]
    want = call(x.clone()).clone()
    s = torch.cuda.Stream()
    t = x.clone()
    torch.cuda.synchronize()
    place = t.data_ptr()
    with torch.cuda.stream(s):
        torch.cuda._sleep(200_000_000)
        call(t, stream=s)
    del t
    again = [torch.zeros_like(x) for _ in range(2)]
    assert not s.query(), "the stream was done too early to show anything"
    assert place not in [a.data_ptr() for a in again]
    s.synchronize()
    assert torch.equal(out, want)
