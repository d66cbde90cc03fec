"""The MXFP4 operators as timed cases: quantising rows and reading them back, and
the experts' SwiGLU products on MXFP4 weights with a routing that the caller has.

MXFP4: blocks of 32 values along a row, 17 bytes each: the exponent byte s of a
scale 2^(s - 127) (255: NaN), then 16 bytes of 4-bit codes, value j in the low and
value j + 16 in the high half of byte j. A code is a sign bit and one of 0, 0.5, 1,
1.5, 2, 3, 4, 6. A block's scale is 2^(floor(log2 amax) - 2), its values are
rounded to the nearest code (ties to the even one, more than 6 is 6); a block that
holds a NaN or an infinity becomes NaN.

Experts: y[t] = sum over j of w[t, j] D_e(silu(G_e x[t]) * U_e x[t]) with
e = idx[t, j] (an idx outside 0 .. E - 1 is no expert), plus shared_w[t] times the
same of the shared expert.
"""
import math

import torch

own = False

CODES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
BLOCK_BYTES = 17
STD = 0.02   # of the weights, before they are quantised


# ------------------------------------------------------------------ cases
def _rows(name, kind, rows, cols):
    return dict(name=name, kind=kind, rows=rows, cols=cols)


def _experts(name, tokens, hidden=2048, experts=512, topk=10, inter=512, shared=512, act="bf16", padded=0.0, skew=0.0):
    return dict(name=name, kind="experts", tokens=tokens, hidden=hidden, experts=experts, topk=topk, inter=inter,
                shared=shared, act=act, padded=padded, skew=skew)


def listed():
    return [
        # one projection of the smallest block, quantised and read back
        _rows("quantise 128 x 256", "quantise", 128, 256),
        # in-situ quantisation of a whole projection stack: 512 experts' gate rows
        _rows("quantise gate stack", "quantise", 512 * 512, 2048),
        # a shared expert's rows read back, an odd number of blocks a row
        _rows("read back 1031 x 2080", "read_back", 1031, 2080),
        # the stack of 512 experts' down rows read back
        _rows("read back down stack", "read_back", 512 * 2048, 512),
        # one user's next token
        _experts("1 token", 1),
        # a few users' next tokens
        _experts("6 tokens", 6),
        # a batch of users' next tokens
        _experts("16 tokens", 16),
        # a padded batch of short continuations: the rows behind the last sequence choose no expert
        _experts("64 tokens, padded", 64, padded=0.2),
        # a chunk of a prompt
        _experts("512 tokens", 512),
        # a whole prompt
        _experts("2048 tokens", 2048),
        # several prompts together, some experts in demand
        _experts("8192 tokens, skewed", 8192, skew=0.8),
        # the smallest block in float32, an odd number of tokens
        _experts("33 tokens, small, f32", 33, hidden=256, experts=16, topk=4, inter=128, shared=128, act="f32",
                 padded=0.1),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    pick = rng.random()
    if pick < 0.4:
        cols = 32 * _log_int(rng, 2, 100)
        rows = _log_int(rng, 64, (1 << 29) // cols)
        return dict(kind="quantise" if pick < 0.22 else "read_back", rows=rows, cols=cols)
    most = max(work(c)["flops"] for c in listed())
    while True:
        form = rng.random()
        if form < 0.4:
            hidden, experts, topk, inter, shared = 2048, 512, 10, 512, 512
        elif form < 0.5:
            hidden, experts, topk, inter, shared = 256, 16, 4, 128, 128
        else:
            hidden, inter = 32 * rng.randint(4, 80), 32 * rng.randint(2, 40)
            experts = _log_int(rng, 4, 256)
            topk = rng.randint(1, min(experts, 12))
            shared = rng.choice((0, inter, 32 * rng.randint(1, 40)))
        c = dict(kind="experts", tokens=_log_int(rng, 1, 8192), hidden=hidden, experts=experts, topk=topk, inter=inter,
                 shared=shared, act=rng.choice(("bf16", "bf16", "bf16", "f32")),
                 padded=rng.choice((0.0, round(rng.uniform(0.0, 0.4), 3))),
                 skew=round(rng.uniform(0.05, 1.2), 3))
        if work(c)["flops"] <= most:
            return c


def work(case):
    if case["kind"] != "experts":
        n = case["rows"] * case["cols"]
        packed = n // 32 * BLOCK_BYTES
        # quantised rows are written, and read again for the values they stand for
        return {"bytes": packed + 4 * n if case["kind"] == "read_back" else 8 * n + 2 * packed, "flops": 0}
    t, h, i, s = case["tokens"], case["hidden"], case["inter"], case["shared"]
    live = t - int(t * case["padded"])
    entries = live * case["topk"]
    # experts that some token chooses, by the chances that prepare() draws with
    p = [(r + 1.0) ** -case["skew"] for r in range(case["experts"])]
    used = sum(1.0 - (1.0 - v / sum(p)) ** entries for v in p)
    matrix = h * i // 32 * BLOCK_BYTES * 3
    acts = t * h * (4 if case["act"] == "f32" else 2) * 2
    return {"bytes": int(used * matrix + (h * s // 32 * BLOCK_BYTES * 3 if s else 0) + acts + t * case["topk"] * 8 + 4 * t),
            "flops": 6 * h * (entries * i + t * s)}


# ------------------------------------------------------------------ inputs
def _seeded(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _weights(g, rows, cols, count=1):
    """float32 rows of a checkpoint: normal values, a few rows of another size"""
    w = torch.randn((count * rows, cols), generator=g, device="cuda").mul_(STD)
    w *= 1.0 + (torch.rand((count * rows, 1), generator=g, device="cuda") < 0.02) * 7.0
    return w


def _packed_weights(g, count, rows, cols):
    """[count, rows, row bytes] of a checkpoint in MXFP4, made 64 matrices at a time"""
    return torch.cat([_quantise(_weights(g, rows, cols, min(64, count - c)))
                      for c in range(0, count, 64)]).view(count, rows, -1)


def _inputs(case, seed):
    g = _seeded(seed)
    if case["kind"] == "quantise":
        return dict(w=_weights(g, case["rows"], case["cols"]))
    if case["kind"] == "read_back":
        return dict(q=_quantise(_weights(g, case["rows"], case["cols"])))
    t, h, e, k, i, s = (case[n] for n in ("tokens", "hidden", "experts", "topk", "inter", "shared"))
    d = dict(gate=_packed_weights(g, e, i, h), up=_packed_weights(g, e, i, h), down=_packed_weights(g, e, h, i))
    if s:
        d.update(sgate=_packed_weights(g, 1, s, h)[0], sup=_packed_weights(g, 1, s, h)[0],
                 sdown=_packed_weights(g, 1, h, s)[0])
    x = torch.randn((t, h), generator=g, device="cuda")
    d["x"] = x if case["act"] == "f32" else x.to(torch.bfloat16)
    # k distinct experts a token, expert of rank r with a chance of (r + 1)^-skew
    order = torch.randperm(e, generator=g, device="cuda")
    chance = torch.empty(e, device="cuda")
    chance[order] = -case["skew"] * torch.log(torch.arange(1, e + 1, device="cuda").float())
    noise = -torch.log(-torch.log(torch.rand((t, e), generator=g, device="cuda").clamp(1e-7, 1 - 1e-7)))
    score, idx = torch.topk(chance + noise, k, dim=1)
    w = torch.softmax(score, dim=1)
    live = t - int(t * case["padded"])
    idx[live:] = -1
    w[live:] = 0.0
    d["idx"], d["w"] = idx.to(torch.int32).contiguous(), w.contiguous()
    d["shared_w"] = torch.sigmoid(torch.randn(t, generator=g, device="cuda")) if s else None
    return d


def prepare(case, seed):
    st = _inputs(case, seed)
    st["kind"] = case["kind"]
    st["cols"] = case.get("cols")
    if own and case["kind"] == "experts":
        import helexa_amd as hx
        cfg = hx.TextConfig(hidden_size=case["hidden"], num_experts=case["experts"], num_experts_per_tok=case["topk"],
                            moe_intermediate_size=case["inter"], shared_expert_intermediate_size=case["shared"])
        weights = {"router": (hx.BF16, torch.zeros((case["experts"], case["hidden"]), dtype=torch.bfloat16, device="cuda"))}
        if case["shared"]:
            weights["seg"] = (hx.BF16, torch.zeros((1, case["hidden"]), dtype=torch.bfloat16, device="cuda"))
        for name in ("gate", "up", "down", "sgate", "sup", "sdown"):
            if name in st:
                weights[name] = (hx.MXFP4, st.pop(name))
        torch.cuda.synchronize()
        st["block"] = hx.Qwen3_5MoeBlock.load(cfg, weights, act_dtype=hx.F32 if case["act"] == "f32" else hx.BF16)
        st["workspace"] = torch.empty(st["block"].workspace_size(case["tokens"]), dtype=torch.uint8, device="cuda")
    return st


# ------------------------------------------------------------------ plain forms
def _quantise(w):
    """float32 [rows, cols] -> uint8 [rows, cols / 32 * 17]. Scaling by a power of two is exact in float32."""
    v = w.view(-1, 32)
    amax = v.abs().amax(dim=1)
    fine = torch.isfinite(amax)
    exponent = torch.frexp(torch.where(fine, amax, 0.0).double())[1] - 3   # amax = m 2^e, m in [0.5, 1)
    exponent = torch.where(amax > 0, exponent, -127).clamp(-127, 127)
    a = v * torch.exp2(-exponent.double()).float()[:, None]
    neg = torch.signbit(a)
    a = a.abs()
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)
            + neg * torch.tensor(8, dtype=torch.uint8, device=w.device))
    code = torch.where(fine[:, None], code, 0)
    scale = torch.where(fine, exponent + 127, 255).to(torch.uint8)
    blocks = torch.cat([scale[:, None], code[:, :16] | (code[:, 16:] << 4)], dim=1)
    return blocks.view(w.shape[0], -1)


def _values(q):
    """uint8 [..., row bytes] -> float32 [..., cols]"""
    scales = torch.exp2(torch.arange(256, device=q.device).double() - 127).float()
    scales[255] = math.nan
    codes = torch.tensor(CODES + tuple(-c for c in CODES), device=q.device)
    b = q.view(*q.shape[:-1], -1, BLOCK_BYTES)
    packed = b[..., 1:].int()
    v = codes[torch.cat([packed & 15, packed >> 4], dim=-1)] * scales[b[..., :1].int()]
    return v.view(*q.shape[:-1], -1)


def _swiglu(x, gate, up, down):
    """x [n, m, hidden] through n experts' packed matrices"""
    g = torch.bmm(x, _values(gate).transpose(1, 2))
    u = torch.bmm(x, _values(up).transpose(1, 2))
    return torch.bmm(g * torch.sigmoid(g) * u, _values(down).transpose(1, 2))


def _experts_plain(st):
    x, idx, w = st["x"].float(), st["idx"].long(), st["w"]
    (tokens, hidden), k, experts = x.shape, idx.shape[1], st["gate"].shape[0]
    idx = torch.where((idx >= 0) & (idx < experts), idx, experts).view(-1)
    order = torch.argsort(idx, stable=True)
    counts = torch.bincount(idx, minlength=experts + 1)[:experts]
    starts = torch.cumsum(counts, 0) - counts
    used = torch.nonzero(counts).view(-1)
    used = used[torch.argsort(counts[used])]   # experts of like counts together
    rows = torch.zeros((tokens * k + 1, hidden), device=x.device)   # the last row takes what is behind a count
    for some in used.split(48):
        m = int(counts[some].max())
        at = starts[some][:, None] + torch.arange(m, device=x.device)
        has = at < (starts + counts)[some][:, None]
        entry = torch.where(has, order[at.clamp(max=tokens * k - 1)], tokens * k)
        xs = x[(entry // k).clamp(max=tokens - 1)]
        rows[entry.view(-1)] = _swiglu(xs, st["gate"][some], st["up"][some], st["down"][some]).view(-1, hidden)
    chosen = (idx < experts).view(tokens, k, 1)
    y = torch.where(chosen, rows[:-1].view(tokens, k, hidden) * w[:, :, None], 0.0).sum(dim=1)
    if st["shared_w"] is not None:
        y += st["shared_w"][:, None] * _swiglu(x[None], st["sgate"][None], st["sup"][None], st["sdown"][None])[0]
    return y.to(st["x"].dtype)


# ------------------------------------------------------------------ one pass
def run(st):
    if own:
        import helexa_amd as hx
        if st["kind"] == "quantise":
            return hx.dequantize(hx.MXFP4, hx.quantize(hx.MXFP4, st["w"]), st["w"].shape[1])
        if st["kind"] == "read_back":
            return hx.dequantize(hx.MXFP4, st["q"], st["cols"])
        return st["block"].experts(st["x"], st["idx"], st["w"], shared_w=st["shared_w"], workspace=st["workspace"])
    if st["kind"] == "quantise":
        return _values(_quantise(st["w"]))
    if st["kind"] == "read_back":
        return _values(st["q"])
    return _experts_plain(st)


# ------------------------------------------------------------------ exact values
def _decoded(q, cols):
    """packed rows -> float64 values: sign, exponent and mantissa bits of each code by arithmetic"""
    b = q.reshape(-1, cols // 32, BLOCK_BYTES)
    c = torch.stack([b[:, :, 1:] % 16, b[:, :, 1:] // 16], dim=2).reshape(b.shape[0], cols // 32, 32).double()
    sign = 1.0 - 2.0 * (c >= 8)
    c = c % 8
    e, m = torch.floor(c / 2), c % 2
    v = sign * torch.where(e > 0, (1.0 + m / 2) * torch.pow(2.0, e - 1), m / 2)
    s = b[:, :, :1].double()
    return (v * torch.where(s < 255, torch.pow(2.0, s - 127), math.nan)).reshape(-1, cols)


def _nearest(w):
    """float64 values on each block's grid: spacing 2^(e - 1) in a value's own binade, half of the smallest below 1"""
    out = torch.empty(w.shape, dtype=torch.float64, device=w.device)
    for r in range(0, w.shape[0], 1 << 15):
        v = w[r:r + (1 << 15)].double().reshape(-1, 32)
        amax = v.abs().amax(dim=1, keepdim=True)
        x = torch.pow(2.0, torch.floor(torch.log2(amax.clamp(min=2.0 ** -149))) - 2).clamp(min=2.0 ** -127)
        a = v / x
        spacing = torch.where(a.abs() >= 4, 2.0, torch.where(a.abs() >= 2, 1.0, 0.5))
        out[r:r + (1 << 15)] = (torch.clamp(torch.round(a / spacing) * spacing, -6.0, 6.0) * x).reshape(-1, w.shape[1])
    return out


def exact(case, seed):
    d = _inputs(case, seed)
    if case["kind"] == "quantise":
        return _nearest(d["w"])
    if case["kind"] == "read_back":
        return torch.cat([_decoded(p, case["cols"]) for p in d["q"].split(1 << 15)])
    h, i = case["hidden"], case["inter"]
    x = d["x"].double()
    y = torch.zeros_like(x)

    def add(tok, weight, gate, up, down, inter):
        xs = x[tok]
        g, u = xs @ _decoded(gate, h).t(), xs @ _decoded(up, h).t()
        y.index_add_(0, tok, weight[:, None].double() * ((g / (1.0 + torch.exp(-g)) * u) @ _decoded(down, inter).t()))

    for e in torch.unique(d["idx"]).tolist():
        if 0 <= e < case["experts"]:
            tok, j = torch.nonzero(d["idx"] == e, as_tuple=True)
            add(tok, d["w"][tok, j], d["gate"][e], d["up"][e], d["down"][e], i)
    if case["shared"]:
        add(torch.arange(case["tokens"], device="cuda"), d["shared_w"], d["sgate"], d["sup"], d["sdown"], case["shared"])
    return y
