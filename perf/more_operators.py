"""The operators on E4M3 weights and the router's balance loss as timed cases.

E4M3 blocks: 8-bit floats (4 exponent, 3 mantissa bits, largest 448) with a float32
scale for each block of 128 x 128 of a weight matrix, or of 128 columns of a row of
activations (shorter blocks at the edges). A block's scale is max(max|x| / 448, 2^-126),
a code the E4M3 value nearest to x / scale, ties to the even one; a block that holds a
NaN or an infinity has the scale NaN and codes of 0.

Linear layer: y = q(x) W^T with q the quantisation of x's rows. Experts: y[t] = sum over
j of w[t, j] D_e(q(silu(G_e q(x[t])) * U_e q(x[t]))) with e = idx[t, j] (an idx outside
0 .. E - 1 is no expert), plus shared_w[t] times the same of the shared expert.

Balance loss of a router: L = coef E sum_e f_e P_e over the live tokens (those with an
index in 0 .. E - 1), f_e = k c_e / sum c of the experts' entries c, P_e the mean of
the tokens' softmax probabilities; its gradient by the logits takes the counts as
given.
"""
import math

import torch
import torch.nn.functional as F

own = False

STD = 0.02       # of the weights, before they are quantised
COEF = 0.001     # of the balance loss


# ------------------------------------------------------------------ cases
def _quant(name, rows, cols, block_rows, act):
    return dict(name=name, kind="quantise", rows=rows, cols=cols, block_rows=block_rows, act=act)


def _linear(name, rows, cols, features, act="bf16"):
    return dict(name=name, kind="linear", rows=rows, cols=cols, features=features, act=act)


def _experts(name, tokens, hidden=2048, experts=512, topk=10, inter=512, shared=512, padded=0.0, skew=0.0):
    return dict(name=name, kind="experts", tokens=tokens, hidden=hidden, experts=experts, topk=topk, inter=inter,
                shared=shared, padded=padded, skew=skew)


def _balance(name, tokens, experts=512, topk=10, act="f32", padded=0.0, skew=0.5):
    return dict(name=name, kind="balance", tokens=tokens, experts=experts, topk=topk, act=act, padded=padded, skew=skew)


def listed():
    return [
        # a few tokens' rows on their way into a product, the last block of a row a short one
        _quant("quantise 17 rows", 17, 2080, 1, "bf16"),
        # in-situ quantisation of a whole projection stack: 512 experts' gate rows
        _quant("quantise gate stack", 512 * 512, 2048, 128, "f32"),
        # one user's next token through a projection
        _linear("linear, 1 row", 1, 2048, 4096),
        # a batch of sequences in float32, no size a whole block
        _linear("linear, 33 rows, odd, f32", 33, 2080, 1031, "f32"),
        # a chunk of a prompt
        _linear("linear, 512 rows", 512, 2048, 4096),
        # several prompts together through a wide projection
        _linear("linear, 8192 rows", 8192, 4096, 8192),
        # one user's next token through the experts
        _experts("experts, 1 token", 1),
        # a padded batch of short continuations: the rows behind the last sequence choose no expert
        _experts("experts, 64 tokens, padded", 64, padded=0.2),
        # several prompts together, some experts in demand
        _experts("experts, 8192 tokens, skewed", 8192, skew=0.8),
        # a padded training batch of the smallest router
        _balance("balance, 33 tokens", 33, experts=16, topk=4, padded=0.1),
        # one layer of a training batch
        _balance("balance, 8192 tokens", 8192),
        # all 48 layers of a training batch, logits in bfloat16, some experts in demand
        _balance("balance, 48 layers", 48 * 4096, act="bf16", skew=1.0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 500)


def draw(rng):
    pick = rng.random()
    while True:
        act = rng.choice(("bf16", "bf16", "f32"))
        if pick < 0.2:
            cols = _log_int(rng, 100, 8192)
            rows = _log_int(rng, 1, (1 << 28) // cols)
            c = dict(kind="quantise", rows=rows, cols=cols, block_rows=rng.choice((1, 128)), act=act)
        elif pick < 0.5:
            c = dict(kind="linear", rows=_log_int(rng, 1, 16384), cols=_log_int(rng, 100, 8192),
                     features=_log_int(rng, 100, 12288), act=act)
            if rng.random() < 0.7:
                c["cols"], c["features"] = (c["cols"] + 127) // 128 * 128, (c["features"] + 63) // 64 * 64
        elif pick < 0.75:
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
            c = dict(kind="experts", tokens=_log_int(rng, 1, 8192), hidden=hidden, experts=experts, topk=topk,
                     inter=inter, shared=shared, padded=rng.choice((0.0, round(rng.uniform(0.0, 0.4), 3))),
                     skew=round(rng.uniform(0.05, 1.2), 3))
        else:
            experts = rng.choice((512, 128, _log_int(rng, 4, 1024)))
            c = dict(kind="balance", tokens=_log_int(rng, 1, 1 << 17), experts=experts,
                     topk=rng.randint(1, min(experts, 12)), act=act,
                     padded=rng.choice((0.0, round(rng.uniform(0.0, 0.4), 3))), skew=round(rng.uniform(0.05, 1.2), 3))
        most = max(_cost(d) for d in listed() if d["kind"] == c["kind"])
        if _cost(c) <= most:
            return c


def _blocks(n):
    return (n + 127) // 128


def work(case):
    size = 4 if case.get("act") == "f32" else 2
    if case["kind"] == "quantise":
        n, br = case["rows"] * case["cols"], case["block_rows"]
        return {"bytes": n * (size + 1) + 4 * ((case["rows"] + br - 1) // br) * _blocks(case["cols"]), "flops": 0}
    if case["kind"] == "linear":
        m, k, n = case["rows"], case["cols"], case["features"]
        return {"bytes": size * m * (k + n) + n * k + 4 * _blocks(n) * _blocks(k), "flops": 2 * m * n * k}
    t = case["tokens"]
    if case["kind"] == "balance":
        e = case["experts"]
        return {"bytes": 2 * size * t * e + 4 * t * case["topk"] + 8 * e, "flops": 10 * t * e}
    h, i, s = case["hidden"], case["inter"], case["shared"]
    live = t - int(t * case["padded"])
    entries = live * case["topk"]
    # experts that some token chooses, by the chances that prepare() draws with
    p = [(r + 1.0) ** -case["skew"] for r in range(case["experts"])]
    used = sum(1.0 - (1.0 - v / sum(p)) ** entries for v in p)
    matrices = 3 * h * i + 12 * _blocks(h) * _blocks(i)
    shared = 3 * h * s + 12 * _blocks(h) * _blocks(s) if s else 0
    return {"bytes": int(used * matrices + shared + 4 * t * h + t * case["topk"] * 8 + 4 * t),
            "flops": 6 * h * (entries * i + t * s)}


# ------------------------------------------------------------------ inputs
def _seeded(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _rows(g, rows, cols, act):
    """activations: normal values, a few columns much larger, as a trained model has them"""
    x = torch.randn((rows, cols), generator=g, device="cuda")
    x *= 1.0 + (torch.rand(cols, generator=g, device="cuda") < 0.01) * 15.0
    return x if act == "f32" else x.to(torch.bfloat16)


def _float_weights(g, rows, cols):
    """float32 rows of a checkpoint: normal values, a few rows of another size"""
    w = torch.randn((rows, cols), generator=g, device="cuda").mul_(STD)
    w *= 1.0 + (torch.rand((rows, 1), generator=g, device="cuda") < 0.02) * 7.0
    return w


def _weights(g, rows, cols):
    return _quantise(_float_weights(g, rows, cols), 128)


def _stack(g, count, rows, cols):
    """codes [count, rows, cols] and scales [count, ...] of a checkpoint's experts"""
    made = [_weights(g, rows, cols) for _ in range(count)]
    return torch.stack([c for c, _ in made]), torch.stack([s for _, s in made])


def _chosen(g, chance, tokens, topk, skew, padded):
    """k distinct experts a token, an expert of rank r with a chance of (r + 1)^-skew; [T, E] scores, indices, live tokens"""
    experts = chance.shape[0]
    order = torch.randperm(experts, generator=g, device="cuda")
    chance[order] = -skew * torch.log(torch.arange(1, experts + 1, device="cuda").float())
    noise = -torch.log(-torch.log(torch.rand((tokens, experts), generator=g, device="cuda").clamp(1e-7, 1 - 1e-7)))
    score = chance + noise
    top, idx = torch.topk(score, topk, dim=1)
    live = tokens - int(tokens * padded)
    idx[live:] = -1
    return score, top, idx.to(torch.int32).contiguous(), live


def _inputs(case, seed):
    g = _seeded(seed)
    if case["kind"] == "quantise":
        if case["block_rows"] == 1:
            return dict(x=_rows(g, case["rows"], case["cols"], case["act"]))
        w = _float_weights(g, case["rows"], case["cols"])
        return dict(x=w if case["act"] == "f32" else w.to(torch.bfloat16))
    if case["kind"] == "linear":
        codes, scales = _weights(g, case["features"], case["cols"])
        return dict(codes=codes, scales=scales, x=_rows(g, case["rows"], case["cols"], case["act"]))
    t, e, k = case["tokens"], case["experts"], case["topk"]
    chance = torch.empty(e, device="cuda")
    if case["kind"] == "balance":
        score, _, idx, live = _chosen(g, chance, t, k, case["skew"], case["padded"])
        logits = score if case["act"] == "f32" else score.to(torch.bfloat16)
        logits[live:] = math.nan   # what lies behind the last sequence
        return dict(logits=logits, idx=idx)
    h, i, s = case["hidden"], case["inter"], case["shared"]
    d = {}
    for name, rows, cols in (("gate", i, h), ("up", i, h), ("down", h, i)):
        d[name], d[name + "_scales"] = _stack(g, e, rows, cols)
    if s:
        for name, rows, cols in (("sgate", s, h), ("sup", s, h), ("sdown", h, s)):
            d[name], d[name + "_scales"] = _weights(g, rows, cols)
    d["x"] = _rows(g, t, h, "bf16")
    _, top, d["idx"], live = _chosen(g, chance, t, k, case["skew"], case["padded"])
    d["w"] = torch.softmax(top, dim=1)
    d["w"][live:] = 0.0
    d["shared_w"] = torch.sigmoid(torch.randn(t, generator=g, device="cuda")) if s else None
    return d


def prepare(case, seed):
    st = _inputs(case, seed)
    st["case"] = case
    if not own:
        return st
    import helexa_amd as hx
    torch.cuda.synchronize()
    if case["kind"] == "linear":
        st["layer"] = hx.F8Linear.load(st.pop("codes"), st.pop("scales"))
        st["workspace"] = torch.empty(st["layer"].workspace_size(case["rows"]), dtype=torch.uint8, device="cuda")
    elif case["kind"] == "balance":
        st["workspace"] = torch.empty(hx.balance_workspace_size(case["tokens"], case["experts"]), dtype=torch.uint8,
                                      device="cuda")
    elif case["kind"] == "experts":
        cfg = hx.TextConfig(hidden_size=case["hidden"], num_experts=case["experts"], num_experts_per_tok=case["topk"],
                            moe_intermediate_size=case["inter"], shared_expert_intermediate_size=case["shared"])
        weights = {"router": (hx.BF16, torch.zeros((case["experts"], case["hidden"]), dtype=torch.bfloat16, device="cuda"))}
        if case["shared"]:
            weights["seg"] = (hx.BF16, torch.zeros((1, case["hidden"]), dtype=torch.bfloat16, device="cuda"))
        for name in ("gate", "up", "down", "sgate", "sup", "sdown"):
            if name in st:
                weights[name] = (hx.F8_E4M3, st.pop(name), st.pop(name + "_scales"))
        torch.cuda.synchronize()
        st["block"] = hx.Qwen3_5MoeBlock.load(cfg, weights, act_dtype=hx.BF16)
        st["workspace"] = torch.empty(st["block"].workspace_size(case["tokens"]), dtype=torch.uint8, device="cuda")
    return st


# ------------------------------------------------------------------ plain forms
def _blocked(x, block_rows):
    """[rows, cols] -> [row blocks, block_rows, column blocks, 128], zeros behind the edges"""
    rows, cols = x.shape
    x = F.pad(x, (0, -cols % 128, 0, -rows % block_rows))
    return x.view(-1, block_rows, x.shape[1] // 128, 128)


def _quantise(x, block_rows):
    """codes in float8_e4m3fn [rows, cols], float32 scales [row blocks, column blocks]"""
    b = _blocked(x.float(), block_rows)
    amax = b.abs().amax(dim=(1, 3))
    fine = torch.isfinite(amax)
    # amax / 448, the float32 nearest to it
    scales = torch.where(fine, (amax.double() / 448.0).float().clamp(min=2.0 ** -126), math.nan)
    q = b.double() / scales.double()[:, None, :, None]   # in 64 bits: values next to the border of two codes
    q = torch.where(fine[:, None, :, None], q, 0.0)
    step = torch.exp2((torch.frexp(q)[1] - 1).clamp(min=-6).double() - 3.0)
    codes = (torch.round(q / step) * step).float().to(torch.float8_e4m3fn)
    return codes.reshape(-1, b.shape[2] * 128)[:x.shape[0], :x.shape[1]].contiguous(), scales


def _values(codes, scales, block_rows):
    """float32 values of codes [..., rows, cols] with scales [..., row blocks, column blocks]"""
    s = scales.repeat_interleave(block_rows, dim=-2)[..., :codes.shape[-2], :]
    return codes.float() * s.repeat_interleave(128, dim=-1)[..., :codes.shape[-1]]


def _requantised(x):
    """float32 [..., cols] -> the values of its quantised rows"""
    rows = x.reshape(-1, x.shape[-1])
    return _values(*_quantise(rows, 1), 1).view(x.shape)


def _swiglu(x, st, some, name):
    """x [n, m, hidden], quantised, through the experts `some` of the stacks (None: the shared expert)"""
    w = lambda n: _values(*((st[name + n][None], st[name + n + "_scales"][None]) if some is None   # noqa: E731
                            else (st[name + n][some], st[name + n + "_scales"][some])), 128)
    g = torch.bmm(x, w("gate").transpose(1, 2))
    u = torch.bmm(x, w("up").transpose(1, 2))
    return torch.bmm(_requantised(g * torch.sigmoid(g) * u), w("down").transpose(1, 2))


def _experts_plain(st):
    x, idx, w = _requantised(st["x"].float()), st["idx"].long(), st["w"]
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
        rows[entry.view(-1)] = _swiglu(xs, st, some, "").view(-1, hidden)
    chosen = (idx < experts).view(tokens, k, 1)
    y = torch.where(chosen, rows[:-1].view(tokens, k, hidden) * w[:, :, None], 0.0).sum(dim=1)
    if st["shared_w"] is not None:
        y += st["shared_w"][:, None] * _swiglu(x[None], st, None, "s")[0]
    return y.to(st["x"].dtype)


def _balance_plain(st):
    logits, idx = st["logits"], st["idx"].long()
    (tokens, experts), k = logits.shape, idx.shape[1]
    valid = (idx >= 0) & (idx < experts)
    live = valid.any(dim=1, keepdim=True)
    counts = torch.zeros(experts + 1, dtype=torch.int32, device=logits.device)
    counts.index_add_(0, torch.where(valid, idx, experts).view(-1), torch.ones_like(idx, dtype=torch.int32).view(-1))
    counts = counts[:experts]
    f = counts.double() * k / counts.sum().clamp(min=1)
    n = live.sum().clamp(min=1)
    x = torch.where(live, logits.float(), 0.0)
    p = torch.exp(x - x.amax(dim=1, keepdim=True))
    p = p / p.sum(dim=1, keepdim=True)
    probs = torch.where(live, p, 0.0).sum(dim=0, dtype=torch.float64) / n
    scale = COEF * experts
    p = p.double()
    grad = torch.where(live, scale / n * p * (f - (p * f).sum(dim=1, keepdim=True)), 0.0)
    return dict(loss=(scale * (f * probs).sum()).float(), counts=counts, probs=probs.float(), dlogits=grad.to(logits.dtype))


# ------------------------------------------------------------------ one pass
def run(st):
    case = st["case"]
    if own:
        import helexa_amd as hx
        if case["kind"] == "quantise":
            return hx.quantize_f8(st["x"], block_rows=case["block_rows"])
        if case["kind"] == "linear":
            return st["layer"].forward(st["x"], workspace=st["workspace"])
        if case["kind"] == "balance":
            return hx.balance_loss(st["logits"], st["idx"], coef=COEF, workspace=st["workspace"])
        return st["block"].experts(st["x"], st["idx"], st["w"], shared_w=st["shared_w"], workspace=st["workspace"])
    if case["kind"] == "quantise":
        return _quantise(st["x"], case["block_rows"])
    if case["kind"] == "linear":
        x = _requantised(st["x"].float())
        return torch.mm(x, _values(st["codes"], st["scales"], 128).t()).to(st["x"].dtype)
    return _balance_plain(st) if case["kind"] == "balance" else _experts_plain(st)


# ------------------------------------------------------------------ exact values
def _grid():
    """the 127 values of E4M3 from 0 to 448, in order"""
    c = torch.arange(127, device="cuda").double()
    e, m = torch.floor(c / 8), c % 8
    return torch.where(e > 0, (1.0 + m / 8) * torch.pow(2.0, e - 7), m * 2.0 ** -9)


def _nearest(x, block_rows):
    """float64 codes [rows, cols] and scales: by the borders between neighbouring values, a tie to the even code"""
    grid = _grid()
    borders = (grid[1:] + grid[:-1]) / 2
    rows, cols = x.shape
    codes = torch.empty((rows, cols), dtype=torch.float64, device=x.device)
    scales = torch.empty(((rows + block_rows - 1) // block_rows, _blocks(cols)), dtype=torch.float64, device=x.device)
    for r in range(0, rows, 1 << 14):
        v = _blocked(x[r:r + (1 << 14)].double(), block_rows)
        s = (v.abs().amax(dim=(1, 3)) / 448.0).float().double().clamp(min=2.0 ** -126)
        a = v.abs() / s[:, None, :, None]
        i = torch.bucketize(a, borders)
        i += (a == borders[i.clamp(max=125)]) & (i % 2 == 1) & (i < 126)
        part = (grid[i] * torch.sign(v)).reshape(-1, v.shape[2] * 128)
        codes[r:r + (1 << 14)] = part[:min(1 << 14, rows - r), :cols]
        scales[r // block_rows:r // block_rows + s.shape[0]] = s
    return codes, scales


def _exact_rows(x):
    codes, scales = _nearest(x, 1)
    at = torch.arange(x.shape[1], device=x.device) // 128
    return codes * scales[:, at]


def _exact_weights(codes, scales):
    at = lambda n: torch.arange(n, device=codes.device) // 128   # noqa: E731
    return codes.double() * scales.double()[at(codes.shape[0])][:, at(codes.shape[1])]


def exact(case, seed):
    d = _inputs(case, seed)
    if case["kind"] == "quantise":
        return _nearest(d["x"], case["block_rows"])
    if case["kind"] == "linear":
        return _exact_rows(d["x"]) @ _exact_weights(d["codes"], d["scales"]).t()
    if case["kind"] == "balance":
        n, e = case["tokens"] - int(case["tokens"] * case["padded"]), case["experts"]
        idx = d["idx"][:n].long()
        counts = torch.stack([(idx == i).sum() for i in range(e)])
        f = counts.double() / n
        p = torch.softmax(d["logits"][:n].double(), dim=1)
        probs = p.mean(dim=0)
        grad = torch.zeros(d["logits"].shape, dtype=torch.float64, device="cuda")
        grad[:n] = COEF * e / n * p * (f - (p @ f)[:, None])
        return dict(loss=COEF * e * (f @ probs), counts=counts, probs=probs, dlogits=grad)
    x = _exact_rows(d["x"])
    y = torch.zeros_like(x)

    def add(tok, weight, name, e):
        part = lambda n: _exact_weights(*((d[name + n], d[name + n + "_scales"]) if e is None   # noqa: E731
                                          else (d[name + n][e], d[name + n + "_scales"][e])))
        g, u = x[tok] @ part("gate").t(), x[tok] @ part("up").t()
        y.index_add_(0, tok, weight[:, None].double() * (_exact_rows(g / (1.0 + torch.exp(-g)) * u) @ part("down").t()))

    for e in torch.unique(d["idx"]).tolist():
        if 0 <= e < case["experts"]:
            tok, j = torch.nonzero(d["idx"] == e, as_tuple=True)
            add(tok, d["w"][tok, j], "", e)
    if case["shared"]:
        add(torch.arange(case["tokens"], device="cuda"), d["shared_w"], "s", None)
    return y
