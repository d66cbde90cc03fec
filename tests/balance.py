"""A router's balance loss in 64 bits, its inputs and the bounds of a kernel in 32."""
import numpy as np

U = 2.0 ** -24   # half a step of float32


def inputs(seed, T, E, k, padded=0, spread=2.0):
    """logits float32 [T, E], indices int32 [T, k]; `padded` tokens at the end without experts, their logits NaN"""
    rng = np.random.default_rng(seed)
    x = (rng.standard_normal((T, E)) * spread).astype(np.float32)
    idx = np.argsort(-x, axis=1, kind="stable")[:, :k].astype(np.int32)
    if padded:
        idx[T - padded:] = rng.choice([-1, E, -2 ** 31, 2 ** 31 - 1], (padded, k))
        x[T - padded:] = np.nan
    return x, idx


def counts_of(idx, E):
    v = idx[(idx >= 0) & (idx < E)]
    return np.bincount(v, minlength=E).astype(np.int64)


def reference(x, idx, coef, counts=None):
    """-> loss, counts, probs, gradient, all in 64 bits, and s_t"""
    x = np.asarray(x, np.float64)
    T, E = x.shape
    k = idx.shape[1]
    live = ((idx >= 0) & (idx < E)).any(axis=1)
    own = counts_of(idx, E)
    c = own if counts is None else np.asarray(counts, np.int64)
    f = k * c / c.sum() if c.sum() else np.zeros(E)
    n = int(live.sum())
    p = np.zeros((T, E))
    if n:
        e = np.exp(x[live] - x[live].max(axis=1, keepdims=True))
        p[live] = e / e.sum(axis=1, keepdims=True)
    s = p @ f
    probs = p.sum(axis=0) / max(n, 1)
    scale = coef * E / n if n else 0.0
    return dict(loss=coef * E * float(f @ probs), counts=own, probs=probs, dlogits=scale * p * (f - s[:, None]) * live[:, None],
                p=p, s=s, f=f, scale=scale, live=live)


def bounds(x, r, T, out_eps):
    """How far a kernel in 32 bits may be off: exp of d = x - max has a relative error of 2.3 |d| + 4
    half steps (the difference's rounding, the product's with log2 e and the constant's, the
    exponential's own), a sum over a row 32 more (16 columns a lane, 6 steps over lanes; products'
    roundings), so that p has 5 D + 72 and the means, over at most 64 + T / 4096 rows in a lane's
    sum and 16 in the tables', 5 D + 160 + T / 4096. The difference f - s keeps the errors of both terms. Probabilities
    below 2^-126 may be zero. out_eps: half a step of the gradient's type."""
    live = r["live"]
    d = 0.0
    if live.any():
        xl = np.asarray(x, np.float64)[live]
        xl = np.where(np.isneginf(xl), xl.max(axis=1, keepdims=True), xl)
        d = min(104.0, float((xl.max(axis=1, keepdims=True) - xl).max()))   # exp(-104) is below float32's smallest
    tiny = 2.0 ** -126
    row, mean = (5 * d + 80) * U, (5 * d + 160 + T / 4096) * U
    grad = row * r["scale"] * r["p"] * (np.abs(r["f"]) + np.abs(r["s"])[:, None]) + out_eps * np.abs(r["dlogits"])
    return dict(loss=mean * abs(r["loss"]) + tiny, probs=mean * r["probs"] + tiny,
                dlogits=(grad * (1 + 2.0 ** -6) + tiny * (1 + r["scale"] * (r["f"].max(initial=0) + 1))) * live[:, None])
