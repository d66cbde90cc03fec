"""The balance loss's entry points without a GPU: what they refuse, and the reference's gradient."""
import ctypes as C
import os
from concurrent.futures import ThreadPoolExecutor

import numpy as np
import pytest

import balance as B
from helexa_amd import moe as hx

pytestmark = pytest.mark.skipif(not os.path.exists(hx.LIB_PATH), reason="libhxmoe.so not built")
P = 4096   # a pointer that a refused call never follows


def alone(f, **kw):
    """f(**kw) and the error text in a thread of its own: the last error is the thread's"""
    with ThreadPoolExecutor(1) as ex:
        return ex.submit(lambda: (f(**kw), hx.last_error())).result()


def loss(logits=P, dt=hx.F32, T=8, E=16, idx=P, k=4, out=P, probs=P, ws=P, ws_n=1 << 20):
    return hx.lib().hx_moe_balance_loss(logits, dt, T, E, idx, k, None, 1.0, out, None, probs, None, ws, ws_n, None)


def counts(idx=P, T=8, k=4, E=16, out=P, ws=P, ws_n=1 << 20):
    return hx.lib().hx_moe_expert_counts(idx, T, k, E, out, ws, ws_n, None)


@pytest.mark.parametrize("call,code", [
    (dict(logits=None), 1), (dict(idx=None), 1), (dict(out=None), 1), (dict(probs=None), 1), (dict(ws=None), 1),
    (dict(T=-1), 1), (dict(E=0), 1), (dict(k=0), 1), (dict(E=1025), 2), (dict(k=65), 2), (dict(dt=hx.F16), 2),
    (dict(T=(1 << 24) + 1), 2), (dict(ws=P + 8), 1), (dict(ws_n=100), 4)])
def test_the_loss_refuses(call, code):
    rc, text = alone(loss, **call)
    assert rc == code and text


@pytest.mark.parametrize("call,code", [
    (dict(idx=None), 1), (dict(out=None), 1), (dict(ws=None), 1), (dict(T=-1), 1), (dict(E=0), 1), (dict(k=0), 1),
    (dict(E=1025), 2), (dict(k=65), 2), (dict(T=(1 << 24) + 1), 2), (dict(ws=P + 4), 1), (dict(ws_n=100), 4)])
def test_the_counts_refuse(call, code):
    rc, text = alone(counts, **call)
    assert rc == code and text


def test_the_workspace_grows_with_tokens_and_experts_to_a_bound():
    sizes = [hx.balance_workspace_size(t, 512) for t in (0, 1, 100, 10000, 1 << 20, 1 << 24)]
    assert sizes == sorted(sizes) and sizes[-1] == sizes[-2] < 4 << 20
    assert hx.balance_workspace_size(100, 16) < hx.balance_workspace_size(100, 1024)
    n = C.c_size_t()
    for T, E, out, code in ((8, 16, None, 1), (-1, 16, C.byref(n), 1), (8, 1025, C.byref(n), 2)):
        assert alone(lambda: hx.lib().hx_moe_balance_workspace_size(T, E, out))[0] == code


def test_the_references_gradient_is_that_of_its_loss():
    """central differences in 64 bits, counts held"""
    x, idx = B.inputs(5, 12, 9, 3, padded=2)
    x = x.astype(np.float64)
    r = B.reference(x, idx, 0.3)
    rng = np.random.default_rng(6)
    for _ in range(5):
        v = rng.standard_normal(x.shape)
        v[10:] = 0.0
        hi, lo = (B.reference(x + h * v, idx, 0.3)["loss"] for h in (1e-5, -1e-5))
        assert abs((hi - lo) / 2e-5 - (r["dlogits"] * v).sum()) < 1e-9


@pytest.mark.parametrize("given,own,code", [(P, P, 1), (P, P + 60, 1), (P + 60, P, 1)])
def test_the_counts_that_are_read_are_not_those_written(given, own, code):
    call = lambda: hx.lib().hx_moe_balance_loss(P, hx.F32, 8, 16, P, 4, given, 1.0, P, own, P, None, P, 1 << 20, None)
    rc, text = alone(call)
    assert rc == code and "overlap" in text
