"""MXFP4 without a GPU: row sizes, the refusals of the entry points (checked
before anything touches a device), and the numpy rules the GPU tests compare with."""
import ctypes as C
from concurrent.futures import ThreadPoolExecutor

import numpy as np
import pytest

import mxfp4 as M


def _alone(f, **kw):
    """f(**kw) in a thread of its own: the last error is the thread's"""
    with ThreadPoolExecutor(1) as ex:
        return ex.submit(f, **kw).result()


def test_row_bytes():
    import helexa_amd as hx
    assert hx.MXFP4 == 39
    assert hx.row_bytes(hx.MXFP4, 32) == 17
    assert hx.row_bytes(hx.MXFP4, 2048) == 1088
    assert hx.row_bytes(hx.MXFP4, 48) == -1
    assert hx.row_bytes(hx.MXFP4, 0) == -1


@pytest.mark.parametrize("fn", ["hx_quantize", "hx_dequantize"])
def test_refusals_of_the_quantiser(fn):
    import helexa_amd as hx
    p = C.c_void_p(4096)   # never reached

    def calls():
        f = getattr(hx.lib(), fn)
        assert f(hx.MXFP4, None, 1, 32, p, None) == 1
        assert f(hx.MXFP4, p, 1, 32, None, None) == 1
        assert f(hx.MXFP4, p, -1, 32, p, None) == 1
        assert f(hx.MXFP4, p, 1, 33, p, None) == 1
        assert f(hx.MXFP4, p, 0, 32, p, None) == 0   # nothing to do

    _alone(calls)


def test_tensors_of_the_host_are_refused():
    import torch
    import helexa_amd as hx
    with pytest.raises(TypeError):
        hx.quantize(hx.MXFP4, torch.zeros(2, 32))
    with pytest.raises(TypeError):
        hx.dequantize(hx.MXFP4, torch.zeros((2, 17), dtype=torch.uint8), 32)


def test_numpy_rules():
    """ties to the even code, saturation, both signs of zero, the scale's range"""
    x = np.zeros((4, 32), np.float32)
    x[0, :16] = [4, .25, .75, 1.25, 1.75, 2.5, 3.5, 5, 7, 6.5, -0.0, -.25, -.2500001, .2500001, 7.99, -5.0001]
    q = M.quantise(x)
    assert q[0, 0] == 127
    assert [int(v) & 15 for v in q[0, 1:17]] == [6, 0, 2, 2, 4, 4, 6, 6, 7, 7, 8, 8, 9, 1, 7, 15]
    x[1] = np.float32(1e-45)
    x[2] = np.float32(3e38)
    x[3, 7] = np.inf
    q = M.quantise(x)
    assert q[1, 0] == 0 and q[2, 0] == 127 + 125 and q[3, 0] == 255 and not q[3, 1:].any()
    assert np.isnan(M.values(q[3])).all()
    assert M.values(q[0])[0] == 4.0 and M.values(q[0])[15] == -6.0


def _create(**kw):
    """hx_moe_create with pointers that no check reads"""
    import helexa_amd.moe as hx
    c = hx.HxConfig(64, 4, 2, 32, kw.pop("shared", 0), 1, hx.BF16)
    w = hx.HxWeights()
    d = dict(location=0, router_dtype=hx.BF16, gate_dtype=hx.MXFP4, up_dtype=hx.MXFP4, down_dtype=hx.MXFP4,
             router=4096, experts_gate=4096, experts_up=4096, experts_down=4096)
    for n in ("hidden_size", "moe_intermediate_size"):
        if n in kw:
            setattr(c, n, kw.pop(n))
    for n, v in {**d, **kw}.items():
        setattr(w, n, v)
    out = C.c_void_p()
    rc = hx.lib().hx_moe_create(C.byref(c), C.byref(w), 0, C.byref(out))
    return rc, hx.last_error()


@pytest.mark.parametrize("kw,rc,what", [
    (dict(down_dtype=8), 2, "all of gate_proj"), (dict(gate_dtype=12, up_dtype=12, hidden_size=256), 2, "all of gate_proj"),
    (dict(up_dtype=8), 2, "share a dtype"), (dict(hidden_size=80), 1, "does not tile"),
    (dict(moe_intermediate_size=48), 1, "does not tile"), (dict(hidden_size=32 * 513), 2, "at most"),
    (dict(shared=32, shared_gate_dtype=8, shared_up_dtype=39, shared_down_dtype=39), 2, "routed experts"),
    (dict(gate_dtype=40, up_dtype=40), 2, "unsupported storage dtype")])
def test_blocks_that_are_refused(kw, rc, what):
    got, msg = _alone(_create, **kw)
    assert got == rc and what in msg, (got, msg)


def test_experts_refuses_bad_arguments():
    import helexa_amd as hx
    p = C.c_void_p(4096)
    assert _alone(lambda: hx.lib().hx_moe_experts(None, p, 1, p, p, None, p, None, 0, None)) == 1
