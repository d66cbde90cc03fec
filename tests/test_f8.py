"""E4M3 without a GPU: the numpy rules, and what the entry points refuse before they touch a device."""
import ctypes as C
import os
from concurrent.futures import ThreadPoolExecutor

import numpy as np
import pytest

import f8 as F
from helexa_amd import moe as hx

built = pytest.mark.skipif(not os.path.exists(hx.LIB_PATH), reason="libhxmoe.so not built")
P = 4096   # a pointer that a refused call never follows


def alone(f):
    """f() and the error text in a thread of its own: the last error is the thread's"""
    with ThreadPoolExecutor(1) as ex:
        return ex.submit(lambda: (f(), hx.last_error())).result()


def test_values_are_torchs():
    import torch
    t = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float().numpy()
    assert np.array_equal(t, F.VALUES.astype(np.float32), equal_nan=True)


def test_quantise_rounds_to_the_nearest_code():
    """against torch's conversion where it rounds once: quotients that float32 holds exactly"""
    import torch
    rng = np.random.default_rng(1)
    x = (rng.standard_normal((40, 256)) * np.exp2(rng.integers(-8, 8, (40, 256)))).astype(np.float32)
    x[:, 0] = x[:, 128] = 448 * 2.0 ** rng.integers(-3, 9, 40)   # scales are powers of two
    x = np.clip(x, -x[:, :1], x[:, :1])
    codes, scales = F.quantise(x, 1)
    assert np.array_equal(scales, np.repeat(x[:, :1] / 448, 2, axis=1))
    want = torch.from_numpy(x / F.spread(scales, 40, 256, 1)).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(codes, want)


def test_quantised_values_are_within_half_a_step():
    x = np.random.default_rng(2).standard_normal((300, 333))
    for rows in (1, 128):
        s = F.spread(F.quantise(x, rows)[1].astype(np.float64), 300, 333, rows)
        assert (np.abs(F.quantised(x, rows) - x) <= np.maximum(2.0 ** -4 * np.abs(x), 2.0 ** -10 * s) * (1 + 1e-6)).all()


@built
@pytest.mark.parametrize("args,code", [
    ((None, 0, 4, 128, 1, P, P), 1), ((P, 0, 4, 128, 1, None, P), 1), ((P, 0, 4, 128, 1, P, None), 1), ((P, 0, -1, 128, 1, P, P), 1),
    ((P, 0, 4, 0, 1, P, P), 1), ((P, 1, 4, 128, 1, P, P), 2), ((P, 0, 4, 128, 64, P, P), 2), ((P + 2, 0, 4, 128, 1, P, P), 1),
    ((P + 1, 30, 4, 128, 1, P, P), 1), ((P, 0, 1 << 40, 128, 1, P, P), 2), ((P, 0, 4, 1 << 40, 1, P, P), 2), ((P, 0, 0, 128, 1, P, P), 0)])
def test_the_quantiser_refuses(args, code):
    assert alone(lambda: hx.lib().hx_quantize_f8(*args, None))[0] == code


@built
@pytest.mark.parametrize("args,code", [
    ((0, 128, P, P, 1, 0), 1), ((128, 0, P, P, 1, 0), 1), ((128, 128, None, P, 1, 0), 1), ((128, 128, P, None, 1, 0), 1),
    ((128, 128, P, P, 2, 0), 1), (((1 << 20) + 1, 128, P, P, 1, 0), 2), ((128, (1 << 17) + 1, P, P, 1, 0), 2)])
def test_a_layer_refuses_to_be_made(args, code):
    out = C.c_void_p(7)
    rc, text = alone(lambda: hx.lib().hx_linear_create(*args, C.byref(out)))
    assert rc == code and text and out.value is None
    assert alone(lambda: hx.lib().hx_linear_create(*args, None))[0] == 1


@built
def test_calls_without_a_layer():
    n = C.c_size_t()
    assert alone(lambda: hx.lib().hx_linear_forward(None, P, 0, 1, P, 0, None, 0, None))[0] == 1
    assert alone(lambda: hx.lib().hx_linear_workspace_size(None, 1, C.byref(n)))[0] == 1
    assert hx.lib().hx_linear_destroy(None) == 0


@built
def test_a_block_refuses_wrong_scales_and_mixtures():
    def create(with_scales=True, **kw):
        c = hx.HxConfig(256, 8, 2, 128, 0, 1, hx.F32)
        for n in ("hidden_size", "moe_intermediate_size"):
            if n in kw:
                setattr(c, n, kw[n])
        w, s, out = hx.HxWeights(), hx.HxF8Scales(P, P, P, None, None, None), C.c_void_p()
        w.location, w.router_dtype, w.router = hx.HX_HOST, hx.F32, P
        w.experts_gate = w.experts_up = w.experts_down = P
        w.gate_dtype, w.up_dtype, w.down_dtype = (kw.get(n, hx.F8_E4M3) for n in ("gate", "up", "down"))
        if with_scales:
            return alone(lambda: hx.lib().hx_moe_create_f8(C.byref(c), C.byref(w), C.byref(s) if kw.get("scales", True) else None, 0, C.byref(out)))
        return alone(lambda: hx.lib().hx_moe_create(C.byref(c), C.byref(w), 0, C.byref(out)))
    assert create(scales=False)[0] == 1
    assert create(with_scales=False)[0] == 1
    assert create(gate=hx.F32, up=hx.F32, down=hx.F32)[0] == 1
    assert create(down=hx.MXFP4)[0] == 2 and create(down=hx.BF16)[0] == 2 and create(up=hx.F32)[0] == 2
    assert create(hidden_size=264)[0] == 2 and create(moe_intermediate_size=40)[0] == 2


@built
@pytest.mark.parametrize("args,code", [
    ((P, 0, 1, 1 << 31, 1, P, P), 2), ((P, 0, 1, 1 << 31, 128, P, P), 2), ((P, 0, 1, (1 << 31) - 127, 1, P, P), 2),
    ((P, 0, 4, 128, 1, P, P + 2), 1), ((P, 0, 0, (1 << 31) - 128, 1, P, P), 0)])
def test_the_quantisers_longest_row(args, code):
    assert alone(lambda: hx.lib().hx_quantize_f8(*args, None))[0] == code
