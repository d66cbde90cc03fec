"""Calls of the E4M3 quantiser and the balance loss that are refused, or done, before they touch a device."""
import os
from concurrent.futures import ThreadPoolExecutor

import pytest

from helexa_amd import moe as hx

pytestmark = pytest.mark.skipif(not os.path.exists(hx.LIB_PATH), reason="libhxmoe.so not built")
P = 1 << 20   # a pointer that a refused call never follows


def alone(f):
    """f() and the error text in a thread of its own: the last error is the thread's"""
    with ThreadPoolExecutor(1) as ex:
        return ex.submit(lambda: (f(), hx.last_error())).result()


@pytest.mark.parametrize("dt,size", [(hx.F32, 4), (hx.BF16, 2)])
def test_a_gradient_over_other_rows_of_the_logits(dt, size):
    """8 tokens x 16 experts: off by an element to all but one, on either side"""
    n = 8 * 16 * size
    for at in (size, -size, 16 * size, n - size, size - n):
        rc, text = alone(lambda: hx.lib().hx_moe_balance_loss(P, dt, 8, 16, 1 << 24, 4, None, 1.0, 1 << 25, None, 1 << 26, P + at, 1 << 27,
                                                              1 << 20, None))
        assert rc == 1 and "overlap" in text


@pytest.mark.parametrize("dt,size", [(hx.F32, 4), (hx.BF16, 2)])
@pytest.mark.parametrize("block_rows", [1, 128])
def test_the_quantiser_in_its_inputs_place(block_rows, dt, size):
    """300 rows of 260: codes in x's place, at its last byte, its first; scales in x, in the codes"""
    n, s = 300 * 260, 4 * 3 * (300 if block_rows == 1 else 3)
    far = 1 << 28
    for codes, scales in ((P, far), (P + n * size - 1, far), (P - n + 1, far), (far, P), (far, P + n * size - 4), (far, P - s + 4),
                          (far, far), (far, far + n - 4), (far, far - s + 4)):
        rc, text = alone(lambda: hx.lib().hx_quantize_f8(P, dt, 300, 260, block_rows, codes, scales, None))
        assert rc == 1 and "overlap" in text, (codes, scales)
    assert alone(lambda: hx.lib().hx_quantize_f8(P, dt, 1 << 38, 1 << 12, block_rows, far, far, None))[0] == 2


def test_no_rows_need_no_memory():
    """an empty tensor has no address"""
    for block_rows in (1, 128):
        assert alone(lambda: hx.lib().hx_quantize_f8(None, hx.F32, 0, 128, block_rows, None, None, None))[0] == 0
        assert alone(lambda: hx.lib().hx_quantize_f8(None, hx.F16, 0, 128, block_rows, None, None, None))[0] == 2
        assert alone(lambda: hx.lib().hx_quantize_f8(None, hx.F32, 1, 128, block_rows, None, None, None))[0] == 1
