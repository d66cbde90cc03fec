"""hx_quantize and hx_dequantize of MXFP4 rows, byte for byte and bit for bit
against numpy: around the 128 blocks a workgroup takes, sources and destinations
off 16-byte alignment, every code on every rounding boundary, special values."""
import numpy as np
import pytest

import mxfp4 as M

pytestmark = pytest.mark.gpu


def _to(x):
    import torch
    return torch.from_numpy(x).cuda()


@pytest.mark.parametrize("rows,cols", [(1, 32), (3, 96), (127, 32), (128, 32), (129, 32), (33, 2080), (7, 4096)])
def test_rows_both_ways(rows, cols):
    from helexa_amd import moe as hx
    rng = np.random.default_rng(rows * 7 + cols)
    x = (rng.standard_normal((rows, cols)) * np.exp2(rng.integers(-20, 20, (rows, 1)))).astype(np.float32)
    ref = M.quantise(x)
    got = hx.quantize(hx.MXFP4, _to(x))
    assert np.array_equal(got.cpu().numpy(), ref)
    back = hx.dequantize(hx.MXFP4, got, cols).cpu().numpy()
    assert np.array_equal(back, M.values(ref).astype(np.float32))
    assert np.array_equal(np.signbit(back), np.signbit(M.values(ref)))


def test_rounding_boundaries():
    """each border between two codes, one float below and one above, at several
    scales; and amax one float below a power of two"""
    from helexa_amd import moe as hx
    edge = np.array([.25, .75, 1.25, 1.75, 2.5, 3.5, 5.0], np.float32)
    vals = np.concatenate([edge, np.nextafter(edge, np.float32(0)), np.nextafter(edge, np.float32(9)), [6, 7, 7.9999995]])
    vals = np.concatenate([vals, -vals]).astype(np.float32)
    x = np.zeros((20, 64), np.float32)
    for r in range(20):
        x[r, :48] = vals
        x[r, 31] = x[r, 63] = 4.0 if r % 2 else np.nextafter(np.float32(8), np.float32(0))
        x[r] *= np.float32(2.0) ** (3 * r - 30)
    ref = M.quantise(x)
    assert np.array_equal(hx.quantize(hx.MXFP4, _to(x)).cpu().numpy(), ref)


def test_special_values():
    from helexa_amd import moe as hx
    inf, nan = np.float32("inf"), np.float32("nan")
    rng = np.random.default_rng(5)
    special = [inf, -inf, nan, 0.0, -0.0, 1e-45, -1e-40, 2.0 ** -126, 2.0 ** -125, 3.4e38, -3.4e38, 1e20, 1e-38]
    x = rng.standard_normal((4 * len(special), 128)).astype(np.float32)
    for i, v in enumerate(special):
        x[4 * i, 5] = v
        x[4 * i + 1, 32:64] = v
        x[4 * i + 2, ::7] = v
        with np.errstate(all="ignore"):
            x[4 * i + 3] *= np.float32(v)
    ref = M.quantise(x)
    got = hx.quantize(hx.MXFP4, _to(x))
    assert np.array_equal(got.cpu().numpy(), ref)
    back = hx.dequantize(hx.MXFP4, got, 128).cpu().numpy()
    with np.errstate(over="ignore"):
        assert np.array_equal(back, M.values(ref).astype(np.float32), equal_nan=True)


def test_every_scale_and_code_read_back():
    from helexa_amd import moe as hx
    q = np.zeros((256, 17), np.uint8)
    q[:, 0] = np.arange(256)
    q[:, 1:] = np.arange(16) | (15 - np.arange(16)) << 4
    got = hx.dequantize(hx.MXFP4, _to(q), 32).cpu().numpy()
    with np.errstate(over="ignore"):
        ref = M.values(q).astype(np.float32)
    assert np.array_equal(got, ref, equal_nan=True)


@pytest.mark.parametrize("rows", [1, 130])
def test_unaligned_pointers(rows):
    """float rows on a 4-byte boundary, packed rows on an odd byte, nothing written
    past either end"""
    import torch
    from helexa_amd import moe as hx
    cols = 96
    rng = np.random.default_rng(rows)
    x = rng.standard_normal((rows, cols)).astype(np.float32)
    ref = M.quantise(x).reshape(-1)
    s = torch.cuda.current_stream().cuda_stream
    src = torch.zeros(rows * cols + 1, device="cuda")
    src[1:] = _to(x.reshape(-1))
    out = torch.zeros(ref.size + 20, dtype=torch.uint8, device="cuda")
    hx.check(hx.lib().hx_quantize(hx.MXFP4, src.data_ptr() + 4, rows, cols, out.data_ptr() + 3, s), "hx_quantize")
    got = out.cpu().numpy()
    assert np.array_equal(got[3:3 + ref.size], ref) and not got[:3].any() and not got[3 + ref.size:].any()
    back = torch.zeros(rows * cols + 9, device="cuda")
    hx.check(hx.lib().hx_dequantize(hx.MXFP4, out.data_ptr() + 3, rows, cols, back.data_ptr() + 4, s), "hx_dequantize")
    b = back.cpu().numpy()
    assert np.array_equal(b[1:1 + rows * cols], M.values(ref).astype(np.float32)) and b[0] == 0 and not b[1 + rows * cols:].any()


def test_rows_that_are_refused_and_no_rows():
    """rows of another length than the columns' would be read or written past their end"""
    import torch
    import helexa_amd as hx
    q = torch.zeros((4, 34), dtype=torch.uint8, device="cuda")
    for bad, cols in ((q, 32), (q.view(-1), 64), (q, 48), (q[:, :17], 64), (q.view(2, 2, 2, 17), 64)):
        with pytest.raises(ValueError):
            hx.dequantize(hx.MXFP4, bad, cols)
    with pytest.raises(TypeError):
        hx.dequantize(hx.MXFP4, q.view(torch.int16), 64)
    assert hx.dequantize(hx.MXFP4, q[:0], 64).shape == (0, 64)
    assert hx.quantize(hx.MXFP4, torch.zeros((0, 64), device="cuda")).shape == (0, 34)
    assert hx.dequantize(hx.MXFP4, q.view(2, 2, 34), 64).shape == (2, 2, 64)
