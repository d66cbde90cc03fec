"""E4M3: the quantiser bit by bit, the linear layer against 64 bits."""
import numpy as np
import pytest

import f8 as F

pytestmark = pytest.mark.gpu


def cuda(a, bf=False):
    import torch
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t.to(torch.bfloat16) if bf else t


def same_codes(got, want, tag=""):
    codes, scales = (t.cpu() for t in got)
    import torch
    assert codes.dtype == torch.float8_e4m3fn
    c, s = codes.view(torch.uint8).numpy(), scales.numpy()
    assert np.array_equal(s, want[1], equal_nan=True), (tag, np.argwhere(~((s == want[1]) | (np.isnan(s) & np.isnan(want[1]))))[:5])
    assert np.array_equal(c, want[0]), (tag, np.argwhere(c != want[0])[:5])


@pytest.mark.parametrize("bf", [False, True])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 128), (3, 130), (17, 2080), (128, 128), (129, 384), (200, 100), (257, 1000), (1, 4096)])
def test_quantise(rows, cols, block_rows, bf):
    import helexa_amd as hx
    rng = np.random.default_rng(rows + cols)
    x = rng.standard_normal((rows, cols), dtype=np.float32) * np.exp2(rng.integers(-12, 12, (rows, cols))).astype(np.float32)
    x[rng.random((rows, cols)) < 0.1] = 0.0
    x[rng.random((rows, cols)) < 0.02] = -0.0
    x = F.bf16(x) if bf else x
    same_codes(hx.quantize_f8(cuda(x, bf), block_rows), F.quantise(x, block_rows))


@pytest.mark.parametrize("block_rows", [1, 128])
def test_borders_of_the_codes(block_rows):
    """values on and next to the borders between codes, for scales that are powers of two and
    others; the largest code of each block is met exactly"""
    import helexa_amd as hx
    rng = np.random.default_rng(1)
    b = np.concatenate([F.BORDERS, F.GRID]).astype(np.float32)
    rows = []
    for s in [1.0, 0.25, 1.7e-3, 3.14159, 2.0 ** -100 * 1.3, 2.0 ** 100 * 1.9, 2.0 ** -126, 7e-37, 1e30] + list(np.exp(rng.uniform(-40, 40, 55))):
        with np.errstate(over="ignore", under="ignore"):
            v = (b.astype(np.float64) * s).astype(np.float32)
        for near in (v, np.nextafter(v, np.float32(0)), np.nextafter(v, np.float32(np.inf))):
            near = np.where(np.isfinite(near), near, 0).astype(np.float32)
            near = np.concatenate([near, -near, np.zeros(512 - 2 * len(b), np.float32)]) if len(b) * 2 <= 512 else near
            near = near.reshape(-1, 128)
            near[:, 0] = np.float32(448.0) * np.float32(s)
            rows.append(near[np.isfinite(near).all(axis=1)])
    x = np.concatenate(rows)
    same_codes(hx.quantize_f8(cuda(x), block_rows), F.quantise(x, block_rows))


@pytest.mark.parametrize("block_rows", [1, 128])
def test_blocks_without_numbers_small_and_large(block_rows):
    import helexa_amd as hx
    x = np.random.default_rng(2).standard_normal((300, 400)).astype(np.float32)
    x[3, 5], x[4, 200], x[5, 399] = np.nan, np.inf, -np.inf
    x[6], x[7] = 0.0, -0.0
    x[8] *= np.float32(2.0 ** -130)
    x[9] = np.float32(2.0 ** -149)
    x[10] *= np.float32(2.0 ** 126)
    x[150:] *= np.float32(2.0 ** -128)
    same_codes(hx.quantize_f8(cuda(x), block_rows), F.quantise(x, block_rows))


def test_quantise_stacks_views_and_nothing():
    import helexa_amd as hx
    import torch
    x = np.random.default_rng(3).standard_normal((3, 200, 260)).astype(np.float32)
    t = cuda(x)
    codes, scales = hx.quantize_f8(t, 128)
    one, s1 = hx.quantize_f8(t)
    assert codes.shape == t.shape and scales.shape == (3, 2, 3) and s1.shape == (3, 200, 3)
    for i in range(3):
        same_codes((codes[i], scales[i]), F.quantise(x[i], 128))
        same_codes((one[i], s1[i]), F.quantise(x[i], 1))
    whole = cuda(x[:, :128])
    codes, scales = hx.quantize_f8(whole, 128)
    for i in range(3):
        same_codes((codes[i], scales[i]), F.quantise(x[i, :128], 128))
    same_codes(hx.quantize_f8(t[0].t()), F.quantise(x[0].T, 1))
    off = torch.empty(128 * 256 + 1, device="cuda")[1:].view(128, 256)   # off 16 bytes
    off.copy_(t[0, :128, :256])
    for rows in (1, 128):
        same_codes(hx.quantize_f8(off, rows), F.quantise(x[0, :128, :256], rows))
    codes, scales = hx.quantize_f8(t[:, :0])
    assert codes.shape == (3, 0, 260) and scales.shape == (3, 0, 3)
    assert hx.quantize_f8(t[0, 0])[1].shape == (3,)


def test_quantise_on_another_stream():
    import helexa_amd as hx
    import torch
    x = np.random.default_rng(4).standard_normal((512, 2048)).astype(np.float32)
    want = hx.quantize_f8(cuda(x))
    t, s = cuda(x), torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        torch.cuda._sleep(20_000_000)
    codes, scales = hx.quantize_f8(t, stream=s)
    del t
    junk = [torch.zeros((512, 2048), device="cuda") for _ in range(3)]
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(codes.view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(scales, want[1])
    del junk


# ------------------------------------------------------------------ linear layer
def rows_of(seed, M, K, bf=False):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((M, K), dtype=np.float32)
    x[:, rng.random(K) < 0.02] *= 20
    return F.bf16(x) if bf else x


def check_linear(y, x, codes, scales):
    import torch
    ref, mag, fixed = F.linear(x, codes, scales)
    bound = F.sum_steps(x.shape[1]) * F.U * mag + 2.0 ** -140
    if y.dtype == torch.bfloat16:   # 8-bit instructions, then the result's own rounding
        bound = (bound + fixed) * (1 + 2.0 ** -8) + 2.0 ** -8 * np.abs(ref)
    got = y.float().cpu().numpy().astype(np.float64).reshape(ref.shape)
    off = np.abs(got - ref)
    print(f"[err] worst {np.max(off / bound, initial=0):.3f} of the bound, norm {np.linalg.norm(off) / max(np.linalg.norm(ref), 1e-300):.2e}", flush=True)
    assert (off <= bound).all(), np.argwhere(off > bound)[:5]


ROWS = [1, 2, 15, 16, 17, 31, 32, 33, 64, 65, 100, 128, 129, 200, 333]
SHAPES = [(1, 1), (16, 16), (128, 128), (130, 100), (1031, 2080), (512, 2048), (64, 4104), (300, 130), (20, 1000), (256, 640)]


@pytest.mark.parametrize("N,K", SHAPES)
def test_linear(N, K):
    import helexa_amd as hx
    import torch
    codes, scales = F.make_weights(N + K, N, K)
    layer = hx.F8Linear.load(cuda(codes), cuda(scales))
    for M in ROWS:
        for bf in (False, True):
            print("case", N, K, M, bf, flush=True)
            x = rows_of(M, M, K, bf)
            check_linear(layer(cuda(x, bf)), x, codes, scales)
        check_linear(layer(cuda(x, True), out_dtype=torch.float32), x, codes, scales)
    layer.close()


@pytest.mark.parametrize("M", [1, 7, 40, 300, 1100])
def test_every_code_and_scale(M):
    """weights of random codes, all 254 that are numbers, with scales of many sizes and signs"""
    import helexa_amd as hx
    rng = np.random.default_rng(M)
    N, K = 272, 400
    codes = rng.integers(0, 256, (N, K)).astype(np.uint8)
    codes[(codes & 127) == 127] = 0
    scales = (rng.standard_normal((3, 4)) * np.exp2(rng.integers(-20, 20, (3, 4)))).astype(np.float32)
    x = rows_of(M, M, K) * np.exp2(rng.integers(-30, 30, (M, 1))).astype(np.float32)
    check_linear(hx.F8Linear.load(cuda(codes), cuda(scales))(cuda(x)), x, codes, scales)


@pytest.mark.parametrize("M", [3, 16, 20, 90, 600])
def test_what_is_no_number_stays_in_its_row_and_feature(M):
    import helexa_amd as hx
    N, K = 150, 300
    codes, scales = F.make_weights(M, N, K)
    x = rows_of(M, M, K)
    plain = hx.F8Linear.load(cuda(codes), cuda(scales))(cuda(x)).cpu().numpy()
    x[1, 200], x[2, 0] = np.nan, np.inf
    codes[77, 3] = 0x7f
    y = hx.F8Linear.load(cuda(codes), cuda(scales))(cuda(x)).cpu().numpy()
    assert np.isnan(y[1:3]).all() and np.isnan(y[:, 77]).all()
    keep = np.ones((M, N), bool)
    keep[1:3], keep[:, 77] = False, False
    assert np.array_equal(y[keep], plain[keep])


@pytest.mark.parametrize("M", [1, 16, 17, 64, 65, 500])
def test_layouts_of_a_call(M):
    """x and y off 16 bytes, strided x, leading dimensions, an output of the caller's whose neighbours stay, no rows"""
    import helexa_amd as hx
    import torch
    N, K = 132, 272
    codes, scales = F.make_weights(9, N, K)
    layer = hx.F8Linear.load(cuda(codes), cuda(scales))
    for bf in (False, True):
        x = cuda(rows_of(M, M, K, bf), bf)
        want = layer(x)
        off = torch.empty(M * K + 1, dtype=x.dtype, device="cuda")[1:].view(M, K)
        off.copy_(x)
        wide = torch.zeros((M, K + 3), dtype=x.dtype, device="cuda")
        wide[:, 2:K + 2] = x
        place = torch.full((M * N + 9,), 5.0, dtype=x.dtype, device="cuda")
        out = place[1:M * N + 1].view(M, N)
        assert torch.equal(layer(off), want) and torch.equal(layer(wide[:, 2:K + 2]), want)
        assert layer(off, out=out) is out and torch.equal(out, want) and (place[0] == 5).all() and (place[M * N + 1:] == 5).all()
        assert torch.equal(layer(x.view(M, 1, K)), want.view(M, 1, N))
        ws = torch.empty(layer.workspace_size(M) + 64, dtype=torch.uint8, device="cuda")
        assert torch.equal(layer(x, workspace=ws), want)
        assert layer(x[:0]).shape == (0, N)


def test_host_weights_and_float8_tensors():
    import helexa_amd as hx
    import torch
    codes, scales = F.make_weights(5, 100, 200)
    x = cuda(rows_of(5, 20, 200))
    a = hx.F8Linear.load(torch.from_numpy(codes), torch.from_numpy(scales))(x)
    b = hx.F8Linear.load(cuda(codes).view(torch.float8_e4m3fn), cuda(scales))(x)
    assert torch.equal(a, b)
    w = torch.randn((100, 200), device="cuda")
    check_linear(hx.F8Linear.load(*hx.quantize_f8(w, 128))(x), x.cpu().numpy(), *F.quantise(w.cpu().numpy(), 128))


@pytest.mark.parametrize("M", [8, 40, 700])
def test_linear_on_another_stream_and_captured(M):
    import helexa_amd as hx
    import torch
    N, K = 260, 520
    codes, scales = F.make_weights(M, N, K)
    layer = hx.F8Linear.load(cuda(codes), cuda(scales))
    xs = [cuda(rows_of(M + i, M, K)) for i in range(3)]
    want = [layer(x) for x in xs]
    s = torch.cuda.Stream()
    ws = torch.empty(layer.workspace_size(M), dtype=torch.uint8, device="cuda")
    t = xs[0].clone()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        torch.cuda._sleep(20_000_000)
    y = layer(t, stream=s, workspace=ws)
    del t
    junk = [torch.zeros((M, K), device="cuda") for _ in range(3)]
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(y, want[0])
    x = xs[0].clone()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = layer(x, workspace=ws)
    for i in (1, 2, 0, 1):
        x.copy_(xs[i])
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i]) and torch.equal(layer(xs[i]), want[i])
    del junk


def test_refusals():
    import helexa_amd as hx
    import torch
    codes, scales = F.make_weights(5, 100, 200)
    layer = hx.F8Linear.load(cuda(codes), cuda(scales))
    x = cuda(rows_of(5, 20, 200))
    short = torch.empty(layer.workspace_size(20) - 1, dtype=torch.uint8, device="cuda")
    for bad, err in ((lambda: hx.F8Linear.load(cuda(codes), cuda(scales[:, :1])), ValueError),
                     (lambda: hx.F8Linear.load(cuda(codes), torch.from_numpy(scales)), ValueError),
                     (lambda: hx.F8Linear.load(cuda(codes).float(), cuda(scales)), ValueError),
                     (lambda: layer(x[:, :199]), ValueError), (lambda: layer(x.cpu()), ValueError), (lambda: layer(x.half()), TypeError),
                     (lambda: layer(x, workspace=short), hx.HxError), (lambda: layer(x, out=x), ValueError),
                     (lambda: layer(x, out_dtype=torch.float16), TypeError),
                     (lambda: hx.quantize_f8(x.half()), TypeError), (lambda: hx.quantize_f8(x.cpu()), TypeError),
                     (lambda: hx.quantize_f8(x, 64), ValueError), (lambda: hx.quantize_f8(x[0], 128), ValueError)):
        with pytest.raises(err):
            bad()


@pytest.mark.parametrize("N,K", [(70, 16400), (33, 60000), (17, 131072)])
def test_long_rows(N, K):
    """rows whose codes do not fit in LDS with few of them, and the longest a layer takes"""
    import helexa_amd as hx
    codes, scales = F.make_weights(K, N, K)
    layer = hx.F8Linear.load(cuda(codes), cuda(scales))
    for M in (1, 3, 5, 20, 70):
        x = rows_of(M, M, K)
        check_linear(layer(cuda(x)), x, codes, scales)


@pytest.mark.parametrize("rows,block_rows", [((1 << 29) + 5, 1), ((1 << 30) + 200, 128)])
def test_more_rows_than_a_launch_takes(rows, block_rows):
    """one column: a launch has less than 2^32 threads. A block's largest has the code of +-448, the
    others are smaller: the codes of 1, 1/2 and 1/4 of it"""
    import torch
    import helexa_amd as hx
    pattern = torch.tensor([4.0, -2.0, 1.0, -4.0, 2.0, 1.0, -1.0], device="cuda", dtype=torch.bfloat16)
    x = pattern.repeat(rows // 7 + 1)[:rows].reshape(rows, 1)
    codes, scales = hx.quantize_f8(x, block_rows)
    want = 4.0 if block_rows == 128 else x.reshape(-1).abs()
    s = torch.as_tensor(want, device="cuda", dtype=torch.float32) / torch.tensor(448.0, device="cuda")
    assert scales.shape == ((rows + block_rows - 1) // block_rows, 1) and bool((scales.reshape(-1) == s).all())
    names = {448.0: 0x7e, 224.0: 0x76, 112.0: 0x6e}
    if block_rows == 128:
        byte = [names[abs(v) * 112] | (0x80 if v < 0 else 0) for v in pattern.tolist()]
    else:
        byte = [0x7e | (0x80 if v < 0 else 0) for v in pattern.tolist()]
    byte = torch.tensor(byte, device="cuda", dtype=torch.uint8).repeat(rows // 7 + 1)[:rows]
    assert bool((codes.view(torch.uint8).reshape(-1) == byte).all())
