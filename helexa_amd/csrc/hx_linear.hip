// C ABI of the E4M3 quantiser and the linear layer on such weights.
#include <algorithm>
#include <new>

#include "hx_abi.h"
#include "hx_f8.h"

using namespace hx;

struct hx_linear {
  int device = 0;
  int64_t N = 0, K = 0;
  uint8_t* w = nullptr;
  void* own_ws = nullptr;
  size_t own_ws_bytes = 0;
};

// largest sizes of a layer: the kernels index a row's columns and a matrix' tiles by 32 bits
static constexpr int64_t MAX_IN = 1 << 17, MAX_OUT = 1 << 20;

extern "C" int hx_quantize_f8(const void* x, int x_dtype, int64_t rows, int64_t cols, int block_rows, void* codes,
                              float* scales, void* stream) {
  if (rows < 0 || cols <= 0 || (rows > 0 && (!x || !codes || !scales))) return fail(HX_ERR_INVALID_ARGUMENT, "bad argument");
  if (x_dtype != HX_F32 && x_dtype != HX_BF16) return fail(HX_ERR_UNSUPPORTED, "hx_quantize_f8: x dtype %d", x_dtype);
  if (block_rows != 1 && block_rows != 128)
    return fail(HX_ERR_UNSUPPORTED, "hx_quantize_f8: blocks of 1 or 128 rows, not %d", block_rows);
  if ((uintptr_t)x & (x_dtype == HX_F32 ? 3 : 1)) return fail(HX_ERR_INVALID_ARGUMENT, "x does not start on an element");
  if ((uintptr_t)scales & 3) return fail(HX_ERR_INVALID_ARGUMENT, "the scales do not start on an element");
  // a row's columns are indexed by 32 bits, bytes by 64
  if (cols > ((int64_t)1 << 31) - 128 || rows > std::min((int64_t)1 << 38, ((int64_t)1 << 48) / cols))
    return fail(HX_ERR_UNSUPPORTED, "hx_quantize_f8: %lld rows of %lld are too many", (long long)rows, (long long)cols);
  if (rows == 0) return HX_OK;
  // a block is read by several threads, its codes and scale leave while others are read
  const size_t n = (size_t)rows * cols, xb = n * (x_dtype == HX_F32 ? 4 : 2),
               sb = sizeof(float) * (size_t)((rows + block_rows - 1) / block_rows) * f8_blocks(cols);
  if (overlap(x, xb, codes, n) || overlap(x, xb, scales, sb) || overlap(codes, n, scales, sb))
    return fail(HX_ERR_INVALID_ARGUMENT, "hx_quantize_f8: x, codes and scales overlap");
  if (block_rows == 1) HX_HIP(launch_f8_rows(x, x_dtype == HX_BF16, rows, cols, codes, scales, false, (hipStream_t)stream));
  else HX_HIP(launch_f8_blocks(x, x_dtype == HX_BF16, rows, cols, codes, scales, (hipStream_t)stream));
  return HX_OK;
}

extern "C" int hx_linear_destroy(hx_linear* l) {
  if (!l) return HX_OK;
  DeviceScope dev(l->device);
  (void)hipDeviceSynchronize();
  if (l->w) (void)hipFree(l->w);
  if (l->own_ws) (void)hipFree(l->own_ws);
  delete l;
  return HX_OK;
}

static int linear_upload(hx_linear* l, const void* codes, const float* scales, int location) {
  const size_t bytes = (size_t)f8_mat_bytes(l->N, l->K), nc = (size_t)(l->N * l->K),
               ns = sizeof(float) * (size_t)f8_blocks(l->N) * f8_blocks(l->K);
  if (hipMalloc((void**)&l->w, bytes) != hipSuccess) return fail(HX_ERR_OUT_OF_MEMORY, "cannot allocate %zu bytes", bytes);
  uint8_t* tmp = nullptr;
  if (location == HX_HOST) {
    const size_t at = (nc + 255) & ~(size_t)255;
    if (hipMalloc((void**)&tmp, at + ns) != hipSuccess)
      return fail(HX_ERR_OUT_OF_MEMORY, "cannot allocate %zu staging bytes", at + ns);
    hipError_t e = hipMemcpy(tmp, codes, nc, hipMemcpyHostToDevice);
    if (e == hipSuccess) e = hipMemcpy(tmp + at, scales, ns, hipMemcpyHostToDevice);
    if (e != hipSuccess) {
      (void)hipFree(tmp);
      return fail(HX_ERR_DEVICE, "upload failed: %s", hipGetErrorString(e));
    }
    codes = tmp;
    scales = (const float*)(tmp + at);
  }
  hipError_t e = launch_f8_repack(codes, scales, 1, l->N, l->K, l->w, 0, 0);
  if (e == hipSuccess) e = hipDeviceSynchronize();
  if (tmp) (void)hipFree(tmp);
  return e == hipSuccess ? HX_OK : fail(HX_ERR_DEVICE, "repack failed: %s", hipGetErrorString(e));
}

extern "C" int hx_linear_create(int64_t out_features, int64_t in_features, const void* codes, const float* scales,
                                int location, int device, hx_linear** out) {
  if (!out) return fail(HX_ERR_INVALID_ARGUMENT, "null argument");
  *out = nullptr;
  if (!codes || !scales || out_features <= 0 || in_features <= 0) return fail(HX_ERR_INVALID_ARGUMENT, "bad argument");
  if (out_features > MAX_OUT || in_features > MAX_IN)
    return fail(HX_ERR_UNSUPPORTED, "at most %lld outputs and %lld inputs are supported", (long long)MAX_OUT, (long long)MAX_IN);
  if (location != HX_HOST && location != HX_DEVICE)
    return fail(HX_ERR_INVALID_ARGUMENT, "location must be HX_HOST or HX_DEVICE");
  DeviceScope dev(device);
  HX_HIP(dev.err);
  hx_linear* l = new (std::nothrow) hx_linear();
  if (!l) return fail(HX_ERR_OUT_OF_MEMORY, "no host memory");
  l->device = device;
  l->N = out_features;
  l->K = in_features;
  const int rc = linear_upload(l, codes, scales, location);
  if (rc) {
    hx_linear_destroy(l);
    return rc;
  }
  *out = l;
  return HX_OK;
}

// what a call of M rows keeps: the quantised rows, where the kernel does not quantise by itself
static size_t linear_codes(const hx_linear* l, int64_t M) { return ((size_t)(M * f8_row(l->K)) + 255) & ~(size_t)255; }
static size_t linear_ws(const hx_linear* l, int64_t M) {
  return f8_quant_inside(M, l->K) ? 0 : linear_codes(l, M) + sizeof(float) * (size_t)M * f8_scale_row(l->K);
}

extern "C" int hx_linear_workspace_size(const hx_linear* l, int64_t n_rows, size_t* bytes) {
  if (!l || !bytes || n_rows < 0) return fail(HX_ERR_INVALID_ARGUMENT, "bad argument");
  *bytes = linear_ws(l, n_rows);
  return HX_OK;
}

extern "C" int hx_linear_forward(hx_linear* l, const void* x, int x_dtype, int64_t n_rows, void* y, int y_dtype,
                                 void* workspace, size_t workspace_bytes, void* stream) {
  if (!l || n_rows < 0 || (n_rows > 0 && (!x || !y))) return fail(HX_ERR_INVALID_ARGUMENT, "bad argument");
  if ((x_dtype != HX_F32 && x_dtype != HX_BF16) || (y_dtype != HX_F32 && y_dtype != HX_BF16))
    return fail(HX_ERR_UNSUPPORTED, "hx_linear_forward: x dtype %d, y dtype %d", x_dtype, y_dtype);
  if (n_rows == 0) return HX_OK;
  if (n_rows > HX_MAX_TOKENS) return fail(HX_ERR_UNSUPPORTED, "too many rows in one call");
  if (((uintptr_t)x & (x_dtype == HX_F32 ? 3 : 1)) || ((uintptr_t)y & (y_dtype == HX_F32 ? 3 : 1)))
    return fail(HX_ERR_INVALID_ARGUMENT, "x or y does not start on an element");
  // few rows: every workgroup quantises all of x, while others write their features of y
  if (overlap(x, (size_t)(n_rows * l->K) * (x_dtype == HX_F32 ? 4 : 2), y, (size_t)(n_rows * l->N) * (y_dtype == HX_F32 ? 4 : 2)))
    return fail(HX_ERR_INVALID_ARGUMENT, "hx_linear_forward: x and y overlap");
  DeviceScope dev(l->device);
  HX_HIP(dev.err);
  hipStream_t s = (hipStream_t)stream;
  const size_t need = linear_ws(l, n_rows);
  if (need && workspace) {
    if (workspace_bytes < need)
      return fail(HX_ERR_WORKSPACE_TOO_SMALL, "workspace of %zu bytes, %zu needed for %lld rows", workspace_bytes, need,
                  (long long)n_rows);
    if ((uintptr_t)workspace & 15) return fail(HX_ERR_INVALID_ARGUMENT, "the workspace must start on 16 bytes");
  } else if (need) {
    if (capturing(s))   // the handle's own may be freed by a later call, the graph would keep it
      return fail(HX_ERR_INVALID_ARGUMENT, "hx_linear_forward: a captured call needs the caller's workspace");
    if (l->own_ws_bytes < need) {
      if (l->own_ws) {
        HX_HIP(hipDeviceSynchronize());
        (void)hipFree(l->own_ws);
        l->own_ws = nullptr;
        l->own_ws_bytes = 0;
      }
      if (hipMalloc(&l->own_ws, need) != hipSuccess) return fail(HX_ERR_OUT_OF_MEMORY, "workspace allocation of %zu bytes", need);
      l->own_ws_bytes = need;
    }
    workspace = l->own_ws;
  }
  F8LinearArgs a{};
  a.w = l->w;
  a.x = x; a.xbf = x_dtype == HX_BF16;
  a.y = y; a.ybf = y_dtype == HX_BF16;
  a.M = n_rows; a.N = (int)l->N; a.K = (int)l->K;
  a.xq = (uint8_t*)workspace;
  a.xs = need ? (float*)((uint8_t*)workspace + linear_codes(l, n_rows)) : nullptr;
  HX_HIP(launch_f8_linear(a, s));
  return HX_OK;
}
