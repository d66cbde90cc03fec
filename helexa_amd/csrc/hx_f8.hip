// E4M3 weights and activations with float32 scales by blocks of 128: quantisation, the
// linear layer y = q(x) W^T, and experts y[t] = sum_j w[t,j] D_e(q(silu(G_e q(x_t)) * U_e q(x_t))).
//
// Quantisation of a block: s = max(max|x| / 448, 2^-126), codes the E4M3 values nearest to
// x / s (the exact quotient, ties to even); a block with a NaN or an infinity has scale NaN.
//
// Products run on v_mfma_f32_16x16x128_f8f6f4 with the weights as its A operand and the
// activations as its B operand: one instruction is one block of K. Its D (lane l: row
// l % 16 of the activations, features 4 (l / 16) + i in register i) starts from zero and
// is added to the sums times sx sw, a lane's one scale of its row and block times the
// scale of the weights' block, which a wave's features share: four multiply-adds a lane
// for the instruction's 32 cycles.
//
// The instruction adds the products that a lane holds in fixed point, 13 bits below the
// exponent of the largest (measured: 2^14 + 2^1 is kept, of 2^14 + 2^0 the second is lost; what
// the four lanes of a row hold is added in float32). A sum is off by 1.4e-5 of its norm so for normal
// inputs, by 3e-5 where one column in 100 is 16 times the others, by 5.5e-5 for h in down (measured); a
// bf16 result's own rounding is 1.7e-3. Float32 results (WIDE) take the codes as bf16, which is exact, and
// v_mfma_f32_16x16x32_bf16, four for a block at half the rate: 1e-8 a block. Gate/up's sums are
// taken so for bf16 too where it costs little (launch_f8_gate_up): h's codes hang on them.
#include <algorithm>

#include "hx_f8.h"
#include "hx_mx_routing.h"

namespace hx {

typedef int f8_v8i __attribute__((ext_vector_type(8)));
typedef float f8_v4f __attribute__((ext_vector_type(4)));
typedef __bf16 f8_v2bf __attribute__((ext_vector_type(2)));
typedef __bf16 f8_v8bf __attribute__((ext_vector_type(8)));

// ---------------------------------------------------------------- quantisation
// a block's scale from the bits of its largest magnitude (NaN and infinity above all
// others), and whether it is a number
HX_DEV bool f8_scale(uint32_t m, float& s) {
  const bool fine = m < 0x7f800000u;
  s = fine ? fmaxf(__uint_as_float(m) / 448.f, 0x1p-126f) : __builtin_nanf("");
  return fine;
}

// x / s for the conversion to E4M3: within half a step of float32 of the quotient, and
// where the quotient is no float32 with the last bit set. The borders between codes have
// few bits, so that the value lies on the same side of each as the quotient, and on one
// only if the quotient does. s is scaled up where the remainders would be subnormal.
struct F8Div {
  float s, r, up;
  HX_DEV explicit F8Div(float scale) {
    up = scale < 0x1p-60f ? 0x1p64f : 1.f;
    s = scale * up;
    r = 1.f / s;
  }
  HX_DEV float operator()(float x) const {
    x *= up;
    const float q0 = x * r;
    // what the quotients are too much: of this sign, -0 stays -0
    const float q = __builtin_fmaf(-__builtin_fmaf(q0, s, -x), r, q0);
    const float rem = __builtin_fmaf(q, s, -x);
    const int b = __float_as_int(q), step = (__float_as_int(rem) ^ b) < 0 ? 1 : -1;
    return __int_as_float(rem != 0.f && (b & 1) == 0 ? b + step : b);
  }
};

// four codes in a word
HX_DEV uint32_t f8_pack(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}

template <int N>
HX_DEV uint32_t f8_amax(const float (&f)[N]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < N; i++) m = max(m, __float_as_uint(f[i]) & 0x7fffffffu);
  return m;
}

// N values with a scale -> N / 4 words of codes; a block that is no number: zeros
template <int N>
HX_DEV void f8_codes(const float (&f)[N], float s, bool fine, uint32_t (&w)[N / 4]) {
  const F8Div div(fine ? s : 1.f);
#pragma unroll
  for (int i = 0; i < N / 4; i++)
    w[i] = fine ? f8_pack(div(f[4 * i]), div(f[4 * i + 1]), div(f[4 * i + 2]), div(f[4 * i + 3])) : 0u;
}

// The same by a product with 1 / s, within 1.5 steps of float32 of the quotient: for h, whose values
// are off by more than that already, a border between codes is no sharper than they are (the exact
// quotients took a third of the gate/up kernel's vector instructions)
template <int N>
HX_DEV void f8_codes_near(const float (&f)[N], float s, bool fine, uint32_t (&w)[N / 4]) {
  const float r = 1.f / (fine ? s : 1.f);
#pragma unroll
  for (int i = 0; i < N / 4; i++)
    w[i] = fine ? f8_pack(f[4 * i] * r, f[4 * i + 1] * r, f[4 * i + 2] * r, f[4 * i + 3] * r) : 0u;
}

// loads and stores of whole words at any address (the hardware splits what crosses a line)
typedef uint32_t f8_any4 __attribute__((ext_vector_type(4), aligned(1)));
typedef uint32_t f8_any1 __attribute__((aligned(1)));

// N elements from p or, at a row's end, n of them, zeros behind
template <bool BF, int N>
HX_DEV void f8_load(const void* base, int64_t at, int n, float (&f)[N]) {
  if (n >= N) {
    constexpr int W = BF ? N / 2 : N;   // words
    uint32_t u[W];
    const uint8_t* p = (const uint8_t*)base + at * (BF ? 2 : 4);
    if constexpr (W >= 4) {
#pragma unroll
      for (int i = 0; i < W / 4; i++) {
        const f8_any4 v = ((const f8_any4*)p)[i];
        u[4 * i] = v[0]; u[4 * i + 1] = v[1]; u[4 * i + 2] = v[2]; u[4 * i + 3] = v[3];
      }
    } else {
#pragma unroll
      for (int i = 0; i < W; i++) u[i] = ((const f8_any1*)p)[i];
    }
#pragma unroll
    for (int i = 0; i < N; i++)
      f[i] = __uint_as_float(!BF ? u[BF ? 0 : i] : i & 1 ? u[i >> 1] & 0xffff0000u : u[i >> 1] << 16);
    return;
  }
#pragma unroll
  for (int i = 0; i < N; i++) f[i] = i < n ? ld_act(base, at + i, BF) : 0.f;
}

struct F8Rows {
  const void* x;
  int64_t rows, cols;
  uint8_t* codes;
  int64_t ldc;       // bytes of a row of codes, cols or more
  float* scales;
  int lds;           // floats of a row of scales
};

// Rows of x, a thread 16 of its values, 8 threads a block. Bound by HBM: 8192 rows of 4096 in bf16, 102
// MB, in 22 to 24 us (4.2 to 4.6 TB/s); few rows by a launch, 3.5 us.
template <bool BF>
HX_DEV void f8_quant_rows(const F8Rows& q, int64_t id) {
  const int nb = f8_blocks(q.cols);
  const int64_t blk = id >> 3, r = blk / nb;
  const int b = (int)(blk % nb), c0 = 128 * b + 16 * (int)(id & 7);
  const bool has = r < q.rows;   // the lanes of a block agree
  float f[16];
  f8_load<BF>(q.x, (has ? r : 0) * q.cols + c0, (int)min<int64_t>(q.cols - c0, 16), f);
  uint32_t m = f8_amax(f);
  m = max(m, (uint32_t)dpp_mov<0xB1>((int)m));    // quad_perm 1,0,3,2
  m = max(m, (uint32_t)dpp_mov<0x4E>((int)m));    // quad_perm 2,3,0,1
  m = max(m, (uint32_t)dpp_mov<0x141>((int)m));   // row_half_mirror
  float s;
  const bool fine = f8_scale(m, s);
  uint32_t w[4];
  f8_codes(f, s, fine, w);
  if (!has) return;
  uint8_t* const p = q.codes + r * q.ldc + c0;
  const int n = (int)min<int64_t>(q.ldc - c0, 16);
  if (n == 16) *(f8_any4*)p = f8_any4{w[0], w[1], w[2], w[3]};
  else
    for (int i = 0; i < n; i++) p[i] = (uint8_t)(w[i >> 2] >> (8 * (i & 3)));
  if ((id & 7) == 0) q.scales[r * q.lds + b] = s;
}
template <bool BF>
__global__ __launch_bounds__(256) void k_f8_rows(F8Rows q) {
  f8_quant_rows<BF>(q, (int64_t)blockIdx.x * 256 + threadIdx.x);
}

// a launch has less than 2^32 threads
constexpr int64_t F8_LAUNCH_THREADS = (int64_t)1 << 31;

hipError_t launch_f8_rows(const void* x, bool xbf, int64_t rows, int64_t cols, void* codes, float* scales, bool padded,
                          hipStream_t s) {
  F8Rows q{x, rows, cols, (uint8_t*)codes, padded ? f8_row(cols) : cols, scales, padded ? f8_scale_row(cols) : f8_blocks(cols)};
  const int64_t most = F8_LAUNCH_THREADS / (8 * (int64_t)f8_blocks(cols));   // rows of a launch
  for (int64_t left = rows; left > 0; left -= most) {
    q.rows = std::min(left, most);
    const dim3 g((unsigned)((q.rows * f8_blocks(cols) * 8 + 255) / 256));
    if (xbf) hx_launch(k_f8_rows<true>, g, dim3(256), 0, s, q);
    else hx_launch(k_f8_rows<false>, g, dim3(256), 0, s, q);
    q.x = (const uint8_t*)q.x + most * cols * (xbf ? 2 : 4);
    q.codes += most * q.ldc;
    q.scales += most * q.lds;
  }
  return hipGetLastError();
}

// Blocks of 128 x 128: a workgroup a block, 64 values a thread in registers, 4 columns of
// 16 rows, 8 rows apart. Bound by HBM: 262144 rows of 2048 in float32, 2.7 GB, in 440 to 470 us by the card (5.7
// to 6.1 TB/s).
template <bool BF>
__global__ __launch_bounds__(256) void k_f8_blocks(F8Rows q) {
  __shared__ uint32_t part[4];
  const int nb = f8_blocks(q.cols), tid = threadIdx.x;
  const int64_t rb = blockIdx.x / nb;
  const int b = (int)(blockIdx.x % nb), c0 = 128 * b + 4 * (tid & 31);
  const int64_t r0 = 128 * rb + (tid >> 5);
  const int n = (int)min<int64_t>(q.cols - c0, 4);
  float f[16][4];
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 16; i++) {
    const int64_t r = r0 + 8 * i;
    f8_load<BF>(q.x, r * q.cols + c0, r < q.rows ? n : 0, f[i]);
  }
#pragma unroll
  for (int i = 0; i < 16; i++) m = max(m, f8_amax(f[i]));
  m = wave_max_u32(m);
  if (lane_id() == 0) part[tid >> 6] = m;
  __syncthreads();
  m = max(max(part[0], part[1]), max(part[2], part[3]));
  float s;
  const bool fine = f8_scale(m, s);
#pragma unroll
  for (int i = 0; i < 16; i++) {
    const int64_t r = r0 + 8 * i;
    uint32_t w[1];
    f8_codes(f[i], s, fine, w);
    if (r >= q.rows) continue;
    uint8_t* p = q.codes + r * q.cols + c0;
    if (n == 4) *(f8_any1*)p = w[0];
    else
      for (int j = 0; j < n; j++) p[j] = (uint8_t)(w[0] >> (8 * j));
  }
  if (tid == 0) q.scales[rb * nb + b] = s;
}

hipError_t launch_f8_blocks(const void* x, bool xbf, int64_t rows, int64_t cols, void* codes, float* scales, hipStream_t s) {
  F8Rows q{x, rows, cols, (uint8_t*)codes, cols, scales, f8_blocks(cols)};
  const int64_t most = std::max<int64_t>(F8_LAUNCH_THREADS / 256 / f8_blocks(cols), 1) * 128;
  for (int64_t left = rows; left > 0; left -= most) {
    q.rows = std::min(left, most);
    const dim3 g((unsigned)((int64_t)f8_blocks(q.rows) * f8_blocks(cols)));
    if (xbf) hx_launch(k_f8_blocks<true>, g, dim3(256), 0, s, q);
    else hx_launch(k_f8_blocks<false>, g, dim3(256), 0, s, q);
    q.x = (const uint8_t*)q.x + most * cols * (xbf ? 2 : 4);
    q.codes += most * cols;
    q.scales += most / 128 * q.lds;
  }
  return hipGetLastError();
}

// ---------------------------------------------------------------- stored weights
// a thread per 16 bytes of a tile, padding included, then the scales
__global__ __launch_bounds__(256) void k_repack_f8(const uint8_t* codes, const float* scales, int64_t count, int64_t rows,
                                                   int64_t K, uint8_t* dst, int64_t dst_stride, int64_t first) {
  const int KB = f8_blocks(K), SR = f8_scale_row(K), RB = f8_blocks(rows);
  const int64_t pieces = (int64_t)f8_tiles(rows) * KB * 128, per = pieces + (int64_t)RB * SR;
  const int64_t id = first + (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= per * count) return;
  const int64_t m = id / per, q = id % per;
  uint8_t* mat = dst + m * dst_stride;
  if (q >= pieces) {
    const int64_t at = q - pieces;
    const int rb = (int)(at / SR), b = (int)(at % SR);
    ((float*)(mat + f8_code_bytes(rows, K)))[at] = b < KB ? scales[(m * RB + rb) * KB + b] : 0.f;
    return;
  }
  const int l = (int)(q & 63), h = (int)((q >> 6) & 1);
  const int64_t tile = q >> 7, row = 16 * (tile / KB) + (l & 15), c0 = 128 * (tile % KB) + 64 * h + 16 * (l >> 4);
  uint32_t w[4] = {0u, 0u, 0u, 0u};
  const uint8_t* src = codes + (m * rows + row) * K + c0;   // the caller's rows: any alignment
  if (row < rows) {
    if (c0 + 16 <= K && ((uintptr_t)src & 15) == 0) {
      const uint4 v = *(const uint4*)src;
      w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    } else {
#pragma unroll
      for (int i = 0; i < 16; i++)
        if (c0 + i < K) w[i >> 2] |= (uint32_t)src[i] << (8 * (i & 3));
    }
  }
  *(uint4*)(mat + q * 16) = make_uint4(w[0], w[1], w[2], w[3]);
}

hipError_t launch_f8_repack(const void* codes, const float* scales, int64_t count, int64_t rows, int64_t K, void* dst,
                            int64_t dst_stride, hipStream_t s) {
  const int64_t per = (int64_t)f8_tiles(rows) * f8_blocks(K) * 128 + (int64_t)f8_blocks(rows) * f8_scale_row(K);
  for (int64_t first = 0; first < per * count; first += F8_LAUNCH_THREADS)
    hipLaunchKernelGGL(k_repack_f8, dim3((unsigned)((std::min(per * count - first, F8_LAUNCH_THREADS) + 255) / 256)), dim3(256),
                       0, s, (const uint8_t*)codes, scales, count, rows, K, (uint8_t*)dst, dst_stride, first);
  return hipGetLastError();
}

// ---------------------------------------------------------------- operands
HX_DEV f8_v4f f8_zero4() { return f8_v4f{0.f, 0.f, 0.f, 0.f}; }

// a lane's two halves as an operand
HX_DEV f8_v8i f8_op(const uint4& a, const uint4& b) {
  return f8_v8i{(int)a.x, (int)a.y, (int)a.z, (int)a.w, (int)b.x, (int)b.y, (int)b.z, (int)b.w};
}
// part c of 4 of an operand's codes as bf16, which is exact
HX_DEV f8_v8bf f8_part(const f8_v8i& v, int c) {
  f8_v8bf r;
#pragma unroll
  for (int j = 0; j < 2; j++) {
    const f8_v2bf lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((uint32_t)v[2 * c + j], 1.f, false);
    const f8_v2bf hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((uint32_t)v[2 * c + j], 1.f, true);
    r[4 * j] = lo[0]; r[4 * j + 1] = lo[1]; r[4 * j + 2] = hi[0]; r[4 * j + 3] = hi[1];
  }
  return r;
}
// an operand as the products take it
template <bool WIDE>
struct F8Arg;
template <>
struct F8Arg<false> {
  f8_v8i v;
  HX_DEV F8Arg() {}
  HX_DEV explicit F8Arg(const f8_v8i& c) : v(c) {}
};
template <>
struct F8Arg<true> {
  f8_v8bf v[4];
  HX_DEV F8Arg() {}
  HX_DEV explicit F8Arg(const f8_v8i& c) {
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = f8_part(c, i);
  }
};
// a block of K: scales of 0 select the instruction's form without any
HX_DEV f8_v4f f8_mfma(const F8Arg<false>& w, const F8Arg<false>& x) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w.v, x.v, f8_zero4(), 0, 0, 0, 0, 0, 0);
}
HX_DEV f8_v4f f8_mfma(const F8Arg<true>& w, const F8Arg<true>& x) {
  f8_v4f d = f8_zero4();
#pragma unroll
  for (int i = 0; i < 4; i++) d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w.v[i], x.v[i], d, 0, 0, 0);
  return d;
}
// two tiles of features with the same rows, exact, a part of the operands at a time (as bf16 all at
// once they took 20 registers more and a CU a workgroup less: 4 tokens' experts 38.3 us for 35.7)
HX_DEV void f8_exact_two(const f8_v8i& w0, const f8_v8i& w1, const f8_v8i& x, f8_v4f& d0, f8_v4f& d1) {
  d0 = d1 = f8_zero4();
#pragma unroll
  for (int c = 0; c < 4; c++) {
    const f8_v8bf xc = f8_part(x, c);
    d0 = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f8_part(w0, c), xc, d0, 0, 0, 0);
    d1 = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f8_part(w1, c), xc, d1, 0, 0, 0);
    __builtin_amdgcn_sched_barrier(0);
  }
}
HX_DEV void f8_add(f8_v4f& acc, const f8_v4f& d, float s) {
#pragma unroll
  for (int i = 0; i < 4; i++) acc[i] = __builtin_fmaf(d[i], s, acc[i]);
}

// the largest of the four lanes that hold a row's block, in all of them
HX_DEV uint32_t f8_max_of_4(uint32_t m) {
  const auto a = __builtin_amdgcn_permlane32_swap(m, m, false, false);
  m = max((uint32_t)a[0], (uint32_t)a[1]);
  const auto b = __builtin_amdgcn_permlane16_swap(m, m, false, false);
  return max((uint32_t)b[0], (uint32_t)b[1]);
}

// A block of a row by 32 lanes, 4 values a lane, into LDS: its 128 codes and its scale. (By the lanes
// that hold an operand each value is quantised by all 16 columns of a row alone: a layer of 4096 x
// 2048 took 7.4 us for a row so, and 5 by this.)
template <bool BF, bool NEAR = false>
HX_DEV void f8_block_to_lds(const void* x, int64_t row_at, int K, int b, uint8_t* codes, float* scale) {
  const int l = lane_id() & 31, c0 = 128 * b + 4 * l;
  float f[4];
  f8_load<BF>(x, row_at + c0, K - c0, f);
  uint32_t m = f8_amax(f);
  m = max(m, (uint32_t)dpp_mov<0xB1>((int)m));    // quad_perm 1,0,3,2
  m = max(m, (uint32_t)dpp_mov<0x4E>((int)m));    // quad_perm 2,3,0,1
  m = max(m, (uint32_t)dpp_mov<0x141>((int)m));   // row_half_mirror
  m = max(m, (uint32_t)dpp_mov<0x140>((int)m));   // row_mirror
  const auto r = __builtin_amdgcn_permlane16_swap(m, m, false, false);
  float s;
  const bool fine = f8_scale(max((uint32_t)r[0], (uint32_t)r[1]), s);
  uint32_t w[1];
  if constexpr (NEAR) f8_codes_near(f, s, fine, w);
  else f8_codes(f, s, fine, w);
  *(uint32_t*)(codes + 4 * l) = w[0];
  if (l == 0) *scale = s;
}
// bytes between rows in LDS: 16 more than the codes, so that the rows' pieces start on other banks
__host__ __device__ inline int f8_pitch(int K) { return f8_blocks(K) * 128 + 16; }

// a lane's part of block b of a quantised row as an operand
HX_DEV f8_v8i f8_operand(const uint8_t* row, int b) {
  const uint8_t* p = row + 128 * b + 16 * (lane_id() >> 4);
  return f8_op(*(const uint4*)p, *(const uint4*)(p + 64));
}

HX_DEV void f8_store(void* y, int64_t at, float v, bool bf) {
  if (bf) ((uint16_t*)y)[at] = f32_to_bf16(v);
  else ((float*)y)[at] = v;
}

// ---------------------------------------------------------------- linear layer, few rows
// Workgroup: 16 features; its 8 waves share K block by block and add up in LDS. CT columns
// of 16 rows. QUANT: a few rows as the caller has them, quantised into LDS by every workgroup (a
// launch less); the weights are on their way meanwhile. Bound by latency: 1 row, 4096 x 2048, 8.4 MB
// in 3.7 us (a launch, two round trips to memory, the sum through LDS).
template <bool BF, int CT, bool QUANT, bool WIDE>
__global__ __launch_bounds__(512) void k_f8_few_rows(F8LinearArgs a) {
  constexpr int PITCH = 16 * CT + 1;
  extern __shared__ __align__(16) uint8_t sm[];
  __shared__ float red[8 * 16 * PITCH];
  const int tid = threadIdx.x, lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = blockIdx.x, KB = f8_blocks(a.K), M = (int)a.M, col = lane & 15;
  const uint8_t* w = a.w + (int64_t)n * KB * 2048 + lane * 16;
  const float* ws = (const float*)(a.w + f8_code_bytes(a.N, a.K)) + (int64_t)(n >> 3) * f8_scale_row(a.K);
  uint4 ring[2][2];
  float rs[2];
  auto fetch = [&](int i, int b) {   // past the last: the last again
    b = min(b, KB - 1);
    ring[i][0] = *(const uint4*)(w + (int64_t)b * 2048);
    ring[i][1] = *(const uint4*)(w + (int64_t)b * 2048 + 1024);
    rs[i] = ws[b];
  };
  fetch(0, wave);
  fetch(1, wave + 8);
  const int pitch = QUANT ? f8_pitch(a.K) : 0;
  float* const qs = (float*)(sm + M * pitch);   // [M][KB]
  if constexpr (QUANT) {
    for (int u = 2 * wave + (lane >> 5); u < M * KB; u += 16) {
      const int r = u / KB, b = u % KB;
      f8_block_to_lds<BF>(a.x, (int64_t)r * a.K, a.K, b, sm + r * pitch + 128 * b, qs + u);
    }
    lds_barrier();
  }
  f8_v4f acc[CT];
#pragma unroll
  for (int c = 0; c < CT; c++) acc[c] = f8_zero4();
  for (int b0 = wave; b0 < KB; b0 += 16) {
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const int b = b0 + 8 * i;
      if (b >= KB) break;
      const F8Arg<WIDE> wv(f8_op(ring[i][0], ring[i][1]));
      const float sw = rs[i];
      f8_v8i x[CT];
      float sx[CT];
#pragma unroll
      for (int c = 0; c < CT; c++) {
        const int r = min(16 * c + col, M - 1);
        x[c] = f8_operand(QUANT ? sm + r * pitch : a.xq + r * f8_row(a.K), b);
        sx[c] = QUANT ? qs[r * KB + b] : a.xs[(int64_t)r * f8_scale_row(a.K) + b];
      }
      fetch(i, b + 16);
#pragma unroll
      for (int c = 0; c < CT; c++) f8_add(acc[c], f8_mfma(wv, F8Arg<WIDE>(x[c])), sx[c] * sw);
    }
  }
#pragma unroll
  for (int c = 0; c < CT; c++)
#pragma unroll
    for (int i = 0; i < 4; i++) red[(wave * 16 + 4 * (lane >> 4) + i) * PITCH + 16 * c + col] = acc[c][i];
  __syncthreads();
  for (int o = tid; o < 16 * min(M, 16 * CT); o += 512) {
    const int f = o & 15, r = o >> 4;
    float y = 0.f;
#pragma unroll
    for (int v = 0; v < 8; v++) y += red[(v * 16 + f) * PITCH + r];
    if (16 * n + f < a.N) f8_store(a.y, (int64_t)r * a.N + 16 * n + f, y, !WIDE);
  }
}

// ---------------------------------------------------------------- products over tiles of rows
// A tile's rows in LDS, 4 blocks of K at a time: [4][TM][128 bytes], 16-byte piece j of row r
// at j ^ r % 8 (the rows' pieces would all start on one bank). They come in by direct
// loads, a chunk ahead.
template <int TM, int NW>
struct F8Tile {
  static constexpr int CB = 4, BYTES = CB * TM * 128, LOADS = BYTES / 1024 / NW;   // KiB a wave and chunk
  const uint8_t* src[LOADS];
  // rowptr(r): the quantised row r of the tile
  template <typename F>
  HX_DEV void init(int wave, F rowptr) {
#pragma unroll
    for (int i = 0; i < LOADS; i++) {
      const int q = (i * NW + wave) * 64 + lane_id(), row = q / 8 % TM;
      src[i] = rowptr(row) + q / (8 * TM) * 128 + ((q % 8) ^ (row & 7)) * 16;
    }
  }
  // blocks b0 .. min(b0 + 4, nblk) - 1
  HX_DEV void load(int wave, int b0, int nblk, uint32_t lds) const {
#pragma unroll
    for (int i = 0; i < LOADS; i++)
      if (b0 + (i * NW + wave) * 8 / TM < nblk) dma16(src[i] + (int64_t)b0 * 128, lds + (i * NW + wave) * 1024);
  }
};

// acc[m][t] = the sums over KB blocks of K of a wave's NM tiles of 16 features (their codes
// from w[m], a lane's place in it included; tiles m with m % 2 == q, or all, by the scales ws[q])
// times the tile's rows; xs[t]: a lane's row's scales. Two blocks of weights are on their way.
template <bool WIDE, int TM, int NW, int NM, int NQ>
HX_DEV void f8_products(const uint8_t* const (&w)[NM], const float* const (&ws)[NQ], const F8Tile<TM, NW>& rows,
                        const float* const (&xs)[TM / 16], int wave, uint8_t* buf, int KB, f8_v4f (&acc)[NM][TM / 16]) {
  constexpr int TT = TM / 16, CB = F8Tile<TM, NW>::CB, BYTES = F8Tile<TM, NW>::BYTES, R = 2;
  const uint32_t lds = (uint32_t)(uintptr_t)(lds_u8*)buf;
  const int lane = lane_id();
#pragma unroll
  for (int m = 0; m < NM; m++)
#pragma unroll
    for (int t = 0; t < TT; t++) acc[m][t] = f8_zero4();
  uint4 ring[R][NM][2];
  auto fetch = [&](int i, int b) {   // past the last: the last again
    const int64_t at = (int64_t)min(b, KB - 1) * 2048;
#pragma unroll
    for (int m = 0; m < NM; m++) {
      ring[i][m][0] = *(const uint4*)(w[m] + at);
      ring[i][m][1] = *(const uint4*)(w[m] + at + 1024);
    }
  };
  rows.load(wave, 0, KB, lds);
#pragma unroll
  for (int i = 0; i < R; i++) fetch(i, i);
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(R * NM * 2) : "memory");   // the rows are the oldest
  lds_barrier();
  const uint8_t* const mine = buf + (lane & 15) * 128;
  const int p0 = ((lane >> 4) ^ (lane & 7)) * 16, p1 = ((4 + (lane >> 4)) ^ (lane & 7)) * 16;
  int h = 0;
  for (int b0 = 0; b0 < KB; b0 += CB, h ^= 1) {
    float4 sx[TT], sw[NQ];
#pragma unroll
    for (int t = 0; t < TT; t++) sx[t] = *(const float4*)(xs[t] + b0);
#pragma unroll
    for (int q = 0; q < NQ; q++) sw[q] = *(const float4*)(ws[q] + b0);
    if (b0 + CB < KB) rows.load(wave, b0 + CB, KB, lds + (h ^ 1) * BYTES);   // that half was read before the barrier
#pragma unroll
    for (int i = 0; i < CB; i++) {
      if (b0 + i >= KB) break;
      F8Arg<WIDE> wv[NM];
#pragma unroll
      for (int m = 0; m < NM; m++) wv[m] = F8Arg<WIDE>(f8_op(ring[i % R][m][0], ring[i % R][m][1]));
      const uint8_t* const at = mine + h * BYTES + i * TM * 128;
#pragma unroll
      for (int t = 0; t < TT; t++) {
        const F8Arg<WIDE> xv(f8_op(*(const uint4*)(at + t * 2048 + p0), *(const uint4*)(at + t * 2048 + p1)));
        const float x = i == 0 ? sx[t].x : i == 1 ? sx[t].y : i == 2 ? sx[t].z : sx[t].w;
        f8_v4f d[NM];
#pragma unroll
        for (int m = 0; m < NM; m++) d[m] = f8_mfma(wv[m], xv);
#pragma unroll
        for (int m = 0; m < NM; m++) {
          const float4& q = sw[m % NQ];
          f8_add(acc[m][t], d[m], x * (i == 0 ? q.x : i == 1 ? q.y : i == 2 ? q.z : q.w));
        }
      }
      fetch(i % R, b0 + i + R);
      __builtin_amdgcn_sched_barrier(0);
    }
    if (b0 + CB >= KB) break;
    // a chunk's blocks of weights came after the next rows
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(R * NM * 2) : "memory");
    lds_barrier();
  }
}

// Both operands through LDS: a workgroup of WF WR waves, a wave FT tiles of 16 features and TT of
// 16 rows. A stage is one block of K: the features' tiles as they are stored, the rows (16-byte
// piece j of row r at j ^ r % 8: the rows' pieces would all start on one bank), the rows' scales, the
// features' scales; NS stages are in LDS, all but one of them on their way. They come in by direct
// loads only: a load into a register would wait for the direct ones before it. KS groups of waves
// take the blocks of K in turn, each with stages of its own, and the first gets all sums.
template <int FT, int TT, int WF, int WR, int NS, int KS = 1>
struct F8Core {
  static constexpr int NW = WF * WR, TF = 16 * FT * WF, TR = 16 * TT * WR;
  static constexpr int ROWS = TF * 128, SX = ROWS + TR * 128, SW = SX + (TR * 4 + 255) / 256 * 256, STAGE = SW + 256;
  static constexpr int APW = TF / 8 / NW, BPW = TR / 8 / NW, SPW = (TR / 64 + NW) / NW;   // loads of a wave
  static constexpr int LOADS = APW + BPW + SPW, GROUP = NS * STAGE, BYTES = KS * GROUP;
  static_assert(TF % (8 * NW) == 0 && TR % (8 * NW) == 0 && TR % 64 == 0, "whole loads");
  // where a wave's loads are: the features' tiles from base registers, rows and scales by the lanes'
  // offsets from theirs
  const uint8_t *a[APW], *rows, *xs, *ws;
  uint32_t b[BPW], s[SPW];   // SPW: one wave's or several waves' loads are of the features' scales
  int wave, group, wf, wr;   // wave: of the group
  // tile(i): the stored tiles of the workgroup's i-th 16 features; row(r), scale(r): the offsets of the
  // quantised row r from `rows` and of its scales from `xs`, within 32 bits; fscale(i): the i-th 16
  // features' scales
  template <typename A, typename B, typename S, typename W>
  HX_DEV F8Core(const uint8_t* rows_, const float* xs_, A tile, B row, S scale, W fscale) : rows(rows_), xs((const uint8_t*)xs_) {
    const int all = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    wave = all % NW;
    group = all / NW;
    wf = wave / WR;
    wr = wave % WR;
    const int lane = lane_id();
#pragma unroll
    for (int i = 0; i < APW; i++) {
      const int q = i * NW + wave;
      a[i] = tile(q >> 1) + (q & 1) * 1024;
    }
#pragma unroll
    for (int i = 0; i < BPW; i++) {
      const int r = (i * NW + wave) * 8 + (lane >> 3);
      b[i] = row(r) + ((lane & 7) ^ (r & 7)) * 16;
    }
#pragma unroll
    for (int i = 0; i < SPW; i++) {   // the last waves' loads of rows that are not there go to the features' place
      const int q = i * NW + wave;
      s[i] = q < TR / 64 ? scale(64 * q + lane) : 0u;
    }
    ws = (const uint8_t*)fscale(min(lane, TF / 16 - 1));
  }
  HX_DEV void load(int k, uint32_t lds) const {
#pragma unroll
    for (int i = 0; i < APW; i++) dma16(a[i] + (int64_t)k * 2048, lane_id() * 16, lds + (i * NW + wave) * 1024);
#pragma unroll
    for (int i = 0; i < BPW; i++) dma16(rows + (int64_t)k * 128, b[i], lds + ROWS + (i * NW + wave) * 1024);
#pragma unroll
    for (int i = 0; i < SPW; i++) {
      if (i * NW + wave < TR / 64) dma4(xs + (int64_t)k * 4, s[i], lds + SX + (i * NW + wave) * 256);
      else dma4(ws + (int64_t)k * 4, lds + SW);
    }
  }
  // acc[f][t] = the sums over KB blocks; tile f's scale is that of tile f % NQ of the wave. A tile's
  // products are added to the sums while the next one's run, its codes come while the one before runs
  // (work false: a wave without rows brings its loads only).
  template <bool WIDE, int NQ>
  HX_DEV void run(int KB, uint8_t* buf, bool work, f8_v4f (&acc)[FT][TT]) const {
    static_assert(FT % 2 == 0 && FT % NQ == 0, "pairs of tiles, whole groups of scales");
    uint8_t* const all = buf;
    buf += group * GROUP;
    const uint32_t lds = (uint32_t)(uintptr_t)(lds_u8*)buf;
    const int lane = lane_id(), KG = (KB + KS - 1) / KS;   // blocks of a group; the last may not be there
    f8_v4f d[2][TT];
    float last[TT];
#pragma unroll
    for (int t = 0; t < TT; t++) {
#pragma unroll
      for (int f = 0; f < FT; f++) acc[f][t] = f8_zero4();
      d[1][t] = f8_zero4();
      last[t] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < NS - 1; i++)
      if (i * KS + group < KB) load(i * KS + group, lds + i * STAGE);
    const uint8_t* const x0 = buf + ROWS + (wr * TT * 16 + (lane & 15)) * 128 + ((lane >> 4) ^ (lane & 7)) * 16;
    const uint8_t* const x1 = buf + ROWS + (wr * TT * 16 + (lane & 15)) * 128 + ((4 + (lane >> 4)) ^ (lane & 7)) * 16;
    const uint8_t* const w0 = buf + wf * FT * 2048 + lane * 16;
    const uint8_t* const s0 = buf + SX + (wr * TT * 16 + (lane & 15)) * 4;
    int at = 0;   // the stage of block k
    for (int k = 0; k < KG; k++) {
      // block k has come; after the barrier also the other waves', and the stage before it has been read
      if ((k + NS - 2) * KS + group < KB) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NS - 2) * LOADS) : "memory");
      else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      lds_barrier();
      if ((k + NS - 1) * KS + group < KB) load((k + NS - 1) * KS + group, lds + (at == 0 ? NS - 1 : at - 1) * STAGE);
      const int st = at * STAGE;
      at = at == NS - 1 ? 0 : at + 1;
      if (!work || (KS > 1 && k * KS + group >= KB)) continue;
      auto tile = [&](int f) { return f8_op(*(const uint4*)(w0 + st + f * 2048), *(const uint4*)(w0 + st + f * 2048 + 1024)); };
      f8_v8i w[2];
      w[0] = tile(0);
      F8Arg<WIDE> x[TT];
#pragma unroll
      for (int t = 0; t < TT; t++)
        x[t] = F8Arg<WIDE>(f8_op(*(const uint4*)(x0 + st + t * 2048), *(const uint4*)(x1 + st + t * 2048)));
      float s[NQ][TT];
      const float* const fs = (const float*)(buf + SW + st) + wf * FT;
#pragma unroll
      for (int t = 0; t < TT; t++)
#pragma unroll
        for (int q = 0; q < NQ; q++) s[q][t] = *(const float*)(s0 + st + t * 64) * fs[q];
#pragma unroll
      for (int f = 0; f < FT; f++) {
        if (f + 1 < FT) w[(f + 1) & 1] = tile(f + 1);
        const F8Arg<WIDE> wv(w[f & 1]);
#pragma unroll
        for (int t = 0; t < TT; t++) {
          d[f & 1][t] = f8_mfma(wv, x[t]);
          f8_add(acc[f == 0 ? FT - 1 : f - 1][t], d[(f & 1) ^ 1][t], f == 0 ? last[t] : s[(f - 1) % NQ][t]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int t = 0; t < TT; t++) last[t] = s[(FT - 1) % NQ][t];
    }
#pragma unroll
    for (int t = 0; t < TT; t++) f8_add(acc[FT - 1][t], d[1][t], last[t]);
    if constexpr (KS > 1) {
      static_assert(KS == 2 && NW * FT * TT * 1024 <= BYTES, "the stages' place holds the second group's sums");
      lds_barrier();   // the last stages have been read
      float4* const p = (float4*)all + (size_t)wave * FT * TT * 64 + lane;
      if (group == 1) {
#pragma unroll
        for (int i = 0; i < FT * TT; i++) {
          const f8_v4f& v = acc[i / TT][i % TT];
          p[i * 64] = make_float4(v[0], v[1], v[2], v[3]);
        }
      }
      lds_barrier();
      if (group == 0) {
#pragma unroll
        for (int i = 0; i < FT * TT; i++) {
          const float4 o = p[i * 64];
          f8_v4f& v = acc[i / TT][i % TT];
          v[0] += o.x; v[1] += o.y; v[2] += o.z; v[3] += o.w;
        }
      }
    }
  }
};

// A wave's results, BYTES a row in LDS, to dst(r): whole rows by neighbouring lanes
template <int BYTES>
struct F8Out {
  static constexpr int PITCH = BYTES + 16, PIECES = BYTES / 16;   // 16 bytes more: fewer rows on the same banks
  template <typename F>
  HX_DEV static void store(const uint8_t* tile, int rows, int bytes, F dst) {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
    for (int i = lane_id(); i < rows * PIECES; i += 64) {
      const int r = i / PIECES, b = i % PIECES * 16;
      if (b < bytes) *(uint4*)(dst(r) + b) = *(const uint4*)(tile + r * PITCH + b);
    }
  }
};
HX_DEV uint32_t f8_bf16x2(float a, float b) { return f32_to_bf16(a) | ((uint32_t)f32_to_bf16(b) << 16); }

// workgroup -> (features, rows) of NF x NR tiles: each XCD (workgroup id mod 8) takes an eighth of a
// list that goes through the features four tiles of rows at a time, so that the workgroups that
// run together on an XCD meet each other's operands in its L2
HX_DEV bool f8_place(int NF, int NR, int& nf, int& nr) {
  const int64_t N = (int64_t)NF * NR, per = (N + 7) / 8, i = blockIdx.x >> 3, j = (blockIdx.x & 7) * per + i;
  if (i >= per || j >= N) return false;
  const int g = (int)(j / (4 * NF)), in = (int)(j % (4 * NF)), h = min(4, NR - 4 * g);
  nf = in / h;
  nr = 4 * g + in % h;
  return true;
}

// Linear layer of many rows. Tiles of 256: 8192 rows, 8192 x 4096, 550 GFLOP in 265 to 295 us (1.9 to 2.1
// PFLOP/s by the card; a library product of the same codes with one scale for all takes 223): the
// matrix cores work half of the time, the scales' multiply-adds take half as many cycles as
// the products, and two waves a SIMD, a stage's barrier and its LDS reads leave gaps. Tiles of 64: bound by
// the chain of stages, 0.6 us each, and the launch before: 512 rows, 4096 x 2048, 12 us. Results in bf16 of features that are
// no multiple of 8 leave element by element, 2 bytes each: 8192 rows, 8196 x 4096, 408 us for 282, 512 rows 46 for 32.
template <int FT, int TT, int WF, int WR, int NS, int KS, bool WIDE>
__global__ __launch_bounds__(64 * WF * WR * KS, 2) void k_f8_linear(F8LinearArgs a) {
  typedef F8Core<FT, TT, WF, WR, NS, KS> Core;
  typedef F8Out<32 * FT> Out;
  constexpr int OUT = WIDE ? 0 : WF * WR * 16 * TT * Out::PITCH;
  __shared__ __align__(16) uint8_t buf[Core::BYTES > OUT ? Core::BYTES : OUT];
  static_assert(128 % (16 * FT) == 0, "a wave's features have one scale");
  const int NT = f8_tiles(a.N), KB = f8_blocks(a.K), lane = lane_id();
  int nf, nr;
  if (!f8_place((a.N + Core::TF - 1) / Core::TF, (int)((a.M + Core::TR - 1) / Core::TR), nf, nr)) return;
  const int64_t r0 = (int64_t)nr * Core::TR;
  const int rows = (int)min<int64_t>(Core::TR, a.M - r0), n0 = nf * (Core::TF / 16);
  const float* const ws = (const float*)(a.w + f8_code_bytes(a.N, a.K));
  const Core core(a.xq + r0 * f8_row(a.K), a.xs + r0 * f8_scale_row(a.K),
                  [&](int i) { return a.w + (int64_t)min(n0 + i, NT - 1) * KB * 2048; },
                  [&](int r) { return (uint32_t)(min(r, rows - 1) * f8_row(a.K)); },
                  [&](int r) { return (uint32_t)(min(r, rows - 1) * f8_scale_row(a.K) * 4); },
                  [&](int i) { return ws + (int64_t)(min(n0 + i, NT - 1) >> 3) * f8_scale_row(a.K); });
  f8_v4f acc[FT][TT];
  core.template run<WIDE, 1>(KB, buf, core.wr * TT * 16 < rows, acc);
  const int f0 = 16 * (n0 + core.wf * FT), wr0 = core.wr * TT * 16, wrows = rows - wr0;   // the wave's
  if (!WIDE && a.N % 8 == 0 && ((uintptr_t)a.y & 15) == 0) {
    lds_barrier();   // the last stage has been read (or the second group's sums)
    if (core.group > 0) return;
    uint8_t* const tl = buf + core.wave * (16 * TT * Out::PITCH);
#pragma unroll
    for (int t = 0; t < TT; t++)
#pragma unroll
      for (int f = 0; f < FT; f++) {
        const f8_v4f& v = acc[f][t];
        *(uint2*)(tl + (16 * t + (lane & 15)) * Out::PITCH + 32 * f + 8 * (lane >> 4)) = make_uint2(f8_bf16x2(v[0], v[1]), f8_bf16x2(v[2], v[3]));
      }
    Out::store(tl, min(wrows, 16 * TT), 2 * (a.N - f0),
               [&](int r) { return (uint8_t*)a.y + ((r0 + wr0 + r) * a.N + f0) * 2; });
    return;
  }
  if (core.group > 0) return;
  const bool vec = WIDE && a.N % 4 == 0 && ((uintptr_t)a.y & 15) == 0;
#pragma unroll
  for (int t = 0; t < TT; t++) {
    const int r = 16 * t + (lane & 15);
    if (r >= wrows) continue;
#pragma unroll
    for (int f = 0; f < FT; f++) {
      const int c = f0 + 16 * f + 4 * (lane >> 4);
      const int64_t at = (r0 + wr0 + r) * a.N + c;
      const f8_v4f& v = acc[f][t];
      if (vec) {
        if (c < a.N) *(float4*)((float*)a.y + at) = make_float4(v[0], v[1], v[2], v[3]);
      } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
          if (c + i < a.N) f8_store(a.y, at + i, v[i], !WIDE);
      }
    }
  }
}

template <int FT, int TT, int WF, int WR, int NS, int KS, bool WIDE>
static void f8_linear_tiled(const F8LinearArgs& a, hipStream_t s) {
  typedef F8Core<FT, TT, WF, WR, NS, KS> Core;
  const int64_t n = ((a.N + Core::TF - 1) / Core::TF) * ((a.M + Core::TR - 1) / Core::TR);
  hx_launch(k_f8_linear<FT, TT, WF, WR, NS, KS, WIDE>, dim3((unsigned)((n + 7) / 8 * 8)), dim3(64 * WF * WR * KS), 0, s, a);
}

// Rows that the few-row kernel quantises itself: every workgroup takes about 0.5 us for 16 blocks, a launch for
// it 2 us. us with one and with the other: layers of 4096 x 2048, 2 rows 4.2 and 5.7, 4 rows 5.2 and 6.0, 5 rows
// (80 blocks) 5.7 and 6.1, 6 rows 6.3 and 6.1; 2048 x 4096, 2 rows 6.1 and 6.9, 3 rows 7.2 and 6.9. A tile
// of rows at most.
bool f8_quant_inside(int64_t M, int64_t K) { return M <= 16 && M * f8_blocks(K) <= F8_QUANT_BLOCKS; }
static uint32_t f8_few_lds(int64_t M, int64_t K) { return (uint32_t)(M * (f8_pitch((int)K) + 4 * f8_blocks(K))); }

// The larger a tile, the fewer loads and LDS reads a product takes, if the tiles fill the chip: one
// of 256 x 256 a CU, two of 128 x 128, which take a third of its time. us with tiles of 256, 128, 64
// (quantisation included): 512 rows x 4096 x 2048 48, 19.4, 15.5; 768 rows 37, 21.6, 20.5; 1024 37, 22.5,
// 25.0; 4096 44.9, 47.9, 64; 5000 (320 tiles of 256) 74, 59, 77; 8192 x 4096: 1024 rows 65, 45, 63; 1536
// 67, 70, 89; 2304 128, 102, 131; 8192 281, 319, -. A workgroup of 64 a CU: twice the waves share K. 128 rows x
// 4096 x 2048 11.6 -> 10.5; 512 (2 a CU) 15.5 -> 18.3. Exact products have operands of 16 bits, which leave
// registers for 128 features x 64 rows.
int f8_linear_tile(int64_t M, int64_t N, bool exact) {
  auto tiles = [&](int t) { return ((N + t - 1) / t) * ((M + t - 1) / t); };
  if (exact) return tiles(128) >= 128 ? 128 : 64;
  if (3 * ((tiles(256) + 255) / 256) <= (tiles(128) + 255) / 256) return 256;
  if (tiles(128) >= 224) return 128;
  return tiles(64) > 256 ? 64 : 0;
}

template <bool WIDE>
static hipError_t f8_linear(const F8LinearArgs& a, hipStream_t s) {
  const dim3 few((unsigned)f8_tiles(a.N));
  if (f8_quant_inside(a.M, a.K)) {
    const uint32_t lds = f8_few_lds(a.M, a.K);
    if (a.xbf) hx_launch(k_f8_few_rows<true, 1, true, WIDE>, few, dim3(512), lds, s, a);
    else hx_launch(k_f8_few_rows<false, 1, true, WIDE>, few, dim3(512), lds, s, a);
    return hipGetLastError();
  }
  hipError_t e = launch_f8_rows(a.x, a.xbf, a.M, a.K, a.xq, a.xs, true, s);
  if (e != hipSuccess) return e;
  if (a.M <= 16) hx_launch(k_f8_few_rows<true, 1, false, WIDE>, few, dim3(512), 0, s, a);
  else if (a.M <= 32) hx_launch(k_f8_few_rows<true, 2, false, WIDE>, few, dim3(512), 0, s, a);
  else if (a.M <= F8_FEW_ROWS)   // 33, 40, 48 rows x 4096 x 2048 8.8, 9.3, 9.9 us, by tiles 10.0 to 10.1; x 2048 x 4096 12.1, 13.4, 14.4 and 13.9
    hx_launch(k_f8_few_rows<true, 3, false, WIDE>, few, dim3(512), 0, s, a);
  else {
    switch (f8_linear_tile(a.M, a.N, WIDE)) {
      case 256: if constexpr (!WIDE) f8_linear_tiled<8, 4, 2, 4, 2, 1, WIDE>(a, s); break;
      case 128: f8_linear_tiled<4, WIDE ? 2 : 4, 2, 2, 2, 1, WIDE>(a, s); break;
      case 64: f8_linear_tiled<2, 2, 2, 2, 3, 1, WIDE>(a, s); break;
      default: if constexpr (!WIDE) f8_linear_tiled<2, 2, 2, 2, 3, 2, WIDE>(a, s); break;
    }
  }
  return hipGetLastError();
}
hipError_t launch_f8_linear(const F8LinearArgs& a, hipStream_t s) { return a.ybf ? f8_linear<false>(a, s) : f8_linear<true>(a, s); }

// ---------------------------------------------------------------- experts, few tokens
// Gate/up of up to 16 tokens. Workgroup: a chosen expert (slot) and 8 / KW groups of 16
// features; KW waves share a group's K and add up in LDS. h leaves in f32: its blocks of 128
// are of several workgroups, the down kernels quantise it. ONE token: an expert a chosen entry. QUANT: the
// tokens are quantised into LDS by every workgroup, their expert's weights on their way meanwhile;
// more tokens come quantised. Bound by latency and the weight stream: one token's 23 MB (11 experts of
// 512 x 2048) in 7.9 to 8.2 us, 2.9 TB/s with a launch and the tokens' round trip in it; 4 tokens' 82 MB in 22 us, the load
// units 77 % of the time at work. The products are exact (launch_f8_gate_up).
template <bool BF, int KW, bool ONE, bool QUANT>
__global__ __launch_bounds__(512) void k_f8_few_gate_up(F8Args a) {
  constexpr int FW = 8 / KW;
  extern __shared__ __align__(16) uint8_t sm[];   // QUANT: the tokens' codes, then their scales
  __shared__ MxFewT<ONE ? 1 : F8_FEW_T> few;
  __shared__ float red[8][2][16][17];
  const int tid = threadIdx.x, lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(tid >> 6), T = ONE ? 1 : a.T;
  const int slot = blockIdx.y, fb = blockIdx.x * FW + wave / KW, kq = wave % KW, KB = f8_blocks(a.H), col = lane & 15;
  int e = a.E;
  if (ONE) {
    if (slot < a.k) e = a.idx[slot];
    if (slot < a.k && (unsigned)e >= (unsigned)a.E) return;
  } else {
    mx_few_bits(a, few);
    int n;
    e = mx_few_slot(few, slot, n);
    if (e < 0) {
      if (slot > n || a.Is == 0) {
        if (blockIdx.x == 0 && tid == 0) a.few[slot * MX_FEW_TAB + 32] = -1;
        return;
      }
      e = a.E;
    }
  }
  e = __builtin_amdgcn_readfirstlane(e);
  const bool sh = e == a.E;
  const int inter = sh ? a.Is : a.I;
  if (!ONE && blockIdx.x == 0 && tid < 33)   // for the down kernel
    a.few[slot * MX_FEW_TAB + tid] = tid == 32 ? e : tid < T ? mx_few_row(a, few, e, tid) : -1;
  if (16 * (int)blockIdx.x * FW >= inter) return;
  const bool work = 16 * fb < inter;
  const uint8_t* const mat[2] = {sh ? a.sgate.base : a.gate.mat(e), sh ? a.sup.base : a.up.mat(e)};
  const int64_t at = (int64_t)(work ? fb : 0) * KB * 2048 + lane * 16;
  const int64_t sat = f8_code_bytes(inter, a.H) + (int64_t)((work ? fb : 0) >> 3) * f8_scale_row(a.H) * 4;
  uint4 ring[2][2][2];   // two blocks, gate and up
  float rs[2][2];
  auto fetch = [&](int i, int b) {
    b = min(b, KB - 1);
#pragma unroll
    for (int m = 0; m < 2; m++) {
      const uint8_t* p = mat[m] + at + (int64_t)b * 2048;
      ring[i][m][0] = *(const uint4*)p;
      ring[i][m][1] = *(const uint4*)(p + 1024);
      rs[i][m] = ((const float*)(mat[m] + sat))[b];
    }
  };
  fetch(0, kq);
  fetch(1, kq + KW);
  const int pitch = f8_pitch(a.H);
  float* const qs = (float*)(sm + T * pitch);   // [T][KB]
  if (QUANT) {
    for (int u = 2 * wave + (lane >> 5); u < T * KB; u += 16) {
      const int t = ONE ? 0 : u / KB, b = ONE ? u : u % KB;
      f8_block_to_lds<BF>(a.x, (int64_t)t * a.H, a.H, b, sm + t * pitch + 128 * b, qs + u);
    }
    lds_barrier();
  }
  f8_v4f ag = f8_zero4(), au = f8_zero4();
  const int tok = min(col, T - 1);
  const uint8_t* const row = QUANT ? sm + tok * pitch : a.xrec + tok * f8_row(a.H);
  const float* const xs = QUANT ? qs + tok * KB : a.xs + (int64_t)tok * f8_scale_row(a.H);
  for (int b0 = kq; b0 < KB; b0 += 2 * KW) {
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const int b = b0 + i * KW;
      if (b >= KB) break;
      const float s = xs[b];
      f8_v4f g, u;
      f8_exact_two(f8_op(ring[i][0][0], ring[i][0][1]), f8_op(ring[i][1][0], ring[i][1][1]), f8_operand(row, b), g, u);
      f8_add(ag, g, s * rs[i][0]);
      f8_add(au, u, s * rs[i][1]);
      fetch(i, b + 2 * KW);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; i++) {
    red[wave][0][4 * (lane >> 4) + i][col] = ag[i];
    red[wave][1][4 * (lane >> 4) + i][col] = au[i];
  }
  lds_barrier();
  for (int o = tid; o < FW * 16 * T; o += 512) {
    const int f = o & 15, t = (o >> 4) % T, w0 = (o >> 4) / T * KW, fo = 16 * (blockIdx.x * FW + w0 / KW) + f;
    const int r = ONE ? (sh ? a.F : slot) : mx_few_row(a, few, e, t);
    if (r < 0 || fo >= inter) continue;
    float g = 0.f, u = 0.f;
#pragma unroll
    for (int w = 0; w < KW; w++) {
      g += red[w0 + w][0][f][t];
      u += red[w0 + w][1][f][t];
    }
    a.hf[(int64_t)r * a.hcols + fo] = silu_rcp(g) * u;
  }
}

// most chosen experts of a call (one token: its entries), and the shared one
static int f8_few_slots(const F8Args& a) { return (a.T == 1 ? a.k : std::min(a.T * a.k, a.E)) + (a.Is > 0 ? 1 : 0); }

// Down and combine of one token. Workgroup: 16 outputs; its 16 waves take the entries in turn, 4 blocks
// of K together, half a wave quantises a block of h, each product is weighed in f32, and the waves
// add up in LDS. Bound by latency: 11.5 MB (11 experts, 2048 outputs) in 4.2 to 4.8 us, on 128 workgroups: the entry, its
// weights and h, the sum.
template <bool WIDE>
__global__ __launch_bounds__(1024) void k_f8_one_down(F8Args a) {
  __shared__ float red[16][16];
  __shared__ __align__(16) uint8_t hq[16][4 * 128];
  __shared__ float hs[16][4];
  const int tid = threadIdx.x, lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(tid >> 6), nb = blockIdx.x, k = a.k;
  f8_v4f acc = f8_zero4();
  for (int j = wave; j < k + (a.Is > 0 ? 1 : 0); j += 16) {
    const bool sh = j == k;
    int e = 0;
    if (!sh) e = __builtin_amdgcn_readfirstlane(a.idx[j]);
    if ((unsigned)e >= (unsigned)a.E) continue;
    const float wt = sh ? a.shared_w[0] : a.w[j];
    const int inter = sh ? a.Is : a.I, KB = f8_blocks(inter);
    const uint8_t* mat = sh ? a.sdown.base : a.down.mat(e);
    const uint8_t* w = mat + (int64_t)nb * KB * 2048 + lane * 16;
    const float* ws = (const float*)(mat + f8_code_bytes(a.H, inter)) + (int64_t)(nb >> 3) * f8_scale_row(inter);
    const int64_t row = (int64_t)(sh ? a.F : j) * a.hcols;
    for (int b0 = 0; b0 < KB; b0 += 4) {
      uint4 wq[4][2];
#pragma unroll
      for (int i = 0; i < 4; i++) {   // past the last: the last again
        const uint8_t* p = w + min(b0 + i, KB - 1) * 2048;
        wq[i][0] = *(const uint4*)p;
        wq[i][1] = *(const uint4*)(p + 1024);
      }
      const float4 sw = *(const float4*)(ws + b0);
#pragma unroll 1
      for (int i = lane >> 5; i < 4; i += 2)
        if (b0 + i < KB) f8_block_to_lds<false, true>(a.hf, row, inter, b0 + i, hq[wave] + 128 * i, &hs[wave][i]);
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
#pragma unroll
      for (int i = 0; i < 4; i++) {
        if (b0 + i >= KB) break;
        const float s = hs[wave][i] * (i == 0 ? sw.x : i == 1 ? sw.y : i == 2 ? sw.z : sw.w);
        f8_add(acc, f8_mfma(F8Arg<WIDE>(f8_op(wq[i][0], wq[i][1])), F8Arg<WIDE>(f8_operand(hq[wave], i))), s * wt);
      }
      __builtin_amdgcn_wave_barrier();   // read before the next blocks are written
    }
  }
  if ((lane & 15) == 0) {
#pragma unroll
    for (int i = 0; i < 4; i++) red[wave][4 * (lane >> 4) + i] = acc[i];
  }
  lds_barrier();
  if (tid < 16) {
    float y = 0.f;
#pragma unroll
    for (int w = 0; w < 16; w++) y += red[w][tid];
    mx_store(a, 16 * nb + tid, y);
  }
}

// Outputs of the experts for 2 to 16 tokens, unweighted and in f32, in the row of the token's
// first entry with the expert. Workgroup: a chosen expert (slot) and 128 outputs, 32 a wave; 4 blocks of
// h at a time, quantised into LDS (its workgroups share no block's codes: 16 of 2048 outputs quantise an h of
// 512 each, less than a launch for it). Bound by the weight stream and its start: a workgroup has 64 KB.
template <bool WIDE>
__global__ __launch_bounds__(256) void k_f8_few_down(F8Args a) {
  constexpr int PITCH = 4 * 128 + 16;
  __shared__ __align__(16) uint8_t hq[16 * PITCH];
  __shared__ float hs[16][4];
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int32_t* tab = a.few + blockIdx.y * MX_FEW_TAB;   // k_f8_few_gate_up's
  const int e = tab[32], row = tab[lane & 15];
  if (e < 0) return;
  const bool sh = e == a.E;
  const int inter = sh ? a.Is : a.I, KB = f8_blocks(inter), NT = a.H / 16;
  const int n0 = min(8 * (int)blockIdx.x + 2 * wave, NT - 2);   // past the last: computed, not stored
  const uint8_t* mat = sh ? a.sdown.base : a.down.mat(e);
  const uint8_t* w = mat + (int64_t)n0 * KB * 2048 + lane * 16;
  const float* ws = (const float*)(mat + f8_code_bytes(a.H, inter)) + (int64_t)(n0 >> 3) * f8_scale_row(inter);
  f8_v4f acc[2] = {f8_zero4(), f8_zero4()};
  const unsigned long long rows = __ballot(row >= 0) & 0xffffu;
  for (int b0 = 0; b0 < KB; b0 += 4) {
    uint4 wq[4][2][2];
    float sw[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int b = min(b0 + i, KB - 1);
      sw[i] = ws[b];
#pragma unroll
      for (int m = 0; m < 2; m++) {
        const uint8_t* p = w + ((int64_t)m * KB + b) * 2048;
        wq[i][m][0] = *(const uint4*)p;
        wq[i][m][1] = *(const uint4*)(p + 1024);
      }
    }
    if (b0 > 0) lds_barrier();   // the blocks before have been read
    int c = -1;
    for (unsigned long long left = rows; left; left &= left - 1) {   // half a wave a block of a row
      c = __ffsll(left) - 1;
      const int i = (wave & 1) * 2 + (lane >> 5), r = __shfl(row, c, 64);
      if ((__popcll(rows & ((1ull << c) - 1)) & 1) == (wave >> 1) && b0 + i < KB)
        f8_block_to_lds<false, true>(a.hf, (int64_t)r * a.hcols, inter, b0 + i, hq + c * PITCH + 128 * i, &hs[c][i]);
    }
    lds_barrier();
    const int mine = row >= 0 ? lane & 15 : c;   // a column without a row: any
#pragma unroll
    for (int i = 0; i < 4; i++) {
      if (b0 + i >= KB) break;
      const F8Arg<WIDE> h(f8_operand(hq + mine * PITCH, i));
      const float s = hs[mine][i] * sw[i];
#pragma unroll
      for (int m = 0; m < 2; m++) f8_add(acc[m], f8_mfma(F8Arg<WIDE>(f8_op(wq[i][m][0], wq[i][m][1])), h), s);
    }
  }
  if (row < 0 || 8 * (int)blockIdx.x + 2 * wave >= NT) return;
#pragma unroll
  for (int m = 0; m < 2; m++)
    *(float4*)((float*)a.obuf + (int64_t)row * a.H + 16 * (n0 + m) + 4 * (lane >> 4)) =
        make_float4(acc[m][0], acc[m][1], acc[m][2], acc[m][3]);
}

bool f8_few(int T) { return T <= F8_FEW_T; }

template <bool BF>
static hipError_t f8_few_gate_up(const F8Args& a, hipStream_t s) {
  const int slots = f8_few_slots(a), groups = (std::max(a.I, a.Is) + 15) / 16;
  const bool in = f8_quant_inside(a.T, a.H);
  const uint32_t lds = in ? f8_few_lds(a.T, a.H) : 0;
  // K shared by 8 waves where there are few groups, else by 4: a workgroup's start is shared by more work. us with 8
  // and 4, experts of 512 x 2048: 672 groups 26.5 and 26.0, 1312 41.0 and 35.9, 5152 105.3 and 98.9; of 256 x 2048: 320
  // groups 18.6 and 17.3; of 128 x 2048: 168 groups 15.1 and 15.7, 248 16.4 and 17.1, 328 19.6 and 18.8; of 1024 x
  // 4096, whose K is long: 512 groups 29.0 and 29.0, 1024 41.3 and 42.1.
  const bool few = a.T == 1 || slots * groups < 300;
  const dim3 g(few ? groups : (groups + 1) / 2, slots);
#define FGU(KW, ONE, QUANT) hx_launch(k_f8_few_gate_up<BF, KW, ONE, QUANT>, g, dim3(512), lds, s, a)
  if (a.T == 1 && in) FGU(8, true, true);
  else if (a.T == 1) FGU(8, true, false);
  else if (in && few) FGU(8, false, true);
  else if (in) FGU(4, false, true);
  else if (few) FGU(8, false, false);
  else FGU(4, false, false);
#undef FGU
  return hipGetLastError();
}

hipError_t launch_f8_few_gate_up(const F8Args& a, hipStream_t s) {
  return a.xbf ? f8_few_gate_up<true>(a, s) : f8_few_gate_up<false>(a, s);
}

template <bool WIDE>
static void f8_few_down(const F8Args& a, hipStream_t s) {
  if (a.T == 1) hx_launch(k_f8_one_down<WIDE>, dim3(a.H / 16), dim3(1024), 0, s, a);
  else hx_launch(k_f8_few_down<WIDE>, dim3((a.H + 127) / 128, f8_few_slots(a)), dim3(256), 0, s, a);
}
hipError_t launch_f8_few_down(const F8Args& a, hipStream_t s) {
  if (a.xbf) f8_few_down<false>(a, s);
  else f8_few_down<true>(a, s);
  return hipGetLastError();
}

// ---------------------------------------------------------------- experts, grouped
// Workgroups 0 .. chunks - 1: the chunk's entries by expert (mx_chunk_entries); the others: the
// tokens' rows, a thread 16 values. Bound by the launch (64 tokens of 2048: 6 us), then by HBM: 8192 tokens,
// 50 MB, 13 to 15 us, the entries by expert meanwhile.
template <bool BF>
__global__ __launch_bounds__(256) void k_f8_prep(F8Args a) {
  __shared__ MxPlace sm;
  const int nch = mx_chunks(a.F);
  if ((int)blockIdx.x < nch) {
    mx_chunk_entries(a, sm, nch);
    return;
  }
  const F8Rows q{a.x, a.T, a.H, a.xrec, f8_row(a.H), a.xs, f8_scale_row(a.H)};
  f8_quant_rows<BF>(q, (int64_t)(blockIdx.x - nch) * 256 + threadIdx.x);
}

hipError_t launch_f8_prep(const F8Args& a, hipStream_t s) {
  const dim3 g((unsigned)(((int64_t)a.T * f8_blocks(a.H) * 8 + 255) / 256 + mx_chunks(a.F)));
  if (a.xbf) hx_launch(k_f8_prep<true>, g, dim3(256), 0, s, a);
  else hx_launch(k_f8_prep<false>, g, dim3(256), 0, s, a);
  return hipGetLastError();
}

// Rows of a tile: F entries over all E experts, so that padding and experts without rows count too
// (the routing is on the device). us for 512 experts of 512 x 2048, 10 chosen, with tiles of 32, 64, 128: 64 tokens
// 219, 225, 265; 512 (10 rows an expert) 310, 322, 380; 900 (18) 322, 332, 393; 1024 (20) 329, 333, 394; 2048 (40) 416, 365, 424;
// 3000 (59) 472, 412, 449; 4096 (80) 579, 519, 487; 8192 (160, skewed) 946, 765, 765. (16, by the fp8 instruction: 241 and
// 341 for 64 and 512 tokens.) 128 of 768 x 2048, 8 chosen: 18 rows an expert 129, 131, 150; 24 142, 134, 154; 60 180, 164, 172; 80 216,
// 197, 182. 64 of 1408 x 4096, 6 chosen: 18 212, 217, 246; 24 238, 221, 250; 60 323, 272, 278; 80 359, 337, 294. Small experts, 256 of
// 256 x 1024, 8 chosen, would take smaller ones a little longer: 24 rows 61, 69, 80; 40 74, 74, 85; 80 104, 101, 102. Few wide ones,
// 16 of 2048 x 2048, 2 chosen, larger ones sooner: 40 63, 52, 53; 60 74, 64, 56; 80 76, 68, 59. Tiles of 128 have kernels of their own, which find a token's codes by 32 bits; f32
// results' operands leave room for 32.
int f8_tile_m(int64_t T, int64_t F, int E, int H, bool xbf) {
  if (!xbf || F <= 18 * (int64_t)E) return 32;
  return F <= 68 * (int64_t)E || T * f8_row(H) >= (int64_t)1 << 32 ? 64 : 128;
}

// h = q(silu(G x) * (U x)). Workgroup: a tile of TM rows and 128 features, a block of h's
// columns: 32 a wave (16 where there are 8), gate and up of a feature in the same lane. Bound by the weights' way
// from HBM into the CU: 512 experts of 512 x 2048, 1.07 GB; 64 tokens, 0.69 GB of it, 116 to 126 us (5.5 to
// 5.9 TB/s); 512 tokens 197 us (5.5 TB/s), the load units 96 % of the time at work, the matrix cores 17.
template <int TM, bool WIDE, int NW>
__global__ __launch_bounds__(64 * NW, NW / 2) void k_f8_gate_up(F8Args a) {
  constexpr int TT = TM / 16, NF = 8 / NW, NM = 2 * NF;   // NF: a wave's tiles of features
  __shared__ __align__(16) uint8_t buf[2 * F8Tile<TM, NW>::BYTES];
  __shared__ uint32_t amax[NW][TM];
  int nt, tile;
  mx_tile(a.hblocks, a.counts[0], nt, tile);
  if (tile < 0) return;
  const int4 ti = ((const int4*)a.tiles)[tile];
  const int e = __builtin_amdgcn_readfirstlane(ti.x), p0 = ti.y, rows = ti.z;
  const bool sh = e == a.E;
  const int inter = sh ? a.Is : a.I;
  if (128 * nt >= inter) return;
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), KB = f8_blocks(a.H);
  auto token = [&](int r) {
    const int p = p0 + min(r, rows - 1);
    return (int64_t)(sh ? p - a.F : a.perm[p] / a.k);
  };
  F8Tile<TM, NW> rw;
  rw.init(wave, [&](int r) { return a.xrec + token(r) * f8_row(a.H); });
  const float* xs[TT];
#pragma unroll
  for (int t = 0; t < TT; t++) xs[t] = a.xs + token(16 * t + (lane & 15)) * f8_scale_row(a.H);
  const uint8_t* const mat[2] = {sh ? a.sgate.base : a.gate.mat(e), sh ? a.sup.base : a.up.mat(e)};
  const uint8_t* w[NM];   // gate, up of each
#pragma unroll
  for (int m = 0; m < NM; m++)
    w[m] = mat[m & 1] + (int64_t)min(8 * nt + NF * wave + (m >> 1), inter / 16 - 1) * KB * 2048 + lane * 16;
  const int64_t sat = f8_code_bytes(inter, a.H) + (int64_t)nt * f8_scale_row(a.H) * 4;
  const float* const ws[2] = {(const float*)(mat[0] + sat), (const float*)(mat[1] + sat)};
  f8_v4f acc[NM][TT];
  f8_products<WIDE, TM, NW, NM, 2>(w, ws, rw, xs, wave, buf, KB, acc);
  float h[TT][4 * NF];
#pragma unroll
  for (int t = 0; t < TT; t++) {
#pragma unroll
    for (int f = 0; f < NF; f++) {
      const bool in = 128 * nt + 16 * (NF * wave + f) < inter;   // features behind the last are zeros
#pragma unroll
      for (int i = 0; i < 4; i++) h[t][4 * f + i] = in ? silu_rcp(acc[2 * f][t][i]) * acc[2 * f + 1][t][i] : 0.f;
    }
    const uint32_t m = f8_max_of_4(f8_amax(h[t]));
    if (lane < 16) amax[wave][16 * t + lane] = m;
  }
  lds_barrier();
#pragma unroll
  for (int t = 0; t < TT; t++) {
    const int r = 16 * t + (lane & 15);
    uint32_t m = 0;
#pragma unroll
    for (int v = 0; v < NW; v++) m = max(m, amax[v][r]);
    float s;
    const bool fine = f8_scale(m, s);
    uint32_t c[NF];
    f8_codes_near(h[t], s, fine, c);
    if (r >= rows) continue;
    uint32_t* o = (uint32_t*)(a.hrec + ((int64_t)(p0 + r) * a.hblocks + nt) * 128 + 16 * NF * wave + 4 * (lane >> 4));
#pragma unroll
    for (int f = 0; f < NF; f++) o[4 * f] = c[f];
    if (wave == 0 && lane < 16) a.hs[(int64_t)(p0 + r) * a.hscale + nt] = s;
  }
}

// A wave's outputs of NM tiles from n0 for rows p0 .. of obuf: f16 with a scale for each 32, a power of
// two that gives the largest finite magnitude of the row's outputs here the exponent 2^14 (infinities and
// NaN stay what they are)
template <int NM, int TT>
HX_DEV void f8_out_rows(const F8Args& a, const f8_v4f (&acc)[NM][TT], uint8_t* tl, int64_t p0, int rows, int n0) {
  static_assert(NM % 2 == 0, "32 outputs have a scale");
  typedef F8Out<32 * NM> Out;
  const int lane = lane_id(), tiles = a.H / 16;
#pragma unroll
  for (int t = 0; t < TT; t++) {
    uint32_t top = 0;
#pragma unroll
    for (int m = 0; m < NM; m++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const uint32_t u = __float_as_uint(acc[m][t][i]) & 0x7fffffffu;
        top = max(top, n0 + m < tiles && u < 0x7f800000u ? u : 0u);
      }
    const int ex = max((int)(f8_max_of_4(top) >> 23), 15), r = 16 * t + (lane & 15);
    const float up = __uint_as_float((uint32_t)(268 - ex) << 23);
#pragma unroll
    for (int m = 0; m < NM; m++) {
      uint32_t h[2];
#pragma unroll
      for (int i = 0; i < 2; i++) {
        const _Float16 lo = (_Float16)(acc[m][t][2 * i] * up), hi = (_Float16)(acc[m][t][2 * i + 1] * up);
        h[i] = (uint32_t)__builtin_bit_cast(uint16_t, lo) | ((uint32_t)__builtin_bit_cast(uint16_t, hi) << 16);
      }
      *(uint2*)(tl + r * Out::PITCH + 32 * m + 8 * (lane >> 4)) = make_uint2(h[0], h[1]);
    }
    if (lane < 16 && r < rows)
#pragma unroll
      for (int m = 0; m < NM; m += 2)
        if (n0 + m < tiles) a.oscale[(p0 + r) * (a.H / 32) + ((n0 + m) >> 1)] = __uint_as_float((uint32_t)(ex - 14) << 23);
  }
  Out::store(tl, min(rows, 16 * TT), 2 * (a.H - 16 * n0), [&](int r) { return (uint8_t*)a.obuf + ((p0 + r) * a.H + 16 * n0) * 2; });
}

// Outputs of the experts, unweighted: D h. Workgroup: a tile of TM rows and 256 outputs. Bound as
// gate/up: 512 tokens, 0.54 GB, in 107 us (5 TB/s); 64 tokens 61 to 65 us. bf16 activations: outputs leave
// as f16 with a scale for each 32, off by 2^-11 of a value at most (or, where that is more, 2^-39 of the power of two
// below the largest that it shares the scale with) for half of the bytes that float32 takes here and in the
// combine (bf16, 2^-8, would be the result's own error once more).
template <int TM, bool WIDE, int NW>
__global__ __launch_bounds__(64 * NW, NW / 2) void k_f8_down(F8Args a) {
  constexpr int TT = TM / 16, NM = 16 / NW;
  __shared__ __align__(16) uint8_t buf[2 * F8Tile<TM, NW>::BYTES];
  int nt, tile;
  mx_tile((a.H + 255) / 256, a.counts[0], nt, tile);
  if (tile < 0) return;
  const int4 ti = ((const int4*)a.tiles)[tile];
  const int e = __builtin_amdgcn_readfirstlane(ti.x), p0 = ti.y, rows = ti.z;
  const bool sh = e == a.E;
  const int inter = sh ? a.Is : a.I, KB = f8_blocks(inter), tiles = a.H / 16;
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n0 = 16 * nt + wave * NM;
  F8Tile<TM, NW> rw;
  rw.init(wave, [&](int r) { return a.hrec + (int64_t)(p0 + min(r, rows - 1)) * a.hblocks * 128; });
  const float* xs[TT];
#pragma unroll
  for (int t = 0; t < TT; t++) xs[t] = a.hs + (int64_t)(p0 + min(16 * t + (lane & 15), rows - 1)) * a.hscale;
  const uint8_t* mat = sh ? a.sdown.base : a.down.mat(e);
  const uint8_t* w[NM];
#pragma unroll
  for (int m = 0; m < NM; m++) w[m] = mat + (int64_t)min(n0 + m, tiles - 1) * KB * 2048 + lane * 16;   // past the last: not stored
  const float* const ws[1] = {(const float*)(mat + f8_code_bytes(a.H, inter)) + (int64_t)(min(n0, tiles - 1) >> 3) * f8_scale_row(inter)};
  f8_v4f acc[NM][TT];
  f8_products<WIDE, TM, NW, NM, 1>(w, ws, rw, xs, wave, buf, KB, acc);
  if constexpr (WIDE) {
#pragma unroll
    for (int t = 0; t < TT; t++) {
      const int r = 16 * t + (lane & 15);
      if (r >= rows) continue;
#pragma unroll
      for (int m = 0; m < NM; m++) {
        if (n0 + m >= tiles) continue;
        const f8_v4f& v = acc[m][t];
        *(float4*)((float*)a.obuf + (int64_t)(p0 + r) * a.H + 16 * (n0 + m) + 4 * (lane >> 4)) = make_float4(v[0], v[1], v[2], v[3]);
      }
    }
  } else {
    static_assert(NW * TM * F8Out<32 * NM>::PITCH <= 2 * F8Tile<TM, NW>::BYTES, "the rows' place holds the results");
    lds_barrier();   // the rows have been read
    f8_out_rows<NM, TT>(a, acc, buf + wave * (TM * F8Out<32 * NM>::PITCH), p0, rows, n0);
  }
}

// The same two products where experts have many rows: both operands through LDS (F8Core), tiles of
// 128 rows; the waves of a tile's second half bring loads only where it has 64 rows or fewer. Bound by the
// loads' latency at two waves a SIMD, with a barrier a stage: 8192 tokens, ten experts each, gate/up 378 GFLOP in 353 us, 441 where
// the routing is skewed (1 PFLOP/s; the load units 73 % at work, the matrix cores 28 %), down 189 GFLOP in 267 and 317 us (87 %, 17 %:
// K is four stages, each output leaves with 2 bytes and the rows' 0.39 GB are written).
__global__ __launch_bounds__(512, 2) void k_f8_gate_up_many(F8Args a) {
  typedef F8Core<4, 4, 4, 2, 2> Core;
  constexpr int TT = 4, TR = Core::TR, PITCH = 128 + 16;
  static_assert(TR * PITCH <= Core::BYTES, "the stages' place holds the results");
  __shared__ __align__(16) uint8_t buf[Core::BYTES];
  __shared__ uint32_t amax[4][TR];
  int nt, tile;
  mx_tile(a.hblocks, a.counts[0], nt, tile);
  if (tile < 0) return;
  const int4 ti = ((const int4*)a.tiles)[tile];
  const int e = __builtin_amdgcn_readfirstlane(ti.x), p0 = ti.y, rows = ti.z;
  const bool sh = e == a.E;
  const int inter = sh ? a.Is : a.I;
  if (128 * nt >= inter) return;
  const int lane = lane_id(), KB = f8_blocks(a.H);
  auto token = [&](int r) {
    const int p = p0 + min(r, rows - 1);
    return sh ? p - a.F : a.perm[p] / a.k;
  };
  const uint8_t* const gm = sh ? a.sgate.base : a.gate.mat(e);
  const uint8_t* const um = sh ? a.sup.base : a.up.mat(e);
  const int64_t sat = f8_code_bytes(inter, a.H) + (int64_t)nt * f8_scale_row(a.H) * 4;
  // a wave's tiles: gate, up, gate, up of its 32 features
  const Core core(a.xrec, a.xs,
                  [&](int i) { return (i & 1 ? um : gm) + (int64_t)min(8 * nt + (i >> 1), inter / 16 - 1) * KB * 2048; },
                  [&](int r) { return (uint32_t)(token(r) * (uint32_t)f8_row(a.H)); },
                  [&](int r) { return (uint32_t)(token(r) * (uint32_t)f8_scale_row(a.H) * 4); },
                  [&](int i) { return (const float*)((i & 1 ? um : gm) + sat); });
  f8_v4f acc[4][TT];
  const int r0 = core.wr * 64;   // the wave's first row
  const bool work = r0 < rows;
  core.run<false, 2>(KB, buf, work, acc);
  const bool in = 128 * nt + 32 * core.wf < inter;   // features behind the last are zeros
  float h[TT][8];
#pragma unroll
  for (int t = 0; t < TT; t++) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const int m = 2 * (i >> 2);
      h[t][i] = in ? silu_rcp(acc[m][t][i & 3]) * acc[m + 1][t][i & 3] : 0.f;
    }
    const uint32_t m = f8_max_of_4(f8_amax(h[t]));
    if (lane < 16) amax[core.wf][r0 + 16 * t + lane] = m;
  }
  lds_barrier();   // the last stage has been read, too
  if (work) {
#pragma unroll
    for (int t = 0; t < TT; t++) {
      const int r = r0 + 16 * t + (lane & 15);
      float s;
      const bool fine = f8_scale(max(max(amax[0][r], amax[1][r]), max(amax[2][r], amax[3][r])), s);
      uint32_t c[2];
      f8_codes_near(h[t], s, fine, c);
      uint8_t* const o = buf + r * PITCH + 32 * core.wf + 4 * (lane >> 4);
      *(uint32_t*)o = c[0];
      *(uint32_t*)(o + 16) = c[1];
      if (core.wf == 0 && lane < 16 && r < rows) a.hs[(int64_t)(p0 + r) * a.hscale + nt] = s;
    }
  }
  lds_barrier();
  for (int i = threadIdx.x; i < rows * 8; i += 512)
    *(uint4*)(a.hrec + ((int64_t)(p0 + (i >> 3)) * a.hblocks + nt) * 128 + (i & 7) * 16) = *(const uint4*)(buf + (i >> 3) * PITCH + (i & 7) * 16);
}

__global__ __launch_bounds__(256, 2) void k_f8_down_many(F8Args a) {
  typedef F8Core<4, 4, 2, 2, 2> Core;
  __shared__ __align__(16) uint8_t buf[Core::BYTES];
  int nt, tile;
  mx_tile((a.H + 127) / 128, a.counts[0], nt, tile);
  if (tile < 0) return;
  const int4 ti = ((const int4*)a.tiles)[tile];
  const int e = __builtin_amdgcn_readfirstlane(ti.x), p0 = ti.y, rows = ti.z;
  const bool sh = e == a.E;
  const int inter = sh ? a.Is : a.I, KB = f8_blocks(inter), tiles = a.H / 16;
  const uint8_t* const mat = sh ? a.sdown.base : a.down.mat(e);
  const float* const ws = (const float*)(mat + f8_code_bytes(a.H, inter)) + (int64_t)nt * f8_scale_row(inter);
  const Core core(a.hrec + (int64_t)p0 * a.hblocks * 128, a.hs + (int64_t)p0 * a.hscale,
                  [&](int i) { return mat + (int64_t)min(8 * nt + i, tiles - 1) * KB * 2048; },
                  [&](int r) { return (uint32_t)(min(r, rows - 1) * a.hblocks * 128); },
                  [&](int r) { return (uint32_t)(min(r, rows - 1) * a.hscale * 4); }, [&](int) { return ws; });
  f8_v4f acc[4][4];
  const int r0 = core.wr * 64;
  core.run<false, 1>(KB, buf, r0 < rows, acc);
  lds_barrier();   // the last stage has been read
  f8_out_rows<4, 4>(a, acc, buf + core.wave * (64 * F8Out<128>::PITCH), p0 + r0, rows - r0, 8 * nt + 4 * core.wf);
}

// workgroups for the tiles of a call, nx for each
static dim3 f8_grid(const F8Args& a, int nx) { return dim3((unsigned)((int64_t)nx * ((a.max_tiles + 7) / 8 * 8))); }

// Gate/up's products are exact for few tokens and with tiles of 32 rows, whichever the activations' type: what the
// fp8 instruction drops moves some of h's codes to a neighbour, and so the outputs by another 1.0e-3 to 2.5e-3 of their
// norm, as much as bf16's own rounding (1.7e-3). us of a call by the fp8 instruction and exact: 1 token 13.0 and 13.4, 4
// 35.2 and 35.7, 16 97.9 and 98.8, 64 219.1 and 217.7, 512 311.2 and 310.4, 900 325.1 and 322.7. With larger tiles it stays with the
// fp8 instruction, which is off by 1.3e-3 there: exact sums cost 12 to 15 % (1024 tokens 332 and 383, 2048 365 and
// 410, 8192 762 and 866).
hipError_t launch_f8_gate_up(const F8Args& a, hipStream_t s) {
  const dim3 g = f8_grid(a, a.hblocks);
  if (a.tile_m == 32) hx_launch(k_f8_gate_up<32, true, 4>, g, dim3(256), 0, s, a);
  else if (a.tile_m == 64) hx_launch(k_f8_gate_up<64, false, 8>, g, dim3(512), 0, s, a);
  else hx_launch(k_f8_gate_up_many, g, dim3(512), 0, s, a);
  return hipGetLastError();
}
hipError_t launch_f8_down(const F8Args& a, hipStream_t s) {
  const dim3 g = f8_grid(a, (a.H + 255) / 256);
  if (!a.xbf) hx_launch(k_f8_down<32, true, 4>, g, dim3(256), 0, s, a);
  else if (a.tile_m == 32) hx_launch(k_f8_down<32, false, 4>, g, dim3(256), 0, s, a);
  else if (a.tile_m == 64) hx_launch(k_f8_down<64, false, 8>, g, dim3(512), 0, s, a);
  else hx_launch(k_f8_down_many, f8_grid(a, (a.H + 127) / 128), dim3(256), 0, s, a);
  return hipGetLastError();
}

}  // namespace hx
