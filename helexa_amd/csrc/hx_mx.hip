// Experts on MXFP4 weights: y[t] = sum_j w[t,j] D_e(silu(G_e x_t) * U_e x_t) with
// e = idx[t,j], plus shared_w[t] times the shared expert's, for a routing the caller
// has or hx_moe_forward's router makes.
//
// Both products run on v_mfma_scale_f32_32x32x64_f8f6f4 with the weights as its A
// operand, their stored codes and scales untouched, and the activations as its B
// operand, cut into E2M3 planes (hx_mx.h). D then holds a token's outputs in a
// column: lane l token l % 32, rows 8 (i / 4) + 4 (l / 32) + i % 4 in register i, so
// that lanes l and l + 32 hold the 32 features of one token that make one record of
// the next product, or 64 bytes of its row.
//
// A few tokens (mx_few): gate/up with a workgroup per expert and 8 / KW groups of 32
// features, then one token's down, which combines, or down with a workgroup per expert and
// 128 outputs, and the combine. More: the tokens' records and the expert counts, the
// dispatch, grouped products over tiles of tile_m rows, and the combine.
#include "hx_mx_routing.h"

#include <type_traits>

namespace hx {

typedef int mx_v8i __attribute__((ext_vector_type(8)));
typedef uint32_t mx_v4u __attribute__((ext_vector_type(4)));
typedef uint32_t mx_v6u __attribute__((ext_vector_type(6)));
typedef float mx_v16f __attribute__((ext_vector_type(16)));
typedef float mx_v32f __attribute__((ext_vector_type(32)));

// ---------------------------------------------------------------- stored weights
// MXFP4 rows -> the layout of hx_mx.h: a thread per lane of a tile, padding included
__global__ __launch_bounds__(256) void k_repack_mx(const uint8_t* src, int64_t count, int rows, int K, uint8_t* dst,
                                                   int64_t dst_stride) {
  const int S = mx_steps(K), S4 = (S + 3) / 4, NB = K / 32;
  const int64_t per = (int64_t)(rows / 32) * S4 * 4 * 64;
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= per * count) return;
  const int64_t m = id / per;
  const int64_t q = id % per;
  const int l = (int)(q & 63), s = (int)((q >> 6) % (S4 * 4)), n = (int)((q >> 6) / (S4 * 4));
  const int row = 32 * n + (l & 31), kb = 2 * s + (l >> 5);
  uint4 c = make_uint4(0u, 0u, 0u, 0u);
  uint8_t e = 127;
  if (kb < NB) {
    const uint8_t* b = src + ((m * rows + row) * NB + kb) * 17;   // the caller's rows: any alignment
    e = b[0];
    uint32_t o[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int j = 0; j < 16; j++) {
      const uint32_t v = b[1 + j];
      o[j >> 3] |= (v & 15u) << (4 * (j & 7));
      o[2 + (j >> 3)] |= (v >> 4) << (4 * (j & 7));
    }
    c = make_uint4(o[0], o[1], o[2], o[3]);
  }
  uint8_t* mat = dst + m * dst_stride;
  if (s < S) *(uint4*)(mat + (((int64_t)n * S + s) * 64 + l) * 16) = c;
  mat[mx_code_bytes(rows, K) + (((int64_t)n * S4 + s / 4) * 64 + l) * 4 + (s & 3)] = e;
}

hipError_t launch_mx_repack(const void* src, int64_t count, int64_t rows, int64_t K, void* dst, int64_t dst_stride,
                            hipStream_t s) {
  const int64_t n = count * (rows / 32) * ((mx_steps((int)K) + 3) / 4) * 256;
  hipLaunchKernelGGL(k_repack_mx, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, (const uint8_t*)src, count,
                     (int)rows, (int)K, (uint8_t*)dst, dst_stride);
  return hipGetLastError();
}

// ---------------------------------------------------------------- records
template <int P>
struct MxRec {
  static constexpr int BYTES = P == 3 ? 80 : 128, VECS = BYTES / 16, SCALE = 6 * P;   // words: codes, then scales
};

// 32 values -> the words of their record
template <int P>
HX_DEV void mx_record(const float (&f)[32], uint4 (&out)[MxRec<P>::VECS]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 32; i++) m = max(m, __float_as_uint(f[i]) & 0x7fffffffu);
  const int e = (int)(m >> 23);
  const bool bad = e == 255;
  // the first scale's exponent byte; at least so much that the last plane's is 1, a
  // normal float for the conversions: 2^-126, in steps of 2^-129. Blocks of a largest
  // magnitude below 2^-116 (three planes; five: 2^-106) lose what is under 2^-130.
  const int sb = bad ? 127 : max(e - 2, 5 * (P - 1) - 1);
  uint32_t w[4 * MxRec<P>::VECS];
#pragma unroll
  for (int i = 0; i < 4 * MxRec<P>::VECS; i++) w[i] = 0;
  mx_v16f ev, od;   // the conversion takes the even and the odd elements; whatever codes a bad block gets
#pragma unroll
  for (int i = 0; i < 16; i++) {
    ev[i] = f[2 * i];
    od[i] = f[2 * i + 1];
  }
#pragma unroll
  for (int p = 0; p < P; p++) {
    const int b = sb - (p == 0 ? 0 : 5 * p - 2);
    const float sc = __uint_as_float((uint32_t)b << 23);
    mx_v6u c = __builtin_amdgcn_cvt_scalef32_2xpk16_fp6_f32(ev, od, sc);
    // these conversions write their first results before they have read all their
    // sources, and the compiler may give both the same registers: the sources are
    // kept alive past them
    asm volatile("" : "+v"(c) : "v"(ev), "v"(od), "v"(sc));
#pragma unroll
    for (int i = 0; i < 6; i++) w[i < 4 ? 4 * p + i : 4 * P + 2 * p + i - 4] = c[i];
    if (p + 1 < P) {
      mx_v32f v = __builtin_amdgcn_cvt_scalef32_pk32_f32_fp6(c, sc);
      asm volatile("" : "+v"(v) : "v"(c), "v"(sc));
#pragma unroll
      for (int i = 0; i < 16; i++) {
        ev[i] -= v[2 * i];
        od[i] -= v[2 * i + 1];
      }
    }
    w[MxRec<P>::SCALE + p / 4] |= (uint32_t)(bad ? 255 : b) << (8 * (p & 3));
  }
#pragma unroll
  for (int i = 0; i < MxRec<P>::VECS; i++) out[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
}

// the record of 32 zeros
template <int P>
HX_DEV void mx_zero_record(uint4 (&out)[MxRec<P>::VECS]) {
#pragma unroll
  for (int i = 0; i < MxRec<P>::VECS; i++) out[i] = make_uint4(0u, 0u, 0u, 0u);
  // by components: a store through a pointer to words puts the record into scratch memory
  constexpr int V = MxRec<P>::SCALE / 4;
  static_assert(MxRec<P>::SCALE % 4 == 2, "the scales' words are .z and .w");
  out[V].z = 0x7f7f7f7fu;
  if (P > 4) out[V].w = 0x7f7f7f7fu;
}

// block kb of token row x (H columns) -> its record; blocks past the row are zeros
template <int P>
HX_DEV void mx_token_record(const void* x, int64_t t, int H, int kb, uint4 (&out)[MxRec<P>::VECS]) {
  if (32 * kb >= H) {
    mx_zero_record<P>(out);
    return;
  }
  float f[32];
  if constexpr (P == 3) {
    const uint16_t* p = (const uint16_t*)x + t * H + 32 * kb;
    if (((uintptr_t)p & 15) == 0) {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const uint4 v = ((const uint4*)p)[i];
        const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 4; j++) {
          f[8 * i + 2 * j] = __uint_as_float(u[j] << 16);
          f[8 * i + 2 * j + 1] = __uint_as_float(u[j] & 0xffff0000u);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 32; i++) f[i] = bf16_to_f32(p[i]);
    }
  } else {
    const float* p = (const float*)x + t * H + 32 * kb;
    if (((uintptr_t)p & 15) == 0) {
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const float4 v = ((const float4*)p)[i];
        f[4 * i] = v.x; f[4 * i + 1] = v.y; f[4 * i + 2] = v.z; f[4 * i + 3] = v.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 32; i++) f[i] = p[i];
    }
  }
  mx_record<P>(f, out);
}

// a plane of a record as the MFMA takes it: 6 words in a row
typedef int mx_v6i __attribute__((ext_vector_type(6)));
template <int P>
HX_DEV mx_v6i mx_plane(const uint8_t* rec, int p) {
  const uint4 a = *(const uint4*)(rec + 16 * p);
  const uint2 b = *(const uint2*)(rec + 16 * P + 8 * p);
  return mx_v6i{(int)a.x, (int)a.y, (int)a.z, (int)a.w, (int)b.x, (int)b.y};
}

// a record's planes and scales as MFMA operands
template <int P>
struct MxB {
  mx_v6i w[P];
  uint32_t sc[(P + 3) / 4];
  HX_DEV void load(const uint8_t* rec) {
#pragma unroll
    for (int p = 0; p < P; p++) w[p] = mx_plane<P>(rec, p);
#pragma unroll
    for (int i = 0; i < (P + 3) / 4; i++) sc[i] = *(const uint32_t*)(rec + 24 * P + 4 * i);
  }
  // a record of 128 bytes whose 16-byte piece j lies at j ^ x
  HX_DEV void load_swizzled(const uint8_t* rec, int x) {
    auto at = [&](int byte) { return rec + ((byte & ~15) ^ (16 * x)) + (byte & 15); };
#pragma unroll
    for (int p = 0; p < P; p++) {
      const uint4 a = *(const uint4*)at(16 * p);
      const uint2 b = *(const uint2*)at(16 * P + 8 * p);
      w[p] = mx_v6i{(int)a.x, (int)a.y, (int)a.z, (int)a.w, (int)b.x, (int)b.y};
    }
    const uint2 q = *(const uint2*)at(24 * P);
    sc[0] = q.x;
    sc[(P - 1) / 4] = q.y;
  }
};

// c[m][n] += weights m (one step's codes, their scale in byte SA of sc[m]) x the planes
// of b; plane by plane, so that neighbouring MFMAs do not wait for each other
template <int P, int SA, int NM, int NC>
HX_DEV void mx_mfma(const mx_v4u (&w)[NM], const uint32_t (&sc)[NM], const MxB<P>& b, mx_v16f (&c)[NM][NC], int n) {
#define MX_PLANE(p)                                                                                               \
  if constexpr (p < P) {                                                                                          \
    const mx_v8i bv = {b.w[p][0], b.w[p][1], b.w[p][2], b.w[p][3], b.w[p][4], b.w[p][5], 0, 0};                   \
    _Pragma("unroll") for (int m = 0; m < NM; m++) {                                                              \
      const mx_v8i av = {(int)w[m].x, (int)w[m].y, (int)w[m].z, (int)w[m].w, 0, 0, 0, 0};                         \
      c[m][n] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(av, bv, c[m][n], 4, 2, SA, (int)sc[m], (p) & 3,   \
                                                                (int)b.sc[(p) / 4]);                              \
    }                                                                                                             \
  }
  MX_PLANE(0) MX_PLANE(1) MX_PLANE(2) MX_PLANE(3) MX_PLANE(4)
#undef MX_PLANE
}

// One plane of a record as an MFMA operand. Where few rows meet the weights, their
// planes are columns of their own (column p n + r: plane p of row r, n rows), one
// MFMA does what takes P with the planes one after the other, and the columns of a
// row are added at the end.
struct MxPlane {
  mx_v6i w;
  uint32_t sc;
  HX_DEV void zero() {
    w = mx_v6i{0, 0, 0, 0, 0, 0};
    sc = 127u;
  }
  template <int P>
  HX_DEV void load(const uint8_t* rec, int p) {
    w = mx_plane<P>(rec, p);
    sc = rec[24 * P + p];
  }
};
template <int SA>
HX_DEV mx_v16f mx_mfma1(const uint4& a, uint32_t sa, const MxPlane& b, mx_v16f c) {
  const mx_v8i av = {(int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0};
  const mx_v8i bv = {b.w[0], b.w[1], b.w[2], b.w[3], b.w[4], b.w[5], 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(av, bv, c, 4, 2, SA, (int)sa, 0, (int)b.sc);
}

HX_DEV mx_v16f mx_zero16() {
  mx_v16f z;
#pragma unroll
  for (int i = 0; i < 16; i++) z[i] = 0.f;
  return z;
}

// silu(g) u, the division by v_rcp_f32 (1 ulp)
HX_DEV float mx_swiglu(float g, float u) { return silu_rcp(g) * u; }

// ---------------------------------------------------------------- few tokens
// steps of K a wave takes where W waves share them: 1, 2 or whole words of scales
__host__ __device__ inline int mx_wave_steps(int S, int W) {
  const int c = (S + W - 1) / W;
  return c <= 1 ? 1 : c == 2 ? 2 : (c + 3) / 4 * 4;
}

// Gate/up of up to 8 tokens. Workgroup: a chosen expert (slot) and 8 / KW groups of 32
// features; KW waves share a group's K and add up in LDS. The tokens' records are
// made in LDS by every workgroup: a kernel of their own would cost a launch (about 4 us).
// The planes are columns: with them one after the other the products alone took 8 us of
// 6 tokens' call.
// ONE token: an expert a chosen entry, its weights on their way before anything else.
// Bound by latency and the weight stream: the routing, the experts' addresses, the weights
// in flight, two sums through LDS. H 2048, I 512, 10 of 512 experts, bf16: one token's 12 MB
// in 6.7 us, 6 tokens' 64 MB in 17.5 (3.7 TB/s), 8 tokens' 85 MB in 21.8 (3.9); five planes
// 7.7 for one token, 17.1 for 5.
template <int P, int KW, bool ONE>
__global__ __launch_bounds__(512, ONE || P == 5 ? 2 : 4) void k_mx_few_gate_up(MxArgs a) {
  constexpr int RB = MxRec<P>::BYTES, RV = MxRec<P>::VECS, FW = 8 / KW;
  extern __shared__ __align__(16) uint8_t sm[];
  __shared__ MxFewT<MX_FEW_T> few;
  const int tid = threadIdx.x, lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(tid >> 6), T = ONE ? 1 : a.T;
  const int slot = blockIdx.y, fb = blockIdx.x * FW + wave / KW, kq = wave % KW;
  const int S = mx_steps(a.H), S4 = (S + 3) / 4, HB = mx_blocks(a.H);
  const int c = mx_wave_steps(S, KW), s0 = kq * c, s1 = min(S, s0 + c);
  int e = a.E, inter = a.Is;
  int64_t at = 0, sat = 0;
  const uint8_t *gm = nullptr, *um = nullptr;
  bool work = false;
  // four steps of weights are on their way at any time
  uint4 wg[4], wu[4];
  auto fetch = [&](int s, int i) {
    wg[i] = *(const uint4*)(gm + (at + s * 1024) + lane * 16);
    wu[i] = *(const uint4*)(um + (at + s * 1024) + lane * 16);
  };
  uint32_t sg, su;
  auto fetch_scales = [&](int s) {
    sg = *(const uint32_t*)(gm + (sat + (s >> 2) * 256) + lane * 4);
    su = *(const uint32_t*)(um + (sat + (s >> 2) * 256) + lane * 4);
  };
  // the slot's expert is known: its weights
  auto start = [&]() {
    e = __builtin_amdgcn_readfirstlane(e);
    const bool sh = e == a.E;
    inter = sh ? a.Is : a.I;
    gm = sh ? a.sgate.base : a.gate.mat(e);
    um = sh ? a.sup.base : a.up.mat(e);
    at = (int64_t)fb * S * 1024;
    sat = mx_code_bytes(inter, a.H) + (int64_t)fb * S4 * 256;
    work = 32 * fb < inter && s0 < s1;   // the others: a record behind the last feature, or none
    if (!work) return;
    fetch_scales(s0);
#pragma unroll
    for (int i = 0; i < 4; i++) fetch(min(s0 + i, s1 - 1), i);
  };
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
  start();
  if (!ONE && blockIdx.x == 0 && tid < 33)   // for the down kernel
    a.few[slot * MX_FEW_TAB + tid] = tid == 32 ? e : tid < P * T ? mx_few_row(a, few, e, tid % T) : -1;
  if ((int)blockIdx.x * FW >= mx_blocks(inter)) return;
  for (int b = tid; b < T * HB; b += 512) {
    const int t = b / HB, kb = b % HB;
    uint4 r[RV];
    mx_token_record<P>(a.x, t, a.H, kb, r);
    uint4* o = (uint4*)(sm + (size_t)(kb * T + t) * RB);
#pragma unroll
    for (int i = 0; i < RV; i++) o[i] = r[i];
  }
  uint8_t* const zrec = sm + (size_t)T * HB * RB;   // what the columns without a token read
  if (tid == 0) {
    uint4 r[RV];
    mx_zero_record<P>(r);
#pragma unroll
    for (int i = 0; i < RV; i++) ((uint4*)zrec)[i] = r[i];
  }
  lds_barrier();
  mx_v16f ag = mx_zero16(), au = mx_zero16();
  const int col = lane & 31, half = lane >> 5, C = P * T, p = col / T, t = col % T;   // column, plane, token
  const uint8_t* rec = col < C ? sm + (half * T + t) * RB : zrec;
  const int rstep = col < C ? 2 * T * RB : 0, pl = col < C ? p : 0;
#define MX_STEP(i)                          \
  {                                         \
    MxPlane b;                              \
    b.load<P>(rec + (s + i) * rstep, pl);   \
    ag = mx_mfma1<i>(wg[i], cg, b, ag);     \
    au = mx_mfma1<i>(wu[i], cu, b, au);     \
  }
  if (work) {
    int s = s0;
    for (; s + 8 <= s1; s += 4) {
      const uint32_t cg = sg >> (8 * (s & 3)), cu = su >> (8 * (s & 3));
      fetch_scales(s + 4);
      // a step's registers are loaded again as soon as it is done (left to itself the
      // compiler loads all four steps into others first, and spills them)
      MX_STEP(0) fetch(s + 4, 0);
      __builtin_amdgcn_sched_barrier(0);
      MX_STEP(1) fetch(s + 5, 1);
      __builtin_amdgcn_sched_barrier(0);
      MX_STEP(2) fetch(s + 6, 2);
      __builtin_amdgcn_sched_barrier(0);
      MX_STEP(3) fetch(s + 7, 3);
      __builtin_amdgcn_sched_barrier(0);
    }
    for (; s < s1; s += 4) {   // one or two last groups, the last one short
      const uint32_t cg = sg >> (8 * (s & 3)), cu = su >> (8 * (s & 3));
      MX_STEP(0)
      if (s + 1 < s1) MX_STEP(1)
      if (s + 2 < s1) MX_STEP(2)
      if (s + 3 < s1) MX_STEP(3)
      if (s + 4 < s1) {
        fetch_scales(s + 4);
#pragma unroll
        for (int i = 0; i < 4; i++) fetch(min(s + 4 + i, s1 - 1), i);
      }
    }
  }
#undef MX_STEP
  lds_barrier();   // the records have been read: their place takes the sums
  float* red = (float*)sm;                  // [8 waves][gate, up][32 features][C]
  float* hv = red + 8 * 2 * 32 * C;         // [FW][T][33]
  if (col < C) {
#pragma unroll
    for (int i = 0; i < 16; i++) {
      const int f = 8 * (i >> 2) + 4 * half + (i & 3);
      red[((wave * 2 + 0) * 32 + f) * C + col] = ag[i];
      red[((wave * 2 + 1) * 32 + f) * C + col] = au[i];
    }
  }
  lds_barrier();
  for (int o = tid; o < FW * 32 * T; o += 512) {
    const int w0 = o / (32 * T) * KW, f = o / T % 32, tt = o % T;
    float g = 0.f, u = 0.f;
#pragma unroll
    for (int w = 0; w < KW; w++)
#pragma unroll
      for (int q = 0; q < P; q++) {
        g += red[((w0 + w) * 2 + 0) * 32 * C + f * C + q * T + tt];
        u += red[((w0 + w) * 2 + 1) * 32 * C + f * C + q * T + tt];
      }
    hv[(w0 / KW * T + tt) * 33 + f] = mx_swiglu(g, u);
  }
  lds_barrier();
  if (tid < FW * T) {
    const int ft = tid / T, tt = tid % T, f0 = blockIdx.x * FW + ft;
    // the row of h: the token's first entry with this expert
    const int row = !ONE ? mx_few_row(a, few, e, tt) : e == a.E ? a.F : slot;
    if (row >= 0 && f0 < mx_blocks(inter)) {
      uint4 r[RV];
      if (32 * f0 >= inter) {
        mx_zero_record<P>(r);
      } else {
        float f[32];
#pragma unroll
        for (int i = 0; i < 32; i++) f[i] = hv[tid * 33 + i];
        mx_record<P>(f, r);
      }
      uint4* o = (uint4*)(a.hrec + ((int64_t)row * a.hblocks + f0) * RB);
#pragma unroll
      for (int i = 0; i < RV; i++) o[i] = r[i];
    }
  }
}

// bytes of LDS of k_mx_few_gate_up: the tokens' records and the one of zeros, then the sums
static size_t mx_few_lds(int T, int H, bool xbf) {
  const size_t rec = ((size_t)T * mx_blocks(H) + 1) * mx_rec_bytes(xbf);
  const size_t red = (size_t)(8 * 2 * 32 * mx_planes(xbf) * T + 8 * 33 * T) * 4;
  return rec > red ? rec : red;
}

// LDS decides. By the sums bf16 has 8 tokens at most (56 KB), f32 5 (55 KB; 6 would be 66);
// by the records that many up to 2944 columns, fewer of more.
constexpr size_t MX_FEW_LDS = 60 * 1024;
static_assert(8 * 2 * 32 * 33 * 4 > MX_FEW_LDS, "the sums of more planes than an MFMA's 32 columns do not fit");
bool mx_few(int T, int k, int H, bool xbf) { return T <= MX_FEW_T && mx_few_lds(T, H, xbf) <= MX_FEW_LDS; }

// most chosen experts of a call (one token: its entries)
static int mx_few_slots(int T, int k, int E) { return T == 1 ? k : min(T * k, E); }

// 8 steps of K of an expert's 32 outputs nb for up to 8 tokens: d += the weights of
// steps s .. of mat (inter columns) x the planes of the lanes' rows (row < 0: zeros)
template <int P>
HX_DEV mx_v16f mx_few_unit(const MxArgs& a, const uint8_t* mat, int inter, int nb, int s, int row, int p, mx_v16f d) {
  constexpr int RB = MxRec<P>::BYTES;
  const int lane = lane_id(), half = lane >> 5, S = mx_steps(inter), S4 = (S + 3) / 4;
  const uint8_t* wp = mat + ((int64_t)nb * S + s) * 1024;
  const uint8_t* sp = mat + (mx_code_bytes(a.H, inter) + ((int64_t)nb * S4 + s / 4) * 256);
  uint4 w[8];
  const uint32_t sa = *(const uint32_t*)(sp + lane * 4);
  const uint32_t sb = *(const uint32_t*)(sp + (s / 4 + 1 < S4 ? 256 : 0) + lane * 4);
#pragma unroll
  for (int i = 0; i < 8; i++) w[i] = *(const uint4*)(wp + min(i, S - 1 - s) * 1024 + lane * 16);
  const uint8_t* hp = a.hrec + ((int64_t)max(row, 0) * a.hblocks + 2 * s + half) * RB;
#define MX_STEP(i)                                            \
  if (s + i < S) {                                            \
    MxPlane b;                                                \
    b.zero();                                                 \
    if (row >= 0) b.load<P>(hp + 2 * i * RB, p);              \
    d = mx_mfma1<(i & 3)>(w[i], i < 4 ? sa : sb, b, d);       \
  }
  MX_STEP(0) MX_STEP(1) MX_STEP(2) MX_STEP(3) MX_STEP(4) MX_STEP(5) MX_STEP(6) MX_STEP(7)
#undef MX_STEP
  return d;
}

// Down and combine of one token. Workgroup: 32 outputs; its 16 waves take the units
// (entry, 8 steps of K) in turn, weigh each product in f32, and add up in LDS. No
// combine, so a launch less. 6.4 us for 10 experts and the shared one of 2048 x 512, 6 MB:
// bound by latency (routing, weights and records, the last sum of 16 P values by one lane
// an output) on 64 workgroups, a quarter of the CUs. Twice the bytes of Q8_0 take 5.4 in
// their own kernel, which spreads them over more.
template <int P>
__global__ __launch_bounds__(1024) void k_mx_one_down(MxArgs a) {
  __shared__ float red[16 * P * 32];
  const int tid = threadIdx.x, lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int k = a.k, nb = blockIdx.x, G = (mx_steps(a.I) + 7) / 8, Gs = a.Is ? (mx_steps(a.Is) + 7) / 8 : 0;
  const int col = lane & 31, half = lane >> 5;
  mx_v16f acc = mx_zero16();
  for (int u = wave; u < k * G + Gs; u += 16) {
    const bool sh = u >= k * G;
    const int j = sh ? k : u / G, g = sh ? u - k * G : u % G;
    int e = a.E;
    if (!sh) e = __builtin_amdgcn_readfirstlane(a.idx[j]);
    if (!sh && (unsigned)e >= (unsigned)a.E) continue;
    const float wt = sh ? a.shared_w[0] : a.w[j];
    const mx_v16f d = mx_few_unit<P>(a, sh ? a.sdown.base : a.down.mat(e), sh ? a.Is : a.I, nb, 8 * g,
                                     col < P ? (sh ? a.F : j) : -1, col, mx_zero16());
#pragma unroll
    for (int i = 0; i < 16; i++) acc[i] = __builtin_fmaf(wt, d[i], acc[i]);
  }
  if (col < P) {
#pragma unroll
    for (int i = 0; i < 16; i++) red[(wave * P + col) * 32 + 8 * (i >> 2) + 4 * half + (i & 3)] = acc[i];
  }
  lds_barrier();
  if (tid < 32) {
    float y = 0.f;
#pragma unroll
    for (int w = 0; w < 16 * P; w++) y += red[w * 32 + tid];
    mx_store(a, 32 * nb + tid, y);
  }
}

// Outputs of the experts for 2 to 8 tokens, unweighted and in f32, in the row of the
// token's first entry with the expert. Workgroup: a chosen expert (slot) and 128
// outputs; a wave 32 of them and all of K, its 8 KB of a step group in flight together.
// 6 tokens' 32 MB of 2048 x 512 experts: 10.8 us (3.0 TB/s; of them about 4 before the
// first weights can be asked for).
template <int P>
__global__ __launch_bounds__(256) void k_mx_few_down(MxArgs a) {
  __shared__ float red[4][32][33];
  const int tid = threadIdx.x, lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int T = a.T, nb = 4 * blockIdx.x + wave, col = lane & 31, half = lane >> 5;
  const int32_t* tab = a.few + blockIdx.y * MX_FEW_TAB;   // k_mx_few_gate_up's
  const int e = tab[32], row = tab[col];
  if (e < 0 || 32 * nb >= a.H) return;   // no barrier behind this
  const bool sh = e == a.E;
  const int inter = sh ? a.Is : a.I, S = mx_steps(inter), p = col / T;
  const uint8_t* mat = sh ? a.sdown.base : a.down.mat(e);
  mx_v16f d = mx_zero16();
  for (int s = 0; s < S; s += 8) d = mx_few_unit<P>(a, mat, inter, nb, s, row, p, d);
#pragma unroll
  for (int i = 0; i < 16; i++) red[wave][col][8 * (i >> 2) + 4 * half + (i & 3)] = d[i];
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
  for (int t0 = 0; t0 < T; t0 += 2) {   // a half wave a token
    const int tt = t0 + half, r = __shfl(row, tt & 31, 64);
    if (tt >= T || r < 0) continue;
    float y = 0.f;
#pragma unroll
    for (int q = 0; q < P; q++) y += red[wave][q * T + tt][col];
    ((float*)a.obuf)[(int64_t)r * a.H + 32 * nb + col] = y;
  }
}

template <int P>
static void mx_few_gate_up(const MxArgs& a, hipStream_t s) {
  const int slots = mx_few_slots(a.T, a.k, a.E) + (a.Is > 0 ? 1 : 0), tasks = slots * a.hblocks;
  const uint32_t lds = (uint32_t)mx_few_lds(a.T, a.H, a.xbf);
  // A wave's start costs as much as some steps of K, so that sharing K pays only where
  // there are too few waves. K shared by 8, 2 and 1 waves, us (512 experts of 512 x 2048
  // and others): 72 tasks 8.3, 9.4, -; 264 11.5, 11.8, -; 336 12.4, 11.0, -; 976 22.8,
  // 19.3, 21.2; 1296 31.4, 24.6, 22.6; 2048 -, 28.8, 28.9.
#define FGU(KW, ONE) \
  hx_launch(k_mx_few_gate_up<P, KW, ONE>, dim3((a.hblocks + 8 / KW - 1) / (8 / KW), slots), dim3(512), lds, s, a)
  if (a.T == 1) FGU(8, true);
  else if (tasks >= 1200) FGU(1, false);
  else if (tasks >= 300) FGU(2, false);
  else FGU(8, false);
#undef FGU
}

hipError_t launch_mx_few_gate_up(const MxArgs& a, hipStream_t s) {
  if (a.xbf) mx_few_gate_up<3>(a, s);
  else mx_few_gate_up<5>(a, s);
  return hipGetLastError();
}

hipError_t launch_mx_few_down(const MxArgs& a, hipStream_t s) {
  if (a.T == 1) {
    if (a.xbf) hx_launch(k_mx_one_down<3>, dim3(a.H / 32), dim3(1024), 0, s, a);
    else hx_launch(k_mx_one_down<5>, dim3(a.H / 32), dim3(1024), 0, s, a);
  } else {
    const dim3 g((a.H + 127) / 128, mx_few_slots(a.T, a.k, a.E) + (a.Is > 0 ? 1 : 0));
    if (a.xbf) hx_launch(k_mx_few_down<3>, g, dim3(256), 0, s, a);
    else hx_launch(k_mx_few_down<5>, g, dim3(256), 0, s, a);
  }
  return hipGetLastError();
}

// ---------------------------------------------------------------- dispatch
// Workgroups 0 .. chunks - 1: the chunk's entries by expert, and where there is one
// chunk alone (a launch less: about 4 us) their places too; the others: the tokens' records,
// a thread a block of 32. Bound by launch and latency up to some hundred tokens (4.5 us),
// then by HBM: 8192 tokens of 2048, 34 MB in and 42 out, 16 us (4.7 TB/s; 24 with a
// record a lane).
template <int P>
__global__ __launch_bounds__(256) void k_mx_prep(MxArgs a) {
  constexpr int RB = MxRec<P>::BYTES, RV = MxRec<P>::VECS;
  static_assert(sizeof(MxPlace) <= 256 * RB, "one of the two is used");
  __shared__ __align__(16) uint8_t rows[256 * RB];
  MxPlace& sm = *(MxPlace*)rows;
  const int nch = mx_chunks(a.F), tid = threadIdx.x;
  if ((int)blockIdx.x < nch) {
    mx_chunk_entries(a, sm, nch);
    return;
  }
  // a wave's 64 records leave through LDS, by whole KiB
  const int HB = mx_blocks(a.H), lane = lane_id(), wave = tid >> 6;
  const int64_t b0 = (int64_t)(blockIdx.x - nch) * 256 + wave * 64, n = (int64_t)a.T * HB - b0;
  uint4* const rec = (uint4*)(rows + wave * 64 * RB);
  if (lane < n) {
    const int64_t b = b0 + lane;
    uint4 r[RV];
    mx_token_record<P>(a.x, b / HB, a.H, (int)(b % HB), r);
#pragma unroll
    for (int i = 0; i < RV; i++) rec[lane * RV + i] = r[i];
  }
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
  uint4* const o = (uint4*)(a.xrec + b0 * RB);
#pragma unroll
  for (int i = 0; i < RV; i++)
    if (i * 64 + lane < n * RV) o[i * 64 + lane] = rec[i * 64 + lane];
}

// several chunks: every workgroup sums the chunks' counts itself and places its own
// entries. Bound by that sum's latency: 4.9 us for 5 chunks, 10 to 12 for 80 (8192 tokens).
__global__ __launch_bounds__(1024) void k_mx_dispatch(MxArgs a) {
  __shared__ MxPlace sm;
  const int e = threadIdx.x, nch = mx_chunks(a.F), c = blockIdx.x;
  int count[1] = {0}, pre[1] = {0};
  if (e < a.E) {
    for (int c0 = 0; c0 < nch; c0 += 8) {
      int h[8];
#pragma unroll
      for (int i = 0; i < 8; i++) h[i] = c0 + i < nch ? a.hist[(int64_t)(c0 + i) * a.E + e] : 0;
#pragma unroll
      for (int i = 0; i < 8; i++) {
        if (c0 + i == c) pre[0] = count[0];
        count[0] += h[i];
      }
    }
  }
  mx_place<1024>(a, sm, c, count, pre);
}

hipError_t launch_mx_prep(const MxArgs& a, hipStream_t s) {
  const int64_t n = ((int64_t)a.T * mx_blocks(a.H) + 255) / 256 + mx_chunks(a.F);
  if (a.xbf) hx_launch(k_mx_prep<3>, dim3((unsigned)n), dim3(256), 0, s, a);
  else hx_launch(k_mx_prep<5>, dim3((unsigned)n), dim3(256), 0, s, a);
  return hipGetLastError();
}

hipError_t launch_mx_dispatch(const MxArgs& a, hipStream_t s) {
  hx_launch(k_mx_dispatch, dim3(mx_chunks(a.F)), dim3(1024), 0, s, a);
  return hipGetLastError();
}

// ---------------------------------------------------------------- grouped products
// Rows of a tile: 32 while the experts have few rows each: F entries over all E experts, so
// that padding and experts without rows count too (the routing is on the device). 512 experts of 10 chosen: at
// 20 rows an expert 197 us with tiles of 32 and 229 of 64, at 25 219 and 236, at 31 258
// and 244, at 40 325 and 259.
int mx_tile_m(int64_t F, int E, bool xbf) { return !xbf || F <= 28 * (int64_t)E ? 32 : 64; }

// Whether an expert's weights are read mostly once: non-temporally then, so that they
// leave the caches to the rows. 64 tokens on 512 experts 123 -> 112 us, 512 tokens (10
// rows an expert) 182 -> 172, 2048 (40) 266 -> 258, 2500 (49) 275 -> 273; 3000 (59) no
// gain, 3500 (68, two tiles) 371 -> 384, 8192 661 -> 688: there the tiles that come
// later want them in the caches. f32, tiles of 32: 512 tokens 197 -> 191, 1000 (20) 216 ->
// 212; 2048 366 -> 383.
static bool mx_once(const MxArgs& a) { return a.F <= (a.tile_m == 32 ? 28 : 50) * (int64_t)a.E; }

// The tile's rows in LDS, CB blocks of K at a time: [CB / G groups][TM rows][G records].
// They come in by direct loads, 16 bytes a lane, in LDS order; a unit of U blocks is whole
// KiB loads. G 2 reads 160 bytes of a row in a piece where G 1 reads 80 (512 tokens, tiles
// of 32: 171 -> 168 us), but the operands' 160-byte steps meet more often on a bank: with
// tiles of 64, 653 -> 659 us at 8192 tokens. f32's records of 128 bytes would all start on
// one bank: piece j of row r lies at j ^ r % 8 (512 tokens of 2048 on 512 experts of 512:
// gate/up 165 -> 128 us, down 88 -> 73).
template <int TM, int P>
struct MxRows {
  static constexpr int RB = MxRec<P>::BYTES, RV = MxRec<P>::VECS;
  static constexpr int CB = 8, BYTES = CB * TM * RB;
  static constexpr int G = P == 3 && TM == 32 ? 2 : 1;   // blocks of a row side by side
  static constexpr int U = G == 1 && TM * RV % 64 == 0 ? 1 : 2, LOADS = U * TM * RV / 64;
  static_assert(U * TM * RV % 64 == 0, "whole loads");
  const uint8_t* src[LOADS];
  // rowptr(r): the records of the tile's row r
  template <typename F>
  HX_DEV void init(F rowptr) {
#pragma unroll
    for (int i = 0; i < LOADS; i++) {
      const int q = i * 64 + lane_id();   // 16-byte piece of the unit
      const int row = q / (G * RV) % TM, piece = q % (G * RV);
      src[i] = rowptr(row) + q / (TM * G * RV) * (G * RB) + (P == 5 ? piece ^ (row & 7) : piece) * 16;
    }
  }
  // blocks b0 .. min(b0 + CB, nblk) - 1 (a multiple of 4)
  HX_DEV void load(int wave, int b0, int nblk, uint32_t lds) const {
    const int n = min(CB, nblk - b0) / U;
    for (int u = wave; u < n; u += 4)
#pragma unroll
      for (int i = 0; i < LOADS; i++) dma16(src[i] + (int64_t)(b0 + u * U) * RB, lds + (u * LOADS + i) * 1024);
  }
};

// A wave's weights: NM matrices' tiles of 32 rows, R steps of K on their way at any
// time; a step's registers are loaded again as soon as its MFMAs are issued. (Loaded a
// stage ahead into a second set, with a barrier and a wait for everything at each
// stage of 128 columns, the wait was never over in time: MFMAs busy 41 % at 8192 tokens.)
// AUX 2: non-temporal (mx_once).
template <int P, int NM, int AUX>
struct MxRing {
  // steps, words of scales; a chunk of rows is whole turns of the ring
  static constexpr int R = 8 / NM, U = R < 4 ? 4 : R, W = U / 4;
  static_assert(MxRows<32, P>::CB / 2 % U == 0, "whole turns");
  // byte offsets of the matrices' tiles from mat[m % 2]; buffer loads, so that the lanes'
  // addresses take one register in all
  __amdgpu_buffer_rsrc_t mat[2];
  int codes[NM], scales[NM];
  mx_v4u w[R][NM];
  uint32_t sc[W][NM], sn[W][NM];   // of this turn and of the next
  HX_DEV void matrix(int q, const uint8_t* base, int rows, int K) {
    mat[q] = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, (int)mx_mat_bytes(rows, K), 0x00027000);
  }
  // Steps past the last (s >= S) are loaded from past the matrix's end, which reads
  // nothing and gives zeros: a branch around the loads would copy the ring where it
  // joins, and so wait for all of it.
  HX_DEV static int lane_offset(int size, bool has) { return lane_id() * size + (has ? 0 : 0x40000000); }
  HX_DEV void fetch(int i, int s, int S) {
    const int o = lane_offset(16, s < S);
#pragma unroll
    for (int m = 0; m < NM; m++)
      w[i][m] = __builtin_amdgcn_raw_buffer_load_b128(mat[m % 2], o, s < S ? codes[m] + s * 1024 : 0, AUX);
  }
  HX_DEV void fetch_scales(int j, int s, int S) {   // of steps s .. s + 3
    const int o = lane_offset(4, s < S);
#pragma unroll
    for (int m = 0; m < NM; m++)
      sn[j][m] = __builtin_amdgcn_raw_buffer_load_b32(mat[m % 2], o, s < S ? scales[m] + (s >> 2) * 256 : 0, 0);
  }
  HX_DEV void start(int S) {
#pragma unroll
    for (int j = 0; j < W; j++) fetch_scales(j, 4 * j, S);
#pragma unroll
    for (int i = 0; i < R; i++) fetch(i, i, S);
  }
  HX_DEV void turn(int s, int S) {   // the scales of steps s .. become this turn's, the next are fetched
#pragma unroll
    for (int j = 0; j < W; j++) {
#pragma unroll
      for (int m = 0; m < NM; m++) sc[j][m] = sn[j][m];
      fetch_scales(j, s + U + 4 * j, S);
    }
  }
};

// a turn of the ring from step s of S: acc += its weights x the rows at rec; LAST: no
// steps of a turn after it are fetched
template <int TM, int P, int NM, bool LAST, int AUX, int I = 0>
HX_DEV void mx_turn(MxRing<P, NM, AUX>& ring, const uint8_t* rec, int s, int S, mx_v16f (&acc)[NM][TM / 32]) {
  constexpr int RB = MxRec<P>::BYTES, R = MxRing<P, NM, AUX>::R, U = MxRing<P, NM, AUX>::U;
  if constexpr (I < U) {
    if (!LAST || s + I < S) {
#pragma unroll
      for (int n = 0; n < TM / 32; n++) {
        MxB<P> b;
        const uint8_t* r = rec + (2 * I * TM + 32 * MxRows<TM, P>::G * n) * RB;
        if constexpr (P == 5) b.load_swizzled(r, lane_id() & 7);
        else b.load(r);
        mx_mfma<P, I & 3>(ring.w[I % R], ring.sc[I / 4], b, acc, n);
      }
      if (!LAST || I + R < U) ring.fetch(I % R, s + I + R, S);
      __builtin_amdgcn_sched_barrier(0);
      mx_turn<TM, P, NM, LAST, AUX, I + 1>(ring, rec, s, S, acc);
    }
  }
}
// acc = the sums over nblk blocks of K of the ring's weights x the tile's rows, which
// come into buf's two halves in turn, a chunk ahead
template <int TM, int P, int NM, int AUX>
HX_DEV void mx_products(MxRing<P, NM, AUX>& ring, const MxRows<TM, P>& rw, int wave, uint8_t* buf, int nblk,
                        mx_v16f (&acc)[NM][TM / 32]) {
  constexpr int RB = MxRec<P>::BYTES, CB = MxRows<TM, P>::CB, BYTES = MxRows<TM, P>::BYTES;
  constexpr int R = MxRing<P, NM, AUX>::R, U = MxRing<P, NM, AUX>::U, W = MxRing<P, NM, AUX>::W;
  const uint32_t lds = (uint32_t)(uintptr_t)(lds_u8*)buf;
  const int lane = lane_id(), S = nblk / 2;
  const uint8_t* rec = buf + (MxRows<TM, P>::G == 2 ? lane % 32 * 2 + lane / 32 : lane / 32 * TM + lane % 32) * RB;
#pragma unroll
  for (int m = 0; m < NM; m++)
#pragma unroll
    for (int n = 0; n < TM / 32; n++) acc[m][n] = mx_zero16();
  rw.load(wave, 0, nblk, lds);
  ring.start(S);
  // the rows are the oldest loads: what may be left are the ring's
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"((R + W) * NM) : "memory");
  lds_barrier();
  int s = 0, b0 = 0, h = 0;   // a chunk is whole turns; the last turn comes after the loop
  for (;;) {
    // the other half was read before the barrier
    if (b0 + CB < nblk) rw.load(wave, b0 + CB, nblk, lds + (h ^ 1) * BYTES);
    for (const int end = min(S - U, (b0 + CB) / 2); s < end; s += U) {
      ring.turn(s, S);
      mx_turn<TM, P, NM, false, AUX>(ring, rec + h * BYTES + (2 * s - b0) * TM * RB, s, S, acc);
    }
    if (b0 + CB >= nblk) break;
    // a turn's loads at least came after the next rows'
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(U * NM) : "memory");
    lds_barrier();
    b0 += CB;
    h ^= 1;
  }
  ring.turn(s, S);
  mx_turn<TM, P, NM, true, AUX>(ring, rec + h * BYTES + (2 * s - b0) * TM * RB, s, S, acc);
  // the sums leave the loop whole: seen through, their elements are carried through it
  // one by one as well, and spilled
#pragma unroll
  for (int m = 0; m < NM; m++)
#pragma unroll
    for (int n = 0; n < TM / 32; n++) asm volatile("" : "+v"(acc[m][n]));
}

// lane l: the 32 values of column l of the tile from D's halves
template <int TM>
HX_DEV void mx_columns(const mx_v16f (&d)[TM / 32], float (&f)[32]) {
#pragma unroll
  for (int i = 0; i < 16; i++) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(d[0][i]), __float_as_uint(d[TM / 32 - 1][i]), false, false);
    const int o = 8 * (i >> 2) + (i & 3);
    f[o] = __uint_as_float(r[0]);
    f[o + 4] = __uint_as_float(r[1]);
  }
}

// A wave's results, BYTES a row in LDS (row r at tile + r PITCH), to dst(r): whole rows by
// neighbouring lanes. (A row a lane, 16 bytes a store, touches 64 rows' lines with every
// store: k_mx_down 260 us at 8192 tokens, 63 at 512; so 228, 58.)
template <int BYTES>
struct MxOut {
  static constexpr int PITCH = BYTES + 16, PIECES = BYTES / 16;   // 16 bytes more: fewer rows on the same banks
  HX_DEV static uint8_t* row(uint8_t* tile, int r) { return tile + r * PITCH; }
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

// h = silu(G x) * (U x), as records. Workgroup: a tile of TM rows and 4 MF groups of 32
// features, MF a wave, with gate and up of a feature in the same lane. TM 32 (few rows an
// expert) is bound by the weight stream: 512 tokens on 512 experts of 2048 x 512, 574 MB
// in 99 us (5.8 TB/s; the load units busy 96 %). TM 64 by the loads' way into the CU: 8192
// tokens 310 to 360 us, the load units busy 86 % of it and the matrix cores 60 %, at a
// clock of about 1.7 GHz; 2048 tokens 150, 96 and 39 % (a wave's weights meet 64 rows; MF 2
// halves the rows' loads, and its sums and ring fill the registers, 213 of 256, two waves a
// SIMD).
template <int TM, int P, int MF, bool NT>
__global__ __launch_bounds__(256, 2) void k_mx_gate_up(MxArgs a) {
  constexpr int RB = MxRec<P>::BYTES, RV = MxRec<P>::VECS;
  __shared__ __align__(16) uint8_t buf[2 * MxRows<TM, P>::BYTES];
  int nt, tile;
  mx_tile((a.hblocks + 4 * MF - 1) / (4 * MF), a.counts[0], nt, tile);
  if (tile < 0) return;
  const int4 ti = ((const int4*)a.tiles)[tile];
  const int e = __builtin_amdgcn_readfirstlane(ti.x), p0 = ti.y, rows = ti.z;
  const bool sh = e == a.E;
  const int inter = sh ? a.Is : a.I;
  if (4 * MF * nt >= mx_blocks(inter)) return;
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int f0 = (4 * nt + wave) * MF, HB = mx_blocks(a.H), S = mx_steps(a.H), S4 = (S + 3) / 4;
  MxRows<TM, P> rw;
  rw.init([&](int r) {
    const int p = p0 + min(r, rows - 1);
    const int t = sh ? p - a.F : a.perm[p] / a.k;
    return a.xrec + (int64_t)t * HB * RB;
  });
  MxRing<P, 2 * MF, NT ? 2 : 0> ring;
  ring.matrix(0, sh ? a.sgate.base : a.gate.mat(e), inter, a.H);
  ring.matrix(1, sh ? a.sup.base : a.up.mat(e), inter, a.H);
#pragma unroll
  for (int m = 0; m < MF; m++) {
    const int fb = min(f0 + m, inter / 32 - 1);
    ring.codes[2 * m] = ring.codes[2 * m + 1] = fb * S * 1024;
    ring.scales[2 * m] = ring.scales[2 * m + 1] = (int)mx_code_bytes(inter, a.H) + fb * S4 * 256;
  }
  mx_v16f acc[2 * MF][TM / 32];
  mx_products<TM, P, 2 * MF, NT ? 2 : 0>(ring, rw, wave, buf, HB, acc);
  using Out = MxOut<MF * RB>;
  static_assert(4 * TM * Out::PITCH <= 2 * MxRows<TM, P>::BYTES, "the rows' place holds the results");
  lds_barrier();   // the rows have been read
  uint8_t* const tl = buf + wave * (TM * Out::PITCH);
#pragma unroll
  for (int m = 0; m < MF; m++) {
    mx_v16f h[TM / 32];
#pragma unroll
    for (int n = 0; n < TM / 32; n++)
#pragma unroll
      for (int i = 0; i < 16; i++) h[n][i] = mx_swiglu(acc[2 * m][n][i], acc[2 * m + 1][n][i]);
    float f[32];
    mx_columns<TM>(h, f);
    uint4 r[RV];
    if (32 * (f0 + m) < inter) mx_record<P>(f, r);
    else mx_zero_record<P>(r);
    if (lane < TM) {
      uint4* o = (uint4*)(Out::row(tl, lane) + m * RB);
#pragma unroll
      for (int i = 0; i < RV; i++) o[i] = r[i];
    }
  }
  Out::store(tl, rows, min(MF, mx_blocks(inter) - f0) * RB,
             [&](int r) { return a.hrec + ((int64_t)(p0 + r) * a.hblocks + f0) * RB; });
}

// Outputs of the experts, unweighted: D h. Workgroup: a tile of TM rows and 256 MF
// features, 64 MF a wave. K is short (I), so that a quarter of the time goes into the
// start and the rows going out. 512 tokens: 287 MB in 55 us (5.2 TB/s); 8192 tokens 212 to
// 239 us, the load units busy 88 %.
// A row leaves in the activations' type: bf16 rows are half of what this kernel writes and
// the combine reads (8192 tokens: 369 MB each way, the combine at the HBM's rate), for a
// rounding of each expert's part by at most 2^-8 of it, as the result's own: 0.0024 of the
// output's norm from 64 bits in place of 0.0017. The weighted sum is in f32.
template <int TM, int P, int MF, bool NT>
__global__ __launch_bounds__(256, 2) void k_mx_down(MxArgs a) {
  constexpr int RB = MxRec<P>::BYTES, NM = 2 * MF;
  __shared__ __align__(16) uint8_t buf[2 * MxRows<TM, P>::BYTES];
  int nt, tile;
  const int nb = a.H / 32;
  mx_tile((nb + 4 * NM - 1) / (4 * NM), a.counts[0], nt, tile);
  if (tile < 0) return;
  const int4 ti = ((const int4*)a.tiles)[tile];
  const int e = __builtin_amdgcn_readfirstlane(ti.x), p0 = ti.y, rows = ti.z;
  const bool sh = e == a.E;
  const int inter = sh ? a.Is : a.I;
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int IB = mx_blocks(inter), S = mx_steps(inter), S4 = (S + 3) / 4, n0 = (4 * nt + wave) * NM;
  MxRows<TM, P> rw;
  rw.init([&](int r) { return a.hrec + (int64_t)(p0 + min(r, rows - 1)) * a.hblocks * RB; });
  MxRing<P, NM, NT ? 2 : 0> ring;
  ring.matrix(0, sh ? a.sdown.base : a.down.mat(e), a.H, inter);
  ring.mat[1] = ring.mat[0];
#pragma unroll
  for (int m = 0; m < NM; m++) {
    const int n = min(n0 + m, nb - 1);   // past the last: computed again, not stored
    ring.codes[m] = n * S * 1024;
    ring.scales[m] = (int)mx_code_bytes(a.H, inter) + n * S4 * 256;
  }
  mx_v16f acc[NM][TM / 32];
  mx_products<TM, P, NM, NT ? 2 : 0>(ring, rw, wave, buf, IB, acc);
  constexpr int ES = P == 3 ? 2 : 4;   // bytes of an output
  using Out = MxOut<32 * NM * ES>;
  static_assert(4 * TM * Out::PITCH <= 2 * MxRows<TM, P>::BYTES, "the rows' place holds the results");
  lds_barrier();   // the rows have been read
  uint8_t* const tl = buf + wave * (TM * Out::PITCH);
#pragma unroll
  for (int m = 0; m < NM; m++) {
    __builtin_amdgcn_sched_barrier(0);   // one matrix's outputs after the other's: all at once do not fit the registers
    float f[32];
    mx_columns<TM>(acc[m], f);
    if (lane < TM) {
      if constexpr (P == 3) {
        uint4* o = (uint4*)(Out::row(tl, lane) + m * 64);
#pragma unroll
        for (int i = 0; i < 4; i++) {
          uint32_t q[4];
#pragma unroll
          for (int j = 0; j < 4; j++)
            q[j] = f32_to_bf16(f[8 * i + 2 * j]) | ((uint32_t)f32_to_bf16(f[8 * i + 2 * j + 1]) << 16);
          o[i] = make_uint4(q[0], q[1], q[2], q[3]);
        }
      } else {
        float4* o = (float4*)(Out::row(tl, lane) + m * 128);
#pragma unroll
        for (int i = 0; i < 8; i++) o[i] = make_float4(f[4 * i], f[4 * i + 1], f[4 * i + 2], f[4 * i + 3]);
      }
    }
  }
  Out::store(tl, rows, min(NM, nb - n0) * 32 * ES,
             [&](int r) { return (uint8_t*)a.obuf + ((int64_t)(p0 + r) * a.H + 32 * n0) * ES; });
}

// groups of 32 features a wave takes at a time where tiles have 64 rows
constexpr int MX_MF = 2;
#define MX_LAUNCH(KERNEL, NX)                                                                    \
  auto go = [&](auto kernel, int mf) {                                                           \
    hx_launch(kernel, dim3((unsigned)((int64_t)(NX) * ((a.max_tiles + 7) / 8 * 8))), dim3(256), 0, s, a); \
  };                                                                                             \
  if (a.xbf && a.tile_m == 32) go(KERNEL<32, 3, 1, true>, 1);                                    \
  else if (a.xbf && mx_once(a)) go(KERNEL<64, 3, MX_MF, true>, MX_MF);                           \
  else if (a.xbf) go(KERNEL<64, 3, MX_MF, false>, MX_MF);                                        \
  else if (mx_once(a)) go(KERNEL<32, 5, 1, true>, 1);                                            \
  else go(KERNEL<32, 5, 1, false>, 1)

hipError_t launch_mx_gate_up(const MxArgs& a, hipStream_t s) {
  MX_LAUNCH(k_mx_gate_up, (a.hblocks + 4 * mf - 1) / (4 * mf));
  return hipGetLastError();
}
hipError_t launch_mx_down(const MxArgs& a, hipStream_t s) {
  MX_LAUNCH(k_mx_down, (a.H / 32 + 8 * mf - 1) / (8 * mf));
  return hipGetLastError();
}

constexpr int64_t MX_CACHE = 256ll << 20;   // bytes of the cache before the memory

template <bool NT>
HX_DEV uint4 mx_row16(const void* p) {
  if constexpr (NT) {
    const mx_v4u v = __builtin_nontemporal_load((const mx_v4u*)p);
    return make_uint4(v[0], v[1], v[2], v[3]);
  } else {
    return *(const uint4*)p;
  }
}

// y[t] = the token's entries' rows times their weights in their order, then the
// shared expert's. A wave: 512 outputs of a token, 8 a lane, 8 rows' loads together
// (an entry without an expert reads row 0 and counts nothing). Bound by HBM, few
// tokens by latency (4 us). FEW: rows in f32, a
// token's entry at that of its first with the same expert; else rows in the
// activations' type by inv, SC: in f16 with a scale for each 32; NT: more of them than MX_CACHE, read non-temporally (8192
// tokens' 369 MB: 65 us against 78; 2048 tokens' 92 MB: 19 against 17). f32 rows of 2048 tokens:
// 34 us.
template <bool BF, bool FEW, bool NT, bool SC>
__global__ __launch_bounds__(256) void k_mx_combine(MxArgs a) {
  constexpr bool R16 = BF && !FEW;
  static_assert(R16 || !SC, "rows of 16 bits");
  constexpr int B = 8;
  const int lane = lane_id(), segs = (a.H + 511) / 512, k = a.k;
  const int64_t id = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t t = id / segs;
  const int n0 = (int)(id % segs) * 512 + lane * 8;
  if (t >= a.T) return;
  // a lane behind the row's end computes the row's first outputs and stores nothing: the
  // others read its entry's row and weight
  const bool mine = n0 < a.H;
  // lane j: entry j; lane k: the shared expert's row (k <= 64: held apart)
  int p;
  if constexpr (FEW) {
    const int e = lane < k ? a.idx[t * k + lane] : -1;
    p = (unsigned)e < (unsigned)a.E ? (int)t * k + lane : -1;
    for (int j = k - 2; j >= 0; j--)
      if (p >= 0 && __builtin_amdgcn_readlane(e, j) == e && j < lane) p = (int)t * k + j;
  } else {
    p = lane < k ? a.inv[t * k + lane] : -1;
  }
  const float w = lane < k ? a.w[t * k + lane] : 0.f;
  const int ps = a.Is > 0 ? a.F + (int)t : -1;
  const float ws = a.Is > 0 ? a.shared_w[t] : 0.f;
  float acc[8];
#pragma unroll
  for (int i = 0; i < 8; i++) acc[i] = 0.f;
  for (int j0 = 0; j0 <= k; j0 += B) {
    uint4 q[B], r[B];
    int pj[B];
    float wj[B], sc[B];
#pragma unroll
    for (int j = 0; j < B; j++) {
      const int jj = j0 + j;
      pj[j] = jj < k ? __builtin_amdgcn_readlane(p, jj) : jj == k ? ps : -1;
      wj[j] = jj < k ? __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w), jj)) : ws;
      const int64_t at = (int64_t)max(pj[j], 0) * a.H + (mine ? n0 : 0);
      if constexpr (SC) sc[j] = a.oscale[(int64_t)max(pj[j], 0) * (a.H / 32) + ((mine ? n0 : 0) >> 5)];
      if constexpr (R16) {
        q[j] = mx_row16<NT>((const uint16_t*)a.obuf + at);
      } else {
        q[j] = mx_row16<NT>((const float*)a.obuf + at);
        r[j] = mx_row16<NT>((const float*)a.obuf + at + 4);
      }
    }
#pragma unroll
    for (int j = 0; j < B; j++) {
      if (pj[j] < 0) continue;
      const uint32_t u[4] = {q[j].x, q[j].y, q[j].z, q[j].w};
      float v[8];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        if constexpr (SC) {
          v[2 * i] = f16_to_f32((uint16_t)u[i]);
          v[2 * i + 1] = f16_to_f32((uint16_t)(u[i] >> 16));
        } else if constexpr (R16) {
          v[2 * i] = __uint_as_float(u[i] << 16);
          v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
        } else {
          v[i] = __uint_as_float(u[i]);
        }
      }
      if constexpr (!R16) {
        v[4] = __uint_as_float(r[j].x); v[5] = __uint_as_float(r[j].y);
        v[6] = __uint_as_float(r[j].z); v[7] = __uint_as_float(r[j].w);
      }
      const float wt = SC ? wj[j] * sc[j] : wj[j];
#pragma unroll
      for (int i = 0; i < 8; i++) acc[i] = __builtin_fmaf(wt, v[i], acc[i]);
    }
  }
  if (!mine) return;
  const int64_t at = t * a.H + n0;
  void* const base = a.resid ? a.resid : a.y;
  if constexpr (BF) {
    uint16_t* o = (uint16_t*)base + at;
    uint32_t h[4];
    if (((uintptr_t)base & 15) == 0) {
      uint32_t x[4] = {0u, 0u, 0u, 0u};
      if (a.resid) {
        const uint4 v = *(const uint4*)o;
        x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
      }
#pragma unroll
      for (int i = 0; i < 4; i++) {
        uint16_t lo = f32_to_bf16(acc[2 * i]), hi = f32_to_bf16(acc[2 * i + 1]);
        if (a.resid) {
          lo = f32_to_bf16(__uint_as_float(x[i] << 16) + bf16_to_f32(lo));
          hi = f32_to_bf16(__uint_as_float(x[i] & 0xffff0000u) + bf16_to_f32(hi));
        }
        h[i] = lo | ((uint32_t)hi << 16);
      }
      *(uint4*)o = make_uint4(h[0], h[1], h[2], h[3]);
    } else {
      for (int i = 0; i < 8; i++) mx_store(a, at + i, acc[i]);
    }
  } else {
    float* o = (float*)base + at;
    if (((uintptr_t)base & 15) == 0) {
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f), y = x;
      if (a.resid) {
        x = ((const float4*)o)[0];
        y = ((const float4*)o)[1];
      }
      // x + 0 only where there is a stream: -0 stays
      ((float4*)o)[0] = a.resid ? make_float4(x.x + acc[0], x.y + acc[1], x.z + acc[2], x.w + acc[3])
                                : make_float4(acc[0], acc[1], acc[2], acc[3]);
      ((float4*)o)[1] = a.resid ? make_float4(y.x + acc[4], y.y + acc[5], y.z + acc[6], y.w + acc[7])
                                : make_float4(acc[4], acc[5], acc[6], acc[7]);
    } else {
      for (int i = 0; i < 8; i++) mx_store(a, at + i, acc[i]);
    }
  }
}

hipError_t launch_mx_combine(const MxArgs& a, hipStream_t s) {
  const int64_t waves = (int64_t)a.T * ((a.H + 511) / 512);
  const dim3 g((unsigned)((waves + 3) / 4));
  const int64_t rows = ((int64_t)a.F + (a.Is > 0 ? a.T : 0)) * a.H * (a.xbf ? 2 : 4);   // bytes
  const bool few = a.few_rows, nt = rows > MX_CACHE;
#define COMBINE(BF, FEW, NT) hx_launch(k_mx_combine<BF, FEW, NT, false>, g, dim3(256), 0, s, a)
  if (a.oscale && !few) {
    if (nt) hx_launch(k_mx_combine<true, false, true, true>, g, dim3(256), 0, s, a);
    else hx_launch(k_mx_combine<true, false, false, true>, g, dim3(256), 0, s, a);
  } else if (a.xbf) {
    if (few) COMBINE(true, true, false);
    else if (nt) COMBINE(true, false, true);
    else COMBINE(true, false, false);
  } else {
    if (few) COMBINE(false, true, false);
    else if (nt) COMBINE(false, false, true);
    else COMBINE(false, false, false);
  }
#undef COMBINE
  return hipGetLastError();
}

}  // namespace hx
