// Per-expert counts of a routing and the router's balance loss with its gradient:
//   L = coef E sum_e f_e P_e,  f_e = k c_e / sum c,  P_e = (1 / n) sum_t p_te,  p_t = softmax(l_t)
// over the n live tokens t, those with an index in 0 .. E - 1; c_e the entries of expert e,
// taken as given. With s_t = sum_j f_j p_tj,
//   L = coef E / n sum_t s_t,   dL / dl_te = coef E / n p_te (f_e - s_t),
// so that one pass over the logits gives the loss, the means and the gradient: the counts
// come first, from the routing alone. Sums over tokens stay in a lane's registers, one a
// column, then go through LDS and a table of one row a workgroup, which a last kernel adds
// up in 64 bits: no float atomics, the same bits every time.
#include <algorithm>

#include "hx_abi.h"
#include "hx_device.h"
#include "hx_internal.h"

namespace hx {

struct BalArgs {
  const void* logits;        // [T, E]
  int64_t T;
  int E, k;
  const int32_t* idx;        // [T, k]
  const int32_t* given;      // [E] counts that f goes by, or null: the routing's own
  float coef;
  int32_t* counts;           // [E] or null
  float* probs;              // [E]
  float* loss;               // [1]
  void* dlogits;             // [T, E] or null
  int32_t* hist;             // [G1][E + 1] entries by expert, live tokens
  float* part;               // [G2][E + 1] sums of p, sum of s
  int G1, G2;
  int lpr;                   // lanes of a row, a power of two
};

// tokens a workgroup of the counts takes, and their most
constexpr int BAL_CHUNK = 1024, BAL_MAX_G1 = 64, BAL_MAX_G2 = 1024;
static int bal_g1(int64_t T) { return (int)std::min<int64_t>((T + BAL_CHUNK - 1) / BAL_CHUNK, BAL_MAX_G1); }
// the most of the row pass: a wave that takes a row at a time has two turns at least (launch_balance: rows of fewer lanes)
static int bal_g2(int64_t T) { return (int)std::max<int64_t>(1, std::min<int64_t>((T + 15) / 16, BAL_MAX_G2)); }

// hist[0 .. E - 1] += the entries by expert of tokens t0 .. t1 - 1, hist[E] += the live ones
HX_DEV void bal_count(const BalArgs& a, int64_t t0, int64_t t1, int* hist) {
  for (int64_t t = t0 + threadIdx.x; t < t1; t += blockDim.x) {
    bool live = false;
    for (int j0 = 0; j0 < a.k; j0 += 8) {   // eight loads on their way together
      int e[8];
#pragma unroll
      for (int j = 0; j < 8; j++) e[j] = j0 + j < a.k ? a.idx[t * a.k + j0 + j] : -1;
#pragma unroll
      for (int j = 0; j < 8; j++) {
        if ((unsigned)e[j] >= (unsigned)a.E) continue;
        live = true;
        atomicAdd(&hist[e[j]], 1);
      }
    }
    if (live) atomicAdd(&hist[a.E], 1);
  }
}

__global__ __launch_bounds__(1024) void k_bal_counts(BalArgs a) {
  __shared__ int hist[HX_MAX_EXPERTS + 1];
  for (int e = threadIdx.x; e <= a.E; e += 1024) hist[e] = 0;
  __syncthreads();
  const int64_t per = (a.T + a.G1 - 1) / a.G1, t0 = blockIdx.x * per;
  bal_count(a, t0, min(a.T, t0 + per), hist);
  __syncthreads();
  for (int e = threadIdx.x; e <= a.E; e += 1024) a.hist[(int64_t)blockIdx.x * (a.E + 1) + e] = hist[e];
}

// the chunks' counts of column e, eight loads on their way together
HX_DEV int bal_sum(const BalArgs& a, int e) {
  int n = 0;
  for (int g0 = 0; g0 < a.G1; g0 += 8) {
    int h[8];
#pragma unroll
    for (int i = 0; i < 8; i++) h[i] = g0 + i < a.G1 ? a.hist[(int64_t)(g0 + i) * (a.E + 1) + e] : 0;
#pragma unroll
    for (int i = 0; i < 8; i++) n += h[i];
  }
  return n;
}

__global__ __launch_bounds__(256) void k_bal_counts_sum(BalArgs a) {
  const int e = blockIdx.x * 256 + threadIdx.x;
  if (e < a.E) a.counts[e] = bal_sum(a, e);
}

// sum / maximum over the lpr lanes of a row, in all of them
HX_DEV float bal_row_sum(float v, int lpr) {
  if (lpr == 64) return wave_sum<64>(v);
  for (int off = lpr / 2; off >= 1; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}
HX_DEV float bal_row_max(float v, int lpr) {
  if (lpr == 64) return wave_max_dpp(v);
  for (int off = lpr / 2; off >= 1; off >>= 1) v = fmaxf(v, __shfl_xor(v, off, 64));
  return v;
}

// V elements at p: as they come, and their values
template <bool BF, int V>
struct BalRaw {
  static constexpr int W = V == 1 ? 1 : 4;   // words
  uint32_t u[W];
  HX_DEV void load(const void* base, int64_t at) {
    if constexpr (V == 1) {
      u[0] = BF ? (uint32_t)((const uint16_t*)base)[at] << 16 : ((const uint32_t*)base)[at];
    } else {
      const uint4 v = *(const uint4*)((const uint8_t*)base + at * (BF ? 2 : 4));
      u[0] = v.x; u[1] = v.y; u[2] = v.z; u[3] = v.w;
    }
  }
  HX_DEV void none() {   // -inf: adds nothing, is no maximum
#pragma unroll
    for (int i = 0; i < W; i++) u[i] = BF && V > 1 ? 0xff80ff80u : 0xff800000u;
  }
  HX_DEV float value(int i) const {
    if constexpr (BF && V > 1) return __uint_as_float(i & 1 ? u[i >> 1] & 0xffff0000u : u[i >> 1] << 16);
    else return __uint_as_float(u[i]);
  }
};
template <bool BF, int V>
HX_DEV void bal_store(void* base, int64_t at, const float (&f)[V]) {
  if constexpr (BF && V == 8) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; i++) u[i] = f32_to_bf16(f[2 * i]) | ((uint32_t)f32_to_bf16(f[2 * i + 1]) << 16);
    *(uint4*)((uint16_t*)base + at) = make_uint4(u[0], u[1], u[2], u[3]);
  } else if constexpr (!BF && V == 4) {
    *(float4*)((float*)base + at) = make_float4(f[0], f[1], f[2], f[3]);
  } else if constexpr (BF) {
    ((uint16_t*)base)[at] = f32_to_bf16(f[0]);
  } else {
    ((float*)base)[at] = f[0];
  }
}

// The row pass: lpr lanes a row (64 / lpr rows a wave at a time), lane j of a row its
// columns (i lpr + j) V .. + V - 1 for i < NJ. WHOLE: lpr is 64. ONE: one workgroup does it all, counts
// and last sums included. Bound by HBM and the vector instructions together (about 16 an element):
// 196608 rows of 512 in bf16, 411 MB, in 92 us (4.5 TB/s); 8192 in float32 11 us, half of it the counts' sum and the start.
template <bool BF, int V, int NJ, bool WHOLE, bool ONE>
__global__ __launch_bounds__(ONE ? 1024 : 512) void k_bal_rows(BalArgs a) {
  constexpr int NW = ONE ? 16 : 8, NT = 64 * NW;
  extern __shared__ __align__(16) float sm[];
  float* const f_of = sm;                         // [E] f
  float* const sums = sm + a.E;                   // [NW][E + 1] the waves' sums
  int* const hist = (int*)(sums + NW * (a.E + 1));   // [E + 1]
  __shared__ double total_of[NW];
  const int tid = threadIdx.x, lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(tid >> 6), E = a.E, k = a.k;
  for (int e = tid; e <= E; e += NT) hist[e] = ONE ? 0 : bal_sum(a, e);
  __syncthreads();
  if (ONE) {
    bal_count(a, 0, a.T, hist);
    __syncthreads();
  }
  const int live_n = hist[E];
  double total = 0.0;   // whole numbers: exact in any order; the counts of many devices may pass 32 bits
  for (int e = tid; e < E; e += NT) {
    total += a.given ? a.given[e] : hist[e];
    if (blockIdx.x == 0 && a.counts) a.counts[e] = hist[e];
  }
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) total += __shfl_xor(total, off, 64);
  if (lane == 0) total_of[wave] = total;
  __syncthreads();
  total = 0.0;
#pragma unroll
  for (int w = 0; w < NW; w++) total += total_of[w];
  for (int e = tid; e < E; e += NT) {
    const int c = a.given ? a.given[e] : hist[e];
    f_of[e] = total > 0.0 ? (float)((double)k * c / total) : 0.f;
  }
  __syncthreads();
  const int lpr = WHOLE ? 64 : a.lpr, rpw = 64 / lpr, sub = lane & (lpr - 1), grp = lane / lpr;
  float f[NJ][V], sum[NJ][V];
#pragma unroll
  for (int i = 0; i < NJ; i++)
#pragma unroll
    for (int v = 0; v < V; v++) {
      const int c = (i * lpr + sub) * V + v;
      f[i][v] = c < E ? f_of[c] : 0.f;
      sum[i][v] = 0.f;
    }
  const float scale = live_n > 0 ? a.coef * E / live_n : 0.f;
  float s_sum = 0.f;
  const int64_t step = (int64_t)gridDim.x * NW * rpw;
  // a row on its way while the one before is computed
  BalRaw<BF, V> next[NJ];
  bool next_mine;
  auto fetch = [&](int64_t t) {
    const bool row = t < a.T;
#pragma unroll
    for (int i = 0; i < NJ; i++) {
      const int c = (i * lpr + sub) * V;
      if (row && c < E) next[i].load(a.logits, t * E + c);
      else next[i].none();
    }
    if (WHOLE) {   // at most 64 entries
      next_mine = lane < k && (unsigned)a.idx[t * k + lane] < (unsigned)E;
    } else {
      next_mine = false;
      for (int j = sub; row && j < k; j += lpr) next_mine |= (unsigned)a.idx[t * k + j] < (unsigned)E;
    }
  };
  int64_t t0 = ((int64_t)blockIdx.x * NW + wave) * rpw;
  if (t0 < a.T) fetch(t0 + grp);
  for (; t0 < a.T; t0 += step) {
    const int64_t t = t0 + grp;
    const bool row = t < a.T;
    float x[NJ][V];
#pragma unroll
    for (int i = 0; i < NJ; i++)
#pragma unroll
      for (int v = 0; v < V; v++) x[i][v] = next[i].value(v);
    const unsigned long long any = __ballot(next_mine);
    if (t0 + step < a.T) fetch(t0 + step + grp);
    const bool live = WHOLE ? any != 0 : ((any >> (grp * lpr)) & ((1ull << lpr) - 1)) != 0;
    // a row that is not live, whatever it holds, adds nothing and has no gradient
    if (WHOLE && !live) {
      const float none[V] = {};
#pragma unroll
      for (int i = 0; i < NJ; i++)
        if (a.dlogits && (i * 64 + lane) * V < E) bal_store<BF, V>(a.dlogits, t * E + (i * 64 + lane) * V, none);
      continue;
    }
    float m = -__builtin_inff();
#pragma unroll
    for (int i = 0; i < NJ; i++)
#pragma unroll
      for (int v = 0; v < V; v++) m = fmaxf(m, x[i][v]);
    m = bal_row_max(m, lpr);
    float z = 0.f, s = 0.f;
    // exp2((x - m) log2 e): two roundings, together 2 |x - m| half steps of the result
#pragma unroll
    for (int i = 0; i < NJ; i++)
#pragma unroll
      for (int v = 0; v < V; v++) {
        x[i][v] = __builtin_amdgcn_exp2f((x[i][v] - m) * 1.44269502e+00f);
        z += x[i][v];
        s = __builtin_fmaf(f[i][v], x[i][v], s);
      }
    z = bal_row_sum(z, lpr);
    s = bal_row_sum(s, lpr);
    const float r = 1.f / z;
    s *= r;
    if (WHOLE || live) s_sum += s;
    const float ss = scale * s;
#pragma unroll
    for (int i = 0; i < NJ; i++) {
      const int c = (i * lpr + sub) * V;
      float g[V];
#pragma unroll
      for (int v = 0; v < V; v++) {
        const float p = WHOLE || live ? x[i][v] * r : 0.f;
        sum[i][v] += p;
        const float d = p * __builtin_fmaf(f[i][v], scale, -ss);
        g[v] = WHOLE || live ? d : 0.f;
      }
      if (row && a.dlogits && c < E) bal_store<BF, V>(a.dlogits, t * E + c, g);
    }
  }
  // the rows' groups, then the waves
#pragma unroll
  for (int i = 0; i < NJ; i++)
#pragma unroll
    for (int v = 0; v < V; v++) {
      for (int off = 32; off >= lpr; off >>= 1) sum[i][v] += __shfl_xor(sum[i][v], off, 64);
      const int c = (i * lpr + sub) * V + v;
      if (grp == 0 && c < E) sums[wave * (E + 1) + c] = sum[i][v];
    }
  for (int off = 32; off >= lpr; off >>= 1) s_sum += __shfl_xor(s_sum, off, 64);
  if (lane == 0) sums[wave * (E + 1) + E] = s_sum;
  __syncthreads();
  for (int e = tid; e <= E; e += NT) {
    if (ONE) {
      double v = 0.0;
      for (int w = 0; w < NW; w++) v += sums[w * (E + 1) + e];
      if (e < E) a.probs[e] = live_n > 0 ? (float)(v / live_n) : 0.f;
      else a.loss[0] = live_n > 0 ? (float)(v * a.coef * E / live_n) : 0.f;
    } else {
      float v = 0.f;
      for (int w = 0; w < NW; w++) v += sums[w * (E + 1) + e];
      a.part[(int64_t)blockIdx.x * (E + 1) + e] = v;
    }
  }
}

// the workgroups' sums: a workgroup 16 columns (of the E + 1), 64 threads a column
__global__ __launch_bounds__(1024) void k_bal_last(BalArgs a) {
  __shared__ double red[64][16];
  __shared__ int live_sm;
  const int c = threadIdx.x & 15, q = threadIdx.x >> 4, e = blockIdx.x * 16 + c;
  if (threadIdx.x == 0) live_sm = 0;
  __syncthreads();
  if (threadIdx.x < a.G1) atomicAdd(&live_sm, a.hist[(int64_t)threadIdx.x * (a.E + 1) + a.E]);
  double v = 0.0;
  if (e <= a.E)
    for (int g0 = q; g0 < a.G2; g0 += 1024) {   // sixteen loads on their way together
      float p[16];
#pragma unroll
      for (int i = 0; i < 16; i++) p[i] = g0 + 64 * i < a.G2 ? a.part[(int64_t)(g0 + 64 * i) * (a.E + 1) + e] : 0.f;
#pragma unroll
      for (int i = 0; i < 16; i++) v += p[i];
    }
  red[q][c] = v;
  __syncthreads();
  if (q == 0 && e <= a.E) {
    const int n = live_sm;
    v = 0.0;
    for (int w = 0; w < 64; w++) v += red[w][c];
    if (e < a.E) a.probs[e] = n > 0 ? (float)(v / n) : 0.f;
    else a.loss[0] = n > 0 ? (float)(v * a.coef * a.E / n) : 0.f;
  }
}

static uint32_t bal_lds(int E, int waves) { return (uint32_t)((E + (waves + 1) * (E + 1)) * 4); }

template <bool BF, int V, int NJ>
static void launch_rows(const BalArgs& a, bool one, hipStream_t s) {
  const dim3 g(one ? 1 : a.G2), b(one ? 1024 : 512);
  const uint32_t lds = bal_lds(a.E, one ? 16 : 8);
  if (a.lpr == 64) {
    if (one) hx_launch(k_bal_rows<BF, V, NJ, true, true>, g, b, lds, s, a);
    else hx_launch(k_bal_rows<BF, V, NJ, true, false>, g, b, lds, s, a);
  } else if constexpr (NJ == 1) {   // rows of fewer lanes
    if (one) hx_launch(k_bal_rows<BF, V, NJ, false, true>, g, b, lds, s, a);
    else hx_launch(k_bal_rows<BF, V, NJ, false, false>, g, b, lds, s, a);
  }
}

// Where one workgroup does it all: few tokens, entries (they are counted by atomics on one LDS) and logits,
// so that what one CU takes longer is less than what two more launches cost. us with one and with
// three, f32: 33 tokens x 512 experts, top 10, 8.0 and 10.9; 64 x 512 10.1 and 11.2; 80 x 512 11.4 and 11.1; 64 x 848 14.2
// and 13.0; 80 x 128, top 8, 9.1 and 10.5; 128 x 128 11.9 and 10.5; 128 x 16, top 4, 6.3 and 10.2.
static bool bal_one(const BalArgs& a) {
  return a.T <= 128 && a.T * a.k <= 768 && a.T * a.E <= 32768 && bal_lds(a.E, 16) <= 60 * 1024;
}

static hipError_t launch_balance(BalArgs a, bool bf, hipStream_t s) {
  const bool one = bal_one(a);
  const int per = bf ? 8 : 4;
  const bool vec = a.E % per == 0 && (((uintptr_t)a.logits | (uintptr_t)a.dlogits) & 15) == 0;
  const int chunks = vec ? a.E / per : a.E;
  a.lpr = 64;
  while (a.lpr > 1 && a.lpr / 2 >= chunks) a.lpr /= 2;
  // a wave takes 64 / lpr rows at a time: a workgroup without rows would sum the counts and leave zeros for the last
  // kernel to add. us for 16 experts in bf16, with as many workgroups as for whole waves and with these: 8192
  // tokens 15.7 and 13.5, 32768 22.2 and 15.6, 131072 26.1 and 22.0; two turns a wave here too: 14.7, 16.4, 21.0.
  const int rows = 8 * (64 / a.lpr);   // of a workgroup's waves
  a.G2 = (int)std::min<int64_t>(a.G2, std::max<int64_t>(1, (a.T + rows - 1) / rows));
  if (!one && a.T > 0) hx_launch(k_bal_counts, dim3(a.G1), dim3(1024), 0, s, a);   // no tokens: no chunks
  const int nj = (chunks + 63) / 64;
  if (bf && vec) {
    if (nj <= 1) launch_rows<true, 8, 1>(a, one, s);
    else launch_rows<true, 8, 2>(a, one, s);
  } else if (vec) {
    if (nj <= 1) launch_rows<false, 4, 1>(a, one, s);
    else if (nj <= 2) launch_rows<false, 4, 2>(a, one, s);
    else launch_rows<false, 4, 4>(a, one, s);
  } else if (bf) {
    if (nj <= 1) launch_rows<true, 1, 1>(a, one, s);
    else if (nj <= 4) launch_rows<true, 1, 4>(a, one, s);
    else launch_rows<true, 1, 16>(a, one, s);
  } else {
    if (nj <= 1) launch_rows<false, 1, 1>(a, one, s);
    else if (nj <= 4) launch_rows<false, 1, 4>(a, one, s);
    else launch_rows<false, 1, 16>(a, one, s);
  }
  if (!one) hx_launch(k_bal_last, dim3((a.E + 1 + 15) / 16), dim3(1024), 0, s, a);
  return hipGetLastError();
}

}  // namespace hx

using namespace hx;

static size_t bal_up(size_t v) { return (v + 255) & ~(size_t)255; }
static size_t bal_hist_bytes(int64_t T, int E) { return bal_up(sizeof(int32_t) * (size_t)bal_g1(T) * (E + 1)); }

static int check_balance(int64_t n_tokens, int num_experts, int k) {
  if (n_tokens < 0 || num_experts < 1 || k < 1) return fail(HX_ERR_INVALID_ARGUMENT, "bad argument");
  if (num_experts > HX_MAX_EXPERTS || k > HX_MAX_TOPK)
    return fail(HX_ERR_UNSUPPORTED, "at most %d experts and top-%d are supported", HX_MAX_EXPERTS, HX_MAX_TOPK);
  if (n_tokens > HX_MAX_TOKENS) return fail(HX_ERR_UNSUPPORTED, "too many tokens in one call");
  return HX_OK;
}

extern "C" int hx_moe_balance_workspace_size(int64_t n_tokens, int num_experts, size_t* bytes) {
  if (!bytes) return fail(HX_ERR_INVALID_ARGUMENT, "bad argument");
  int rc = check_balance(n_tokens, num_experts, 1);
  if (rc) return rc;
  *bytes = bal_hist_bytes(n_tokens, num_experts) + bal_up(sizeof(float) * (size_t)bal_g2(n_tokens) * (num_experts + 1));
  return HX_OK;
}

// the workspace of a call, checked
static int bal_args(BalArgs& a, const int32_t* topk_idx, int64_t T, int k, int E, void* ws, size_t ws_bytes) {
  size_t need;
  int rc = hx_moe_balance_workspace_size(T, E, &need);
  if (rc) return rc;
  if (!ws) return fail(HX_ERR_INVALID_ARGUMENT, "null workspace");
  if (ws_bytes < need)
    return fail(HX_ERR_WORKSPACE_TOO_SMALL, "workspace of %zu bytes, %zu needed for %lld tokens", ws_bytes, need, (long long)T);
  if ((uintptr_t)ws & 15) return fail(HX_ERR_INVALID_ARGUMENT, "the workspace must start on 16 bytes");
  a.T = T; a.E = E; a.k = k; a.idx = topk_idx;
  a.G1 = bal_g1(T); a.G2 = bal_g2(T);
  a.hist = (int32_t*)ws;
  a.part = (float*)((uint8_t*)ws + bal_hist_bytes(T, E));
  return HX_OK;
}

extern "C" int hx_moe_expert_counts(const int32_t* topk_idx, int64_t n_tokens, int k, int num_experts, int32_t* counts,
                                    void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_balance(n_tokens, num_experts, k);
  if (rc) return rc;
  if (!counts || (n_tokens > 0 && !topk_idx)) return fail(HX_ERR_INVALID_ARGUMENT, "bad argument");
  BalArgs a{};
  if ((rc = bal_args(a, topk_idx, n_tokens, k, num_experts, workspace, workspace_bytes))) return rc;
  a.counts = counts;
  hipStream_t s = (hipStream_t)stream;
  if (n_tokens > 0) hx_launch(k_bal_counts, dim3(a.G1), dim3(1024), 0, s, a);
  hx_launch(k_bal_counts_sum, dim3((num_experts + 255) / 256), dim3(256), 0, s, a);
  HX_HIP(hipGetLastError());
  return HX_OK;
}

extern "C" int hx_moe_balance_loss(const void* logits, int logits_dtype, int64_t n_tokens, int num_experts,
                                   const int32_t* topk_idx, int k, const int32_t* given_counts, float coef,
                                   float* loss, int32_t* counts, float* probs, void* dlogits, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  int rc = check_balance(n_tokens, num_experts, k);
  if (rc) return rc;
  if (!loss || !probs || (n_tokens > 0 && (!logits || !topk_idx))) return fail(HX_ERR_INVALID_ARGUMENT, "bad argument");
  if (logits_dtype != HX_F32 && logits_dtype != HX_BF16)
    return fail(HX_ERR_UNSUPPORTED, "hx_moe_balance_loss: logits dtype %d", logits_dtype);
  // one workgroup writes the routing's own counts while the others read the given ones
  if (given_counts && counts && given_counts < counts + num_experts && counts < given_counts + num_experts)
    return fail(HX_ERR_INVALID_ARGUMENT, "hx_moe_balance_loss: counts and given_counts overlap");
  // a row's gradient goes where the row was, or where no row is
  const size_t row_bytes = (size_t)n_tokens * num_experts * (logits_dtype == HX_F32 ? 4 : 2);
  if (dlogits && dlogits != logits && overlap(logits, row_bytes, dlogits, row_bytes))
    return fail(HX_ERR_INVALID_ARGUMENT, "hx_moe_balance_loss: logits and dlogits overlap in part");
  BalArgs a{};
  if ((rc = bal_args(a, topk_idx, n_tokens, k, num_experts, workspace, workspace_bytes))) return rc;
  a.logits = logits; a.given = given_counts; a.coef = coef;
  a.loss = loss; a.counts = counts; a.probs = probs; a.dlogits = dlogits;
  HX_HIP(launch_balance(a, logits_dtype == HX_BF16, (hipStream_t)stream));
  return HX_OK;
}
