// What the kernels of block-scaled experts (hx_mx.hip, hx_f8.hip) share: the routing of
// a few tokens, the experts' tiles and rows, a tile's place on the chip.
#pragma once
#include "hx_device.h"
#include "hx_mx.h"

namespace hx {

// The routing of a few tokens in LDS.
template <int MAX_T>
struct MxFewT {
  int idx[MAX_T * HX_MAX_TOPK];
  uint32_t bits[32];   // the experts that some token chose
};
template <int MAX_T>
HX_DEV void mx_few_bits(const MxArgs& a, MxFewT<MAX_T>& sm) {
  if (threadIdx.x < 32) sm.bits[threadIdx.x] = 0u;
  lds_barrier();
  for (int f = threadIdx.x; f < a.F; f += blockDim.x) {
    const int e = a.idx[f];
    sm.idx[f] = e;
    if ((unsigned)e < (unsigned)a.E) atomicOr(&sm.bits[e >> 5], 1u << (e & 31));
  }
  lds_barrier();
}
// the number of chosen experts, and (in every lane) the s-th of them in ascending
// order, -1 if there are fewer
template <int MAX_T>
HX_DEV int mx_few_slot(const MxFewT<MAX_T>& sm, int s, int& n) {
  const int l = lane_id();
  const uint32_t w = l < 32 ? sm.bits[l] : 0u;
  int c = __popc(w), x = c;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int y = __shfl_up(x, off, 64);
    if (l >= off) x += y;
  }
  n = __shfl(x, 31, 64);
  const unsigned long long hit = __ballot(l < 32 && x - c <= s && s < x);
  if (!hit) return -1;
  const int L = __ffsll(hit) - 1;
  const uint32_t word = (uint32_t)__shfl((int)w, L, 64);
  const int r = s - __shfl(x - c, L, 64);
  const unsigned long long b =
      __ballot(l < 32 && ((word >> l) & 1u) && __popc(word & ((1u << l) - 1u)) == r);
  return 32 * L + __ffsll(b) - 1;
}

// the row of h and of the outputs of token t with expert e (E: the shared one): at the
// token's first entry with it, -1 if there is none
template <int MAX_T>
HX_DEV int mx_few_row(const MxArgs& a, const MxFewT<MAX_T>& sm, int e, int t) {
  int row = e == a.E ? a.F + t : -1;
  if (e != a.E)
    for (int j = a.k - 1; j >= 0; j--)
      if (sm.idx[t * a.k + j] == e) row = t * a.k + j;
  return row;
}

// Positions of a chunk's entries by expert, and (chunk 0) the tiles, from the experts'
// counts: thread i has the counts of experts EPT i .. and how many of each come in
// earlier chunks. The entries get their places by LDS counters; their order among an
// expert's rows is free: a row's results do not depend on its place in a tile, and the
// combine sums a token's entries in their order.
struct MxPlace {
  int base[HX_MAX_EXPERTS], off[HX_MAX_EXPERTS], cnt[HX_MAX_EXPERTS], first[HX_MAX_EXPERTS];
  int sh[2][17];
};
template <int NT>
HX_DEV void mx_place(const MxArgs& a, MxPlace& sm, int c, const int (&count)[HX_MAX_EXPERTS / NT],
                     const int (&pre)[HX_MAX_EXPERTS / NT]) {
  constexpr int EPT = HX_MAX_EXPERTS / NT, NW = NT / 64;
  const int tid = threadIdx.x, lane = lane_id(), wave = tid >> 6, e0 = EPT * tid;
  int n0 = 0, n1 = 0;   // rows, tiles
#pragma unroll
  for (int i = 0; i < EPT; i++) {
    n0 += count[i];
    n1 += (count[i] + a.tile_m - 1) / a.tile_m;
  }
  int x0 = n0, x1 = n1;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int y0 = __shfl_up(x0, off, 64), y1 = __shfl_up(x1, off, 64);
    if (lane >= off) {
      x0 += y0;
      x1 += y1;
    }
  }
  if (lane == 63) {
    sm.sh[0][wave] = x0;
    sm.sh[1][wave] = x1;
  }
  __syncthreads();
  if (tid < 2) {
    int run = 0;
    for (int w = 0; w < NW; w++) {
      const int v = sm.sh[tid][w];
      sm.sh[tid][w] = run;
      run += v;
    }
    sm.sh[tid][16] = run;
  }
  __syncthreads();
  int off = sm.sh[0][wave] + x0 - n0, first = sm.sh[1][wave] + x1 - n1;
  const int total = sm.sh[1][16];
#pragma unroll
  for (int i = 0; i < EPT; i++) {
    sm.base[e0 + i] = off + pre[i];
    sm.off[e0 + i] = off;
    sm.cnt[e0 + i] = count[i];
    sm.first[e0 + i] = first;
    off += count[i];
    first += (count[i] + a.tile_m - 1) / a.tile_m;
  }
  __syncthreads();
  const int per = mx_chunk(a.F), f0 = c * per, f1 = min(a.F, f0 + per);
  for (int f = f0 + tid; f < f1; f += NT) {
    const int x = a.idx[f];
    int pos = -1;
    if ((unsigned)x < (unsigned)a.E) {
      pos = atomicAdd(&sm.base[x], 1);
      a.perm[pos] = f;
    }
    a.inv[f] = pos;
  }
  if (c != 0) return;
  for (int i = tid; i < total; i += NT) {
    int lo = 0, hi = a.E - 1;   // the largest expert with first <= i
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (sm.first[mid] <= i) lo = mid;
      else hi = mid - 1;
    }
    const int m0 = (i - sm.first[lo]) * a.tile_m;
    ((int4*)a.tiles)[i] = make_int4(lo, sm.off[lo] + m0, min(a.tile_m, sm.cnt[lo] - m0), 0);
  }
  const int nst = a.Is > 0 ? (a.T + a.tile_m - 1) / a.tile_m : 0;
  for (int i = tid; i < nst; i += NT) {
    const int m0 = i * a.tile_m;
    ((int4*)a.tiles)[total + i] = make_int4(a.E, a.F + m0, min(a.tile_m, a.T - m0), 0);
  }
  if (tid == 0) a.counts[0] = total + nst;
}

// A chunk of a prep kernel's first nch workgroups (256 threads): the chunk's entries by
// expert, and where there is one chunk alone (a launch less: about 4 us) their places too.
HX_DEV void mx_chunk_entries(const MxArgs& a, MxPlace& sm, int nch) {
  constexpr int EPT = HX_MAX_EXPERTS / 256;
  const int tid = threadIdx.x;
  for (int e = tid; e < HX_MAX_EXPERTS; e += 256) sm.cnt[e] = 0;
  __syncthreads();
  const int per = mx_chunk(a.F), f0 = blockIdx.x * per, f1 = min(a.F, f0 + per);
  for (int f = f0 + tid; f < f1; f += 256) {
    const int e = a.idx[f];
    if ((unsigned)e < (unsigned)a.E) atomicAdd(&sm.cnt[e], 1);
  }
  __syncthreads();
  if (nch > 1) {
    for (int e = tid; e < a.E; e += 256) a.hist[(int64_t)blockIdx.x * a.E + e] = sm.cnt[e];
    return;
  }
  int count[EPT], pre[EPT];
#pragma unroll
  for (int i = 0; i < EPT; i++) {
    count[i] = sm.cnt[EPT * tid + i];
    pre[i] = 0;
  }
  mx_place<256>(a, sm, 0, count, pre);
}

// workgroup -> (feature group, tile) of N tiles; tile -1: none. XCD x (workgroup id
// mod 8) takes the x-th eighth of the list in order, so that the tiles of an expert,
// which are neighbours in the list, and the NX workgroups of a tile run side by side
// on one XCD and meet each other's weights and rows in its L2. (Tiles dealt to the XCDs
// in turn: every XCD fetched every expert.)
HX_DEV void mx_tile(int NX, int N, int& nt, int& tile) {
  const int L = blockIdx.x, per = (N + 7) / 8, i = L / (8 * NX);
  nt = (L >> 3) % NX;
  tile = (L & 7) * per + i;
  if (i >= per || tile >= N) tile = -1;
}

// an output of the block, or its addition to the residual stream
HX_DEV void mx_store(const MxArgs& a, int64_t at, float y) {
  if (a.xbf) {
    uint16_t* p = (uint16_t*)(a.resid ? a.resid : a.y) + at;
    const uint16_t b = f32_to_bf16(y);
    *p = a.resid ? f32_to_bf16(bf16_to_f32(*p) + bf16_to_f32(b)) : b;
  } else {
    float* p = (float*)(a.resid ? a.resid : a.y) + at;
    *p = a.resid ? *p + y : y;
  }
}

}  // namespace hx
