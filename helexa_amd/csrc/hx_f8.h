// Products of E4M3 weights and activations with a float32 scale for each block of 128:
// layouts, argument blocks and launchers of hx_f8.hip.
//
// The caller's form: codes [rows][K], one byte each, scales [ceil(rows / 128)][ceil(K / 128)].
//
// Stored weights. A matrix is kept as the operand tiles of v_mfma_f32_16x16x128_f8f6f4:
// tile (n, b) holds rows 16 n .. + 15 and the columns of block b, in two halves of 1 KiB;
// half h, lane l: the 16 codes of row 16 n + l % 16, columns 128 b + 64 h + 16 (l / 16) .. + 15,
// so that one 16-byte load a lane fills four of the operand's registers. (Which of the
// instruction's k a byte is does not matter as long as both operands agree.) A row of tiles
// is contiguous along K. K is padded to whole blocks and the rows to whole tiles with zero
// codes. The scales follow, f8_scale_row(K) floats a row of blocks.
//
// Quantised activations: [rows][f8_blocks(K) 128] codes, zeros behind K, and
// [rows][f8_scale_row(K)] scales.
#pragma once
#include "hx_internal.h"
#include "hx_mx.h"

namespace hx {

__host__ __device__ inline int f8_blocks(int64_t K) { return (int)((K + 127) / 128); }
__host__ __device__ inline int f8_tiles(int64_t rows) { return (int)((rows + 15) / 16); }
__host__ __device__ inline int f8_scale_row(int64_t K) { return (f8_blocks(K) + 3) / 4 * 4; }   // floats: whole 16 bytes
__host__ __device__ inline int64_t f8_code_bytes(int64_t rows, int64_t K) {
  return (int64_t)f8_tiles(rows) * f8_blocks(K) * 2048;
}
__host__ __device__ inline int64_t f8_mat_bytes(int64_t rows, int64_t K) {
  return f8_code_bytes(rows, K) + (int64_t)f8_blocks(rows) * f8_scale_row(K) * 4;
}
// bytes of a row of quantised activations
__host__ __device__ inline int64_t f8_row(int64_t K) { return (int64_t)f8_blocks(K) * 128; }

// tokens up to which a block takes the few-token kernels: an MFMA's 16 columns
constexpr int F8_FEW_T = 16;
// rows up to which a layer takes the few-row kernel, and blocks of rows up to which that one and the
// few-token gate/up quantise them themselves (f8_quant_inside)
constexpr int F8_FEW_ROWS = 48, F8_QUANT_BLOCKS = 80;

// experts: MxArgs with xrec and hrec the quantised rows of x and h, hblocks the blocks of
// a row of h
struct F8Args : MxArgs {
  float* xs;      // [T][f8_scale_row(H)]
  float* hs;      // [F + T][hscale]
  float* hf;      // few tokens: [F + T][hcols] h in f32
  int hscale, hcols;
};

struct F8LinearArgs {
  const uint8_t* w;      // stored weights
  const void* x;         // [M, K]
  bool xbf, ybf;
  int64_t M;
  int N, K;
  void* y;               // [M, N]
  uint8_t* xq;           // [M][f8_row(K)]
  float* xs;             // [M][f8_scale_row(K)]
};

hipError_t launch_f8_repack(const void* codes, const float* scales, int64_t count, int64_t rows, int64_t K, void* dst,
                            int64_t dst_stride, hipStream_t s);
// rows of x quantised by 1 x 128; padded: to the layout of quantised activations, else to the caller's
hipError_t launch_f8_rows(const void* x, bool xbf, int64_t rows, int64_t cols, void* codes, float* scales, bool padded,
                          hipStream_t s);
hipError_t launch_f8_blocks(const void* x, bool xbf, int64_t rows, int64_t cols, void* codes, float* scales, hipStream_t s);
bool f8_quant_inside(int64_t M, int64_t K);
// features (and rows, if not exact) of a tile of a layer of more than F8_FEW_ROWS rows: 256, 128, 64, or 0: 64 with K
// shared by two groups of waves
int f8_linear_tile(int64_t M, int64_t N, bool exact);
hipError_t launch_f8_linear(const F8LinearArgs& a, hipStream_t s);

bool f8_few(int T);
int f8_tile_m(int64_t T, int64_t F, int E, int H, bool xbf);   // rows of a tile
hipError_t launch_f8_few_gate_up(const F8Args& a, hipStream_t s);
hipError_t launch_f8_few_down(const F8Args& a, hipStream_t s);
hipError_t launch_f8_prep(const F8Args& a, hipStream_t s);
hipError_t launch_f8_gate_up(const F8Args& a, hipStream_t s);
hipError_t launch_f8_down(const F8Args& a, hipStream_t s);

}  // namespace hx
