// MXFP4 experts: layouts, argument block and launchers of hx_mx.hip.
//
// Stored weights. A projection matrix [rows][K] is kept as the operand tiles of
// v_mfma_scale_f32_32x32x64_f8f6f4: tile (n, s) holds rows 32 n .. + 31 and columns
// 64 s .. + 63, lane l the 32 codes of row 32 n + l % 32, columns 64 s + 32 (l / 32)
// .. + 31, in column order, low half first: 16 bytes a lane, 1 KiB a tile, loaded by
// one 16-byte load a lane straight into the MFMA's registers. The scales' exponent
// bytes follow all tiles: byte s % 4 of word ((n S4 + s / 4) 64 + l). K is padded to
// whole stages of 128 columns with codes 0 of scale 1.
//
// Activation records. A 32-wide block of a row of activations (the tokens, then h)
// is cut into P planes of E2M3 codes (4 significant bits, largest 7.5), each with its
// own power-of-two scale: S = 2^(floor(log2 amax) - 2) for the first, S 2^-3 for what
// it leaves (at most S / 2), then 2^-5 of the one before for each next. Each step leaves at
// most 2^-5 of the one before, so that three planes hold a value to S 2^-11, at most
// 2^-13 of the block's largest, and five to S 2^-21; no plane is held to less than 2^-130.
// A bf16 value below about 2^-6 of its block's largest so loses some of its bits. That is
// far below the rounding of a product with the large value; it shows only where that one's
// weight is zero, and a fourth plane would cost a third more MFMAs. The products of the
// codes are exact and the MFMA sums them in f32. A product with bf16 activations costs
// three MFMAs at the 4 / 6-bit rate (9.3 PFLOP/s measured), four times the bf16 rate: less
// than one bf16 MFMA, and no weight is ever expanded.
// A record is the first 16 of each plane's 24 bytes of codes, then the last 8 of each
// (both are loaded straight into the registers of an MFMA operand), then the P scale
// bytes; 80 bytes with three planes, 128 with five. A block with a NaN or an infinity has
// scale NaN: its token's outputs are NaN.
#pragma once
#include "hx_internal.h"

namespace hx {

constexpr int MX_STAGE = 128;                         // K columns of a stage
__host__ __device__ inline int mx_blocks(int K) { return (K + MX_STAGE - 1) / MX_STAGE * 4; }   // records of a row
__host__ __device__ inline int mx_steps(int K) { return mx_blocks(K) / 2; }                     // MFMA steps
__host__ __device__ inline int64_t mx_code_bytes(int rows, int K) { return (int64_t)(rows / 32) * mx_steps(K) * 1024; }
__host__ __device__ inline int64_t mx_mat_bytes(int rows, int K) {
  return mx_code_bytes(rows, K) + (int64_t)(rows / 32) * ((mx_steps(K) + 3) / 4) * 256;
}
__host__ __device__ inline int mx_planes(bool xbf) { return xbf ? 3 : 5; }
__host__ __device__ inline int mx_rec_bytes(bool xbf) { return xbf ? 80 : 128; }

// tokens up to which the few-token kernels may be used (mx_few)
constexpr int MX_FEW_T = 8;
constexpr int MX_FEW_TAB = 64;   // ints of a slot: the row of each of 32 columns (-1: none), the expert (-1: no work)
// entries of the routing a dispatch workgroup takes, and the most workgroups
constexpr int MX_CHUNK = 1024, MX_MAX_CHUNKS = 256;
__host__ __device__ inline int mx_chunk(int64_t F) {   // entries a chunk, a multiple of MX_CHUNK
  const int64_t n = (F + MX_CHUNK - 1) / MX_CHUNK;
  return (int)((n + MX_MAX_CHUNKS - 1) / MX_MAX_CHUNKS * MX_CHUNK);
}
__host__ __device__ inline int mx_chunks(int64_t F) { return (int)((F + mx_chunk(F) - 1) / mx_chunk(F)); }

struct MxArgs {
  WMat gate, up, down, sgate, sup, sdown;   // fmt HX_MXFP4
  int E, k, H, I, Is, T, F;                 // Is 0: no shared expert in this call
  const void* x;                            // [T, H] act dtype
  bool xbf;
  const int32_t* idx;                       // [T, k], entries outside 0 .. E - 1 are skipped
  const float* w;                           // [T, k]
  const float* shared_w;                    // [T]
  void* y;                                  // [T, H] act dtype
  void* resid;                              // or null: resid += y in place of writing y
  uint8_t* xrec;                            // [T][mx_blocks(H)] records
  uint8_t* hrec;                            // [F + T][mx_blocks(max(I, Is))] records
  int hblocks;                              // records of a row of hrec
  void* obuf;                               // [F + T, H] expert outputs, act dtype (few tokens: f32)
  float* oscale;                            // or null; [F + T][H / 32]: obuf is f16 times these
  int32_t* few;                             // [slots][MX_FEW_TAB], 2 to 8 tokens: rows of the columns, then the expert
  int32_t* perm;                            // [F] entries by expert
  int32_t* inv;                             // [F] their positions, -1: no expert
  int32_t* hist;                            // [chunks][E]
  int32_t* tiles;                           // [max_tiles][4]: expert (E: shared), first row, rows
  int32_t* counts;                          // [1] tiles
  int tile_m, max_tiles;
  bool few_rows;                            // obuf as the few-token kernels leave it
};

// whether a call of T tokens takes the few-token kernels
bool mx_few(int T, int k, int H, bool xbf);
int mx_tile_m(int64_t F, int E, bool xbf);
hipError_t launch_mx_repack(const void* src, int64_t count, int64_t rows, int64_t K, void* dst, int64_t dst_stride,
                            hipStream_t s);
hipError_t launch_mx_few_gate_up(const MxArgs& a, hipStream_t s);
hipError_t launch_mx_few_down(const MxArgs& a, hipStream_t s);
hipError_t launch_mx_prep(const MxArgs& a, hipStream_t s);       // records of the tokens, expert counts
hipError_t launch_mx_dispatch(const MxArgs& a, hipStream_t s);   // positions and tiles
hipError_t launch_mx_gate_up(const MxArgs& a, hipStream_t s);
hipError_t launch_mx_down(const MxArgs& a, hipStream_t s);
hipError_t launch_mx_combine(const MxArgs& a, hipStream_t s);

}  // namespace hx
