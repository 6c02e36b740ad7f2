// Microscaled rows: their layout in memory, and the calls of the operators over them (comp_amd.mx).
//
// A row of K elements (K a multiple of 32) is K e2m1 or e4m3 elements and one scale byte s a block of 32, which stands for
// 2^(s - 127); s = 255 makes the block NaN.  Rows lie in tiles of 16, and a tile is cut along K into steps of 128 elements:
// the operands of one matrix instruction v_mfma_scale_f32_16x16x128_f8f6f4.  Lane l = 16 g + r of a wave holds block g
// (32 elements) of row r:
//   codes   e2m1: [row tile][step][lane][16 bytes] (element e in nibble e, the low one of a byte first)
//           e4m3: [row tile][step][half of the block][lane][16 bytes]
//   scales  [row tile][four steps][lane][4 bytes]: one dword a lane holds its blocks' scales of four steps
// so a wave loads any operand with contiguous 1 KB loads and each byte is used in the lane where it lands: 4.25 (8.25) bits
// an element, nothing to turn.  Rows and blocks behind the last ones of a tile are zeros (scale byte 0, 2^-127).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace komp {

enum MxFmt { MX_E2M1 = 0, MX_E4M3 = 1 };
enum MxType { MX_F32 = 0, MX_F16 = 1, MX_BF16 = 2 };
enum MxAct { MX_PLAIN = 0, MX_SILU = 1, MX_RELU2 = 2 };

struct MxRows {
  uint8_t* codes;
  uint8_t* scales;
  int64_t rows;
  int64_t k;
  int fmt;
};

__host__ __device__ inline int64_t mx_tiles(int64_t rows) { return (rows + 15) >> 4; }
__host__ __device__ inline int64_t mx_steps(int64_t k) { return (k + 127) >> 7; }
__host__ __device__ inline int64_t mx_supers(int64_t k) { return (k + 511) >> 9; }
// bytes of a row tile
__host__ __device__ inline int64_t mx_code_bytes(int64_t k, int fmt) { return mx_steps(k) << (fmt == MX_E4M3 ? 11 : 10); }
__host__ __device__ inline int64_t mx_scale_bytes(int64_t k) { return mx_supers(k) << 8; }

// rows from X [rows][k] (act MX_PLAIN), or from X [rows][2 k]: the gates, then the values that they multiply
struct MxQuantCall {
  MxRows r;
  const void* x;
  int type;
  int64_t stride;
  int act;
};

// rows[ids[t]] * factor (ids NULL: rows[t]) -> OUT [count][k]
struct MxLookupCall {
  MxRows r;
  const int64_t* ids;
  int64_t count;
  void* out;
  int type;
  int64_t stride;
  float factor;
};

// rows <-> plain planes: codes [rows][k / 2 or k], scales [rows][k / 32]; ggml: codes are 17-byte block_mxfp4 blocks
struct MxPackCall {
  MxRows r;
  uint8_t* codes;
  uint8_t* scales;
  bool ggml;
  bool unpack;
};

// Y [x rows][w rows] = x w^T; x either quantized rows (src NULL) or src [x.rows][k], quantized to x.fmt on the way
struct MxGemmCall {
  MxRows x;
  MxRows w;
  const void* src;
  int src_type;
  int64_t src_stride;
  void* y;
  int type;
  int64_t stride;
};

// The kernel that a product runs on, and the tiles of 16 rows of W and of X that a workgroup has at once.
enum MxKernel { MX_STEP = 0, MX_STREAM = 1, MX_TILE = 2 };
struct MxGemmPlan {
  MxKernel kernel;
  int row_tiles;
  int col_tiles;
};
MxGemmPlan mx_gemm_plan(int64_t t, int64_t n, int64_t k);

constexpr int kMxLinearRows = 16;  // rows that one launch quantizes on the way: one column tile

hipError_t launch_mx_quantize(const MxQuantCall& c, hipStream_t stream);
hipError_t launch_mx_lookup(const MxLookupCall& c, hipStream_t stream);
hipError_t launch_mx_pack(const MxPackCall& c, hipStream_t stream);
hipError_t launch_mx_gemm(const MxGemmCall& c, hipStream_t stream);

}  // namespace komp
