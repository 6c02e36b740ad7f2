// Layout of the quantized key/value cache, shared by the kernels that write, read and attend over it.
//
// A cache has pages of `page` tokens (a multiple of 32, a power of two).  For each page and kv head the codes and the
// f16 scales of the page's keys, and of its values, lie together.  Keys come in tiles of 16 tokens and values in tiles of
// 32, ordered as the matrix instruction's operands (v_mfma_f32_16x16x32_f16: lane 16 q + i holds row i, contraction
// places 8 q .. 8 q + 7), so that a wave reads a tile with full-width contiguous loads and uses every dword where it
// lands:
//   keys    operand A of S^T = K Q^T: row = token of the 16, contraction = a block's 32 channels; quarter q of the wave
//           holds channels 8 q .. 8 q + 7 of each block.  Q4_0: channel 8 q + e in bits 4 e of one dword; Q8_0: in byte e
//           of two.  KB blocks lie side by side in a lane's load.
//   values  operand A of O^T = V^T P^T: row = channel, contraction = tokens; quarter q holds the tokens 4 q + r and
//           16 + 4 q + r (r = 0..3), which are the rows of S^T that the same lane holds, so the probabilities go from the
//           softmax into the second product without leaving their lane.  Q4_0: byte 4 t + r of the 8-byte group (block,
//           q, channel c < 16) holds channel c of token 16 t + 4 q + r in its low nibble and channel c + 16 in its high
//           one (no byte is shared by two tokens, so a token is written without reading).  Q8_0: two such groups.
//   scales  keys: [token of the 16][block]; values: [quarter][block][8 tokens, in the order r = 0, 2, 1, 3 of each four:
//           the order in which masks and shifts take a dword's bytes apart]
// A Q4_0 code is stored as ggml's nibble (value + 8), a Q8_0 code as value + 128 (an unsigned byte).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>
#include <utility>

namespace komp {

// f(integral_constant<int, 0>{}) .. f(integral_constant<int, N - 1>{})
template <typename F, int... I>
__device__ __forceinline__ void each_impl(F&& f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void each(F&& f) {
  each_impl(static_cast<F&&>(f), std::make_integer_sequence<int, N>{});
}

enum KvFmt { KV_Q4_0 = 0, KV_Q8_0 = 2 };  // Fmt's values
enum KvType { KV_F32 = 0, KV_F16 = 1, KV_BF16 = 2 };

struct KvCache {
  uint8_t* kq;
  uint16_t* ks;
  uint8_t* vq;
  uint16_t* vs;
  int64_t pages;
  int heads;
  int dim;
  int page;
  int page_log2;
  int kf;
  int vf;
};

// code bytes of a block of 32
__host__ __device__ constexpr int kv_code_bytes(int fmt) { return fmt == KV_Q8_0 ? 32 : 16; }

// blocks that lie side by side in one lane's load of key codes, and of value codes
__host__ __device__ constexpr int kv_kb(int nb, int fmt) {
  return fmt == KV_Q8_0 ? (nb % 2 == 0 ? 2 : 1) : nb % 4 == 0 ? 4 : nb % 3 == 0 ? 3 : nb % 2 == 0 ? 2 : 1;
}
__host__ __device__ constexpr int kv_vb(int nb, int fmt) { return fmt == KV_Q8_0 ? 1 : nb % 2 == 0 ? 2 : 1; }

// Dword of the 16-token key tile that holds channels 8 quarter + 4 half .. of block b (Q4_0: `half` selects the 16 bits
// inside it).
__host__ __device__ inline int kv_k_dword(int nb, int fmt, int token16, int b, int quarter, int half) {
  const int kb = kv_kb(nb, fmt);
  const int lane = (b / kb) * 64 + quarter * 16 + token16;
  return fmt == KV_Q8_0 ? (lane * kb + b % kb) * 2 + half : lane * kb + b % kb;
}
// Byte of the 32-token value tile that holds channel c (0..15) of block b, and of channel c + 16 for Q8_0's half 1.
__host__ __device__ inline int kv_v_byte(int nb, int fmt, int token32, int b, int c, int half) {
  const int t = token32 >> 4, quarter = (token32 >> 2) & 3, r = token32 & 3;
  const int vb = kv_vb(nb, fmt);
  const int group = ((b / vb) * 64 + quarter * 16 + c) * vb + b % vb;
  return (fmt == KV_Q8_0 ? group * 2 + half : group) * 8 + t * 4 + r;
}
__host__ __device__ inline int kv_k_scale(int nb, int token16, int b) { return token16 * nb + b; }
__host__ __device__ inline int kv_v_scale(int nb, int token32, int b) {
  const int t = token32 >> 4, quarter = (token32 >> 2) & 3, r = token32 & 3;
  return (quarter * nb + b) * 8 + t * 4 + ((r & 1) << 1 | r >> 1);
}

// ---- the operators' calls (abi.hip's checked arguments) --------------------------------------------------------------
struct KvWriteCall {
  KvCache cache;
  const void* k;
  const void* v;
  int type;
  const int64_t* slots;
  int64_t tokens;
  int64_t stride_t[2];  // keys, values: elements between tokens and between heads
  int64_t stride_h[2];
};
struct KvReadCall {
  KvCache cache;
  const int64_t* slots;
  int64_t tokens;
  void* k;  // [tokens][heads][dim]
  void* v;
  int type;
};
struct KvAttendCall {
  KvCache cache;
  const void* q;
  int64_t q_stride_t, q_stride_h;
  void* out;
  int64_t out_stride_t, out_stride_h;
  float* lse;
  int type;
  const int32_t* tables;
  int64_t table_stride;
  int table_cols;
  const int32_t* lengths;
  const int32_t* starts;
  const int32_t* prefix;
  const float* slopes;
  int64_t rows;
  int batch;
  int heads;
  int64_t max_queries;
  int64_t max_length;
  float scale;
  float softcap;
  int window;
  void* work;
  int64_t work_bytes;
};
hipError_t launch_kv_write(const KvWriteCall& w, hipStream_t stream);
hipError_t launch_kv_read(const KvReadCall& r, hipStream_t stream);
// bytes of workspace that the attention call needs (0: none)
int64_t kv_attend_work_bytes(const KvAttendCall& c);
hipError_t launch_kv_attend(const KvAttendCall& c, hipStream_t stream);

}  // namespace komp
