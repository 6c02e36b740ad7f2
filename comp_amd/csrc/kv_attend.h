// Attention over the quantized key/value cache (layout and the order of its bytes: kv_layout.h).
//
//   s_ij = scale * q_i . k_j ;  s = cap * tanh(s / cap) ;  s -= slope_h * |i - j|
//   o_i  = sum_j softmax(s)_ij v_j  over the visible j:  j < length, j <= i or j < prefix, i - j < window
//
// The columns of a wave are (query token, query head of the group) pairs that share one kv head, 16 a matrix tile; it
// walks tiles of 32 keys, with a softmax that keeps a reference M a column and rescales when a score passes it.
//
// Both products run transposed, S^T = K Q^T and O^T = V^T P^T, with the cache's codes as operand A in f16:
//   * a nibble (or byte) n, masked out of its dword, IS an f16: the subnormal n * 2^-24.  Key codes are used that way: the
//     product is exact, 2^-24 goes into the score's factor and the offset (code = n - 8) into the product's initial
//     accumulator, -8 * 2^-24 * sum(q) over the block.  Where registers are short, or many columns share the unpacking,
//     keys are signed codes ((n | 0x6400) - 1032, exact) instead, which needs no accumulators kept for it, and so do f32 queries:
//     the matrix unit sums products of subnormals with some 20 bits.
//   * a block's key scale multiplies its 32-channel partial dot in f32, so keys are not rounded at all;
//   * value codes are exact signed f16, and the value scale of (token, block) goes onto the probability: P' = P * d.
// What bounds it: few columns, by bytes (18 or 34 a block of keys and of values, once a kv head) and by vector
// instructions: 346 counted a 32-key tile of 128 4-bit channels, bf16 (630 with f32 queries and 8-bit keys), which is 1400
// cycles of a SIMD, whose share of the rate of a large read (6.85 TB/s) is the tile's bytes in 1650; many columns, by the
// softmax's instructions beside the products (kv_many.h).  Measured, 32 query heads over 8 of 128 channels, 4-bit, bf16: 64
// sequences of up to 8192 keys 85-88 us (4.2 TB/s), one of 131072 38 us (4.0 TB/s), where a read of as many bytes takes 53
// and 22 us.
// What is rounded: queries to f16 after a power of two that puts a column's largest at 2^13 (f16 and bf16 queries are
// exact, except values 2^-27 of the largest), P' to f16 (2^-12, to nearest), and for bf16 queries P before it.  f32 queries
// (PREC) are held in two f16 parts and P' in two, 22 bits each, two matrix instructions for one.  Scores, sums and
// accumulators are f32.  Relative error against 64 bits, and of f32 operations rounded once: f16 2.4e-4 and 2.1e-4 (many
// columns 2.9e-4), bf16 1.7e-3 and 1.6e-3, f32 2.8e-7 and 5.3e-7.
//
// One wave's keys are a range of tiles that no mask of its columns empties; inside it only the tiles at a mask's edge are
// masked, and there a masked key's P' is set to 0, so what a masked or unwritten place holds (NaN scales too) is not seen.
#pragma once

#include <hip/hip_ext.h>

#include <type_traits>
#include <utility>

#include "komp_device.h"
#include "komp_internal.h"
#include "kv_layout.h"

namespace komp {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

struct AttendArgs {
  KvCache c;
  const void* q;
  int64_t q_stride_t, q_stride_h;
  void* out;
  int64_t out_stride_t, out_stride_h;
  float* lse;  // [rows][heads] or null
  const int32_t* tables;
  int64_t table_stride;
  int table_cols;
  const int32_t* lengths;
  const int32_t* starts;  // null: one query a sequence
  const int32_t* prefix;  // or null
  const float* slopes;    // or null
  int64_t rows;           // query tokens in all
  int heads;
  int group;     // query heads a kv head
  int type;
  int window;
  float scale;   // times log2(e)
  float cap;     // softcap, or 0
  float twice;   // 2 / softcap
  bool wide_q;   // query rows may be loaded 16 bytes at a time
  bool wide_out; // output rows stored four elements at a time
  int splits;
  int least;     // splits of any sequence with as many tiles
  int per;       // tiles a split of longer ones
  int groups;    // column groups a sequence may have
  float* part_o;   // [split][row][head][dim]
  float2* part_m;  // [split][row][head]: M and l
};

// many: the kernel of kv_many.h; else 16 columns a workgroup.  Column groups a sequence, splits of its keys
struct AttendPlan {
  bool many;
  int groups;
  int splits;
  int least;
  int per;
};

hipError_t launch_attend_q4_q4(const AttendArgs& a, const AttendPlan& plan, int batch, hipStream_t stream);
hipError_t launch_attend_q8_q4(const AttendArgs& a, const AttendPlan& plan, int batch, hipStream_t stream);
hipError_t launch_attend_q8_q8(const AttendArgs& a, const AttendPlan& plan, int batch, hipStream_t stream);

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kAttendWaves = 4;
constexpr int many_cols(int dim, int type) { return dim == 256 ? 128 : type == KV_F32 ? 192 : 256; }  // of a workgroup of kv_many.h

template <typename T>
__device__ __forceinline__ T quarters_max(T v) {  // over the lanes of a column: lane ^ 16, lane ^ 32
  auto p = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
  v = fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
  auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float quarters_sum(float v) {
  auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(p[0]) + __uint_as_float(p[1]);
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// N dwords of a 16-, 12-, 8- or 4-byte aligned address, in loads of W
template <int N, int W>
__device__ __forceinline__ void load_words(const uint8_t* p, unsigned* out) {
  typedef unsigned int vec __attribute__((ext_vector_type(W), aligned(4)));
#pragma unroll
  for (int i = 0; i < N / W; ++i) {
    const vec v = reinterpret_cast<const vec*>(p)[i];
#pragma unroll
    for (int j = 0; j < W; ++j) out[i * W + j] = v[j];
  }
}

__device__ __forceinline__ f16x2 as_f16x2(unsigned v) { return __builtin_bit_cast(f16x2, v); }
__device__ __forceinline__ f16x8 as_f16x8(unsigned a, unsigned b, unsigned c, unsigned d) {
  const u32x4 v = {a, b, c, d};
  return __builtin_bit_cast(f16x8, v);
}
__device__ __forceinline__ unsigned pack_f16(float a, float b) {  // to nearest even
  const f32x2 v = {a, b};
  return __builtin_bit_cast(unsigned, __builtin_convertvector(v, f16x2));
}
// signed codes of two masked nibbles or bytes n: (1024 + n) - (1024 + offset), and of nibbles still shifted left by 4
__device__ __forceinline__ unsigned signed_low(unsigned masked, float offset) {
  const _Float16 o = static_cast<_Float16>(-1024.0f - offset);
  const f16x2 v = as_f16x2(masked | 0x64006400u) + f16x2{o, o};
  return __builtin_bit_cast(unsigned, v);
}
__device__ __forceinline__ unsigned signed_high(unsigned masked) {  // (1024 + 16 n) / 16 - 72 = n - 8, exact in one fma
  const f16x2 k = {static_cast<_Float16>(0.0625f), static_cast<_Float16>(0.0625f)};
  const f16x2 o = {static_cast<_Float16>(-72.0f), static_cast<_Float16>(-72.0f)};
  const f16x2 v = __builtin_elementwise_fma(as_f16x2(masked | 0x64006400u), k, o);
  return __builtin_bit_cast(unsigned, v);
}

// The visible keys of query position i are [lo, hi).
struct Span {
  int lo, hi;
};
__device__ __forceinline__ Span visible(int i, int length, int prefix, int window) {
  Span s;
  s.hi = max(0, min(length, max(i + 1, prefix)));
  s.lo = window ? max(0, i - window + 1) : 0;
  return s;
}

// Key codes of a lane's dword (Q4_0) or two (Q8_0) as operand A: subnormals (exact multiples of 2^-24; the channels of a
// high nibble 16 times that) or signed values.
template <bool SIGNED, int KF>
__device__ __forceinline__ f16x8 key_codes(unsigned w, unsigned y) {
  if constexpr (KF == KV_Q4_0) {
    const unsigned x = w >> 8;
    if constexpr (SIGNED)
      return as_f16x8(signed_low(w & 0x000F000Fu, 8.f), signed_high(w & 0x00F000F0u), signed_low(x & 0x000F000Fu, 8.f),
                      signed_high(x & 0x00F000F0u));
    return as_f16x8(w & 0x000F000Fu, w & 0x00F000F0u, x & 0x000F000Fu, x & 0x00F000F0u);
  } else {
    if constexpr (SIGNED)
      return as_f16x8(signed_low(w & 0x00FF00FFu, 128.f), signed_low(w >> 8 & 0x00FF00FFu, 128.f),
                      signed_low(y & 0x00FF00FFu, 128.f), signed_low(y >> 8 & 0x00FF00FFu, 128.f));
    return as_f16x8(w & 0x00FF00FFu, w >> 8 & 0x00FF00FFu, y & 0x00FF00FFu, y >> 8 & 0x00FF00FFu);
  }
}
// Signed value codes of a lane's two dwords (tokens 4 quarter + r, 16 + 4 quarter + r) as operand A.  Q4_0: channels c
// (half 0) or c + 16.
template <int VF>
__device__ __forceinline__ f16x8 value_codes(unsigned w0, unsigned w1, int half) {
  if constexpr (VF == KV_Q4_0) {
    const unsigned x0 = w0 >> 8, x1 = w1 >> 8;
    if (half == 0)
      return as_f16x8(signed_low(w0 & 0x000F000Fu, 8.f), signed_low(x0 & 0x000F000Fu, 8.f), signed_low(w1 & 0x000F000Fu, 8.f),
                      signed_low(x1 & 0x000F000Fu, 8.f));
    return as_f16x8(signed_high(w0 & 0x00F000F0u), signed_high(x0 & 0x00F000F0u), signed_high(w1 & 0x00F000F0u),
                    signed_high(x1 & 0x00F000F0u));
  } else {
    return as_f16x8(signed_low(w0 & 0x00FF00FFu, 128.f), signed_low(w0 >> 8 & 0x00FF00FFu, 128.f),
                    signed_low(w1 & 0x00FF00FFu, 128.f), signed_low(w1 >> 8 & 0x00FF00FFu, 128.f));
  }
}

// lane I of each 16 lanes, in all of them
template <int I>
__device__ __forceinline__ unsigned row_lane(unsigned v) {
  return __builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x150 | I, 0xF, 0xF, true);  // (no lane keeps an old value)
}

// One 32-key tile as it lies in a wave's registers.  The scales that a quarter needs are the same in its 16 lanes: each
// lane loads one dword of them, and a DPP broadcast hands it to the row where it is used, which costs 8 NB instructions a
// tile and saves 8 NB - 2 registers a tile in flight.
template <int NB, int KF, int VF>
struct KvTile {
  static constexpr int KW = NB * kv_code_bytes(KF) / 16;  // key dwords a lane of each 16 tokens
  static constexpr int VW = NB * kv_code_bytes(VF) / 8;   // value dwords a lane
  static constexpr int SW = (4 * NB + 15) / 16;           // scale dwords a lane
  unsigned kc[2][KW];
  unsigned ks[SW];  // of a quarter, t * 2 NB + j: halves 2 j and 2 j + 1 of its 4 keys of the 16 tokens t (r * NB + b)
  unsigned vc[VW];
  unsigned vs[SW];  // of a quarter, 4 b + i: its tokens' pair i of block b

  __device__ __forceinline__ void load(const KvCache& c, int64_t unit, int lane) {
    constexpr int kbd = kv_kb(NB, KF) * (KF == KV_Q8_0 ? 2 : 1);  // dwords of one load
    constexpr int vbd = kv_vb(NB, VF) * (VF == KV_Q8_0 ? 4 : 2);
    const int quarter = lane >> 4;
    const uint8_t* k = c.kq + unit * (NB * 32 * kv_code_bytes(KF));
    const uint8_t* v = c.vq + unit * (NB * 32 * kv_code_bytes(VF));
    const unsigned* ksp = reinterpret_cast<const unsigned*>(c.ks) + unit * (16 * NB);
    const unsigned* vsp = reinterpret_cast<const unsigned*>(c.vs) + unit * (16 * NB);
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < KW / kbd; ++i)
        load_words<kbd, kbd>(k + (t * KW * 64 + i * kbd * 64 + lane * kbd) * 4, &kc[t][i * kbd]);
#pragma unroll
    for (int i = 0; i < SW; ++i) {
      const int at = min(i * 16 + (lane & 15), 4 * NB - 1), t = at / (2 * NB);
      ks[i] = ksp[t * 8 * NB + quarter * 2 * NB + at - t * 2 * NB];
      vs[i] = vsp[quarter * 4 * NB + at];
    }
#pragma unroll
    for (int i = 0; i < VW / vbd; ++i) load_words<vbd, vbd>(v + (i * vbd * 64 + lane * vbd) * 4, &vc[i * vbd]);
  }
  // key codes of tokens 16 t ..., block b: operand A, as subnormals (exact multiples of 2^-24; the channels of a high
  // nibble 16 times that) or signed
  template <bool SIGNED>
  __device__ __forceinline__ f16x8 key(int t, int b) const {
    if constexpr (KF == KV_Q4_0) {
      return key_codes<SIGNED, KF>(kc[t][b], 0u);
    } else {
      return key_codes<SIGNED, KF>(kc[t][2 * b], kc[t][2 * b + 1]);
    }
  }
  // signed value codes of block b, channels 16 half ...: operand A
  __device__ __forceinline__ f16x8 value(int b, int half) const {
    if constexpr (VF == KV_Q4_0) return value_codes<VF>(vc[2 * b], vc[2 * b + 1], half);
    return value_codes<VF>(vc[4 * b + 2 * half], vc[4 * b + 2 * half + 1], half);
  }
};

// channel (in its quarter's 8) of a key operand's place e
template <int KF>
__device__ constexpr int key_place(int e) {
  // Q4_0: nibbles 0,4 1,5 2,6 3,7; Q8_0: bytes 0,2 1,3 of each dword
  constexpr int n4[8] = {0, 4, 1, 5, 2, 6, 3, 7};
  constexpr int n8[8] = {0, 2, 1, 3, 4, 6, 5, 7};
  return KF == KV_Q4_0 ? n4[e] : n8[e];
}

// four consecutive channels of an output row
__device__ __forceinline__ void store_out(void* out, int type, bool wide, int64_t i, f32x4 o) {
  typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));
  if (type == KV_F32) {
    float* p = static_cast<float*>(out) + i;
    if (wide) {
      *reinterpret_cast<f32x4*>(p) = o;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) p[e] = o[e];
    }
    return;
  }
  u16x4 u;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    u[e] = type == KV_F16 ? __builtin_bit_cast(uint16_t, static_cast<_Float16>(o[e]))
                          : __builtin_bit_cast(uint16_t, static_cast<__bf16>(o[e]));
  uint16_t* p = static_cast<uint16_t*>(out) + i;
  if (wide) {
    *reinterpret_cast<u16x4*>(p) = u;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) p[e] = u[e];
  }
}

// What a call asks of one (sequence, kv head): its rows, its keys, and the visible ones.
struct Sequence {
  int64_t row0;
  int cols;    // columns: rows * group
  int length;  // keys
  int shift;   // position of the first row
  int prefix;
  __device__ __forceinline__ Sequence(const AttendArgs& a, int seq) {
    row0 = a.starts ? a.starts[seq] : seq;
    const int64_t row1 = a.starts ? a.starts[seq + 1] : seq + 1;
    // rows past the query tensor do not exist, whatever `starts` says
    const int count = row0 < 0 || row1 > a.rows || row1 < row0 ? 0 : static_cast<int>(row1 - row0);
    length = max(int64_t{0}, min(static_cast<int64_t>(a.lengths[seq]), static_cast<int64_t>(a.table_cols) << a.c.page_log2));
    shift = a.lengths[seq] - count;
    cols = count * a.group;
    prefix = a.prefix ? a.prefix[seq] : 0;
  }
  __device__ __forceinline__ Span seen(const AttendArgs& a, int token) const {
    return visible(shift + token, length, prefix, a.window);
  }
};

// A wave's columns and their softmax: queries, references and sums.  MODE: the type of the queries.  SIGNED: how it takes
// key codes.
template <int NB, int KF, int VF, int MODE, int CT, bool SIGNED>
struct Columns {
  static constexpr int COLS = 16 * CT;
  static constexpr bool PREC = MODE == KV_F32;
  static constexpr int PARTS = PREC ? 2 : 1;
  static constexpr int OT = 2 * NB;  // 16-channel tiles of the output
  static constexpr float NONE = -__builtin_inff();
  static constexpr float UNSEEN = 0x1p127f;  // neg before anything was seen: any score is above its reference, and masked ones give 0
  // M moves to a column's largest score less this, and moves again when a score is 8 above that: P is 2^(ROOM + 8) at most,
  // and P' = P d below 2^15 for value scales of exponent fields up to 21 - ROOM.  Keys with larger ones leave less room.
  static constexpr int ROOM = PREC ? 20 : 6;

  Span all;           // keys that some column sees
  Span span[CT];      // of the lane's columns
  int pos[CT];
  f16x8 qf[CT][NB][PARTS];
  f32x4 init[SIGNED ? 1 : NB];
  float fx[CT];       // of y, the raw or capped and biased score, to log2 units
  float raw[CT];      // of the raw score to log2 units, when it is capped or biased
  float slope[CT];
  f32x4 acc[CT][OT];
  float neg[CT];      // -M, or UNSEEN
  float l[CT];
  int room;           // of the tiles so far (Columns::step)

  // the lane's column ct: its query row and head; false where there is none
  __device__ __forceinline__ bool place(const AttendArgs& a, const Sequence& s, int h, int col0, int ct, int lane,
                                        int64_t& row, int& head) const {
    const int c = col0 + ct * 16 + (lane & 15);
    const int token = c < s.cols ? c / a.group : 0;
    row = s.row0 + token;
    head = h * a.group + (c < s.cols ? c - token * a.group : 0);
    return c < s.cols;
  }

  // M of column ct (-inf before anything was seen)
  __device__ __forceinline__ float reference(int ct) const { return neg[ct] == UNSEEN ? NONE : -neg[ct]; }

  // a lane's query channels, as they are in memory: the loads are under way before the keys', which take longer
  struct Raw {
    u32x4 w[CT][NB][PREC ? 2 : 1];
  };
  __device__ __forceinline__ void fetch(const AttendArgs& a, const Sequence& s, int h, int col0, int lane, Raw& q) const {
    const int quarter = lane >> 4;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      int64_t row;
      int head;
      const bool live = place(a, s, h, col0, ct, lane, row, head);
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const int64_t at = row * a.q_stride_t + head * a.q_stride_h + b * 32 + quarter * 8;
#pragma unroll
        for (int i = 0; i < (PREC ? 2 : 1); ++i) q.w[ct][b][i] = u32x4{0, 0, 0, 0};
        if (!live) continue;
        if (a.wide_q) {
          const u32x4* p = PREC ? reinterpret_cast<const u32x4*>(static_cast<const float*>(a.q) + at)
                                : reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(a.q) + at);
#pragma unroll
          for (int i = 0; i < (PREC ? 2 : 1); ++i) q.w[ct][b][i] = p[i];
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            if constexpr (PREC) q.w[ct][b][e >> 2][e & 3] = static_cast<const unsigned*>(a.q)[at + e];
            else q.w[ct][b][0][e >> 1] |= static_cast<unsigned>(static_cast<const uint16_t*>(a.q)[at + e]) << (16 * (e & 1));
          }
        }
      }
    }
  }

  __device__ __forceinline__ void begin(const AttendArgs& a, const Sequence& s, int h, int col0, int lane, const Raw& q) {
    room = ROOM;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      int64_t row;
      int head;
      const bool live = place(a, s, h, col0, ct, lane, row, head);
      pos[ct] = s.shift + static_cast<int>(row - s.row0);
      span[ct] = live ? s.seen(a, static_cast<int>(row - s.row0)) : Span{0, 0x7FFFFFFF};  // no column: never masked or stored
      slope[ct] = a.slopes ? a.slopes[head] * kLog2e : 0.f;
      // queries: f16 parts, scaled so that a column's largest is in [2^13, 2^14)
      float v[NB][8];
      float top = 0.f;
      const float sign = a.scale < 0.f ? -1.f : 1.f;
#pragma unroll
      for (int b = 0; b < NB; ++b) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const unsigned w = PREC ? q.w[ct][b][PREC ? e >> 2 : 0][e & 3] : q.w[ct][b][0][e >> 1];
          const unsigned u = e & 1 ? w >> 16 : w & 0xFFFFu;
          const float x = PREC            ? __uint_as_float(w)
                          : MODE == KV_F16 ? static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(u)))
                                           : __uint_as_float(u << 16);
          top = fmaxf(top, fabsf(x));
          v[b][e] = x * sign;
        }
      }
      top = quarters_max(top);
      int up = 0;  // 2^up brings the largest to [2^13, 2^14); none for 0, infinity and NaN
      if (top > 0.f && top < __builtin_inff()) up = 13 - (static_cast<int>(__builtin_amdgcn_frexp_expf(top)) - 1);
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float x = __builtin_ldexpf(v[b][key_place<KF>(e)], up);
          const bool high = !SIGNED && KF == KV_Q4_0 && (e & 2);  // meets 16 times its code
          const float y = high ? x * 0.0625f : x;
          const _Float16 hi = static_cast<_Float16>(y);
          qf[ct][b][0][e] = hi;
          if constexpr (PREC) qf[ct][b][1][e] = static_cast<_Float16>(y - static_cast<float>(hi));
          sum += high ? static_cast<float>(hi) * 16.f : static_cast<float>(hi);
        }
        if constexpr (!SIGNED) {
          const float o = (KF == KV_Q4_0 ? -8.f : -128.f) * 0x1p-24f * quarters_sum(sum);
          init[b] = f32x4{o, o, o, o};
        }
      }
      const float unit = __builtin_ldexpf(fabsf(a.scale), (SIGNED ? 0 : 24) - up);
      raw[ct] = unit;
      fx[ct] = a.cap > 0.f || a.slopes ? 1.f : fmaxf(unit, 0x1p-126f);
      neg[ct] = UNSEEN;
      l[ct] = 0.f;
#pragma unroll
      for (int i = 0; i < OT; ++i) acc[ct][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
  }

  // Capped and biased scores from raw ones.  With s the score in log2 units and v = 2 s / cap, tanh(score / cap) = tanh(v ln2 /
  // 2) is 1 - 2 / (2^v + 1), whose two terms cancel where |v| is small; there the capped score is s (1 + z P(z)), z = v^2, P
  // fitted to tanh(u) / u on |u| <= 1/2 (relative error 2^-25.9, coefficients times (ln2 / 2)^2k).  A wave whose scores are
  // all that small, as with most caps in use, computes nothing else.
  __device__ __forceinline__ void shape(const AttendArgs& a, int ct, int key0, float unit, float (&y)[2][4]) const {
    constexpr float BEND = kLog2e;  // |v| of |u| = 1/2
    const float back = static_cast<float>(pos[ct] - key0), to = raw[ct] * unit;
    bool bent = false;
    if (a.cap > 0.f) {
      float most = 0.f;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) most = fmaxf(most, fabsf(y[t][r]));
      bent = __builtin_amdgcn_ballot_w64(most * to * a.twice > BEND) != 0;
    }
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float x = y[t][r] * to;
        if (a.cap > 0.f) {
          const float v = x * a.twice, z = v * v;
          const float p = fmaf(fmaf(fmaf(0x1.e1ab3p-19f, z, -0x1.818ceap-14f), z, 0x1.f7fc2cp-10f), z, -0x1.47fcc6p-5f);
          const float low = fmaf(x * z, p, x);
          if (bent) {
            const float one = fmaf(-2.f, __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(v) + 1.f), 1.f);
            x = fabsf(v) > BEND ? a.cap * one * kLog2e : low;
          } else {
            x = low;
          }
        }
        y[t][r] = fmaf(-slope[ct], fabsf(back - (16 * t + r)), x);
      }
  }

  // The columns' room over 32 keys of which some are masked, whose value scales lie as in KvTile::vs: of each column, by the
  // finite scales that it sees, so that a large one that it does not see takes no bits from it.
  __device__ __forceinline__ void settle(const unsigned (&vs)[(4 * NB + 15) / 16], int key0, int (&own)[CT]) const {
    unsigned keep[CT][4];
    int top[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      seen_pairs(ct, key0, keep[ct]);
      top[ct] = 21 - ROOM;
    }
    each<4 * NB>([&](auto nc) {
      constexpr int at = nc.value;
      const unsigned d = row_lane<at % 16>(vs[at / 16]);
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        const unsigned w = d & keep[ct][at & 3];
        const int lo = w >> 10 & 31, hi = w >> 26 & 31;
        top[ct] = max(top[ct], max(lo == 31 ? 0 : lo, hi == 31 ? 0 : hi));
      }
    });
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) own[ct] = 21 - static_cast<int>(quarters_max(static_cast<float>(top[ct])));
  }

  // Where a column's largest score has left its room, M moves there, and what was summed with it.
  __device__ __forceinline__ void move(const int (&own)[CT], float unit, const float (&y)[CT][2][4]) {
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      float top = y[ct][0][0];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) top = fmaxf(top, y[ct][t][r]);
      top = quarters_max(top * (fx[ct] * unit));
      const float to = top + neg[ct] > own[ct] + 8 ? own[ct] - top : neg[ct];
      // (nothing seen yet: nothing to rescale)
      const float by = neg[ct] == UNSEEN ? 0.f : __builtin_amdgcn_exp2f(to - neg[ct]);
      l[ct] *= by;
#pragma unroll
      for (int i = 0; i < OT; ++i) acc[ct][i] *= by;
      neg[ct] = to;
    }
  }

  // Raw scores (in the tile's unit) to probabilities 2^(x - M + ev), and the sums of 2^(x - M).  `left`: the room that the
  // tile's value scales leave, seen or not.  `scales`: them, or nothing where they are in the operands.
  template <typename S>
  __device__ __forceinline__ void soften(const AttendArgs& a, bool masked, int key0, int left, float unit, int ev, float (&y)[CT][2][4],
                                         S&& scales) {
    const bool shaped = a.cap > 0.f || a.slopes != nullptr;
    bool go = false;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      if (shaped) shape(a, ct, key0, unit, y[ct]);
      if (masked) {  // (2^(-inf fx - M) is 0: fx is not)
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int j = key0 + 16 * t + r;
            if (j < span[ct].lo || j >= span[ct].hi) y[ct][t][r] = NONE;
          }
      }
    }
    if (shaped) unit = 1.f;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      const float top = fmaxf(fmaxf(fmaxf(y[ct][0][0], y[ct][0][1]), fmaxf(y[ct][0][2], y[ct][0][3])),
                              fmaxf(fmaxf(y[ct][1][0], y[ct][1][1]), fmaxf(y[ct][1][2], y[ct][1][3])));
      go |= fmaf(top, fx[ct] * unit, neg[ct]) > left + 8;
    }
    if (__builtin_amdgcn_ballot_w64(go) != 0) {
      int own[CT];
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) own[ct] = left;
      if constexpr (!std::is_same_v<std::decay_t<S>, std::nullptr_t>) {
        if (masked) settle(scales(), key0, own);
      }
      move(own, unit, y);
    }
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      const float f = fx[ct] * unit, n = neg[ct] + ev;
      float sum = 0.f;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          y[ct][t][r] = __builtin_amdgcn_exp2f(fmaf(y[ct][t][r], f, n));
          sum += y[ct][t][r];
        }
      l[ct] += __builtin_ldexpf(sum, -ev);
    }
  }

  // probabilities in f16, in the order of the value codes' places
  __device__ __forceinline__ static void pack(const float (&p)[2][4], unsigned (&w)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = pack_f16(p[i >> 1][i & 1], p[i >> 1][2 + (i & 1)]);
  }
  // masks of the pairs of keys that column ct sees
  __device__ __forceinline__ void seen_pairs(int ct, int key0, unsigned (&keep)[4]) const {
    auto in = [&](int j) { return j >= span[ct].lo && j < span[ct].hi; };
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int j = key0 + 16 * (i >> 1) + (i & 1);
      keep[i] = (in(j) ? 0xFFFFu : 0u) | (in(j + 2) ? 0xFFFF0000u : 0u);
    }
  }
  // P' = P * d of a pair of keys, in f16 parts
  __device__ __forceinline__ static void weigh(float p0, float p1, f16x2 d, unsigned (&w)[PARTS][4], int i) {
    const float y0 = p0 * static_cast<float>(d[0]), y1 = p1 * static_cast<float>(d[1]);
    w[0][i] = pack_f16(y0, y1);
    if constexpr (PREC) {
      const f16x2 hi = as_f16x2(w[0][i]);
      w[PARTS - 1][i] = pack_f16(y0 - static_cast<float>(hi[0]), y1 - static_cast<float>(hi[1]));
    }
  }

  // Queries of 8 blocks in shared memory (one column tile, the same for all waves): 32 registers, or 64 in two parts, that a
  // wave beside its tile and sums does not have.
  static constexpr bool SHARED_QUERIES = NB == 8 && CT == 1;
  typedef f16x8 Queries[NB * PARTS][64];
  __device__ __forceinline__ void share(Queries& to, int lane) const {
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int p = 0; p < PARTS; ++p) to[b * PARTS + p][lane] = qf[0][b][p];
  }

  // A tile of 32 keys from key `first` on.  masked: some column does not see some of them; a key that a column does not
  // see gets a P' of 0 there whatever its scale holds.
  __device__ __forceinline__ void step(const AttendArgs& a, const KvTile<NB, KF, VF>& kv, const Queries* shared, bool masked, int first,
                                       int lane) {
    const int quarter = lane >> 4, key0 = first + quarter * 4;
    float y[CT][2][4];
    if constexpr (SHARED_QUERIES) {
      static_assert(SIGNED, "the accumulators begin at zero");
      int at = lane;
      asm volatile("" : "+v"(at));  // (read here, a tile at a time: held over the loop they would take their registers again)
      each<NB / 2>([&](auto gc) {
        constexpr int g = gc.value;
        f32x4 c[2][2] = {};
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int p = 0; p < PARTS; ++p) {
            const f16x8 q = (*shared)[(2 * g + b) * PARTS + p][at];
#pragma unroll
            for (int t = 0; t < 2; ++t)
              c[t][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kv.template key<SIGNED>(t, 2 * g + b), q, c[t][b], 0, 0, 0);
          }
        each<8>([&](auto rc) {
          constexpr int t = rc.value / 4, r = rc.value % 4, i = t * 2 * NB + r * NB / 2 + g;  // (dword of row r, blocks 2 g and 2 g + 1)
          const f16x2 d = as_f16x2(row_lane<i % 16>(kv.ks[i / 16]));
          y[0][t][r] = g == 0 ? static_cast<float>(d[0]) * c[t][0][r] : fmaf(static_cast<float>(d[0]), c[t][0][r], y[0][t][r]);
          y[0][t][r] = fmaf(static_cast<float>(d[1]), c[t][1][r], y[0][t][r]);
        });
      });
    } else each<2>([&](auto tc) {
      constexpr int t = tc.value;
      f32x4 c[CT][NB];
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const f16x8 k = kv.template key<SIGNED>(t, b);
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
          c[ct][b] = SIGNED ? f32x4{0.f, 0.f, 0.f, 0.f} : init[SIGNED ? 0 : b];
#pragma unroll
          for (int p = 0; p < PARTS; ++p) c[ct][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, qf[ct][b][p], c[ct][b], 0, 0, 0);
        }
      }
      each<2 * NB>([&](auto jc) {
        constexpr int j = jc.value, at = t * 2 * NB + j;
        const f16x2 d = as_f16x2(row_lane<at % 16>(kv.ks[at / 16]));
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          constexpr int i0 = 2 * j;
          const int r = (i0 + e) / NB, b = (i0 + e) % NB;
#pragma unroll
          for (int ct = 0; ct < CT; ++ct)
            y[ct][t][r] = b == 0 ? static_cast<float>(d[e]) * c[ct][b][r] : fmaf(static_cast<float>(d[e]), c[ct][b][r], y[ct][t][r]);
        }
      });
    });
    // larger value scales may leave less room; the scales of keys that no column sees are not looked at
    unsigned vs[KvTile<NB, KF, VF>::SW];
    bool above = false;
#pragma unroll
    for (int i = 0; i < KvTile<NB, KF, VF>::SW; ++i) {
      vs[i] = kv.vs[i];
      if (masked) {
        const int pair = min(i * 16 + (lane & 15), 4 * NB - 1) & 3, j = key0 + 16 * (pair >> 1) + (pair & 1);
        vs[i] &= (j >= all.lo && j < all.hi ? 0xFFFFu : 0u) | (j + 2 >= all.lo && j + 2 < all.hi ? 0xFFFF0000u : 0u);
      }
      const unsigned lo = vs[i] & 0x7C00u, hi = vs[i] >> 16 & 0x7C00u, most = static_cast<unsigned>(21 - room) << 10;
      above |= (lo > most && lo != 0x7C00u) || (hi > most && hi != 0x7C00u);
    }
    if (__builtin_amdgcn_ballot_w64(above) != 0) {
      unsigned e = 0;  // the largest finite scale's exponent field
#pragma unroll
      for (int i = 0; i < KvTile<NB, KF, VF>::SW; ++i) {
        const unsigned lo = vs[i] >> 10 & 31, hi = vs[i] >> 26 & 31;
        e = max(e, max(lo == 31 ? 0u : lo, hi == 31 ? 0u : hi));
      }
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) e = max(e, static_cast<unsigned>(__shfl_xor(static_cast<int>(e), o, 64)));
      room = __builtin_amdgcn_readfirstlane(min(room, 21 - static_cast<int>(max(e, 1u))));
    }
    soften(a, masked, key0, room, 1.f, 0, y, [&]() -> auto& { return vs; });
    unsigned ph[CT][4], keep[CT][4];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      if constexpr (MODE == KV_BF16) pack(y[ct], ph[ct]);
      if (masked) seen_pairs(ct, key0, keep[ct]);
    }
    each<NB>([&](auto bc) {
      constexpr int b = bc.value;
      unsigned w[CT][PARTS][4];
      each<4>([&](auto ic) {
        constexpr int i = ic.value, at = 4 * b + i;
        const f16x2 d = as_f16x2(row_lane<at % 16>(vs[at / 16]));
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
          if constexpr (MODE == KV_BF16) {
            w[ct][0][i] = __builtin_bit_cast(unsigned, as_f16x2(ph[ct][i]) * d);
          } else {
            weigh(y[ct][i >> 1][i & 1], y[ct][i >> 1][2 + (i & 1)], d, w[ct], i);
          }
          if (masked) {
#pragma unroll
            for (int part = 0; part < PARTS; ++part) w[ct][part][i] &= keep[ct][i];
          }
        }
      });
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const f16x8 v = kv.value(b, half);
#pragma unroll
        for (int ct = 0; ct < CT; ++ct)
#pragma unroll
          for (int part = 0; part < PARTS; ++part)
            acc[ct][2 * b + half] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                v, as_f16x8(w[ct][part][0], w[ct][part][1], w[ct][part][2], w[ct][part][3]), acc[ct][2 * b + half], 0, 0, 0);
      }
    });
  }

  // the parts of a split without keys
  __device__ __forceinline__ void store_none(const AttendArgs& a, const Sequence& s, int h, int col0, int split, int lane) const {
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      int64_t row;
      int head;
      if (place(a, s, h, col0, ct, lane, row, head)) a.part_m[(split * a.rows + row) * a.heads + head] = float2{NONE, 0.f};
    }
  }

  // the columns' results, or their part of a split
  __device__ __forceinline__ void store(const AttendArgs& a, const Sequence& s, int h, int col0, int split, int lane) const {
    constexpr int D = NB * 32;
    const int quarter = lane >> 4;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      int64_t row;
      int head;
      if (!place(a, s, h, col0, ct, lane, row, head)) continue;
      const float M = reference(ct);
      if (a.splits > 1) {
        const int64_t at = (split * a.rows + row) * a.heads + head;
        if (lane < 16) a.part_m[at] = float2{M, l[ct]};
        if (M == NONE) continue;
#pragma unroll
        for (int i = 0; i < OT; ++i)
          *reinterpret_cast<f32x4*>(a.part_o + at * D + i * 16 + quarter * 4) = acc[ct][i];
      } else {
        const float inv = l[ct] == 0.f ? 0.f : 1.f / l[ct];
        if (a.lse && lane < 16)
          a.lse[row * a.heads + head] = l[ct] == 0.f ? NONE : (M + __log2f(l[ct])) * (1.f / kLog2e);
        const int64_t at = row * a.out_stride_t + head * a.out_stride_h + quarter * 4;
#pragma unroll
        for (int i = 0; i < OT; ++i) store_out(a.out, MODE, a.wide_out, at + i * 16, acc[ct][i] * inv);
      }
    }
  }
};

// The pages of a sequence and head: where a tile of 32 keys lies, in units of 32 tokens of a page and head; -1 for a page
// that the cache does not have.
struct Pages {
  const int32_t* table;
  int64_t pages;
  int heads, h, log2;
  __device__ __forceinline__ Pages(const AttendArgs& a, int seq, int h)
      : table(a.tables + seq * a.table_stride), pages(a.c.pages), heads(a.c.heads), h(h), log2(a.c.page_log2 - 5) {}
  __device__ __forceinline__ int64_t unit(int tile) const {
    const int page = table[tile >> log2];
    const int64_t u = ((static_cast<int64_t>(page) * heads + h) << log2) + (tile & ((1 << log2) - 1));
    return ((page < 0) | (page >= pages)) ? -1 : u;
  }
};

// Few columns over many keys: the waves of a workgroup have the same 16 columns and share its keys out among them, a tile
// each in turn; they join their sums in shared memory.  Registers decide how it hides the memory's latency: 3 waves a SIMD
// (4 of 64 channels, 2 of 256, or 1 with f32 queries) with one tile in flight each, or for 8-bit tiles, twice as large, 2 waves
// with two.  256 channels, 64 sequences of up to 8192 keys, 32 heads over 4: 4-bit 102 us (f32 queries 128), 8-bit 138 (209).
// No kernel may spill registers (the compiler has stored a spilled one where only some lanes were on, and all lanes read it
// again: wild addresses): 256 channels have their queries in shared memory.
template <int NB, int KF, int VF, int MODE>
struct Few {
  static constexpr int DEEP = KF == KV_Q8_0 && VF == KV_Q8_0 && NB <= 4 ? 2 : 1;
  static constexpr int WAVES = NB == 2 ? 4 : NB == 8 ? (MODE == KV_F32 ? 1 : 2) : NB == 4 && DEEP == 2 ? 2 : 3;  // a SIMD
  static constexpr bool SIGNED = NB == 8;  // (the subnormals' accumulators would take 32 registers)
};
template <int NB, int KF, int VF, int MODE>
__global__ void __launch_bounds__(kAttendWaves * 64, (Few<NB, KF, VF, MODE>::WAVES)) kv_attend_few_kernel(const AttendArgs a) {
  constexpr int W = kAttendWaves, DEEP = Few<NB, KF, VF, MODE>::DEEP, CT = 1;
  using Cols = Columns<NB, KF, VF, MODE, CT, (Few<NB, KF, VF, MODE>::SIGNED || MODE == KV_F32)>;
  constexpr int COLS = Cols::COLS, OT = Cols::OT;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int h = blockIdx.y, seq = blockIdx.z;
  // Workgroups go round the XCDs in order.  So that the first groups and splits, which are never empty, do not all meet on
  // the same ones, a sequence and head begins with a group and split of its own (16 sequences of 1-5 rows, f32, with 1024
  // workgroups, half of them second groups, mostly empty: 50 us without, 41 with).
  const int parts = a.groups * a.splits, place = parts == 1 ? 0 : static_cast<int>(blockIdx.x + h + seq) % parts;
  const int split = a.groups == 1 ? place : place / a.groups, col0 = (place - split * a.groups) * COLS;
  const Sequence s(a, seq);
  if (col0 >= s.cols) return;
  Cols cols;
  const Span s0 = s.seen(a, col0 / a.group), s1 = s.seen(a, (min(s.cols, col0 + COLS) - 1) / a.group);
  // the workgroup's tiles, and those of them that all columns see
  int tile0 = s0.lo >> 5, tile1 = (s1.hi + 31) >> 5;
  if (tile0 > tile1) tile0 = tile1 = 0;
  if (a.splits > 1) {
    // pieces of a length that the plan sets, but `least` of a sequence, and no more than there are splits
    const int n = tile1 - tile0, per = max((n + a.splits - 1) / a.splits, min((n + a.least - 1) / a.least, a.per));
    tile0 = min(tile1, tile0 + split * per);
    tile1 = min(tile1, tile0 + per);
    if (tile0 == tile1) {  // nothing for this one
      if (wave == 0 && lane < 16) cols.store_none(a, s, h, col0, split, lane);
      return;
    }
  }
  typename Cols::Raw query;
  cols.fetch(a, s, h, col0, lane, query);
  int full0 = max(tile0, (s1.lo + 31) >> 5), full1 = min(tile1, s0.hi >> 5);
  if (full0 >= full1) full0 = full1 = tile1;

  __shared__ f32x4 so[W / 2][OT][64];  // the waves' sums on their way to each other; until then, the queries
  __shared__ float2 sm[W / 2][16];
  auto* const queries = reinterpret_cast<typename Cols::Queries*>(so);
  cols.all = Span{s0.lo, s1.hi};
  if constexpr (Cols::SHARED_QUERIES) {
    static_assert(sizeof(typename Cols::Queries) <= sizeof(so), "the queries fit");
    cols.begin(a, s, h, col0, lane, query);
    if (wave == 0) cols.share(*queries, lane);
    __syncthreads();
  }
  const Pages pages(a, seq, h);
  KvTile<NB, KF, VF> kv[DEEP];
  int64_t unit[DEEP];
#pragma unroll
  for (int i = 0; i < DEEP; ++i) {
    const int tile = full0 + wave + i * W;
    unit[i] = tile < full1 ? pages.unit(tile) : -1;
    if (unit[i] >= 0) kv[i].load(a.c, unit[i], lane);
  }
  if constexpr (!Cols::SHARED_QUERIES) cols.begin(a, s, h, col0, lane, query);
  for (int tile = full0 + wave; tile < full1; tile += DEEP * W) {
#pragma unroll
    for (int i = 0; i < DEEP; ++i) {
      const int now = tile + i * W, next = now + DEEP * W;
      if (unit[i] >= 0) cols.step(a, kv[i], queries, false, now * 32, lane);
      unit[i] = next < full1 ? pages.unit(next) : -1;
      if (unit[i] >= 0) kv[i].load(a.c, unit[i], lane);
    }
  }
  // the tiles at the masks' edges: before the full ones, and after them
  const int before = min(full0, tile1) - tile0, edges = before + tile1 - full1;
  for (int e = wave; e < edges; e += W) {
    const int tile = e < before ? tile0 + e : full1 + e - before;
    const int64_t u = pages.unit(tile);
    if (u < 0) continue;
    KvTile<NB, KF, VF> one;
    one.load(a.c, u, lane);
    cols.step(a, one, queries, true, tile * 32, lane);
  }

  // join the waves, a column tile at a time: the upper half hands its sums to the lower half, then wave 1 to wave 0
  if constexpr (Cols::SHARED_QUERIES) __syncthreads();
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    float M = cols.reference(ct);
    cols.l[ct] = quarters_sum(cols.l[ct]);
#pragma unroll
    for (int half = W / 2; half >= 1; half >>= 1) {
      if (wave >= half && wave < 2 * half) {
        if (lane < 16) sm[wave - half][lane] = float2{M, cols.l[ct]};
#pragma unroll
        for (int i = 0; i < OT; ++i) so[wave - half][i][lane] = cols.acc[ct][i];
      }
      __syncthreads();
      if (wave < half) {
        const float2 other = sm[wave][lane & 15];
        const float top = fmaxf(M, other.x);
        const float f0 = M == Cols::NONE ? 0.f : __builtin_amdgcn_exp2f(M - top);
        const float f1 = other.x == Cols::NONE ? 0.f : __builtin_amdgcn_exp2f(other.x - top);
        cols.l[ct] = cols.l[ct] * f0 + other.y * f1;
        M = top;
#pragma unroll
        for (int i = 0; i < OT; ++i) cols.acc[ct][i] = cols.acc[ct][i] * f0 + so[wave][i][lane] * f1;
      }
      __syncthreads();
    }
    cols.neg[ct] = M == Cols::NONE ? Cols::UNSEEN : -M;
  }
  if (wave == 0) cols.store(a, s, h, col0, split, lane);
}

}  // namespace komp
