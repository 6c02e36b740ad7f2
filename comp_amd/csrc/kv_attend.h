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
//     accumulator, -8 * 2^-24 * sum(q) over the block (one column).  Several columns share the unpacking and take
//     signed codes ((n | 0x6400) - 1032, exact) instead, which needs no accumulators kept for it, and so do f32 queries:
//     the matrix unit sums products of subnormals with some 20 bits.
//   * a block's key scale multiplies its 32-channel partial dot in f32, so keys are not rounded at all;
//   * value codes are exact signed f16, and the value scale of (token, block) goes onto the probability: P' = P * d.
// What is rounded: queries to f16 after a power of two that puts a column's largest at 2^13 (f16 and bf16 queries are
// exact, except values 2^-27 of the largest), P and P' to f16 (2^-12 each, to nearest).  f32 queries (PREC) are held in
// two f16 parts and P' in two, 22 bits each, two matrix instructions for one.  Scores, sums and accumulators are f32.
//
// One wave's keys are a range of tiles that no mask of its columns empties; inside it only the tiles at a mask's edge are
// masked, and there a masked key's P' is set to 0, so what a masked or unwritten place holds (NaN scales too) is not seen.
#pragma once

#include <hip/hip_ext.h>

#include <type_traits>

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
  bool wide_q;   // query rows may be loaded 16 bytes at a time
  bool wide_out; // output rows stored four elements at a time
  int splits;
  int groups;    // column groups a sequence may have
  float* part_o;   // [split][row][head][dim]
  float2* part_m;  // [split][row][head]: M and l
};

// column tiles of 16 a wave, own columns a wave or shared ones, column groups a sequence, splits of its keys
struct AttendPlan {
  int ct;
  bool wide;
  int groups;
  int splits;
};

hipError_t launch_attend_q4_q4(const AttendArgs& a, const AttendPlan& plan, int batch, hipStream_t stream);
hipError_t launch_attend_q8_q4(const AttendArgs& a, const AttendPlan& plan, int batch, hipStream_t stream);
hipError_t launch_attend_q8_q8(const AttendArgs& a, const AttendPlan& plan, int batch, hipStream_t stream);

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kAttendWaves = 4;

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

template <int N>
struct Words {
  unsigned w[N];
};
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

// One 32-key tile as it lies in a lane's registers.
template <int NB, int KF, int VF>
struct KvTile {
  static constexpr int KW = NB * kv_code_bytes(KF) / 16;  // key dwords a lane of each 16 tokens
  static constexpr int VW = NB * kv_code_bytes(VF) / 8;   // value dwords a lane
  unsigned kc[2][KW];
  unsigned ks[2][2 * NB];  // the f16 scales of keys 4 quarter + r: half r * NB + b
  unsigned vc[VW];
  unsigned vs[4 * NB];  // of the lane's 8 tokens, block by block

  __device__ __forceinline__ void load(const KvCache& c, int64_t unit, int lane) {
    constexpr int kbd = kv_kb(NB, KF) * (KF == KV_Q8_0 ? 2 : 1);  // dwords of one load
    constexpr int vbd = kv_vb(NB, VF) * (VF == KV_Q8_0 ? 4 : 2);
    const int quarter = lane >> 4;
    const uint8_t* k = c.kq + unit * (NB * 32 * kv_code_bytes(KF));
    const uint8_t* v = c.vq + unit * (NB * 32 * kv_code_bytes(VF));
    const uint8_t* ksp = reinterpret_cast<const uint8_t*>(c.ks) + unit * (64 * NB);
    const uint8_t* vsp = reinterpret_cast<const uint8_t*>(c.vs) + unit * (64 * NB);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int i = 0; i < KW / kbd; ++i)
        load_words<kbd, kbd>(k + (t * KW * 64 + i * kbd * 64 + lane * kbd) * 4, &kc[t][i * kbd]);
      load_words<2 * NB, NB % 2 == 0 ? 4 : 2>(ksp + t * 32 * NB + quarter * 8 * NB, ks[t]);
    }
#pragma unroll
    for (int i = 0; i < VW / vbd; ++i) load_words<vbd, vbd>(v + (i * vbd * 64 + lane * vbd) * 4, &vc[i * vbd]);
    load_words<4 * NB, 4>(vsp + quarter * 16 * NB, vs);
  }
  // key codes of tokens 16 t ..., block b: operand A, as subnormals (exact multiples of 2^-24; the channels of a high
  // nibble 16 times that) or signed
  template <bool SIGNED>
  __device__ __forceinline__ f16x8 key(int t, int b) const {
    if constexpr (KF == KV_Q4_0) {
      const unsigned w = kc[t][b], x = w >> 8;
      if constexpr (SIGNED)
        return as_f16x8(signed_low(w & 0x000F000Fu, 8.f), signed_high(w & 0x00F000F0u), signed_low(x & 0x000F000Fu, 8.f),
                        signed_high(x & 0x00F000F0u));
      return as_f16x8(w & 0x000F000Fu, w & 0x00F000F0u, x & 0x000F000Fu, x & 0x00F000F0u);
    } else {
      const unsigned w = kc[t][2 * b], x = kc[t][2 * b + 1];
      if constexpr (SIGNED)
        return as_f16x8(signed_low(w & 0x00FF00FFu, 128.f), signed_low(w >> 8 & 0x00FF00FFu, 128.f),
                        signed_low(x & 0x00FF00FFu, 128.f), signed_low(x >> 8 & 0x00FF00FFu, 128.f));
      return as_f16x8(w & 0x00FF00FFu, w >> 8 & 0x00FF00FFu, x & 0x00FF00FFu, x >> 8 & 0x00FF00FFu);
    }
  }
  __device__ __forceinline__ float key_scale(int t, int r, int b) const {
    const int i = r * NB + b;
    return static_cast<float>(as_f16x2(ks[t][i >> 1])[i & 1]);
  }
  // signed value codes of block b, channels 16 half ...: operand A
  __device__ __forceinline__ f16x8 value(int b, int half) const {
    if constexpr (VF == KV_Q4_0) {
      const unsigned w0 = vc[2 * b], w1 = vc[2 * b + 1], x0 = w0 >> 8, x1 = w1 >> 8;
      if (half == 0)
        return as_f16x8(signed_low(w0 & 0x000F000Fu, 8.f), signed_low(x0 & 0x000F000Fu, 8.f),
                        signed_low(w1 & 0x000F000Fu, 8.f), signed_low(x1 & 0x000F000Fu, 8.f));
      return as_f16x8(signed_high(w0 & 0x00F000F0u), signed_high(x0 & 0x00F000F0u), signed_high(w1 & 0x00F000F0u),
                      signed_high(x1 & 0x00F000F0u));
    } else {
      const unsigned w0 = vc[4 * b + 2 * half], w1 = vc[4 * b + 2 * half + 1];
      return as_f16x8(signed_low(w0 & 0x00FF00FFu, 128.f), signed_low(w0 >> 8 & 0x00FF00FFu, 128.f),
                      signed_low(w1 & 0x00FF00FFu, 128.f), signed_low(w1 >> 8 & 0x00FF00FFu, 128.f));
    }
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

__device__ __forceinline__ float load_query(const void* q, int type, int64_t i) {
  if (type == KV_F32) return static_cast<const float*>(q)[i];
  const uint16_t u = static_cast<const uint16_t*>(q)[i];
  return type == KV_F16 ? static_cast<float>(__builtin_bit_cast(_Float16, u)) : __uint_as_float(static_cast<unsigned>(u) << 16);
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

// `WIDE`: the workgroup's waves have columns of their own and walk the same keys; else they have the same columns and
// share the keys out among them.
template <int NB, int KF, int VF, bool PREC, int CT, bool WIDE>
__global__ void __launch_bounds__(kAttendWaves * 64, 2) kv_attend_kernel(const AttendArgs a) {
  constexpr int W = kAttendWaves, D = NB * 32, COLS = 16 * CT;
  constexpr bool SIGNED = CT > 1 || PREC;
  constexpr int PARTS = PREC ? 2 : 1;
  constexpr int OT = 2 * NB;  // 16-channel tiles of the output
  const int lane = threadIdx.x & 63, quarter = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int h = blockIdx.y, seq = blockIdx.z;
  const int split = blockIdx.x / a.groups;
  const int grp = blockIdx.x - split * a.groups;
  const int64_t row0 = a.starts ? a.starts[seq] : seq;
  const int64_t row1 = a.starts ? a.starts[seq + 1] : seq + 1;
  // rows past the query tensor do not exist, whatever `starts` says
  const int count = row0 < 0 || row1 > a.rows || row1 < row0 ? 0 : static_cast<int>(row1 - row0);
  const int length = max(0, min(static_cast<int64_t>(a.lengths[seq]), static_cast<int64_t>(a.table_cols) << a.c.page_log2));
  const int shift = a.lengths[seq] - count;  // position of the sequence's first query
  const int cols = count * a.group;
  const int col0 = (WIDE ? grp * W + wave : grp) * COLS;
  if (col0 >= cols) return;  // (the same for all waves where they join)
  const int prefix = a.prefix ? a.prefix[seq] : 0;

  // this lane's columns
  Span span[CT];
  int64_t row[CT];
  int head[CT];
  int pos[CT];
  bool live[CT];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const int c = col0 + ct * 16 + (lane & 15);
    live[ct] = c < cols;
    const int token = live[ct] ? c / a.group : 0;
    head[ct] = h * a.group + (live[ct] ? c - token * a.group : 0);
    row[ct] = row0 + token;
    pos[ct] = shift + token;
    span[ct] = visible(pos[ct], length, prefix, a.window);
    if (!live[ct]) span[ct] = Span{0, 0x7FFFFFFF};  // no column: never masked, never stored
  }
  // the wave's keys: from its first token's window to its last token's last key, and where all of them see every key
  const int first_token = col0 / a.group, last_token = (min(cols, col0 + COLS) - 1) / a.group;
  const Span s0 = visible(shift + first_token, length, prefix, a.window);
  const Span s1 = visible(shift + last_token, length, prefix, a.window);
  int tile0 = s0.lo >> 5, tile1 = (s1.hi + 31) >> 5;
  if (tile0 > tile1) tile0 = tile1 = 0;
  const int full_lo = s1.lo, full_hi = s0.hi;
  if (a.splits > 1) {
    const int per = (tile1 - tile0 + a.splits - 1) / a.splits;
    tile0 = min(tile1, tile0 + split * per);
    tile1 = min(tile1, tile0 + per);
  }
  constexpr int STEP = WIDE ? 1 : W;
  if (!WIDE) tile0 += wave;

  // queries: f16 parts, scaled so that a column's largest is in [2^13, 2^14)
  f16x8 qf[CT][NB][PARTS];
  f32x4 init[SIGNED ? 1 : NB];
  float factor[CT];  // of the raw score, towards log2 units
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    float v[NB][8];
    float top = 0.f;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const int64_t at = row[ct] * a.q_stride_t + head[ct] * a.q_stride_h + b * 32 + quarter * 8;
      if (!live[ct]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[b][e] = 0.f;
      } else if (a.wide_q) {
        if (a.type == KV_F32) {
          const f32x4* p = reinterpret_cast<const f32x4*>(static_cast<const float*>(a.q) + at);
          const f32x4 x = p[0], y = p[1];
#pragma unroll
          for (int e = 0; e < 4; ++e) v[b][e] = x[e], v[b][4 + e] = y[e];
        } else {
          const u32x4 x = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(a.q) + at);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const unsigned u = e & 1 ? x[e >> 1] >> 16 : x[e >> 1] & 0xFFFFu;
            v[b][e] = a.type == KV_F16 ? static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(u)))
                                       : __uint_as_float(u << 16);
          }
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[b][e] = load_query(a.q, a.type, at + e);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(v[b][e]));
    }
    top = quarters_max(top);
    int up = 0;  // 2^up brings the largest to [2^13, 2^14); none for 0, infinity and NaN
    if (top > 0.f && top < __builtin_inff()) up = 13 - (static_cast<int>(__builtin_amdgcn_frexp_expf(top)) - 1);
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      float sum = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int ch = key_place<KF>(e);
        float x = __builtin_ldexpf(v[b][ch], up);
        const bool high = !SIGNED && KF == KV_Q4_0 && (e & 2);  // meets 16 times its code
        const float y = high ? x * 0.0625f : x;
        const _Float16 hi = static_cast<_Float16>(y);
        qf[ct][b][0][e] = hi;
        float used = static_cast<float>(hi);
        if constexpr (PREC) {
          const _Float16 lo = static_cast<_Float16>(y - used);
          qf[ct][b][1][e] = lo;
          used += static_cast<float>(lo);
        }
        sum += high ? used * 16.f : used;
      }
      if constexpr (!SIGNED) {
        const float off = (KF == KV_Q4_0 ? -8.f : -128.f) * 0x1p-24f * quarters_sum(sum);
        init[b] = f32x4{off, off, off, off};
      }
    }
    factor[ct] = __builtin_ldexpf(a.cap > 0.f ? 2.f * a.scale / a.cap : a.scale, (SIGNED ? 0 : 24) - up);
  }
  const float cap2 = a.cap * kLog2e;
  float slope[CT];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) slope[ct] = a.slopes ? a.slopes[head[ct]] * kLog2e : 0.f;

  // P = 2^(x - M), M = max - off.  A score may pass the max by 8 before M moves, so P <= 2^(8 + off), and P' stays below
  // 2^15 with value scales below 2^(7 - off).  P in f16 allows off = 6, which serves scales below 2; f32 queries, whose P'
  // is a product in f32, begin higher, so that P' of small scales keeps its bits.  Larger scales lower it.
  int off = PREC ? 20 : 6;
  f32x4 acc[CT][OT];
  float M[CT], lim[CT], l[CT];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    M[ct] = -__builtin_inff();
    lim[ct] = -__builtin_inff();
    l[ct] = 0.f;
#pragma unroll
    for (int i = 0; i < OT; ++i) acc[ct][i] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  const int tiles_log2 = a.c.page_log2 - 5;
  const int32_t* table = a.tables + seq * a.table_stride;
  // the unit (32 tokens of a page and head) of a tile, or -1 for a page that the cache does not have
  auto unit_of = [&](int tile) -> int64_t {
    const int page = table[tile >> tiles_log2];
    if (page < 0 || page >= a.c.pages) return -1;
    return ((static_cast<int64_t>(page) * a.c.heads + h) << tiles_log2) + (tile & ((1 << tiles_log2) - 1));
  };

  auto step = [&](const KvTile<NB, KF, VF>& kv, int tile, auto masked_c) {
    constexpr bool MASKED = decltype(masked_c)::value;
    const int key0 = tile * 32 + quarter * 4;
    float x[CT][2][4];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const f16x8 k = kv.template key<SIGNED>(t, b);
        float d[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) d[r] = kv.key_scale(t, r, b);
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
          f32x4 c = SIGNED ? f32x4{0.f, 0.f, 0.f, 0.f} : init[SIGNED ? 0 : b];
#pragma unroll
          for (int p = 0; p < PARTS; ++p) c = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, qf[ct][b][p], c, 0, 0, 0);
#pragma unroll
          for (int r = 0; r < 4; ++r) x[ct][t][r] = b == 0 ? d[r] * c[r] : fmaf(d[r], c[r], x[ct][t][r]);
        }
      }
    }
    // the scales of keys that no column sees are not looked at (they may hold anything)
    unsigned vs[4 * NB];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      unsigned m = 0xFFFFFFFFu;
      if constexpr (MASKED) {
        auto in = [&](int r) {
          const int j = key0 + 16 * (i >> 1) + r;
          return j >= s0.lo && j < s1.hi;
        };
        m = (in(i & 1) ? 0xFFFFu : 0u) | (in(2 + (i & 1)) ? 0xFFFF0000u : 0u);
      }
#pragma unroll
      for (int b = 0; b < NB; ++b) vs[4 * b + i] = kv.vs[4 * b + i] & m;
    }
    // larger scales may need a lower `off`: f32 queries look at every tile's largest, the others at scales of 2 or more
    // (an f16 with bit 14 set)
    int off_now = off;
    bool look = PREC;
    if constexpr (!PREC) {
      unsigned bits = 0;
#pragma unroll
      for (int i = 0; i < 4 * NB; ++i) bits |= vs[i];
      look = __builtin_amdgcn_ballot_w64((bits & 0x40004000u) != 0) != 0;
    }
    if (look) {
      unsigned e = 0;  // the largest finite scale's exponent field, in bits 10..14
#pragma unroll
      for (int i = 0; i < 4 * NB; ++i) {
        const unsigned lo = vs[i] & 0x7C00u, hi = vs[i] >> 16 & 0x7C00u;
        e = max(e, max(lo == 0x7C00u ? 0u : lo, hi == 0x7C00u ? 0u : hi));
      }
      const int top = static_cast<int>(quarters_max(static_cast<float>(e >> 10)));
      off_now = __builtin_amdgcn_readfirstlane(min(off, 21 - max(top, 1)));
    }
    bool move = off_now < off;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) x[ct][t][r] *= factor[ct];
      if (a.cap > 0.f) {  // cap tanh(s / cap), tanh u = 1 - 2 / (e^2u + 1)
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            x[ct][t][r] = cap2 - 2.f * cap2 * __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(x[ct][t][r]) + 1.f);
      }
      if (a.slopes) {
        const float back = static_cast<float>(pos[ct] - key0);
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) x[ct][t][r] = fmaf(-slope[ct], fabsf(back - (16 * t + r)), x[ct][t][r]);
      }
      if constexpr (MASKED) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int j = key0 + 16 * t + r;
            if (j < span[ct].lo || j >= span[ct].hi) x[ct][t][r] = -__builtin_inff();
          }
      }
      const float top = fmaxf(fmaxf(fmaxf(x[ct][0][0], x[ct][0][1]), fmaxf(x[ct][0][2], x[ct][0][3])),
                              fmaxf(fmaxf(x[ct][1][0], x[ct][1][1]), fmaxf(x[ct][1][2], x[ct][1][3])));
      move |= top > lim[ct];
    }
    if (__builtin_amdgcn_ballot_w64(move) != 0) {
      const int before = off;
      off = off_now;
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        float top = M[ct] + before;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) top = fmaxf(top, x[ct][t][r]);
        top = quarters_max(top);
        const float now = top - off;
        // (nothing seen yet: M stays -inf, and there is nothing to rescale)
        const float by = M[ct] == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(M[ct] - now);
        l[ct] *= by;
#pragma unroll
        for (int i = 0; i < OT; ++i) acc[ct][i] *= by;
        M[ct] = now;
        lim[ct] = top + 8.f;
      }
    }
    unsigned keep[CT][4];  // masked tiles: a masked key's P' is 0 whatever its scale holds
    float p[CT][2][4];
    unsigned ph[CT][4];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      const float ref = M[ct] == -__builtin_inff() ? 0.f : M[ct];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          p[ct][t][r] = __builtin_amdgcn_exp2f(x[ct][t][r] - ref);
          l[ct] += p[ct][t][r];
        }
        ph[ct][2 * t] = pack_f16(p[ct][t][0], p[ct][t][2]);
        ph[ct][2 * t + 1] = pack_f16(p[ct][t][1], p[ct][t][3]);
        if constexpr (MASKED) {
          auto in = [&](int r) {
            const int j = key0 + 16 * t + r;
            return j >= span[ct].lo && j < span[ct].hi;
          };
          keep[ct][2 * t] = (in(0) ? 0xFFFFu : 0u) | (in(2) ? 0xFFFF0000u : 0u);
          keep[ct][2 * t + 1] = (in(1) ? 0xFFFFu : 0u) | (in(3) ? 0xFFFF0000u : 0u);
        }
      }
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      unsigned w[CT][PARTS][4];
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (PREC) {
            const f16x2 d = as_f16x2(vs[4 * b + i]);
            const float y0 = p[ct][i >> 1][i & 1] * static_cast<float>(d[0]);
            const float y1 = p[ct][i >> 1][2 + (i & 1)] * static_cast<float>(d[1]);
            w[ct][0][i] = pack_f16(y0, y1);
            const f16x2 hi = as_f16x2(w[ct][0][i]);
            w[ct][1][i] = pack_f16(y0 - static_cast<float>(hi[0]), y1 - static_cast<float>(hi[1]));
          } else {
            w[ct][0][i] = __builtin_bit_cast(unsigned, as_f16x2(ph[ct][i]) * as_f16x2(vs[4 * b + i]));
          }
          if constexpr (MASKED) {
#pragma unroll
            for (int part = 0; part < PARTS; ++part) w[ct][part][i] &= keep[ct][i];
          }
        }
      }
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
    }
  };

  for (int tile = tile0; tile < tile1; tile += STEP) {
    const int64_t unit = unit_of(tile);
    if (unit < 0) continue;
    KvTile<NB, KF, VF> kv;
    kv.load(a.c, unit, lane);
    if (tile * 32 >= full_lo && tile * 32 + 32 <= full_hi)
      step(kv, tile, std::false_type{});
    else
      step(kv, tile, std::true_type{});
  }

#pragma unroll
  for (int ct = 0; ct < CT; ++ct) l[ct] = quarters_sum(l[ct]);

  if constexpr (!WIDE) {
    // join the waves, a column tile at a time: the upper half hands its sums to the lower half, then wave 1 to wave 0
    __shared__ f32x4 so[W / 2][OT][64];
    __shared__ float2 sm[W / 2][16];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
#pragma unroll
      for (int half = W / 2; half >= 1; half >>= 1) {
        if (wave >= half && wave < 2 * half) {
          if (lane < 16) sm[wave - half][lane] = float2{M[ct], l[ct]};
#pragma unroll
          for (int i = 0; i < OT; ++i) so[wave - half][i][lane] = acc[ct][i];
        }
        __syncthreads();
        if (wave < half) {
          const float2 other = sm[wave][lane & 15];
          const float top = fmaxf(M[ct], other.x);
          const float f0 = M[ct] == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(M[ct] - top);
          const float f1 = other.x == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(other.x - top);
          l[ct] = l[ct] * f0 + other.y * f1;
          M[ct] = top;
#pragma unroll
          for (int i = 0; i < OT; ++i) acc[ct][i] = acc[ct][i] * f0 + so[wave][i][lane] * f1;
        }
        __syncthreads();
      }
    }
    if (wave != 0) return;
  }

#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    if (!live[ct]) continue;
    if (a.splits > 1) {
      const int64_t at = (split * a.rows + row[ct]) * a.heads + head[ct];
      if (lane < 16) a.part_m[at] = float2{M[ct], l[ct]};
      if (M[ct] == -__builtin_inff()) continue;
#pragma unroll
      for (int i = 0; i < OT; ++i)
        *reinterpret_cast<f32x4*>(a.part_o + at * D + i * 16 + quarter * 4) = acc[ct][i];
    } else {
      const float inv = l[ct] == 0.f ? 0.f : 1.f / l[ct];
      if (a.lse && lane < 16)
        a.lse[row[ct] * a.heads + head[ct]] = l[ct] == 0.f ? -__builtin_inff() : (M[ct] + __log2f(l[ct])) * (1.f / kLog2e);
      const int64_t at = row[ct] * a.out_stride_t + head[ct] * a.out_stride_h + quarter * 4;
#pragma unroll
      for (int i = 0; i < OT; ++i) {
        const f32x4 o = acc[ct][i] * inv;
        store_out(a.out, a.type, a.wide_out, at + i * 16, o);
      }
    }
  }
}

// `plan` says the kernel: column tiles a wave, and whether the waves have columns of their own
template <int NB, int KF, int VF>
hipError_t launch_attend_blocks(const AttendArgs& a, const AttendPlan& plan, int batch, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(a.splits) * static_cast<unsigned>(a.groups), static_cast<unsigned>(a.c.heads),
                  static_cast<unsigned>(batch));
  auto run = [&](auto kern) {
    const Timing tm = timing_slot(KIND_PROBE);
    if (tm.on) {
      hipExtLaunchKernelGGL(kern, grid, dim3(kAttendWaves * 64), 0, stream, tm.start, tm.stop, 0, a);
    } else {
      hipLaunchKernelGGL(kern, grid, dim3(kAttendWaves * 64), 0, stream, a);
    }
    return hipGetLastError();
  };
  if (a.type == KV_F32) {
    if (plan.wide) return run(kv_attend_kernel<NB, KF, VF, true, 2, true>);
    if (plan.ct == 1) return run(kv_attend_kernel<NB, KF, VF, true, 1, false>);
    return run(kv_attend_kernel<NB, KF, VF, true, 2, false>);
  }
  constexpr int MOST = NB <= 4 ? 4 : 2;
  if (plan.wide) return run(kv_attend_kernel<NB, KF, VF, false, MOST, true>);
  if (plan.ct == 1) return run(kv_attend_kernel<NB, KF, VF, false, 1, false>);
  if (plan.ct == 2 || MOST == 2) return run(kv_attend_kernel<NB, KF, VF, false, 2, false>);
  return run(kv_attend_kernel<NB, KF, VF, false, MOST, false>);
}

template <int KF, int VF>
hipError_t launch_attend_format(const AttendArgs& a, const AttendPlan& plan, int batch, hipStream_t stream) {
  switch (a.c.dim) {
    case 64: return launch_attend_blocks<2, KF, VF>(a, plan, batch, stream);
    case 96: return launch_attend_blocks<3, KF, VF>(a, plan, batch, stream);
    case 128: return launch_attend_blocks<4, KF, VF>(a, plan, batch, stream);
    default: return launch_attend_blocks<8, KF, VF>(a, plan, batch, stream);
  }
}

}  // namespace komp
