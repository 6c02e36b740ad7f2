// Writing tokens into the quantized key/value cache, and reading them back (layout: kv_layout.h).
//
// The quantizers are ggml's, with correctly rounded f32 steps: Q8_0 d = amax / 127, q = roundf(x * (1 / d)); Q4_0 d = max
// / -8 with max the signed value of largest magnitude (the first of equals), q = min(15, floor(x * (1 / d) + 8.5)); the
// stored scale is f16(d).  A block that holds a NaN gets a NaN scale, so it reads back as NaN.
//
// Bound by bytes: 65536 tokens of 8 heads of 128 channels, f32 and Q8_0, are written in 158-173 us and read in 114-146 (679 MB
// each way; a copy of as many bytes 141), 49999 tokens read from Q8_0 and Q4_0 as bf16 in 71 us (288 MB; 60).  One token
// each of 64 sequences: 2.8 and 2.7 us, a launch's own time.
#include <hip/hip_ext.h>

#include <type_traits>
#include <utility>

#include "komp_device.h"
#include "komp_internal.h"
#include "kv_layout.h"

namespace komp {
namespace {

constexpr int kThreads = 256, kGroups = kThreads / 8;

struct WriteArgs {
  KvCache c;
  const void* x[2];  // keys, values
  int64_t stride_t[2];
  int64_t stride_h[2];
  const int64_t* slots;
  int64_t tokens;
  bool wide[2];   // four elements of a row may be loaded at once
};

struct ReadArgs {
  KvCache c;
  void* x[2];
  const int64_t* slots;
  int64_t tokens;
};

template <int TYPE>
__device__ __forceinline__ float to_f32(const void* p, int64_t i) {
  if constexpr (TYPE == KV_F32) return static_cast<const float*>(p)[i];
  const uint16_t u = static_cast<const uint16_t*>(p)[i];
  if constexpr (TYPE == KV_F16) return static_cast<float>(__builtin_bit_cast(_Float16, u));
  return __uint_as_float(static_cast<unsigned>(u) << 16);
}

// four elements of a row, which is `wide` when it may be read 4 elements at a time
template <int TYPE>
__device__ __forceinline__ f32x4 load4(const void* p, int64_t i, bool wide) {
  if (wide) {
    if constexpr (TYPE == KV_F32) return *reinterpret_cast<const f32x4*>(static_cast<const float*>(p) + i);
    typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));
    const u16x4 u = *reinterpret_cast<const u16x4*>(static_cast<const uint16_t*>(p) + i);
    f32x4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint16_t w = u[e];
      v[e] = TYPE == KV_F16 ? static_cast<float>(__builtin_bit_cast(_Float16, w))
                            : __uint_as_float(static_cast<unsigned>(w) << 16);
    }
    return v;
  }
  return f32x4{to_f32<TYPE>(p, i), to_f32<TYPE>(p, i + 1), to_f32<TYPE>(p, i + 2), to_f32<TYPE>(p, i + 3)};
}

__device__ __forceinline__ uint16_t f16_bits(float v) { return __builtin_bit_cast(uint16_t, static_cast<_Float16>(v)); }

// Blocks of 32, each held by 8 aligned lanes of 4 values, N of them: the lane's four codes of each as unsigned bytes (Q4_0:
// 0..15, Q8_0: value + 128).  The divisions of N blocks are shared out: lane n of each four does block n's, and holds its
// scale's bits afterwards (N = 1: every lane).
template <int FMT, int N>
__device__ __forceinline__ void quantize8(const f32x4 (&v)[N], int lane8, unsigned (&packed)[N], uint16_t& scale) {
#pragma clang fp contract(off)
  static_assert(N == 1 || N == 4, "blocks of a quad of lanes");
  float d[N];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    // |x|'s bits order like the floats, and a NaN's are above infinity's
    int a[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) a[e] = __float_as_int(v[n][e]) & 0x7FFFFFFF;
    int top = max(max(a[0], a[1]), max(a[2], a[3]));
    top = max(top, dpp_i<KOMP_DPP_XOR1>(top));
    top = max(top, dpp_i<KOMP_DPP_XOR2>(top));
    top = max(top, dpp_i<KOMP_DPP_HALF_MIRROR>(top));
    if constexpr (FMT == KV_Q8_0) {
      d[n] = __int_as_float(top);
    } else {
      int first = 64;  // 2 * index + sign of the first value of that magnitude
#pragma unroll
      for (int e = 3; e >= 0; --e) first = a[e] == top ? 2 * (4 * lane8 + e) + (__float_as_uint(v[n][e]) >> 31) : first;
      first = min(first, dpp_i<KOMP_DPP_XOR1>(first));
      first = min(first, dpp_i<KOMP_DPP_XOR2>(first));
      first = min(first, dpp_i<KOMP_DPP_HALF_MIRROR>(first));
      d[n] = __int_as_float(top) * ((first & 1) ? 0.125f : -0.125f);
    }
  }
  float own = d[0];
  if constexpr (N == 4) {
    const int q = lane8 & 3;
    own = q == 0 ? d[0] : q == 1 ? d[1] : q == 2 ? d[2] : d[3];
  }
  if constexpr (FMT == KV_Q8_0) own = own / 127.0f;
  scale = f16_bits(own);
  float id = own != 0.0f ? 1.0f / own : 0.0f;
  if constexpr (FMT == KV_Q8_0) id = id + id;
  each<N>([&](auto nc) __attribute__((always_inline)) {
    constexpr int n = nc.value;
    // quad_perm [n, n, n, n]: lane n of each four
    const float f = N == 1 ? id : __int_as_float(dpp_i<N == 1 ? 0 : n * 0x55>(__float_as_int(id)));
    unsigned q[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (FMT == KV_Q8_0) {
        // t = trunc(2 y), y = x * id (2 id is exact): roundf(y) is (t + 1) >> 1 for t >= 0, t >> 1 below; and 128 more
        const int t = static_cast<int>(v[n][e] * f);
        q[e] = static_cast<unsigned>(t + (t >> 31) + 257) >> 1 & 255;
      } else {
        q[e] = min(15u, static_cast<unsigned>(v[n][e] * f + 8.5f));
      }
    }
    packed[n] = q[0] | q[1] << 8 | q[2] << 16 | q[3] << 24;
  });
}

// where a tile of 32 tokens of a page and head lies, in units of such tiles
__device__ __forceinline__ int64_t unit_of(const KvCache& c, int64_t tile, int h) {
  const int log2 = c.page_log2 - 5;
  return (((tile >> log2) * c.heads + h) << log2) + (tile & ((int64_t{1} << log2) - 1));
}

constexpr int kNext4 = 0x104;  // row_shl:4, lane + 4 of a row

// A block's codes, four of eight lanes each, into the 32-token tile at `codes` and `scales` (global or shared memory).
// Only this token's bytes are written.
template <int FMT, int NB, bool VALUE>
__device__ __forceinline__ void put(uint8_t* codes, uint16_t* scales, int token32, int b, int lane8, unsigned q, uint16_t scale) {
  const int token16 = token32 & 15;
  if constexpr (!VALUE) {
    uint8_t* tile = codes + (token32 >> 4) * (16 * NB * kv_code_bytes(FMT));
    const int dword = kv_k_dword(NB, FMT, token16, b, lane8 >> 1, lane8 & 1);
    if constexpr (FMT == KV_Q8_0) {
      reinterpret_cast<unsigned*>(tile)[dword] = q;
    } else {
      const unsigned n = (q & 15) | (q >> 4 & 0xF0) | (q >> 8 & 0xF00) | (q >> 12 & 0xF000);
      reinterpret_cast<uint16_t*>(tile)[dword * 2 + (lane8 & 1)] = static_cast<uint16_t>(n);
    }
    if (lane8 == 0) scales[(token32 >> 4) * (16 * NB) + kv_k_scale(NB, token16, b)] = scale;
  } else {
    if constexpr (FMT == KV_Q4_0) q |= static_cast<unsigned>(dpp_i<kNext4>(static_cast<int>(q))) << 4;  // lanes 0..3: channels + 16
    if (FMT == KV_Q8_0 || lane8 < 4) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        codes[kv_v_byte(NB, FMT, token32, b, (lane8 & 3) * 4 + e, lane8 >> 2)] = static_cast<uint8_t>(q >> (8 * e));
    }
    if (lane8 == 0) scales[kv_v_scale(NB, token32, b)] = scale;
  }
}

// the four values of a lane of eight
template <int FMT, int NB, bool VALUE>
__device__ __forceinline__ f32x4 get(const uint8_t* codes, const uint16_t* scales, int token32, int b, int lane8) {
  const int token16 = token32 & 15;
  uint16_t scale;
  int q[4];
  if constexpr (!VALUE) {
    const uint8_t* tile = codes + (token32 >> 4) * (16 * NB * kv_code_bytes(FMT));
    const int dword = kv_k_dword(NB, FMT, token16, b, lane8 >> 1, lane8 & 1);
    scale = scales[(token32 >> 4) * (16 * NB) + kv_k_scale(NB, token16, b)];
    if constexpr (FMT == KV_Q8_0) {
      const unsigned w = reinterpret_cast<const unsigned*>(tile)[dword];
#pragma unroll
      for (int e = 0; e < 4; ++e) q[e] = static_cast<int>(w >> (8 * e) & 255) - 128;
    } else {
      const unsigned w = reinterpret_cast<const uint16_t*>(tile)[dword * 2 + (lane8 & 1)];
#pragma unroll
      for (int e = 0; e < 4; ++e) q[e] = static_cast<int>(w >> (4 * e) & 15) - 8;
    }
  } else {
    scale = scales[kv_v_scale(NB, token32, b)];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int w = codes[kv_v_byte(NB, FMT, token32, b, (lane8 & 3) * 4 + e, lane8 >> 2)];
      q[e] = FMT == KV_Q8_0 ? w - 128 : (lane8 < 4 ? w & 15 : w >> 4) - 8;
    }
  }
  const float d = f16_bits_to_f32(static_cast<int16_t>(scale));
  return f32x4{q[0] * d, q[1] * d, q[2] * d, q[3] * d};
}

// keys or values of a cache
struct Plane {
  uint8_t* codes;
  uint16_t* scales;
};
template <bool VALUE>
__device__ __forceinline__ Plane plane_of(const KvCache& c) {
  return VALUE ? Plane{c.vq, c.vs} : Plane{c.kq, c.ks};
}
template <int FMT, int NB>
__device__ __forceinline__ Plane at_unit(const Plane& p, int64_t unit) {
  return Plane{p.codes + unit * (32 * NB * kv_code_bytes(FMT)), p.scales + unit * (32 * NB)};
}

// Few tokens: eight lanes a block, a workgroup's blocks those of `tokens` tokens of one head.
template <int FMT, int NB, int TYPE, bool VALUE>
__device__ __forceinline__ void write_few(const WriteArgs& a) {
  const int lane8 = threadIdx.x & 7, group = threadIdx.x >> 3, h = blockIdx.x % a.c.heads;
  const int64_t t = static_cast<int64_t>(blockIdx.x / a.c.heads) * (kGroups / NB) + group / NB;
  const int b = group % NB;
  if (group >= kGroups / NB * NB || t >= a.tokens) return;  // in groups of 8 lanes
  const int64_t slot = a.slots[t];
  if (slot < 0 || slot >= a.c.pages << a.c.page_log2) return;
  const f32x4 v[1] = {load4<TYPE>(a.x[VALUE], t * a.stride_t[VALUE] + h * a.stride_h[VALUE] + b * 32 + lane8 * 4, a.wide[VALUE])};
  uint16_t scale;
  unsigned q[1];
  quantize8<FMT>(v, lane8, q, scale);
  const Plane p = at_unit<FMT, NB>(plane_of<VALUE>(a.c), unit_of(a.c, slot >> 5, h));
  put<FMT, NB, VALUE>(p.codes, p.scales, static_cast<int>(slot & 31), b, lane8, q[0], scale);
}

// Four tokens' codes of a block, four channels a lane, as four channels' codes, four tokens each, and back.
__device__ __forceinline__ void transpose4(unsigned (&q)[4]) {
  const unsigned a = __builtin_amdgcn_perm(q[1], q[0], 0x05010400u), b = __builtin_amdgcn_perm(q[1], q[0], 0x07030602u);
  const unsigned c = __builtin_amdgcn_perm(q[3], q[2], 0x05010400u), d = __builtin_amdgcn_perm(q[3], q[2], 0x07030602u);
  q[0] = __builtin_amdgcn_perm(c, a, 0x05040100u);
  q[1] = __builtin_amdgcn_perm(c, a, 0x07060302u);
  q[2] = __builtin_amdgcn_perm(d, b, 0x05040100u);
  q[3] = __builtin_amdgcn_perm(d, b, 0x07060302u);
}

// Many tokens: a workgroup has 32 tokens of the list and one head.  Consecutive slots fall into two tiles of 32 at most (one
// where the list begins at a tile's start, which the first tokens are left out of the first workgroup for); a group of
// eight lanes takes a block of four neighbouring places of a tile at a time, and the workgroup puts the tiles together in
// shared memory and moves them by dwords, four tokens of value codes in one.  Tokens of further tiles go one by one.
template <int FMT, int NB>
struct Tiles {
  static constexpr int CODES = 32 * NB * kv_code_bytes(FMT), SCALES = 32 * NB;
  uint8_t codes[2][CODES];
  uint16_t scales[2][SCALES];
  int64_t slot[32];  // of the tokens of further tiles; -1 for the others
  int token[2][32];  // which of the 32 a place of a tile belongs to; -1: none
  int quads[16];     // the fours of places that have a token, 8 * tile + four
  unsigned mask[2];  // the places that have one
  int further;       // whether there are tokens of further tiles
};
// What lies where; the two tiles are the first and the last valid slot's (-1 for none).  Returns the list's index of the
// first token, and in `count` how many fours of places there are.
template <int FMT, int NB>
__device__ __forceinline__ int64_t find_tiles(const KvCache& c, const int64_t* slots, int64_t tokens, Tiles<FMT, NB>& sh, int64_t (&tile)[2], int& count) {
  const int lane = threadIdx.x & 63;
  const int64_t first = static_cast<int64_t>(blockIdx.x / c.heads) * 32 - (slots[0] & 31), t = first + (lane & 31);
  int64_t slot = t >= 0 && t < tokens ? slots[t] : -1;
  if (slot < 0 || slot >= c.pages << c.page_log2) slot = -1;
  const unsigned there = static_cast<unsigned>(__builtin_amdgcn_ballot_w64(slot >= 0 && lane < 32));
  tile[0] = tile[1] = -1;
  const int64_t own = slot >> 5;
  if (there) {
    tile[0] = __shfl(own, __builtin_ctz(there), 64);
    tile[1] = __shfl(own, 31 - __builtin_clz(there), 64);
    if (tile[1] == tile[0]) tile[1] = -1;
  }
  if (threadIdx.x < 64) (&sh.token[0][0])[threadIdx.x] = -1;
  if (threadIdx.x < 2) sh.mask[threadIdx.x] = 0;
  const int to = slot < 0 || lane >= 32 ? -1 : own == tile[0] ? 0 : own == tile[1] ? 1 : -2;
  const bool further = __builtin_amdgcn_ballot_w64(to == -2) != 0;
  __syncthreads();
  if (threadIdx.x < 32) {
    sh.slot[threadIdx.x] = to == -2 ? slot : -1;
    if (to >= 0) {
      sh.token[to][slot & 31] = threadIdx.x;
      atomicOr(&sh.mask[to], 1u << (slot & 31));
    }
  }
  if (threadIdx.x == 0) sh.further = further;
  __syncthreads();
  unsigned fours = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) fours |= (sh.mask[i >> 3] >> ((i & 7) * 4) & 15) ? 1u << i : 0u;
  count = __builtin_popcount(fours);
  if (threadIdx.x < 16 && (fours >> threadIdx.x & 1)) sh.quads[__builtin_popcount(fours & ((1u << threadIdx.x) - 1))] = threadIdx.x;
  __syncthreads();
  return first;
}

template <int FMT, int NB, int TYPE, bool VALUE>
__device__ __forceinline__ void write_many(const WriteArgs& a, Tiles<FMT, NB>& sh) {
  const int lane8 = threadIdx.x & 7, group = threadIdx.x >> 3, h = blockIdx.x % a.c.heads;
  int64_t tile[2];
  int count;
  const int64_t first = find_tiles(a.c, a.slots, a.tokens, sh, tile, count);
  const Plane plane = plane_of<VALUE>(a.c);
  auto row = [&](int token, int b) {
    return load4<TYPE>(a.x[VALUE], (first + token) * a.stride_t[VALUE] + h * a.stride_h[VALUE] + b * 32 + lane8 * 4, a.wide[VALUE]);
  };
  for (int task = group; task < count * NB; task += kGroups) {
    const int quad = sh.quads[task / NB], b = task % NB, to = quad >> 3, at = (quad & 7) * 4;
    f32x4 v[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const int token = sh.token[to][at + n];
      v[n] = f32x4{0.f, 0.f, 0.f, 0.f};  // (a place without a token: what becomes of it is not stored)
      if (token >= 0) v[n] = row(token, b);
    }
    unsigned q[4];
    uint16_t scale;
    quantize8<FMT>(v, lane8, q, scale);
    if constexpr (VALUE) {
      if constexpr (FMT == KV_Q4_0) {
#pragma unroll
        for (int n = 0; n < 4; ++n) q[n] |= static_cast<unsigned>(dpp_i<kNext4>(static_cast<int>(q[n]))) << 4;
      }
      if (FMT == KV_Q8_0 || lane8 < 4) {
        transpose4(q);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          *reinterpret_cast<unsigned*>(&sh.codes[to][kv_v_byte(NB, FMT, at, b, (lane8 & 3) * 4 + e, lane8 >> 2)]) = q[e];
      }
      if (lane8 < 4) sh.scales[to][kv_v_scale(NB, at + lane8, b)] = scale;
    } else {
      each<4>([&](auto nc) __attribute__((always_inline)) {
        constexpr int n = nc.value;
        put<FMT, NB, VALUE>(sh.codes[to], sh.scales[to], at + n, b, lane8, q[n], static_cast<uint16_t>(dpp_i<n * 0x55>(scale)));
      });
    }
  }
  if (sh.further) {
    for (int task = group; task < 32 * NB; task += kGroups) {
      const int64_t slot = sh.slot[task / NB];
      const int b = task % NB;
      if (slot < 0) continue;
      const f32x4 v[1] = {row(task / NB, b)};
      unsigned q[1];
      uint16_t scale;
      quantize8<FMT>(v, lane8, q, scale);
      const Plane p = at_unit<FMT, NB>(plane, unit_of(a.c, slot >> 5, h));
      put<FMT, NB, VALUE>(p.codes, p.scales, static_cast<int>(slot & 31), b, lane8, q[0], scale);
    }
  }
  __syncthreads();
#pragma unroll
  for (int to = 0; to < 2; ++to) {
    if (tile[to] < 0) continue;
    const unsigned mask = sh.mask[to];
    const Plane p = at_unit<FMT, NB>(plane, unit_of(a.c, tile[to], h));
    if (mask == 0xFFFFFFFFu) {  // the whole tile
      for (int w = threadIdx.x; w < Tiles<FMT, NB>::CODES / 16; w += kThreads)
        reinterpret_cast<u32x4*>(p.codes)[w] = reinterpret_cast<const u32x4*>(sh.codes[to])[w];
      for (int w = threadIdx.x; w < Tiles<FMT, NB>::SCALES / 8; w += kThreads)
        reinterpret_cast<u32x4*>(p.scales)[w] = reinterpret_cast<const u32x4*>(sh.scales[to])[w];
      continue;
    }
    const unsigned* codes = reinterpret_cast<const unsigned*>(sh.codes[to]);
    for (int w = threadIdx.x; w < Tiles<FMT, NB>::CODES / 4; w += kThreads) {
      if constexpr (!VALUE) {
        constexpr int lane_words = kv_kb(NB, FMT) * (FMT == KV_Q8_0 ? 2 : 1), half = 4 * NB * kv_code_bytes(FMT);
        if (mask >> (w / half * 16 + w / lane_words % 16) & 1) reinterpret_cast<unsigned*>(p.codes)[w] = codes[w];
      } else {
        constexpr int lane_words = kv_vb(NB, FMT) * (FMT == KV_Q8_0 ? 4 : 2);
        const unsigned own = mask >> ((w & 1) * 16 + (w / lane_words >> 4 & 3) * 4) & 15;
        if (own == 15) {
          reinterpret_cast<unsigned*>(p.codes)[w] = codes[w];
        } else {
          for (int e = 0; e < 4; ++e)
            if (own >> e & 1) p.codes[w * 4 + e] = sh.codes[to][w * 4 + e];
        }
      }
    }
    for (int i = threadIdx.x; i < Tiles<FMT, NB>::SCALES; i += kThreads) {
      // the token of scale i: kv_k_scale, kv_v_scale
      const int k = i & 3, value = (i >> 2 & 1) * 16 + i / (8 * NB) * 4 + (k & 1) * 2 + (k >> 1);
      if (mask >> (VALUE ? value : i / NB) & 1) p.scales[i] = sh.scales[to][i];
    }
  }
}

template <int KF, int VF, int NB, int TYPE, bool MANY>
__global__ void __launch_bounds__(kThreads) kv_write_kernel(const WriteArgs a) {
  if constexpr (MANY) {
    constexpr size_t bytes = sizeof(Tiles<KF, NB>) > sizeof(Tiles<VF, NB>) ? sizeof(Tiles<KF, NB>) : sizeof(Tiles<VF, NB>);
    __shared__ __attribute__((aligned(16))) unsigned char shared[bytes];
    if (blockIdx.y == 0) write_many<KF, NB, TYPE, false>(a, *reinterpret_cast<Tiles<KF, NB>*>(shared));
    else write_many<VF, NB, TYPE, true>(a, *reinterpret_cast<Tiles<VF, NB>*>(shared));
  } else {
    if (blockIdx.y == 0) write_few<KF, NB, TYPE, false>(a);
    else write_few<VF, NB, TYPE, true>(a);
  }
}

template <int TYPE>
__device__ __forceinline__ void store4(void* p, int64_t i, f32x4 v) {
  if constexpr (TYPE == KV_F32) {
    *reinterpret_cast<f32x4*>(static_cast<float*>(p) + i) = v;
  } else {
    typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));
    u16x4 u;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      u[e] = TYPE == KV_F16 ? f16_bits(v[e]) : __builtin_bit_cast(uint16_t, static_cast<__bf16>(v[e]));
    *reinterpret_cast<u16x4*>(static_cast<uint16_t*>(p) + i) = u;
  }
}

template <int FMT, int NB, int TYPE, bool VALUE>
__device__ __forceinline__ void read_few(const ReadArgs& a) {
  const int lane8 = threadIdx.x & 7, group = threadIdx.x >> 3, h = blockIdx.x % a.c.heads;
  const int64_t t = static_cast<int64_t>(blockIdx.x / a.c.heads) * (kGroups / NB) + group / NB;
  const int b = group % NB;
  if (group >= kGroups / NB * NB || t >= a.tokens) return;
  const int64_t slot = a.slots[t];
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  if (slot >= 0 && slot < a.c.pages << a.c.page_log2) {
    const Plane p = at_unit<FMT, NB>(plane_of<VALUE>(a.c), unit_of(a.c, slot >> 5, h));
    v = get<FMT, NB, VALUE>(p.codes, p.scales, static_cast<int>(slot & 31), b, lane8);
  }
  store4<TYPE>(a.x[VALUE], ((t * a.c.heads + h) * NB + b) * 32 + lane8 * 4, v);
}

// (a tile is loaded whole, 16 bytes a lane, whatever part of it is read)
template <int FMT, int NB, int TYPE, bool VALUE>
__device__ __forceinline__ void read_many(const ReadArgs& a, Tiles<FMT, NB>& sh) {
  const int lane8 = threadIdx.x & 7, group = threadIdx.x >> 3, h = blockIdx.x % a.c.heads;
  int64_t tile[2];
  int count;
  const int64_t first = find_tiles(a.c, a.slots, a.tokens, sh, tile, count);
  const Plane plane = plane_of<VALUE>(a.c);
#pragma unroll
  for (int to = 0; to < 2; ++to) {
    if (tile[to] < 0) continue;
    const Plane p = at_unit<FMT, NB>(plane, unit_of(a.c, tile[to], h));
    for (int w = threadIdx.x; w < Tiles<FMT, NB>::CODES / 16; w += kThreads)
      reinterpret_cast<u32x4*>(sh.codes[to])[w] = reinterpret_cast<const u32x4*>(p.codes)[w];
    for (int w = threadIdx.x; w < Tiles<FMT, NB>::SCALES / 8; w += kThreads)
      reinterpret_cast<u32x4*>(sh.scales[to])[w] = reinterpret_cast<const u32x4*>(p.scales)[w];
  }
  __syncthreads();
  auto store = [&](int token, int b, f32x4 v) {
    store4<TYPE>(a.x[VALUE], (((first + token) * a.c.heads + h) * NB + b) * 32 + lane8 * 4, v);
  };
  for (int task = group; task < count * NB; task += kGroups) {
    const int quad = sh.quads[task / NB], b = task % NB, to = quad >> 3, at = (quad & 7) * 4;
    f32x4 v[4];
    if constexpr (VALUE) {
      unsigned q[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        q[e] = *reinterpret_cast<const unsigned*>(&sh.codes[to][kv_v_byte(NB, FMT, at, b, (lane8 & 3) * 4 + e, lane8 >> 2)]);
        if constexpr (FMT == KV_Q4_0) q[e] = (lane8 < 4 ? q[e] : q[e] >> 4) & 0x0F0F0F0Fu;
      }
      transpose4(q);
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const float d = f16_bits_to_f32(static_cast<int16_t>(sh.scales[to][kv_v_scale(NB, at + n, b)]));
#pragma unroll
        for (int e = 0; e < 4; ++e) v[n][e] = (static_cast<float>(q[n] >> (8 * e) & 255u) - (FMT == KV_Q8_0 ? 128.f : 8.f)) * d;
      }
    } else {
#pragma unroll
      for (int n = 0; n < 4; ++n) v[n] = get<FMT, NB, VALUE>(sh.codes[to], sh.scales[to], at + n, b, lane8);
    }
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const int token = sh.token[to][at + n];
      if (token >= 0) store(token, b, v[n]);
    }
  }
  // tokens of further tiles, and those without a slot (or a second time the same one): one by one
  const int left = static_cast<int>(min(int64_t{32}, a.tokens - first));
  if (__builtin_popcount(sh.mask[0]) + __builtin_popcount(sh.mask[1]) < left - static_cast<int>(max(int64_t{0}, -first))) {
    for (int task = group; task < 32 * NB; task += kGroups) {
      const int token = task / NB, b = task % NB;
      const int64_t t = first + token;
      if (t < 0 || t >= a.tokens) continue;
      const int64_t slot = a.slots[t], own = slot >> 5;
      f32x4 v = {0.f, 0.f, 0.f, 0.f};
      if (slot >= 0 && slot < a.c.pages << a.c.page_log2) {
        const int to = own == tile[0] ? 0 : own == tile[1] ? 1 : -1;
        if (to >= 0 && sh.token[to][slot & 31] == token) continue;
        const Plane p = at_unit<FMT, NB>(plane, unit_of(a.c, own, h));
        v = get<FMT, NB, VALUE>(p.codes, p.scales, static_cast<int>(slot & 31), b, lane8);
      }
      store(token, b, v);
    }
  }
}

template <int KF, int VF, int NB, int TYPE, bool MANY>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(const ReadArgs a) {
  if constexpr (MANY) {
    constexpr size_t bytes = sizeof(Tiles<KF, NB>) > sizeof(Tiles<VF, NB>) ? sizeof(Tiles<KF, NB>) : sizeof(Tiles<VF, NB>);
    __shared__ __attribute__((aligned(16))) unsigned char shared[bytes];
    if (blockIdx.y == 0) read_many<KF, NB, TYPE, false>(a, *reinterpret_cast<Tiles<KF, NB>*>(shared));
    else read_many<VF, NB, TYPE, true>(a, *reinterpret_cast<Tiles<VF, NB>*>(shared));
  } else {
    if (blockIdx.y == 0) read_few<KF, NB, TYPE, false>(a);
    else read_few<VF, NB, TYPE, true>(a);
  }
}

// Workgroups of one call: `per` tokens of one head each, keys and values apart.  The heads of the same tokens follow one
// another, so that a token's rows are read and written together.
dim3 grid_of(int64_t tokens, int per, int heads) {
  return dim3(static_cast<unsigned>((tokens + per - 1) / per * heads), 2);
}

// The kernels of 32-token tiles, from the size on where they fill the CUs (and their lists begin 0 to 31 tokens early).  Few and
// tiles, us, 8 heads of 128 channels, of 8192, 16384 and 32768 tokens times heads: write bf16 into Q8_0 keys and Q4_0 values
// 4.3 and 5.7, 6.1 and 6.9, 10.2 and 10.1; f32 into Q8_0 4.9 and 5.6, 7.9 and 7.0, 14.5 and 10.8; read bf16 from the first 3.7 and
// 4.4, 5.5 and 5.6, 8.9 and 8.5; f32 from the second 4.6 and 4.8, 7.1 and 6.8, 11.7 and 10.3.
bool many_tokens(int64_t tokens, int heads) { return tokens * heads >= 32 * 512; }

template <typename F, typename A>
hipError_t launch(F kern, const dim3& grid, hipStream_t stream, const A& a) {
  const Timing tm = timing_slot(KIND_PROBE);
  if (tm.on) {
    hipExtLaunchKernelGGL(kern, grid, dim3(kThreads), 0, stream, tm.start, tm.stop, 0, a);
  } else {
    hipLaunchKernelGGL(kern, grid, dim3(kThreads), 0, stream, a);
  }
  return hipGetLastError();
}

// run f with the cache's formats, blocks a head and element type as constants
template <int KF, int VF, int NB, typename F>
hipError_t with_type(int type, F&& f) {
  if (type == KV_F32) return f(std::integral_constant<int, KF>{}, std::integral_constant<int, VF>{}, std::integral_constant<int, NB>{}, std::integral_constant<int, KV_F32>{});
  if (type == KV_F16) return f(std::integral_constant<int, KF>{}, std::integral_constant<int, VF>{}, std::integral_constant<int, NB>{}, std::integral_constant<int, KV_F16>{});
  return f(std::integral_constant<int, KF>{}, std::integral_constant<int, VF>{}, std::integral_constant<int, NB>{}, std::integral_constant<int, KV_BF16>{});
}
template <int KF, int VF, typename F>
hipError_t with_blocks(int nb, int type, F&& f) {
  switch (nb) {
    case 2: return with_type<KF, VF, 2>(type, f);
    case 3: return with_type<KF, VF, 3>(type, f);
    case 4: return with_type<KF, VF, 4>(type, f);
    default: return with_type<KF, VF, 8>(type, f);
  }
}
template <typename F>
hipError_t with_constants(const KvCache& c, int type, F&& f) {
  const int nb = c.dim / 32;
  if (c.kf == KV_Q4_0) return with_blocks<KV_Q4_0, KV_Q4_0>(nb, type, f);
  if (c.vf == KV_Q4_0) return with_blocks<KV_Q8_0, KV_Q4_0>(nb, type, f);
  return with_blocks<KV_Q8_0, KV_Q8_0>(nb, type, f);
}

}  // namespace

hipError_t launch_kv_write(const KvWriteCall& w, hipStream_t stream) {
  WriteArgs a;
  a.c = w.cache;
  a.slots = w.slots;
  a.tokens = w.tokens;
  const int size = w.type == KV_F32 ? 4 : 2;
  for (int i = 0; i < 2; ++i) {
    a.x[i] = i ? w.v : w.k;
    a.stride_t[i] = w.stride_t[i];
    a.stride_h[i] = w.stride_h[i];
    a.wide[i] = reinterpret_cast<uintptr_t>(a.x[i]) % (4 * size) == 0 && w.stride_t[i] % 4 == 0 && w.stride_h[i] % 4 == 0;
  }
  return with_constants(w.cache, w.type, [&](auto kf, auto vf, auto nb, auto type) {
    constexpr int KF = kf.value, VF = vf.value, NB = nb.value, TYPE = type.value;
    if (many_tokens(a.tokens, a.c.heads))
      return launch(kv_write_kernel<KF, VF, NB, TYPE, true>, grid_of(a.tokens + 31, 32, a.c.heads), stream, a);
    return launch(kv_write_kernel<KF, VF, NB, TYPE, false>, grid_of(a.tokens, kGroups / NB, a.c.heads), stream, a);
  });
}

hipError_t launch_kv_read(const KvReadCall& r, hipStream_t stream) {
  ReadArgs a;
  a.c = r.cache;
  a.slots = r.slots;
  a.tokens = r.tokens;
  a.x[0] = r.k;
  a.x[1] = r.v;
  return with_constants(r.cache, r.type, [&](auto kf, auto vf, auto nb, auto type) {
    constexpr int KF = kf.value, VF = vf.value, NB = nb.value, TYPE = type.value;
    if (many_tokens(a.tokens, a.c.heads))
      return launch(kv_read_kernel<KF, VF, NB, TYPE, true>, grid_of(a.tokens + 31, 32, a.c.heads), stream, a);
    return launch(kv_read_kernel<KF, VF, NB, TYPE, false>, grid_of(a.tokens, kGroups / NB, a.c.heads), stream, a);
  });
}

}  // namespace komp
