// Writing tokens into the quantized key/value cache, and reading them back (layout: kv_layout.h).
//
// The quantizers are ggml's, with correctly rounded f32 steps: Q8_0 d = amax / 127, q = roundf(x * (1 / d)); Q4_0 d = max
// / -8 with max the signed value of largest magnitude (the first of equals), q = min(15, floor(x * (1 / d) + 8.5)); the
// stored scale is f16(d).  A block that holds a NaN gets a NaN scale, so it reads back as NaN.
#include <hip/hip_ext.h>

#include <type_traits>

#include "komp_device.h"
#include "komp_internal.h"
#include "kv_layout.h"

namespace komp {
namespace {

constexpr int kThreads = 256;

struct WriteArgs {
  KvCache c;
  const void* x[2];  // keys, values
  int64_t stride_t[2];
  int64_t stride_h[2];
  const int64_t* slots;
  int64_t lanes;  // tokens * heads * blocks * 8
  bool wide[2];   // four elements of a row may be loaded at once
};

struct ReadArgs {
  KvCache c;
  void* x[2];
  const int64_t* slots;
  int64_t lanes;
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

// One block of 32 held by 8 aligned lanes of 4 values: the lane's four codes as unsigned bytes (Q4_0: 0..15, Q8_0:
// value + 128), and the block's scale bits in every lane.
template <int FMT>
__device__ __forceinline__ unsigned quantize8(f32x4 v, int lane8, uint16_t& scale) {
#pragma clang fp contract(off)
  // |x|'s bits order like the floats, and a NaN's are above infinity's
  int a[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) a[e] = __float_as_int(v[e]) & 0x7FFFFFFF;
  int top = max(max(a[0], a[1]), max(a[2], a[3]));
  top = max(top, dpp_i<KOMP_DPP_XOR1>(top));
  top = max(top, dpp_i<KOMP_DPP_XOR2>(top));
  top = max(top, dpp_i<KOMP_DPP_HALF_MIRROR>(top));
  float d;
  if constexpr (FMT == KV_Q8_0) {
    d = __int_as_float(top) / 127.0f;
  } else {
    int first = 64;  // 2 * index + sign of the first value of that magnitude
#pragma unroll
    for (int e = 3; e >= 0; --e) first = a[e] == top ? 2 * (4 * lane8 + e) + (__float_as_uint(v[e]) >> 31) : first;
    first = min(first, dpp_i<KOMP_DPP_XOR1>(first));
    first = min(first, dpp_i<KOMP_DPP_XOR2>(first));
    first = min(first, dpp_i<KOMP_DPP_HALF_MIRROR>(first));
    d = __int_as_float(top) * ((first & 1) ? 0.125f : -0.125f);
  }
  const float id = d != 0.0f ? 1.0f / d : 0.0f;
  scale = f16_bits(d);
  unsigned packed = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float y = v[e] * id;
    int q;
    if constexpr (FMT == KV_Q8_0) {
      q = max(0, min(255, static_cast<int>(round_half_away(y)) + 128));
    } else {
      q = max(0, min(15, static_cast<int>(floorf(y + 8.5f))));
    }
    packed |= static_cast<unsigned>(q) << (8 * e);
  }
  return packed;
}

// where the page and head of a slot begin, in units of 32 tokens * blocks (times bytes of each plane)
__device__ __forceinline__ int64_t unit_of(const KvCache& c, int64_t slot, int h) {
  const int64_t page = slot >> c.page_log2;
  const int tile = static_cast<int>(slot & (c.page - 1)) >> 5;
  return (page * c.heads + h) * (c.page >> 5) + tile;
}

// Eight lanes a block; a token's slot decides where its codes go.  Only this token's bytes are written, so tokens of
// any slots may be written together.
template <int KF, int VF, int NB, int TYPE>
__global__ void __launch_bounds__(kThreads) kv_write_kernel(const WriteArgs a) {
  const int64_t gid = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (gid >= a.lanes) return;  // in groups of 8 lanes
  const int lane8 = static_cast<int>(gid & 7);
  const int64_t blk = gid >> 3;
  const int b = static_cast<int>(blk % NB);
  const int64_t th = blk / NB;
  const int64_t t = th / a.c.heads;
  const int h = static_cast<int>(th - t * a.c.heads);
  const int64_t slot = a.slots[t];
  if (slot < 0 || slot >= a.c.pages << a.c.page_log2) return;
  const int64_t unit = unit_of(a.c, slot, h);
  const int token32 = static_cast<int>(slot & 31), token16 = token32 & 15;
  uint16_t scale;
  if (blockIdx.y == 0) {
    const f32x4 v = load4<TYPE>(a.x[0], t * a.stride_t[0] + h * a.stride_h[0] + b * 32 + lane8 * 4, a.wide[0]);
    const unsigned q = quantize8<KF>(v, lane8, scale);
    const int64_t tile = unit * 2 + (token32 >> 4);  // 16 tokens
    const int dword = kv_k_dword(NB, KF, token16, b, lane8 >> 1, lane8 & 1);
    if constexpr (KF == KV_Q8_0) {
      reinterpret_cast<unsigned*>(a.c.kq)[tile * (128 * NB) + dword] = q;
    } else {
      const unsigned n = (q & 15) | (q >> 4 & 0xF0) | (q >> 8 & 0xF00) | (q >> 12 & 0xF000);
      reinterpret_cast<uint16_t*>(a.c.kq)[(tile * (64 * NB) + dword) * 2 + (lane8 & 1)] = static_cast<uint16_t>(n);
    }
    if (lane8 == 0) a.c.ks[tile * (16 * NB) + kv_k_scale(NB, token16, b)] = scale;
  } else {
    const f32x4 v = load4<TYPE>(a.x[1], t * a.stride_t[1] + h * a.stride_h[1] + b * 32 + lane8 * 4, a.wide[1]);
    unsigned q = quantize8<VF>(v, lane8, scale);
    uint8_t* base = a.c.vq + unit * (32 * NB * kv_code_bytes(VF));
    const int channel = (lane8 & 3) * 4;
    if constexpr (VF == KV_Q4_0) q |= __shfl_xor(static_cast<int>(q), 4, 64) << 4;  // used by lanes 0..3: channels + 16
    if (VF == KV_Q8_0 || lane8 < 4) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        base[kv_v_byte(NB, VF, token32, b, channel + e, lane8 >> 2)] = static_cast<uint8_t>(q >> (8 * e));
    }
    if (lane8 == 0) a.c.vs[unit * (32 * NB) + kv_v_scale(NB, token32, b)] = scale;
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

template <int KF, int VF, int NB, int TYPE>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(const ReadArgs a) {
  const int64_t gid = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (gid >= a.lanes) return;
  const int lane8 = static_cast<int>(gid & 7);
  const int64_t blk = gid >> 3;
  const int b = static_cast<int>(blk % NB);
  const int64_t th = blk / NB;
  const int64_t t = th / a.c.heads;
  const int h = static_cast<int>(th - t * a.c.heads);
  const int64_t slot = a.slots[t];
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  if (slot >= 0 && slot < a.c.pages << a.c.page_log2) {
    const int64_t unit = unit_of(a.c, slot, h);
    const int token32 = static_cast<int>(slot & 31), token16 = token32 & 15;
    uint16_t scale;
    int q[4];
    if (blockIdx.y == 0) {
      const int64_t tile = unit * 2 + (token32 >> 4);
      const int dword = kv_k_dword(NB, KF, token16, b, lane8 >> 1, lane8 & 1);
      scale = a.c.ks[tile * (16 * NB) + kv_k_scale(NB, token16, b)];
      if constexpr (KF == KV_Q8_0) {
        const unsigned w = reinterpret_cast<const unsigned*>(a.c.kq)[tile * (128 * NB) + dword];
#pragma unroll
        for (int e = 0; e < 4; ++e) q[e] = static_cast<int>(w >> (8 * e) & 255) - 128;
      } else {
        const unsigned w = reinterpret_cast<const uint16_t*>(a.c.kq)[(tile * (64 * NB) + dword) * 2 + (lane8 & 1)];
#pragma unroll
        for (int e = 0; e < 4; ++e) q[e] = static_cast<int>(w >> (4 * e) & 15) - 8;
      }
    } else {
      const uint8_t* base = a.c.vq + unit * (32 * NB * kv_code_bytes(VF));
      scale = a.c.vs[unit * (32 * NB) + kv_v_scale(NB, token32, b)];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int w = base[kv_v_byte(NB, VF, token32, b, (lane8 & 3) * 4 + e, lane8 >> 2)];
        q[e] = VF == KV_Q8_0 ? w - 128 : (lane8 < 4 ? w & 15 : w >> 4) - 8;
      }
    }
    const float d = f16_bits_to_f32(static_cast<int16_t>(scale));
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = static_cast<float>(q[e]) * d;
  }
  store4<TYPE>(a.x[blockIdx.y], (th * NB + b) * 32 + lane8 * 4, v);
}

template <typename F, typename A>
hipError_t launch(F kern, int64_t lanes, hipStream_t stream, const A& a) {
  const dim3 grid(static_cast<unsigned>((lanes + kThreads - 1) / kThreads), 2);
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
  a.lanes = w.tokens * w.cache.heads * (w.cache.dim / 4);
  const int size = w.type == KV_F32 ? 4 : 2;
  for (int i = 0; i < 2; ++i) {
    a.x[i] = i ? w.v : w.k;
    a.stride_t[i] = w.stride_t[i];
    a.stride_h[i] = w.stride_h[i];
    a.wide[i] = reinterpret_cast<uintptr_t>(a.x[i]) % (4 * size) == 0 && w.stride_t[i] % 4 == 0 && w.stride_h[i] % 4 == 0;
  }
  return with_constants(w.cache, w.type, [&](auto kf, auto vf, auto nb, auto type) {
    return launch(kv_write_kernel<kf.value, vf.value, nb.value, type.value>, a.lanes, stream, a);
  });
}

hipError_t launch_kv_read(const KvReadCall& r, hipStream_t stream) {
  ReadArgs a;
  a.c = r.cache;
  a.slots = r.slots;
  a.lanes = r.tokens * r.cache.heads * (r.cache.dim / 4);
  a.x[0] = r.k;
  a.x[1] = r.v;
  return with_constants(r.cache, r.type, [&](auto kf, auto vf, auto nb, auto type) {
    return launch(kv_read_kernel<kf.value, vf.value, nb.value, type.value>, a.lanes, stream, a);
  });
}

}  // namespace komp
