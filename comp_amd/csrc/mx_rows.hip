// Rows into microscaled elements and back: quantize, gate, lookup, pack (layout: mx_layout.h, formats: mx_device.h).
//
// A workgroup has a tile of 16 rows and four steps of 128 elements, a step a wave: lane 4 r + q holds elements 8 q .. 8 q + 7
// of a block of row r, for the step's four blocks.  A row's reads are 128 contiguous elements a wave, a tile's codes leave in
// runs of 256 bytes, and the four steps' scale bytes meet in shared memory and leave as dwords.
#include <hip/hip_ext.h>

#include <type_traits>

#include "komp_internal.h"
#include "mx_device.h"

namespace komp {
namespace {

constexpr int kThreads = 256;
// workgroups of a launch at most (a grid holds 2^32 threads); they walk over more tiles than that
constexpr unsigned kGrid = 1u << 22;

// The product whose rounding to f32 is quantized, from 64 bits: an f32 exp would be off by enough to move values over an
// element's border.
template <int ACT>
__device__ __forceinline__ float mx_act(float g, float u) {
  const double a = g, b = u;
  if constexpr (ACT == MX_SILU) return static_cast<float>(a / (1.0 + exp(-a)) * b);
  const double p = a > 0.0 ? a : a != a ? a : 0.0;
  return static_cast<float>(p * p * b);
}

struct QuantArgs {
  MxRows r;
  const void* x;
  int64_t stride;
  unsigned tiles;  // row tiles times four-step pieces, below 2^31
};

template <int FMT, int TYPE, int ACT>
__global__ __launch_bounds__(kThreads) void mx_quantize_kernel(const QuantArgs a) {
  __shared__ unsigned scales[64];
  const int wave = threadIdx.x >> 6, row = (threadIdx.x & 63) >> 2, q = threadIdx.x & 3;
  const int64_t steps = mx_steps(a.r.k), blocks = a.r.k >> 5;
  const unsigned supers = static_cast<unsigned>(mx_supers(a.r.k));
  for (unsigned tile = blockIdx.x; tile < a.tiles; tile += gridDim.x) {
    const int64_t rt = tile / supers, piece = tile % supers;
    const int64_t step = piece * 4 + wave, r = rt * 16 + row;
    float v[4][8];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int64_t b = step * 4 + g;
      if (b < blocks && r < a.r.rows) {
        mx_load<TYPE>(a.x, r * a.stride + b * 32 + q * 8, v[g]);
        if constexpr (ACT != MX_PLAIN) {
          float u[8];
          mx_load<TYPE>(a.x, r * a.stride + a.r.k + b * 32 + q * 8, u);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[g][e] = mx_act<ACT>(v[g][e], u[e]);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[g][e] = 0.f;
      }
    }
    uint8_t* const codes = a.r.codes + rt * mx_code_bytes(a.r.k, FMT);
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      unsigned most = mx_most(v[g]);
      most = umax(most, static_cast<unsigned>(dpp_i<KOMP_DPP_XOR1>(static_cast<int>(most))));
      most = umax(most, static_cast<unsigned>(dpp_i<KOMP_DPP_XOR2>(static_cast<int>(most))));
      const unsigned s = mx_scale<FMT>(most);
      if (step < steps) {
        if constexpr (FMT == MX_E2M1) {
          unsigned c[1];
          mx_codes8<FMT>(v[g], s, c);
          *reinterpret_cast<unsigned*>(codes + step * 1024 + (g * 16 + row) * 16 + q * 4) = c[0];
        } else {
          unsigned c[2];
          mx_codes8<FMT>(v[g], s, c);
          *reinterpret_cast<u32x2*>(codes + step * 2048 + (q >> 1) * 1024 + (g * 16 + row) * 16 + (q & 1) * 8) = u32x2{c[0], c[1]};
        }
      }
      if (q == 0) reinterpret_cast<uint8_t*>(scales)[(g * 16 + row) * 4 + wave] = static_cast<uint8_t>(s);
    }
    __syncthreads();
    if (threadIdx.x < 64)
      reinterpret_cast<unsigned*>(a.r.scales + rt * mx_scale_bytes(a.r.k) + piece * 256)[threadIdx.x] = scales[threadIdx.x];
    __syncthreads();
  }
}

struct LookupArgs {
  MxRows r;
  const int64_t* ids;
  int64_t count;
  void* out;
  int64_t stride;
  float factor;
  unsigned tiles;
};

template <int FMT, int TYPE>
__global__ __launch_bounds__(kThreads) void mx_lookup_kernel(const LookupArgs a) {
  const int wave = threadIdx.x >> 6, row = (threadIdx.x & 63) >> 2, q = threadIdx.x & 3;
  const int64_t blocks = a.r.k >> 5;
  const unsigned supers = static_cast<unsigned>(mx_supers(a.r.k));
  for (unsigned tile = blockIdx.x; tile < a.tiles; tile += gridDim.x) {
    const int64_t t16 = tile / supers, piece = tile % supers;
    const int64_t step = piece * 4 + wave, t = t16 * 16 + row;
    if (t >= a.count) continue;
    const int64_t id = a.ids == nullptr ? t : a.ids[t];
    const bool in = id >= 0 && id < a.r.rows;
    const int64_t rt = in ? id >> 4 : 0;
    const int lane = in ? static_cast<int>(id & 15) : 0;
    const uint8_t* const codes = a.r.codes + rt * mx_code_bytes(a.r.k, FMT);
    const uint8_t* const scales = a.r.scales + rt * mx_scale_bytes(a.r.k) + piece * 256;
    unsigned c[4][FMT == MX_E2M1 ? 1 : 2], s[4];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      c[g][0] = 0;
      if constexpr (FMT == MX_E4M3) c[g][1] = 0;
      s[g] = 0;
      if (in && step * 4 + g < blocks) {
        s[g] = scales[(g * 16 + lane) * 4 + wave];
        if constexpr (FMT == MX_E2M1) {
          c[g][0] = *reinterpret_cast<const unsigned*>(codes + step * 1024 + (g * 16 + lane) * 16 + q * 4);
        } else {
          const u32x2 w = *reinterpret_cast<const u32x2*>(codes + step * 2048 + (q >> 1) * 1024 + (g * 16 + lane) * 16 + (q & 1) * 8);
          c[g][0] = w[0];
          c[g][1] = w[1];
        }
      }
    }
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int64_t b = step * 4 + g;
      if (b >= blocks) continue;
      float v[8];
      mx_values8<FMT>(c[g], s[g], v);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[e] = in ? v[e] * a.factor : 0.f;
        // the compiler makes v_fma_mixlo_f16 with an addend of +0 of a product and its rounding to f16, which loses -0
        if constexpr (TYPE == MX_F16) asm("" : "+v"(v[e]));
      }
      mx_store<TYPE>(a.out, t * a.stride + b * 32 + q * 8, v);
    }
  }
}

struct PackArgs {
  MxRows r;
  uint8_t* codes;
  uint8_t* scales;
  unsigned tiles;
};

// Plain planes into rows, UNPACK: rows into plain planes.  ggml's 17-byte blocks hold the scale byte and 16 bytes whose byte j has
// element j in its low and element j + 16 in its high nibble.
template <int FMT, bool GGML, bool UNPACK>
__global__ __launch_bounds__(kThreads) void mx_pack_kernel(const PackArgs a) {
  __shared__ unsigned scales[64];
  const int wave = threadIdx.x >> 6, row = (threadIdx.x & 63) >> 2, q = threadIdx.x & 3;
  const int64_t steps = mx_steps(a.r.k), blocks = a.r.k >> 5;
  const unsigned supers = static_cast<unsigned>(mx_supers(a.r.k));
  typedef u32x2 loose2 __attribute__((aligned(1)));
  typedef unsigned loose __attribute__((aligned(1)));
  for (unsigned tile = blockIdx.x; tile < a.tiles; tile += gridDim.x) {
    const int64_t rt = tile / supers, piece = tile % supers;
    const int64_t step = piece * 4 + wave, r = rt * 16 + row;
    uint8_t* const codes = a.r.codes + rt * mx_code_bytes(a.r.k, FMT);
    uint8_t* const held = a.r.scales + rt * mx_scale_bytes(a.r.k) + piece * 256;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int64_t b = step * 4 + g, at = r * blocks + b;
      const bool in = b < blocks && r < a.r.rows;
      unsigned* const place = reinterpret_cast<unsigned*>(
          FMT == MX_E2M1 ? codes + step * 1024 + (g * 16 + row) * 16 + q * 4
                         : codes + step * 2048 + (q >> 1) * 1024 + (g * 16 + row) * 16 + (q & 1) * 8);
      uint8_t* const plain = a.codes + (GGML ? at * 17 + 1 : FMT == MX_E2M1 ? at * 16 + q * 4 : at * 32 + q * 8);
      if constexpr (UNPACK) {
        if (!in) continue;
        if constexpr (FMT == MX_E2M1) {
          *reinterpret_cast<loose*>(plain) = place[0];
        } else {
          *reinterpret_cast<loose2*>(plain) = u32x2{place[0], place[1]};
        }
        if (q == 0) a.scales[at] = held[(g * 16 + row) * 4 + wave];
      } else {
        u32x2 c = {0, 0};
        uint8_t s = 0;
        if (in) {
          if constexpr (GGML) {
            const u32x2 w = *reinterpret_cast<const loose2*>(plain + (q & 1) * 8);
            const int shift = (q >> 1) * 4;
#pragma unroll
            for (int e = 0; e < 8; ++e) c[0] |= ((w[e >> 2] >> ((e & 3) * 8 + shift)) & 15u) << (4 * e);
            s = plain[-1];
          } else {
            if constexpr (FMT == MX_E2M1) c[0] = *reinterpret_cast<const loose*>(plain);
            else c = *reinterpret_cast<const loose2*>(plain);
            s = a.scales[at];
          }
        }
        if (step < steps) {
          place[0] = c[0];
          if constexpr (FMT == MX_E4M3) place[1] = c[1];
        }
        if (q == 0) reinterpret_cast<uint8_t*>(scales)[(g * 16 + row) * 4 + wave] = s;
      }
    }
    if constexpr (!UNPACK) {
      __syncthreads();
      if (threadIdx.x < 64) reinterpret_cast<unsigned*>(held)[threadIdx.x] = scales[threadIdx.x];
      __syncthreads();
    }
  }
}

unsigned piece_count(int64_t rows, int64_t k) { return static_cast<unsigned>(mx_tiles(rows) * mx_supers(k)); }

template <typename Args>
hipError_t launch(void (*kern)(Args), hipStream_t stream, const Args& a) {
  const dim3 grid(a.tiles < kGrid ? a.tiles : kGrid);
  const Timing tm = timing_slot(KIND_PROBE);
  if (tm.on) {
    hipExtLaunchKernelGGL(kern, grid, dim3(kThreads), 0, stream, tm.start, tm.stop, 0, a);
  } else {
    hipLaunchKernelGGL(kern, grid, dim3(kThreads), 0, stream, a);
  }
  return hipGetLastError();
}

// f(format) and f(format, type) with constants
template <typename F>
hipError_t with_format(int fmt, F&& f) {
  if (fmt == MX_E2M1) return f(std::integral_constant<int, MX_E2M1>());
  return f(std::integral_constant<int, MX_E4M3>());
}
template <typename F>
hipError_t with_type(int type, F&& f) {
  if (type == MX_F32) return f(std::integral_constant<int, MX_F32>());
  if (type == MX_F16) return f(std::integral_constant<int, MX_F16>());
  return f(std::integral_constant<int, MX_BF16>());
}

}  // namespace

hipError_t launch_mx_quantize(const MxQuantCall& c, hipStream_t stream) {
  const QuantArgs a{c.r, c.x, c.stride, piece_count(c.r.rows, c.r.k)};
  return with_format(c.r.fmt, [&](auto fmt) {
    return with_type(c.type, [&](auto type) {
      constexpr int FMT = fmt.value, TYPE = type.value;
      if (c.act == MX_SILU) return launch(mx_quantize_kernel<FMT, TYPE, MX_SILU>, stream, a);
      if (c.act == MX_RELU2) return launch(mx_quantize_kernel<FMT, TYPE, MX_RELU2>, stream, a);
      return launch(mx_quantize_kernel<FMT, TYPE, MX_PLAIN>, stream, a);
    });
  });
}

hipError_t launch_mx_lookup(const MxLookupCall& c, hipStream_t stream) {
  const LookupArgs a{c.r, c.ids, c.count, c.out, c.stride, c.factor, piece_count(c.count, c.r.k)};
  return with_format(c.r.fmt, [&](auto fmt) {
    return with_type(c.type, [&](auto type) { return launch(mx_lookup_kernel<fmt.value, type.value>, stream, a); });
  });
}

hipError_t launch_mx_pack(const MxPackCall& c, hipStream_t stream) {
  const PackArgs a{c.r, c.codes, c.scales, piece_count(c.r.rows, c.r.k)};
  if (c.ggml) return launch(mx_pack_kernel<MX_E2M1, true, false>, stream, a);
  return with_format(c.r.fmt, [&](auto fmt) {
    constexpr int FMT = fmt.value;
    return c.unpack ? launch(mx_pack_kernel<FMT, false, true>, stream, a) : launch(mx_pack_kernel<FMT, false, false>, stream, a);
  });
}

}  // namespace komp
