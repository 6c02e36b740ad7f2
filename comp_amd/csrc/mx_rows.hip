// Rows into microscaled elements and back: quantize, gate, lookup, pack (layout: mx_layout.h, formats: mx_device.h).
//
// A workgroup has a tile of 16 rows and four steps of 128 elements (of shorter rows several tiles), a step a wave: lane 4 r + q holds elements 8 q .. 8 q + 7
// of a block of row r, for the step's four blocks.  A row's reads are 128 contiguous elements a wave, a tile's codes leave in
// runs of 256 bytes, and the four steps' scale bytes meet in shared memory and leave as dwords.
//
// Bound by bytes: 28672 x 8192 f16 values become e2m1 in 110 us (595 MB, 5.4 TB/s) and bf16 values again in 92-107; 3001 x 14336 gated
// bf16 pairs e2m1 in 46-49 us (4.0 TB/s; vector instructions issue 56% of the time); 16383 rows of 2560 are looked up in 40 us (a row's blocks
// lie 256 bytes apart, so 16 bytes are used of each line that is fetched), one row of 4096 is quantized in 2.9 us and read in 2.3.
// Short rows share a wave or a workgroup: a million rows of 32 (f32 to e4m3) are quantized in 41 us (a workgroup a row tile 69), gated
// in 73, looked up in 18 (80).
//
// Plain planes of 28672 x 8192 become rows in 67 us (e2m1; 113 in e4m3), ggml's blocks in 81, and rows plain planes in 142 (199); copying the codes
// alone takes 45 (88).  An instruction of a wave has only 16 bytes (32) of each of 16 rows on the plain side; a weight goes this way once.
#include <hip/hip_ext.h>

#include <type_traits>

#include "komp_internal.h"
#include "mx_device.h"

namespace komp {
namespace {

constexpr int kThreads = 256;
// workgroups of a launch at most (a grid holds 2^32 threads); they walk over more tiles than that
constexpr unsigned kGrid = 1u << 22;

// The product whose rounding to f32 is quantized, from 64 bits.
template <int ACT>
__device__ __forceinline__ float mx_act(float g, float u) {
  const double a = g, b = u;
  if constexpr (ACT == MX_SILU) return static_cast<float>(a / (1.0 + exp(-a)) * b);
  const double p = a > 0.0 ? a : a != a ? a : 0.0;
  return static_cast<float>(p * p * b);
}

// The same in f32, within 2^-20 of it for products from 2^-126 on and gates from -80 on.  e^-g is 2^t with t = -g log2(e) in two
// parts, so that t's rounding (up to 2^-18) does not count; the exponential and the reciprocal are off by one step each.  The
// gate meets the other factor first: a step that leaves f32's range on the way to a product inside it is infinite, never a zero.
template <int ACT>
__device__ __forceinline__ float mx_act_near(float g, float u) {
  if constexpr (ACT == MX_SILU) {
    const float t = g * -1.44269502f, rest = __builtin_fmaf(g, -1.92596303e-8f, __builtin_fmaf(g, -1.44269502f, -t));
    const float e = __builtin_amdgcn_exp2f(t);
    return g * u * __builtin_amdgcn_rcpf(1.f + __builtin_fmaf(e, rest * 0.693147182f, e));
  } else {
    const float p = __builtin_fmaxf(g, 0.f);
    return p * u * p;
  }
}

// the largest of a quad of lanes
__device__ __forceinline__ unsigned most4(unsigned most) {
  most = umax(most, static_cast<unsigned>(dpp_i<KOMP_DPP_XOR1>(static_cast<int>(most))));
  return umax(most, static_cast<unsigned>(dpp_i<KOMP_DPP_XOR2>(static_cast<int>(most))));
}

// A quad of lanes' block of gated products: scale and codes.  They come from f32 products where all that these may stand for, 2^-19 to
// either side, give the same ones (scale and rounding are monotonous), and from 64 bits otherwise: with e4m3 one block in a thousand
// (2^-15 an element).  Blocks of products below 2^-60, with values that are no numbers, or with gates below -80 take 64 bits too, and so do
// blocks with a product of -0, whose two ends have different signs: with squared ReLU nearly every block (g <= 0 beside u < 0).  That
// costs nothing that shows: 8192 x 4096 to e4m3 take 42 us with either activation.
template <int FMT, int ACT>
__device__ __forceinline__ void gate8(const float (&g)[8], const float (&u)[8], unsigned& s, unsigned (&c)[FMT == MX_E2M1 ? 1 : 2]) {
  float low[8], high[8], largest = 0.f, least = 0.f, zero = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float v = mx_act_near<ACT>(g[e], u[e]);
    largest = __builtin_fmaxf(largest, __builtin_fabsf(v));
    zero = __builtin_fmaf(v, 0.f, zero);  // NaN from an infinity or a NaN on
    if constexpr (ACT == MX_SILU) least = __builtin_fminf(least, g[e]);
    else zero = __builtin_fmaf(g[e], 0.f, zero);
    low[e] = v - v * 0x1p-19f;
    high[e] = v + v * 0x1p-19f;
  }
  const unsigned most = most4(__float_as_uint(largest));
  s = mx_scale<FMT>(most);
  // (2^-19 are up to 32 steps of an f32)
  bool far = !(zero == 0.f) || least < -80.f || most < (67u << 23) || mx_scale<FMT>(most - 32) != s || mx_scale<FMT>(most + 32) != s;
  unsigned d[FMT == MX_E2M1 ? 1 : 2];
  mx_codes8<FMT>(low, s, c);
  mx_codes8<FMT>(high, s, d);
#pragma unroll
  for (int h = 0; h < (FMT == MX_E2M1 ? 1 : 2); ++h) far |= c[h] != d[h];
  if (most4(far) != 0) {
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = mx_act<ACT>(g[e], u[e]);
    s = mx_scale<FMT>(most4(mx_most(v)));
    mx_codes8<FMT>(v, s, c);
  }
}

struct QuantArgs {
  MxRows r;
  const void* x;
  int64_t stride;
  unsigned tiles;  // groups of row tiles times four-step pieces, below 2^31
  int waves_log2;  // waves a row tile: 4, or as many as a shorter row has steps (a power of two)
};

template <int FMT, int TYPE, int ACT>
__global__ __launch_bounds__(kThreads) void mx_quantize_kernel(const QuantArgs a) {
  __shared__ unsigned scales[kThreads / 64][64];
  const int wave = threadIdx.x >> 6, row = (threadIdx.x & 63) >> 2, q = threadIdx.x & 3;
  const int own = wave & ((1 << a.waves_log2) - 1), which = wave >> a.waves_log2;  // step of the piece, row tile of the group
  const int64_t steps = mx_steps(a.r.k), blocks = a.r.k >> 5;
  const unsigned supers = static_cast<unsigned>(mx_supers(a.r.k));
  for (unsigned tile = blockIdx.x; tile < a.tiles; tile += gridDim.x) {
    const int64_t rt = static_cast<int64_t>(tile / supers) * (4 >> a.waves_log2) + which, piece = tile % supers;
    const int64_t step = piece * 4 + own, r = rt * 16 + row;
    const bool there = rt * 16 < a.r.rows;
    if (a.waves_log2 < 2) {  // steps that no wave has
      if (own == 0) scales[which][threadIdx.x & 63] = 0;
      __syncthreads();
    }
    float v[4][8], u[ACT == MX_PLAIN ? 1 : 4][8];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int64_t b = step * 4 + g;
      if (b < blocks && r < a.r.rows) {
        mx_load<TYPE>(a.x, r * a.stride + b * 32 + q * 8, v[g]);
        if constexpr (ACT != MX_PLAIN) mx_load<TYPE>(a.x, r * a.stride + a.r.k + b * 32 + q * 8, u[g]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[g][e] = 0.f;
        if constexpr (ACT != MX_PLAIN) {
#pragma unroll
          for (int e = 0; e < 8; ++e) u[g][e] = 0.f;
        }
      }
    }
    uint8_t* const codes = a.r.codes + rt * mx_code_bytes(a.r.k, FMT);
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      unsigned s, c[FMT == MX_E2M1 ? 1 : 2];
      if constexpr (ACT == MX_PLAIN) {
        s = mx_scale<FMT>(most4(mx_most(v[g])));
        mx_codes8<FMT>(v[g], s, c);
      } else if (step * 4 + g < blocks && r < a.r.rows) {  // (quads of lanes; blocks of zeros would take 64 bits)
        gate8<FMT, ACT>(v[g], u[g], s, c);
      } else {
        s = 0;
#pragma unroll
        for (unsigned& code : c) code = 0;
      }
      if (there && step < steps) {
        if constexpr (FMT == MX_E2M1) {
          *reinterpret_cast<unsigned*>(codes + step * 1024 + (g * 16 + row) * 16 + q * 4) = c[0];
        } else {
          *reinterpret_cast<u32x2*>(codes + step * 2048 + (q >> 1) * 1024 + (g * 16 + row) * 16 + (q & 1) * 8) = u32x2{c[0], c[1]};
        }
      }
      if (q == 0) reinterpret_cast<uint8_t*>(scales[which])[(g * 16 + row) * 4 + own] = static_cast<uint8_t>(s);
    }
    __syncthreads();
    if (there && own == 0)
      reinterpret_cast<unsigned*>(a.r.scales + rt * mx_scale_bytes(a.r.k) + piece * 256)[threadIdx.x & 63] = scales[which][threadIdx.x & 63];
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
  unsigned tiles;  // groups of rows times pieces of 512 elements
  int lanes_log2;  // lanes a row: 16, or as many as a shorter row has blocks (a power of two)
};

// A wave has 64 blocks: 512 elements of four of the rows asked for, or more rows that are shorter.  A lane loads one block, 16 or
// 32 bytes from anywhere, and through shared memory the wave turns them into whole rows, 1 KB a store.
template <int FMT, int TYPE>
__global__ __launch_bounds__(kThreads) void mx_lookup_kernel(const LookupArgs a) {
  constexpr int kParts = FMT == MX_E2M1 ? 1 : 2;
  constexpr int kE = TYPE == MX_F32 ? 4 : 8;  // elements a store
  constexpr unsigned kMissing = 1u << 31;     // in a scale's place: no such row
  __shared__ u32x4 codes_of[kThreads / 64][64 * kParts];
  __shared__ unsigned scales_of[kThreads / 64][64];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, block = lane & ((1 << a.lanes_log2) - 1);
  const int64_t blocks = a.r.k >> 5;
  const unsigned supers = static_cast<unsigned>(mx_supers(a.r.k));
  for (unsigned tile = blockIdx.x; tile < a.tiles; tile += gridDim.x) {
    const int64_t t0 = (static_cast<int64_t>(tile / supers) * 4 + wave) * (64 >> a.lanes_log2), piece = tile % supers;
    const int64_t t = t0 + (lane >> a.lanes_log2);
    int64_t id = -1;
    if (t < a.count) id = a.ids == nullptr ? t : a.ids[t];
    const bool there = id >= 0 && id < a.r.rows;
    u32x4 c[kParts];
    unsigned s = 0;
#pragma unroll
    for (int h = 0; h < kParts; ++h) c[h] = u32x4{0, 0, 0, 0};
    if (there && piece * 16 + block < blocks) {
      const int at = (block & 3) * 16 + static_cast<int>(id & 15);
      const u32x4* const from =
          reinterpret_cast<const u32x4*>(a.r.codes + (id >> 4) * mx_code_bytes(a.r.k, FMT)) + (piece * 4 + (block >> 2)) * 64 * kParts + at;
#pragma unroll
      for (int h = 0; h < kParts; ++h) c[h] = from[h * 64];
      s = (a.r.scales + (id >> 4) * mx_scale_bytes(a.r.k) + piece * 256)[at * 4 + (block >> 2)];
    }
    // (a wave's own places: its reads of the turn before are done, in order)
#pragma unroll
    for (int h = 0; h < kParts; ++h) codes_of[wave][lane * kParts + h] = c[h];
    scales_of[wave][lane] = there ? s << 23 : kMissing;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int p = 0; p < 32 / kE; ++p) {
      const int f = (p * 64 + lane) * kE;  // of the wave's 2048 elements
      const int row = f >> (5 + a.lanes_log2), e = f & ((32 << a.lanes_log2) - 1);
      if (t0 + row >= a.count || piece * 16 + (e >> 5) >= blocks) continue;
      const unsigned scale = scales_of[wave][f >> 5];
      const uint8_t* const from = reinterpret_cast<const uint8_t*>(codes_of[wave]) + (FMT == MX_E2M1 ? f / 2 : f);
      float v[kE];
      mx_values<FMT, kE>(from, __uint_as_float(scale), v);
#pragma unroll
      for (int i = 0; i < kE; ++i) {
        v[i] = scale == kMissing ? 0.f : v[i] * a.factor;
        // the compiler makes v_fma_mixlo_f16 with an addend of +0 of a product and its rounding to f16, which loses -0
        if constexpr (TYPE == MX_F16) asm("" : "+v"(v[i]));
      }
      mx_store<TYPE>(a.out, (t0 + row) * a.stride + piece * 512 + e, v);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
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
  const int waves_log2 = c.r.k <= 128 ? 0 : c.r.k <= 256 ? 1 : 2;
  const int64_t group = 4 >> waves_log2;  // row tiles of a workgroup
  const QuantArgs a{c.r, c.x, c.stride, static_cast<unsigned>((mx_tiles(c.r.rows) + group - 1) / group * mx_supers(c.r.k)), waves_log2};
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
  int lanes_log2 = 0;
  while (lanes_log2 < 4 && (INT64_C(32) << lanes_log2) < c.r.k) ++lanes_log2;
  const int64_t rows = 256 >> lanes_log2;  // a workgroup
  const LookupArgs a{c.r, c.ids, c.count, c.out, c.stride, c.factor,
                     static_cast<unsigned>((c.count + rows - 1) / rows * mx_supers(c.r.k)), lanes_log2};
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
