// Products of microscaled rows: Y [T][N] = X W^T, W in e2m1, X in e2m1 or e4m3 or quantized on the way (layout: mx_layout.h).
//
// The weights are the matrix instruction's A operand and the activations its B operand, so a lane's four results are four
// consecutive outputs of one row of X.  X in e2m1: v_mfma_scale_f32_16x16x128_f8f6f4 takes codes and scale bytes as they lie in
// memory; a product of two e2m1 elements has at most four bits, and its sums are f32's.  X in e4m3: that instruction adds a
// block's products of e2m1 and e4m3 with some 15 bits below the largest one (measured: 2688 - 2688 + 1/16 gives 0), which
// is not a 32-bit sum.  So both operands become bf16, scale included, which is exact (four bits at most, and bf16's exponents
// are f32's; only activations below 2^-126 may lose bits), and v_mfma_f32_16x16x32_bf16 adds them in f32.
#include <hip/hip_ext.h>

#include <type_traits>

#include "komp_internal.h"
#include "mx_device.h"

namespace komp {
namespace {

struct GemmArgs {
  const uint8_t* w;        // weight codes and scales
  const uint8_t* ws;
  const uint8_t* x;        // codes (rows), or elements (quantized on the way)
  const uint8_t* xs;
  int64_t x_stride;        // elements between rows, quantized on the way
  int64_t n, t;
  int k;
  void* y;
  int64_t y_stride;
};

// One step's operand of one row tile: codes, and the dword of its four steps' scales.
template <int FMT>
struct Operand {
  u32x4 q[FMT == MX_E2M1 ? 1 : 2];
};

// The B or A operands of v_mfma_f32_16x16x32_bf16 that a lane's block makes: its elements 8 j .. 8 j + 7 for j = 0..3.
template <int FMT>
__device__ __forceinline__ bf16x8 bf16_part(const Operand<FMT>& o, int j, float scale) {
  bf16x2 p[4];
  if constexpr (FMT == MX_E2M1) {
    const unsigned q = o.q[0][j];
    p[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 0);
    p[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 1);
    p[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 2);
    p[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 3);
  } else {
    const unsigned q = o.q[j >> 1][2 * (j & 1)], r = o.q[j >> 1][2 * (j & 1) + 1];
    p[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q, scale, false);
    p[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q, scale, true);
    p[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(r, scale, false);
    p[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(r, scale, true);
  }
  return __builtin_shufflevector(__builtin_shufflevector(p[0], p[1], 0, 1, 2, 3), __builtin_shufflevector(p[2], p[3], 0, 1, 2, 3),
                                 0, 1, 2, 3, 4, 5, 6, 7);
}

__device__ __forceinline__ float scale_of(unsigned four, int step) {
  return __uint_as_float(((four >> (8 * step)) & 255u) << 23);
}

// acc += one step's products; STEP (0..3) picks the scale bytes.
template <int FMT, int STEP, int RT, int CT>
__device__ __forceinline__ void mma_step(f32x4 (&acc)[RT][CT], const Operand<MX_E2M1> (&w)[RT], const unsigned (&ws)[RT],
                                         const Operand<FMT> (&x)[CT], const unsigned (&xs)[CT]) {
  if constexpr (FMT == MX_E2M1) {
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int j = 0; j < CT; ++j) {
        const u32x4 a = w[i].q[0], b = x[j].q[0];
        const i32x8 a8 = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
        const i32x8 b8 = {(int)b[0], (int)b[1], (int)b[2], (int)b[3], 0, 0, 0, 0};
        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a8, b8, acc[i][j], 4, 4, STEP, static_cast<int>(ws[i]), STEP,
                                                                     static_cast<int>(xs[j]));
      }
  } else {
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      bf16x8 b[CT];
#pragma unroll
      for (int j = 0; j < CT; ++j) b[j] = bf16_part(x[j], p, scale_of(xs[j], STEP));
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        const bf16x8 a = bf16_part(w[i], p, scale_of(ws[i], STEP));
#pragma unroll
        for (int j = 0; j < CT; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b[j], acc[i][j], 0, 0, 0);
      }
    }
  }
}

// Four outputs n .. n + 3 of row t.
template <int TYPE>
__device__ __forceinline__ void store4(const GemmArgs& a, int64_t t, int64_t n, f32x4 v) {
  if (t >= a.t || n >= a.n) return;
  const int64_t at = t * a.y_stride + n;
  if (n + 4 <= a.n) {
    const float f[4] = {v[0], v[1], v[2], v[3]};
    mx_store<TYPE>(a.y, at, f);
  } else {
#pragma unroll
    for (int e = 0; e < 3; ++e) {
      const float f[1] = {v[e]};
      if (n + e < a.n) mx_store<TYPE>(a.y, at + e, f);
    }
  }
}

// ---- few rows of X ---------------------------------------------------------------------------------------------------

// Operands come straight from memory: a workgroup has RT row tiles of W and CT tiles of X, its waves take four-step pieces of
// K in turn and join in shared memory, in the waves' order.  SRC: the type of the rows that are quantized on the way (each wave
// its own pieces), -1: X is quantized already.
template <int FMT, int SRC, int TYPE, int RT, int CT>
__global__ __launch_bounds__(512) void mx_stream_kernel(const GemmArgs a) {
  extern __shared__ f32x4 join[];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const int steps = static_cast<int>(mx_steps(a.k)), supers = static_cast<int>(mx_supers(a.k));
  const int64_t w_tiles = mx_tiles(a.n), x_tiles = mx_tiles(a.t);
  const int64_t w0 = static_cast<int64_t>(blockIdx.x) * RT, x0 = static_cast<int64_t>(blockIdx.y) * CT;
  const int64_t w_bytes = mx_code_bytes(a.k, MX_E2M1), x_bytes = mx_code_bytes(a.k, FMT), s_bytes = mx_scale_bytes(a.k);
  // a tile past the last one is read again as the last one, and not stored
  auto tile_of = [](int64_t tile, int64_t tiles) { return tile < tiles ? tile : tiles - 1; };
  f32x4 acc[RT][CT];
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int j = 0; j < CT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int sp = wave; sp < supers; sp += waves) {
    Operand<MX_E2M1> w[4][RT];
    unsigned ws[RT], xs[CT];
    Operand<FMT> x[4][CT];
    const int here = steps - sp * 4;  // steps of this piece
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      const int64_t tile = tile_of(w0 + i, w_tiles);
      ws[i] = reinterpret_cast<const unsigned*>(a.ws + tile * s_bytes)[sp * 64 + lane];
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const int step = sp * 4 + (s < here ? s : here - 1);
        w[s][i].q[0] = reinterpret_cast<const u32x4*>(a.w + tile * w_bytes)[step * 64 + lane];
      }
    }
    if constexpr (SRC < 0) {
#pragma unroll
      for (int j = 0; j < CT; ++j) {
        const int64_t tile = tile_of(x0 + j, x_tiles);
        xs[j] = reinterpret_cast<const unsigned*>(a.xs + tile * s_bytes)[sp * 64 + lane];
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          const int step = sp * 4 + (s < here ? s : here - 1);
          constexpr int parts = FMT == MX_E2M1 ? 1 : 2;
#pragma unroll
          for (int h = 0; h < parts; ++h)
            x[s][j].q[h] = reinterpret_cast<const u32x4*>(a.x + tile * x_bytes)[(step * parts + h) * 64 + lane];
        }
      }
    } else {
      static_assert(SRC < 0 || CT == 1, "one column tile");
      xs[0] = 0;
      const int64_t row = lane & 15;
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const int block = (sp * 4 + s) * 4 + (lane >> 4);
        float v[32];
        if (row < a.t && block * 32 < a.k) {
#pragma unroll
          for (int e = 0; e < 4; ++e) mx_load<SRC>(a.x, row * a.x_stride + block * 32 + e * 8, *reinterpret_cast<float(*)[8]>(v + 8 * e));
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) v[e] = 0.f;
        }
        const unsigned scale = mx_scale<FMT>(mx_most(v));
        xs[0] |= scale << (8 * s);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          unsigned c[FMT == MX_E2M1 ? 1 : 2];
          mx_codes8<FMT>(v + 8 * e, scale, c);
          if constexpr (FMT == MX_E2M1) {
            x[s][0].q[0][e] = c[0];
          } else {
            x[s][0].q[e >> 1][2 * (e & 1)] = c[0];
            x[s][0].q[e >> 1][2 * (e & 1) + 1] = c[1];
          }
        }
      }
    }
    mma_step<FMT, 0>(acc, w[0], ws, x[0], xs);
    if (here > 1) mma_step<FMT, 1>(acc, w[1], ws, x[1], xs);
    if (here > 2) mma_step<FMT, 2>(acc, w[2], ws, x[2], xs);
    if (here > 3) mma_step<FMT, 3>(acc, w[3], ws, x[3], xs);
  }
  auto put = [&](int i, int j, int l, f32x4 v) {
    store4<TYPE>(a, (x0 + j) * 16 + (l & 15), (w0 + i) * 16 + (l >> 4) * 4, v);
  };
  if (waves == 1) {
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int j = 0; j < CT; ++j) put(i, j, lane, acc[i][j]);
    return;
  }
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int j = 0; j < CT; ++j) join[(wave * RT * CT + i * CT + j) * 64 + lane] = acc[i][j];
  __syncthreads();
  for (int p = wave; p < RT * CT; p += waves) {
    f32x4 sum = join[p * 64 + lane];
    for (int w = 1; w < waves; ++w) sum += join[(w * RT * CT + p) * 64 + lane];
    put(p / CT, p % CT, lane, sum);
  }
}

// ---- many rows of X --------------------------------------------------------------------------------------------------

// A workgroup of GN x GT waves has GN * WN row tiles of W and GT * WT of X: a step's codes go through shared memory, two
// buffers, the next step's loads in flight during one step's products; scales come straight from memory, four steps at once.
template <int FMT, int TYPE, int WN, int WT, int GN, int GT>
__global__ __launch_bounds__(GN* GT * 64) void mx_tile_kernel(const GemmArgs a) {
  constexpr int kParts = FMT == MX_E2M1 ? 1 : 2, kWaves = GN * GT;
  constexpr int kW = GN * WN, kX = GT * WT * kParts, kPieces = kW + kX, kLoads = (kPieces + kWaves - 1) / kWaves;  // 1 KB each
  __shared__ u32x4 buffer[2][kPieces * 64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wn = wave % GN, wt = wave / GN;
  const int steps = static_cast<int>(mx_steps(a.k)), supers = static_cast<int>(mx_supers(a.k));
  const int64_t w_tiles = mx_tiles(a.n), x_tiles = mx_tiles(a.t);
  const int64_t w0 = static_cast<int64_t>(blockIdx.x) * kW, x0 = static_cast<int64_t>(blockIdx.y) * (GT * WT);
  const int64_t w_bytes = mx_code_bytes(a.k, MX_E2M1), x_bytes = mx_code_bytes(a.k, FMT), s_bytes = mx_scale_bytes(a.k);
  auto tile_of = [](int64_t tile, int64_t tiles) { return tile < tiles ? tile : tiles - 1; };
  // this wave's pieces of a step: where they come from
  const u32x4* from[kLoads];
  int pace[kLoads];
#pragma unroll
  for (int l = 0; l < kLoads; ++l) {
    const int p = wave + l * kWaves;
    if (p < kW) {
      from[l] = reinterpret_cast<const u32x4*>(a.w + tile_of(w0 + p, w_tiles) * w_bytes) + lane;
      pace[l] = 64;
    } else {
      const int c = p < kPieces ? p - kW : 0;
      from[l] = reinterpret_cast<const u32x4*>(a.x + tile_of(x0 + c / kParts, x_tiles) * x_bytes) + (c % kParts) * 64 + lane;
      pace[l] = 64 * kParts;
    }
  }
  const unsigned *ws_at[WN], *xs_at[WT];
#pragma unroll
  for (int i = 0; i < WN; ++i)
    ws_at[i] = reinterpret_cast<const unsigned*>(a.ws + tile_of(w0 + wn * WN + i, w_tiles) * s_bytes) + lane;
#pragma unroll
  for (int j = 0; j < WT; ++j)
    xs_at[j] = reinterpret_cast<const unsigned*>(a.xs + tile_of(x0 + wt * WT + j, x_tiles) * s_bytes) + lane;
  f32x4 acc[WN][WT];
#pragma unroll
  for (int i = 0; i < WN; ++i)
#pragma unroll
    for (int j = 0; j < WT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  u32x4 next[kLoads];
  unsigned ws[WN], xs[WT], ws_next[WN], xs_next[WT];
  auto fetch = [&](int step) {
#pragma unroll
    for (int l = 0; l < kLoads; ++l)
      if (kPieces % kWaves == 0 || wave + l * kWaves < kPieces) next[l] = from[l][static_cast<int64_t>(step) * pace[l]];
  };
  auto place = [&](int b) {
#pragma unroll
    for (int l = 0; l < kLoads; ++l)
      if (kPieces % kWaves == 0 || wave + l * kWaves < kPieces) buffer[b][(wave + l * kWaves) * 64 + lane] = next[l];
  };
  auto fetch_scales = [&](int sp) {
#pragma unroll
    for (int i = 0; i < WN; ++i) ws_next[i] = ws_at[i][sp * 64];
#pragma unroll
    for (int j = 0; j < WT; ++j) xs_next[j] = xs_at[j][sp * 64];
  };
  fetch(0);
  fetch_scales(0);
  place(0);
  __syncthreads();
  auto one = [&](auto step_in, int step) {
    constexpr int STEP = decltype(step_in)::value;
    if (step >= steps) return;
    if (step + 1 < steps) fetch(step + 1);
    if constexpr (STEP == 0) {
#pragma unroll
      for (int i = 0; i < WN; ++i) ws[i] = ws_next[i];
#pragma unroll
      for (int j = 0; j < WT; ++j) xs[j] = xs_next[j];
      if (step + 4 < steps) fetch_scales(step / 4 + 1);
    }
    const u32x4* const held = buffer[STEP & 1] + lane;
    Operand<MX_E2M1> w[WN];
    Operand<FMT> x[WT];
#pragma unroll
    for (int i = 0; i < WN; ++i) w[i].q[0] = held[(wn * WN + i) * 64];
#pragma unroll
    for (int j = 0; j < WT; ++j)
#pragma unroll
      for (int h = 0; h < kParts; ++h) x[j].q[h] = held[(kW + (wt * WT + j) * kParts + h) * 64];
    mma_step<FMT, STEP>(acc, w, ws, x, xs);
    if (step + 1 < steps) place((STEP + 1) & 1);
    __syncthreads();
  };
  for (int sp = 0; sp < supers; ++sp) {
    one(std::integral_constant<int, 0>(), sp * 4);
    one(std::integral_constant<int, 1>(), sp * 4 + 1);
    one(std::integral_constant<int, 2>(), sp * 4 + 2);
    one(std::integral_constant<int, 3>(), sp * 4 + 3);
  }
#pragma unroll
  for (int i = 0; i < WN; ++i)
#pragma unroll
    for (int j = 0; j < WT; ++j)
      store4<TYPE>(a, (x0 + wt * WT + j) * 16 + (lane & 15), (w0 + wn * WN + i) * 16 + (lane >> 4) * 4, acc[i][j]);
}

// ---- launches --------------------------------------------------------------------------------------------------------

hipError_t run(void (*kern)(GemmArgs), dim3 grid, int threads, size_t lds, hipStream_t stream, const GemmArgs& a) {
  const Timing tm = timing_slot(KIND_PROBE);
  if (tm.on) {
    hipExtLaunchKernelGGL(kern, grid, dim3(threads), lds, stream, tm.start, tm.stop, 0, a);
  } else {
    hipLaunchKernelGGL(kern, grid, dim3(threads), lds, stream, a);
  }
  return hipGetLastError();
}

template <int FMT, int SRC, int TYPE, int RT, int CT>
hipError_t launch_stream(const GemmArgs& a, int waves, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>((mx_tiles(a.n) + RT - 1) / RT), static_cast<unsigned>((mx_tiles(a.t) + CT - 1) / CT));
  return run(mx_stream_kernel<FMT, SRC, TYPE, RT, CT>, grid, waves * 64, waves > 1 ? waves * RT * CT * 1024 : 0, stream, a);
}

template <int FMT, int TYPE, int WN, int WT, int GN, int GT>
hipError_t launch_tile(const GemmArgs& a, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>((mx_tiles(a.n) + GN * WN - 1) / (GN * WN)),
                  static_cast<unsigned>((mx_tiles(a.t) + GT * WT - 1) / (GT * WT)));
  return run(mx_tile_kernel<FMT, TYPE, WN, WT, GN, GT>, grid, GN * GT * 64, 0, stream, a);
}

int stream_waves(int64_t k) {
  const int64_t supers = mx_supers(k);
  return static_cast<int>(supers < 8 ? supers : 8);
}

template <int FMT, int TYPE>
hipError_t launch_rows(const MxGemmCall& c, const GemmArgs& a, hipStream_t stream) {
  if (c.src != nullptr) {
    const int waves = stream_waves(c.w.k);
    if (c.src_type == MX_F32) return launch_stream<FMT, MX_F32, TYPE, 1, 1>(a, waves, stream);
    if (c.src_type == MX_F16) return launch_stream<FMT, MX_F16, TYPE, 1, 1>(a, waves, stream);
    return launch_stream<FMT, MX_BF16, TYPE, 1, 1>(a, waves, stream);
  }
  const int waves = stream_waves(c.w.k);
  if (a.t <= 16) return launch_stream<FMT, -1, TYPE, 1, 1>(a, waves, stream);
  if (a.t <= 32) return launch_stream<FMT, -1, TYPE, 1, 2>(a, waves, stream);
  if (a.t <= 64) return launch_stream<FMT, -1, TYPE, 1, 4>(a, waves, stream);
  return launch_tile<FMT, TYPE, 4, 4, 2, 2>(a, stream);
}

template <int FMT>
hipError_t launch_format(const MxGemmCall& c, const GemmArgs& a, hipStream_t stream) {
  if (c.type == MX_F32) return launch_rows<FMT, MX_F32>(c, a, stream);
  if (c.type == MX_F16) return launch_rows<FMT, MX_F16>(c, a, stream);
  return launch_rows<FMT, MX_BF16>(c, a, stream);
}

}  // namespace

hipError_t launch_mx_gemm(const MxGemmCall& c, hipStream_t stream) {
  GemmArgs a;
  a.w = c.w.codes;
  a.ws = c.w.scales;
  a.x = c.src != nullptr ? static_cast<const uint8_t*>(c.src) : c.x.codes;
  a.xs = c.x.scales;
  a.x_stride = c.src_stride;
  a.n = c.w.rows;
  a.t = c.x.rows;
  a.k = static_cast<int>(c.w.k);
  a.y = c.y;
  a.y_stride = c.stride;
  return c.x.fmt == MX_E2M1 ? launch_format<MX_E2M1>(c, a, stream) : launch_format<MX_E4M3>(c, a, stream);
}

}  // namespace komp
