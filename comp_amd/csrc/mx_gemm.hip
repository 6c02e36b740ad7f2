// Products of microscaled rows: Y [T][N] = X W^T, W in e2m1, X in e2m1 or e4m3 or quantized on the way (layout: mx_layout.h).
//
// The weights are the matrix instruction's A operand and the activations its B operand, so a lane's four results are four
// consecutive outputs of one row of X.  X in e2m1: v_mfma_scale_f32_16x16x128_f8f6f4 takes codes and scale bytes as they lie in
// memory; a product of two e2m1 elements has at most four bits, and its sums are f32's.  X in e4m3: that instruction aligns the
// products of eight consecutive elements and drops what lies 14 binades and more below the group's largest (measured: 256 - 256 + 2^-5 is
// kept, + 2^-6 is not), which is not a 32-bit sum.  So both operands become bf16, scale included, which is exact (four bits at most, and bf16's exponents
// are f32's, subnormals included; only elements of X with scale bytes 0 to 2 lie between bf16's multiples of 2^-133, and values past
// f32's largest are infinite), and v_mfma_f32_16x16x32_bf16 adds them in f32.  (The scaled instruction
// would save the conversions and half the matrix cores' time; on random codes its results were off by 2.7 times what f32 sums and
// the rounding to bf16 allow.)
//
// Three kernels: one column tile of X (decode steps), tiles straight from memory (batches), tiles through shared memory (prompts).
// Figures: one MI355X, 6.9 TB/s read, 1.22 PFLOP/s in an 8192^3 bf16 library product.
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
  int type;                // of y
  int x_type;              // of x, quantized on the way
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
__device__ __forceinline__ void store4_as(const GemmArgs& a, int64_t t, int64_t n, f32x4 v) {
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
__device__ __forceinline__ void store4(const GemmArgs& a, int64_t t, int64_t n, f32x4 v) {
  if (t >= a.t || n >= a.n) return;
  if (a.type == MX_F32) store4_as<MX_F32>(a, t, n, v);
  else if (a.type == MX_F16) store4_as<MX_F16>(a, t, n, v);
  else store4_as<MX_BF16>(a, t, n, v);
}

// ---- one column tile of X --------------------------------------------------------------------------------------------

// X's operands of a four-step piece, ready for mma_piece: as they are (e2m1; e4m3 in eight registers a step), or in bf16.
template <int FMT, bool WIDE>
struct PieceX {
  Operand<FMT> x[4];
  unsigned scales;
};
template <>
struct PieceX<MX_E4M3, true> {
  bf16x8 b[4][4];
};

struct PieceW {
  Operand<MX_E2M1> w[4];
  unsigned scales;
};

// acc += a piece's products.  A step behind K's end has zero codes in X (the codes of W are the last step's again).
template <int FMT, bool WIDE>
__device__ __forceinline__ void mma_piece(f32x4& acc, const PieceW& w, const PieceX<FMT, WIDE>& x) {
  f32x4 out[1][1] = {{acc}};
  if constexpr (FMT == MX_E4M3 && WIDE) {
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const float scale = scale_of(w.scales, s);
#pragma unroll
      for (int p = 0; p < 4; ++p)
        out[0][0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bf16_part(w.w[s], p, scale), x.b[s][p], out[0][0], 0, 0, 0);
    }
  } else {
    auto step = [&](auto at) {
      constexpr int S = decltype(at)::value;
      const Operand<MX_E2M1> ws[1] = {w.w[S]};
      const Operand<FMT> xs[1] = {x.x[S]};
      const unsigned w_scales[1] = {w.scales}, x_scales[1] = {x.scales};
      mma_step<FMT, S>(out, ws, w_scales, xs, x_scales);
    };
    step(std::integral_constant<int, 0>());
    step(std::integral_constant<int, 1>());
    step(std::integral_constant<int, 2>());
    step(std::integral_constant<int, 3>());
  }
  acc = out[0][0];
}

// A wave's piece of the rows of X into shared memory: codes by rows, scales as the operands' dwords.  As many rows' loads are on their
// way together as the registers beside W's hold.
template <int FMT, int TYPE, int P>
__device__ __forceinline__ void quantize_rows(const GemmArgs& a, int sp, bool in, int lane, uint8_t* codes, uint8_t* scales, int column) {
  constexpr int kAtOnce = P > 1 ? 2 : TYPE == MX_F32 || FMT == MX_E4M3 ? 4 : 8;
  typedef typename MxElement<TYPE>::type T;
  typedef T vec __attribute__((ext_vector_type(8), aligned(sizeof(T))));
  const int count = static_cast<int>(a.t);
  const T* const from = reinterpret_cast<const T*>(a.x) + sp * 512 + lane * 8;
  for (int t0 = 0; t0 < count; t0 += kAtOnce) {
    vec raw[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
#pragma unroll
      for (int e = 0; e < 8; ++e) raw[i][e] = static_cast<T>(0.f);
      if (in && t0 + i < count) raw[i] = *reinterpret_cast<const vec*>(from + (t0 + i) * a.x_stride);
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int t = t0 + i;
      if (t >= count) break;
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = static_cast<float>(raw[i][e]);
      unsigned most = mx_most(v);
      most = umax(most, static_cast<unsigned>(dpp_i<KOMP_DPP_XOR1>(static_cast<int>(most))));
      most = umax(most, static_cast<unsigned>(dpp_i<KOMP_DPP_XOR2>(static_cast<int>(most))));
      const unsigned scale = mx_scale<FMT>(most);
      unsigned c[FMT == MX_E2M1 ? 1 : 2];
      mx_codes8<FMT>(v, scale, c);
      if constexpr (FMT == MX_E2M1) *reinterpret_cast<unsigned*>(codes + t * column + lane * 4) = c[0];
      else *reinterpret_cast<u32x2*>(codes + t * column + lane * 8) = u32x2{c[0], c[1]};
      // block 4 s + g of the piece: byte s of group g's dword
      if ((lane & 3) == 0) scales[(((lane >> 2) & 3) * 16 + t) * 4 + (lane >> 4)] = static_cast<uint8_t>(scale);
    }
  }
}

// Up to 16 rows of X.  A workgroup keeps X in registers, each wave P pieces of K, and walks over row tiles of W, whose codes
// it loads D pieces ahead; its waves join in shared memory, in their order.  FLOATS: the rows are quantized on the way, by each
// wave its own pieces, eight elements a lane, through shared memory into the operands' order.
//
// Bound by W's bytes where there are many: 128256 x 4096, one bf16 row to e4m3, in 44.7 us (6.3 TB/s; with W's loads through the
// caches 48.9, quantizing X again for every row tile 182), 28672 x 4096, five rows to e2m1, in 13.0 us cold.  Small products are a chain of
// latencies: 6912 x 2560 and one f32 row in 6.0 us in a graph, of which reading 9.4 MB is 1.4.  X as bf16 operands in registers costs
// e4m3 64 conversions a piece of W and none of X; from 16 pieces on (K above 8192) a wave holds four pieces, as codes.  D = 2: one
// piece on its way beside the one in use; with three the registers of P = 1 (128 for 16 waves) spill.
template <int FMT, bool FLOATS, int P, int D>
__global__ __launch_bounds__(P == 1 ? 1024 : 512) void mx_step_kernel(const GemmArgs a) {
  constexpr bool kWide = P == 1;
  constexpr int kTiles = D > P ? D / P : 1;                   // row tiles a turn of the loop
  constexpr int kColumn = (FMT == MX_E2M1 ? 256 : 512) + 16;  // bytes of a column's piece, apart in the banks
  extern __shared__ f32x4 shared[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const int steps = static_cast<int>(mx_steps(a.k)), supers = static_cast<int>(mx_supers(a.k));
  const int tiles = static_cast<int>(mx_tiles(a.n)), pace = gridDim.x;
  const int64_t w_bytes = mx_code_bytes(a.k, MX_E2M1), s_bytes = mx_scale_bytes(a.k);
  const int column = lane & 15, group = lane >> 4;
  PieceW w[D];
  auto fetch = [&](PieceW& into, int tile, int p) {
    const int sp = wave + waves * p;
    if (tile >= tiles || sp >= supers) return;
    into.scales = reinterpret_cast<const unsigned*>(a.ws + tile * s_bytes)[sp * 64 + lane];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int step = sp * 4 + s < steps ? sp * 4 + s : steps - 1;
      into.w[s].q[0] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(a.w + tile * w_bytes) + step * 64 + lane);
    }
  };
#pragma unroll
  for (int d = 0; d < D; ++d) fetch(w[d], blockIdx.x + d / P * pace, d % P);
  PieceX<FMT, kWide> x[P];
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const int sp = wave + waves * p;
    Operand<FMT> q[4];
    unsigned scales = 0;
    if (sp < supers) {
      if constexpr (FLOATS) {
        uint8_t* const mine = reinterpret_cast<uint8_t*>(shared) + wave * (static_cast<int>(a.t) * kColumn + 256);
        uint8_t* const mine_scales = mine + a.t * kColumn;
        const bool in = (sp * 16 + (lane >> 2)) * 32 < a.k;
        if (a.x_type == MX_F32) quantize_rows<FMT, MX_F32, P>(a, sp, in, lane, mine, mine_scales, kColumn);
        else if (a.x_type == MX_F16) quantize_rows<FMT, MX_F16, P>(a, sp, in, lane, mine, mine_scales, kColumn);
        else quantize_rows<FMT, MX_BF16, P>(a, sp, in, lane, mine, mine_scales, kColumn);
        // lanes read what others of their wave wrote
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if (column < a.t) {
          scales = reinterpret_cast<const unsigned*>(mine_scales)[lane];
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            const u32x4* const from = reinterpret_cast<const u32x4*>(mine + column * kColumn) + (s * 4 + group) * (FMT == MX_E2M1 ? 1 : 2);
            q[s].q[0] = from[0];
            if constexpr (FMT == MX_E4M3) q[s].q[1] = from[1];
          }
        }
      } else {
        scales = reinterpret_cast<const unsigned*>(a.xs)[sp * 64 + lane];
        constexpr int parts = FMT == MX_E2M1 ? 1 : 2;
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
          for (int h = 0; h < parts; ++h) {
            const int step = sp * 4 + s < steps ? sp * 4 + s : steps - 1;
            q[s].q[h] = reinterpret_cast<const u32x4*>(a.x)[(step * parts + h) * 64 + lane];
          }
      }
    }
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const bool in = column < a.t && sp * 4 + s < steps;
#pragma unroll
      for (int h = 0; h < (FMT == MX_E2M1 ? 1 : 2); ++h) q[s].q[h] = in ? q[s].q[h] : u32x4{0, 0, 0, 0};
      if (!in) scales &= ~(255u << (8 * s));
    }
    if constexpr (FMT == MX_E4M3 && kWide) {
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int j = 0; j < 4; ++j) x[p].b[s][j] = bf16_part(q[s], j, scale_of(scales, s));
    } else {
#pragma unroll
      for (int s = 0; s < 4; ++s) x[p].x[s] = q[s];
      x[p].scales = scales;
    }
  }
  if constexpr (FLOATS) __syncthreads();  // the waves' places are the join's from here on
  int turn = 0;
  for (int base = blockIdx.x; base < tiles; base += kTiles * pace) {
#pragma unroll
    for (int u = 0; u < kTiles; ++u) {
      const int tile = base + u * pace;
      if (tile >= tiles) break;
      f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int p = 0; p < P; ++p) {
        // (opaque scales: nothing made from x is kept over the tiles, which would not fit)
        if constexpr (!(FMT == MX_E4M3 && kWide)) asm volatile("" : "+v"(x[p].scales));
        const int item = u * P + p;  // of this turn; D items on, its place is free again
        if (wave + waves * p < supers) mma_piece<FMT, kWide>(acc, w[item % D], x[p]);
        fetch(w[item % D], base + (item + D) / P * pace, (item + D) % P);
      }
      const int64_t n = static_cast<int64_t>(tile) * 16 + group * 4;
      if (waves == 1) {
        store4(a, column, n, acc);
        continue;
      }
      f32x4* const join = shared + (turn & 1) * waves * 64 + lane;
      if (column < a.t) join[wave * 64] = acc;
      __syncthreads();
      if (wave == turn % waves && column < a.t) {
        f32x4 sum = join[0];
        for (int v = 1; v < waves; ++v) sum += join[v * 64];
        store4(a, column, n, sum);
      }
      ++turn;
    }
  }
}

// ---- few rows of X ---------------------------------------------------------------------------------------------------

// Operands come straight from memory: a workgroup has RT row tiles of W and CT tiles of X, its waves take four-step pieces of
// K in turn and join in shared memory, in the waves' order.  SRC: the type of the rows that are quantized on the way (each wave
// its own pieces; rows of more than 16384 elements, which mx_step_kernel cannot hold), -1: X is quantized already.
//
// For batches, whose tiles are too few for the device unless a tile is small and K is shared out inside the workgroup.  Bound by
// latency: 64 x 4096 x 14336 takes 15.9 us with cold weights, in e2m1 11.8, at one wave a SIMD, of whose time the vector instructions are
// 25% and the matrix cores 16%; 100 x 4096 x 4096 8.3 us.  Through wide weights the caches count too (each operand is read by N / (16 RT) or
// T / (16 CT) workgroups): 32 x 131072 x 4096 in 71 us, in e2m1 59 (4.1 and 5.0 TB/s).  (K shared out over workgroups, tiles of 128 x 64 through shared
// memory and the sums joined by a second launch: 19.0 and 14.4 us; two pieces of a wave's on their way: 18.4 and 12.6 us.)
template <int FMT, int SRC, int RT, int CT, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void mx_stream_kernel(const GemmArgs a) {
  constexpr int kParts = FMT == MX_E2M1 ? 1 : 2;
  extern __shared__ f32x4 join[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
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
  Operand<MX_E2M1> w[4][RT];
  Operand<FMT> x[4][CT];
  unsigned ws[RT], xs[CT], ws_next[RT], xs_next[CT];
  // step `s` of piece `sp`; a step past the last one is the last one again, and not used
  auto fetch = [&](int sp, int s) {
    const int step = sp * 4 + s < steps ? sp * 4 + s : steps - 1;
#pragma unroll
    for (int i = 0; i < RT; ++i)
      w[s][i].q[0] = reinterpret_cast<const u32x4*>(a.w + tile_of(w0 + i, w_tiles) * w_bytes)[step * 64 + lane];
    if constexpr (SRC < 0) {
#pragma unroll
      for (int j = 0; j < CT; ++j)
#pragma unroll
        for (int h = 0; h < kParts; ++h)
          x[s][j].q[h] = reinterpret_cast<const u32x4*>(a.x + tile_of(x0 + j, x_tiles) * x_bytes)[(step * kParts + h) * 64 + lane];
    }
  };
  auto fetch_scales = [&](int sp) {
#pragma unroll
    for (int i = 0; i < RT; ++i) ws_next[i] = reinterpret_cast<const unsigned*>(a.ws + tile_of(w0 + i, w_tiles) * s_bytes)[sp * 64 + lane];
    if constexpr (SRC < 0) {
#pragma unroll
      for (int j = 0; j < CT; ++j)
        xs_next[j] = reinterpret_cast<const unsigned*>(a.xs + tile_of(x0 + j, x_tiles) * s_bytes)[sp * 64 + lane];
    }
  };
  if (wave < supers) {
    fetch_scales(wave);
#pragma unroll
    for (int s = 0; s < 4; ++s) fetch(wave, s);
  }
  for (int sp = wave; sp < supers; sp += waves) {
#pragma unroll
    for (int i = 0; i < RT; ++i) ws[i] = ws_next[i];
    if constexpr (SRC < 0) {
#pragma unroll
      for (int j = 0; j < CT; ++j) xs[j] = xs_next[j];
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
    // a step's registers take the wave's next piece as soon as they are used
    const int next = sp + waves;
    const bool more = next < supers;
    if (more) fetch_scales(next);
    auto one = [&](auto at) {
      constexpr int STEP = decltype(at)::value;
      if (sp * 4 + STEP < steps) mma_step<FMT, STEP>(acc, w[STEP], ws, x[STEP], xs);
      if (more) fetch(next, STEP);
    };
    one(std::integral_constant<int, 0>());
    one(std::integral_constant<int, 1>());
    one(std::integral_constant<int, 2>());
    one(std::integral_constant<int, 3>());
  }
  auto put = [&](int i, int j, int l, f32x4 v) {
    store4(a, (x0 + j) * 16 + (l & 15), (w0 + i) * 16 + (l >> 4) * 4, v);
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

// 1 KB (16 bytes a lane) or 256 bytes (4 a lane) from memory straight into shared memory at `place`, lane after lane.  The
// compiler does not see these loads: dma_wait waits for them, and the barrier behind it for the other waves'.
__device__ __forceinline__ void dma16(unsigned place, const uint8_t* base, unsigned offset) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(place), "v"(offset), "s"(base) : "m0", "memory");
}
__device__ __forceinline__ void dma4(unsigned place, const uint8_t* base, unsigned offset) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"(place), "v"(offset), "s"(base) : "m0", "memory");
}
// until at most N of this wave's loads are on their way, and its reads of shared memory are done
template <int N>
__device__ __forceinline__ void dma_wait() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
}

// Row tiles of W in a workgroup, column tiles of X, and the loads of a wave a step.
template <int FMT, int WN, int WT, int GN, int GT>
struct TileShape {
  static constexpr int kParts = FMT == MX_E2M1 ? 1 : 2, kWaves = GN * GT;
  static constexpr int kW = GN * WN, kX = GT * WT, kPieces = kW + kX * kParts;  // 1 KB each
  static constexpr int kLoads = (kPieces + kWaves - 1) / kWaves;
  static constexpr int kScaleLoads = (kW + kX + 4 * kWaves - 1) / (4 * kWaves);  // of 256 bytes
  static constexpr int kStage = kLoads * kWaves * 1024, kScales = kScaleLoads * 4 * kWaves * 256;
};

// Places in shared memory for a step's codes.  (Scales are read before the next but one's loads: four at most.)
constexpr int kPlaces = 3;

// A workgroup of GN x GT waves has GN * WN row tiles of W and GT * WT of X.  A step's codes lie in one of kPlaces places in shared memory,
// loaded kPlaces - 1 steps ahead; the scales of the next four steps are loaded beside them, a quarter a step, into one of two places.
//
// Bound by the matrix cores, at the clock that their power leaves: 8192 x 14336 x 4096 in 632 us in e4m3 (1.52 PFLOP/s; the matrix cores
// busy 66% of the time, conversions 46% of the issue slots) and 267 us in e2m1 (3.6 PFLOP/s, of which storing Y is some 55 us).  256 x
// 256 tiles of eight waves, 128 x 64 each (a step reads 12 operands for 32 products); two or three places measured the same, loads by way
// of registers and one step ahead 758 us.
template <int FMT, int WN, int WT, int GN, int GT>
__global__ __launch_bounds__(GN* GT * 64) void mx_tile_kernel(const GemmArgs a) {
  using S = TileShape<FMT, WN, WT, GN, GT>;
  extern __shared__ f32x4 shared[];
  uint8_t* const lds = reinterpret_cast<uint8_t*>(shared);
  uint8_t* const lds_scales = lds + kPlaces * S::kStage;
  const unsigned place0 = static_cast<unsigned>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) uint8_t*)lds));
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wn = wave % GN, wt = wave / GN;
  const int supers = static_cast<int>(mx_supers(a.k));
  const int last = static_cast<int>(mx_steps(a.k)) - 1;
  const int64_t w_tiles = mx_tiles(a.n), x_tiles = mx_tiles(a.t);
  const int64_t w0 = static_cast<int64_t>(blockIdx.x) * S::kW, x0 = static_cast<int64_t>(blockIdx.y) * S::kX;
  const int64_t w_bytes = mx_code_bytes(a.k, MX_E2M1), x_bytes = mx_code_bytes(a.k, FMT), s_bytes = mx_scale_bytes(a.k);
  // a tile past the last one is read again as the last one, and not stored
  auto tile_of = [](int64_t tile, int64_t tiles) { return tile < tiles ? tile : tiles - 1; };
  const uint8_t *from[S::kLoads], *from_scales[4][S::kScaleLoads];
  unsigned pace[S::kLoads];
#pragma unroll
  for (int l = 0; l < S::kLoads; ++l) {
    const int p = wave + l * S::kWaves;
    if (p < S::kW) {
      from[l] = a.w + tile_of(w0 + p, w_tiles) * w_bytes;
      pace[l] = 1024;
    } else {  // (past the last piece: the last one again)
      const int c = p < S::kPieces ? p - S::kW : S::kX * S::kParts - 1;
      from[l] = a.x + tile_of(x0 + c / S::kParts, x_tiles) * x_bytes + c % S::kParts * 1024;
      pace[l] = 1024 * S::kParts;
    }
  }
#pragma unroll
  for (int q = 0; q < 4; ++q)
#pragma unroll
    for (int l = 0; l < S::kScaleLoads; ++l) {
      const int p = (q * S::kScaleLoads + l) * S::kWaves + wave;
      const int c = p < S::kW + S::kX ? p : S::kW + S::kX - 1;
      from_scales[q][l] = c < S::kW ? a.ws + tile_of(w0 + c, w_tiles) * s_bytes : a.xs + tile_of(x0 + c - S::kW, x_tiles) * s_bytes;
    }
  // the loads of a step, and a quarter of the next piece's scales; steps and pieces past the end are the last one again
  auto fetch_scales = [&](int q, int sp) {
    const unsigned at = place0 + kPlaces * S::kStage + (sp & 1) * S::kScales;
    const int64_t offset = static_cast<int64_t>(sp < supers ? sp : supers - 1) * 256;
#pragma unroll
    for (int l = 0; l < S::kScaleLoads; ++l)
      dma4(at + ((q * S::kScaleLoads + l) * S::kWaves + wave) * 256, from_scales[q][l] + offset, lane * 4);
  };
  auto fetch = [&](int step, int slot) {
    const int64_t at = step < last ? step : last;
#pragma unroll
    for (int l = 0; l < S::kLoads; ++l)
      dma16(place0 + slot * S::kStage + (wave + l * S::kWaves) * 1024, from[l] + at * pace[l], lane * 16);
  };
  f32x4 acc[WN][WT];
#pragma unroll
  for (int i = 0; i < WN; ++i)
#pragma unroll
    for (int j = 0; j < WT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int q = 0; q < 4; ++q) fetch_scales(q, 0);
#pragma unroll
  for (int s = 0; s < kPlaces - 1; ++s) {
    fetch(s, s);
    fetch_scales(s, 1);
  }
  unsigned ws[WN], xs[WT];
  int slot = 0;
  auto one = [&](auto step_in, int sp) {
    constexpr int STEP = decltype(step_in)::value;
    const int step = sp * 4 + STEP;
    if (step > last) return;
    dma_wait<(kPlaces - 2) * (S::kLoads + S::kScaleLoads)>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");  // (no read of shared memory moves up)
    if constexpr (STEP == 0) {
      const unsigned* const held = reinterpret_cast<const unsigned*>(lds_scales + (sp & 1) * S::kScales) + lane;
#pragma unroll
      for (int i = 0; i < WN; ++i) ws[i] = held[(wn * WN + i) * 64];
#pragma unroll
      for (int j = 0; j < WT; ++j) xs[j] = held[(S::kW + wt * WT + j) * 64];
    }
    const u32x4* const held = reinterpret_cast<const u32x4*>(lds + slot * S::kStage) + lane;
    Operand<MX_E2M1> w[WN];
    Operand<FMT> x[WT];
#pragma unroll
    for (int i = 0; i < WN; ++i) w[i].q[0] = held[(wn * WN + i) * 64];
#pragma unroll
    for (int j = 0; j < WT; ++j)
#pragma unroll
      for (int h = 0; h < S::kParts; ++h) x[j].q[h] = held[(S::kW + (wt * WT + j) * S::kParts + h) * 64];
    // the next loads, while the reads are on their way: every wave is done with the place of the step before
    const int free_slot = slot == 0 ? kPlaces - 1 : slot - 1;
    constexpr int AHEAD = STEP + kPlaces - 1;
    fetch(step + kPlaces - 1, free_slot);
    fetch_scales(AHEAD & 3, sp + AHEAD / 4 + 1);
    mma_step<FMT, STEP>(acc, w, ws, x, xs);
    slot = slot == kPlaces - 1 ? 0 : slot + 1;
  };
  for (int sp = 0; sp < supers; ++sp) {
    one(std::integral_constant<int, 0>(), sp);
    one(std::integral_constant<int, 1>(), sp);
    one(std::integral_constant<int, 2>(), sp);
    one(std::integral_constant<int, 3>(), sp);
  }
  dma_wait<0>();  // no load is on its way into this workgroup's shared memory when it ends
#pragma unroll
  for (int i = 0; i < WN; ++i)
#pragma unroll
    for (int j = 0; j < WT; ++j)
      store4(a, (x0 + wt * WT + j) * 16 + (lane & 15), (w0 + wn * WN + i) * 16 + (lane >> 4) * 4, acc[i][j]);
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

template <int FMT, int SRC, int RT, int CT, int WAVES>
hipError_t launch_stream(const GemmArgs& a, hipStream_t stream) {
  static std::atomic<unsigned> limit[kMaxDevices];
  const int waves = static_cast<int>(mx_supers(a.k) < WAVES ? mx_supers(a.k) : WAVES);
  const dim3 grid(static_cast<unsigned>((mx_tiles(a.n) + RT - 1) / RT), static_cast<unsigned>((mx_tiles(a.t) + CT - 1) / CT));
  const size_t lds = waves > 1 ? waves * RT * CT * 1024 : 0;
  const auto kern = mx_stream_kernel<FMT, SRC, RT, CT, WAVES>;
  const hipError_t e = allow_dynamic_lds(reinterpret_cast<const void*>(kern), lds, limit);
  return e != hipSuccess ? e : run(kern, grid, waves * 64, lds, stream, a);
}

template <int FMT, int WN, int WT, int GN, int GT>
hipError_t launch_tile(const GemmArgs& a, hipStream_t stream) {
  using S = TileShape<FMT, WN, WT, GN, GT>;
  static std::atomic<unsigned> limit[kMaxDevices];
  const dim3 grid(static_cast<unsigned>((mx_tiles(a.n) + S::kW - 1) / S::kW), static_cast<unsigned>((mx_tiles(a.t) + S::kX - 1) / S::kX));
  const size_t lds = kPlaces * S::kStage + 2 * S::kScales;
  const auto kern = mx_tile_kernel<FMT, WN, WT, GN, GT>;
  const hipError_t e = allow_dynamic_lds(reinterpret_cast<const void*>(kern), lds, limit);
  return e != hipSuccess ? e : run(kern, grid, GN * GT * 64, lds, stream, a);
}

template <int FMT, bool FLOATS, int P, int D>
hipError_t launch_step(const GemmArgs& a, hipStream_t stream) {
  static std::atomic<unsigned> limit[kMaxDevices];
  const int waves = static_cast<int>((mx_supers(a.k) + P - 1) / P);
  const int column = (FMT == MX_E2M1 ? 256 : 512) + 16;
  const size_t place = FLOATS ? waves * (a.t * column + 256) : 0, join = waves > 1 ? 2 * waves * 1024 : 0;
  const size_t lds = place > join ? place : join;
  // as many workgroups as make 16 waves a CU, each with several row tiles; 8 waves where each workgroup quantizes many rows (16 rows of
  // 4096, 14336 of W: 15.8 us against 18.9; one row: the same)
  const int64_t tiles = mx_tiles(a.n), most = static_cast<int64_t>(device_cu_count()) * (FLOATS && a.t > 8 ? (waves < 8 ? 8 / waves : 1) : 16 / waves);
  const auto kern = mx_step_kernel<FMT, FLOATS, P, D>;
  const hipError_t e = allow_dynamic_lds(reinterpret_cast<const void*>(kern), lds, limit);
  if (e != hipSuccess) return e;
  return run(kern, dim3(static_cast<unsigned>(tiles < most ? tiles : most)), waves * 64, lds, stream, a);
}

template <int FMT>
hipError_t launch_format(const MxGemmCall& c, const GemmArgs& a, hipStream_t stream) {
  const bool floats = c.src != nullptr;
  const MxGemmPlan p = mx_gemm_plan(a.t, a.n, a.k);
  if (p.kernel == MX_STEP) {
    if (mx_supers(a.k) <= 16) return floats ? launch_step<FMT, true, 1, 2>(a, stream) : launch_step<FMT, false, 1, 2>(a, stream);
    return floats ? launch_step<FMT, true, 4, 2>(a, stream) : launch_step<FMT, false, 4, 2>(a, stream);
  }
  if (p.kernel == MX_TILE) {
    if (p.row_tiles == 16) return launch_tile<FMT, 8, 4, 2, 4>(a, stream);
    return launch_tile<FMT, 4, 4, 2, 2>(a, stream);
  }
  if (p.col_tiles == 2) {
    if (p.row_tiles == 4) return launch_stream<FMT, -1, 4, 2, 8>(a, stream);
    if (p.row_tiles == 2) return launch_stream<FMT, -1, 2, 2, 8>(a, stream);
    return launch_stream<FMT, -1, 1, 2, 8>(a, stream);
  }
  if (!floats) return launch_stream<FMT, -1, 1, 1, 8>(a, stream);
  if (c.src_type == MX_F32) return launch_stream<FMT, MX_F32, 1, 1, 8>(a, stream);
  if (c.src_type == MX_F16) return launch_stream<FMT, MX_F16, 1, 1, 8>(a, stream);
  return launch_stream<FMT, MX_BF16, 1, 1, 8>(a, stream);
}

}  // namespace

MxGemmPlan mx_gemm_plan(int64_t t, int64_t n, int64_t k) {
  // (mx_step_kernel holds rows of up to 16384 elements)
  if (t <= 16) return mx_supers(k) <= 32 ? MxGemmPlan{MX_STEP, 1, 1} : MxGemmPlan{MX_STREAM, 1, 1};
  // The largest tiles that are enough for the device.  Both sides, us (T x N x K):
  //   256 x 256 tiles against 128 x 128: 8192 x 14336 x 4096 (1792 of 256 x 256) 647 and 698 in e4m3, 282 and 309 in e2m1; 2048 x 4096 x
  //     4096 (128) 87 and 55
  //   128 x 128 against 64 x 32: 256 x 14336 x 4096 (224 of 128 x 128) 17.5 and 31.5 in e2m1; 256 x 4096 x 14336 (64) 99 and 38 in e4m3
  //   64 x 32 against 32 x 32: 100 x 4096 x 4096 (256 of 64 x 32) 9.0 and 10.0; 64 x 4096 x 14336 (128) 21.0 and 16.1
  //   32 x 32 against 16 x 32: 64 x 4096 x 14336 (256 of 32 x 32) 16.1 and 20.8; 32 x 4096 x 14336 (128) 16.7 and 14.2
  //
  // A group that ends past T or N takes its full time for what it throws away, so a tile must also be mostly filled.  Both sides, us:
  //   256 x 256 covers at most 5/4 of what 128 x 128 tiles cover: with 131072 of W and K = 4096, 17 rows of X (twice as much) 177 and 108 in
  //     e4m3, 85 and 58 in e2m1; 300 rows (4/3) 376 and 318, 178 and 179; 640 rows (6/5) 577 and 547, 281 and 304; 144 rows (as much) 187 and 211
  //   128 x 128 against 64 x 32 where one of these holds all rows of X or of W: 32 x 28672 x 4096 30.7 and 19.7 in e4m3, 17.6 and 16.2 in
  //     e2m1, 32 x 128256 x 4096 106 and 71, 57 and 58; 262144 x 64 x 1024 69 and 63, 40 and 29; past that, 33 x 131072 x 4096 110 and 127, 59 and
  //     105; 262144 x 80 x 1024 69 and 101, 41 and 53
  //   64 x 32 against 32 x 32 for W of 32 rows: 262144 x 32 x 1024 52 and 42 in e4m3, 24 and 23 in e2m1; 32 x 32 against 16 x 32 for 16
  //     rows: 8192 x 16 x 4096 5.4 and 4.8, 3.9 and 3.7
  const int64_t cus = device_cu_count(), n16 = mx_tiles(n), t16 = mx_tiles(t);
  auto groups = [&](int64_t rows, int64_t cols) { return ((n16 + rows - 1) / rows) * ((t16 + cols - 1) / cols); };
  if (groups(16, 16) >= 2 * cus && 16 * groups(16, 16) <= 5 * groups(8, 8)) return {MX_TILE, 16, 16};
  if (8 * groups(8, 8) >= 5 * cus && n16 > 4 && t16 > 2) return {MX_TILE, 8, 8};
  if (groups(4, 2) >= cus && n16 > 2) return {MX_STREAM, 4, 2};
  if (groups(2, 2) >= cus && n16 > 1) return {MX_STREAM, 2, 2};
  return {MX_STREAM, 1, 2};
}

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
  a.type = c.type;
  a.x_type = c.src_type;
  return c.x.fmt == MX_E2M1 ? launch_format<MX_E2M1>(c, a, stream) : launch_format<MX_E4M3>(c, a, stream);
}

}  // namespace komp
