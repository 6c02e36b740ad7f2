// The plan of an attention call over the quantized key/value cache, and the join of a sequence's splits.
#include <algorithm>

#include "kv_attend.h"

namespace komp {
namespace {

constexpr int kMaxSplits = 64;

AttendPlan plan_of(const KvAttendCall& c) {
  const int group = c.heads / c.cache.heads;
  const int64_t cols = c.max_queries * group;
  const int64_t units = static_cast<int64_t>(c.batch) * c.cache.heads;
  AttendPlan p;
  // The many-column kernel unpacks a key once for 256 columns rather than 16, but starts slower and fills a CU with one
  // workgroup.  8 sequences of 4096 keys, 8 kv heads of 128 channels, 4-bit, few and many, us: 48 columns bf16 35 and 62, f32
  // 46 and 59; 96 columns bf16 57 and 67, f16 61 and 72, f32 73 and 80; 128 columns bf16 68 and 69, f16 73 and 76, f32 88 and 84.
  p.many = cols > 96;
  const int wide = p.many ? many_cols(c.cache.dim, c.type) : 16;
  p.groups = std::max(1, static_cast<int>((cols + wide - 1) / wide));  // (none without query rows: such a call launches nothing)
  // Workgroups to fill the CUs (one of many columns each; of few three fit, and a fourth evens out what masks and short
  // sequences leave empty: 16 sequences of up to 8192 keys and 1-5 rows, f32, 56 us with 512 workgroups, 45 with 768, 37
  // with 1024, 39 with 1536; 8 of up to 3000 keys, 12 heads of 96 channels, f16, 18, 20, 20 and 20), twice that where there are
  // many sequences of unlike lengths (64 of up to 8192 keys, bf16: 100 us with 1024, 89 with 2048, 90 with 4096; 40 of up to
  // 3000, 20 heads over 5: 24 with each); and no split of less than two tiles a wave or two buffers.  Pieces of few
  // columns have the longest length's share of the splits, so that shorter sequences are cut into fewer, but enough
  // (`least`) to fill the CUs if all are that short.
  const int64_t fill = p.many ? 256 : 1024, aim = !p.many && units * p.groups >= 256 ? 2 * fill : fill;
  p.least = static_cast<int>((fill + units * p.groups - 1) / (units * p.groups));
  p.per = 1;
  const int64_t want = (aim + units * p.groups - 1) / (units * p.groups);
  const int64_t most = p.many ? c.max_length / 256 : (c.max_length + 31) / 32 / (2 * kAttendWaves);
  if (c.rows * c.heads > 1 << 22) {  // rows that no sequence holds, most likely: the join has a workgroup for each row and head
    p.splits = 1;
    return p;
  }
  p.splits = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({want, most, kMaxSplits})));
  p.least = std::min(p.least, p.splits);
  p.per = static_cast<int>(((c.max_length + 31) / 32 + p.splits - 1) / p.splits);
  return p;
}

// One workgroup a row and head: the splits' sums, brought to the largest of their references.  A wave takes every fourth
// split, D / 4 lanes a split; their sums meet in shared memory.
template <int D>
__global__ void __launch_bounds__(256) kv_attend_join_kernel(const AttendArgs a) {
  constexpr int LANES = D / 4, PAR = 64 / LANES;  // lanes a split, splits a wave at a time
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t n = a.rows * a.heads, at = blockIdx.x;
  float2 m = float2{-__builtin_inff(), 0.f};
  if (lane < a.splits) m = a.part_m[lane * n + at];
  const int part = lane / LANES, ch = lane - part * LANES;
  // every split's sums are loaded before its reference is known (kMaxSplits / 4 / PAR loads at most, all in flight)
  constexpr int MOST = kMaxSplits / 4 / PAR;
  f32x4 x[MOST];
#pragma unroll
  for (int i = 0; i < MOST; ++i) {
    const int s = (i * 4 + wave) * PAR + part;
    x[i] = part < PAR && s < a.splits ? *reinterpret_cast<const f32x4*>(a.part_o + (s * n + at) * D + ch * 4) : f32x4{0.f, 0.f, 0.f, 0.f};
  }
  float top = m.x;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
  const float f = m.x == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(m.x - top);
  const float l = group_sum(f * m.y, 64);
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < MOST; ++i) {
    const int s = (i * 4 + wave) * PAR + part;
    const float fs = __shfl(f, s & 63, 64), ms = __shfl(m.x, s & 63, 64);
    if (ms != -__builtin_inff()) o += fs * x[i];  // (a split that saw nothing has stored no sums)
  }
  __shared__ f32x4 sum[4][64];
  sum[wave][lane] = o;
  __syncthreads();
  if (threadIdx.x < LANES) {
    o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 4; ++w)
#pragma unroll
      for (int p = 0; p < PAR; ++p) o += sum[w][p * LANES + threadIdx.x];
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int64_t row = at / a.heads;
    const int head = static_cast<int>(at - row * a.heads);
    store_out(a.out, a.type, a.wide_out, row * a.out_stride_t + head * a.out_stride_h + ch * 4, o * inv);
    if (a.lse && lane == 0) a.lse[at] = l == 0.f ? -__builtin_inff() : (top + __log2f(l)) * (1.f / kLog2e);
  }
}

int64_t round256(int64_t v) { return (v + 255) / 256 * 256; }

}  // namespace

int64_t kv_attend_work_bytes(const KvAttendCall& c) {
  if (c.batch == 0 || c.rows == 0 || c.max_queries == 0) return 0;
  const AttendPlan p = plan_of(c);
  if (p.splits == 1) return 0;
  const int64_t n = p.splits * c.rows * c.heads;
  return round256(n * c.cache.dim * 4) + n * 8;
}

hipError_t launch_kv_attend(const KvAttendCall& c, hipStream_t stream) {
  const AttendPlan p = plan_of(c);
  AttendArgs a;
  a.c = c.cache;
  a.q = c.q;
  a.q_stride_t = c.q_stride_t;
  a.q_stride_h = c.q_stride_h;
  a.out = c.out;
  a.out_stride_t = c.out_stride_t;
  a.out_stride_h = c.out_stride_h;
  a.lse = c.lse;
  a.tables = c.tables;
  a.table_stride = c.table_stride;
  a.table_cols = c.table_cols;
  a.lengths = c.lengths;
  a.starts = c.starts;
  a.prefix = c.prefix;
  a.slopes = c.slopes;
  a.rows = c.rows;
  a.heads = c.heads;
  a.group = c.heads / c.cache.heads;
  a.type = c.type;
  a.window = c.window;
  a.scale = c.scale * kLog2e;
  a.cap = c.softcap;
  a.twice = c.softcap > 0.f ? std::min(2.f / c.softcap, 3.0e38f) : 0.f;  // (a number for the smallest caps too)
  const int size = c.type == KV_F32 ? 4 : 2;
  auto fits = [&](const void* p, int64_t st, int64_t sh, int bytes) {
    return reinterpret_cast<uintptr_t>(p) % bytes == 0 && st * size % bytes == 0 && sh * size % bytes == 0;
  };
  a.wide_q = fits(c.q, c.q_stride_t, c.q_stride_h, 16);
  a.wide_out = fits(c.out, c.out_stride_t, c.out_stride_h, 4 * size);
  a.splits = p.splits;
  a.least = p.least;
  a.per = p.per;
  a.groups = p.groups;
  a.part_o = static_cast<float*>(c.work);
  const int64_t n = p.splits * c.rows * c.heads;
  a.part_m = reinterpret_cast<float2*>(static_cast<char*>(c.work) + round256(n * c.cache.dim * 4));
  hipError_t e;
  if (c.cache.kf == KV_Q4_0) e = launch_attend_q4_q4(a, p, c.batch, stream);
  else if (c.cache.vf == KV_Q4_0) e = launch_attend_q8_q4(a, p, c.batch, stream);
  else e = launch_attend_q8_q8(a, p, c.batch, stream);
  if (e != hipSuccess || p.splits == 1) return e;
  const dim3 grid(static_cast<unsigned>(c.rows * c.heads));
  auto run = [&](auto kern) {
    const Timing tm = timing_slot(KIND_PROBE);
    if (tm.on) {
      hipExtLaunchKernelGGL(kern, grid, dim3(256), 0, stream, tm.start, tm.stop, 0, a);
    } else {
      hipLaunchKernelGGL(kern, grid, dim3(256), 0, stream, a);
    }
    return hipGetLastError();
  };
  switch (c.cache.dim) {
    case 64: return run(kv_attend_join_kernel<64>);
    case 96: return run(kv_attend_join_kernel<96>);
    case 128: return run(kv_attend_join_kernel<128>);
    default: return run(kv_attend_join_kernel<256>);
  }
}

}  // namespace komp
