// Attention over the quantized key/value cache for many columns, as a prompt has: the keys and values are unpacked once
// for all of a workgroup's columns (kv_attend.h has the mathematics and the columns' softmax).
//
// The waves of a workgroup have CT column tiles each and walk the same keys, which the workgroup unpacks into shared
// memory as the f16 operands that the waves then read (16 bytes a lane, in lane order: no bank conflicts).  Two buffers of
// KEYS keys, one barrier a buffer: while a wave computes with one, it unpacks its share of the next and has the codes
// after that in flight.
//
// f16 and f32 queries: the operands hold the codes, exact; the scales lie beside them and are used as in Columns::step.
// bf16 queries: the operands hold d * code, rounded to f16 after a power of two that brings the tile's largest scale to [1, 2)
// and that the scores' factor or the probabilities' exponent takes back.  2^-12 of a key or value is an eighth of what bf16
// keeps of the result, and saves the f32 products of the partial dots and of the probabilities, half of a column's
// instructions.  (Where the logarithms of the sums are asked for, in f32, keys stay exact: KV_VALUES_SCALED.)  A value block
// whose scale is no number is held as zeros then, and makes NaN of its channels in the columns that see it.  f16 holds a scale
// times that power whole down to 2^-14 of the largest (or at all, where the largest is below 2); where a tile has a smaller one,
// of keys that some column sees or not, the workgroup begins again with exact operands.
// Measured, 32 query heads over 8 of 128 channels, 4-bit: a prompt of 4096 tokens 268 us in bf16 (with the sums' logarithms
// 309, f16 354, f32 515), 600 TFLOP/s where every key is seen (f16 450, f32 283, twice the products), where a large library
// product reaches 1160: the vector unit is busy 43% of the time, the matrix unit 20%.
#pragma once

#include "kv_attend.h"

namespace komp {

// what of the operands is multiplied by its scales: nothing, values, values and keys
enum { KV_EXACT = 0, KV_VALUES_SCALED = 1, KV_ALL_SCALED = 2 };

template <int NB, int KF, int VF, int MODE, int SCALED>
struct Many {
  static constexpr bool V_SCALED = SCALED != KV_EXACT, K_SCALED = SCALED == KV_ALL_SCALED;
  static constexpr int BLOCKS = NB;
  // Exact keys, and values multiplied by their scales on their way, of 128 channels: more than 256 registers, and a kernel may not
  // spill.  Partial dots are held two blocks at a time then, and a lane's addresses are formed where they are used (which costs
  // the kernels that have the room some 5%).
  static constexpr bool TIGHT = SCALED == KV_VALUES_SCALED && NB == 4;
  static __device__ __forceinline__ int here(int lane) {
    if constexpr (TIGHT) asm volatile("" : "+v"(lane));
    return lane;
  }
  // two column tiles a wave halve the operand reads and the unpacking a column, where the registers (of two waves a SIMD)
  // hold their queries and sums: not f32 queries, in two parts, nor 256 channels
  static constexpr bool PAIR = NB <= 4 && MODE != KV_F32;
  static constexpr int CT = PAIR ? 2 : 1, WAVES = PAIR || NB == 8 ? 8 : 12, COLS = 16 * CT;
  static constexpr int HALVES = NB == 8 ? 2 : PAIR ? 4 : 3, KEYS = 32 * HALVES;  // (a "half" is 32 keys: two key tiles)
  static constexpr int KB = kv_kb(NB, KF), VB = kv_vb(NB, VF);
  static constexpr int KD = KB * kv_code_bytes(KF) / 16, VD = VB * kv_code_bytes(VF) / 8;  // code dwords of a lane's chunk
  static constexpr int MD = KD > VD ? KD : VD;
  static constexpr int KG = NB / KB, VG = NB / VB;                                         // chunks a 16- or 32-token tile
  static constexpr int KCHUNKS = KEYS / 16 * KG, VCHUNKS = HALVES * VG, CHUNKS = KCHUNKS + VCHUNKS;
  static constexpr int TURNS = (CHUNKS + WAVES - 1) / WAVES;  // chunks of one wave
  static constexpr int SW = (16 * NB + 63) / 64;              // dwords a lane of a half's scales, in a wave
  // the largest exponent fields of a tile: of the values' and the keys' scales, or of each half's values' scales (KV_EXACT)
  static constexpr int MOST = V_SCALED ? 2 : HALVES;
  using Cols = Columns<NB, KF, VF, MODE, CT, true>;

  struct Shared {
    f16x8 k[2][HALVES * 2 * NB][64];  // [16 tokens][block]
    f16x8 v[2][HALVES * NB * 2][64];  // [32 tokens][block][channels 0..15, 16..31]
    unsigned ks[2][K_SCALED ? 1 : HALVES][K_SCALED ? 1 : 16 * NB];
    unsigned vs[2][V_SCALED ? 1 : HALVES][V_SCALED ? 1 : 16 * NB];
    unsigned most[4][MOST];
    unsigned bad[4][V_SCALED ? 1 + HALVES * NB : 1];  // a tile's flags; which tokens of a half and block have a value scale
                                                    // that is no number
  };
  // flags: there are value scales that are no numbers; scales too far below the largest
  static constexpr unsigned SPOILT = 1, SCATTERED = 2;
  // a wave's chunks on their way from the cache to shared memory, and for the first waves the scales of a half
  struct Chunk {
    unsigned code[MD];
    unsigned scale[V_SCALED ? 4 * VB : 1];
  };
  Chunk chunk[TURNS];
  bool there[TURNS];
  unsigned ks[K_SCALED ? 1 : SW], vs[V_SCALED ? 1 : SW];

  static __device__ __forceinline__ int half_of(int c) { return c < KCHUNKS ? c / KG >> 1 : (c - KCHUNKS) / VG; }

  // `unit(half)`: where a half of the tile lies, -1 for nowhere
  template <typename F>
  __device__ __forceinline__ void load(const KvCache& cache, F&& unit, int wave, int lane) {
#pragma unroll
    for (int i = 0; i < TURNS; ++i) {
      const int c = i * WAVES + wave;
      const int64_t u = c < CHUNKS ? unit(half_of(c)) : -1;
      there[i] = u >= 0;
      if (!there[i]) continue;
      if constexpr (KD != VD) {  // (a length that depends on the kind would put the codes into scratch memory)
#pragma unroll
        for (int j = KD < VD ? KD : VD; j < MD; ++j) chunk[i].code[j] = 0;
      }
      if (c < KCHUNKS) {
        const int t16 = c / KG & 1, g = c % KG;
        load_words<KD, KD>(cache.kq + u * (NB * 32 * kv_code_bytes(KF)) + t16 * (NB * 16 * kv_code_bytes(KF)) + (g * 64 + lane) * (KD * 4),
                           chunk[i].code);
        if constexpr (K_SCALED) {
          const uint16_t* sp = cache.ks + u * (32 * NB) + (t16 * 16 + (lane & 15)) * NB + g * KB;
          if constexpr (KB % 2 == 0) {
            load_words<KB / 2, KB / 2>(reinterpret_cast<const uint8_t*>(sp), chunk[i].scale);
          } else {
#pragma unroll
            for (int b = 0; b < KB; ++b) chunk[i].scale[b] = sp[b];
          }
        }
      } else {
        const int g = (c - KCHUNKS) % VG;
        load_words<VD, VD>(cache.vq + u * (NB * 32 * kv_code_bytes(VF)) + (g * 64 + lane) * (VD * 4), chunk[i].code);
        if constexpr (V_SCALED) {
          const uint16_t* sp = cache.vs + u * (32 * NB) + ((lane >> 4) * NB + g * VB) * 8;
          load_words<4 * VB, 4>(reinterpret_cast<const uint8_t*>(sp), chunk[i].scale);
        }
      }
    }
    if constexpr (!K_SCALED) if (wave < HALVES) {
      const int64_t u = unit(wave);
#pragma unroll
      for (int i = 0; i < SW; ++i) {
        const int at = min(i * 64 + lane, 16 * NB - 1);
        ks[i] = u < 0 ? 0u : reinterpret_cast<const unsigned*>(cache.ks)[u * (16 * NB) + at];
        if constexpr (!V_SCALED) vs[i] = u < 0 ? 0u : reinterpret_cast<const unsigned*>(cache.vs)[u * (16 * NB) + at];
      }
    }
  }

  // the tokens of a pair of value scales, place i of a quarter's four: this one and the one 2 on
  static __device__ __forceinline__ int value_token(int quarter, int i) { return 16 * (i >> 1 & 1) + 4 * quarter + (i & 1); }
  static __device__ __forceinline__ unsigned value_mask(int quarter, int i, int left) {  // leaves those before `left`
    const int token = value_token(quarter, i);
    return (token < left ? 0xFFFFu : 0u) | (token + 2 < left ? 0xFFFF0000u : 0u);
  }

  // The loaded scales: those of keys from `length` on become 0, and so do values' that are no numbers, which go into
  // bad[slot]; the largest exponents go to most[slot].  (Scales beside the operands: the masks keep the products numbers.)
  __device__ __forceinline__ void look(Shared& sh, int slot, int first, int length, int wave, int lane) {
    unsigned e = 0, ek = 0;
    if constexpr (V_SCALED) {
#pragma unroll
      for (int i = 0; i < TURNS; ++i) {
        const int c = i * WAVES + wave;
        if (!there[i]) continue;
        if (c < KCHUNKS) {
          if constexpr (K_SCALED) {
            const bool in = (c / KG & 1) * 16 + (lane & 15) < length - first - half_of(c) * 32;
#pragma unroll
            for (int b = 0; b < (KB % 2 == 0 ? KB / 2 : KB); ++b) {
              chunk[i].scale[b] = in ? chunk[i].scale[b] : 0u;
              const unsigned lo = chunk[i].scale[b] & 0x7C00u, hi = chunk[i].scale[b] >> 16 & 0x7C00u;
              ek = max(ek, max(lo == 0x7C00u ? 0u : lo, hi == 0x7C00u ? 0u : hi));
            }
          }
          continue;
        }
        const int left = length - first - half_of(c) * 32;
        unsigned worst = 0;
#pragma unroll
        for (int j = 0; j < 4 * VB; ++j) {
          if (left < 32) chunk[i].scale[j] &= value_mask(lane >> 4, j, left);
          worst = max(worst, max(chunk[i].scale[j] & 0x7C00u, chunk[i].scale[j] >> 16 & 0x7C00u));
        }
        if (__builtin_amdgcn_ballot_w64(worst == 0x7C00u) != 0) {
          worst = 0;
#pragma unroll
          for (int j = 0; j < 4 * VB; ++j) {
            unsigned lo = chunk[i].scale[j] & 0xFFFFu, hi = chunk[i].scale[j] >> 16;
            const unsigned token = value_token(lane >> 4, j & 3);
            unsigned none = 0;
            if ((lo & 0x7C00u) == 0x7C00u) none |= 1u << token, lo = 0;
            if ((hi & 0x7C00u) == 0x7C00u) none |= 4u << token, hi = 0;
            if (none && (lane & 15) == 0) {
              atomicOr(&sh.bad[slot][1 + half_of(c) * NB + (c - KCHUNKS) % VG * VB + (j >> 2)], none);
              atomicOr(&sh.bad[slot][0], SPOILT);
            }
            chunk[i].scale[j] = lo | hi << 16;
            worst = max(worst, max(lo & 0x7C00u, hi & 0x7C00u));
          }
        }
        e = max(e, worst >> 10);
      }
    } else if (wave < HALVES) {
#pragma unroll
      for (int i = 0; i < SW; ++i) {
        const int at = min(i * 64 + lane, 16 * NB - 1);
        vs[i] &= value_mask(at / (4 * NB), at, length - first - wave * 32);
        const unsigned lo = vs[i] >> 10 & 31, hi = vs[i] >> 26 & 31;
        e = max(e, max(lo == 31 ? 0u : lo, hi == 31 ? 0u : hi));
      }
    }
    int top = static_cast<int>(e);
    if constexpr (!V_SCALED) top = row16_max_i(top);  // (value operands: a row's lanes have the same scales)
    top = static_cast<int>(quarters_max(static_cast<float>(top)));
    if constexpr (!V_SCALED) {
      if (wave < HALVES && lane == 0) sh.most[slot][wave] = static_cast<unsigned>(top);
    } else {
      if (top && lane == 0) atomicMax(&sh.most[slot][0], static_cast<unsigned>(top));
      if constexpr (K_SCALED) {
        const int k = row16_max_i(static_cast<int>(ek >> 10));  // (the quarters have the same keys)
        if (k && lane == 0) atomicMax(&sh.most[slot][1], static_cast<unsigned>(k));
      }
    }
  }

  // the loaded codes as operands in buffer `buf`
  __device__ __forceinline__ void unpack(Shared& sh, int buf, int slot, int wave, int lane) {
    f16x2 fv = {}, fk = {};  // 2^(15 - field)
    auto power = [&](int which) {
      const _Float16 f = static_cast<_Float16>(__builtin_ldexpf(1.f, 15 - static_cast<int>(max(sh.most[slot][which], 1u))));
      return f16x2{f, f};
    };
    if constexpr (V_SCALED) {
      fv = power(0), fk = power(1);
      // f16 scales (but 0) of exponent fields below this, 2 at least, lose bits to the power
      auto least = [&](int which) { return __builtin_amdgcn_readfirstlane(static_cast<int>(sh.most[slot][which])) - 14; };
      auto below = [](unsigned pair, int field) {
        const unsigned lo = pair & 0x7FFFu, hi = pair >> 16 & 0x7FFFu, to = static_cast<unsigned>(field) << 10;
        return (lo != 0 && lo < to) || (hi != 0 && hi < to);
      };
      const int kl = K_SCALED ? least(1) : 0, vl = least(0);
      if (kl > 1 || vl > 1) {
        bool scattered = false;
#pragma unroll
        for (int i = 0; i < TURNS; ++i) {
          if (!there[i]) continue;
          if (i * WAVES + wave < KCHUNKS) {
#pragma unroll
            for (int b = 0; K_SCALED && b < (KB % 2 == 0 ? KB / 2 : KB); ++b) scattered |= kl > 1 && below(chunk[i].scale[b], kl);
          } else {
#pragma unroll
            for (int j = 0; j < 4 * VB; ++j) scattered |= vl > 1 && below(chunk[i].scale[j], vl);
          }
        }
        if (scattered) atomicOr(&sh.bad[slot][0], SCATTERED);
      }
    }
#pragma unroll
    for (int i = 0; i < TURNS; ++i) {
      const int c = i * WAVES + wave;
      if (!there[i]) continue;
      if (c < KCHUNKS) {
        f16x8* to = &sh.k[buf][c / KG * NB + c % KG * KB][lane];
#pragma unroll
        for (int b = 0; b < KB; ++b) {
          f16x8 x;
          if constexpr (KF == KV_Q4_0) x = key_codes<true, KF>(chunk[i].code[b], 0u);
          else x = key_codes<true, KF>(chunk[i].code[2 * b], chunk[i].code[2 * b + 1]);
          if constexpr (K_SCALED) {
            const _Float16 d = KB % 2 == 0 ? as_f16x2(chunk[i].scale[b >> 1])[b & 1] : as_f16x2(chunk[i].scale[b])[0];
            const f16x2 dd = f16x2{d, d} * fk;
            x *= f16x8{dd[0], dd[0], dd[0], dd[0], dd[0], dd[0], dd[0], dd[0]};
          }
          to[b * 64] = x;
        }
      } else {
        f16x8* to = &sh.v[buf][(c - KCHUNKS) * VB * 2][lane];
#pragma unroll
        for (int b = 0; b < VB; ++b) {
          u32x4 d;
          if constexpr (V_SCALED) {
#pragma unroll
            for (int j = 0; j < 4; ++j) d[j] = __builtin_bit_cast(unsigned, as_f16x2(chunk[i].scale[4 * b + j]) * fv);
          }
#pragma unroll
          for (int hh = 0; hh < 2; ++hh) {
            f16x8 x;
            if constexpr (VF == KV_Q4_0) x = value_codes<VF>(chunk[i].code[2 * b], chunk[i].code[2 * b + 1], hh);
            else x = value_codes<VF>(chunk[i].code[4 * b + 2 * hh], chunk[i].code[4 * b + 2 * hh + 1], 0);
            if constexpr (V_SCALED) x *= __builtin_bit_cast(f16x8, d);
            to[(b * 2 + hh) * 64] = x;
          }
        }
      }
    }
    if constexpr (!K_SCALED) if (wave < HALVES) {
#pragma unroll
      for (int i = 0; i < SW; ++i) {
        const int at = min(i * 64 + lane, 16 * NB - 1);
        sh.ks[buf][wave][at] = ks[i];
        if constexpr (!V_SCALED) sh.vs[buf][wave][at] = vs[i];
      }
    }
  }

  // a wave's columns over half `half` of the tile in `buf`, its keys from `first` on
  static __device__ __forceinline__ void step(Cols& cols, const AttendArgs& a, const Shared& sh, bool masked, int buf, int slot,
                                              int half, int first, int lane) {
    constexpr int ROWS = (4 * NB + 15) / 16;  // a quarter's scales: dwords a lane of its 16
    const int quarter = lane >> 4, key0 = first + quarter * 4;
    const int e = __builtin_amdgcn_readfirstlane(static_cast<int>(max(sh.most[slot][V_SCALED ? 0 : half], 1u)));
    unsigned ks[ROWS] = {};
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const int at = min(i * 16 + (lane & 15), 4 * NB - 1), t = at / (2 * NB);
      if constexpr (!K_SCALED) ks[i] = sh.ks[buf][half][t * 8 * NB + quarter * 2 * NB + at - t * 2 * NB];
    }
    float y[CT][2][4];
    each<2>([&](auto tc) {
      constexpr int t = tc.value;
      // blocks at a time, whose partial dots are held until their scales come
      constexpr int AT = TIGHT ? 2 : NB;
      each<NB / AT>([&](auto gc) {
        constexpr int b0 = gc.value * AT;
        f32x4 c[CT][AT];
#pragma unroll
        for (int b = 0; b < AT; ++b) {
          const f16x8 k = sh.k[buf][(half * 2 + t) * NB + b0 + b][lane];
#pragma unroll
          for (int ct = 0; ct < CT; ++ct) {
            f32x4& x = c[ct][K_SCALED ? 0 : b];
            if (!K_SCALED || b == 0) x = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int p = 0; p < Cols::PARTS; ++p) x = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, cols.qf[ct][b0 + b][p], x, 0, 0, 0);
          }
        }
        if constexpr (K_SCALED) {
#pragma unroll
          for (int ct = 0; ct < CT; ++ct)
#pragma unroll
            for (int r = 0; r < 4; ++r) y[ct][t][r] = c[ct][0][r];
        } else {
          // dword j has the scales of places 2 j and 2 j + 1 of [4 keys][NB]
          each<2 * AT>([&](auto ic) {
            constexpr int i = ic.value, j = AT == NB ? i : i * (NB / 2) + b0 / 2, at = t * 2 * NB + j;
            const f16x2 d = as_f16x2(row_lane<at % 16>(ks[at / 16]));
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int r = (2 * j + h) / NB, b = (2 * j + h) % NB - b0;
#pragma unroll
              for (int ct = 0; ct < CT; ++ct)
                y[ct][t][r] = b0 + b == 0 ? static_cast<float>(d[h]) * c[ct][b][r] : fmaf(static_cast<float>(d[h]), c[ct][b][r], y[ct][t][r]);
            }
          });
        }
      });
    });
    const int left = min(Cols::ROOM, 21 - e);
    if constexpr (V_SCALED) {
      float unit = 1.f;
      if constexpr (K_SCALED)
        unit = __builtin_ldexpf(1.f, __builtin_amdgcn_readfirstlane(static_cast<int>(max(sh.most[slot][1], 1u))) - 15);
      // (the power of two is the whole tile's, and so is what P may reach)
      cols.soften(a, masked, key0, left, unit, e - 15, y, nullptr);
    } else {
      unsigned own[ROWS];
      cols.soften(a, masked, key0, left, 1.f, 0, y, [&]() -> auto& {
#pragma unroll
        for (int i = 0; i < ROWS; ++i) own[i] = sh.vs[buf][half][quarter * 4 * NB + min(i * 16 + (lane & 15), 4 * NB - 1)];
        return own;
      });
    }
    if constexpr (V_SCALED) {
      unsigned w[CT][4];
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) Cols::pack(y[ct], w[ct]);
#pragma unroll
      for (int i = 0; i < 2 * NB; ++i) {
        const f16x8 v = sh.v[buf][half * NB * 2 + i][lane];
#pragma unroll
        for (int ct = 0; ct < CT; ++ct)
          cols.acc[ct][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, as_f16x8(w[ct][0], w[ct][1], w[ct][2], w[ct][3]),
                                                                  cols.acc[ct][i], 0, 0, 0);
      }
    } else {
      unsigned vs[ROWS], keep[CT][4];
#pragma unroll
      for (int i = 0; i < ROWS; ++i) vs[i] = sh.vs[buf][half][quarter * 4 * NB + min(i * 16 + (lane & 15), 4 * NB - 1)];
      if (masked) {
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) cols.seen_pairs(ct, key0, keep[ct]);
      }
      each<NB>([&](auto bc) {
        constexpr int b = bc.value;
        unsigned w[CT][Cols::PARTS][4];
        each<4>([&](auto ic) {
          constexpr int i = ic.value, at = 4 * b + i;
          const f16x2 d = as_f16x2(row_lane<at % 16>(vs[at / 16]));
#pragma unroll
          for (int ct = 0; ct < CT; ++ct) {
            Cols::weigh(y[ct][i >> 1][i & 1], y[ct][i >> 1][2 + (i & 1)], d, w[ct], i);
            if (masked) {
#pragma unroll
              for (int p = 0; p < Cols::PARTS; ++p) w[ct][p][i] &= keep[ct][i];
            }
          }
        });
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          const f16x8 v = sh.v[buf][(half * NB + b) * 2 + hh][lane];
#pragma unroll
          for (int ct = 0; ct < CT; ++ct)
#pragma unroll
            for (int p = 0; p < Cols::PARTS; ++p)
              cols.acc[ct][2 * b + hh] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                  v, as_f16x8(w[ct][p][0], w[ct][p][1], w[ct][p][2], w[ct][p][3]), cols.acc[ct][2 * b + hh], 0, 0, 0);
        }
      });
    }
  }

  // the channels of blocks without a scale, in the columns that see their tokens
  static __device__ __forceinline__ void spoil(Cols& cols, const Shared& sh, int slot, int half, int first) {
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      const int lo = max(0, cols.span[ct].lo - first), hi = min(32, cols.span[ct].hi - first);
      const unsigned seen = lo >= hi ? 0u : (hi == 32 ? ~0u : (1u << hi) - 1) & ~((1u << lo) - 1);
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const bool to = (sh.bad[slot][V_SCALED ? 1 + half * NB + b : 0] & seen) != 0;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          cols.acc[ct][2 * b][r] = to ? __builtin_nanf("") : cols.acc[ct][2 * b][r];
          cols.acc[ct][2 * b + 1][r] = to ? __builtin_nanf("") : cols.acc[ct][2 * b + 1][r];
        }
      }
    }
  }
};

// A workgroup's columns over its keys; false where a tile's scales are scattered, for all of its waves at the same point, and
// nothing is stored then.
template <typename M>
__device__ __forceinline__ bool attend_many(const AttendArgs& a, typename M::Shared& sh, int thread, int h, int seq) {
  constexpr int NB = M::BLOCKS;
  const int lane = thread & 63, wave = __builtin_amdgcn_readfirstlane(thread >> 6);
  __builtin_assume(wave >= 0 && wave < M::WAVES);
  const int split = blockIdx.z / a.groups;
  // the groups of the latest positions, which see the most keys, begin first, those of all heads and sequences together
  const int group0 = (a.groups - 1 - (static_cast<int>(blockIdx.z) - split * a.groups)) * (M::WAVES * M::COLS);
  const Sequence s(a, seq);
  if (group0 >= s.cols) return true;
  const Span g0 = s.seen(a, group0 / a.group), g1 = s.seen(a, (min(s.cols, group0 + M::WAVES * M::COLS) - 1) / a.group);
  int tile0 = g0.lo / M::KEYS, tile1 = (g1.hi + M::KEYS - 1) / M::KEYS;
  if (tile0 > tile1) tile0 = tile1 = 0;
  const int per = (tile1 - tile0 + a.splits - 1) / a.splits;
  tile0 = min(tile1, tile0 + split * per);
  tile1 = min(tile1, tile0 + per);

  // the wave's own columns: what they see, and what all of them see
  const int col0 = group0 + wave * M::COLS;
  const bool any = col0 < s.cols;
  const Span w0 = s.seen(a, any ? col0 / a.group : 0), w1 = s.seen(a, any ? (min(s.cols, col0 + M::COLS) - 1) / a.group : 0);

  const Pages pages(a, seq, h);
  auto unit = [&](int tile, int half) -> int64_t {
    // (no branch, so that a tile's table entries are loaded together; there is a first key where there is a tile)
    const int at = tile * M::HALVES + half, last = (s.length - 1) >> 5;
    const int64_t u = pages.unit(min(at, last));
    return ((tile < tile1) & (at <= last)) ? u : -1;
  };
  auto halves = [&](int tile) {  // a bit for each half that lies somewhere
    unsigned there = 0;
#pragma unroll
    for (int i = 0; i < M::HALVES; ++i) there |= unit(tile, i) < 0 ? 0u : 1u << i;
    return there;
  };
  typename M::Cols cols;
  cols.all = Span{w0.lo, w1.hi};
  typename M::Cols::Raw query;
  cols.fetch(a, s, h, col0, lane, query);
  cols.begin(a, s, h, col0, lane, query);
  if (tile0 < tile1) {
    M m;
    if (M::V_SCALED && thread < 4 * M::MOST) (&sh.most[0][0])[thread] = 0;
    constexpr int BAD = M::V_SCALED ? 1 + M::HALVES * NB : 0;
    if (thread < 4 * BAD) (&sh.bad[0][0])[thread] = 0;
    unsigned now = halves(tile0);
    m.load(a.c, [&](int half) { return unit(tile0, half); }, wave, lane);
    __syncthreads();
    m.look(sh, 0, tile0 * M::KEYS, s.length, wave, lane);
    __syncthreads();
    m.unpack(sh, 0, 0, wave, lane);
    unsigned next = halves(tile0 + 1);
    m.load(a.c, [&](int half) { return unit(tile0 + 1, half); }, wave, lane);
    m.look(sh, 1, (tile0 + 1) * M::KEYS, s.length, wave, lane);
    __syncthreads();
    for (int tile = tile0; tile < tile1; ++tile) {
      // most[] and bad[]: this tile's are in slot i, the next one's in i + 1, the one after's are filled in i + 2, and i + 3,
      // last read a turn ago, is cleared for the turn to come
      const int i = tile - tile0, buf = i & 1;
      if (M::V_SCALED && thread < M::MOST) sh.most[(i + 3) & 3][thread] = 0;
      if (thread < BAD) sh.bad[(i + 3) & 3][thread] = 0;
      const int at = M::here(lane);
      m.unpack(sh, buf ^ 1, (i + 1) & 3, wave, at);
      const unsigned after = halves(tile + 2);
      m.load(a.c, [&](int half) { return unit(tile + 2, half); }, wave, at);
      const unsigned flags = M::V_SCALED ? __builtin_amdgcn_readfirstlane(sh.bad[i & 3][0]) : 0u;
      if (flags & M::SCATTERED) return false;  // (set before the last barrier: every wave sees it here)
#pragma unroll 1
      for (int half = 0; half < M::HALVES; ++half) {
        const int first = tile * M::KEYS + half * 32;
        if (!any || first >= w1.hi || first + 32 <= w0.lo || !(now >> half & 1)) continue;
        M::step(cols, a, sh, first < w1.lo || first + 32 > w0.hi, buf, i & 3, half, first, M::here(lane));
      }
      if (flags & M::SPOILT) {
#pragma unroll 1
        for (int half = 0; half < M::HALVES; ++half)
          if (any && (now >> half & 1)) M::spoil(cols, sh, i & 3, half, tile * M::KEYS + half * 32);
      }
      m.look(sh, (i + 2) & 3, (tile + 2) * M::KEYS, s.length, wave, at);
      now = next;
      next = after;
      __syncthreads();
    }
  }
  if (!any) return true;
#pragma unroll
  for (int ct = 0; ct < M::CT; ++ct) cols.l[ct] = quarters_sum(cols.l[ct]);
  cols.store(a, s, h, col0, split, lane);
  return true;
}

template <int NB, int KF, int VF, int MODE, int SCALED>
struct ManyKernel {
  using First = Many<NB, KF, VF, MODE, SCALED>;
  using Exact = Many<NB, KF, VF, MODE, KV_EXACT>;
  static constexpr int THREADS = 64 * First::WAVES;
  static constexpr size_t SHARED = sizeof(typename First::Shared) > sizeof(typename Exact::Shared) ? sizeof(typename First::Shared)
                                                                                                   : sizeof(typename Exact::Shared);
  static_assert(First::WAVES == Exact::WAVES && First::COLS == Exact::COLS, "one launch serves both");
};
template <int NB, int KF, int VF, int MODE, int SCALED>
__global__ void __launch_bounds__((ManyKernel<NB, KF, VF, MODE, SCALED>::THREADS), (ManyKernel<NB, KF, VF, MODE, SCALED>::THREADS / 256))
kv_attend_many_kernel(const AttendArgs a) {
  using K = ManyKernel<NB, KF, VF, MODE, SCALED>;
  extern __shared__ __attribute__((aligned(16))) unsigned char shared_bytes[];
  int thread = threadIdx.x, h = blockIdx.x, seq = blockIdx.y;
  const bool done = attend_many<typename K::First>(a, *reinterpret_cast<typename K::First::Shared*>(shared_bytes), thread, h, seq);
  if constexpr (SCALED != KV_EXACT) {
    if (done) return;
    __syncthreads();
    // (nothing of the first pass is held for this one: it loads the arguments again)
    auto args = __builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+v"(thread), "+s"(h), "+s"(seq), "+s"(args));
    const AttendArgs again = *(const AttendArgs*)(const void*)args;
    attend_many<typename K::Exact>(again, *reinterpret_cast<typename K::Exact::Shared*>(shared_bytes), thread, h, seq);
  }
}

template <int NB, int KF, int VF, int MODE, int SCALED>
hipError_t launch_attend_many(const AttendArgs& a, const dim3& grid, hipStream_t stream) {
  using K = ManyKernel<NB, KF, VF, MODE, SCALED>;
  static std::atomic<unsigned> limit[kMaxDevices];
  const auto kern = kv_attend_many_kernel<NB, KF, VF, MODE, SCALED>;
  constexpr size_t bytes = K::SHARED;
  const hipError_t e = allow_dynamic_lds(reinterpret_cast<const void*>(kern), bytes, limit);
  if (e != hipSuccess) return e;
  const Timing tm = timing_slot(KIND_PROBE);
  if (tm.on) {
    hipExtLaunchKernelGGL(kern, grid, dim3(K::THREADS), bytes, stream, tm.start, tm.stop, 0, a);
  } else {
    hipLaunchKernelGGL(kern, grid, dim3(K::THREADS), bytes, stream, a);
  }
  return hipGetLastError();
}

}  // namespace komp
