// Device helpers of the microscaled rows: loads and stores of the three float types, and a block's quantization.
//
// The conversions are the CDNA4 instructions v_cvt_scalef32_*: nearest even, a scale operand of which only the exponent counts
// (bits s << 23: 2^(s - 127), s = 0 and 255 included).  To e2m1 they saturate; to e4m3 they do not, so values are clamped first.
#pragma once

#include "komp_device.h"
#include "mx_layout.h"

namespace komp {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef short s16x2v __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

template <int TYPE>
struct MxElement {
  typedef float type;
};
template <>
struct MxElement<MX_F16> {
  typedef _Float16 type;
};
template <>
struct MxElement<MX_BF16> {
  typedef __bf16 type;
};

// N consecutive elements, as f32; their address need only be aligned to one element (gfx950 loads and stores them as wide all
// the same).
template <int TYPE, int N>
__device__ __forceinline__ void mx_load(const void* p, int64_t i, float (&v)[N]) {
  typedef typename MxElement<TYPE>::type T;
  typedef T vec __attribute__((ext_vector_type(N), aligned(sizeof(T))));
  const vec x = *reinterpret_cast<const vec*>(static_cast<const T*>(p) + i);
#pragma unroll
  for (int e = 0; e < N; ++e) v[e] = static_cast<float>(x[e]);
}

template <int TYPE, int N>
__device__ __forceinline__ void mx_store(void* p, int64_t i, const float (&v)[N]) {
  typedef typename MxElement<TYPE>::type T;
  typedef T vec __attribute__((ext_vector_type(N), aligned(sizeof(T))));
  vec x;
#pragma unroll
  for (int e = 0; e < N; ++e) x[e] = static_cast<T>(v[e]);  // nearest even
  *reinterpret_cast<vec*>(static_cast<T*>(p) + i) = x;
}

__device__ __forceinline__ unsigned umax(unsigned a, unsigned b) { return a > b ? a : b; }

// The largest |value|'s f32 bits: they order as the magnitudes do, with infinity and the NaNs above all others.
template <int N>
__device__ __forceinline__ unsigned mx_most(const float (&v)[N]) {
  unsigned m = 0;
#pragma unroll
  for (int e = 0; e < N; ++e) m = umax(m, __float_as_uint(v[e]) & 0x7FFFFFFFu);
  return m;
}

// A block's scale byte from the bits of its largest magnitude: the exponent that brings it into the elements' last binade,
// [4, 8) of e2m1 (to 6) and [256, 512) of e4m3 (to 448); 255 where it is no number.
template <int FMT>
__device__ __forceinline__ unsigned mx_scale(unsigned most) {
  const unsigned e = most >> 23;
  constexpr unsigned high = FMT == MX_E2M1 ? 2 : 8;
  return e == 255 ? 255u : e > high ? e - high : 0u;
}

// Eight elements: a dword of e2m1 or two of e4m3.  A block without a number holds zeros.
template <int FMT>
__device__ __forceinline__ void mx_codes8(const float* v, unsigned s, unsigned (&out)[FMT == MX_E2M1 ? 1 : 2]) {
  const float scale = __uint_as_float(s << 23);
  if constexpr (FMT == MX_E2M1) {
    unsigned p = 0;
    p = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(p, v[0], v[1], scale, 0);
    p = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(p, v[2], v[3], scale, 1);
    p = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(p, v[4], v[5], scale, 2);
    p = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(p, v[6], v[7], scale, 3);
    out[0] = s == 255 ? 0 : p;
  } else {
    const float top = __builtin_ldexpf(448.f, static_cast<int>(s) - 127);
    float c[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) c[e] = __builtin_amdgcn_fmed3f(v[e], -top, top);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      s16x2v p = {0, 0};
      p = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(p, c[4 * h], c[4 * h + 1], scale, false);
      p = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(p, c[4 * h + 2], c[4 * h + 3], scale, true);
      out[h] = s == 255 ? 0 : __builtin_bit_cast(unsigned, p);
    }
  }
}

// What four or eight elements in shared memory stand for, in f32 (exact).
template <int FMT, int N>
__device__ __forceinline__ void mx_values(const uint8_t* from, float scale, float (&v)[N]) {
  f32x2 p[N / 2];
  if constexpr (FMT == MX_E2M1) {
    const unsigned q = N == 8 ? *reinterpret_cast<const unsigned*>(from) : *reinterpret_cast<const uint16_t*>(from);
    p[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, scale, 0);
    p[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, scale, 1);
    if constexpr (N == 8) {
      p[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, scale, 2);
      p[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, scale, 3);
    }
  } else {
    const unsigned q = reinterpret_cast<const unsigned*>(from)[0];
    p[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(q, scale, false);
    p[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(q, scale, true);
    if constexpr (N == 8) {
      const unsigned r = reinterpret_cast<const unsigned*>(from)[1];
      p[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(r, scale, false);
      p[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(r, scale, true);
    }
  }
#pragma unroll
  for (int e = 0; e < N; ++e) v[e] = p[e / 2][e % 2];
}

}  // namespace komp
