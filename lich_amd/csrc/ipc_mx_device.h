// ipc_mx_device.h - device helpers of the microscaled formats (gfx950).
#pragma once

#include "ipc_device.h"
#include "ipc_mx.h"

namespace ipc {
namespace mx {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

// Scale byte of a block from the largest of its values' magnitudes, as bits of
// a float (so NaN counts as more than infinity).  Half a unit of the element's
// last place is added before the exponent is read: 1 mantissa bit of E2M1, 6
// fraction bits of int8.  Magnitudes that would round past the largest float
// saturate.  0 for a block of zeros; 1 (2^-126) at the least
// otherwise, so that every scale in use is a normal float.
template <int FMT>
__device__ __forceinline__ unsigned scale_byte(unsigned amax) {
  const int e = (int)((amax + (FMT == MX_FP4 ? 0x200000u : 0x10000u)) >> 23) - (FMT == MX_FP4 ? 2 : 0);
  constexpr int TOP = FMT == MX_FP4 ? 252 : 254;  // 6 * 2^125, 127/64 * 2^127: the largest finite results
  const int s = e < 1 ? 1 : e > TOP ? TOP : e;
  return amax >= 0x7f800000u ? 255u : amax == 0u ? 0u : (unsigned)s;
}

__device__ __forceinline__ unsigned abs_bits(float v) { return __builtin_bit_cast(unsigned, v) & 0x7fffffffu; }

// N (4 or 8) values of a block with scale byte s as E2M1 codes, 4 bits each.  The
// conversion divides by the scale, rounds to nearest even and saturates at 6,
// which only values the rule above lets through (6 .. 7, next to the largest float
// 6 .. 8) reach.
template <int N>
__device__ __forceinline__ unsigned fp4_codes(const float (&v)[N], unsigned s) {
  const float scale = __builtin_bit_cast(float, (s == 255u ? 0u : s) << 23);
  unsigned o = 0;
  o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, v[0], v[1], scale, 0);
  o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, v[2], v[3], scale, 1);
  if constexpr (N == 8) {
    o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, v[4], v[5], scale, 2);
    o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, v[6], v[7], scale, 3);
  }
  return s == 0u || s == 255u ? 0u : o;  // (a zero scale divides by nothing: all codes are 0)
}

// 4 values as a dword of int8 codes: v * 2^(133 - s), an exact product, rounded
// to the nearest even integer; 128 (possible only at s = 254) saturates.
__device__ __forceinline__ unsigned int8_codes4(float a, float b, float c, float d, unsigned s) {
  if (s == 0u || s == 255u) return 0u;
  const int k = 133 - (int)s;
  auto q = [&](float v) -> unsigned {
    const float r = __builtin_rintf(__builtin_ldexpf(v, k));
    return (unsigned)(int)__builtin_amdgcn_fmed3f(r, -127.0f, 127.0f) & 255u;
  };
  return q(a) | (q(b) << 8) | (q(c) << 16) | (q(d) << 24);
}

// 2^(s - 133), the value of code 1 in an int8 block with scale byte s: code times
// this is exact (NaN for s = 255).
__device__ __forceinline__ float int8_scale(unsigned s) {
  return s == 255u ? __builtin_nanf("") : __builtin_ldexpf(1.0f, (int)s - 133);
}
__device__ __forceinline__ int sext8(unsigned w, int byte) { return (int)(w << (24 - 8 * byte)) >> 24; }

// N (4 or 8) values of E2M1 codes in a block with scale byte s.
template <int N>
__device__ __forceinline__ void fp4_values(unsigned q, unsigned s, float (&o)[N]) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  const float scale = __builtin_bit_cast(float, s << 23);
  const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, scale, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, scale, 1);
  o[0] = a[0]; o[1] = a[1]; o[2] = b[0]; o[3] = b[1];
  if constexpr (N == 8) {
    const f32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, scale, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, scale, 3);
    o[4] = c[0]; o[5] = c[1]; o[6] = d[0]; o[7] = d[1];
  }
  if (s == 255u) {
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = __builtin_nanf("");
  }
}

// N consecutive elements (16 bytes) at any element-aligned address: gfx950's
// global loads and stores take any alignment.
template <typename ST, int N>
struct Run {
  typedef ST V __attribute__((ext_vector_type(N)));
  struct __attribute__((packed, aligned(sizeof(ST)))) U { V v; };
};
template <typename ST, int N>
__device__ __forceinline__ void load_run(const ST* p, float (&o)[N]) {
  const typename Run<ST, N>::V v = reinterpret_cast<const typename Run<ST, N>::U*>(p)->v;
#pragma unroll
  for (int i = 0; i < N; ++i) o[i] = to_f32(v[i]);
}
template <typename ST, int N>
__device__ __forceinline__ void store_run(ST* p, const float (&o)[N]) {
  typename Run<ST, N>::V v;
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = cvt<ST>(o[i]);
  reinterpret_cast<typename Run<ST, N>::U*>(p)->v = v;
}

}  // namespace mx
}  // namespace ipc
