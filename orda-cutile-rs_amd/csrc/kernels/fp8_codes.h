// fp8_codes.h — e4m3 codes of a block's values: shared by the quantiser and by the
// kernels that quantise what they compute.
#pragma once

#include <float.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace orda {
namespace {

typedef uint32_t fp8_u32x2 __attribute__((ext_vector_type(2)));
constexpr float kE4m3Max = 448.f;

__device__ __forceinline__ float scale_of(uint32_t amax_bits) {
  if (amax_bits >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
  return fmaxf(__uint_as_float(amax_bits) / kE4m3Max, FLT_MIN);
}
__device__ __forceinline__ float coded(float x, float s) {
  const float q = x / s;
  return q != q ? q : fminf(fmaxf(q, -kE4m3Max), kE4m3Max);
}
// Whether x / s might round to another code than q = x * (1/s), which is at most 3
// units in the last place off the rounded quotient: near a midpoint of two
// codes (three bits of mantissa are kept: the other 20 near one half), or below
// the smallest normal code, where the midpoints lie elsewhere.
__device__ __forceinline__ bool doubtful(float q) {
  const uint32_t u = __float_as_uint(q) & 0x7fffffffu;
  return (u & 0xfffffu) - 0x7fffcu <= 8u || (u < 0x3c800004u && u != 0u) || u >= 0x7f800000u;
}
__device__ __forceinline__ uint32_t codes4(const float* x, float s, float r) {
  float q[4];
  bool doubt = false;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    q[k] = x[k] * r;
    doubt |= doubtful(q[k]);
    q[k] = fminf(fmaxf(q[k], -kE4m3Max), kE4m3Max);
  }
  if (doubt) {
#pragma unroll
    for (int k = 0; k < 4; ++k) q[k] = coded(x[k], s);
  }
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], w, true);
  return static_cast<uint32_t>(w);
}
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
// The codes of eight neighbouring values, the eight that hold the last column whole.
__device__ __forceinline__ void store8(uint8_t* row, int64_t c, int64_t cols, const float (&x)[8], float s) {
  const float r = __builtin_amdgcn_rcpf(s);
  if (c < cols) *reinterpret_cast<fp8_u32x2*>(row + c) = fp8_u32x2{codes4(x, s, r), codes4(x + 4, s, r)};
}

// The same scale and codes without divisions or a branch on the values: with r the
// rounded 1/s and q = x·r rounded, q·s - x is exact and q - (q·s - x)·r the rounded
// quotient (P. Markstein, 1990) where nothing of it is under the normal range: values
// whose largest is over 2^-90. (Signs as written: a zero keeps its own.)
__device__ __forceinline__ float quotient(float x, float s, float r) {
  const float q = x * r;
  return fmaf(-fmaf(q, s, -x), r, q);
}
__device__ __forceinline__ float scale_divided(uint32_t amax_bits) {
  constexpr float kReciprocal = 1.f / kE4m3Max;
  const float m = __uint_as_float(amax_bits);
  return amax_bits - 0x12800000u < 0x7f800000u - 0x12800000u ? quotient(m, kE4m3Max, kReciprocal) : scale_of(amax_bits);
}
__device__ __forceinline__ void store8_divided(uint8_t* row, int64_t c, int64_t cols, const float (&x)[8], float s) {
  if (c >= cols) return;
  if (!(s >= 1.8e-30f)) {   // 2^-99; also NaN
    store8(row, c, cols, x, s);
    return;
  }
  float r = __builtin_amdgcn_rcpf(s);
  r = fmaf(fmaf(-s, r, 1.f), r, r);
  r = fmaf(fmaf(-s, r, 1.f), r, r);
  float q[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) q[k] = __builtin_amdgcn_fmed3f(quotient(x[k], s, r), -kE4m3Max, kE4m3Max);
  uint32_t w[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    int u = __builtin_amdgcn_cvt_pk_fp8_f32(q[4 * k], q[4 * k + 1], 0, false);
    u = __builtin_amdgcn_cvt_pk_fp8_f32(q[4 * k + 2], q[4 * k + 3], u, true);
    w[k] = static_cast<uint32_t>(u);
  }
  *reinterpret_cast<fp8_u32x2*>(row + c) = fp8_u32x2{w[0], w[1]};
}

}  // namespace
}  // namespace orda
