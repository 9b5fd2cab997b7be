// ce_few.hip — the logits of a few rows for the linear cross entropy: a token or a
// small batch against the whole vocabulary.
//
// Bound by the weight's bytes, which each go once from memory to the registers of
// one wave, with no LDS and no barrier before the end. A wave takes 16 classes and
// all rows (F fragments of 16, from the caches) and loads the next 256 bytes of each,
// or 512, while it multiplies these; the workgroup's 64 classes are one tile
// of statistics. The weight's rows may have any pitch and alignment: its vectors
// need none but their elements'. A tile of the large product holds 256 classes, so that 14000
// classes are 56 workgroups on 256 CUs. One row at 32000 x 2048: 23 us, 5.8 TB/s (on
// the tiles 41); 18 rows at 14334 x 4032 31 us, 3.7 TB/s (75), where the rows' way
// from the second-level caches, as many bytes as the weight's for each 16 rows,
// bounds it. fp32, one row at 32000 x 4096: 117 us, 4.5 TB/s (on fp32 tiles 526).
#include <float.h>
#include <math.h>

#include <type_traits>

#include "orda_kernels.h"
#include "row_terms.h"

namespace orda {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int kCols = 64;   // classes of a workgroup

__device__ __forceinline__ float quad_max(float x) {
  x = fmaxf(x, __shfl_xor(x, 16));
  return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float quad_sum(float x) {
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

// A lane's 16 bytes of a row, four lanes a fragment's K: 32 columns of bf16, or 16
// of fp32, multiplied four at a time (which of a lane's columns an instruction takes
// is the same for both operands).
template <typename E>
struct Vec;
template <>
struct Vec<__bf16> {
  typedef bf16x8 T;
  static __device__ __forceinline__ f32x4 mul(T b, T a, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(b, a, c, 0, 0, 0);
  }
};
template <>
struct Vec<float> {
  typedef f32x4 T;
  static __device__ __forceinline__ f32x4 mul(T b, T a, f32x4 c) {
#pragma unroll
    for (int k = 0; k < 4; ++k) c = __builtin_amdgcn_mfma_f32_16x16x4f32(b[k], a[k], c, 0, 0, 0);
    return c;
  }
};

template <typename E, int F, bool GRAD>
__global__ __launch_bounds__(256) void ce_few_kernel(CeFewArgs a) {
  using T = typename Vec<E>::T;
  constexpr int U = F == 1 ? 2 : 1;   // blocks in flight
  constexpr int kV = 16 / sizeof(E), kBlock = 16 * kV;
  constexpr bool kAllRows = GRAD && sizeof(E) == 4;   // the gradient's rows from the count on are zeros
  __shared__ float4 part[4][F * 16];
  const int m = static_cast<int>(*a.rows.count);
  if (m <= 0 && !kAllRows) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lrow = lane & 15, lgrp = lane >> 4;
  const int64_t n0 = blockIdx.x * static_cast<int64_t>(kCols) + wave * 16;
  f32x4 acc[F];
#pragma unroll
  for (int i = 0; i < F; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (n0 < a.cols && m > 0) {
    // rows and classes past the last: the last one again, not counted
    const E* pa[F];
#pragma unroll
    for (int i = 0; i < F; ++i)
      pa[i] = static_cast<const E*>(a.x) + (i * 16 + lrow < m ? i * 16 + lrow : m - 1) * a.ldx + lgrp * kV;
    const E* const pb = static_cast<const E*>(a.w) + (n0 + lrow < a.cols ? n0 + lrow : a.cols - 1) * a.ldw + lgrp * kV;
    struct Block {
      T a[F][4], b[4];
    };
    auto load = [&](Block& w, int64_t kb) {
#pragma unroll
      for (int q = 0; q < 4; ++q) __builtin_memcpy(&w.b[q], pb + kb * kBlock + q * 4 * kV, 16);
#pragma unroll
      for (int i = 0; i < F; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) w.a[i][q] = *reinterpret_cast<const T*>(pa[i] + kb * kBlock + q * 4 * kV);
    };
    auto use = [&](const Block& w) {
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int i = 0; i < F; ++i) acc[i] = Vec<E>::mul(w.b[q], w.a[i][q], acc[i]);
    };
    const int64_t nfull = a.k / kBlock;
    int64_t kb = 0;
    if (nfull >= 2 * U) {
      Block w[2][U];
#pragma unroll
      for (int u = 0; u < U; ++u) load(w[0][u], u);
      for (; kb + 3 * U <= nfull; kb += 2 * U) {
#pragma unroll
        for (int u = 0; u < U; ++u) load(w[1][u], kb + U + u);
#pragma unroll
        for (int u = 0; u < U; ++u) use(w[0][u]);
#pragma unroll
        for (int u = 0; u < U; ++u) load(w[0][u], kb + 2 * U + u < nfull ? kb + 2 * U + u : nfull - 1);
#pragma unroll
        for (int u = 0; u < U; ++u) use(w[1][u]);
      }
      // w[0] holds blocks kb .. kb + U - 1, where they exist
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (kb + u < nfull) use(w[0][u]);
      kb = kb + U < nfull ? kb + U : nfull;
    }
    for (; kb < nfull; ++kb) {
      Block w;
      load(w, kb);
      use(w);
    }
    if (nfull * kBlock < a.k) {   // the rest: zeros past k (in x up to whole vectors already)
      Block w;
      const T zero = {};
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int64_t c = nfull * kBlock + q * 4 * kV;
        const int64_t left = a.k - c - lgrp * kV;
        w.b[q] = zero;
        if (left >= kV) {
          __builtin_memcpy(&w.b[q], pb + c, 16);
        } else {
#pragma unroll
          for (int k = 0; k < kV; ++k)
            if (k < left) w.b[q][k] = pb[c + k];
        }
#pragma unroll
        for (int i = 0; i < F; ++i) {
          w.a[i][q] = zero;
          if (left > 0) w.a[i][q] = *reinterpret_cast<const T*>(pa[i] + c);
        }
      }
      use(w);
    }
  }
  // Lane: row i * 16 + lrow, classes n0 + 4 * lgrp + e.
  const int64_t col = n0 + 4 * lgrp, ncol = a.cols - col;
#pragma unroll
  for (int i = 0; i < F; ++i) {
    const int row = i * 16 + lrow;
    const f32x4 v = acc[i];
    const int64_t y = row < m ? a.rows.labels[row] - a.col0 - col : -1;   // among the lane's classes, or not
    if constexpr (GRAD) {
      const float4 c = row < m ? a.coef[row] : make_float4(0.f, 0.f, 0.f, 0.f);
      f32x4 d;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        d[e] = fmaf(c.y, __builtin_amdgcn_exp2f(fmaf(v[e], kLog2e, -c.x)), -c.z);
        if (e == y) d[e] -= c.w;
        d[e] = e < ncol && row < m ? d[e] : 0.f;
      }
      if constexpr (sizeof(E) == 2) {   // rounded for the matrix units, as on the tiles
        bf16x4 o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = static_cast<__bf16>(d[e]);
        if (row < m && col < (a.cols + 7) / 8 * 8)
          *reinterpret_cast<bf16x4*>(static_cast<__bf16*>(a.ds) + row * a.ldds + col) = o;
      } else if (row < a.n && col < a.cols) {
        *reinterpret_cast<f32x4*>(static_cast<float*>(a.ds) + row * a.ldds + col) = d;
      }
    } else {
      float mx = -INFINITY;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < ncol) mx = fmaxf(mx, v[e]);
      mx = quad_max(mx);
      // (an infinite maximum: the sum is that infinity or 0, without inf - inf)
      const float ref = fabsf(mx) <= kCeLargest ? mx : 0.f;
      float sum = 0.f, sx = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < ncol) {
          sum += __builtin_amdgcn_exp2f(fmaf(v[e], kLog2e, -ref * kLog2e));
          sx += v[e];
          if (e == y) a.xy[row] = v[e];
        }
      sum = quad_sum(sum);
      sx = quad_sum(sx);
      if (lgrp == 0) part[wave][row] = make_float4(mx < -kCeLargest ? -INFINITY : ref, sum, 0.f, sx);
    }
  }
  if constexpr (!GRAD) {
    __syncthreads();
    const int row = threadIdx.x;
    if (row >= F * 16 || row >= m) return;
    float top = -INFINITY, all = 0.f;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < 4; ++w) top = fmaxf(top, part[w][row].x);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float4 p = part[w][row];
      if (p.x != -INFINITY) s.y += p.y * __builtin_amdgcn_exp2f((p.x - top) * kLog2e);
      all += p.y;
      s.w += p.w;
    }
    s.x = top;
    if (!(all <= FLT_MAX)) s.y = all;   // an infinite or NaN sum stays one
    a.stats[row * a.stats_ld + blockIdx.x] = s;
  }
}

}  // namespace

int64_t ce_few_tiles(int64_t cols) { return (cols + kCols - 1) / kCols; }

hipError_t launch_ce_few(const CeFewArgs& a, DType t, bool grad, hipStream_t stream) {
  if (a.n <= 0 || a.cols <= 0) return hipSuccess;
  const int64_t es = dtype_size(t);
  if (a.n > kCeFewRows || a.ldx * es % 16 != 0 || (grad && a.ldds * es % 16 != 0) ||
      a.ldx < (a.k * es + 15) / 16 * 16 / es || reinterpret_cast<uintptr_t>(a.x) % 16 != 0)
    return hipErrorInvalidValue;
  using K = void (*)(CeFewArgs);
  auto pick = [&](auto e, auto g) -> K {
    using E = decltype(e);
    constexpr bool kGrad = decltype(g)::value;
    return a.n <= 16 ? ce_few_kernel<E, 1, kGrad> : a.n <= 32 ? ce_few_kernel<E, 2, kGrad> : ce_few_kernel<E, 4, kGrad>;
  };
  const K k = t == DType::BF16 ? (grad ? pick(__bf16{}, std::true_type{}) : pick(__bf16{}, std::false_type{}))
                               : (grad ? pick(float{}, std::true_type{}) : pick(float{}, std::false_type{}));
  hipLaunchKernelGGL(k, dim3(static_cast<unsigned>(ce_few_tiles(a.cols))), dim3(256), 0, stream, a);
  return hipGetLastError();
}

}  // namespace orda
