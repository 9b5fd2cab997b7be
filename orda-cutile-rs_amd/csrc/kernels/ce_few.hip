// ce_few.hip — the logits of a few rows for the linear cross entropy: a token or a
// small batch against the whole vocabulary, in bf16.
//
// Bound by the weight's bytes, which each go once from memory to the registers of
// one wave, with no LDS and no barrier before the end. A wave takes 16 classes and
// all rows (F fragments of 16, from the caches) and loads the next 128 columns, or
// two times 128, while it multiplies these; the workgroup's 64 classes are one tile
// of statistics. A tile of the large product holds 256 classes, so that 14000
// classes are 56 workgroups on 256 CUs. One row at 32000 x 2048: 23 us, 5.8 TB/s (on
// the tiles 41); 18 rows at 14334 x 4032 31 us, 3.7 TB/s (75), where the rows' way
// from the second-level caches, as many bytes as the weight's for each 16 rows,
// bounds it.
#include <float.h>
#include <math.h>

#include "orda_kernels.h"
#include "row_terms.h"

namespace orda {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
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

template <int F, bool GRAD>
__global__ __launch_bounds__(256) void ce_few_kernel(CeFewArgs a) {
  constexpr int U = F == 1 ? 2 : 1;   // blocks of 128 columns in flight
  __shared__ float4 part[4][F * 16];
  const int m = static_cast<int>(*a.rows.count);
  if (m <= 0) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lrow = lane & 15, lgrp = lane >> 4;
  const int64_t n0 = blockIdx.x * static_cast<int64_t>(kCols) + wave * 16;
  f32x4 acc[F];
#pragma unroll
  for (int i = 0; i < F; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (n0 < a.cols) {
    // rows and classes past the last: the last one again, not counted
    const __bf16* pa[F];
#pragma unroll
    for (int i = 0; i < F; ++i)
      pa[i] = static_cast<const __bf16*>(a.x) + (i * 16 + lrow < m ? i * 16 + lrow : m - 1) * a.ldx + lgrp * 8;
    const __bf16* const pb = static_cast<const __bf16*>(a.w) + (n0 + lrow < a.cols ? n0 + lrow : a.cols - 1) * a.ldw + lgrp * 8;
    struct Block {
      bf16x8 a[F][4], b[4];
    };
    auto load = [&](Block& w, int64_t kb) {
#pragma unroll
      for (int q = 0; q < 4; ++q) w.b[q] = *reinterpret_cast<const bf16x8*>(pb + kb * 128 + q * 32);
#pragma unroll
      for (int i = 0; i < F; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) w.a[i][q] = *reinterpret_cast<const bf16x8*>(pa[i] + kb * 128 + q * 32);
    };
    auto use = [&](const Block& w) {
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int i = 0; i < F; ++i) acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w.b[q], w.a[i][q], acc[i], 0, 0, 0);
    };
    const int64_t nfull = a.k / 128;
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
    if (nfull * 128 < a.k) {   // k is a multiple of 8: vectors from there on are zeros
      Block w;
      const bf16x8 zero = {};
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int64_t c = nfull * 128 + q * 32;
        const bool in = c + lgrp * 8 < a.k;
        w.b[q] = zero;
        if (in) w.b[q] = *reinterpret_cast<const bf16x8*>(pb + c);
#pragma unroll
        for (int i = 0; i < F; ++i) {
          w.a[i][q] = zero;
          if (in) w.a[i][q] = *reinterpret_cast<const bf16x8*>(pa[i] + c);
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
      bf16x4 o;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float d = fmaf(c.y, __builtin_amdgcn_exp2f(fmaf(v[e], kLog2e, -c.x)), -c.z);
        if (e == y) d -= c.w;
        o[e] = static_cast<__bf16>(e < ncol ? d : 0.f);   // rounded for the matrix units, as on the tiles
      }
      if (row < m && col < (a.cols + 7) / 8 * 8)
        *reinterpret_cast<bf16x4*>(static_cast<__bf16*>(a.ds) + row * a.ldds + col) = o;
    } else {
      float mx = -INFINITY;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < ncol) mx = fmaxf(mx, v[e]);
      mx = quad_max(mx);
      // (an infinite maximum: the sum is that infinity or 0, without inf - inf)
      const float ref = fabsf(mx) <= FLT_MAX ? mx : 0.f;
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
      if (lgrp == 0) part[wave][row] = make_float4(mx == -INFINITY ? mx : ref, sum, 0.f, sx);
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

hipError_t launch_ce_few(const CeFewArgs& a, int64_t n, bool grad, hipStream_t stream) {
  if (n <= 0 || a.cols <= 0) return hipSuccess;
  if (n > kCeFewRows || a.k % 8 != 0 || a.ldx % 8 != 0 || a.ldw % 8 != 0 || (grad && a.ldds % 8 != 0) ||
      reinterpret_cast<uintptr_t>(a.x) % 16 != 0 || reinterpret_cast<uintptr_t>(a.w) % 16 != 0)
    return hipErrorInvalidValue;
  using K = void (*)(CeFewArgs);
  const K k = n <= 16   ? (grad ? static_cast<K>(ce_few_kernel<1, true>) : ce_few_kernel<1, false>)
              : n <= 32 ? (grad ? static_cast<K>(ce_few_kernel<2, true>) : ce_few_kernel<2, false>)
                        : (grad ? static_cast<K>(ce_few_kernel<4, true>) : ce_few_kernel<4, false>);
  hipLaunchKernelGGL(k, dim3(static_cast<unsigned>(ce_few_tiles(a.cols))), dim3(256), 0, stream, a);
  return hipGetLastError();
}

}  // namespace orda
