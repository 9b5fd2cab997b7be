// ce_rows.hip — the row kernels of the linear cross entropy that keeps no
// logits (its products run in gemm.hip with the CeStats and CeGrad epilogues).
//
// Rows whose label is ignore_index contribute nothing, so they are taken out
// first: the labelled rows' numbers and labels are compacted (their count stays
// on the device: the call waits for nothing and can be captured), their hidden
// rows gathered, and every product runs over those rows alone.
#include <float.h>
#include <math.h>

#include "orda_kernels.h"

namespace orda {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
constexpr float kLog2e = 1.4426950408889634f;

// ------------------------------------------------------------ compaction
// One workgroup walks the labels in order, 8 consecutive ones a thread and
// 8192 an iteration: counts within a thread, a prefix sum over the lanes of a
// wave and over the waves, then the stores. Bound by latency, a load and two
// barriers an iteration.
constexpr int kScanThreads = 1024, kScanPer = 8;

__global__ __launch_bounds__(kScanThreads) void ce_rows_kernel(const int64_t* labels, int64_t n, int64_t v,
                                                               int64_t ignore, CeRows r, float* nll, float* lse) {
  __shared__ int wave_sum[kScanThreads / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int64_t base = 0;
  for (int64_t i0 = 0; i0 < n; i0 += kScanThreads * kScanPer) {
    const int64_t first = i0 + tid * kScanPer;
    int64_t y[kScanPer];
    int mine = 0;
#pragma unroll
    for (int k = 0; k < kScanPer; ++k) {
      y[k] = first + k < n ? labels[first + k] : ignore;
      mine += y[k] != ignore ? 1 : 0;
    }
    int incl = mine;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int t = __shfl_up(incl, d);
      if (lane >= d) incl += t;
    }
    if (lane == 63) wave_sum[wave] = incl;
    __syncthreads();
    int before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < kScanThreads / 64; ++w) {
      const int s = wave_sum[w];
      before += w < wave ? s : 0;
      total += s;
    }
    __syncthreads();
    int64_t at = base + before + incl - mine;
#pragma unroll
    for (int k = 0; k < kScanPer; ++k) {
      const int64_t i = first + k;
      if (i >= n) continue;
      if (y[k] != ignore) {
        r.src[at] = static_cast<int32_t>(i);
        r.labels[at] = y[k] >= 0 && y[k] < v ? y[k] : -1;
        r.pos[i] = static_cast<int32_t>(at++);
      } else {
        r.pos[i] = -1;
        if (nll != nullptr) nll[i] = 0.f, lse[i] = 0.f;
      }
    }
    base += total;
  }
  if (tid == 0) *r.count = base;
}

// ------------------------------------------------------------ hidden rows
// A wave copies a row to its compact place: 16-byte vectors where the source
// allows, zeros up to the pitch, and zero rows from the count up to the next
// multiple of 64 (finite values beside the zeros of the backward products). With
// coef, the row's CeGrad coefficients too (CeArgs::coef).
template <typename E, bool VEC>
__global__ __launch_bounds__(256) void ce_gather_kernel(const E* x, int64_t ldx, int64_t h, CeRows r, E* dst,
                                                        int64_t ldd, CeGradRows g) {
  const int lane = threadIdx.x & 63;
  const int64_t row = blockIdx.x * int64_t{4} + (threadIdx.x >> 6);
  const int64_t n = *r.count;
  if (row >= (n + 63) / 64 * 64) return;
  E* d = dst + row * ldd;
  constexpr int kVec = 16 / sizeof(E);
  const int64_t i = row < n ? r.src[row] : 0;
  const E* s = x + i * ldx;
  for (int64_t c = lane * kVec; c < ldd; c += 64 * kVec) {
    alignas(16) E w[kVec] = {};
    if (row < n) {
      if (VEC && c + kVec <= h) {
        *reinterpret_cast<u32x4*>(w) = *reinterpret_cast<const u32x4*>(s + c);
      } else {
#pragma unroll
        for (int k = 0; k < kVec; ++k)
          if (c + k < h) w[k] = s[c + k];
      }
    }
    *reinterpret_cast<u32x4*>(d + c) = *reinterpret_cast<const u32x4*>(w);
  }
  if (g.coef != nullptr && lane == 0 && row < n) {
    const float gn = g.grad_nll != nullptr ? g.grad_nll[i] : 0.f, gl = g.grad_lse != nullptr ? g.grad_lse[i] : 0.f;
    float4 c = make_float4(g.lse[i] * kLog2e, gn + gl, gn * g.smooth_each, gn * g.target);
    if (r.labels[row] < 0) c = make_float4(NAN, NAN, NAN, NAN);   // no such class
    g.coef[row] = c;
  }
}

// ------------------------------------------------------------ losses
// A wave merges a row's tile statistics, the maximum first and then the sums
// relative to it (the second read comes from the cache), and on the last piece
// of the vocabulary forms the row's loss. An infinite or NaN sum goes past the
// scaling as it is.
__global__ __launch_bounds__(256) void ce_losses_kernel(CeLossArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t row = blockIdx.x * int64_t{4} + (threadIdx.x >> 6);
  if (row >= *a.rows.count) return;
  const float4* st = a.stats + row * a.stats_ld;
  float4 old = make_float4(-INFINITY, 0.f, 0.f, 0.f);   // {max, sum, sum of logits, infinite sums}
  if (!a.first) old = a.state[row];
  float m = old.x;
  for (int64_t t = lane; t < a.tiles; t += 64) m = fmaxf(m, st[t].x);
#pragma unroll
  for (int d = 32; d > 0; d /= 2) m = fmaxf(m, __shfl_xor(m, d));
  float sum = 0.f, sx = 0.f, ext = 0.f;
  for (int64_t t = lane; t < a.tiles; t += 64) {
    const float4 s = st[t];
    sx += s.z;
    if (!(s.y <= FLT_MAX)) ext += s.y;
    else if (s.x != -INFINITY) sum += s.y * __builtin_amdgcn_exp2f((s.x - m) * kLog2e);
  }
#pragma unroll
  for (int d = 32; d > 0; d /= 2) {
    sum += __shfl_xor(sum, d);
    sx += __shfl_xor(sx, d);
    ext += __shfl_xor(ext, d);
  }
  if (lane != 0) return;
  if (old.x != -INFINITY) sum += old.y * __builtin_amdgcn_exp2f((old.x - m) * kLog2e);
  sx += old.z;
  ext += old.w;
  if (!a.last) {
    a.state[row] = make_float4(m, sum, sx, ext);
    return;
  }
  const float l = ext != 0.f ? ext : m == -INFINITY ? m : m + logf(sum);
  const int64_t i = a.rows.src[row];
  a.lse[i] = l;
  float nll = NAN;
  if (a.rows.labels[row] >= 0) {
    nll = l - a.target * a.xy[row];
    if (a.smooth_each != 0.f) nll -= a.smooth_each * sx;
  }
  a.nll[i] = nll;
}

// ------------------------------------------------------------ grad_hidden
// The compact fp32 gradient rows to their places in the output's type; rows
// without a label (with pos null: all) are zero.
template <typename O, bool VEC>
__global__ __launch_bounds__(256) void ce_scatter_kernel(const float* src, int64_t lds, const int32_t* pos,
                                                         int64_t rows, int64_t h, O* dst, int64_t ldd) {
  const int lane = threadIdx.x & 63;
  const int64_t row = blockIdx.x * int64_t{4} + (threadIdx.x >> 6);
  if (row >= rows) return;
  const int64_t p = pos != nullptr ? pos[row] : -1;
  const float* s = src + (p < 0 ? 0 : p) * lds;
  O* d = dst + row * ldd;
  for (int64_t c = lane * 4; c < h; c += 256) {
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
    if (p >= 0) x = *reinterpret_cast<const f32x4*>(s + c);   // lds is a multiple of 4, >= h
    if (VEC && c + 4 <= h) {
      alignas(16) O o[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) o[k] = static_cast<O>(x[k]);
      if constexpr (sizeof(O) == 4) *reinterpret_cast<u32x4*>(d + c) = *reinterpret_cast<const u32x4*>(o);
      else *reinterpret_cast<uint64_t*>(d + c) = *reinterpret_cast<const uint64_t*>(o);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (c + k < h) d[c + k] = static_cast<O>(x[k]);
    }
  }
}

unsigned row_blocks(int64_t rows) { return static_cast<unsigned>((rows + 3) / 4); }

}  // namespace

hipError_t launch_ce_rows(const int64_t* labels, int64_t n, int64_t v, int64_t ignore, const CeRows& r, float* nll,
                          float* lse, hipStream_t stream) {
  hipLaunchKernelGGL(ce_rows_kernel, dim3(1), dim3(kScanThreads), 0, stream, labels, n, v, ignore, r, nll, lse);
  return hipGetLastError();
}

hipError_t launch_ce_gather(DType t, const void* x, int64_t ldx, int64_t n, int64_t h, const CeRows& r, void* dst,
                            int64_t ldd, const CeGradRows& g, hipStream_t stream) {
  if (ldd % 8 != 0 || ldd < h || reinterpret_cast<uintptr_t>(dst) % 16 != 0) return hipErrorInvalidValue;
  const dim3 grid(row_blocks((n + 63) / 64 * 64));
  const bool vec = (ldx * dtype_size(t)) % 16 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0;
  auto run = [&](auto kernel, auto* e) {
    using E = std::remove_pointer_t<decltype(e)>;
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, stream, static_cast<const E*>(x), ldx, h, r, static_cast<E*>(dst),
                       ldd, g);
  };
  if (t == DType::BF16) {
    uint16_t* e = nullptr;
    if (vec) run(ce_gather_kernel<uint16_t, true>, e);
    else run(ce_gather_kernel<uint16_t, false>, e);
  } else {
    uint32_t* e = nullptr;
    if (vec) run(ce_gather_kernel<uint32_t, true>, e);
    else run(ce_gather_kernel<uint32_t, false>, e);
  }
  return hipGetLastError();
}

hipError_t launch_ce_losses(const CeLossArgs& a, int64_t n, hipStream_t stream) {
  hipLaunchKernelGGL(ce_losses_kernel, dim3(row_blocks(n)), dim3(256), 0, stream, a);
  return hipGetLastError();
}

hipError_t launch_ce_scatter(const float* src, int64_t lds, const int32_t* pos, int64_t rows, int64_t h, DType t,
                             void* dst, int64_t ldd, hipStream_t stream) {
  if (lds % 4 != 0 || reinterpret_cast<uintptr_t>(src) % 16 != 0) return hipErrorInvalidValue;
  const int64_t align = 4 * dtype_size(t);
  const bool vec = (ldd * dtype_size(t)) % align == 0 && reinterpret_cast<uintptr_t>(dst) % align == 0;
  const dim3 grid(row_blocks(rows));
  if (t == DType::BF16) {
    auto* d = static_cast<__bf16*>(dst);
    if (vec) hipLaunchKernelGGL((ce_scatter_kernel<__bf16, true>), grid, dim3(256), 0, stream, src, lds, pos, rows, h, d, ldd);
    else hipLaunchKernelGGL((ce_scatter_kernel<__bf16, false>), grid, dim3(256), 0, stream, src, lds, pos, rows, h, d, ldd);
  } else {
    auto* d = static_cast<float*>(dst);
    if (vec) hipLaunchKernelGGL((ce_scatter_kernel<float, true>), grid, dim3(256), 0, stream, src, lds, pos, rows, h, d, ldd);
    else hipLaunchKernelGGL((ce_scatter_kernel<float, false>), grid, dim3(256), 0, stream, src, lds, pos, rows, h, d, ldd);
  }
  return hipGetLastError();
}

}  // namespace orda
