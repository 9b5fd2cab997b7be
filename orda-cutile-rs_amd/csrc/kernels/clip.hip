// clip.hip — the norm of many gradients together, and their scaling to a limit.
//
// n = sqrt(Σ g²), then g·min(1, max_norm / (n + eps)). Squares and sums are held in
// 64 bits: the square of an fp32 or bf16 value is exact there, and neither a large
// gradient overflows nor a small one vanishes. The gradients travel in the
// launches' arguments, so that nothing is copied to the device and a captured graph
// holds them. Bound by HBM: one read for the norm, and where it is over the limit
// another read and a write.
#include <math.h>

#include "orda_kernels.h"
#include "wave.h"

namespace orda {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ double block_sum(double x, double* part) {
  x = wave_sum(x);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
  __syncthreads();
  x = 0.;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) x += part[w];
  return x;
}

// Piece i: its gradient, and where it begins and how many values it has.
struct Piece {
  int part;
  int64_t row, col, n;
};
__device__ __forceinline__ Piece piece_of(const GradArgs& a, int64_t i) {
  int lo = 0, hi = a.count - 1;   // the last part whose first piece is not after i
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (a.part[mid].first <= i) lo = mid;
    else hi = mid - 1;
  }
  const GradPart& p = a.part[lo];
  const int64_t across = (p.cols + a.piece - 1) / a.piece, k = i - p.first;
  const int64_t row = p.rows == 1 ? 0 : k / across, col = (k - row * across) * a.piece;
  return {lo, row, col, p.cols - col < a.piece ? p.cols - col : a.piece};
}

template <typename E>
__device__ __forceinline__ double squares(const E* p, int64_t n) {
  double s = 0.;
  const int64_t whole = n / 8 * 8;
  for (int64_t c = threadIdx.x * int64_t{8}; c < whole; c += kThreads * 8) {
    E v[8];
    __builtin_memcpy(v, p + c, sizeof v);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const double x = static_cast<float>(v[k]);
      s = fma(x, x, s);
    }
  }
  const int64_t c = whole + threadIdx.x;
  if (c < n) {
    const double x = static_cast<float>(p[c]);
    s = fma(x, x, s);
  }
  return s;
}

__global__ __launch_bounds__(kThreads) void grad_sums_kernel(GradArgs a) {
  __shared__ double part[kThreads / 64];
  double s = 0.;
  for (int64_t i = blockIdx.x; i < a.pieces; i += gridDim.x) {
    const Piece q = piece_of(a, i);
    const GradPart& p = a.part[q.part];
    const int64_t at = q.row * p.lds + q.col;
    s += p.src_bf16 ? squares(static_cast<const __bf16*>(p.src) + at, q.n)
                    : squares(static_cast<const float*>(p.src) + at, q.n);
  }
  s = block_sum(s, part);
  if (threadIdx.x == 0) a.sums[blockIdx.x] = s;
}

__device__ __forceinline__ double total(const double* sums, int n, double* part) {
  double s = 0.;
  for (int i = threadIdx.x; i < n; i += kThreads) s += sums[i];
  return block_sum(s, part);
}

template <typename S, typename D>
__device__ __forceinline__ void scaled(const S* s, D* d, int64_t n, float f) {
  const int64_t whole = n / 8 * 8;
  for (int64_t c = threadIdx.x * int64_t{8}; c < whole; c += kThreads * 8) {
    S v[8];
    D o[8];
    __builtin_memcpy(v, s + c, sizeof v);
#pragma unroll
    for (int k = 0; k < 8; ++k) o[k] = static_cast<D>(static_cast<float>(v[k]) * f);
    __builtin_memcpy(d + c, o, sizeof o);
  }
  const int64_t c = whole + threadIdx.x;
  if (c < n) d[c] = static_cast<D>(static_cast<float>(s[c]) * f);
}

__global__ __launch_bounds__(kThreads) void grad_scale_kernel(GradArgs a) {
  __shared__ double part[kThreads / 64];
  const double n = sqrt(total(a.all, a.n_sums, part));
  if (a.norm && blockIdx.x == 0 && threadIdx.x == 0) *a.norm = static_cast<float>(n);
  const double f64 = a.max_norm / (n + a.eps);
  const float f = f64 >= 1. ? 1.f : static_cast<float>(f64);   // (a NaN stays one)
  if (a.in_place && f == 1.f) return;
  for (int64_t i = blockIdx.x; i < a.pieces; i += gridDim.x) {
    const Piece q = piece_of(a, i);
    const GradPart& p = a.part[q.part];
    const int64_t at = q.row * p.lds + q.col, to = q.row * p.ldd + q.col;
    if (p.src_bf16) {
      const __bf16* s = static_cast<const __bf16*>(p.src) + at;
      if (p.dst_bf16) scaled(s, static_cast<__bf16*>(p.dst) + to, q.n, f);
      else scaled(s, static_cast<float*>(p.dst) + to, q.n, f);
    } else {
      const float* s = static_cast<const float*>(p.src) + at;
      if (p.dst_bf16) scaled(s, static_cast<__bf16*>(p.dst) + to, q.n, f);
      else scaled(s, static_cast<float*>(p.dst) + to, q.n, f);
    }
  }
}

__global__ __launch_bounds__(kThreads) void grad_norm_kernel(const double* sums, int n, float* norm) {
  __shared__ double part[kThreads / 64];
  const double s = total(sums, n, part);
  if (threadIdx.x == 0) *norm = static_cast<float>(sqrt(s));
}

}  // namespace

hipError_t launch_grad_sums(const GradArgs& a, int blocks, hipStream_t stream) {
  hipLaunchKernelGGL(grad_sums_kernel, dim3(blocks), dim3(kThreads), 0, stream, a);
  return hipGetLastError();
}

hipError_t launch_grad_scale(const GradArgs& a, int blocks, hipStream_t stream) {
  hipLaunchKernelGGL(grad_scale_kernel, dim3(blocks), dim3(kThreads), 0, stream, a);
  return hipGetLastError();
}

hipError_t launch_grad_norm(const double* sums, int n, float* norm, hipStream_t stream) {
  hipLaunchKernelGGL(grad_norm_kernel, dim3(1), dim3(kThreads), 0, stream, sums, n, norm);
  return hipGetLastError();
}

}  // namespace orda
