// clip.hip — the norm of many gradients together, and their scaling to a limit.
//
// n = sqrt(Σ g²), then g·min(1, max_norm / (n + eps)). Squares and sums are held in
// 64 bits: the square of an fp32 or bf16 value is exact there, and neither a large
// gradient overflows nor a small one vanishes. The gradients travel in the
// launches' arguments, so that nothing is copied to the device and a captured graph
// holds them. Bound by HBM: one read for the norm, and where it is over the limit
// another read and a write. 4.29 GB of fp32: 613 us (7.0 TB/s) and 1640 (5.2 both ways; a
// copy reaches 4.8); 1.05 GB of bf16 in 110 tensors at any address, two launches: 181 (5.8;
// 208 before the loads began at whole 16 bytes).
//
// The gradients' values are one row of pieces, of which each workgroup has an equal run:
// with whole tensors or a piece at a time the last ones left the others waiting.
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

// A run of values of one row, which begins `at` values (`to` in the destination) from
// its gradient's first.
struct Run {
  int part;
  int64_t at, to, n, pieces;
};
__device__ __forceinline__ int part_of(const GradArgs& a, int64_t i) {
  int lo = 0, hi = a.count - 1;   // the last part whose first piece is not after i
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (a.part[mid].first <= i) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}
// The last run of the pieces from `from` to `to`, which is after `from`.
__device__ __forceinline__ Run last_run(const GradArgs& a, int64_t from, int64_t to) {
  const int k = part_of(a, to - 1);
  const GradPart& p = a.part[k];
  const int64_t across = (p.cols + kGradPiece - 1) / kGradPiece, i = to - 1 - p.first;
  const int64_t row = p.rows == 1 ? 0 : i / across, begin = p.first + row * across;
  const int64_t first = from > begin ? from : begin, col = (first - begin) * kGradPiece;
  const int64_t end = (to - begin) * kGradPiece;
  return {k, row * p.lds + col, row * p.ldd + col, (p.cols < end ? p.cols : end) - col, to - first};
}

// 16 bytes at any address. ONCE: past the caches.
template <bool ONCE, typename E, int N>
__device__ __forceinline__ void take(E (&v)[N], const E* p) {
  typedef uint32_t Words __attribute__((ext_vector_type(4), aligned(2)));
  static_assert(sizeof v == sizeof(Words));
  Words w;
  if constexpr (ONCE) w = __builtin_nontemporal_load(reinterpret_cast<const Words*>(p));
  else __builtin_memcpy(&w, p, sizeof w);
  __builtin_memcpy(v, &w, sizeof v);
}

// Values before the first that lies at 16 bytes, of n.
template <typename E>
__device__ __forceinline__ int64_t to_aligned(const E* p, int64_t n) {
  const int64_t k = (16 - reinterpret_cast<uintptr_t>(p) % 16) % 16 / sizeof(E);
  return k < n ? k : n;
}

// Loads that a thread has under way: 64 bytes of fp32 (4.29 GB past the caches: 612 us,
// 640 with 32) or 32 of bf16, whose values take twice the registers (1.05 GB: 180 us, 188
// with 64).
template <typename E>
constexpr int kAhead = sizeof(E) == 4 ? 4 : 2;

template <bool ONCE, typename E>
__device__ __forceinline__ double squares(const E* p, int64_t n) {
  constexpr int N = 16 / sizeof(E), kStep = kThreads * N, kU = kAhead<E>;
  double s[kU] = {};
  auto add = [](double& s, float v) { s = fma(static_cast<double>(v), static_cast<double>(v), s); };
  const int64_t first = to_aligned(p, n);
  if (threadIdx.x < first) add(s[1], p[threadIdx.x]);
  p += first;
  n -= first;
  const int64_t whole = n / N * N;
  int64_t c = threadIdx.x * int64_t{N};
  for (; c + (kU - 1) * kStep < whole; c += kU * kStep) {
    E v[kU][N];
#pragma unroll
    for (int u = 0; u < kU; ++u) take<ONCE>(v[u], p + c + u * kStep);
#pragma unroll
    for (int u = 0; u < kU; ++u)
#pragma unroll
      for (int k = 0; k < N; ++k) add(s[u], v[u][k]);
  }
  for (; c < whole; c += kStep) {
    E v[N];
    take<ONCE>(v, p + c);
#pragma unroll
    for (int k = 0; k < N; ++k) add(s[0], v[k]);
  }
  c = whole + threadIdx.x;
  if (c < n) add(s[1], p[c]);
#pragma unroll
  for (int u = 1; u < kU; ++u) s[0] += s[u];
  return s[0];
}

// The pieces from which and to which this workgroup's are.
__device__ __forceinline__ int64_t share(const GradArgs& a, int64_t block) { return a.pieces * block / gridDim.x; }

// ONCE: gradients that the cache will not hold until they are scaled.
template <bool ONCE>
__global__ __launch_bounds__(kThreads) void grad_sums_kernel(GradArgs a) {
  __shared__ double part[kThreads / 64];
  double s = 0.;
  const int64_t from = share(a, blockIdx.x);
  for (int64_t to = share(a, blockIdx.x + 1); to > from;) {
    const Run r = last_run(a, from, to);
    const GradPart& p = a.part[r.part];
    s += p.src_bf16 ? squares<ONCE>(static_cast<const __bf16*>(p.src) + r.at, r.n)
                    : squares<ONCE>(static_cast<const float*>(p.src) + r.at, r.n);
    to -= r.pieces;
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
  constexpr int N = 16 / sizeof(S), kStep = kThreads * N, kU = 4;
  auto put = [&](int64_t c, const S (&v)[N]) {
    D o[N];
#pragma unroll
    for (int k = 0; k < N; ++k) o[k] = static_cast<D>(static_cast<float>(v[k]) * f);
    __builtin_memcpy(d + c, o, sizeof o);
  };
  const int64_t first = to_aligned(s, n);
  if (threadIdx.x < first) d[threadIdx.x] = static_cast<D>(static_cast<float>(s[threadIdx.x]) * f);
  s += first;
  d += first;
  n -= first;
  const int64_t whole = n / N * N;
  int64_t c = threadIdx.x * int64_t{N};
  for (; c + (kU - 1) * kStep < whole; c += kU * kStep) {
    S v[kU][N];
#pragma unroll
    for (int u = 0; u < kU; ++u) take<false>(v[u], s + c + u * kStep);
#pragma unroll
    for (int u = 0; u < kU; ++u) put(c + u * kStep, v[u]);
  }
  for (; c < whole; c += kStep) {
    S v[N];
    take<false>(v, s + c);
    put(c, v);
  }
  c = whole + threadIdx.x;
  if (c < n) d[c] = static_cast<D>(static_cast<float>(s[c]) * f);
}

__global__ __launch_bounds__(kThreads) void grad_scale_kernel(GradArgs a) {
  __shared__ double part[kThreads / 64];
  const double n = sqrt(total(a.all, a.n_sums, part));
  if (a.norm && blockIdx.x == 0 && threadIdx.x == 0) *a.norm = static_cast<float>(n);
  // (1 too where both are 0 or both infinite; a NaN stays one)
  const float f = n + a.eps <= a.max_norm ? 1.f : static_cast<float>(a.max_norm / (n + a.eps));
  if (a.in_place && f == 1.f) return;
  const int64_t from = share(a, blockIdx.x);
  for (int64_t to = share(a, blockIdx.x + 1); to > from;) {
    const Run r = last_run(a, from, to);
    const GradPart& p = a.part[r.part];
    if (p.src_bf16) {
      const __bf16* s = static_cast<const __bf16*>(p.src) + r.at;
      if (p.dst_bf16) scaled(s, static_cast<__bf16*>(p.dst) + r.to, r.n, f);
      else scaled(s, static_cast<float*>(p.dst) + r.to, r.n, f);
    } else {
      const float* s = static_cast<const float*>(p.src) + r.at;
      if (p.dst_bf16) scaled(s, static_cast<__bf16*>(p.dst) + r.to, r.n, f);
      else scaled(s, static_cast<float*>(p.dst) + r.to, r.n, f);
    }
    to -= r.pieces;
  }
}

__global__ __launch_bounds__(kThreads) void grad_norm_kernel(const double* sums, int n, float* norm) {
  __shared__ double part[kThreads / 64];
  const double s = total(sums, n, part);
  if (threadIdx.x == 0) *norm = static_cast<float>(sqrt(s));
}

}  // namespace

hipError_t launch_grad_sums(const GradArgs& a, int blocks, bool once, hipStream_t stream) {
  hipLaunchKernelGGL(once ? grad_sums_kernel<true> : grad_sums_kernel<false>, dim3(blocks), dim3(kThreads), 0, stream, a);
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
