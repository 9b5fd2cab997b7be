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
#include "split3.h"

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
constexpr int64_t kScanRows = 16384;   // up to here each workgroup of ce_prep_kernel counts for itself

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
// A workgroup takes 64 rows of the batch and CePrepArgs::cols of their columns, and
// writes what the products read of those that have a label, at their compact
// places: the rows (a pitch of whole vectors, zeros past h), and for the backward
// products the transposed rows, which pass through LDS 64 x 64 at a time. OUT 0
// keeps the type, OUT 1 writes fp32 values as three bf16 planes (split3.h). The
// workgroups of the last 64 rows also write the zeros up to the next multiple of 64
// (finite values beside the zeros of the backward products), those of the first
// columns the rows' numbers, classes, losses of ignored rows and coefficients.
//
// SCAN: the places are counted here, from all labels before (a batch of up to
// kScanRows: 4 us at 8192, where a kernel of its own takes 13 and a launch), else
// read from pos, which ce_rows_kernel has written.
//
// cols: 64 while that makes at most 2048 workgroups (1000 x 1536, both directions:
// 8 + 12 us, of 256 columns 15 + 24), then up to 256 (8192 x 4096, forward: 28 us,
// of 64 columns 48, as each workgroup counts for itself).
constexpr int kMinPrepCols = 64, kMaxPrepCols = 256;

template <typename E, int OUT, bool VEC, bool SCAN>
__global__ __launch_bounds__(256) void ce_prep_kernel(CePrepArgs a) {
  constexpr int kVec = 16 / sizeof(E), kLanes = 64 / kVec, kPass = 256 / kLanes;   // rows a pass
  __shared__ int place[64];
  __shared__ int sums[4];
  __shared__ E tile[64][65];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t r0 = static_cast<int64_t>(blockIdx.x) * 64, first = static_cast<int64_t>(blockIdx.y) * a.cols;
  const CeRows& r = a.rows;
  const bool lead = blockIdx.y == 0, last_rows = r0 + 64 >= a.n;
  int64_t base = 0;   // labelled rows before r0
  if constexpr (SCAN) {
    int mine = 0;
    for (int64_t i = tid * 8; i < r0; i += 2048) {   // r0 is a multiple of 64
#pragma unroll
      for (int k = 0; k < 8; ++k) mine += a.labels[i + k] != a.ignore ? 1 : 0;
    }
#pragma unroll
    for (int d = 32; d > 0; d /= 2) mine += __shfl_xor(mine, d);
    if (lane == 0) sums[wave] = mine;
    __syncthreads();
    base = sums[0] + sums[1] + sums[2] + sums[3];
  }
  if (wave == 0) {
    const int64_t i = r0 + lane;
    const int64_t y = i < a.n ? a.labels[i] : a.ignore;
    int p = -1;
    if constexpr (SCAN) {
      const uint64_t has = __ballot(y != a.ignore);
      if (y != a.ignore) p = static_cast<int>(base) + __popcll(has & ((uint64_t{1} << lane) - 1));
      if (lead && last_rows && lane == 0) *r.count = base + __popcll(has);
      if (lead && i < a.n) {
        r.pos[i] = p;
        if (p >= 0) {
          r.src[p] = static_cast<int32_t>(i);
          r.labels[p] = y >= 0 && y < a.v ? y : -1;
        } else if (a.nll != nullptr) {
          a.nll[i] = 0.f;
          a.lse_out[i] = 0.f;
        }
      }
    } else {
      if (i < a.n) p = r.pos[i];
    }
    if (lead && a.grad.coef != nullptr && p >= 0) {
      const CeGradRows& g = a.grad;
      const float gn = g.grad_nll != nullptr ? g.grad_nll[i] : 0.f, gl = g.grad_lse != nullptr ? g.grad_lse[i] : 0.f;
      float4 c = make_float4(g.lse[i] * kLog2e, gn + gl, gn * g.smooth_each, gn * g.target);
      if (y < 0 || y >= a.v) c = make_float4(NAN, NAN, NAN, NAN);   // no such class
      g.coef[p] = c;
    }
    place[lane] = p;
  }
  __syncthreads();
  const E* const x = static_cast<const E*>(a.x);
  const int row_in = tid / kLanes, col_in = tid % kLanes * kVec;
  for (int64_t c0 = first; c0 < first + a.cols && c0 < a.pitch; c0 += 64) {
#pragma unroll
    for (int q = 0; q < 64 / kPass; ++q) {
      const int rl = q * kPass + row_in, p = place[rl];
      const int64_t i = r0 + rl, c = c0 + col_in;
      alignas(16) E w[kVec] = {};
      if (p >= 0) {
        const E* src = x + i * a.ldx + c;
        if (VEC && c + kVec <= a.h) {
          *reinterpret_cast<u32x4*>(w) = *reinterpret_cast<const u32x4*>(src);
        } else {
#pragma unroll
          for (int k = 0; k < kVec; ++k)
            if (c + k < a.h) w[k] = src[k];
        }
        if (a.dst != nullptr && c < a.pitch) {
          if constexpr (OUT == 0) {
            *reinterpret_cast<u32x4*>(static_cast<E*>(a.dst) + p * a.pitch + c) = *reinterpret_cast<const u32x4*>(w);
          } else {
            uint32_t lo[3], hi[3];
            split3_pack(w[0], w[1], lo);
            split3_pack(w[2], w[3], hi);
            uint16_t* d = static_cast<uint16_t*>(a.dst) + 3 * p * a.pitch + c;
#pragma unroll
            for (int k = 0; k < 3; ++k) *reinterpret_cast<uint2*>(d + k * a.pitch) = make_uint2(lo[k], hi[k]);
          }
        }
      } else if (a.zero != nullptr && i < a.n && c < a.h) {   // an ignored row's gradient
        E* d = static_cast<E*>(a.zero) + i * a.ldz + c;
        if (a.zero_vec && c + kVec <= a.h) {
          *reinterpret_cast<u32x4*>(d) = u32x4{0, 0, 0, 0};
        } else {
#pragma unroll
          for (int k = 0; k < kVec; ++k)
            if (c + k < a.h) d[k] = E(0);
        }
      }
      if (a.trans != nullptr) {
#pragma unroll
        for (int k = 0; k < kVec; ++k) tile[rl][col_in + k] = w[k];
      }
    }
    if (a.trans == nullptr) continue;
    __syncthreads();
    const int p = place[lane];
    for (int q = wave; q < 64; q += 4) {
      const int64_t c = c0 + q;
      if (c >= a.h || p < 0) continue;
      const E e = tile[lane][q];
      if constexpr (OUT == 0) {
        static_cast<E*>(a.trans)[c * a.ldt + p] = e;
      } else {
        float h, m, l;
        split3(e, h, m, l);
        __bf16* d = static_cast<__bf16*>(a.trans) + 3 * c * a.ldt + p;
        d[0] = static_cast<__bf16>(h);
        d[a.ldt] = static_cast<__bf16>(m);
        d[2 * a.ldt] = static_cast<__bf16>(l);
      }
    }
    __syncthreads();
  }
  if (!last_rows) return;
  // zeros from the count up
  const int64_t n = SCAN ? base + __popcll(__ballot(place[lane] >= 0)) : *r.count;
  const int64_t end = a.whole ? (a.n + 63) / 64 * 64 : (n + 63) / 64 * 64;
  constexpr int kPlanes = OUT == 0 ? 1 : 3;
  constexpr int kOutBytes = OUT == 0 ? sizeof(E) : 2;
  const int64_t c1 = first + a.cols < a.pitch ? first + a.cols : a.pitch;
  if (lead && a.whole)
    for (int64_t p = n + tid; p < end; p += 256) {
      if (p < a.n) r.labels[p] = -1;
      if (p < a.n && a.grad.coef != nullptr) a.grad.coef[p] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
  for (int64_t p = n + wave; p < end; p += 4) {
    for (int k = 0; a.dst != nullptr && k < kPlanes; ++k)
      for (int64_t c = first + lane; c < c1; c += 64) {
        char* d = static_cast<char*>(a.dst) + ((p * kPlanes + k) * a.pitch + c) * kOutBytes;
        if constexpr (kOutBytes == 2) *reinterpret_cast<uint16_t*>(d) = 0;
        else *reinterpret_cast<uint32_t*>(d) = 0;
      }
    for (int k = 0; a.trans != nullptr && k < kPlanes; ++k)
      for (int64_t c = first + lane; c < c1 && c < a.h; c += 64) {
        char* d = static_cast<char*>(a.trans) + ((c * kPlanes + k) * a.ldt + p) * kOutBytes;
        if constexpr (kOutBytes == 2) *reinterpret_cast<uint16_t*>(d) = 0;
        else *reinterpret_cast<uint32_t*>(d) = 0;
      }
  }
}

// ------------------------------------------------------------ weights
// Rows of any pitch and alignment at a pitch of whole 16 bytes, zeros past cols: a
// wave a row, four 16-byte vectors a lane in flight, which need no alignment but
// their elements'. Bound by HBM: 51192 x 2426 of bf16 84 us, 5.9 TB/s (with loads as
// wide as a row's alignment allows, a vector a thread, 252).
template <typename E>
__global__ __launch_bounds__(256) void ce_stage_kernel(const E* src, int64_t lds, E* dst, int64_t ldd, int64_t rows,
                                                       int64_t cols) {
  constexpr int kV = 16 / sizeof(E), kLoads = 4, kStep = 64 * kV;
  const int lane = threadIdx.x & 63;
  const int64_t r = blockIdx.x * int64_t{4} + (threadIdx.x >> 6);
  if (r >= rows) return;
  const E* s = src + r * lds;
  E* d = dst + r * ldd;
  for (int64_t c = lane * kV; c < ldd; c += kLoads * kStep) {
    u32x4 w[kLoads];
    if (c + (kLoads - 1) * kStep + kV <= cols) {
#pragma unroll
      for (int q = 0; q < kLoads; ++q) __builtin_memcpy(&w[q], s + c + q * kStep, 16);
#pragma unroll
      for (int q = 0; q < kLoads; ++q) *reinterpret_cast<u32x4*>(d + c + q * kStep) = w[q];
      continue;
    }
    for (int q = 0; q < kLoads; ++q) {
      const int64_t at = c + q * kStep;
      if (at >= ldd) break;
      E x[kV];
      if (at + kV <= cols) {
        __builtin_memcpy(x, s + at, 16);
      } else {
#pragma unroll
        for (int k = 0; k < kV; ++k) x[k] = at + k < cols ? s[at + k] : E(0);
      }
      __builtin_memcpy(__builtin_assume_aligned(d + at, 16), x, 16);
    }
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
    sx += s.w;
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

// ------------------------------------------------------------ logits in memory
// Small fp32 calls (CeDirectArgs): a workgroup sums 2048 columns of a row over
// the parts of a product that was split, in order, and leaves their statistics,
// or writes the gradient of the logits (rows from the count on: zeros). 8 columns
// a thread, 16-byte vectors; the rows' pitches hold whole ones.
constexpr int kDirectCols = 2048;

__device__ __forceinline__ void direct_logits(const CeDirectArgs& a, int64_t row, int64_t c0, f32x4 (&x)[2]) {
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int64_t c = c0 + q * (kDirectCols / 2) + threadIdx.x * 4;
    x[q] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (c >= a.v) continue;
    const float* p = a.logits + row * a.ld + c;
    x[q] = *reinterpret_cast<const f32x4*>(p);
#pragma unroll 8
    for (int s = 1; s < a.splits; ++s) x[q] += *reinterpret_cast<const f32x4*>(p + s * a.stride);
  }
}

__global__ __launch_bounds__(256) void ce_direct_stats_kernel(CeDirectArgs a) {
  __shared__ float red[4][3];
  const int64_t row = blockIdx.y, c0 = static_cast<int64_t>(blockIdx.x) * kDirectCols;
  if (row >= *a.rows.count) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  f32x4 x[2];
  direct_logits(a, row, c0, x);
  const int64_t y = a.rows.labels[row];
  float m = -INFINITY, sx = 0.f;
#pragma unroll
  for (int q = 0; q < 2; ++q)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int64_t c = c0 + q * (kDirectCols / 2) + threadIdx.x * 4 + e;
      if (c >= a.v) continue;
      m = fmaxf(m, x[q][e]);
      sx += x[q][e];
      if (c == y) a.xy[row] = x[q][e];
    }
#pragma unroll
  for (int d = 32; d > 0; d /= 2) {
    m = fmaxf(m, __shfl_xor(m, d));
    sx += __shfl_xor(sx, d);
  }
  if (lane == 0) red[wave][0] = m, red[wave][1] = sx;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 4; ++w) m = fmaxf(m, red[w][0]);
  sx = red[0][1] + red[1][1] + red[2][1] + red[3][1];
  const float ref = fabsf(m) <= kCeLargest ? m : 0.f;   // as in the products' epilogue
  float sum = 0.f;
#pragma unroll
  for (int q = 0; q < 2; ++q)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (c0 + q * (kDirectCols / 2) + threadIdx.x * 4 + e < a.v)
        sum += __builtin_amdgcn_exp2f(fmaf(x[q][e], kLog2e, -ref * kLog2e));
#pragma unroll
  for (int d = 32; d > 0; d /= 2) sum += __shfl_xor(sum, d);
  if (lane == 0) red[wave][2] = sum;
  __syncthreads();
  if (threadIdx.x == 0)
    a.stats[row * a.stats_ld + blockIdx.x] =
        make_float4(m < -kCeLargest ? -INFINITY : ref, red[0][2] + red[1][2] + red[2][2] + red[3][2], 0.f, sx);
}

__global__ __launch_bounds__(256) void ce_direct_grad_kernel(CeDirectArgs a) {
  const int64_t row = blockIdx.y, c0 = static_cast<int64_t>(blockIdx.x) * kDirectCols;
  f32x4 x[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
  const bool live = row < *a.rows.count;
  float4 k = make_float4(0.f, 0.f, 0.f, 0.f);
  int64_t y = -1;
  if (live) {
    direct_logits(a, row, c0, x);
    k = a.coef[row];
    y = a.rows.labels[row];
  }
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int64_t c = c0 + q * (kDirectCols / 2) + threadIdx.x * 4;
    if (c >= a.v) continue;
    f32x4 d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (live && c + e < a.v) {
        d[e] = fmaf(k.y, __builtin_amdgcn_exp2f(fmaf(x[q][e], kLog2e, -k.x)), -k.z);
        if (c + e == y) d[e] -= k.w;
      }
    *reinterpret_cast<f32x4*>(a.grad + row * a.grad_ld + c) = d;
  }
}

// Compact fp32 gradient rows to their places; rows without a label are zero
// already (CePrepArgs::zero).
__global__ __launch_bounds__(256) void ce_scatter_kernel(const float* src, int64_t lds, CeRows r, int64_t h, float* dst,
                                                         int64_t ldd) {
  const int64_t row = blockIdx.x * int64_t{4} + (threadIdx.x >> 6);
  if (row >= *r.count) return;
  float* d = dst + r.src[row] * ldd;
  for (int64_t c = threadIdx.x & 63; c < h; c += 64) d[c] = src[row * lds + c];
}

template <typename E>
__global__ __launch_bounds__(256) void zero_rows_kernel(E* p, int64_t ld, int64_t rows, int64_t cols) {
  const int64_t row = blockIdx.x * int64_t{4} + (threadIdx.x >> 6);
  if (row >= rows) return;
  for (int64_t c = threadIdx.x & 63; c < cols; c += 64) p[row * ld + c] = E(0);
}

unsigned row_blocks(int64_t rows) { return static_cast<unsigned>((rows + 3) / 4); }

}  // namespace

hipError_t launch_ce_prep(const CePrepArgs& in, DType t, bool planes, hipStream_t stream) {
  CePrepArgs a = in;
  if (a.n <= 0) return hipSuccess;
  if (a.pitch % 8 != 0 || a.pitch < a.h || (planes && t != DType::F32)) return hipErrorInvalidValue;
  if (reinterpret_cast<uintptr_t>(a.dst) % 16 != 0 || reinterpret_cast<uintptr_t>(a.trans) % 16 != 0)
    return hipErrorInvalidValue;
  const int64_t es = dtype_size(t);
  const bool vec = (a.ldx * es) % 16 == 0 && reinterpret_cast<uintptr_t>(a.x) % 16 == 0;
  a.zero_vec = (a.ldz * es) % 16 == 0 && reinterpret_cast<uintptr_t>(a.zero) % 16 == 0;
  const bool scan = a.n <= kScanRows;
  if (!scan) {
    hipLaunchKernelGGL(ce_rows_kernel, dim3(1), dim3(kScanThreads), 0, stream, a.labels, a.n, a.v, a.ignore, a.rows, a.nll,
                       a.lse_out);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  const int64_t rows = (a.n + 63) / 64;
  a.cols = kMinPrepCols;
  while (a.cols < kMaxPrepCols && rows * ((a.pitch + a.cols - 1) / a.cols) > 2048) a.cols *= 2;
  const dim3 grid(static_cast<unsigned>(rows), static_cast<unsigned>((a.pitch + a.cols - 1) / a.cols));
  using K = void (*)(CePrepArgs);
  auto pick = [&](auto e, auto out_c) -> K {
    using E = decltype(e);
    constexpr int kOut = decltype(out_c)::value;
    if (scan) return vec ? ce_prep_kernel<E, kOut, true, true> : ce_prep_kernel<E, kOut, false, true>;
    return vec ? ce_prep_kernel<E, kOut, true, false> : ce_prep_kernel<E, kOut, false, false>;
  };
  const K k = t == DType::BF16 ? pick(uint16_t{}, std::integral_constant<int, 0>{})
              : planes         ? pick(float{}, std::integral_constant<int, 1>{})
                               : pick(float{}, std::integral_constant<int, 0>{});
  hipLaunchKernelGGL(k, grid, dim3(256), 0, stream, a);
  return hipGetLastError();
}

hipError_t launch_ce_stage(DType t, const void* src, int64_t lds, void* dst, int64_t ldd, int64_t rows, int64_t cols,
                           hipStream_t stream) {
  if (rows <= 0 || cols <= 0) return hipSuccess;
  if (ldd * dtype_size(t) % 16 != 0 || reinterpret_cast<uintptr_t>(dst) % 16 != 0 || ldd < cols)
    return hipErrorInvalidValue;
  const dim3 grid(static_cast<unsigned>((rows + 3) / 4));
  if (t == DType::BF16)
    hipLaunchKernelGGL(ce_stage_kernel<uint16_t>, grid, dim3(256), 0, stream, static_cast<const uint16_t*>(src), lds,
                       static_cast<uint16_t*>(dst), ldd, rows, cols);
  else
    hipLaunchKernelGGL(ce_stage_kernel<float>, grid, dim3(256), 0, stream, static_cast<const float*>(src), lds,
                       static_cast<float*>(dst), ldd, rows, cols);
  return hipGetLastError();
}

hipError_t launch_ce_losses(const CeLossArgs& a, int64_t n, hipStream_t stream) {
  hipLaunchKernelGGL(ce_losses_kernel, dim3(row_blocks(n)), dim3(256), 0, stream, a);
  return hipGetLastError();
}

int64_t ce_direct_tiles(int64_t v) { return (v + kDirectCols - 1) / kDirectCols; }

hipError_t launch_ce_direct(const CeDirectArgs& a, int64_t n, bool grad, hipStream_t stream) {
  if (n <= 0) return hipSuccess;
  if (a.ld % 4 != 0 || a.stride % 4 != 0 || reinterpret_cast<uintptr_t>(a.logits) % 16 != 0 || n > 65535 ||
      (grad && (a.grad_ld % 4 != 0 || reinterpret_cast<uintptr_t>(a.grad) % 16 != 0)))
    return hipErrorInvalidValue;
  const dim3 grid(static_cast<unsigned>(ce_direct_tiles(a.v)), static_cast<unsigned>(n));
  if (grad) hipLaunchKernelGGL(ce_direct_grad_kernel, grid, dim3(256), 0, stream, a);
  else hipLaunchKernelGGL(ce_direct_stats_kernel, grid, dim3(256), 0, stream, a);
  return hipGetLastError();
}

hipError_t launch_ce_scatter(const float* src, int64_t lds, const CeRows& r, int64_t n, int64_t h, float* dst, int64_t ldd,
                             hipStream_t stream) {
  if (n <= 0) return hipSuccess;
  hipLaunchKernelGGL(ce_scatter_kernel, dim3(row_blocks(n)), dim3(256), 0, stream, src, lds, r, h, dst, ldd);
  return hipGetLastError();
}

hipError_t launch_zero_rows(DType t, void* p, int64_t ld, int64_t rows, int64_t cols, hipStream_t stream) {
  auto run = [&](auto* d) {
    using E = std::remove_pointer_t<decltype(d)>;
    constexpr int64_t kMost = most_blocks(256) * 4;   // rows of a launch
    for (int64_t r = 0; r < rows; r += kMost) {
      const int64_t m = rows - r < kMost ? rows - r : kMost;
      hipLaunchKernelGGL(zero_rows_kernel<E>, dim3(row_blocks(m)), dim3(256), 0, stream, d + r * ld, ld, m, cols);
    }
  };
  if (t == DType::BF16) run(static_cast<uint16_t*>(p));
  else run(static_cast<uint32_t*>(p));
  return hipGetLastError();
}

}  // namespace orda
