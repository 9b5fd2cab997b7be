// norm.hip — the root-mean-square norm with the residual's addition, its output in
// the rows' type or in e4m3, and its gradients.
//
// With t = x + r and s = (mean t² + eps)^-1/2: out = t·s·(w + o), and, with q = g·(w + o),
// dt = s·q - t·s³·mean(q·t) + gt, dw = Σ over rows of g·t·s. Bound by HBM: each input is read
// once and each output written once, a row held in registers in between as it lies in
// memory (bf16 keeps half the registers of its values); the gradient of the weight stays in
// registers over a workgroup's rows. Squares are summed in 64 bits, which costs nothing
// beside the loads; the products of the gradients in 32.
// 8192 x 4096 bf16 with a residual: forward 44 us (6.0 TB/s; to e4m3 45, where codes are 1
// byte), gradients 43 with the sum's gradient (6.2 TB/s), and 4 for the weight's join.
#include <math.h>

#include "fp8_codes.h"
#include "orda_kernels.h"
#include "wave.h"

namespace orda {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Eight neighbouring values as they lie in memory.
template <typename E>
struct Raw8 {
  u32x4 q[sizeof(E) / 2];
};

// Columns c to c + 7 of a row of h. Every lane loads, those past the row's end from
// within it, so that no branch makes a load wait for the one before; `settle` then puts
// zeros there. TAIL (h no multiple of 8): the last eight that the row has, which it moves
// into place.
template <typename E, bool TAIL>
__device__ __forceinline__ Raw8<E> fetch8(const E* row, int64_t c, int64_t h) {
  Raw8<E> r;
  if (TAIL && h < 8) {
    E v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = c + k < h ? row[c + k] : static_cast<E>(0.f);
    __builtin_memcpy(&r, v, sizeof r);
  } else {
    const int64_t at = TAIL ? (c <= h - 8 ? c : h - 8) : (c < h ? c : 0);
    __builtin_memcpy(&r, row + at, sizeof r);
  }
  return r;
}
template <typename E, bool TAIL>
__device__ __forceinline__ void settle(Raw8<E>& r, int64_t c, int64_t h) {
  constexpr int kWords = 2 * sizeof(E);
  const int64_t past = TAIL ? c - (h - 8) : c < h ? 0 : 8;
  if ((TAIL && h < 8) || !__any(past > 0)) return;   // (whole waves: most)
  const int d = past < 0 ? 0 : past < 8 ? static_cast<int>(past) : 8;
  uint32_t w[kWords];
  __builtin_memcpy(w, &r, sizeof r);
  if constexpr (TAIL) {   // by d values: 4, 2 and 1 of them
    auto move = [&](int b, int words) {
#pragma unroll
      for (int k = 0; k < kWords; ++k) w[k] = (d & b) ? (k + words < kWords ? w[k + words] : 0u) : w[k];
    };
    move(4, sizeof(E));
    move(2, sizeof(E) / 2);
    if constexpr (sizeof(E) == 4) {
      move(1, 1);
    } else {
#pragma unroll
      for (int k = 0; k < kWords; ++k) {
        const uint32_t next = k + 1 < kWords ? w[k + 1] : 0u;
        w[k] = (d & 1) ? __builtin_amdgcn_alignbit(next, w[k], 16) : w[k];
      }
    }
  }
#pragma unroll
  for (int k = 0; k < kWords; ++k) w[k] = d >= 8 ? 0u : w[k];
  __builtin_memcpy(&r, w, sizeof r);
}
template <typename E, bool TAIL>
__device__ __forceinline__ Raw8<E> settled8(const E* row, int64_t c, int64_t h) {
  Raw8<E> r = fetch8<E, TAIL>(row, c, h);
  settle<E, TAIL>(r, c, h);
  return r;
}
// Makes the compiler convert them anew where they are used next, instead of keeping the
// values, twice the registers, over a barrier.
template <typename E>
__device__ __forceinline__ void again(Raw8<E>& r) {
#pragma unroll
  for (size_t i = 0; i < sizeof(E) / 2; ++i) asm volatile("" : "+v"(r.q[i]));
}
template <typename E>
__device__ __forceinline__ void widened(const Raw8<E>& r, float (&x)[8]) {
  E v[8];
  __builtin_memcpy(v, &r, sizeof r);
#pragma unroll
  for (int k = 0; k < 8; ++k) x[k] = static_cast<float>(v[k]);
}
template <typename E, bool TAIL>
__device__ __forceinline__ void put8(E* row, int64_t c, int64_t h, const Raw8<E>& x) {
  E v[8];
  __builtin_memcpy(v, &x, sizeof v);
  if (c + 8 <= h) {
    __builtin_memcpy(row + c, v, sizeof v);
  } else if (TAIL) {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (c + k < h) row[c + k] = v[k];
  }
}

template <typename E, bool TAIL>
__device__ __forceinline__ void put8(E* row, int64_t c, int64_t h, const float (&x)[8]) {
  E v[8];
  Raw8<E> r;
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = static_cast<E>(x[k]);
  __builtin_memcpy(&r, v, sizeof v);
  put8<E, TAIL>(row, c, h, r);
}

// Codes and scales of a lane's eight values; 16 lanes hold a block of 128.
__device__ __forceinline__ void put_codes(const NormArgs& a, int64_t row, int64_t c, const float (&v)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) m = abs_bits(v[k]) > m ? abs_bits(v[k]) : m;
  m = most_of<16>(m);
  const float s = scale_divided(m);
  store8_divided(a.codes + row * a.ldc, c, a.h, v, s);
  if ((threadIdx.x & 15) == 0 && c < a.h) a.scales[row * a.scale_row + c / 128 * a.scale_col] = s;
}

// v = t·s·(w + offset). To e4m3 the factors and products are pairs of fp32 values, each the
// other's rounding error, and v is their sum, rounded once: next to a border of two codes
// fp32's own roundings would decide, and the codes are those of the formula. (In 64 bits
// it took 27 us more at 8192 x 4096.)
struct Factor {
  float s, rest;   // of the row
};
// 1/sqrt(x) from the instruction's 24 bits and Newton's steps (0 and infinity as they
// come): a sixth of the instructions of a square root and a division.
__device__ __forceinline__ double reciprocal_root(double x) {
  const double y0 = __builtin_amdgcn_rsq(x);
  const double half = .5 * x;
  double y = y0;
  y = fma(y, fma(-half * y, y, .5), y);
  y = fma(y, fma(-half * y, y, .5), y);
  return y0 > 0. && y0 < INFINITY ? y : y0;
}
__device__ __forceinline__ Factor factor_of(double sum, const NormArgs& a) {
  const double s = reciprocal_root(fma(sum, a.per_column, a.eps));
  const float f = static_cast<float>(s);
  return {f, static_cast<float>(s - static_cast<double>(f))};
}
// OFFSET: there is one.
template <bool OFFSET>
__device__ __forceinline__ float paired(float t, const Factor& f, float w, float o, float o_rest) {
#pragma clang fp contract(off)   // (a rounding error is of the rounded product)
  const float u = t * f.s, u_rest = fmaf(t, f.rest, fmaf(t, f.s, -u));
  float q = w, q_rest = 0.f;
  if constexpr (OFFSET) {
    q = w + o;
    const float b = q - w;
    q_rest = (w - (q - b)) + (o - b) + o_rest;
  }
  // (what is to be added with its sign turned: a -0 stays one)
  const float p = u * q;
  float less = fmaf(-u_rest, q, fmaf(-u, q, p));
  if constexpr (OFFSET) less = fmaf(-u, q_rest, less);
  return p - less;
}
template <bool FP8>
__device__ __forceinline__ void normed(const float (&t)[8], const Factor& f, const float (&w)[8], double offset,
                                       float (&v)[8]) {
  const float o = static_cast<float>(offset);
  if constexpr (!FP8) {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = t[k] * f.s * (w[k] + o);
  } else if (offset == 0.) {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = paired<false>(t[k], f, w[k], 0.f, 0.f);
  } else {
    const float o_rest = static_cast<float>(offset - static_cast<double>(o));
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = paired<true>(t[k], f, w[k], o, o_rest);
  }
}

// NT threads hold a row in registers, NV vectors of eight columns each.
template <typename E, typename W, int NT, int NV, bool TAIL, bool FP8>
__global__ __launch_bounds__(NT < 256 ? 256 : NT) void norm_kernel(NormArgs a) {
  constexpr int kTeams = NT < 256 ? 256 / NT : 1, kWaves = NT / 64;
  __shared__ double part[kTeams][kWaves];
  const int team = threadIdx.x / NT, at = threadIdx.x % NT;
  const int64_t row0 = blockIdx.x * int64_t{kTeams} + team;
  const bool live = row0 < a.n;
  const int64_t row = live ? row0 : a.n - 1;
  Raw8<E> t[NV];   // the sum, as it lies in memory
  const E* px = static_cast<const E*>(a.x) + row * a.ldx;
#pragma unroll
  for (int i = 0; i < NV; ++i) t[i] = fetch8<E, TAIL>(px, (i * NT + at) * int64_t{8}, a.h);
  double sum = 0.;
  auto add = [&](const float (&v)[8]) {
#pragma unroll
    for (int k = 0; k < 8; ++k) sum = fma(static_cast<double>(v[k]), static_cast<double>(v[k]), sum);
  };
  if (a.r) {
    Raw8<E> r[NV];
    const E* pr = static_cast<const E*>(a.r) + row * a.ldr;
#pragma unroll
    for (int i = 0; i < NV; ++i) r[i] = fetch8<E, TAIL>(pr, (i * NT + at) * int64_t{8}, a.h);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int64_t c = (i * NT + at) * int64_t{8};
      float v[8], y[8];
      E e[8];
      settle<E, TAIL>(t[i], c, a.h);
      settle<E, TAIL>(r[i], c, a.h);
      widened(t[i], v);
      widened(r[i], y);
#pragma unroll
      for (int k = 0; k < 8; ++k) e[k] = static_cast<E>(v[k] + y[k]);
      __builtin_memcpy(&t[i], e, sizeof e);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = static_cast<float>(e[k]);
      add(v);
      if (a.total && live) put8<E, TAIL>(static_cast<E*>(a.total) + row * a.ldt, c, a.h, t[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int64_t c = (i * NT + at) * int64_t{8};
      float v[8];
      settle<E, TAIL>(t[i], c, a.h);
      widened(t[i], v);
      add(v);
      if (a.total && live) put8<E, TAIL>(static_cast<E*>(a.total) + row * a.ldt, c, a.h, t[i]);
    }
  }
  Raw8<W> wr[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) wr[i] = fetch8<W, TAIL>(static_cast<const W*>(a.w), (i * NT + at) * int64_t{8}, a.h);
  sum = wave_sum(sum);
  if constexpr (kWaves > 1) {
    if ((at & 63) == 0) part[team][at >> 6] = sum;
    __syncthreads();
    sum = 0.;
#pragma unroll
    for (int q = 0; q < kWaves; ++q) sum += part[team][q];
  }
  const Factor f = factor_of(sum, a);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int64_t c = (i * NT + at) * int64_t{8};
    float w[8], v[8], y[8];
    again(t[i]);
    settle<W, TAIL>(wr[i], c, a.h);
    widened(wr[i], w);
    widened(t[i], y);
    normed<FP8>(y, f, w, a.offset, v);
    if constexpr (FP8) {
      if (live) put_codes(a, row, c, v);
    } else {
      if (live) put8<E, TAIL>(static_cast<E*>(a.out) + row * a.ldo, c, a.h, v);
    }
  }
}

// Rows longer than registers hold: a workgroup a row, read twice.
template <typename E, typename W, bool FP8>
__global__ __launch_bounds__(1024) void norm_long_kernel(NormArgs a) {
  __shared__ double part[16];
  const int64_t row = blockIdx.x;
  const E* px = static_cast<const E*>(a.x) + row * a.ldx;
  const E* pr = a.r ? static_cast<const E*>(a.r) + row * a.ldr : nullptr;
  auto totals = [&](int64_t c, float (&t)[8]) {
    widened(settled8<E, true>(px, c, a.h), t);
    if (!pr) return;
    float y[8];
    widened(settled8<E, true>(pr, c, a.h), y);
#pragma unroll
    for (int k = 0; k < 8; ++k) t[k] = static_cast<float>(static_cast<E>(t[k] + y[k]));
  };
  double sum = 0.;
  for (int64_t c = threadIdx.x * int64_t{8}; c < a.h; c += 8192) {
    float t[8];
    totals(c, t);
    if (a.total) put8<E, true>(static_cast<E*>(a.total) + row * a.ldt, c, a.h, t);
#pragma unroll
    for (int k = 0; k < 8; ++k) sum = fma(static_cast<double>(t[k]), static_cast<double>(t[k]), sum);
  }
  sum = wave_sum(sum);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = sum;
  __syncthreads();
  sum = 0.;
#pragma unroll
  for (int q = 0; q < 16; ++q) sum += part[q];
  const Factor f = factor_of(sum, a);
  // (Whole waves take part in a block's maximum: the columns past the end are 0.)
  for (int64_t c = threadIdx.x * int64_t{8}; c - threadIdx.x % 64 * 8 < a.h; c += 8192) {
    float t[8], w[8], v[8];
    totals(c, t);
    widened(settled8<W, true>(static_cast<const W*>(a.w), c, a.h), w);
    normed<FP8>(t, f, w, a.offset, v);
    if constexpr (FP8) put_codes(a, row, c, v);
    else put8<E, true>(static_cast<E*>(a.out) + row * a.ldo, c, a.h, v);
  }
}

// ------------------------------------------------------------ gradients
// A row's two sums and what follows from them.
struct RowGrad {
  float s, k;   // dx = s·(g·q - t·k) + gt
};
__device__ __forceinline__ RowGrad row_grad(double sq, float dot, const NormGradArgs& a) {
  const double s = reciprocal_root(fma(sq, a.per_column, a.eps));
  return {static_cast<float>(s), static_cast<float>(s * s * (static_cast<double>(dot) * a.per_column))};
}

// Workgroups of teams of NT threads, a row a team at a time, the next row's loads under
// way; a thread's columns of the weight and of its gradient stay in registers. ws: a row
// of fp32 a workgroup.
constexpr int kGradThreads = 512;   // 256 registers each: the loads under way and the sums
template <typename E, typename W, int NT, int NV, bool TAIL>
__global__ __launch_bounds__(kGradThreads) void norm_grad_kernel(NormGradArgs a) {
  constexpr int kTeams = kGradThreads / NT, kWaves = NT / 64;
  __shared__ double part_sq[2][kTeams][kWaves];
  __shared__ float part_dot[2][kTeams][kWaves];
  __shared__ float acc[NT * NV * 8];
  const int team = threadIdx.x / NT, at = threadIdx.x % NT;
  const float offset = static_cast<float>(a.offset);
  Raw8<W> wr[NV];
  float dw[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    wr[i] = settled8<W, TAIL>(static_cast<const W*>(a.w), (i * NT + at) * int64_t{8}, a.h);
#pragma unroll
    for (int k = 0; k < 8; ++k) dw[i][k] = 0.f;
  }
  Raw8<E> rg[NV], rt[NV], rx[NV];
  auto fetch = [&](int64_t r) {
    const int64_t row = r + team < a.n ? r + team : a.n - 1;
    const E* pg = static_cast<const E*>(a.g) + row * a.ldg;
    const E* pt = static_cast<const E*>(a.t) + row * a.ldt;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      rg[i] = fetch8<E, TAIL>(pg, (i * NT + at) * int64_t{8}, a.h);
      rt[i] = fetch8<E, TAIL>(pt, (i * NT + at) * int64_t{8}, a.h);
    }
    if (a.gt) {
      const E* px = static_cast<const E*>(a.gt) + row * a.ldgt;
#pragma unroll
      for (int i = 0; i < NV; ++i) rx[i] = fetch8<E, TAIL>(px, (i * NT + at) * int64_t{8}, a.h);
    }
  };
  const int64_t step = gridDim.x * int64_t{kTeams};
  int turn = 0;
  fetch(blockIdx.x * int64_t{kTeams});
  for (int64_t r0 = blockIdx.x * int64_t{kTeams}; r0 < a.n; r0 += step, turn ^= 1) {
    const bool live = r0 + team < a.n;
    const int64_t row = r0 + team;
    Raw8<E> g8[NV], t8[NV], x8[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int64_t c = (i * NT + at) * int64_t{8};
      g8[i] = rg[i], t8[i] = rt[i], x8[i] = rx[i];
      settle<E, TAIL>(g8[i], c, a.h);
      settle<E, TAIL>(t8[i], c, a.h);
      if (a.gt) settle<E, TAIL>(x8[i], c, a.h);
    }
    if (r0 + step < a.n) fetch(r0 + step);
    double sq = 0.;
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float g[8], t[8], q[8];
      widened(g8[i], g);
      widened(t8[i], t);
      widened(wr[i], q);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        sq = fma(static_cast<double>(t[k]), static_cast<double>(t[k]), sq);
        dot = fmaf(g[k] * (q[k] + offset), t[k], dot);
      }
    }
    sq = wave_sum(sq);
    dot = wave_sum(dot);
    if constexpr (kWaves > 1) {
      if ((at & 63) == 0) {
        part_sq[turn][team][at >> 6] = sq;
        part_dot[turn][team][at >> 6] = dot;
      }
      __syncthreads();
      sq = 0.;
      dot = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        sq += part_sq[turn][team][w];
        dot += part_dot[turn][team][w];
      }
    }
    const RowGrad f = row_grad(sq, dot, a);
    if (!live) continue;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int64_t c = (i * NT + at) * int64_t{8};
      float g[8], t[8], q[8], y[8], d[8];
      again(g8[i]);
      again(t8[i]);
      again(wr[i]);
      widened(g8[i], g);
      widened(t8[i], t);
      widened(wr[i], q);
      if (a.gt) widened(x8[i], y);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        d[k] = f.s * (g[k] * (q[k] + offset) - t[k] * f.k);
        if (a.gt) d[k] += y[k];
        dw[i][k] = fmaf(g[k], t[k] * f.s, dw[i][k]);
      }
      if (a.dx) put8<E, TAIL>(static_cast<E*>(a.dx) + row * a.ldd, c, a.h, d);
    }
  }
  if (!a.dw) return;
  // the teams' sums in their order
  for (int p = 0; p < kTeams; ++p) {
    if (p == team) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          float& s = acc[(k * NV + i) * NT + at];
          s = p ? s + dw[i][k] : dw[i][k];
        }
    }
    __syncthreads();
  }
  float* out = static_cast<float*>(a.ws) + blockIdx.x * a.h;
  for (int64_t c = threadIdx.x; c < a.h; c += kGradThreads) {
    const int v = static_cast<int>(c / 8);
    out[c] = acc[(static_cast<int>(c % 8) * NV + v / NT) * NT + v % NT];
  }
}

// Longer rows: their factors first (a workgroup a row), then tiles of 2048 columns
// and `each` rows.
template <typename E, typename W>
__global__ __launch_bounds__(1024) void norm_grad_rows_kernel(NormGradArgs a) {
  __shared__ double part_sq[16];
  __shared__ float part_dot[16];
  const int64_t row = blockIdx.x;
  const E* pg = static_cast<const E*>(a.g) + row * a.ldg;
  const E* pt = static_cast<const E*>(a.t) + row * a.ldt;
  double sq = 0.;
  float dot = 0.f;
  for (int64_t c = threadIdx.x * int64_t{8}; c < a.h; c += 8192) {
    float g[8], t[8], q[8];
    widened(settled8<E, true>(pg, c, a.h), g);
    widened(settled8<E, true>(pt, c, a.h), t);
    widened(settled8<W, true>(static_cast<const W*>(a.w), c, a.h), q);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      sq = fma(static_cast<double>(t[k]), static_cast<double>(t[k]), sq);
      dot = fmaf(g[k] * (q[k] + static_cast<float>(a.offset)), t[k], dot);
    }
  }
  sq = wave_sum(sq);
  dot = wave_sum(dot);
  if ((threadIdx.x & 63) == 0) {
    part_sq[threadIdx.x >> 6] = sq;
    part_dot[threadIdx.x >> 6] = dot;
  }
  __syncthreads();
  if (threadIdx.x) return;
  sq = 0.;
  dot = 0.f;
  for (int w = 0; w < 16; ++w) {
    sq += part_sq[w];
    dot += part_dot[w];
  }
  static_cast<RowGrad*>(a.ws)[row] = row_grad(sq, dot, a);
}
template <typename E, typename W>
__global__ __launch_bounds__(256) void norm_grad_tiles_kernel(NormGradArgs a, const RowGrad* rows, float* parts,
                                                              int64_t each) {
  const int64_t across = (a.h + 2047) / 2048, tile = blockIdx.x % across, band = blockIdx.x / across;
  const int64_t c = (tile * 256 + threadIdx.x) * 8;
  float q[8], dw[8];
  widened(settled8<W, true>(static_cast<const W*>(a.w), c, a.h), q);
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    q[k] += static_cast<float>(a.offset);
    dw[k] = 0.f;
  }
  const int64_t end = (band + 1) * each < a.n ? (band + 1) * each : a.n;
  for (int64_t row = band * each; row < end; ++row) {
    float g[8], t[8], y[8], d[8];
    widened(settled8<E, true>(static_cast<const E*>(a.g) + row * a.ldg, c, a.h), g);
    widened(settled8<E, true>(static_cast<const E*>(a.t) + row * a.ldt, c, a.h), t);
    if (a.gt) widened(settled8<E, true>(static_cast<const E*>(a.gt) + row * a.ldgt, c, a.h), y);
    const RowGrad f = rows[row];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      d[k] = f.s * (g[k] * q[k] - t[k] * f.k);
      if (a.gt) d[k] += y[k];
      dw[k] = fmaf(g[k], t[k] * f.s, dw[k]);
    }
    if (a.dx) put8<E, true>(static_cast<E*>(a.dx) + row * a.ldd, c, a.h, d);
  }
  if (a.dw) put8<float, true>(parts + band * a.h, c, a.h, dw);
}

// dw[c] = Σ_p parts[p][c]: 64 columns a workgroup, 16 threads a column.
template <typename W>
__global__ __launch_bounds__(1024) void norm_grad_join_kernel(const float* parts, int64_t count, int64_t h, W* dw) {
  __shared__ float sums[16][64];
  const int k = threadIdx.x & 63, p0 = threadIdx.x >> 6;
  const int64_t c = blockIdx.x * int64_t{64} + k;
  float s = 0.f;
  if (c < h)
    for (int64_t p = p0; p < count; p += 256) {
      float v[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = p + 16 * i < count ? parts[(p + 16 * i) * h + c] : 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) s += v[i];
    }
  sums[p0][k] = s;
  __syncthreads();
  if (p0 == 0 && c < h) {
    for (int p = 1; p < 16; ++p) s += sums[p][k];
    dw[c] = static_cast<W>(s);
  }
}

// ------------------------------------------------------------ launches
using NormKernel = void (*)(NormArgs);
struct NormLaunch {
  NormKernel k;
  int threads, teams;
};
template <typename E, typename W, bool TAIL, bool FP8>
NormLaunch norm_launch(int64_t n, int64_t h) {
  // Few rows: as many threads as a row has vectors (bf16 with residual, 1 and 64 rows: 2048
  // columns 2.0 and 2.8 us, in the other form 3.0 and 3.9; 4096 2.4 and 3.6, 3.0 and 4.1;
  // 512 rows of 4096 5.6 and 5.2).
  if (n < 512) {
    if (h <= 2048) return {norm_kernel<E, W, 256, 1, TAIL, FP8>, 256, 1};
    if (h <= 8192) return {norm_kernel<E, W, 1024, 1, TAIL, FP8>, 1024, 1};
  }
  // Many: four vectors a thread, whose loads are under way together, and few waves that
  // wait for one another (8192 x 4096 to e4m3: two waves a row 44 us, four 62).
  if (h <= 1024) return {norm_kernel<E, W, 64, 2, TAIL, FP8>, 256, 4};
  if (h <= 2048) return {norm_kernel<E, W, 64, 4, TAIL, FP8>, 256, 4};
  if (h <= 4096) return {norm_kernel<E, W, 128, 4, TAIL, FP8>, 256, 2};
  if (h <= 8192) return {norm_kernel<E, W, 256, 4, TAIL, FP8>, 256, 1};
  if (h <= 32768) return {norm_kernel<E, W, 1024, 4, TAIL, FP8>, 1024, 1};
  return {norm_long_kernel<E, W, FP8>, 1024, 1};
}
template <typename E, typename W>
NormLaunch norm_launch(const NormArgs& a) {
  if (a.codes)
    return a.h % 8 ? norm_launch<E, W, true, true>(a.n, a.h) : norm_launch<E, W, false, true>(a.n, a.h);
  return a.h % 8 ? norm_launch<E, W, true, false>(a.n, a.h) : norm_launch<E, W, false, false>(a.n, a.h);
}

constexpr int64_t kLongRow = 16384, kLongRowF32 = 8192;   // longer ones are read twice
using GradKernel = void (*)(NormGradArgs);
struct GradLaunch {
  GradKernel k;   // null: rows too long for registers
  int teams;
};
template <typename E, typename W, bool TAIL>
GradLaunch grad_launch(int64_t h) {
  // As many rows at a time as registers hold (8192 rows of bf16, one thread a vector and
  // two rows in their place: 1024 columns 13 us against 25, 2048 19 against 27; 64 rows
  // take 5 us against 4).
  if (h <= 512) return {norm_grad_kernel<E, W, 64, 1, TAIL>, 8};
  if (h <= 1024) return {norm_grad_kernel<E, W, 64, 2, TAIL>, 8};
  if (h <= 2048) return {norm_grad_kernel<E, W, 128, 2, TAIL>, 4};
  if (h <= 4096) return {norm_grad_kernel<E, W, 256, 2, TAIL>, 2};
  if (h <= 8192) return {norm_grad_kernel<E, W, 512, 2, TAIL>, 1};
  // (fp32's do not fit: with spills 2000 x 16384 took 153 us, read twice 114; bf16 takes 36,
  // and read twice half of 32768 columns' 112.)
  if constexpr (sizeof(E) == 2)
    if (h <= kLongRow) return {norm_grad_kernel<E, W, 512, 4, TAIL>, 1};
  return {nullptr, 0};
}
int grad_teams(int64_t h) { return h <= 1024 ? 8 : h <= 2048 ? 4 : h <= 4096 ? 2 : 1; }

// Workgroups that keep sums of the weight's gradient, one a CU (of 512 the kernel takes as long
// and the join 4 us more; 8192 x 4096 bf16).
constexpr int64_t kGradBlocks = 256;
int64_t grad_blocks(int64_t n, int64_t h) {
  const int64_t b = (n + grad_teams(h) - 1) / grad_teams(h);
  return b < kGradBlocks ? b : kGradBlocks;
}
// Bands of rows of the tiles of long rows: enough tiles to fill the device.
int64_t grad_bands(int64_t n, int64_t h) {
  const int64_t across = (h + 2047) / 2048, want = (1024 + across - 1) / across;
  return n < want ? n : want;
}

template <typename E, typename W>
hipError_t norm_grad(const NormGradArgs& a, hipStream_t stream) {
  const float* parts = static_cast<const float*>(a.ws);
  int64_t count;
  const GradLaunch l = a.h % 8 ? grad_launch<E, W, true>(a.h) : grad_launch<E, W, false>(a.h);
  if (l.k) {
    count = grad_blocks(a.n, a.h);
    hipLaunchKernelGGL(l.k, dim3(static_cast<unsigned>(count)), dim3(kGradThreads), 0, stream, a);
  } else {
    float* p = static_cast<float*>(a.ws) + (a.n * 2 + 63) / 64 * 64;
    const int64_t bands = grad_bands(a.n, a.h), each = (a.n + bands - 1) / bands;
    count = (a.n + each - 1) / each;
    constexpr int64_t kMost = most_blocks(1024);
    if (a.n > kMost) return hipErrorInvalidValue;   // 128 GiB of rows
    hipLaunchKernelGGL((norm_grad_rows_kernel<E, W>), dim3(static_cast<unsigned>(a.n)), dim3(1024), 0, stream, a);
    hipLaunchKernelGGL((norm_grad_tiles_kernel<E, W>), dim3(static_cast<unsigned>(count * ((a.h + 2047) / 2048))),
                       dim3(256), 0, stream, a, static_cast<const RowGrad*>(a.ws), p, each);
    parts = p;
  }
  if (a.dw)
    hipLaunchKernelGGL((norm_grad_join_kernel<W>), dim3(static_cast<unsigned>((a.h + 63) / 64)), dim3(1024), 0, stream,
                       parts, count, a.h, static_cast<W*>(a.dw));
  return hipGetLastError();
}

}  // namespace

hipError_t launch_norm(const NormArgs& a, DType rows, DType weight, hipStream_t stream) {
  const NormLaunch l = rows == DType::BF16
                           ? (weight == DType::BF16 ? norm_launch<__bf16, __bf16>(a) : norm_launch<__bf16, float>(a))
                           : (weight == DType::BF16 ? norm_launch<float, __bf16>(a) : norm_launch<float, float>(a));
  const int64_t es = dtype_size(rows), most = most_blocks(l.threads) / l.teams * l.teams;   // rows of a launch
  for (int64_t r = 0; r < a.n; r += most) {
    NormArgs p = a;
    p.n = a.n - r < most ? a.n - r : most;
    auto past = [&](const void* d, int64_t ld) {
      return d ? static_cast<char*>(const_cast<void*>(d)) + r * ld * es : nullptr;
    };
    p.x = past(a.x, a.ldx);
    p.r = past(a.r, a.ldr);
    p.total = past(a.total, a.ldt);
    p.out = past(a.out, a.ldo);
    if (a.codes) {
      p.codes = a.codes + r * a.ldc;
      p.scales = a.scales + r * a.scale_row;
    }
    hipLaunchKernelGGL(l.k, dim3(static_cast<unsigned>((p.n + l.teams - 1) / l.teams)), dim3(l.threads), 0, stream, p);
  }
  return hipGetLastError();
}

int64_t norm_grad_scratch(int64_t n, int64_t h) {
  if (n == 0 || h == 0) return 0;
  // (of either type)
  const int64_t sums = h <= kLongRow ? grad_blocks(n, h) * h : 0;
  const int64_t twice = h > kLongRowF32 ? (n * 2 + 63) / 64 * 64 + grad_bands(n, h) * h : 0;
  return ((sums > twice ? sums : twice) * 4 + 255) / 256 * 256;
}

hipError_t launch_norm_grad(const NormGradArgs& a, DType rows, DType weight, hipStream_t stream) {
  if (rows == DType::BF16)
    return weight == DType::BF16 ? norm_grad<__bf16, __bf16>(a, stream) : norm_grad<__bf16, float>(a, stream);
  return weight == DType::BF16 ? norm_grad<float, __bf16>(a, stream) : norm_grad<float, float>(a, stream);
}

}  // namespace orda
