// sampling.hip — tokens drawn from rows of logits with temperature, top-k, top-p and
// min-p, by one given number a row.
//
// The distribution function of a row has as many borders as tokens, so an error of
// d in it gives another token with a probability of about 2·d·V: masses and their
// sums are held in 64 bits.
#include <math.h>

#include "orda_kernels.h"

namespace orda {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;   // of the kernel that picks: a workgroup a row
constexpr int kGroup = 1024;                             // tokens whose mass is summed up first
constexpr int kBins = 2048, kList = 4096;

// ---------------------------------------------------------------- keys, masses
// Keys order as the values do; equal values (0 and -0) have equal keys, NaN the
// largest.
constexpr uint32_t kNan = 0xffffffffu, kInf = 0xff800000u, kNone = 0x007fffffu;   // kNone: -infinity
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return x != x ? kNan : u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

// e^z of z <= 0, 0 below e^-700: z = n·ln 2 + y, and e^y by its series (|y| <= ln 2 / 2:
// the first term left out is 6e-15).
__device__ __forceinline__ double exp_of(double z) {
  const double n = rint(z * 1.4426950408889634074);
  double y = fma(n, -0.69314718055994528623, z);
  y = fma(n, -2.3190468138462995584e-17, y);
  double p = 1. / 39916800.;
  p = fma(p, y, 1. / 3628800.);
  p = fma(p, y, 1. / 362880.);
  p = fma(p, y, 1. / 40320.);
  p = fma(p, y, 1. / 5040.);
  p = fma(p, y, 1. / 720.);
  p = fma(p, y, 1. / 120.);
  p = fma(p, y, 1. / 24.);
  p = fma(p, y, 1. / 6.);
  p = fma(p, y, .5);
  p = fma(p, y, 1.);
  p = fma(p, y, 1.);
  const int e = static_cast<int>(n);
  const double r = __hiloint2double(__double2hiint(p) + e * (1 << 20), __double2loint(p));
  return z > -700. ? r : 0.;   // (and where z is NaN)
}

struct Row {
  float t, p, m, u;
  int64_t k;
  double inv_t;
  bool bad, first;   // first: only the largest logit is kept
};
__device__ __forceinline__ Row row_of(const SampleArgs& a, int64_t row) {
  Row r;
  r.t = a.t ? a.t[row] : a.t1;
  r.p = a.p ? a.p[row] : a.p1;
  r.m = a.m ? a.m[row] : a.m1;
  r.k = a.k ? a.k[row] : a.k1;
  r.u = a.u[row];
  r.bad = !(r.t >= 0.f) || r.t == INFINITY || r.p != r.p || r.m != r.m || !(r.u >= 0.f && r.u <= 1.f);
  if (r.k <= 0 || r.k >= a.v) r.k = 0;
  r.first = r.t == 0.f || r.k == 1 || r.p <= 0.f || r.m > 1.f;
  r.inv_t = 1. / static_cast<double>(r.t);
  return r;
}
// Whether the masses of all tokens are needed.
__device__ __forceinline__ bool whole(const Row& r) {
  return !r.bad && !r.first && r.k == 0 && (r.p < 1.f || r.m <= 0.f);
}

__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
  for (int d = 32; d; d /= 2) x += __shfl_xor(x, d);
  return x;
}

// A lane's 16 of a group's tokens, kPer neighbouring ones a load; -infinity past the
// row's end.
template <typename E>
struct Tokens {
  static constexpr int kPer = 16 / sizeof(E), kLoads = 16 / kPer;
  float x[16];
  __device__ __forceinline__ static int64_t column(int64_t group, int i) {   // of load i
    return group * kGroup + (i * 64 + static_cast<int>(threadIdx.x & 63)) * int64_t{kPer};
  }
  __device__ __forceinline__ void load(const E* row, int64_t group, int64_t v) {
    E w[kLoads][kPer];
    if ((group + 1) * kGroup <= v) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) __builtin_memcpy(w[i], row + column(group, i), sizeof w[i]);
    } else {
#pragma unroll
      for (int i = 0; i < kLoads; ++i)
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
          const int64_t c = column(group, i) + k;
          w[i][k] = c < v ? row[c] : static_cast<E>(-INFINITY);
        }
    }
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
#pragma unroll
      for (int k = 0; k < kPer; ++k) x[i * kPer + k] = static_cast<float>(w[i][k]);
  }
};

// ---------------------------------------------------------------- first pass
// A wave a group: the largest keys of its 64s and of all of it, and where they are
// needed its masses' sum, relative to its largest.
template <typename E>
__global__ __launch_bounds__(256) void sample_groups_kernel(SampleArgs a) {
  using T = Tokens<E>;
  const int64_t id = blockIdx.x * int64_t{4} + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (id >= a.n * a.n1024) return;
  const int64_t row = id / a.n1024, group = id - row * a.n1024;
  T t;
  t.load(static_cast<const E*>(a.x) + row * a.ldx, group, a.v);
  constexpr int kLanes = 64 / T::kPer;   // that hold 64 neighbouring tokens
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < T::kLoads; ++i) {
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < T::kPer; ++k) {
      const uint32_t key = key_of(t.x[i * T::kPer + k]);
      m = key > m ? key : m;
    }
#pragma unroll
    for (int d = 1; d < kLanes; d *= 2) {
      const uint32_t o = __shfl_xor(m, d);
      m = o > m ? o : m;
    }
    const int64_t at = group * (kGroup / 64) + i * T::kPer + lane / kLanes;
    if (lane % kLanes == 0 && at < a.n64) a.tops[row * a.n64 + at] = m;
    top = m > top ? m : top;
  }
#pragma unroll
  for (int d = kLanes; d < 64; d *= 2) {
    const uint32_t o = __shfl_xor(top, d);
    top = o > top ? o : top;
  }
  if (lane == 0) a.firsts[row * a.n1024 + group] = top;
  const Row r = row_of(a, row);
  if (!whole(r)) return;
  double mass = 0.;
  if (top >= kInf) {
#pragma unroll
    for (int k = 0; k < 16; ++k) mass += t.x[k] == INFINITY ? 1. : 0.;
  } else if (top > kNone) {
    const double most = static_cast<double>(value_of(top));
#pragma unroll
    for (int k = 0; k < 16; ++k) mass += exp_of((static_cast<double>(t.x[k]) - most) * r.inv_t);
  }
  mass = wave_sum(mass);
  if (lane == 0) a.masses[row * a.n1024 + group] = mass;
}

// ---------------------------------------------------------------- picking
struct Shared {
  uint64_t list[kList];        // candidates, key over the token's complement
  uint64_t mass[kBins];        // fixed point
  uint32_t count[2 * kBins];   // of bins; or the 64s that hold candidates
  double group[kGroup];
  double waves[kWaves];
  uint64_t waves64[kWaves];
  uint32_t n;
  uint32_t found;
  double before;
};

__device__ __forceinline__ uint64_t order_of(float x, int64_t c) {
  return static_cast<uint64_t>(key_of(x)) << 32 | static_cast<uint32_t>(~static_cast<uint32_t>(c));
}

template <typename T>
__device__ __forceinline__ T block_most(T v, T* waves) {   // largest of the block's
#pragma unroll
  for (int d = 32; d; d /= 2) {
    const T o = __shfl_xor(v, d);
    v = o > v ? o : v;
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = v;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) v = waves[w] > v ? waves[w] : v;
  return v;
}
// Sum of the values up to this thread's, and of all.
template <typename T>
__device__ __forceinline__ T block_scan(T v, T* waves, T& all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const T o = __shfl_up(v, d);
    if (lane >= d) v += o;
  }
  __syncthreads();
  if (lane == 63) waves[wave] = v;
  __syncthreads();
  T before = 0;
  all = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    if (w == wave) before = all;
    all += waves[w];
  }
  return before + v;
}

// One row's picking; every thread of the workgroup calls each member.
template <typename E>
struct Pick {
  const SampleArgs& a;
  Shared& s;
  const int64_t row;
  const Row r;
  const E* x;
  float top;
  bool inf;   // the largest is +infinity: those tokens count as 0, the others as -infinity

  __device__ __forceinline__ float value(float y) const { return inf ? (y == INFINITY ? 0.f : -INFINITY) : y; }
  __device__ __forceinline__ float at(int64_t c) const { return value(static_cast<float>(x[c])); }
  __device__ __forceinline__ double exponent(float y) const { return (static_cast<double>(y) - static_cast<double>(top)) * r.inv_t; }
  __device__ __forceinline__ double weight(float y) const { return exp_of(exponent(y)); }

  __device__ __forceinline__ void done(int64_t c, double logp) const {
    a.token[row] = c;
    if (a.logprob) a.logprob[row] = static_cast<float>(logp);
  }

  // Thread t's share of a sum that crosses `target`: the first whose sum up to it is
  // over the target, the last with a share where none is. Leaves the sum before it in
  // s.before.
  __device__ __forceinline__ int crossing(double share, double upto, double target) {
    uint32_t mine = 0;   // larger: earlier
    if (share > 0.) mine = upto > target ? 0x80000000u | (kThreads - threadIdx.x) : 1u + threadIdx.x;
    const uint32_t best = block_most(mine, reinterpret_cast<uint32_t*>(s.waves64));
    const int t = best & 0x80000000u ? kThreads - static_cast<int>(best & 0x7fffffffu) : best ? static_cast<int>(best) - 1 : 0;
    if (static_cast<int>(threadIdx.x) == t) s.before = upto - share;
    __syncthreads();
    return t;
  }

  // The token of `group` where the kept masses, `before` those of its groups before,
  // cross the target.
  __device__ __forceinline__ void in_group(int64_t group, double before, double target, double mass, uint64_t cut, double least) {
    const int64_t c = group * kGroup + threadIdx.x;
    float y = -INFINITY;
    double w = 0.;
    if (c < a.v) {
      y = at(c);
      w = weight(y);
      if (order_of(y, c) < cut || w < least) w = 0.;
    }
    double all;
    const double upto = before + block_scan(w, s.waves, all);
    const int t = crossing(w, upto, target);
    if (static_cast<int>(threadIdx.x) == t) done(c, exponent(y) - log(mass));
  }

  // Where the groups' masses cross u times their sum.
  __device__ __forceinline__ void by_groups(double mine, uint64_t cut, double least) {
    double mass;
    const double upto = block_scan(mine, s.waves, mass);
    const double target = static_cast<double>(r.u) * mass;
    const int g = crossing(mine, upto, target);
    in_group(g, s.before, target, mass, cut, least);
  }

  // The mass of thread t's group, all tokens counted.
  __device__ __forceinline__ double group_mass() const {
    if (static_cast<int64_t>(threadIdx.x) >= a.n1024) return 0.;
    const uint32_t k = a.firsts[row * a.n1024 + threadIdx.x];
    if (k <= kNone) return 0.;
    if (inf) return k == kInf ? a.masses[row * a.n1024 + threadIdx.x] : 0.;
    return a.masses[row * a.n1024 + threadIdx.x] * weight(value_of(k));
  }

  // The largest logit, the first such token.
  __device__ __forceinline__ void largest(uint32_t key) {
    uint32_t mine = 0;
    if (static_cast<int64_t>(threadIdx.x) < a.n1024 && a.firsts[row * a.n1024 + threadIdx.x] == key) mine = kThreads - threadIdx.x;
    const int64_t group = kThreads - static_cast<int64_t>(block_most(mine, reinterpret_cast<uint32_t*>(s.waves64)));
    const int64_t c = group * kGroup + threadIdx.x;
    mine = c < a.v && key_of(static_cast<float>(x[c])) == key ? kThreads - threadIdx.x : 0;
    const int t = kThreads - static_cast<int>(block_most(mine, reinterpret_cast<uint32_t*>(s.waves64)));
    if (static_cast<int>(threadIdx.x) == t) done(c, 0.);
  }

  // The k-th largest of the 64s' largest keys (1 <= k <= n64), 11, 11 and 10 bits at a time.
  __device__ __forceinline__ uint32_t kth_top(int64_t k) {
    const uint32_t* tops = a.tops + row * a.n64;
    uint32_t prefix = 0, mask = 0;
    uint32_t rank = static_cast<uint32_t>(k);
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
      const uint32_t digits = pass == 2 ? 1023 : 2047;
      __syncthreads();
      for (int b = threadIdx.x; b < kBins; b += kThreads) s.count[b] = 0;
      __syncthreads();
      for (int64_t i = threadIdx.x; i < a.n64; i += kThreads) {
        const uint32_t key = tops[i];
        if ((key & mask) == prefix) atomicAdd(&s.count[key >> shift & digits], 1u);
      }
      __syncthreads();
      const int b = kBins - 2 - 2 * static_cast<int>(threadIdx.x);   // bins b + 1, then b
      const uint64_t hi = s.count[b + 1], lo = s.count[b];
      uint64_t all;
      const uint64_t upto = block_scan<uint64_t>(hi + lo, s.waves64, all);
      if (upto >= rank && upto - hi - lo < rank) {
        const uint64_t before = upto - hi - lo;
        const bool in_hi = before + hi >= rank;
        s.found = static_cast<uint32_t>(in_hi ? b + 1 : b);
        s.n = static_cast<uint32_t>(rank - (in_hi ? before : before + hi));
      }
      __syncthreads();
      prefix |= s.found << shift;
      mask |= digits << shift;
      rank = s.n;
    }
    __syncthreads();
    return prefix;
  }

  // Puts o into the list where `take`.
  __device__ __forceinline__ void append(bool take, uint64_t o) {
    const uint64_t who = __ballot(take);
    if (!who) return;
    const int lane = threadIdx.x & 63;
    uint32_t base = 0;
    if (lane == 0) base = atomicAdd(&s.n, static_cast<uint32_t>(__popcll(who)));
    base = __shfl(base, 0);
    const uint32_t place = base + static_cast<uint32_t>(__popcll(who & ((uint64_t{1} << lane) - 1)));
    if (take && place < kList) s.list[place] = o;
  }

  // Tokens with keys from `least` on; how many there are (over kList: too many).
  __device__ __forceinline__ uint32_t candidates(uint32_t least) {
    __syncthreads();
    if (threadIdx.x == 0) {
      s.n = 0;
      s.found = 0;
    }
    __syncthreads();
    const uint32_t* tops = a.tops + row * a.n64;
    for (int64_t i = threadIdx.x; i < a.n64; i += kThreads)
      if (tops[i] >= least) {
        const uint32_t at = atomicAdd(&s.found, 1u);
        if (at < 2 * kBins) s.count[at] = static_cast<uint32_t>(i);
      }
    __syncthreads();
    const uint32_t spans = s.found;
    if (spans > 2 * kBins) return kList + 1;
    for (uint32_t i = threadIdx.x >> 6; i < spans; i += kWaves) {
      const int64_t c = s.count[i] * int64_t{64} + (threadIdx.x & 63);
      const float y = c < a.v ? static_cast<float>(x[c]) : -INFINITY;
      append(c < a.v && key_of(y) >= least, order_of(y, c));
    }
    __syncthreads();
    return s.n;
  }

  // The list's first n in descending order; how many entries that are with the zeros
  // after them (a power of two).
  __device__ __forceinline__ uint32_t sort(uint32_t n) {
    uint32_t size = 64;
    while (size < n) size *= 2;
    __syncthreads();
    for (uint32_t i = n + threadIdx.x; i < size; i += kThreads) s.list[i] = 0;
    __syncthreads();
    for (uint32_t run = 2; run <= size; run *= 2) {
      for (uint32_t d = run / 2; d; d /= 2) {
        for (uint32_t q = threadIdx.x; q < size / 2; q += kThreads) {
          const uint32_t i = q / d * 2 * d + q % d, j = i + d;
          const uint64_t u = s.list[i], w = s.list[j];
          if ((u < w) == ((i & run) == 0)) {
            s.list[i] = w;
            s.list[j] = u;
          }
        }
        __syncthreads();
      }
    }
    return size;
  }

  __device__ __forceinline__ float listed(uint32_t i) const { return value_of(static_cast<uint32_t>(s.list[i] >> 32)); }

  // From the tokens whose keys are at least `least`, where they are few enough and
  // known to hold all that are kept (`complete`, or the cut is among them).
  __device__ __forceinline__ bool from_list(uint32_t least, bool complete, double all_mass) {
    const uint32_t n = candidates(least);
    if (n > kList) return false;
    const uint32_t size = sort(n), per = size > kThreads ? size / kThreads : 1, i0 = threadIdx.x * per;
    const uint32_t most = r.k ? static_cast<uint32_t>(r.k) : n;
    double w[kList / kThreads], mine = 0., all;
#pragma unroll
    for (uint32_t q = 0; q < kList / kThreads; ++q) {
      w[q] = q < per && i0 + q < n && i0 + q < most ? weight(listed(i0 + q)) : 0.;
      mine += w[q];
    }
    const double upto = block_scan(mine, s.waves, all);
    const double limit = r.p < 1.f ? static_cast<double>(r.p) * (r.k ? all : all_mass) : INFINITY;
    double before = upto - mine;
    uint32_t kept = 0;
#pragma unroll
    for (uint32_t q = 0; q < kList / kThreads; ++q) {
      const uint32_t i = i0 + q;
      if (q < per && i < n && i < most && (i == 0 || (before < limit && w[q] >= static_cast<double>(r.m)))) kept = i + 1;
      before += w[q];
    }
    const uint32_t count = block_most(kept, reinterpret_cast<uint32_t*>(s.waves64));
    if (!r.k && !complete && count == n) return false;
    // the kept ones in the order of the vocabulary
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < count; i += kThreads) s.list[i] = s.list[i] << 32 | s.list[i] >> 32;
    const uint32_t size2 = sort(count), per2 = size2 > kThreads ? size2 / kThreads : 1, j0 = threadIdx.x * per2;
    mine = 0.;
#pragma unroll
    for (uint32_t q = 0; q < kList / kThreads; ++q) {
      w[q] = q < per2 && j0 + q < count ? weight(value_of(static_cast<uint32_t>(s.list[j0 + q]))) : 0.;
      mine += w[q];
    }
    const double upto2 = block_scan(mine, s.waves, all);
    const double target = static_cast<double>(r.u) * all;
    const int t = crossing(mine, upto2, target);
    if (static_cast<int>(threadIdx.x) == t) {
      double sum = upto2 - mine;
      uint32_t pick = j0;
#pragma unroll
      for (uint32_t q = 0; q < kList / kThreads; ++q) {
        if (q < per2 && j0 + q < count && w[q] > 0.) {
          if (!(sum > target)) pick = j0 + q;
          sum += w[q];
        }
      }
      const uint64_t e = s.list[pick];
      done(static_cast<int64_t>(static_cast<uint32_t>(~static_cast<uint32_t>(e >> 32))),
           exponent(value_of(static_cast<uint32_t>(e))) - log(all));
    }
    return true;
  }

  // ---- rows whose kept tokens are many: selection over the whole row
  template <typename F>
  __device__ __forceinline__ void each(F&& f) const {
    for (int64_t c = threadIdx.x; c < (a.v + kThreads - 1) / kThreads * kThreads; c += kThreads)
      f(c, c < a.v ? at(c) : -INFINITY);
  }

  // Of the tokens from `cut` on in descending order, the last one kept: the k-th (`by`
  // k), or the first up to which the masses add to `goal` (k 0). `mass`: of the tokens
  // up to it.
  __device__ __forceinline__ uint64_t select(uint64_t cut, int64_t k, double goal, double& mass) {
    // Bins of equal width below the largest value; where one of them holds too many
    // tokens, bins of equal width of its keys.
    const float width = fminf(static_cast<float>(kBins) / 24.f * static_cast<float>(r.inv_t), 1e30f);
    uint32_t first = 0, lo = 0, hi = 0;
    int level = 0, shift = 0;
    double above = 0.;
    int64_t n_above = 0;
    // weights in fixed point, at most 2^42 each: added in any order they are the same
    constexpr double kOne = 4398046511104.;
    auto bin0 = [&](float y) { return static_cast<uint32_t>(fminf((top - y) * width, static_cast<float>(kBins - 1))); };
    auto member = [&](int64_t c, float y) {
      return y > -INFINITY && order_of(y, c) >= cut && (level == 0 || (bin0(y) == first && key_of(y) >= lo && key_of(y) <= hi));
    };
    while (true) {
      __syncthreads();
      for (int b = threadIdx.x; b < kBins; b += kThreads) {
        s.count[b] = 0;
        s.mass[b] = 0;
      }
      __syncthreads();
      each([&](int64_t c, float y) {
        if (!member(c, y)) return;
        const uint32_t b = level == 0 ? bin0(y) : (hi - key_of(y)) >> shift;
        atomicAdd(&s.count[b], 1u);
        atomicAdd(reinterpret_cast<unsigned long long*>(&s.mass[b]),
                  static_cast<unsigned long long>(weight(y) * kOne + .5));
      });
      __syncthreads();
      const int b = 2 * static_cast<int>(threadIdx.x);
      const uint64_t c0 = s.count[b], c1 = s.count[b + 1], m0 = s.mass[b], m1 = s.mass[b + 1];
      uint64_t n_all, m_all;
      const uint64_t n_upto = block_scan<uint64_t>(c0 + c1, s.waves64, n_all);
      const uint64_t m_upto = block_scan<uint64_t>(m0 + m1, s.waves64, m_all);
      auto reached = [&](uint64_t n, uint64_t m) {
        return k ? n_above + static_cast<int64_t>(n) >= k : above + static_cast<double>(m) / kOne >= goal;
      };
      // the first bin that reaches it, or else the last one with tokens
      uint32_t mine = 0;
      if (c0 && reached(n_upto - c1, m_upto - m1)) mine = 0x80000000u | (kBins - b);
      else if (c1 && reached(n_upto, m_upto)) mine = 0x80000000u | (kBins - b - 1);
      else if (c1) mine = 2u + b;
      else if (c0) mine = 1u + b;
      const uint32_t best = block_most(mine, reinterpret_cast<uint32_t*>(s.waves));
      const uint32_t bin = best & 0x80000000u ? kBins - (best & 0x7fffffffu) : best - 1;
      if (bin / 2 == threadIdx.x) {
        const bool odd = bin & 1;
        s.waves64[0] = n_upto - c1 - (odd ? 0 : c0);
        s.waves64[1] = m_upto - m1 - (odd ? 0 : m0);
      }
      __syncthreads();
      n_above += static_cast<int64_t>(s.waves64[0]);
      above += static_cast<double>(s.waves64[1]) / kOne;
      const uint32_t here = s.count[bin];
      __syncthreads();
      if (level == 0) {
        first = bin;
        lo = 0;
        hi = kNan;
      } else {
        const uint32_t h = hi - (bin << shift);
        lo = h - lo > (uint32_t{1} << shift) - 1 ? h - ((uint32_t{1} << shift) - 1) : lo;
        hi = h;
      }
      ++level;
      if (here <= kList) break;
      // the members' own range of keys
      uint32_t least = kNan, most = 0;
      each([&](int64_t c, float y) {
        if (!member(c, y)) return;
        const uint32_t key = key_of(y);
        least = key < least ? key : least;
        most = key > most ? key : most;
      });
      hi = block_most(most, reinterpret_cast<uint32_t*>(s.waves));
      lo = ~block_most(~least, reinterpret_cast<uint32_t*>(s.waves));
      if (lo == hi) {   // more equal values than the list holds
        const double w = weight(value_of(hi));
        int64_t want = k ? k - n_above : static_cast<int64_t>(fmin(ceil((goal - above) / w), static_cast<double>(here)));
        want = want < 1 ? 1 : want > here ? here : want;
        mass = above + static_cast<double>(want) * w;
        // the want-th of them
        uint64_t seen = 0, o = 0;
        for (int64_t c0 = 0; c0 < a.v; c0 += kThreads) {
          const int64_t c = c0 + threadIdx.x;
          const float y = c < a.v ? at(c) : -INFINITY;
          const bool is = c < a.v && key_of(y) == hi && member(c, y);
          uint64_t all;
          const uint64_t upto = seen + block_scan<uint64_t>(is ? 1 : 0, s.waves64, all);
          if (is && static_cast<int64_t>(upto) == want) o = order_of(y, c);
          seen += all;
          if (static_cast<int64_t>(seen) >= want) break;
        }
        return block_most(o, s.waves64);
      }
      shift = 0;
      while ((hi - lo) >> shift >= kBins) ++shift;
    }
    if (threadIdx.x == 0) s.n = 0;
    __syncthreads();
    each([&](int64_t c, float y) { append(member(c, y), order_of(y, c)); });
    __syncthreads();
    const uint32_t n = s.n, size = sort(n), per = size > kThreads ? size / kThreads : 1, i0 = threadIdx.x * per;
    double w[kList / kThreads], mine = 0., all;
#pragma unroll
    for (uint32_t q = 0; q < kList / kThreads; ++q) {
      w[q] = q < per && i0 + q < n ? weight(listed(i0 + q)) : 0.;
      mine += w[q];
    }
    double sum = above + block_scan(mine, s.waves, all) - mine;
    uint32_t best = 0;   // larger: earlier
    double through = 0.;
#pragma unroll
    for (uint32_t q = 0; q < kList / kThreads; ++q) {
      const uint32_t i = i0 + q;
      sum += w[q];
      if (q < per && i < n && !(best & 0x80000000u)) {
        const bool is = k ? n_above + i + 1 >= k : sum >= goal;
        best = is ? 0x80000000u | (kList - i) : 1u + i;
        through = sum;
      }
    }
    const uint32_t found = block_most(best, reinterpret_cast<uint32_t*>(s.waves64));
    const uint32_t i = found & 0x80000000u ? kList - (found & 0x7fffffffu) : found - 1;
    if (best == found) s.before = through;
    __syncthreads();
    mass = s.before;
    const uint64_t o = s.list[i];
    __syncthreads();
    return o;
  }

  __device__ __forceinline__ void general(double all_mass) {
    uint64_t cut = static_cast<uint64_t>(kNone + 1) << 32;
    double mass = all_mass;
    if (r.k) cut = select(cut, r.k, 0., mass);
    if (r.p < 1.f) {
      double through;
      cut = select(cut, 0, static_cast<double>(r.p) * mass, through);
    }
    const double least = static_cast<double>(r.m);
    // the kept masses of the groups, a wave a group
    __syncthreads();
    for (int64_t g = threadIdx.x >> 6; g < a.n1024; g += kWaves) {
      Tokens<E> t;
      t.load(x, g, a.v);
      double sum = 0.;
#pragma unroll
      for (int i = 0; i < Tokens<E>::kLoads; ++i)
#pragma unroll
        for (int k = 0; k < Tokens<E>::kPer; ++k) {
          const float y = value(t.x[i * Tokens<E>::kPer + k]);
          const double w = weight(y);
          if (order_of(y, Tokens<E>::column(g, i) + k) >= cut && w >= least) sum += w;
        }
      sum = wave_sum(sum);
      if ((threadIdx.x & 63) == 0) s.group[g] = sum;
    }
    __syncthreads();
    by_groups(static_cast<int64_t>(threadIdx.x) < a.n1024 ? s.group[threadIdx.x] : 0., cut, least);
  }

  __device__ __forceinline__ void run() {
    const uint32_t key = block_most(
        static_cast<int64_t>(threadIdx.x) < a.n1024 ? a.firsts[row * a.n1024 + threadIdx.x] : 0u,
        reinterpret_cast<uint32_t*>(s.waves64));
    if (r.bad || key == kNan || key <= kNone) {
      if (threadIdx.x == 0) done(-1, NAN);
      return;
    }
    if (r.first) {
      largest(key);
      return;
    }
    inf = key == kInf;
    top = inf ? 0.f : value_of(key);
    const bool all = whole(r);
    double mass = 0.;
    if (all) {
      const double mine = group_mass();
      if (r.p >= 1.f) {
        by_groups(mine, 0, 0.);
        return;
      }
      block_scan(mine, s.waves, mass);
    }
    if (!inf) {
      if (r.k) {
        if (r.k <= a.n64 && from_list(kth_top(r.k), true, 0.)) return;
      } else {
        uint32_t floor = kNone + 1;
        if (r.m > 0.f) {   // nothing under it is kept
          const double y = top + static_cast<double>(r.t) * log(static_cast<double>(r.m));
          // (under it by more than the roundings of y, of f and of a mass)
          const float f = static_cast<float>(y - 1e-6 * (fabs(y) + fabs(static_cast<double>(top)) + static_cast<double>(r.t)));
          floor = f > -INFINITY ? key_of(f) : kNone + 1;
          if (from_list(floor, true, mass)) return;
        }
        if (r.p < 1.f) {
          for (int64_t c = 64; c <= 1024 && c <= a.n64; c *= 16) {
            const uint32_t least = kth_top(c);
            if (from_list(least > floor ? least : floor, least <= floor, mass)) return;
          }
        }
      }
    }
    general(mass);
  }
};

template <typename E>
__global__ __launch_bounds__(kThreads) void sample_pick_kernel(SampleArgs a) {
  __shared__ Shared s;
  const int64_t row = blockIdx.x;
  Pick<E> p{a, s, row, row_of(a, row), static_cast<const E*>(a.x) + row * a.ldx, 0.f, false};
  p.run();
}

template <typename E>
hipError_t sample(const SampleArgs& a, hipStream_t stream) {
  const int64_t blocks = (a.n * a.n1024 + 3) / 4;
  if (blocks > most_blocks(256) || a.n > most_blocks(kThreads)) return hipErrorInvalidValue;
  hipLaunchKernelGGL(sample_groups_kernel<E>, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, stream, a);
  hipLaunchKernelGGL(sample_pick_kernel<E>, dim3(static_cast<unsigned>(a.n)), dim3(kThreads), 0, stream, a);
  return hipGetLastError();
}

}  // namespace

int64_t sample_scratch(int64_t n, int64_t v, int64_t* tops, int64_t* firsts) {
  auto up = [](int64_t b) { return (b + 255) / 256 * 256; };
  const int64_t n64 = (v + 63) / 64, n1024 = (v + kGroup - 1) / kGroup;
  *tops = up(n * n1024 * 8);
  *firsts = *tops + up(n * n64 * 4);
  return *firsts + up(n * n1024 * 4);
}

hipError_t launch_sample(const SampleArgs& a, DType t, hipStream_t stream) {
  return t == DType::BF16 ? sample<__bf16>(a, stream) : sample<float>(a, stream);
}

}  // namespace orda
