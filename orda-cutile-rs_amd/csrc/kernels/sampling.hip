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

// e^z of z <= 0 in 64 bits: z·32/ln 2 = 32·n + j + f, |f| <= 1/2, and e^z = 2^n · 2^(j/32)
// · e^(f ln 2/32), the last by its series (the first term left out is 1.2e-12), 2^(j/32)
// from a table in LDS whose 64 words lie in 64 banks. 15 vector instructions and a read
// of LDS; without a table the series takes eight terms more.
__device__ const double kPowers[32] = {
    1.0, 1.0218971486541166, 1.0442737824274138, 1.0671404006768237,
    1.0905077326652577, 1.1143867425958924, 1.1387886347566916, 1.1637248587775775,
    1.189207115002721, 1.215247359980469, 1.241857812073484, 1.2690509571917332,
    1.2968395546510096, 1.3252366431597413, 1.3542555469368927, 1.383909881963832,
    1.4142135623730951, 1.4451808069770467, 1.4768261459394993, 1.5091644275934228,
    1.5422108254079407, 1.5759808451078865, 1.6104903319492543, 1.645755478153965,
    1.681792830507429, 1.718619298122478, 1.7562521603732995, 1.7947090750031072,
    1.8340080864093424, 1.8741676341103, 1.9152065613971474, 1.9571441241754002,
};
struct Exp {
  const double* powers;   // kPowers, in LDS
  double top, scale;      // of e^((x - top) / t): scale = 32 / (t ln 2)
  // (Next to nothing, not 0, below e^-690.)
  __device__ __forceinline__ double rough(float x) const {
    constexpr double kMagic = 6755399441055744., y = 0.021660849392498290084;   // 1.5 · 2^52; ln 2 / 32
    const double t = fmax((static_cast<double>(x) - top) * scale, -32000.);
    const double d = t + kMagic;   // its low word is round(t)
    const double f = t - (d - kMagic);
    double p = fma(f, y * y * y * y / 24., y * y * y / 6.);
    p = fma(p, f, y * y / 2.);
    p = fma(p, f, y);
    p = fma(p, f, 1.);
    const int k = __double2loint(d);
    p *= powers[k & 31];
    return __hiloint2double(__double2hiint(p) + (k >> 5) * (1 << 20), __double2loint(p));
  }
  // 0 below e^-690 (and of -infinity).
  __device__ __forceinline__ double operator()(float x) const {
    return (static_cast<double>(x) - top) * scale > -690. * 46.166241308446828384 ? rough(x) : 0.;
  }
};
__device__ __forceinline__ void load_powers(double* powers) {
  if (threadIdx.x < 32) powers[threadIdx.x] = kPowers[threadIdx.x];
}

struct Row {
  float t, p, m, u;
  int64_t k;
  double scale;      // 32 / (t ln 2)
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
  r.scale = 46.166241308446828384 / static_cast<double>(r.t);
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
// The largest of each 64 and of each 1024 tokens, as keys, and where they are needed
// the sum of each 1024's masses, relative to its largest: one read of the logits.
__device__ __forceinline__ float max3(float a, float b, float c) {   // (a NaN is looked for apart)
  float m;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(m) : "v"(a), "v"(b), "v"(c));
  return m;
}
template <typename E>
__global__ __launch_bounds__(256) void sample_groups_kernel(SampleArgs a) {
  using T = Tokens<E>;
  __shared__ double powers[32];
  load_powers(powers);
  __syncthreads();
  const int64_t row = blockIdx.y, group = blockIdx.x * int64_t{4} + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (group >= a.n1024) return;
  T t;
  t.load(static_cast<const E*>(a.x) + row * a.ldx, group, a.v);
  constexpr int kLanes = 64 / T::kPer;   // that hold 64 neighbouring tokens
  float top = -INFINITY;
  bool nan = false;
#pragma unroll
  for (int i = 0; i < T::kLoads; ++i) {
    const float* y = t.x + i * T::kPer;
    float m = max3(y[0], y[1], y[2]);
    bool bad = __builtin_isunordered(y[0], y[1]) || __builtin_isunordered(y[2], y[3]);
    if constexpr (T::kPer == 8) {
      m = max3(max3(m, y[3], y[4]), y[5], max3(y[6], y[7], y[7]));
      bad = bad || __builtin_isunordered(y[4], y[5]) || __builtin_isunordered(y[6], y[7]);
    } else {
      m = max3(m, y[3], y[3]);
    }
    uint32_t key = bad ? kNan : key_of(m);
#pragma unroll
    for (int d = 1; d < kLanes; d *= 2) {
      const uint32_t o = __shfl_xor(key, d);
      key = o > key ? o : key;
    }
    const int64_t at = group * (kGroup / 64) + i * T::kPer + lane / kLanes;
    if (lane % kLanes == 0 && at < a.n64) a.tops[row * a.n64 + at] = key;
    nan = nan || key == kNan;
    top = max3(top, value_of(key), top);
  }
  uint32_t key = nan ? kNan : key_of(top);
#pragma unroll
  for (int d = kLanes; d < 64; d *= 2) {
    const uint32_t o = __shfl_xor(key, d);
    key = o > key ? o : key;
  }
  if (lane == 0) a.firsts[row * a.n1024 + group] = key;
  const Row r = row_of(a, row);
  if (!whole(r)) return;
  double mass = 0.;
  if (key >= kInf) {
#pragma unroll
    for (int k = 0; k < 16; ++k) mass += t.x[k] == INFINITY ? 1. : 0.;
  } else if (key > kNone) {
    const Exp e{powers, static_cast<double>(value_of(key)), r.scale};
    double part = 0.;
#pragma unroll
    for (int k = 0; k < 16; k += 2) {
      mass += e.rough(t.x[k]);
      part += e.rough(t.x[k + 1]);
    }
    mass += part;
  }
  mass = wave_sum(mass);
  if (lane == 0) a.masses[row * a.n1024 + group] = mass;
}

// ---------------------------------------------------------------- picking
struct Shared {
  uint64_t list[kList];        // candidates, key over the token's complement
  uint64_t mass[kBins];        // of bins, in fixed point; or of groups
  uint32_t count[2 * kBins];   // of bins; or the 64s that hold candidates
  double group[kGroup];
  double powers[32];
  uint64_t waves[2][kWaves];
  uint32_t n, found;
  double value;
};

__device__ __forceinline__ uint64_t order_of(float x, int64_t c) {
  return static_cast<uint64_t>(key_of(x)) << 32 | static_cast<uint32_t>(~static_cast<uint32_t>(c));
}
__device__ __forceinline__ int64_t token_of(uint32_t low) { return static_cast<int64_t>(static_cast<uint32_t>(~low)); }

// A mass of at most 1 in fixed point, added in any order the same: 2^20 of them fit
// in 64 bits. (The sum's mantissa holds it: 512 has 2^-43 as its last bit.)
constexpr double kFixed = 8796093022208.;
__device__ __forceinline__ unsigned long long fixed_of(double w) {
  return static_cast<unsigned long long>(__double_as_longlong(w + 512.)) & ((1ull << 52) - 1);
}

// What one lane writes to LDS is there for the others of its wave.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}
// Over the workgroup: the largest.
template <typename T>
__device__ __forceinline__ T block_most(T v, Shared& s) {
  T* waves = reinterpret_cast<T*>(s.waves[0]);
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
template <typename T>
__device__ __forceinline__ T wave_scan(T v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const T o = __shfl_up(v, d);
    if (lane >= d) v += o;
  }
  return v;
}
// Sum of the values up to this thread's, and of all.
template <typename T>
__device__ __forceinline__ T block_scan(T v, Shared& s, T& all) {
  T* waves = reinterpret_cast<T*>(s.waves[1]);
  const int wave = threadIdx.x >> 6;
  v = wave_scan(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) waves[wave] = v;
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
  Exp mass_of;
  bool inf;   // the largest is +infinity: those tokens count as 0, the others as -infinity

  __device__ __forceinline__ float top() const { return static_cast<float>(mass_of.top); }
  __device__ __forceinline__ float value(float y) const { return inf ? (y == INFINITY ? 0.f : -INFINITY) : y; }
  __device__ __forceinline__ double weight(float y) const { return mass_of(y); }

  __device__ __forceinline__ void none() const {
    if (threadIdx.x) return;
    a.token[row] = -1;
    if (a.logprob) a.logprob[row] = NAN;
  }
  __device__ __forceinline__ void done(int64_t c, double logp) const {
    a.token[row] = c;
    if (a.logprob) a.logprob[row] = static_cast<float>(logp);
  }
  __device__ __forceinline__ void done(int64_t c, float y, double mass) const {
    done(c, (static_cast<double>(y) - mass_of.top) / static_cast<double>(r.t) - log(mass));
  }

  // The thread in whose share a sum crosses `target`: the first whose sum up to it is
  // over the target, the last with a share where none is. Leaves the sum before it in
  // s.value.
  __device__ __forceinline__ int crossing(double share, double upto, double target) {
    uint32_t mine = 0;   // larger: earlier
    if (share > 0.) mine = upto > target ? 0x80000000u | (kThreads - threadIdx.x) : 1u + threadIdx.x;
    const uint32_t best = block_most(mine, s);
    const int t = best & 0x80000000u ? kThreads - static_cast<int>(best & 0x7fffffffu) : best ? static_cast<int>(best) - 1 : 0;
    if (static_cast<int>(threadIdx.x) == t) s.value = upto - share;
    __syncthreads();
    return t;
  }

  // Where the groups' masses, thread t's group's here, cross u times their sum, the
  // group's token: of the tokens from `cut` on in descending order, with masses of at
  // least `least`.
  __device__ __forceinline__ void by_groups(double mine, uint64_t cut, double least) {
    double mass, all;
    const double upto = block_scan(mine, s, mass);
    const double target = static_cast<double>(r.u) * mass;
    const int64_t c = crossing(mine, upto, target) * int64_t{kGroup} + threadIdx.x;
    const double before = s.value;
    float y = -INFINITY;
    double w = 0.;
    if (c < a.v) {
      y = value(static_cast<float>(x[c]));
      w = weight(y);
      if (order_of(y, c) < cut || w < least) w = 0.;
    }
    const double sum = before + block_scan(w, s, all);
    const int t = crossing(w, sum, target);
    if (static_cast<int>(threadIdx.x) == t) done(c, y, mass);
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
    const int64_t group = kThreads - static_cast<int64_t>(block_most(mine, s));
    const int64_t c = group * kGroup + threadIdx.x;
    mine = c < a.v && key_of(static_cast<float>(x[c])) == key ? kThreads - threadIdx.x : 0;
    const int t = kThreads - static_cast<int>(block_most(mine, s));
    if (static_cast<int>(threadIdx.x) == t) done(c, 0.);
  }

  // ---- few tokens: lists
  // A key that at least k of the 64s' largest keys reach, and not many more: from their
  // counts in bins of equal width.
  __device__ __forceinline__ uint32_t near_top(int64_t k) {
    const uint32_t* tops = a.tops + row * a.n64;
    uint32_t most = 0;   // of the complements
    for (int64_t i = threadIdx.x; i < a.n64; i += kThreads) {
      const uint32_t key = tops[i];
      if (key > kNone) most = ~key > most ? ~key : most;
    }
    for (int b = threadIdx.x; b < kBins; b += kThreads) s.count[b] = 0;
    const float high = top(), low = value_of(~block_most(most, s));
    const float width = static_cast<float>(kBins - 1) / (high - low);   // (none: infinite)
    auto bin = [&](float y) { return static_cast<uint32_t>(fminf(fmaxf((high - y) * width, 0.f), kBins - 1.f)); };
    for (int64_t i = threadIdx.x; i < a.n64; i += kThreads) {
      const uint32_t key = tops[i];
      if (key > kNone) atomicAdd(&s.count[bin(value_of(key))], 1u);
    }
    __syncthreads();
    const int b = 2 * static_cast<int>(threadIdx.x);
    const uint32_t c0 = s.count[b], c1 = s.count[b + 1];
    uint32_t all;
    const uint32_t upto = block_scan(c0 + c1, s, all);
    if (threadIdx.x == 0) s.found = kBins - 1;
    __syncthreads();
    if (upto >= k && upto - c0 - c1 < k) s.found = upto - c1 >= k ? b : b + 1;
    __syncthreads();
    // its lower end, and a little less for the roundings
    const float end = high - (static_cast<float>(s.found) + 1.f) / width;
    const float less = end - 1e-6f * (fabsf(high) + fabsf(end));
    return less > -INFINITY && s.found < kBins - 1 ? key_of(less) : kNone + 1;
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
      const uint32_t hi = s.count[b + 1], lo = s.count[b];
      uint32_t all;
      const uint32_t upto = block_scan(hi + lo, s, all);
      if (upto >= rank && upto - hi - lo < rank) {
        const uint32_t before = upto - hi - lo;
        const bool in_hi = before + hi >= rank;
        s.found = static_cast<uint32_t>(in_hi ? b + 1 : b);
        s.n = rank - (in_hi ? before : before + hi);
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
  // after them (a power of two). Distances under 64 go from lane to lane.
  __device__ __forceinline__ uint32_t sort(uint32_t n) {
    uint32_t size = 64;
    while (size < n) size *= 2;
    __syncthreads();
    for (uint32_t i = n + threadIdx.x; i < size; i += kThreads) s.list[i] = 0;
    __syncthreads();
    // runs of up to 64, and after each longer distance the ones under 64, in registers
    auto lanes = [&](uint32_t run_from, uint32_t run_to) {
      for (uint32_t i = threadIdx.x; i < size; i += kThreads) {
        uint64_t o = s.list[i];
        for (uint32_t run = run_from; run <= run_to; run *= 2)
          for (uint32_t d = run / 2 < 32 ? run / 2 : 32; d; d /= 2) {
            const uint64_t w = __shfl_xor(o, d);
            const bool larger = ((i & run) == 0) == ((i & d) == 0);   // keeps the larger of the two
            o = (o > w) == larger ? o : w;
          }
        s.list[i] = o;
      }
      __syncthreads();
    };
    lanes(2, 64);
    for (uint32_t run = 128; run <= size; run *= 2) {
      for (uint32_t d = run / 2; d >= 64; d /= 2) {
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
      lanes(run, run);
    }
    return size;
  }

  __device__ __forceinline__ static float listed(uint64_t o) { return value_of(static_cast<uint32_t>(o >> 32)); }

  // Up to 64 candidates by one wave (the others wait): each entry's rank is how many are
  // over it. The token, or false where the cut is not among them; `share`: of all masses.
  __device__ __forceinline__ bool from_few(uint32_t n, bool complete, double all_mass, double& share) {
    if (threadIdx.x < 64) {
      const uint32_t i = threadIdx.x;
      uint64_t o = i < n ? s.list[i] : 0;
      uint32_t rank = 0;
      for (uint32_t j = 0; j < n; ++j) rank += s.list[j] > o;
      wave_sync();
      if (i < n) s.list[rank] = o;
      wave_sync();
      const uint32_t most = r.k && r.k < n ? static_cast<uint32_t>(r.k) : n;
      o = i < most ? s.list[i] : 0;
      const double w = i < most ? weight(listed(o)) : 0.;
      const double upto = wave_scan(w), all = __shfl(upto, 63);
      const double limit = r.p < 1.f ? static_cast<double>(r.p) * (r.k ? all : all_mass) : INFINITY;
      const bool keep = i < most && (i == 0 || (upto - w < limit && w >= static_cast<double>(r.m)));
      const uint32_t count = static_cast<uint32_t>(__popcll(__ballot(keep)));
      const bool found = r.k || complete || count < n;
      if (found) {
        // in the order of the vocabulary
        if (keep) s.list[i] = o << 32 | o >> 32;
        wave_sync();
        const uint64_t mine = keep ? s.list[i] : 0;
        uint32_t place = 0;
        for (uint32_t j = 0; j < count; ++j) place += s.list[j] > mine;
        wave_sync();
        if (keep) s.list[place] = mine;
        wave_sync();
        const uint64_t e = i < count ? s.list[i] : 0;
        const float y = value_of(static_cast<uint32_t>(e));
        const double m = i < count ? weight(y) : 0.;
        const double sum = wave_scan(m), mass = __shfl(sum, 63);
        const double target = static_cast<double>(r.u) * mass;
        const uint64_t over = __ballot(m > 0. && sum > target), any = __ballot(m > 0.);
        const int t = over ? __ffsll(static_cast<unsigned long long>(over)) - 1 : 63 - __clzll(static_cast<long long>(any));
        if (static_cast<int>(i) == t) done(token_of(static_cast<uint32_t>(e >> 32)), y, mass);
      }
      if (i == 0) {
        s.found = found;
        s.value = all;
      }
    }
    __syncthreads();
    share = s.value / all_mass;
    const bool found = s.found;
    __syncthreads();
    return found;
  }

  // From the tokens whose keys are at least `least`, where they are few enough and
  // known to hold all that are kept (`complete`, or the cut is among them).
  __device__ __forceinline__ bool from_list(uint32_t least, bool complete, double all_mass, double& share) {
    share = 1.;
    const uint32_t n = candidates(least);
    if (n > kList) return false;
    if (n <= 64) return from_few(n, complete, all_mass, share);
    const uint32_t size = sort(n), per = size > kThreads ? size / kThreads : 1, i0 = threadIdx.x * per;
    const uint32_t most = r.k && r.k < n ? static_cast<uint32_t>(r.k) : n;
    double w[kList / kThreads], mine = 0., all;
#pragma unroll
    for (uint32_t q = 0; q < kList / kThreads; ++q) {
      w[q] = q < per && i0 + q < most ? weight(listed(s.list[i0 + q])) : 0.;
      mine += w[q];
    }
    double before = block_scan(mine, s, all) - mine;
    const double limit = r.p < 1.f ? static_cast<double>(r.p) * (r.k ? all : all_mass) : INFINITY;
    uint32_t kept = 0;
#pragma unroll
    for (uint32_t q = 0; q < kList / kThreads; ++q) {
      const uint32_t i = i0 + q;
      if (q < per && i < most && (i == 0 || (before < limit && w[q] >= static_cast<double>(r.m)))) kept = i + 1;
      before += w[q];
    }
    const uint32_t count = block_most(kept, s);
    share = all / all_mass;
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
    const double upto = block_scan(mine, s, all);
    const double target = static_cast<double>(r.u) * all;
    const int t = crossing(mine, upto, target);
    if (static_cast<int>(threadIdx.x) == t) {
      double sum = upto - mine;
      uint32_t pick = j0;
#pragma unroll
      for (uint32_t q = 0; q < kList / kThreads; ++q) {
        if (w[q] > 0.) {
          if (!(sum > target)) pick = j0 + q;
          sum += w[q];
        }
      }
      const uint64_t e = s.list[pick];
      done(token_of(static_cast<uint32_t>(e >> 32)), value_of(static_cast<uint32_t>(e)), all);
    }
    return true;
  }

  // ---- many tokens: selection over the whole row
  // f(token, value) of every token, a wave a group; ended(group) after each.
  template <typename F, typename G>
  __device__ __forceinline__ void each(F&& f, G&& ended) const {
    for (int64_t g = threadIdx.x >> 6; g < a.n1024; g += kWaves) {
      Tokens<E> t;
      t.load(x, g, a.v);
#pragma unroll
      for (int i = 0; i < Tokens<E>::kLoads; ++i)
#pragma unroll
        for (int k = 0; k < Tokens<E>::kPer; ++k)
          f(Tokens<E>::column(g, i) + k, value(t.x[i * Tokens<E>::kPer + k]));
      ended(g);
    }
  }

  // The groups' masses of the tokens from `cut` on, those of at least `least`.
  __device__ __forceinline__ void group_masses(uint64_t cut, double least) {
    double sum = 0.;
    __syncthreads();
    each([&](int64_t c, float y) {
      const double w = weight(y);
      if (order_of(y, c) >= cut && w >= least) sum += w;
    }, [&](int64_t g) {
      sum = wave_sum(sum);
      if ((threadIdx.x & 63) == 0) s.group[g] = sum;
      sum = 0.;
    });
    __syncthreads();
  }

  // Of the tokens from `cut` on in descending order the last one kept: the k-th (COUNT),
  // or the first up to which the masses add to `goal`. With `last` leaves the kept
  // tokens' masses of at least `least` in s.group and, those that stood in the list,
  // in s.mass; else returns all kept tokens' mass in `mass`.
  //
  // A pass counts or weighs the tokens in bins of equal width below the largest; the
  // bin that the cut is in goes to a list in the next, which also adds up what lies
  // above it, and the list is sorted. Where it is too long its keys are cut into bins
  // again.
  template <bool COUNT>
  __device__ __forceinline__ uint64_t select(uint64_t cut, bool cut_is, int64_t k, double goal, bool last, double least, double& mass) {
    // 24 units of e^x hold all masses that count; by ranks, what the 64s' largest span.
    float span = 24.f * r.t;
    if constexpr (COUNT) {
      uint32_t most = 0;
      for (int64_t i = threadIdx.x; i < a.n64; i += kThreads) {
        const uint32_t key = a.tops[row * a.n64 + i];
        if (key > kNone) most = ~key > most ? ~key : most;
      }
      const float low = value_of(~block_most(most, s));
      if (!inf) span = (top() - low) * 1.25f;
    }
    const float high = top(), width = fminf(static_cast<float>(kBins) / span, 1e30f);
    uint32_t first = 0, lo = 0, hi = 0;
    int level = 0, shift = 0;
    double above = 0.;
    uint32_t n_above = 0, n;
    auto bin0 = [&](float y) { return static_cast<uint32_t>(fminf((high - y) * width, kBins - 1.f)); };
    auto eligible = [&](int64_t c, float y) { return y > -INFINITY && (!cut_is || order_of(y, c) >= cut); };
    while (true) {
      __syncthreads();
      for (int b = threadIdx.x; b < kBins; b += kThreads) {
        if constexpr (COUNT) s.count[b] = 0;
        else s.mass[b] = 0;
      }
      __syncthreads();
      each([&](int64_t c, float y) {
        if (!eligible(c, y)) return;
        uint32_t b = bin0(y);
        if (level) {
          const uint32_t key = key_of(y);
          if (b != first || key < lo || key > hi) return;
          b = (hi - key) >> shift;
        }
        if constexpr (COUNT) atomicAdd(&s.count[b], 1u);
        else atomicAdd(reinterpret_cast<unsigned long long*>(&s.mass[b]), fixed_of(mass_of.rough(y)));
      }, [](int64_t) {});
      __syncthreads();
      // the first bin that reaches it, or else the last one with tokens
      const int b = 2 * static_cast<int>(threadIdx.x);
      uint64_t v0, v1;
      if constexpr (COUNT) v0 = s.count[b], v1 = s.count[b + 1];
      else v0 = s.mass[b], v1 = s.mass[b + 1];
      uint64_t all;
      const uint64_t upto = block_scan<uint64_t>(v0 + v1, s, all);
      auto reached = [&](uint64_t q) {
        if constexpr (COUNT) return n_above + static_cast<int64_t>(q) >= k;
        else return above + static_cast<double>(q) / kFixed >= goal;
      };
      uint32_t mine = 0;
      if (v0 && reached(upto - v1)) mine = 0x80000000u | (kBins - b);
      else if (v1 && reached(upto)) mine = 0x80000000u | (kBins - b - 1);
      else if (v1) mine = 2u + b;
      else if (v0) mine = 1u + b;
      const uint32_t best = block_most(mine, s);
      const uint32_t bin = best & 0x80000000u ? kBins - (best & 0x7fffffffu) : best ? best - 1 : 0;
      if (bin / 2 == threadIdx.x) s.list[0] = upto - v1 - (bin & 1 ? 0 : v0);
      __syncthreads();
      if constexpr (COUNT) n_above += static_cast<uint32_t>(s.list[0]);
      else above += static_cast<double>(s.list[0]) / kFixed;
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
      // the bin's tokens, the range of their keys, and the masses above them
      __syncthreads();
      if (threadIdx.x == 0) s.n = 0;
      __syncthreads();
      uint32_t low = kNan, most = 0;
      double sum = 0.;
      each([&](int64_t c, float y) {
        const bool is = eligible(c, y);
        const uint32_t b = is ? bin0(y) : kBins, key = key_of(y);
        const bool member = b == first && key >= lo && key <= hi;
        if (b < first || (b == first && key > hi)) {
          const double w = weight(y);
          if (w >= least) sum += w;
        }
        if (member) {
          low = key < low ? key : low;
          most = key > most ? key : most;
        }
        append(member, order_of(y, c));
      }, [&](int64_t g) {
        sum = wave_sum(sum);
        if ((threadIdx.x & 63) == 0) s.group[g] = sum;
        sum = 0.;
      });
      __syncthreads();
      n = s.n;
      if (n <= kList) break;
      hi = block_most(most, s);
      lo = ~block_most(~low, s);
      if (lo == hi) {   // more equal values than the list holds
        const double w = weight(value_of(hi));
        int64_t want;
        if constexpr (COUNT) want = k - n_above;
        else want = static_cast<int64_t>(fmin(ceil((goal - above) / w), static_cast<double>(n)));
        want = want < 1 ? 1 : want > n ? n : want;
        // the want-th of them
        uint64_t seen = 0, o = 0;
        for (int64_t c0 = 0; c0 < a.v && static_cast<int64_t>(seen) < want; c0 += kThreads) {
          const int64_t c = c0 + threadIdx.x;
          const float y = c < a.v ? value(static_cast<float>(x[c])) : -INFINITY;
          const bool is = c < a.v && key_of(y) == hi && eligible(c, y);
          uint64_t here;
          const uint64_t at = seen + block_scan<uint64_t>(is ? 1 : 0, s, here);
          if (is && static_cast<int64_t>(at) == want) o = order_of(y, c);
          seen += here;
        }
        o = block_most(o, s);
        if (last) {
          group_masses(o, least);
          for (int g = threadIdx.x; g < kGroup; g += kThreads) s.mass[g] = 0;
          __syncthreads();
        } else {
          block_scan(static_cast<int64_t>(threadIdx.x) < a.n1024 ? s.group[threadIdx.x] : 0., s, mass);
          mass += static_cast<double>(want) * w;
        }
        return o;
      }
      shift = 0;
      while ((hi - lo) >> shift >= kBins) ++shift;
    }
    const uint32_t size = sort(n), per = size > kThreads ? size / kThreads : 1, i0 = threadIdx.x * per;
    double w[kList / kThreads], mine = 0., all;
#pragma unroll
    for (uint32_t q = 0; q < kList / kThreads; ++q) {
      w[q] = q < per && i0 + q < n ? weight(listed(s.list[i0 + q])) : 0.;
      mine += w[q];
    }
    const double before = block_scan(mine, s, all) - mine;
    double sum = before;
    uint32_t best = 0;   // larger: earlier
#pragma unroll
    for (uint32_t q = 0; q < kList / kThreads; ++q) {
      const uint32_t i = i0 + q;
      sum += w[q];
      if (q < per && i < n && !(best & 0x80000000u)) {
        bool is;
        if constexpr (COUNT) is = n_above + i + 1 >= k;
        else is = above + sum >= goal;
        best = is ? 0x80000000u | (kList - i) : 1u + i;
      }
    }
    const uint32_t found = block_most(best, s);
    const uint32_t end = found & 0x80000000u ? kList - (found & 0x7fffffffu) : found ? found - 1 : 0;
    const uint64_t o = s.list[end];
    if (last) {
      for (int g = threadIdx.x; g < kGroup; g += kThreads) s.mass[g] = 0;
      __syncthreads();
#pragma unroll
      for (uint32_t q = 0; q < kList / kThreads; ++q)
        if (q < per && i0 + q <= end && w[q] >= least)
          atomicAdd(reinterpret_cast<unsigned long long*>(&s.mass[token_of(static_cast<uint32_t>(s.list[i0 + q])) / kGroup]),
                    fixed_of(w[q]));
      __syncthreads();
    } else {
      double through = 0.;
      sum = before;
#pragma unroll
      for (uint32_t q = 0; q < kList / kThreads; ++q) {
        sum += w[q];
        if (q < per && i0 + q == end) through = sum;
      }
      through = block_most(through, s);
      block_scan(static_cast<int64_t>(threadIdx.x) < a.n1024 ? s.group[threadIdx.x] : 0., s, mass);
      mass += through;
    }
    return o;
  }

  __device__ __forceinline__ void general(double all_mass) {
    const double least = static_cast<double>(r.m);
    uint64_t cut = static_cast<uint64_t>(kNone + 1) << 32;
    if (r.k && r.p < 1.f) cut = select<true>(cut, false, r.k, 0., false, 0., all_mass);
    if (r.p < 1.f) {
      double unused;
      cut = select<false>(cut, r.k != 0, 0, static_cast<double>(r.p) * all_mass, true, least, unused);
    } else if (r.k) {
      double unused;
      cut = select<true>(cut, false, r.k, 0., true, least, unused);
    } else {
      group_masses(cut, least);
    }
    double mine = 0.;
    if (static_cast<int64_t>(threadIdx.x) < a.n1024) {
      mine = s.group[threadIdx.x];
      if (r.k || r.p < 1.f) mine += static_cast<double>(s.mass[threadIdx.x]) / kFixed;
    }
    by_groups(mine, cut, least);
  }

  __device__ __forceinline__ void run() {
    const uint32_t key = block_most(static_cast<int64_t>(threadIdx.x) < a.n1024 ? a.firsts[row * a.n1024 + threadIdx.x] : 0u, s);
    if (r.bad || key == kNan || key <= kNone) {
      none();
      return;
    }
    if (r.first) {
      largest(key);
      return;
    }
    inf = key == kInf;
    mass_of.top = inf ? 0. : static_cast<double>(value_of(key));
    double mass = 1.;
    if (whole(r)) {
      const double mine = group_mass();
      if (r.p >= 1.f) {
        by_groups(mine, 0, 0.);
        return;
      }
      block_scan(mine, s, mass);
    }
    double share;
    if (!inf) {
      if (r.k) {
        if (r.k <= a.n64) {
          if (from_list(near_top(r.k), true, mass, share)) return;
          if (from_list(kth_top(r.k), true, mass, share)) return;   // (far from evenly spread)
        }
      } else {
        uint32_t floor = kNone + 1;
        if (r.m > 0.f) {   // nothing under it is kept
          const double y = mass_of.top + static_cast<double>(r.t) * log(static_cast<double>(r.m));
          // (under it by more than the roundings of y, of f and of a mass)
          const float f = static_cast<float>(y - 1e-6 * (fabs(y) + fabs(mass_of.top) + static_cast<double>(r.t)));
          floor = f > -INFINITY ? key_of(f) : kNone + 1;
          if (from_list(floor, true, mass, share)) return;
        }
        if (r.p < 1.f) {
          // Some 64 tokens, and where they hold a good part of the masses some 1000.
          for (int64_t c = 64; c <= 1024 && c <= a.n64; c *= 16) {
            const uint32_t least = near_top(c);
            if (from_list(least > floor ? least : floor, least <= floor, mass, share)) return;
            if (share < .5 * static_cast<double>(r.p)) break;
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
  load_powers(s.powers);   // (barriers follow before they are read)
  const Row r = row_of(a, row);
  Pick<E> p{a, s, row, r, static_cast<const E*>(a.x) + row * a.ldx, Exp{s.powers, 0., r.scale}, false};
  p.run();
}

template <typename E>
hipError_t sample(const SampleArgs& a, hipStream_t stream) {
  constexpr int64_t kRows = 65535;   // of a launch's second dimension
  const auto across = static_cast<unsigned>((a.n1024 + 3) / 4);
  for (int64_t r = 0; r < a.n; r += kRows) {
    SampleArgs p = a;
    const int64_t n = a.n - r < kRows ? a.n - r : kRows;
    auto past = [&](auto* q, int64_t each) { return q ? q + r * each : nullptr; };
    p.x = static_cast<const E*>(a.x) + r * a.ldx;
    p.u = a.u + r;
    p.t = past(a.t, 1);
    p.p = past(a.p, 1);
    p.m = past(a.m, 1);
    p.k = past(a.k, 1);
    p.token = a.token + r;
    p.logprob = past(a.logprob, 1);
    p.tops = a.tops + r * a.n64;
    p.firsts = a.firsts + r * a.n1024;
    p.masses = a.masses + r * a.n1024;
    hipLaunchKernelGGL(sample_groups_kernel<E>, dim3(across, static_cast<unsigned>(n)), dim3(256), 0, stream, p);
    hipLaunchKernelGGL(sample_pick_kernel<E>, dim3(static_cast<unsigned>(n)), dim3(kThreads), 0, stream, p);
  }
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
