// sampling.hip — tokens drawn from rows of logits with temperature, top-k, top-p and
// min-p, by one given number a row.
//
// The distribution function of a row has as many borders as tokens, so an error of
// d in it gives another token with a probability of about 2·d·V: masses and their
// sums are held in 64 bits.
//
// Nothing is sorted but a list of at most 2048 candidates. A first pass over the logits
// leaves the largest of each 64 tokens and, where all masses are needed, the mass of each
// 1024; then a workgroup a row takes the candidates from the 64s whose largest reach a
// bound (`pick`), and where the kept tokens are more than the list holds it finds the cut by
// bins, of which it lists one (`select`). (Both in one kernel, 42 KB of code: with
// `select` in a launch of its own the rows that need it waited for all others, 61 us in
// place of 45 for 64 x 50257 of mixed parameters.) The drawn token is then sought in its
// group of 1024 alone. Largest logits, masses and counts do not depend on the order
// in which they are formed, or are summed in fixed point or in a fixed order: the same bits
// in every run.
//
// By the profiler, which keeps launches apart (a call of those after one another beside it):
// 1 x 131072 fp32, top-k 50 and top-p 0.9: 3 us and 9 (16, of the host).
// 256 x 131072 fp32, top-p 0.95 of a flat distribution, the slowest kind: 34 us (4.0 TB/s)
// and 83 (107), of which the binning's and the listing's passes over the row, one workgroup
// a row, are the most. 512 x 131072 bf16, unfiltered: 58 us (20 instructions a token, nine
// of them in 64 bits) and 10 (58); greedy, without masses: 30 (4.5 TB/s)
// and 6 (35).
#include <math.h>

#include "orda_kernels.h"
#include "wave.h"

namespace orda {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;   // of the kernel that picks: a workgroup a row
constexpr int kGroup = 1024;                             // tokens whose mass is summed up first
constexpr int kBins = 2048, kList = 2048, kRing = 512;

// ---------------------------------------------------------------- keys, masses
// Keys order as the values do; equal values (0 and -0) have equal keys, NaN the
// largest.
constexpr uint32_t kNan = 0xffffffffu, kInf = 0xff800000u, kNone = 0x007fffffu;   // kNone: -infinity
__device__ __forceinline__ uint32_t key_of_number(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
}
__device__ __forceinline__ uint32_t key_of(float x) { return x != x ? kNan : key_of_number(x); }
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

// e^z of z <= 0 in 64 bits: z·256/ln 2 = 256·n + j + f, |f| <= 1/2, and e^z = 2^n · 2^(j/256)
// · e^y, y = f ln 2/256, the last by its series (the first term left out is 1.4e-13),
// 2^(j/256) from a table in LDS. Nine instructions of 64 bits (2.2 ns a wave's on its SIMD,
// where one of 32 takes 1.9) and three more, which bound the passes that weigh tokens.
constexpr int kPowers = 256;
__device__ const double kPower[kPowers] = {
    1.0, 1.0027112750502025, 1.0054299011128027, 1.0081558981184175,
    1.0108892860517005, 1.0136300849514894, 1.016378314910953, 1.019133996077738,
    1.0218971486541166, 1.0246677928971357, 1.0274459491187637, 1.030231637686041,
    1.0330248790212284, 1.0358256936019572, 1.0386341019613787, 1.041450124688316,
    1.0442737824274138, 1.0471050958792898, 1.0499440858006872, 1.0527907730046264,
    1.0556451783605572, 1.0585073227945128, 1.061377227289262, 1.0642549128844645,
    1.0671404006768237, 1.0700337118202419, 1.0729348675259756, 1.075843889062791,
    1.0787607977571199, 1.0816856149932152, 1.0846183622133092, 1.0875590609177697,
    1.0905077326652577, 1.0934643990728858, 1.0964290818163769, 1.099401802630222,
    1.102382583307841, 1.1053714457017412, 1.1083684117236787, 1.1113735033448175,
    1.1143867425958924, 1.1174081515673693, 1.1204377524096067, 1.12347556733302,
    1.1265216186082418, 1.129575928566288, 1.1326385195987192, 1.1357094141578055,
    1.1387886347566916, 1.1418762039695616, 1.1449721444318042, 1.148076478840179,
    1.1511892299529827, 1.154310420590216, 1.1574400736337511, 1.1605782120274988,
    1.1637248587775775, 1.1668800369524817, 1.1700437696832502, 1.1732160801636373,
    1.1763969916502812, 1.1795865274628758, 1.182784710984341, 1.1859915656609938,
    1.189207115002721, 1.1924313825831512, 1.1956643920398273, 1.1989061670743806,
    1.202156731452703, 1.2054161090051239, 1.2086843236265816, 1.2119613992768012,
    1.215247359980469, 1.2185422298274085, 1.2218460329727576, 1.2251587936371455,
    1.22848053610687, 1.2318112847340759, 1.2351510639369334, 1.2384998981998165,
    1.241857812073484, 1.245224830175258, 1.2486009771892048, 1.2519862778663162,
    1.255380757024691, 1.2587844395497165, 1.2621973503942507, 1.2656195145788063,
    1.2690509571917332, 1.2724917033894028, 1.275941778396392, 1.2794012075056693,
    1.2828700160787783, 1.2863482295460256, 1.2898358734066657, 1.2933329732290895,
    1.2968395546510096, 1.3003556433796506, 1.3038812651919358, 1.3074164459346773,
    1.3109612115247644, 1.3145155879493546, 1.318079601266064, 1.3216532776031575,
    1.3252366431597413, 1.3288297242059544, 1.3324325470831615, 1.3360451382041458,
    1.339667524053303, 1.3432997311868353, 1.3469417862329458, 1.3505937158920345,
    1.3542555469368927, 1.3579273062129011, 1.3616090206382248, 1.365300717204012,
    1.3690024229745905, 1.3727141650876684, 1.3764359707545302, 1.380167867260238,
    1.383909881963832, 1.387662042298529, 1.3914243757719262, 1.3951969099662003,
    1.3989796725383112, 1.4027726912202048, 1.4065759938190154, 1.4103896082172707,
    1.4142135623730951, 1.4180478843204152, 1.4218926021691656, 1.4257477441054942,
    1.42961333839197, 1.433489413367789, 1.4373759974489824, 1.4412731191286257,
    1.4451808069770467, 1.449099089642035, 1.4530279958490526, 1.4569675544014438,
    1.460917794180647, 1.4648787441464057, 1.4688504333369818, 1.4728328908693675,
    1.4768261459394993, 1.4808302278224719, 1.4848451658727524, 1.488870989524397,
    1.4929077282912648, 1.4969554117672355, 1.5010140696264256, 1.5050837316234065,
    1.5091644275934228, 1.5132561874526098, 1.5173590411982147, 1.5214730189088146,
    1.5255981507445384, 1.529734466947287, 1.533881997840956, 1.5380407738316568,
    1.5422108254079407, 1.5463921831410214, 1.550584877685, 1.5547889397770887,
    1.559004400237837, 1.5632312899713576, 1.567469639965553, 1.5717194812923414,
    1.5759808451078865, 1.5802537626528246, 1.5845382652524937, 1.588834384317164,
    1.593142151342267, 1.597461597908627, 1.6017927556826934, 1.606135656416771,
    1.6104903319492543, 1.6148568142048607, 1.6192351351948637, 1.6236253270173289,
    1.6280274218573478, 1.632441451987275, 1.6368674497669644, 1.6413054476440063,
    1.645755478153965, 1.6502175739206177, 1.6546917676561943, 1.6591780921616162,
    1.6636765803267364, 1.6681872651305825, 1.6727101796415966, 1.6772453570178785,
    1.681792830507429, 1.6863526334483934, 1.6909247992693053, 1.6955093614893326,
    1.7001063537185235, 1.7047158096580513, 1.709337763100463, 1.713972247929926,
    1.718619298122478, 1.723278947746274, 1.7279512309618377, 1.732636182022311,
    1.7373338352737062, 1.7420442251551564, 1.746767386199169, 1.7515033530318782,
    1.7562521603732995, 1.761013843037584, 1.7657884359332727, 1.7705759740635547,
    1.7753764925265212, 1.7801900265154245, 1.785016611318935, 1.789856282321401,
    1.7947090750031072, 1.7995750249405351, 1.804454167806624, 1.809346539371032,
    1.8142521755003989, 1.8191711121586085, 1.8241033854070534, 1.8290490314048973,
    1.8340080864093424, 1.8389805867758937, 1.843966568958626, 1.8489660695104508,
    1.8539791250833855, 1.8590057724288205, 1.864046048397789, 1.8690999899412386,
    1.8741676341103, 1.8792490180565602, 1.8843441790323345, 1.8894531543909392,
    1.8945759815869656, 1.8997126981765553, 1.9048633418176741, 1.9100279502703899,
    1.9152065613971474, 1.9203992131630474, 1.925605943636125, 1.930826790987627,
    1.9360617934922943, 1.9413109895286405, 1.9465744175792332, 1.9518521162309783,
    1.9571441241754002, 1.9624504802089273, 1.9677712232331759, 1.9731063922552343,
    1.978456026387951, 1.9838201648502194, 1.9891988469672663, 1.9945921121709402,
};
struct Exp {
  const double* powers;   // in LDS, as load_powers puts them there
  double top, inv;        // of e^((x - top) / t): inv = 1 / t
  double shift;           // top / t, rounded
  float t, low;           // low: of a mass next to nothing
  __device__ __forceinline__ Exp(const double* p, float t)
      : powers(p), top(0.), inv(1. / static_cast<double>(t)), shift(0.), t(t), low(0.f) {}
  __device__ __forceinline__ void from(float largest) {
    top = static_cast<double>(largest);
    shift = top * inv;
    low = fmaf(-700.f, t, largest);
  }
  // A sum of `sum`'s terms, which are e^shift / e^(top / t) too large: by a factor of 1 and
  // next to nothing.
  __device__ __forceinline__ double corrected(double sum) const { return fma(-fma(top, inv, -shift), sum, sum); }
  // e^u, -707 <= u <= 0, and `sum`.
  __device__ __forceinline__ double plus(double u, double sum) const {
    constexpr double kMagic = 6755399441055744., kStep = 2.7076061740622863e-3;   // 1.5 · 2^52; ln 2 / 256
    const double d = fma(u, 1. / kStep, kMagic);   // its low word is the nearest whole number
    const double y = fma(d - kMagic, -kStep, u);
    double p = fma(y, 1. / 6., .5);
    p = fma(p, y, 1.);
    p = fma(p, y, 1.);
    const int k = __double2loint(d);
    const double q = powers[k & (kPowers - 1)];
    return fma(p, __hiloint2double(__double2hiint(q) + k * (1 << 12), __double2loint(q)), sum);
  }
  // x/t - shift is one rounding of a value of its own size off: an instruction less than
  // the difference first. Not where shift's own rounding is more than `corrected` corrects,
  // nor where 700 t is no fp32 value. Masses under e^-700 are next to nothing, not 0: the
  // logit is held from `low` on (in 32 bits: a maximum in 64 takes twice as long).
  __device__ __forceinline__ bool near() const { return fabs(shift) < 1e6 && t < 1e35f && low > -INFINITY; }
  __device__ __forceinline__ double near_plus(float x, double sum) const {
    return plus(fma(static_cast<double>(__builtin_amdgcn_fmed3f(x, low, INFINITY)), inv, -shift), sum);
  }
  __device__ __forceinline__ double far_plus(float x, double sum) const {
    return plus(fmax((static_cast<double>(x) - top) * inv, -700.), sum);
  }
  // The mass itself, 0 below e^-690 (and of -infinity).
  __device__ __forceinline__ double operator()(float x) const {
    const double u = (static_cast<double>(x) - top) * inv;
    return u > -690. ? plus(u, 0.) : 0.;
  }
};
// k = 256 n + j added to the exponent as k · 2^12 is n and j / 256: the latter is taken out
// of the table's entry j before, for an instruction less than n alone.
__device__ __forceinline__ void load_powers(double* powers) {
  const int j = threadIdx.x;
  if (j >= kPowers) return;
  const double q = kPower[j];
  powers[j] = __hiloint2double(__double2hiint(q) - j * (1 << 12), __double2loint(q));
}

struct Row {
  float t, p, m, u;
  int64_t k;
  bool bad, first;   // first: only the largest logit is kept
};
__device__ __forceinline__ Row row_of(const SampleArgs& a, int64_t row) {
  Row r;
  r.t = uniform(a.t ? a.t[row] : a.t1);
  r.p = uniform(a.p ? a.p[row] : a.p1);
  r.m = uniform(a.m ? a.m[row] : a.m1);
  r.k = uniform(a.k ? a.k[row] : a.k1);
  r.u = uniform(a.u[row]);
  r.bad = !(r.t >= 0.f) || r.t == INFINITY || r.p != r.p || r.m != r.m || !(r.u >= 0.f && r.u <= 1.f);
  if (r.k <= 0 || r.k >= a.v) r.k = 0;
  r.first = r.t == 0.f || r.k == 1 || r.p <= 0.f || r.m > 1.f;
  return r;
}
// Whether the masses of all tokens are needed.
__device__ __forceinline__ bool whole(const Row& r) {
  return !r.bad && !r.first && r.k == 0 && (r.p < 1.f || r.m <= 0.f);
}


// A lane's 16 of a group's tokens, kPer neighbouring ones a load, as they lie in memory,
// so that a next group's can be under way.
template <typename E>
struct Tokens {
  static constexpr int kPer = 16 / sizeof(E), kLoads = 16 / kPer;
  E w[kLoads][kPer];
  __device__ __forceinline__ static int column(int i) {   // within the group, of load i
    return (i * 64 + static_cast<int>(threadIdx.x & 63)) * kPer;
  }
  __device__ __forceinline__ void fetch(const E* group) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) __builtin_memcpy(w[i], group + column(i), sizeof w[i]);
  }
  // -infinity past the row's end, n tokens on.
  __device__ __forceinline__ void fetch(const E* group, int64_t n) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
#pragma unroll
      for (int k = 0; k < kPer; ++k) w[i][k] = column(i) + k < n ? group[column(i) + k] : static_cast<E>(-INFINITY);
  }
  __device__ __forceinline__ void store(E* group) const {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) __builtin_memcpy(group + column(i), w[i], sizeof w[i]);
  }
  __device__ __forceinline__ float at(int i, int k) const { return static_cast<float>(w[i][k]); }
};

// ---------------------------------------------------------------- first pass
// The largest of each 64 and of each 1024 tokens, as keys, and where they are needed
// the sum of each 1024's masses, relative to its largest: one read of the logits, a wave
// a group (so that many rows and one row alike fill the device). A row's last 1024, where
// they are fewer, are copied and filled up, so that later passes read whole ones. Bound by
// HBM for fp32 and by 20 instructions a token for bf16; reads past the
// caches gain 2 us of 66 there and nothing for fp32, and would take from the next pass
// what it finds in them.
__device__ __forceinline__ float max3(float a, float b, float c) {   // (a NaN is looked for apart)
  float m;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(m) : "v"(a), "v"(b), "v"(c));
  return m;
}
template <typename E>
__global__ __launch_bounds__(256) void sample_groups_kernel(SampleArgs a, int each) {
  using T = Tokens<E>;
  __shared__ double powers[kPowers];
  const int64_t row = blockIdx.y, from = blockIdx.x * int64_t{4} * each;
  const int64_t end = from + 4 * each < a.n1024 ? from + 4 * each : a.n1024;
  const int lane = threadIdx.x & 63;
  int64_t group = from + uniform(static_cast<int>(threadIdx.x >> 6));
  const E* const logits = static_cast<const E*>(a.x) + row * a.ldx;
  T raw;
  auto fetch = [&](int64_t g) {
    if ((g + 1) * kGroup <= a.v) {
      raw.fetch(logits + g * kGroup);
    } else {
      raw.fetch(logits + g * kGroup, a.v - g * kGroup);
      raw.store(static_cast<E*>(a.tails) + row * kGroup);
    }
  };
  if (group < end) fetch(group);
  load_powers(powers);
  const Row r = row_of(a, row);
  const bool weigh = whole(r);
  Exp e(powers, r.t);
  __syncthreads();
  for (; group < end; group += 4) {
    float x[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) x[k] = raw.at(k / T::kPer, k % T::kPer);
    if (group + 4 < end) fetch(group + 4);
    constexpr int kLanes = 64 / T::kPer;   // that hold 64 neighbouring tokens
    uint32_t key = 0, mine = 0;            // the largest; of lane i of each kLanes, load i's
#pragma unroll
    for (int i = 0; i < T::kLoads; ++i) {
      const float* y = x + i * T::kPer;
      float m = max3(y[0], y[1], y[2]);
      bool bad = __builtin_isunordered(y[0], y[1]) | __builtin_isunordered(y[2], y[3]);
      if constexpr (T::kPer == 8) {
        m = max3(max3(m, y[3], y[4]), y[5], max3(y[6], y[7], y[7]));
        bad |= __builtin_isunordered(y[4], y[5]) | __builtin_isunordered(y[6], y[7]);
      } else {
        m = max3(m, y[3], y[3]);
      }
      const uint32_t k64 = most_of<kLanes>(bad ? kNan : key_of_number(m));
      mine = lane % kLanes == i ? k64 : mine;
      key = k64 > key ? k64 : key;
    }
    const int64_t at = group * (kGroup / 64) + lane % kLanes * (64 / kLanes) + lane / kLanes;
    if (lane % kLanes < T::kLoads && at < a.n64) a.tops[row * a.n64 + at] = mine;
    key = most_of_rows<kLanes>(key);
    if (lane == 0) a.firsts[row * a.n1024 + group] = key;
    if (!weigh) continue;
    double mass = 0.;
    if (key >= kInf) {
#pragma unroll
      for (int k = 0; k < 16; ++k) mass += x[k] == INFINITY ? 1. : 0.;
    } else if (key > kNone) {
      e.from(value_of(key));
      if (e.near()) {
        double part = 0.;
#pragma unroll
        for (int k = 0; k < 16; k += 2) {
          mass = e.near_plus(x[k], mass);
          part = e.near_plus(x[k + 1], part);
        }
        mass = e.corrected(mass + part);
      } else {
#pragma unroll
        for (int k = 0; k < 16; ++k) mass = e.far_plus(x[k], mass);
      }
    }
    mass = wave_sum(mass);
    if (lane == 0) a.masses[row * a.n1024 + group] = mass;
  }
}

// ---------------------------------------------------------------- picking
struct Shared {
  uint64_t list[kList];            // candidates, key over the token's complement
  union {
    struct {
      uint64_t mass[kBins];        // of bins, in fixed point; or of groups
      uint32_t count[2 * kBins];   // of bins; or the 64s that hold candidates
    };
    float ring[kWaves][kRing];     // a wave's values to be weighed
  };
  double group[kGroup];
  double powers[kPowers];
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
  uint32_t tops[2];   // this thread's first two of the 64s' largest keys (most have no more)
  int turn = 0;       // of two places in LDS for the waves' values: a barrier a use is enough

  // Over the workgroup: the largest; the sum of the values up to this thread's, and of all.
  template <typename T>
  __device__ __forceinline__ T block_most(T v) {
    T* waves = reinterpret_cast<T*>(s.waves[turn]);
    turn ^= 1;
    v = wave_scan(v, Most{});
    if ((threadIdx.x & 63) == 63) waves[threadIdx.x >> 6] = v;
    __syncthreads();
    return lane_of(row_scan(waves[threadIdx.x % kWaves], Most{}), kWaves - 1);
  }
  template <typename T>
  __device__ __forceinline__ T block_scan(T v, T& all) {
    T* waves = reinterpret_cast<T*>(s.waves[turn]);
    turn ^= 1;
    v = wave_scan(v, Sum{});
    const int wave = uniform(static_cast<int>(threadIdx.x >> 6));
    if ((threadIdx.x & 63) == 63) waves[wave] = v;
    __syncthreads();
    const T upto = row_scan(waves[threadIdx.x % kWaves], Sum{});
    all = lane_of(upto, kWaves - 1);
    return wave ? v + lane_of(upto, wave - 1) : v;
  }

  __device__ __forceinline__ float top() const { return static_cast<float>(mass_of.top); }
  __device__ __forceinline__ float value(float y) const { return inf ? (y == INFINITY ? 0.f : -INFINITY) : y; }
  __device__ __forceinline__ double weight(float y) const { return mass_of(y); }

  // What the thread that finds the token sets, for finish().
  int64_t token = INT64_MIN;   // none
  double log_mass = 0., of = 1.;   // the log of its mass, the sum of the kept ones
  __device__ __forceinline__ void found(int64_t c, float y, double mass) {
    token = c;
    log_mass = (static_cast<double>(y) - mass_of.top) / static_cast<double>(r.t);
    of = mass;
  }
  __device__ __forceinline__ void finish() const {
    if (token == INT64_MIN) return;
    a.token[row] = token;
    if (a.logprob) a.logprob[row] = static_cast<float>(log_mass - log(of));
  }

  // The thread in whose share a sum crosses `target`: the first whose sum up to it is
  // over the target, the last with a share where none is. Leaves the sum before it in
  // s.value.
  __device__ __forceinline__ int crossing(double share, double upto, double target) {
    uint32_t mine = 0;   // larger: earlier
    if (share > 0.) mine = upto > target ? 0x80000000u | (kThreads - threadIdx.x) : 1u + threadIdx.x;
    const uint32_t best = block_most(mine);
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
    const double upto = block_scan(mine, mass);
    const double target = static_cast<double>(r.u) * mass;
    const int64_t c = crossing(mine, upto, target) * int64_t{kGroup} + threadIdx.x;
    const double before = uniform(s.value);
    float y = -INFINITY;
    double w = 0.;
    if (c < a.v) {
      y = value(static_cast<float>(x[c]));
      w = weight(y);
      if (order_of(y, c) < cut || w < least) w = 0.;
    }
    const double sum = before + block_scan(w, all);
    const int t = crossing(w, sum, target);
    if (static_cast<int>(threadIdx.x) == t) found(c, y, mass);
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
    const int64_t group = kThreads - static_cast<int64_t>(block_most(mine));
    const int64_t c = group * kGroup + threadIdx.x;
    mine = c < a.v && key_of(static_cast<float>(x[c])) == key ? kThreads - threadIdx.x : 0;
    const int t = kThreads - static_cast<int>(block_most(mine));
    if (static_cast<int>(threadIdx.x) == t) token = c;
  }

  // ---- few tokens: lists
  template <typename F>
  __device__ __forceinline__ void each_top(F&& f) const {
#pragma unroll
    for (int k = 0; k < 2; ++k) f(static_cast<int64_t>(threadIdx.x) + k * kThreads, tops[k]);
    for (int64_t i = threadIdx.x + 2 * int64_t{kThreads}; i < a.n64; i += kThreads) f(i, a.tops[row * a.n64 + i]);
  }
  // The smallest of them over -infinity.
  __device__ __forceinline__ float least_top() {
    uint32_t most = 0;   // of the complements
    each_top([&](int64_t, uint32_t key) { most = key > kNone && ~key > most ? ~key : most; });
    return value_of(~block_most(most));
  }
  // A key that at least k of them reach, and not many more: from their counts in bins of
  // equal width.
  __device__ __forceinline__ uint32_t near_top(int64_t k) {
    for (int b = threadIdx.x; b < kBins; b += kThreads) s.count[b] = 0;
    const float high = top(), low = least_top();
    const float width = static_cast<float>(kBins - 1) / (high - low);   // (none: infinite)
    each_top([&](int64_t, uint32_t key) {
      if (key > kNone)
        atomicAdd(&s.count[static_cast<uint32_t>(fminf(fmaxf((high - value_of(key)) * width, 0.f), kBins - 1.f))], 1u);
    });
    __syncthreads();
    const int b = 2 * static_cast<int>(threadIdx.x);
    const uint32_t c0 = s.count[b], c1 = s.count[b + 1];
    uint32_t all;
    const uint32_t upto = block_scan(c0 + c1, all);
    if (threadIdx.x == 0 && all < k) s.found = kBins - 1;
    if (upto >= k && upto - c0 - c1 < k) s.found = upto - c1 >= k ? b : b + 1;
    __syncthreads();
    // its lower end, and a little less for the roundings
    const uint32_t found = uniform(s.found);
    const float end = high - (static_cast<float>(found) + 1.f) / width;
    const float less = end - 1e-6f * (fabsf(high) + fabsf(end));
    return less > -INFINITY && found < kBins - 1 ? key_of(less) : kNone + 1;
  }
  // The k-th largest of them (1 <= k <= n64), 11, 11 and 10 bits at a time.
  __device__ __forceinline__ uint32_t kth_top(int64_t k) {
    uint32_t prefix = 0, mask = 0;
    uint32_t rank = static_cast<uint32_t>(k);
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
      const uint32_t digits = pass == 2 ? 1023 : 2047;
      __syncthreads();
      for (int b = threadIdx.x; b < kBins; b += kThreads) s.count[b] = 0;
      __syncthreads();
      each_top([&](int64_t i, uint32_t key) {
        if (i < a.n64 && (key & mask) == prefix) atomicAdd(&s.count[key >> shift & digits], 1u);
      });
      __syncthreads();
      const int b = kBins - 2 - 2 * static_cast<int>(threadIdx.x);   // bins b + 1, then b
      const uint32_t hi = s.count[b + 1], lo = s.count[b];
      uint32_t all;
      const uint32_t upto = block_scan(hi + lo, all);
      if (upto >= rank && upto - hi - lo < rank) {
        const uint32_t before = upto - hi - lo;
        const bool in_hi = before + hi >= rank;
        s.found = static_cast<uint32_t>(in_hi ? b + 1 : b);
        s.n = rank - (in_hi ? before : before + hi);
      }
      __syncthreads();
      prefix |= uniform(s.found) << shift;
      mask |= digits << shift;
      rank = uniform(s.n);
    }
    __syncthreads();
    return prefix;
  }

  // Puts a lane's N neighbouring tokens from c on into the list where `take`.
  template <int N>
  __device__ __forceinline__ void append(const bool (&take)[N], const float (&y)[N], int64_t c) {
    uint64_t who[N];
    uint32_t n = 0;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      who[k] = __ballot(take[k]);
      n += static_cast<uint32_t>(__popcll(who[k]));
    }
    if (!n) return;
    const int lane = threadIdx.x & 63;
    uint32_t place = 0;
    if (lane == 0) place = atomicAdd(&s.n, n);
    place = __builtin_amdgcn_readfirstlane(place);
    const uint64_t under = (uint64_t{1} << lane) - 1;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const uint32_t at = place + static_cast<uint32_t>(__popcll(who[k] & under));
      if (take[k] && at < kList) s.list[at] = order_of(y[k], c + k);
      place += static_cast<uint32_t>(__popcll(who[k]));
    }
  }

  // Tokens with keys from `least` on, from the 64s whose largest reach it, several of
  // them a load; how many tokens there are (over kList: too many).
  __device__ __forceinline__ uint32_t candidates(uint32_t least) {
    using T = Tokens<E>;
    __syncthreads();
    if (threadIdx.x == 0) {
      s.n = 0;
      s.found = 0;
    }
    __syncthreads();
    each_top([&](int64_t i, uint32_t key) {
      if (i >= a.n64 || key < least) return;
      const uint32_t at = atomicAdd(&s.found, 1u);
      if (at < 2 * kBins) s.count[at] = static_cast<uint32_t>(i);
    });
    __syncthreads();
    const uint32_t spans = uniform(s.found);
    if (spans > 2 * kBins) return kList + 1;
    constexpr uint32_t kLanes = 64 / T::kPer, kMany = 2;   // lanes of a span; loads under way
    const uint32_t lane = threadIdx.x & 63, step = 64 / kLanes;
    for (uint32_t i0 = (threadIdx.x >> 6) * step; i0 < spans; i0 += kWaves * step * kMany) {
      E w[kMany][T::kPer];
      int64_t c[kMany];
#pragma unroll
      for (uint32_t q = 0; q < kMany; ++q) {
        const uint32_t i = i0 + q * kWaves * step + lane / kLanes;
        c[q] = i < spans ? s.count[i] * int64_t{64} + lane % kLanes * T::kPer : a.v;
        if (c[q] + T::kPer <= a.v) {
          __builtin_memcpy(w[q], x + c[q], sizeof w[q]);
        } else {
#pragma unroll
          for (int k = 0; k < T::kPer; ++k) w[q][k] = c[q] + k < a.v ? x[c[q] + k] : static_cast<E>(-INFINITY);
        }
      }
#pragma unroll
      for (uint32_t q = 0; q < kMany; ++q) {
        float y[T::kPer];
        bool take[T::kPer];
#pragma unroll
        for (int k = 0; k < T::kPer; ++k) {
          y[k] = static_cast<float>(w[q][k]);
          take[k] = c[q] + k < a.v && key_of(y[k]) >= least;
        }
        append(take, y, c[q]);
      }
    }
    __syncthreads();
    return uniform(s.n);
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
  // over it. The token, or false where the cut is not among them.
  __device__ __forceinline__ bool from_few(uint32_t n, bool complete, double all_mass) {
    if (threadIdx.x < 64) {
      const uint32_t i = threadIdx.x;
      uint64_t o = i < n ? s.list[i] : 0;
      wave_sync();
      s.list[i] = o;
      wave_sync();
      uint32_t rank = 0;
      for (uint32_t j = 0; j < n; j += 8)
#pragma unroll
        for (uint32_t q = 0; q < 8; ++q) rank += s.list[j + q] > o;
      wave_sync();
      if (i < n) s.list[rank] = o;
      wave_sync();
      const uint32_t most = r.k && r.k < n ? static_cast<uint32_t>(r.k) : n;
      o = i < most ? s.list[i] : 0;
      const double w = i < most ? weight(listed(o)) : 0.;
      const double upto = wave_scan(w, Sum{}), all = lane_of(upto, 63);
      const double limit = r.p < 1.f ? static_cast<double>(r.p) * (r.k ? all : all_mass) : INFINITY;
      const bool keep = i < most && (i == 0 || (upto - w < limit && w >= static_cast<double>(r.m)));
      const uint32_t count = static_cast<uint32_t>(__popcll(__ballot(keep)));
      const bool is = r.k || complete || count < n;
      if (is) {
        // in the order of the vocabulary
        const uint64_t mine = keep ? o << 32 | o >> 32 : 0;
        s.list[i] = mine;
        wave_sync();
        uint32_t place = 0;
        for (uint32_t j = 0; j < count; j += 8)
#pragma unroll
          for (uint32_t q = 0; q < 8; ++q) place += s.list[j + q] > mine;
        wave_sync();
        if (keep) s.list[place] = mine;
        wave_sync();
        const uint64_t e = i < count ? s.list[i] : 0;
        const float y = value_of(static_cast<uint32_t>(e));
        const double m = i < count ? weight(y) : 0.;
        const double sum = wave_scan(m, Sum{}), mass = lane_of(sum, 63);
        const double target = static_cast<double>(r.u) * mass;
        const uint64_t over = __ballot(m > 0. && sum > target), any = __ballot(m > 0.);
        const int t = over ? __ffsll(static_cast<unsigned long long>(over)) - 1 : 63 - __clzll(static_cast<long long>(any));
        if (static_cast<int>(i) == t) found(token_of(static_cast<uint32_t>(e >> 32)), y, mass);
      }
      if (i == 0) s.found = is;
    }
    __syncthreads();
    const bool is = uniform(s.found);
    __syncthreads();
    return is;
  }

  // ---- many tokens: passes over the whole row
  // f(group, unit, first token, values): four neighbouring tokens a lane, four units a
  // group, a wave a group; the next group's under way. (One copy of f: the whole kernel
  // is to stay in the instruction cache. With f 16 times it was 237 KB, and every
  // stage waited for its code.)
  template <typename F>
  __device__ __forceinline__ void each(F&& f) const {
    using T = Tokens<E>;
    int g = uniform(static_cast<int>(threadIdx.x >> 6));
    const int groups = static_cast<int>(a.n1024), whole = static_cast<int>(a.v / kGroup);
    if (g >= groups) return;
    const E* tail = static_cast<const E*>(a.tails) + row * kGroup;
    T t;
    t.fetch(g < whole ? x + g * int64_t{kGroup} : tail);
    while (true) {
      float y[4][4];
#pragma unroll
      for (int k = 0; k < 16; ++k) y[k / 4][k % 4] = t.at(k / T::kPer, k % T::kPer);
      if (inf) {
#pragma unroll
        for (int k = 0; k < 16; ++k) y[k / 4][k % 4] = value(y[k / 4][k % 4]);
      }
      const int next = g + kWaves;
      if (next < groups) t.fetch(next < whole ? x + next * int64_t{kGroup} : tail);
#pragma unroll
      for (int unit = 0; unit < 4; ++unit)
        f(g, unit, g * int64_t{kGroup} + T::column(unit * 4 / T::kPer) + unit * 4 % T::kPer, y[unit]);
      if (next >= groups) return;
      g = next;
    }
  }

  __device__ __forceinline__ double sum_of_groups() {
    double all;
    block_scan(static_cast<int64_t>(threadIdx.x) < a.n1024 ? s.group[threadIdx.x] : 0., all);
    return all;
  }

  // What a pass over the row looks at: the tokens from `limit` on in descending order,
  // where there is one; of these it takes the ones over `hi` and lists the members, from
  // `lo` to `hi`.
  struct Cut {
    uint64_t limit;
    bool limited, by_count;
    float lo, hi;
    uint32_t most;              // hi's key, from which the bins of keys count down
    int level, shift;
    float high, width, slope, unit;   // bins of equal width below the largest; of log2 of a mass; what 1 weighs
  };
  __device__ __forceinline__ static uint32_t bin_of(const Cut& q, float y) {
    return static_cast<uint32_t>(fminf((q.high - y) * q.width, kBins - 1.f));
  }
  // The largest finite key whose value is in bin b or a later one (0: none), 64 of them
  // looked at at a time.
  __device__ __forceinline__ static uint32_t last_of(const Cut& q, uint32_t b) {
    uint32_t at = kNone + 1, n = key_of(q.high) - at;   // `at` is one, none of the n after it known
    if (bin_of(q, value_of(at)) < b) return 0;
    const uint32_t lane = threadIdx.x & 63;
    while (n) {
      const uint32_t step = (n + 63) / 64, past = (lane + 1) * step < n ? (lane + 1) * step : n;
      const uint32_t is = static_cast<uint32_t>(__popcll(__ballot(bin_of(q, value_of(at + past)) >= b)));
      const uint32_t move = is * step < n ? is * step : n;
      at += move;
      n = n - move < step - 1 ? n - move : step - 1;
    }
    return at;
  }

  // Counts or weighs the members in bins: all in 32 bits first, then (and by keys) in 64.
  __device__ __forceinline__ void fill_bins(const Cut& q) {
    __syncthreads();
    for (int b = threadIdx.x; b < kBins; b += kThreads) {
      s.mass[b] = 0;
      s.count[b] = 0;
    }
    __syncthreads();
    each([&](int, int, int64_t c, const float(&y)[4]) {
      if (q.level == 0) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (!(y[k] >= q.lo) || (q.limited && order_of(y[k], c + k) < q.limit)) continue;
          const uint32_t w = q.by_count ? 1u : static_cast<uint32_t>(__builtin_amdgcn_exp2f((q.high - y[k]) * q.slope) * q.unit);
          atomicAdd(&s.count[bin_of(q, y[k])], w);
        }
        return;
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (!(y[k] >= q.lo && y[k] <= q.hi) || (q.limited && order_of(y[k], c + k) < q.limit)) continue;
        atomicAdd(reinterpret_cast<unsigned long long*>(&s.mass[(q.most - key_of(y[k])) >> q.shift]),
                  q.by_count ? 1ull : fixed_of(weight(y[k])));
      }
    });
    __syncthreads();
  }

  // The first bin for which reached(its sum and those of the bins before), the last one
  // with a share where there is none.
  template <typename F>
  __device__ __forceinline__ uint32_t bin_where(uint64_t v0, uint64_t v1, uint64_t upto, F&& reached) {
    const int b = 2 * static_cast<int>(threadIdx.x);
    uint32_t mine = 0;
    if (v0 && reached(upto - v1)) mine = 0x80000000u | (kBins - b);
    else if (v1 && reached(upto)) mine = 0x80000000u | (kBins - b - 1);
    else if (v1) mine = 2u + b;
    else if (v0) mine = 1u + b;
    const uint32_t best = block_most(mine);
    return best & 0x80000000u ? kBins - (best & 0x7fffffffu) : best ? best - 1 : 0;
  }

  // Adds up the masses of at least `least` of the tokens taken, by group in s.group, and
  // lists the members: `n` of them, false where they are too many for their wave's part
  // of the list; `above`: how many are taken; `low` and `most`: this thread's smallest
  // and largest member. The taken ones are put together and weighed 64 at a time, so that
  // the others cost no exponential.
  __device__ __forceinline__ bool gather(const Cut& q, double least, uint32_t& n, uint32_t& above, float& low, float& most) {
    constexpr uint32_t kPart = kList / kWaves, kOgt = 2, kOge = 3;   // (comparisons' codes)
    __syncthreads();
    if (threadIdx.x == 0) s.found = 0;
    const int wave = uniform(static_cast<int>(threadIdx.x >> 6)), lane = threadIdx.x & 63;
    float* ring = s.ring[wave];
    uint64_t* part = s.list + wave * kPart;
    uint32_t from = 0, held = 0, taken = 0, members = 0;
    double sum = 0.;
    low = INFINITY;
    most = -INFINITY;
    // this lane's place after `base` among those of a mask
    auto place = [](uint64_t who, uint32_t base) {
      return __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(who >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(who), base));
    };
    each([&](int g, int unit, int64_t c, const float(&y)[4]) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uint64_t take = __builtin_amdgcn_fcmpf(y[k], q.hi, kOgt), list = __builtin_amdgcn_fcmpf(y[k], q.lo, kOge) & ~take;
        if (q.limited) {
          const uint64_t is = __ballot(order_of(y[k], c + k) >= q.limit);
          take &= is;
          list &= is;
        }
        if (take >> lane & 1) ring[place(take, from + held) % kRing] = y[k];
        held += static_cast<uint32_t>(__popcll(take));
        if (list) {
          if (list >> lane & 1) {
            const uint32_t at = place(list, members);
            if (at < kPart) part[at] = order_of(y[k], c + k);
            low = fminf(low, y[k]);
            most = fmaxf(most, y[k]);
          }
          members += static_cast<uint32_t>(__popcll(list));
        }
      }
      while (held >= (unit < 3 ? 64u : 1u)) {
        const uint32_t m = held < 64 ? held : 64;
        wave_sync();
        const float v = ring[(from + lane) % kRing];
        wave_sync();
        const double w = lane < static_cast<int>(m) ? weight(v) : 0.;
        if (w >= least) sum += w;
        from += m;
        held -= m;
        taken += m;
      }
      if (unit == 3) {
        sum = wave_sum(sum);
        if (lane == 0) s.group[g] = sum;
        sum = 0.;
      }
    });
    // the waves' parts one after another
    uint32_t* counts = reinterpret_cast<uint32_t*>(s.waves[turn]);
    turn ^= 1;
    if (lane == 0) {
      counts[wave] = members;
      counts[kWaves + wave] = taken;
    }
    const uint32_t mine = members < kPart ? members : kPart;
    uint64_t o[kPart / 64];
#pragma unroll
    for (uint32_t i = 0; i < kPart / 64; ++i) o[i] = i * 64 + lane < mine ? part[i * 64 + lane] : 0;
    __syncthreads();
    const uint32_t count = counts[threadIdx.x % kWaves], upto = row_scan(count, Sum{});
    n = lane_of(upto, kWaves - 1);
    above = lane_of(row_scan(counts[kWaves + threadIdx.x % kWaves], Sum{}), kWaves - 1);
    const bool fits = lane_of(row_scan(count, Most{}), kWaves - 1) <= kPart;
    const uint32_t to = wave ? lane_of(upto, wave - 1) : 0;
    if (fits) {
#pragma unroll
      for (uint32_t i = 0; i < kPart / 64; ++i)
        if (i * 64 + lane < mine) s.list[to + i * 64 + lane] = o[i];
    }
    if (threadIdx.x == 0) s.found = above;
    __syncthreads();
    return fits;
  }

  // The `want`-th in the order of the vocabulary of the tokens with this key.
  __device__ __forceinline__ uint64_t tied(uint32_t key, int64_t want, uint64_t limit) {
    uint64_t seen = 0, o = 0;
    for (int64_t c0 = 0; c0 < a.v && static_cast<int64_t>(seen) < want; c0 += kThreads) {
      const int64_t c = c0 + threadIdx.x;
      const float y = c < a.v ? value(static_cast<float>(x[c])) : -INFINITY;
      const bool is = c < a.v && key_of(y) == key && order_of(y, c) >= limit;
      uint64_t here;
      const uint64_t at = seen + block_scan<uint64_t>(is ? 1 : 0, here);
      if (is && static_cast<int64_t>(at) == want) o = order_of(y, c);
      seen += here;
    }
    return block_most(o);
  }

  // The token after the one at o, in descending order (o where none is over -infinity
  // and at or over `limit`).
  __device__ __forceinline__ uint64_t after(uint64_t o, uint64_t limit) {
    uint64_t best = 0;
    for (int64_t c = threadIdx.x; c < a.v; c += kThreads) {
      const uint64_t at = order_of(value(static_cast<float>(x[c])), c);
      if (at < o && at > best) best = at;
    }
    best = block_most(best);
    return best >> 32 > kNone && best >= limit ? best : o;
  }

  // ---- a row
  // Whether the row has an answer that needs no masses, and what its masses refer to.
  __device__ __forceinline__ bool begin() {
    const uint32_t first = static_cast<int64_t>(threadIdx.x) < a.n1024 ? a.firsts[row * a.n1024 + threadIdx.x] : 0u;
    if (r.k || r.p < 1.f || r.m > 0.f) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int64_t i = threadIdx.x + k * int64_t{kThreads};
        tops[k] = i < a.n64 ? a.tops[row * a.n64 + i] : 0u;
      }
    }
    const uint32_t key = block_most(first);
    if (r.bad || key == kNan || key <= kNone) {
      if (threadIdx.x == 0) token = -1, log_mass = NAN;
      return true;
    }
    if (r.first) {
      largest(key);
      return true;
    }
    inf = key == kInf;
    mass_of.from(inf ? 0.f : value_of(key));
    return false;
  }
  // A key that every token of a mass of at least m reaches.
  __device__ __forceinline__ uint32_t least_key() const {
    if (!(r.m > 0.f)) return kNone + 1;
    const double y = mass_of.top + static_cast<double>(r.t) * static_cast<double>(logf(r.m));
    // (under it by more than the roundings of the logarithm, of y, of f and of a mass)
    const float f = static_cast<float>(y - 1e-6 * (fabs(y) + fabs(mass_of.top) + 100. * static_cast<double>(r.t)));
    return f > -INFINITY ? key_of(f) : kNone + 1;
  }

  // The kept ones of a list's n tokens, `above` the masses and `before` the number of
  // those that stand before them: `end` of the list, by top-k where by_k, top-p and
  // min-p. Their masses go to their groups in s.mass. all_mass: of what top-p refers to,
  // where top-k does not set it. 0: min-p's cut is above the list. passed: top-p's cut is
  // not in the list, by_k above it, else below.
  __device__ __forceinline__ uint32_t cut_list(uint32_t n, bool by_k, double above, uint32_t before, double& all_mass,
                                               bool& passed) {
    const uint32_t size = sort(n), per = size > kThreads ? 2 : 1, i0 = threadIdx.x * per;
    uint32_t end = n;
    if (by_k && static_cast<int64_t>(end) > r.k - before) end = static_cast<uint32_t>(r.k - before);
    double w[2], all;
#pragma unroll 1
    for (uint32_t i = 0; i < 2; ++i) {
      const double v = i < per && i0 + i < end ? weight(listed(s.list[i0 + i])) : 0.;
      w[0] = i ? w[0] : v;
      w[1] = v;
    }
    if (per == 1) w[1] = 0.;
    const double sum = above + block_scan(w[0] + w[1], all) - (w[0] + w[1]);
    if (by_k) all_mass = above + all;
    const double goal = static_cast<double>(r.p) * all_mass, limit = r.p < 1.f ? goal : INFINITY;
    passed = by_k && !(limit > above);
    if (passed) return end;
    const double least = static_cast<double>(r.m);
    uint32_t kept = 0;
    if (i0 < end && ((i0 == 0 && before == 0) || (sum < limit && w[0] >= least))) kept = i0 + 1;
    if (per == 2 && i0 + 1 < end && sum + w[0] < limit && w[1] >= least) kept = i0 + 2;
    end = block_most(kept);
    passed = !by_k && n && end == n && above + all < limit;
    for (int g = threadIdx.x; g < kGroup; g += kThreads) s.mass[g] = 0;
    __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i)
      if (i < per && i0 + i < end && w[i] > 0.) {
        // (a mass of next to nothing is one all the same, u may be 0: the highest bit, which
        // 2048 masses do not reach)
        const unsigned long long f = fixed_of(w[i]);
        auto* m = reinterpret_cast<unsigned long long*>(&s.mass[token_of(static_cast<uint32_t>(s.list[i0 + i])) / kGroup]);
        if (f) atomicAdd(m, f);
        else atomicOr(m, 1ull << 63);
      }
    __syncthreads();
    return end;
  }
  // What cut_list has left for thread t's group.
  __device__ __forceinline__ double listed_mass() const {
    const uint64_t m = s.mass[threadIdx.x];
    return static_cast<double>(m & ~(uint64_t{1} << 63)) / kFixed + (m >> 63 ? 1e-300 : 0.);
  }

  // A row that is not filtered, or of which a list of at most kList tokens is known to
  // hold the kept ones; else false. Lists are, in the order in which they are tried: the
  // tokens over what min-p keeps (all of few), those over what about 64 or k of the 64s'
  // largest reach. (64: one wave settles them, 5 us where a sort of 1024 takes 8; with 256 top-p
  // took 14 us in place of 4.6 on a row whose list did not suffice, and 17 in place of 13 on
  // one whose did. Where top-p's share is over what so many can have, by a quarter, no
  // list is made: 4.5 us in place of 9.)
  __device__ __forceinline__ bool pick() {
    if (begin()) return true;
    double mine = 0., all_mass = 1.;
    uint64_t cut = 0;
    if (whole(r)) mine = group_mass();
    if (!whole(r) || r.p < 1.f) {
      if (inf) return false;
      if (whole(r)) block_scan(mine, all_mass);
      enum Source { kFloor, kSome, kNear, kExact };
      const uint32_t floor = r.k ? kNone + 1 : least_key();
      int source = a.v <= kList ? kFloor : r.k ? kNear : r.m > 0.f ? kFloor : kSome;
      if (r.k > a.n64 && source == kNear) return false;
      while (true) {
        uint32_t from = floor;
        bool complete = true;
        if (source != kFloor) {
          const int64_t c = source == kSome ? 64 : r.k;
          // (No mass is over 1.)
          if (source == kSome && (static_cast<double>(r.p) * all_mass > 1.25 * static_cast<double>(c) || c > a.n64)) return false;
          const uint32_t least = source == kExact ? kth_top(c) : near_top(c);
          complete = r.k || least <= floor;
          if (least > from) from = least;
        }
        const uint32_t n = candidates(from);
        if (n <= 64) {
          if (from_few(n, complete, all_mass)) return true;
          return false;
        }
        if (n <= kList) {
          bool passed;
          const uint32_t end = cut_list(n, r.k != 0, 0., 0, all_mass, passed);
          if (!complete && end == n) return false;   // it may go on below the list
          cut = uniform(s.list[end - 1]);
          mine = listed_mass();
          break;
        }
        if (source == kNear) source = kExact;   // (far from evenly spread)
        else if (source == kFloor && r.p < 1.f) source = kSome;
        else return false;
      }
    }
    by_groups(mine, cut, 0.);
    return true;
  }

  // The other rows: bins of which one is listed. A pass counts or weighs the tokens in
  // bins of equal width below the largest (24 units of e^x hold all masses that count; by
  // ranks, what the 64s' largest span), the next lists the bin that the cut is in and
  // adds up what lies above it. The first weighing is in 32 bits and takes all bins that
  // the cut may be in by what its sums can be off: a mass by 1e-5 of itself (24 units of
  // the exponent, four roundings each) and by 2^-31 of all (a whole number of them is
  // added). A list that is too long has its keys cut into bins again.
  __device__ __forceinline__ void select() {
    if (begin()) return;
    double all_mass = 1.;
    if (whole(r)) block_scan(group_mass(), all_mass);
    const uint64_t floor = static_cast<uint64_t>(least_key()) << 32;
    Cut q{};
    q.high = top();
    double off = 0., mine, cut_least = 0.;
    uint64_t cut = 0;
    enum Source { kCount, kMass, kDirect };   // direct: the cut is known
    int source = r.k ? kCount : r.p < 1.f ? kMass : kDirect;
    while (true) {
      const double goal = static_cast<double>(r.p) * all_mass;
      if (source == kDirect) {   // with the cut in q.limit, or min-p's
        if (!q.limited || q.limit < floor) q.limit = floor;
        q.limited = true;
        q.lo = INFINITY;
        q.hi = -INFINITY;
      } else {
        if (q.level == 0) {
          q.by_count = source == kCount;
          const float span = q.by_count && !inf ? (q.high - least_top()) * 1.25f : 24.f * r.t;
          q.width = fminf(static_cast<float>(kBins) / span, 1e30f);
          q.slope = -1.44269504f * fminf(static_cast<float>(mass_of.inv), 1e30f);
          q.unit = static_cast<float>(2147483648. / all_mass);
          off = mass_of.inv > 1e30 ? INFINITY : (1e-5 + static_cast<double>(a.v) / 2147483648.) * all_mass;
          q.lo = -3.4028234664e38f;
          q.hi = q.high;
        }
        fill_bins(q);
        const int b = 2 * static_cast<int>(threadIdx.x);
        const uint64_t v0 = q.level ? s.mass[b] : s.count[b], v1 = q.level ? s.mass[b + 1] : s.count[b + 1];
        uint64_t all;
        const uint64_t upto = block_scan<uint64_t>(v0 + v1, all);
        const double base = uniform(s.value);   // the masses above the bins, from level 1 on
        const int64_t k = r.k - (q.level ? static_cast<int64_t>(uniform(s.found)) : 0);
        const double unit = q.level ? 1. / kFixed : all_mass / 2147483648.;
        const double low = q.level ? goal - base : goal - off, high = q.level ? low : goal + off;
        const bool count = q.by_count;
        const uint32_t b0 = bin_where(v0, v1, upto, [&](uint64_t m) { return count ? static_cast<int64_t>(m) >= k : static_cast<double>(m) * unit >= low; });
        uint32_t b1 = b0;
        if (!count && q.level == 0) {
          b1 = bin_where(v0, v1, upto, [&](uint64_t m) { return static_cast<double>(m) * unit >= high; });
          if (static_cast<double>(all) * unit < high) b1 = kBins - 1;
        }
        if (q.level == 0) {
          q.hi = b0 ? value_of(last_of(q, b0)) : q.high;
          const uint32_t under = b1 < kBins - 1 ? last_of(q, b1 + 1) : 0;
          q.lo = under ? value_of(under + 1) : -3.4028234664e38f;
        } else {
          const uint32_t h = q.most - (b0 << q.shift), l = h - ((uint32_t{1} << q.shift) - 1), least = key_of(q.lo);
          q.hi = value_of(h);
          q.lo = l <= h && l > least ? value_of(l) : q.lo;
        }
      }
      uint32_t n, before;
      float low, most;
      const bool fits = gather(q, source == kDirect ? static_cast<double>(r.m) : 0., n, before, low, most);
      if (source == kDirect) {
        mine = static_cast<int64_t>(threadIdx.x) < a.n1024 ? s.group[threadIdx.x] : 0.;
        cut = q.limit;
        cut_least = static_cast<double>(r.m);
        break;
      }
      const double above = sum_of_groups();
      if (source == kMass && above >= goal) {
        // Sums in fixed point, off by up to 2^-44 a token, found the cut a bin too late:
        // kept is what lies above the members. (A bin too early: `after`.)
        const uint64_t over = (static_cast<uint64_t>(key_of(q.hi)) + 1) << 32;
        if (!q.limited || q.limit < over) q.limit = over;
        q.limited = true;
        source = kDirect;
        continue;
      }
      if (!fits) {
        q.most = block_most(key_of(most));
        const uint32_t span = q.most - ~block_most(~key_of(low));
        q.hi = value_of(q.most);
        q.lo = value_of(q.most - span);
        ++q.level;
        q.shift = 0;
        while (span >> q.shift >= kBins) ++q.shift;
        if (threadIdx.x == 0) s.value = above;
        __syncthreads();
        if (span) continue;
        // more equal values than the list holds
        const double w = weight(q.hi);
        double want = static_cast<double>(n);
        if (source == kCount) {
          want = fmin(want, static_cast<double>(r.k - before));   // (fewer than k may be over -infinity)
          all_mass = above + want * w;
        }
        const double limit = r.p < 1.f ? static_cast<double>(r.p) * all_mass : INFINITY;
        if (limit > above) want = fmin(want, ceil((limit - above) / w));
        const uint64_t old = q.limited ? q.limit : 0;
        q.limit = tied(q.most, static_cast<int64_t>(fmax(want, 1.)), old);
        if (source == kMass && limit > above + static_cast<double>(n) * w) q.limit = after(q.limit, old);   // (a bin too early)
        q.limited = true;
        q.level = 0;
        source = limit > above ? kDirect : kMass;   // (or top-p's cut is among the ones above)
        continue;
      }
      bool passed;
      const uint32_t end = cut_list(n, source == kCount, above, before, all_mass, passed);
      if (end) cut = uniform(s.list[end - 1]);
      if (source == kCount ? passed : q.level && passed) {
        // above a list of top-k's; or a bin too early, when one more token is kept
        q.limit = source == kCount ? cut : after(cut, q.limited ? q.limit : 0);
        q.limited = true;
        source = source == kCount ? kMass : kDirect;
        q.level = 0;
        continue;
      }
      if (end == 0) {
        source = kDirect;
        continue;
      }
      mine = listed_mass() + (static_cast<int64_t>(threadIdx.x) < a.n1024 ? s.group[threadIdx.x] : 0.);
      break;
    }
    by_groups(mine, cut, cut_least);
  }
};

template <typename E>
__global__ __launch_bounds__(kThreads) void sample_row_kernel(SampleArgs a) {
  __shared__ Shared s;
  const int64_t row = blockIdx.x;
  load_powers(s.powers);   // (barriers follow before they are read)
  const Row r = row_of(a, row);
  Pick<E> p{a, s, row, r, static_cast<const E*>(a.x) + row * a.ldx, Exp(s.powers, r.t), false, {0, 0}};
  if (!p.pick()) {
    __syncthreads();
    p.select();
  }
  p.finish();
}

// Of the first pass: groups of a wave, one after another, where there are enough of them
// for two waves a SIMD all the same (512 x 131072 bf16, the whole call: one 66 us, two 65.7,
// four 63.1, eight and sixteen 62.5, before the maxima took fewer instructions).
constexpr int64_t kMostEach = 8;
template <typename E>
hipError_t sample(const SampleArgs& a, hipStream_t stream) {
  constexpr int64_t kRows = 65535;   // of a launch's second dimension
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
    p.tails = static_cast<E*>(a.tails) + r * kGroup;
    const int64_t quads = (a.n1024 + 3) / 4, many = n * quads / 2048, each = many < 1 ? 1 : many > kMostEach ? kMostEach : many;
    hipLaunchKernelGGL(sample_groups_kernel<E>, dim3(static_cast<unsigned>((quads + each - 1) / each), static_cast<unsigned>(n)),
                       dim3(256), 0, stream, p, static_cast<int>(each));
    hipLaunchKernelGGL(sample_row_kernel<E>, dim3(static_cast<unsigned>(n)), dim3(kThreads), 0, stream, p);
  }
  return hipGetLastError();
}

}  // namespace

int64_t sample_scratch(DType t, int64_t n, int64_t v, int64_t* tops, int64_t* firsts, int64_t* tails) {
  auto up = [](int64_t b) { return (b + 255) / 256 * 256; };
  const int64_t n64 = (v + 63) / 64, n1024 = (v + kGroup - 1) / kGroup;
  *tops = up(n * n1024 * 8);
  *firsts = *tops + up(n * n64 * 4);
  *tails = *firsts + up(n * n1024 * 4);
  return *tails + (v % kGroup ? up(n * kGroup * dtype_size(t)) : 0);
}

hipError_t launch_sample(const SampleArgs& a, DType t, hipStream_t stream) {
  return t == DType::BF16 ? sample<__bf16>(a, stream) : sample<float>(a, stream);
}

}  // namespace orda
