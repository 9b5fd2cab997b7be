// embedding.hip — rows of the vocabulary weight by token id, and the gradient of
// that weight by sorted tokens.
//
// Both are bound by HBM: the lookup reads and writes a row a token, the gradient
// reads a row a token and writes every row of the weight, those a token names
// twice. 65536 tokens x 4096 of bf16 and 131072 rows: the lookup 145 us (7.4 TB/s),
// the gradient 380 us, 177 of them the sort's, in which 1.07 GB are zeroed.
//
// The gradient sorts (id, place) pairs by id, stable, so that a token's rows are
// added in the order they stand in the batch whatever the launch; the sums are
// fp32 and rounded once. Work is cut over the sorted pairs, not over the ids: a
// wave takes a chunk of pairs and 1 KB of columns, so that an id that makes up a
// tenth of the batch costs no more than any other tenth. A sum that a chunk's
// border cuts goes to scratch and is joined by a second kernel, in order.
#include <math.h>

#include "orda_kernels.h"

namespace orda {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Columns of a wave's lane, 16 bytes of E. The vectors need no alignment but their
// elements' (rows of any pitch move as wide).
template <typename E>
struct Cols {
  static constexpr int kV = 16 / sizeof(E);
};

// ------------------------------------------------------------ lookup
// A wave moves up to kLookBytes of one row, so that a lane has four 16-byte
// loads in flight.
constexpr int kLookBytes = 4096;

template <typename E, typename I>
__global__ __launch_bounds__(256) void embedding_kernel(const I* ids, int64_t n, const E* w, int64_t ldw, int64_t v,
                                                        int64_t h, float scale, E* out, int64_t ldo, int64_t parts) {
  constexpr int kV = 16 / sizeof(E), kLoads = kLookBytes / 1024;
  constexpr int kCols = kLookBytes / sizeof(E);
  const int lane = threadIdx.x & 63;
  const int64_t unit = blockIdx.x * int64_t{4} + (threadIdx.x >> 6);
  const int64_t t = unit / parts;
  if (t >= n) return;
  const int64_t c0 = (unit - t * parts) * kCols;
  const int64_t id = static_cast<int64_t>(ids[t]);
  const bool ok = id >= 0 && id < v;
  const E* s = w + (ok ? id : 0) * ldw + c0;
  E* d = out + t * ldo + c0;
  const int cols = static_cast<int>(h - c0 < kCols ? h - c0 : kCols);
  E x[kLoads][kV];
  if (ok) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int c = (i * 64 + lane) * kV;
      if (c + kV <= cols) __builtin_memcpy(x[i], s + c, sizeof(x[i]));
    }
  }
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int c = (i * 64 + lane) * kV;
    if (c + kV <= cols) {
#pragma unroll
      for (int k = 0; k < kV; ++k)
        x[i][k] = ok ? static_cast<E>(static_cast<float>(x[i][k]) * scale) : static_cast<E>(NAN);
      __builtin_memcpy(d + c, x[i], sizeof(x[i]));
    } else {
      for (int k = 0; k < kV && c + k < cols; ++k)
        d[c + k] = ok ? static_cast<E>(static_cast<float>(s[c + k]) * scale) : static_cast<E>(NAN);
    }
  }
}

// ------------------------------------------------------------ sort
constexpr int kFillBytes = 16384;   // of a wave: 1 GB in 163 us, of 4096 bytes in 180

// Ids that take no gradient (padding, or no row of the weight) sort as v, last.
template <typename I>
__device__ __forceinline__ uint32_t key_of(I id, int64_t v, int64_t pad) {
  const int64_t i = static_cast<int64_t>(id);
  return static_cast<uint32_t>(i >= 0 && i < v && i != pad ? i : v);
}

// A launch's share of the zeroes: its workgroups from `first` on, of 16 waves, each
// a span of kFillBytes at a time. The gradient is zeroed whole while the tokens are
// sorted, which leaves most of the chip idle, and the sums then write the rows that
// a token names: zeroing just the others takes a search of the sorted keys and
// writes in rows. (Stores past the caches, here and in the sums, gain nothing over 16
// batches and sizes from 0.3 to 1.6 GB of gradient: from 2 % faster to 3 % slower.)
__device__ __forceinline__ void fill_zero(const EmbedFill& f, int first) {
  const int lane = threadIdx.x & 63;
  const int64_t waves = (static_cast<int64_t>(gridDim.x) - first) * 16;
  for (int64_t u = f.from + (static_cast<int64_t>(blockIdx.x) - first) * 16 + (threadIdx.x >> 6); u < f.to; u += waves) {
    const int64_t row = u / f.spans;
    // spans begin at whole lines, the first one before the row
    const uintptr_t begin = reinterpret_cast<uintptr_t>(f.out) + row * f.pitch, end = begin + f.bytes;
    const uintptr_t at = begin / 128 * 128 + (u - row * f.spans) * kFillBytes;
#pragma unroll
    for (int i = 0; i < kFillBytes / 1024; ++i) {
      const uintptr_t d = at + i * 1024 + lane * 16;
      const u32x4 zero = {0, 0, 0, 0};
      if (d >= begin && d + 16 <= end) __builtin_memcpy(reinterpret_cast<void*>(d), &zero, 16);
      else
        for (uintptr_t e = d; e < d + 16; e += 2)   // elements of 2 or 4 bytes
          if (e >= begin && e < end) *reinterpret_cast<uint16_t*>(e) = 0;
    }
  }
}

// Few tokens: a token's place is the number of pairs before it, counted against
// all of them from LDS, with (key, place) packed into 32 bits: 64 tokens a
// workgroup, each wave against a sixteenth of the pairs. One launch, where the
// passes below take two a digit.
template <typename I>
__global__ __launch_bounds__(1024) void embed_rank_kernel(const I* ids, int n, int64_t v, int64_t pad, uint32_t* keys,
                                                          uint32_t* vals, EmbedFill fill) {
  extern __shared__ __attribute__((aligned(16))) uint32_t all[];   // n, up to whole 64s, then the waves' counts
  const int blocks = (n + 63) / 64;
  if (static_cast<int>(blockIdx.x) >= blocks) return fill_zero(fill, blocks);
  const int np = blocks * 64, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t* part = all + np;
#pragma unroll 4
  for (int i = threadIdx.x; i < np; i += 1024)
    all[i] = i < n ? key_of(ids[i], v, pad) * static_cast<uint32_t>(n) + i : 0xffffffffu;
  __syncthreads();
  const int i = blockIdx.x * 64 + lane;
  const uint32_t me = all[i];
  uint32_t before = 0;
#pragma unroll 4
  for (int j = wave * (np / 16); j < (wave + 1) * (np / 16); j += 4) {
    const u32x4 o = *reinterpret_cast<const u32x4*>(all + j);
#pragma unroll
    for (int k = 0; k < 4; ++k) before += o[k] < me ? 1u : 0u;
  }
  part[wave * 64 + lane] = before;
  __syncthreads();
  if (wave != 0 || i >= n) return;
  before = 0;
#pragma unroll
  for (int w = 0; w < 16; ++w) before += part[w * 64 + lane];
  keys[before] = me / static_cast<uint32_t>(n);
  vals[before] = static_cast<uint32_t>(i);
}

// More: stable passes over digits of kDigitBits, from the lowest. A workgroup
// holds kSortTile pairs, a wave 64·kSortSteps consecutive ones; lanes of one digit
// find each other by a ballot for each of its bits, and a wave's counters in LDS
// carry the ranks from step to step.
constexpr int kDigitBits = 9, kDigits = 1 << kDigitBits;
constexpr int kSortWaves = 16, kSortSteps = 4, kSortTile = kSortWaves * 64 * kSortSteps;

// Pairs of a pass: from the ids (first pass), or the last pass's.
template <typename I>
struct Pairs {
  const I* ids;
  const uint32_t *keys, *vals;
  int64_t n, v, pad;
  __device__ __forceinline__ uint32_t key(int64_t i) const { return ids != nullptr ? key_of(ids[i], v, pad) : keys[i]; }
  __device__ __forceinline__ uint32_t val(int64_t i) const { return ids != nullptr ? static_cast<uint32_t>(i) : vals[i]; }
};

template <typename I>
__global__ __launch_bounds__(1024) void embed_count_kernel(Pairs<I> p, int shift, int blocks, uint32_t* counts,
                                                           EmbedFill fill) {
  __shared__ uint32_t c[kDigits];
  if (static_cast<int>(blockIdx.x) >= blocks) return fill_zero(fill, blocks);
  for (int d = threadIdx.x; d < kDigits; d += 1024) c[d] = 0;
  __syncthreads();
  const int64_t i0 = blockIdx.x * static_cast<int64_t>(kSortTile);
  for (int k = threadIdx.x; k < kSortTile; k += 1024)
    if (i0 + k < p.n) atomicAdd(&c[(p.key(i0 + k) >> shift) & (kDigits - 1)], 1u);   // whole numbers: any order
  __syncthreads();
  for (int d = threadIdx.x; d < kDigits; d += 1024) counts[blockIdx.x * kDigits + d] = c[d];
}

// Up to kSumBlocks workgroups, each sums the others' counts itself as it places its
// pairs, which grows with their square; beyond, a launch before it turns them into
// sums: row b of counts into the pairs of each digit before workgroup b, the row
// after the last into all. A workgroup takes 8 digits, each of its 128 threads a
// digit a run of rows, read twice (2^30 tokens: 0.5 GB). Gradients of 8 columns, us
// without the launch and with it: 2^17 tokens 172 and 171, 2^18 176 and 168, 2^20 229
// and 176, 2^24 17910 and 2195.
constexpr int64_t kSumBlocks = 32;
constexpr int kSumDigits = 8, kSumRuns = 1024 / kSumDigits;

__global__ __launch_bounds__(1024) void embed_sums_kernel(uint32_t* counts, int64_t blocks) {
  __shared__ uint32_t runs[kSumRuns][kSumDigits];
  const int d = threadIdx.x % kSumDigits, run = threadIdx.x / kSumDigits;
  uint32_t* const c = counts + blockIdx.x * kSumDigits + d;
  const int64_t per = (blocks + kSumRuns - 1) / kSumRuns;
  const int64_t from = run * per < blocks ? run * per : blocks, to = from + per < blocks ? from + per : blocks;
  uint32_t mine = 0;
#pragma unroll 8
  for (int64_t b = from; b < to; ++b) mine += c[b * kDigits];
  runs[run][d] = mine;
  __syncthreads();
  for (int k = 1; k < kSumRuns; k *= 2) {
    const uint32_t other = run >= k ? runs[run - k][d] : 0;
    __syncthreads();
    runs[run][d] += other;
    __syncthreads();
  }
  uint32_t at = runs[run][d] - mine;
  if (run == kSumRuns - 1) c[blocks * kDigits] = at + mine;
#pragma unroll 8
  for (int64_t b = from; b < to; ++b) {
    const uint32_t n = c[b * kDigits];
    c[b * kDigits] = at;
    at += n;
  }
}

template <typename I>
__global__ __launch_bounds__(1024) void embed_place_kernel(Pairs<I> p, int shift, int blocks, const uint32_t* counts,
                                                           uint32_t* keys, uint32_t* vals, EmbedFill fill) {
  if (static_cast<int>(blockIdx.x) >= blocks) return fill_zero(fill, blocks);
  __shared__ uint32_t wave_n[kSortWaves][kDigits];   // a wave's pairs of each digit, then where they begin
  __shared__ uint32_t part[2][kDigits], wave_sum[kDigits / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (int d = lane; d < kDigits; d += 64) wave_n[wave][d] = 0;
  // Pairs of digit d in earlier workgroups and in all: read (many workgroups, see
  // embed_sums_kernel), or each half of the workgroup sums half of the counts.
  const int d = tid & (kDigits - 1), half = tid >> kDigitBits;
  static_assert(2 * kDigits == 1024, "two threads a digit");
  uint32_t earlier = 0, total = 0;
  if (blocks > kSumBlocks) {
    if (half == 0) {
      earlier = counts[static_cast<int64_t>(blockIdx.x) * kDigits + d];
      total = counts[static_cast<int64_t>(blocks) * kDigits + d];
    }
  } else {
    for (int b = half; b < blocks; b += 2) {
      const uint32_t c = counts[static_cast<int64_t>(b) * kDigits + d];
      total += c;
      if (b < static_cast<int>(blockIdx.x)) earlier += c;
    }
  }
  __syncthreads();
  if (half == 1) {
    part[0][d] = earlier;
    part[1][d] = total;
  }
  // Ranks within the wave, step by step.
  const int64_t i0 = blockIdx.x * static_cast<int64_t>(kSortTile) + wave * (64 * kSortSteps) + lane;
  uint32_t key[kSortSteps], val[kSortSteps], rank[kSortSteps];
#pragma unroll
  for (int s = 0; s < kSortSteps; ++s) {
    const bool in = i0 + s * 64 < p.n;
    key[s] = in ? p.key(i0 + s * 64) : 0;
    val[s] = in ? p.val(i0 + s * 64) : 0;
  }
#pragma unroll
  for (int s = 0; s < kSortSteps; ++s) {
    const bool in = i0 + s * 64 < p.n;
    const uint32_t dig = (key[s] >> shift) & (kDigits - 1);
    uint64_t same = __ballot(in);
#pragma unroll
    for (int b = 0; b < kDigitBits; ++b) {
      const bool bit = ((dig >> b) & 1) != 0;
      const uint64_t m = __ballot(bit);
      same &= bit ? m : ~m;
    }
    const int below = __popcll(same & ((uint64_t{1} << lane) - 1));
    const uint32_t had = in ? wave_n[wave][dig] : 0;
    rank[s] = had + below;
    __builtin_amdgcn_wave_barrier();   // every lane has read before the first of each digit writes
    if (in && below == 0) wave_n[wave][dig] = had + static_cast<uint32_t>(__popcll(same));
    __builtin_amdgcn_wave_barrier();
  }
  __syncthreads();
  // Where each digit begins: all smaller digits, then earlier workgroups, then
  // earlier waves.
  if (half == 0) {
    earlier += part[0][d];
    total += part[1][d];
    uint32_t incl = total;
#pragma unroll
    for (int k = 1; k < 64; k *= 2) {
      const uint32_t t = __shfl_up(incl, k);
      if (lane >= k) incl += t;
    }
    if (lane == 63) wave_sum[wave] = incl;
    part[1][d] = incl - total;
  }
  __syncthreads();
  if (half == 0) {
    uint32_t at = part[1][d] + earlier;
    for (int w = 0; w < wave; ++w) at += wave_sum[w];
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) {
      const uint32_t c = wave_n[w][d];
      wave_n[w][d] = at;
      at += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int s = 0; s < kSortSteps; ++s) {
    if (i0 + s * 64 >= p.n) continue;
    const uint32_t at = wave_n[wave][(key[s] >> shift) & (kDigits - 1)] + rank[s];
    keys[at] = key[s];
    vals[at] = val[s];
  }
}

// ------------------------------------------------------------ gradient
// First sorted place whose key is at least k: the wave's lanes probe 64 places
// a step.
__device__ __forceinline__ int64_t first_at_least(const uint32_t* keys, int64_t n, uint32_t k, int lane) {
  int64_t lo = 0, hi = n;   // keys[lo - 1] < k <= keys[hi]
  while (lo < hi) {
    const int64_t step = (hi - lo + 63) / 64, at = lo + lane * step;
    const bool less = at < hi && keys[at] < k;
    const int c = __popcll(__ballot(less));   // the first c probes are less
    if (c == 0) return lo;
    const int64_t last = lo + (c - 1) * step;
    hi = last + step < hi ? last + step : hi;
    lo = last + 1;
  }
  return lo;
}

// One lane's columns of a gradient row from column c on, scaled and rounded (added
// to what is there with accumulate).
template <typename E, typename O>
__device__ __forceinline__ void put_row(const EmbedGradArgs& a, int64_t row, int64_t c, const float (&x)[Cols<E>::kV]) {
  constexpr int kV = Cols<E>::kV;
  O* d = static_cast<O*>(a.out) + row * a.ldo + c;
  const int left = static_cast<int>(a.h - c);
  if (left >= kV) {
    O o[kV];
    if (a.accumulate) __builtin_memcpy(o, d, sizeof(o));
#pragma unroll
    for (int k = 0; k < kV; ++k) {
      const float s = x[k] * a.scale;
      o[k] = static_cast<O>(a.accumulate ? static_cast<float>(o[k]) + s : s);
    }
    if constexpr (sizeof(o) % 16 == 0) {   // vector by vector: copied whole, 2 % slower
#pragma unroll
      for (int k = 0; k < static_cast<int>(sizeof(o)) / 16; ++k) {
        u32x4 w;
        __builtin_memcpy(&w, o + k * (16 / sizeof(O)), 16);
        __builtin_memcpy(d + k * (16 / sizeof(O)), &w, 16);
      }
    } else {
      __builtin_memcpy(d, o, sizeof(o));
    }
  } else {
#pragma unroll
    for (int k = 0; k < kV; ++k)
      if (k < left) {
        const float s = x[k] * a.scale;
        d[k] = static_cast<O>(a.accumulate ? static_cast<float>(d[k]) + s : s);
      }
  }
}

// Partial sums of a chunk: its first sum where an earlier chunk began it (slot
// 0), its last where it goes on (slot 1; slot 0 where it is the first too). Their
// rows hold whole waves' columns.
__device__ __forceinline__ float* partial(const EmbedGradArgs& a, int64_t chunk, int slot, int64_t c) {
  return a.parts + (chunk * 2 + slot) * a.ldp + c;
}
template <int kV>
__device__ __forceinline__ void put_partial(float* d, const float (&x)[kV]) {
#pragma unroll
  for (int k = 0; k < kV; k += 4) *reinterpret_cast<f32x4*>(d + k) = f32x4{x[k], x[k + 1], x[k + 2], x[k + 3]};
}
template <int kV>
__device__ __forceinline__ void add_partial(const float* s, float (&x)[kV]) {
#pragma unroll
  for (int k = 0; k < kV; k += 4) {
    const f32x4 v = *reinterpret_cast<const f32x4*>(s + k);
#pragma unroll
    for (int q = 0; q < 4; ++q) x[k + q] += v[q];
  }
}

// The sums of a chunk of sorted pairs, a wave for each chunk and its columns,
// kLoads rows in flight.
template <typename E, typename O>
__global__ __launch_bounds__(256) void embed_sum_kernel(EmbedGradArgs a) {
  constexpr int kV = Cols<E>::kV, kLoads = 8;
  const int lane = threadIdx.x & 63;
  const int64_t unit = blockIdx.x * int64_t{4} + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (unit >= a.chunks * a.slabs) return;
  const int64_t chunk = unit / a.slabs, c = (unit - chunk * a.slabs) * (64 * kV) + lane * kV;
  const int64_t b = chunk * a.chunk, e = b + a.chunk < a.n ? b + a.chunk : a.n;
  const int left = static_cast<int>(a.h - c);
  const E* src = static_cast<const E*>(a.grad) + c;
  float x[kV] = {};
  uint32_t key = a.keys[b];
  bool head = b > 0 && a.keys[b - 1] == key;   // the sum began in an earlier chunk
  auto flush = [&](bool tail) {   // tail: it goes on in the next one
    if (static_cast<int64_t>(key) < a.v) {
      if (head || tail) put_partial(partial(a, chunk, head ? 0 : 1, c), x);
      else if (left > 0) put_row<E, O>(a, key, c, x);
    }
#pragma unroll
    for (int k = 0; k < kV; ++k) x[k] = 0.f;
    head = false;
  };
  for (int64_t i = b; i < e; i += kLoads) {
    E w[kLoads][kV];
    uint32_t ks[kLoads];
    int64_t at[kLoads];
#pragma unroll
    for (int q = 0; q < kLoads; ++q) {
      const int64_t j = i + q < e ? i + q : e - 1;
      ks[q] = a.keys[j];
      at[q] = a.vals[j] * a.ldg;   // (a row without a gradient is read, not added)
    }
    if (left >= kV) {   // one branch for all rows: around each load it made them wait for one another
#pragma unroll
      for (int q = 0; q < kLoads; ++q) __builtin_memcpy(w[q], src + at[q], sizeof(w[q]));
    } else {
#pragma unroll
      for (int q = 0; q < kLoads; ++q)
#pragma unroll
        for (int k = 0; k < kV; ++k) w[q][k] = k < left ? src[at[q] + k] : static_cast<E>(0.f);
    }
#pragma unroll
    for (int q = 0; q < kLoads; ++q) {
      if (i + q < e) {
        if (ks[q] != key) {
          flush(false);
          key = ks[q];
        }
#pragma unroll
        for (int k = 0; k < kV; ++k) x[k] += static_cast<float>(w[q][k]);
      }
    }
  }
  flush(e < a.n && a.keys[e] == key);
}

// Sums that a chunk begins and a later one ends, a wave for each chunk and its
// columns: the parts in order.
template <typename E, typename O>
__global__ __launch_bounds__(256) void embed_join_kernel(EmbedGradArgs a) {
  constexpr int kV = Cols<E>::kV;
  const int lane = threadIdx.x & 63;
  const int64_t unit = blockIdx.x * int64_t{4} + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (unit >= (a.chunks - 1) * a.slabs) return;
  const int64_t chunk = unit / a.slabs, c = (unit - chunk * a.slabs) * (64 * kV) + lane * kV;
  const int64_t b = chunk * a.chunk, e = b + a.chunk;   // not the last chunk: whole
  const uint32_t key = a.keys[e - 1];
  if (static_cast<int64_t>(key) >= a.v || a.keys[e] != key) return;    // nothing goes on
  if (b > 0 && a.keys[b] == key && a.keys[b - 1] == key) return;       // begun earlier
  // the last chunk that begins with this key
  const int64_t end = first_at_least(a.keys, a.n, key + 1, lane);
  const int64_t last = (end - 1) / a.chunk;
  float x[kV] = {};
  add_partial(partial(a, chunk, 1, c), x);
  int64_t j = chunk + 1;
  for (; j + 7 <= last; j += 8) {   // eight loads in flight, added in order
    float y[8][kV] = {};
#pragma unroll
    for (int q = 0; q < 8; ++q) add_partial(partial(a, j + q, 0, c), y[q]);
#pragma unroll
    for (int q = 0; q < 8; ++q)
#pragma unroll
      for (int k = 0; k < kV; ++k) x[k] += y[q][k];
  }
  for (; j <= last; ++j) add_partial(partial(a, j, 0, c), x);
  if (c < a.h) put_row<E, O>(a, key, c, x);
}

int passes_of(int64_t v) {   // digits of keys 0..v
  int bits = 0;
  while (bits < 32 && (v >> bits) != 0) ++bits;
  return bits <= kDigitBits ? 1 : (bits + kDigitBits - 1) / kDigitBits;
}

// Tokens whose ranks are counted: the packed pairs must fit 32 bits and 64 KB of
// LDS, less the waves' counts. 8192 tokens' ranks take 14 us and the passes 25,
// 15000 tokens' 23 and 27, 1024 tokens' 4 and 15.
constexpr int64_t kRankTokens = 15360;
bool ranked(int64_t n, int64_t v) { return n <= kRankTokens && (v + 1) * n <= int64_t{0xffffffff}; }

}  // namespace

hipError_t launch_embedding(DType t, const void* ids, bool ids64, int64_t n, const void* w, int64_t ldw, int64_t v,
                            int64_t h, float scale, void* out, int64_t ldo, hipStream_t stream) {
  if (n <= 0 || h <= 0) return hipSuccess;
  const int64_t es = dtype_size(t);
  const int64_t parts = (h * es + kLookBytes - 1) / kLookBytes;
  const int64_t most = most_blocks(256) * 4 / parts;   // tokens of a launch
  auto run = [&](auto* e, auto* i) {
    using E = std::remove_pointer_t<decltype(e)>;
    using I = std::remove_pointer_t<decltype(i)>;
    for (int64_t t = 0; t < n; t += most) {
      const int64_t m = n - t < most ? n - t : most;
      hipLaunchKernelGGL((embedding_kernel<E, I>), dim3(static_cast<unsigned>((m * parts + 3) / 4)), dim3(256), 0, stream,
                         static_cast<const I*>(ids) + t, m, static_cast<const E*>(w), ldw, v, h, scale,
                         static_cast<E*>(out) + t * ldo, ldo, parts);
    }
  };
  int64_t* i64 = nullptr;
  int32_t* i32 = nullptr;
  __bf16* b = nullptr;
  float* f = nullptr;
  if (t == DType::BF16) ids64 ? run(b, i64) : run(b, i32);
  else ids64 ? run(f, i64) : run(f, i32);
  return hipGetLastError();
}

EmbedScratch embed_scratch(DType grad, int64_t n, int64_t v, int64_t h) {
  EmbedScratch s{};
  const int64_t cols = 64 * 16 / dtype_size(grad);   // of a wave
  s.chunk = 8;   // pairs a wave sums: enough waves of few tokens (1000 x 1531: 9 us, of 32 pairs 22), few joins of many
  while (s.chunk < 256 && n / s.chunk > 512) s.chunk *= 2;
  s.chunks = (n + s.chunk - 1) / s.chunk;
  s.slabs = (h + cols - 1) / cols;
  s.ldp = s.slabs * cols;
  auto up = [](int64_t b) { return (b + 255) / 256 * 256; };
  const int64_t pair = up(n * 4);
  s.keys[0] = 0;
  s.vals[0] = pair;
  s.bytes = 2 * pair;
  if (!ranked(n, v)) {
    s.keys[1] = s.bytes;
    s.vals[1] = s.bytes + pair;
    s.counts = s.bytes + 2 * pair;
    const int64_t blocks = (n + kSortTile - 1) / kSortTile;
    s.bytes = s.counts + up((blocks + (blocks > kSumBlocks ? 1 : 0)) * kDigits * 4);
  }
  s.parts = s.bytes;
  if (s.chunks > 1) s.bytes += up(s.chunks * 2 * s.ldp * 4);
  return s;
}

EmbedFill embed_fill(DType out, void* d, int64_t ldo, int64_t v, int64_t h) {
  const int64_t es = dtype_size(out);
  EmbedFill f{};
  f.out = d;
  const bool whole = ldo == h || v == 1;   // rows that follow each other are one
  f.rows = whole ? 1 : v;
  f.bytes = (whole ? v * h : h) * es;
  f.pitch = ldo * es;
  f.spans = f.bytes > 0 ? (f.bytes + 126 + kFillBytes - 1) / kFillBytes : 0;   // (a row begins up to 126 bytes into its line)
  return f;
}

hipError_t launch_embed_sort(const void* ids, bool ids64, int64_t n, int64_t v, int64_t pad, void* ws,
                             const EmbedScratch& s, EmbedFill fill, const uint32_t** keys, const uint32_t** vals,
                             hipStream_t stream) {
  char* base = static_cast<char*>(ws);
  auto u32 = [&](int64_t at) { return reinterpret_cast<uint32_t*>(base + at); };
  auto run = [&](auto* i) {
    using I = std::remove_pointer_t<decltype(i)>;
    const I* id = static_cast<const I*>(ids);
    const int64_t units = fill.rows * fill.spans;
    // launch l of `of` zeroes its part, a wave a span until the grid is large
    auto share = [&](int l, int of) {
      fill.from = units * l / of;
      fill.to = units * (l + 1) / of;
      const int64_t wgs = (fill.to - fill.from + 15) / 16;
      return static_cast<unsigned>(wgs < 8192 ? wgs : 8192);
    };
    if (ranked(n, v)) {
      const unsigned blocks = static_cast<unsigned>((n + 63) / 64), more = share(0, 1);
      *keys = u32(s.keys[0]);
      *vals = u32(s.vals[0]);
      if (blocks + more > 0)
        hipLaunchKernelGGL(embed_rank_kernel<I>, dim3(blocks + more), dim3(1024), blocks * 256 + 4096, stream, id,
                           static_cast<int>(n), v, pad, u32(s.keys[0]), u32(s.vals[0]), fill);
      return;
    }
    const int passes = passes_of(v);
    const unsigned blocks = static_cast<unsigned>((n + kSortTile - 1) / kSortTile);
    for (int p = 0; p < passes; ++p) {
      const int to = p & 1;
      const Pairs<I> pr{p == 0 ? id : nullptr, u32(s.keys[1 - to]), u32(s.vals[1 - to]), n, v, pad};
      unsigned more = share(2 * p, 2 * passes);
      hipLaunchKernelGGL(embed_count_kernel<I>, dim3(blocks + more), dim3(1024), 0, stream, pr, p * kDigitBits,
                         static_cast<int>(blocks), u32(s.counts), fill);
      if (blocks > kSumBlocks)
        hipLaunchKernelGGL(embed_sums_kernel, dim3(kDigits / kSumDigits), dim3(1024), 0, stream, u32(s.counts),
                           static_cast<int64_t>(blocks));
      more = share(2 * p + 1, 2 * passes);
      hipLaunchKernelGGL(embed_place_kernel<I>, dim3(blocks + more), dim3(1024), 0, stream, pr, p * kDigitBits,
                         static_cast<int>(blocks), static_cast<const uint32_t*>(u32(s.counts)), u32(s.keys[to]),
                         u32(s.vals[to]), fill);
      *keys = u32(s.keys[to]);
      *vals = u32(s.vals[to]);
    }
  };
  int64_t* i64 = nullptr;
  int32_t* i32 = nullptr;
  ids64 ? run(i64) : run(i32);
  return hipGetLastError();
}

hipError_t launch_embed_grad(const EmbedGradArgs& a, DType grad, DType out, hipStream_t stream) {
  const int64_t sum = (a.chunks * a.slabs + 3) / 4, join = ((a.chunks - 1) * a.slabs + 3) / 4;
  if (sum > most_blocks(256)) return hipErrorInvalidValue;   // 68 GB of fp32 parts: more than the gradients that fit
  auto run = [&](auto* e, auto* o) {
    using E = std::remove_pointer_t<decltype(e)>;
    using O = std::remove_pointer_t<decltype(o)>;
    if (sum > 0) hipLaunchKernelGGL((embed_sum_kernel<E, O>), dim3(static_cast<unsigned>(sum)), dim3(256), 0, stream, a);
    if (join > 0) hipLaunchKernelGGL((embed_join_kernel<E, O>), dim3(static_cast<unsigned>(join)), dim3(256), 0, stream, a);
  };
  __bf16* b = nullptr;
  float* f = nullptr;
  if (grad == DType::BF16) out == DType::BF16 ? run(b, b) : run(b, f);
  else out == DType::BF16 ? run(f, b) : run(f, f);
  return hipGetLastError();
}

}  // namespace orda
