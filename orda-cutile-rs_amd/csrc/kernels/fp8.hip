// fp8.hip — matrices in e4m3 with one fp32 scale for each block of 128 columns
// (and of 1 or 128 rows): the quantiser and the product.
#include <float.h>
#include <math.h>

#include "fp8_codes.h"
#include "lds_dma.h"
#include "orda_kernels.h"

namespace orda {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) const u32x4 lds_u32x4;
typedef __attribute__((address_space(3))) const float lds_f32;

// ------------------------------------------------------------ quantiser
// scale = max(amax / 448, 2^-126), code = x / scale rounded to nearest even, both
// quotients in fp32: |x / scale| is at most 448 but for its rounding, which the
// clamp takes back. A block with an infinity or a NaN has the scale NaN and codes
// NaN. Bound by HBM, each value being read once into registers: the quotient is a
// product with the reciprocal wherever that cannot change the code (`doubtful`),
// an IEEE division for every value took twice as long (fp8_codes.h).

// kC neighbouring values from column c on (0 past cols) of N rows by one load each,
// aligned to their size or of any alignment. One branch for all the rows: a branch
// around each load made it wait for the one before.
template <typename E, int N, int kC, bool ALIGNED>
__device__ __forceinline__ void load_rows(const E* const (&row)[N], int64_t c, int64_t cols, float (&x)[N][kC]) {
  E w[N][kC];
  if (c + kC <= cols) {
#pragma unroll
    for (int q = 0; q < N; ++q) {
      if constexpr (ALIGNED) __builtin_memcpy(w[q], __builtin_assume_aligned(row[q] + c, sizeof(w[q])), sizeof(w[q]));
      else __builtin_memcpy(w[q], row[q] + c, sizeof(w[q]));
    }
  } else {
#pragma unroll
    for (int q = 0; q < N; ++q)
#pragma unroll
      for (int k = 0; k < kC; ++k) w[q][k] = c + k < cols ? row[q][c + k] : static_cast<E>(0.f);
  }
#pragma unroll
  for (int q = 0; q < N; ++q)
#pragma unroll
    for (int k = 0; k < kC; ++k) x[q][k] = static_cast<float>(w[q][k]);
}

// Blocks of one row: 16 lanes a block of 128, a wave 4 blocks of each of 4 rows,
// a workgroup 16 rows, whose scales leave as 64 bytes a block.
template <typename E>
__global__ __launch_bounds__(256) void fp8_quant_rows_kernel(Fp8QuantArgs a) {
  __shared__ float sc[4][16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t groups = (a.cols + 511) / 512;
  const int64_t r0 = blockIdx.x / groups * 16, c0 = blockIdx.x % groups * 512;
  const int64_t c = c0 + lane * 8;
  const E* src = static_cast<const E*>(a.src);
  float x[4][8];
  const E* row[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int64_t r = r0 + wave * 4 + q;
    row[q] = src + (r < a.rows ? r : a.rows - 1) * a.lds;
  }
  load_rows<E, 4, 8, false>(row, c, a.cols, x);
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int64_t r = r0 + wave * 4 + q;
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) m = abs_bits(x[q][k]) > m ? abs_bits(x[q][k]) : m;
#pragma unroll
    for (int d = 1; d < 16; d *= 2) {
      const uint32_t o = __shfl_xor(m, d);
      m = o > m ? o : m;
    }
    const float s = scale_of(m);
    if (r < a.rows) store8(a.codes + r * a.ldc, c, a.cols, x[q], s);
    if ((lane & 15) == 0) sc[lane >> 4][wave * 4 + q] = s;
  }
  __syncthreads();
  const int b = threadIdx.x >> 4, k = threadIdx.x & 15;
  if (b < 4 && c0 + b * 128 < a.cols && r0 + k < a.rows)
    a.scales[(r0 + k) * a.scale_row + (c0 / 128 + b) * a.scale_col] = sc[b][k];
}

// Blocks of 128 rows: a workgroup holds a block in registers, 64 / kC rows of kC
// columns a thread, kC as wide as the rows' alignment allows.
template <typename E, int kC, bool ALIGNED>
__global__ __launch_bounds__(256) void fp8_quant_blocks_kernel(Fp8QuantArgs a) {
  constexpr int kLanes = 128 / kC, kRows = 64 / kC, kStep = 256 / kLanes;
  __shared__ uint32_t top[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t cb = (a.cols + 127) / 128;
  // (Neighbouring blocks on one XCD: where rows are no whole lines they share them.)
  const int64_t per = gridDim.x / 8, at = blockIdx.x < per * 8 ? blockIdx.x % 8 * per + blockIdx.x / 8 : blockIdx.x;
  const int64_t rb = at / cb, kb = at % cb;
  const int64_t c = kb * 128 + threadIdx.x % kLanes * kC, r0 = rb * 128 + threadIdx.x / kLanes;
  const E* src = static_cast<const E*>(a.src);
  float x[kRows][kC];
  const E* row[kRows];
  uint32_t m = 0;
#pragma unroll
  for (int q = 0; q < kRows; ++q) {
    const int64_t r = r0 + kStep * q;
    row[q] = src + (r < a.rows ? r : a.rows - 1) * a.lds;   // the last row again
  }
  load_rows<E, kRows, kC, ALIGNED>(row, c, a.cols, x);
#pragma unroll
  for (int q = 0; q < kRows; ++q)
#pragma unroll
    for (int k = 0; k < kC; ++k) m = abs_bits(x[q][k]) > m ? abs_bits(x[q][k]) : m;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const uint32_t o = __shfl_xor(m, d);
    m = o > m ? o : m;
  }
  if (lane == 0) top[wave] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 4; ++w) m = top[w] > m ? top[w] : m;
  const float s = scale_of(m), r1 = __builtin_amdgcn_rcpf(s);
#pragma unroll
  for (int q = 0; q < kRows; ++q) {
    const int64_t r = r0 + kStep * q;
    if (r >= a.rows || c >= a.cols) continue;
    uint8_t* d = a.codes + r * a.ldc + c;
    if constexpr (kC >= 4) {
#pragma unroll
      for (int k = 0; k < kC; k += 4) *reinterpret_cast<uint32_t*>(d + k) = codes4(x[q] + k, s, r1);
    } else {
      float y[4] = {x[q][0], kC > 1 ? x[q][kC - 1] : 0.f, 0.f, 0.f};
      const uint32_t w = codes4(y, s, r1);
      if constexpr (kC == 2) *reinterpret_cast<uint16_t*>(d) = static_cast<uint16_t>(w);
      else *d = static_cast<uint8_t>(w);
    }
  }
  if (threadIdx.x == 0) a.scales[rb * a.scale_row + kb * a.scale_col] = s;
}

// Rows of codes at a pitch of whole 16s, zeros past cols.
__global__ __launch_bounds__(256) void fp8_pack_kernel(const uint8_t* src, int64_t lds, int64_t rows, int64_t cols,
                                                       uint8_t* dst, int64_t ldd) {
  const int64_t per = ldd / 16;
  for (int64_t i = blockIdx.x * int64_t{256} + threadIdx.x; i < rows * per; i += gridDim.x * int64_t{256}) {
    const int64_t r = i / per, c = (i - r * per) * 16;
    alignas(16) uint8_t w[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) w[k] = c + k < cols ? src[r * lds + c + k] : 0;
    *reinterpret_cast<u32x4*>(dst + r * ldd + c) = *reinterpret_cast<const u32x4*>(w);
  }
}

// ------------------------------------------------------------ product
// C[m, n] = Σ_b sa[m, b] · sb[n / 128, b] · Σ_{k in block b} a[m, k] · b[n, k].
//
// One 16x16x128 MFMA is one block of K: its result is a block's plain sum, which
// is scaled into the fp32 accumulators by a fma an element. The vector units
// reach only half of a wave's 512 registers, so a wave holds 128 x 64 of C there
// (128 registers), and a workgroup of 8 waves 256 x 256; while one of a SIMD's two
// waves scales, the other multiplies. K advances one block at a time through two
// 64 KB stages in LDS, moved by DMA while the other is read: rows of 128 bytes,
// their eight 16-byte chunks swizzled by row (by the choice of the chunk a lane
// fetches). Lane group g reads chunks g and 4 + g of its row: a 16-byte read
// serves lanes 0-3, 12-15 and 20-27 together, then the others of 32, and these meet
// no bank twice; with chunks 2g and 2g + 1 every read took twice as long. (Which K
// a lane holds does not matter while both operands hold the same.) The operands
// enter the MFMA swapped: a lane then owns four consecutive columns of a row.
//
// Bound by the SIMDs' instruction and register ports: 16 cycles an MFMA, 4 a vector
// instruction and 4 a register that an LDS read returns are 47 for each MFMA, where
// the matrix unit is busy for 32 (this fits the loop without transfers, 3.6 ms at
// 8192 x 4096 x 131072, without barriers too, 3.3, and without reads, 2.3, against
// 4.1 with all). 32x32x64
// MFMAs, half the port time, leave too few registers to keep two pairs apart: 4.6.
//
// The e4m3 MFMAs (all four shapes, measured) add their products to fewer bits than
// fp32: a sum of 4 to 128 comes out 1.5e-5 of the root of the sum of squares off,
// 1e-4 at most. Beside bf16 outputs, rounded at 1.7e-3, that is nothing; for fp32
// outputs (WIDE) the codes are widened to bf16, exactly, as fragments are read, and
// a block is four 16x16x32 bf16 MFMAs (9e-9 off), at half the matrix rate.
constexpr int kTile = 256, kThreads = 512;
constexpr int kOp = kTile * 128;                      // an operand's stage
constexpr int kScales = kTile * 4 + 64;               // A's row scales, B's two
constexpr int kStage = 2 * kOp;

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  const bf16x2 v = {static_cast<__bf16>(a), static_cast<__bf16>(b)};
  return __builtin_bit_cast(uint32_t, v);
}

// Tile t of the raster: XCDs take contiguous ranges, walked in groups of 8
// M-tiles, so that the tiles of an XCD share operand strips in its L2.
__device__ __forceinline__ void tile_of(int64_t t, int64_t mt, int64_t nt, int64_t& m, int64_t& n) {
  const int64_t per = mt * nt / 8;
  if (t < per * 8) t = (t % 8) * per + t / 8;
  const int64_t group = 8 * nt, first = t / group * 8, size = mt - first < 8 ? mt - first : 8, r = t % group;
  m = first + r % size;
  n = r / size;
}

// A fragment's 32 codes of a lane as bf16, eight for each of four MFMAs.
struct Wide {
  bf16x8 k[4];
};
__device__ __forceinline__ Wide widened(const i32x8& f) {
  Wide w;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const auto lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(f[2 * q + h], 1.f, false);
      const auto hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(f[2 * q + h], 1.f, true);
      w.k[q][4 * h] = lo[0];
      w.k[q][4 * h + 1] = lo[1];
      w.k[q][4 * h + 2] = hi[0];
      w.k[q][4 * h + 3] = hi[1];
    }
  }
  return w;
}

template <typename OT, bool WIDE>
__global__ __launch_bounds__(kThreads, 2) void fp8_mm_kernel(Fp8MmArgs a) {
  __shared__ __attribute__((aligned(1024))) unsigned char smem[2 * kStage + 2 * kScales];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave >> 2, wn = wave & 3;
  int64_t mi, ni;
  tile_of(blockIdx.x, (a.m + kTile - 1) / kTile, (a.n + kTile - 1) / kTile, mi, ni);
  const int64_t m0 = mi * kTile, n0 = ni * kTile;
  // This thread's four 16-byte chunks of each operand's stage: LDS chunk p =
  // t·512 + tid is chunk p % 8 of row p / 8. Rows past the edge are the last one
  // (their outputs are not stored).
  uint32_t offA[4], offB[4];
  int kcol;   // first K of the chunk, the same for all four
  {
    const int r = tid >> 3, q = (tid & 7) ^ (r & 7);
    kcol = q * 16;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int64_t rr = r + 64 * t;
      const int64_t ra = m0 + rr < a.m ? rr : a.m - 1 - m0, rb = n0 + rr < a.n ? rr : a.n - 1 - n0;
      offA[t] = static_cast<uint32_t>(ra * a.lda + kcol);
      offB[t] = static_cast<uint32_t>(rb * a.ldb + kcol);
    }
  }
  const unsigned char* const pa = a.a + m0 * a.lda;
  const unsigned char* const pb = a.b + n0 * a.ldb;
  // Scales of a stage: waves 0-3 fetch a row's each, the others B's two blocks'.
  const float* const psa = a.sa + m0 * a.sa_row;
  const int64_t nb0 = n0 / 128, nbs = (a.n + 127) / 128;
  const float* const psb = a.sb + nb0 * a.sb_row;
  uint32_t offS = 0;
  if (wave < 4) {
    const int64_t r = m0 + tid < a.m ? tid : a.m - 1 - m0;
    offS = static_cast<uint32_t>(r * a.sa_row * 4);
  } else {
    offS = static_cast<uint32_t>(((lane & 1) != 0 && nb0 + 1 < nbs ? 1 : 0) * a.sb_row * 4);
  }
  const uint32_t lds0 = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(
      static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_void*)smem))));
  // Block kb into stage `buf`: nine transfers a wave in all (waves 4-7 all move B's
  // scales, the same values to the same place, so that every wave counts alike).
  auto issue_scales = [&](int kb, int buf) {
    const uint32_t sc = lds0 + 2 * kStage + buf * kScales;
    if (wave < 4) dma4(uniform64(psa + kb * a.sa_col), offS, sc + wave * 256);
    else if (lane < 2) dma4(uniform64(psb + kb * a.sb_col), offS, sc + 1024);
  };
  auto issue_a = [&](int kb, int buf) {   // and the scales: five transfers a wave
    const uint32_t st = lds0 + buf * kStage + wave * 1024;
    const uint64_t u = uniform64(pa + kb * int64_t{128});
    dma16_at<0>(u, offA[0], st);
    dma16_at<8192>(u, offA[1], st);
    dma16_at<16384>(u, offA[2], st);
    dma16_at<24576>(u, offA[3], st);
    issue_scales(kb, buf);
  };
  auto issue_b = [&](int kb, int buf) {   // four
    const uint32_t st = lds0 + buf * kStage + kOp + wave * 1024;
    const uint64_t u = uniform64(pb + kb * int64_t{128});
    dma16_at<0>(u, offB[0], st);
    dma16_at<8192>(u, offB[1], st);
    dma16_at<16384>(u, offB[2], st);
    dma16_at<24576>(u, offB[3], st);
  };
  f32x4 acc[8][4];
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int lrow = lane & 15, lgrp = lane >> 4;
  // Fragment of 16 rows: lane (row lrow, group lgrp) holds chunks lgrp and
  // 4 + lgrp. Addresses of fragment 0 in stage 0, which lies 64 KB below stage 1.
  const uint32_t f0 = lds0 + static_cast<uint32_t>(lrow * 128 + ((lgrp ^ (lrow & 7)) << 4));
  const uint32_t f1 = lds0 + static_cast<uint32_t>(lrow * 128 + (((4 + lgrp) ^ (lrow & 7)) << 4));
  uint32_t a0 = f0 + wm * 16384, a1 = f1 + wm * 16384;
  uint32_t b0 = f0 + kOp + wn * 8192, b1 = f1 + kOp + wn * 8192;
  uint32_t sa_at = lds0 + 2 * kStage + (wm * 128 + lrow) * 4, sb_at = lds0 + 2 * kStage + 1024 + (wn >> 1) * 4;
  auto frag = [&](uint32_t lo_at, uint32_t hi_at, int f) {
    const u32x4 lo = *(const lds_u32x4*)(static_cast<uintptr_t>(lo_at + f * 2048));
    const u32x4 hi = *(const lds_u32x4*)(static_cast<uintptr_t>(hi_at + f * 2048));
    return __builtin_bit_cast(i32x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  };
  auto scale = [&](uint32_t at, int f) { return *(const lds_f32*)(static_cast<uintptr_t>(at + f * 64)); };
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  // One block from stage `buf`, which has landed for all waves.
  auto block = [&](int buf) {
    const uint32_t at = buf * kStage, sc = buf * kScales;
    using F = std::conditional_t<WIDE, Wide, i32x8>;
    auto operand = [&](uint32_t lo_at, uint32_t hi_at, int f) -> F {
      if constexpr (WIDE) return widened(frag(lo_at, hi_at, f));
      else return frag(lo_at, hi_at, f);
    };
    F b[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) b[j] = operand(b0 + at, b1 + at, j);
    const float s_b = scale(sb_at + sc, 0);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const F x = operand(a0 + at, a1 + at, i);
      const float s = s_b * scale(sa_at + sc, i);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        f32x4 p = zero;
        if constexpr (WIDE) {
#pragma unroll
          for (int q = 0; q < 4; ++q) p = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b[j].k[q], x.k[q], p, 0, 0, 0);
        } else {
          p = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b[j], x, p, 0, 0, 0, 0, 0, 0);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][j][e] = fmaf(s, p[e], acc[i][j][e]);
      }
    }
  };
  const int nfull = static_cast<int>(a.k / 128);
  if constexpr (WIDE) {
    if (nfull > 0) issue_b(0, 0), issue_a(0, 0);
    for (int kb = 0; kb < nfull; ++kb) {
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_waitcnt(kWaitAll);
      __builtin_amdgcn_s_barrier();
      __builtin_amdgcn_sched_barrier(0);
      if (kb + 1 < nfull) issue_b(kb + 1, (kb + 1) & 1), issue_a(kb + 1, (kb + 1) & 1);
      __builtin_amdgcn_sched_barrier(0);
      block(kb & 1);
    }
  } else if (nfull > 0) {
    // Row i of the wave's fragments is four MFMAs; beside them run the fmas of
    // row i - 1 and the reads of row i + 2. By row 1 every wave holds its fragments
    // of B: a barrier, and B of block kb + 2 moves into their place. By row 6 it has
    // read all of A, and its own transfers of the next block have landed (all but
    // the four of B just begun): a barrier, A and the scales of block kb + 2 move in,
    // and the next block's first fragments are read under rows 6 and 7. So A has
    // one iteration to land, B one and five eighths. (Both from row 6 on: the
    // matrix units 48 % busy, waiting for the transfers.)
    i32x8 b[4], x[4];
    f32x4 p[2][4];
    float row_scale[4], s[2] = {0.f, 0.f};
    issue_b(0, 0);
    issue_a(0, 0);
    if (nfull > 1) {
      issue_b(1, 1);
      issue_a(1, 1);
      __builtin_amdgcn_s_waitcnt(vm_wait(9));
    } else {
      __builtin_amdgcn_s_waitcnt(kWaitAll);
    }
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    x[0] = frag(a0, a1, 0);
    x[1] = frag(a0, a1, 1);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      b[j] = frag(b0, b1, j);
      p[1][j] = zero;   // row -1: nothing
    }
    float s_b = scale(sb_at, 0);
    row_scale[0] = scale(sa_at, 0);
    row_scale[1] = scale(sa_at, 1);
    // (The last block's iteration reads ahead too, what is in the other stage.)
    for (int kb = 0; kb < nfull; ++kb) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        __builtin_amdgcn_sched_barrier(0);
        if (i == 1) {
          __builtin_amdgcn_s_waitcnt(kWaitLds);
          __builtin_amdgcn_s_barrier();
          __builtin_amdgcn_sched_barrier(0);
          if (kb + 2 < nfull) issue_b(kb + 2, kb & 1);
          __builtin_amdgcn_sched_barrier(0);
        }
        if (i == 6) {
          if (kb + 2 < nfull) __builtin_amdgcn_s_waitcnt(vm_wait(4));
          else __builtin_amdgcn_s_waitcnt(kWaitAll);
          __builtin_amdgcn_s_barrier();
          __builtin_amdgcn_sched_barrier(0);
          if (kb + 2 < nfull) issue_a(kb + 2, kb & 1);
          const uint32_t flip = (kb & 1) != 0 ? 0u - kStage : kStage;   // to the other stage
          const uint32_t flip_s = (kb & 1) != 0 ? 0u - kScales : kScales;
          a0 += flip;
          a1 += flip;
          b0 += flip;
          b1 += flip;
          sa_at += flip_s;
          sb_at += flip_s;
          __builtin_amdgcn_sched_barrier(0);
        }
        const int ahead = (i + 2) & 7;   // rows 0 and 1: of the next block
        x[(i + 2) & 3] = frag(a0, a1, ahead);
        row_scale[(i + 2) & 3] = scale(sa_at, ahead);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          p[i & 1][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b[j], x[i & 3], zero, 0, 0, 0, 0, 0, 0);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            acc[(i + 7) & 7][j][e] = fmaf(s[(i + 1) & 1], p[(i + 1) & 1][j][e], acc[(i + 7) & 7][j][e]);
          asm volatile("" : "+v"(acc[(i + 7) & 7][j]));   // here, not behind the loop's other blocks
          if (i == 7) b[j] = frag(b0, b1, j);
        }
        s[i & 1] = s_b * row_scale[i & 3];
        if (i == 7) s_b = scale(sb_at, 0);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[7][j][e] = fmaf(s[1], p[1][j][e], acc[7][j][e]);
    // back to stage 0's addresses for the partial block
    if ((nfull & 1) != 0) {
      a0 -= kStage;
      a1 -= kStage;
      b0 -= kStage;
      b1 -= kStage;
      sa_at -= kScales;
      sb_at -= kScales;
    }
  }
  if (nfull * int64_t{128} < a.k) {   // the last, partial block: zeros past K
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(kWaitAll);
    __builtin_amdgcn_s_barrier();
    const int krem = static_cast<int>(a.k - nfull * int64_t{128});
    unsigned char* const l = smem + wave * 1024 + lane * 16;
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      const unsigned char* const src = (t < 4 ? pa + offA[t & 3] : pb + offB[t & 3]) + nfull * int64_t{128};
      alignas(16) unsigned char w[16];
      if (kcol + 16 <= krem) {
        *reinterpret_cast<u32x4*>(w) = *reinterpret_cast<const u32x4*>(src);
      } else {
#pragma unroll
        for (int k = 0; k < 16; ++k) w[k] = kcol + k < krem ? src[k] : 0;
      }
      *reinterpret_cast<u32x4*>(l + (t & 3) * 8192 + (t < 4 ? 0 : kOp)) = *reinterpret_cast<const u32x4*>(w);
    }
    issue_scales(nfull, 0);
    __builtin_amdgcn_s_waitcnt(kWaitAll);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    block(0);
  }
  // acc[i][j][e] is row m0 + wm·128 + 16i + lrow, column n0 + wn·64 + 16j + 4·lgrp + e.
  // Rows of bf16 leave as 16 bytes a lane: a swap of neighbouring groups of 16
  // lanes gives each eight consecutive columns of one fragment of a pair. Stored
  // past the caches: nothing here reads them again.
  OT* const C = static_cast<OT*>(a.c);
  const int64_t colw = n0 + wn * 64;
  const bool vec = n0 + kTile <= a.n && a.ldc * static_cast<int64_t>(sizeof(OT)) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(C) % 16 == 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t row = m0 + wm * 128 + i * 16 + lrow;
    OT* const d = C + row * a.ldc + colw;
    if (vec) {
      if constexpr (sizeof(OT) == 2) {
#pragma unroll
        for (int j = 0; j < 4; j += 2) {
          const f32x4 v = acc[i][j], w = acc[i][j + 1];
          const auto lo = __builtin_amdgcn_permlane16_swap(pack_bf16(v[0], v[1]), pack_bf16(w[0], w[1]), false, false);
          const auto hi = __builtin_amdgcn_permlane16_swap(pack_bf16(v[2], v[3]), pack_bf16(w[2], w[3]), false, false);
          if (row < a.m)
            __builtin_nontemporal_store(u32x4{lo[0], hi[0], lo[1], hi[1]},
                                        reinterpret_cast<u32x4*>(d + 16 * (j + (lgrp & 1)) + 8 * (lgrp >> 1)));
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (row < a.m) __builtin_nontemporal_store(acc[i][j], reinterpret_cast<f32x4*>(d + 16 * j + 4 * lgrp));
      }
    } else if (row < a.m) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int c = 16 * j + 4 * lgrp + e;
          if (colw + c < a.n) d[c] = static_cast<OT>(acc[i][j][e]);
        }
    }
  }
}

// ------------------------------------------------------------ few rows
// A token, a small batch: bound by the bytes of B, which each go once from memory
// to the registers of one wave, with no LDS and no barrier. A wave takes 16 rows of
// B and all rows of A (F fragments of 16, from the caches), loads the next two
// blocks while it multiplies these, and scales as above. One row at 131072 x 4096:
// 92 us, 5.9 TB/s (64 rows of B a wave, a block at a time, 115; four blocks 95; on
// the tiles 142).
template <typename OT, bool WIDE, int F>
__global__ __launch_bounds__(256) void fp8_few_kernel(Fp8MmArgs a) {
  constexpr int R = 1, U = 2;   // fragments of B, blocks in flight
  const int lane = threadIdx.x & 63;
  const int64_t n0 = (blockIdx.x * int64_t{4} + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * (16 * R);
  if (n0 >= a.n) return;
  const int lrow = lane & 15, lgrp = lane >> 4;
  const unsigned char *pa[F], *pb[R];
  const float* sa[F];
#pragma unroll
  for (int i = 0; i < F; ++i) {
    const int64_t r = i * 16 + lrow < a.m ? i * 16 + lrow : a.m - 1;   // the last row again: not stored
    pa[i] = a.a + r * a.lda + lgrp * 16;
    sa[i] = a.sa + r * a.sa_row;
  }
#pragma unroll
  for (int j = 0; j < R; ++j) {
    const int64_t r = n0 + j * 16 + lrow < a.n ? n0 + j * 16 + lrow : a.n - 1;
    pb[j] = a.b + r * a.ldb + lgrp * 16;
  }
  const float* const sb = a.sb + n0 / 128 * a.sb_row;
  f32x4 acc[F][R];
#pragma unroll
  for (int i = 0; i < F; ++i)
#pragma unroll
    for (int j = 0; j < R; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  struct Block {
    i32x8 a[F], b[R];
    float s[F];
  };
  // Chunks lgrp and 4 + lgrp of a row's block kb (as on the tiles).
  auto chunk = [&](const unsigned char* p, int64_t kb) {
    const u32x4 lo = *reinterpret_cast<const u32x4*>(p + kb * 128);
    const u32x4 hi = *reinterpret_cast<const u32x4*>(p + kb * 128 + 64);
    return __builtin_bit_cast(i32x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  };
  auto load = [&](Block& w, int64_t kb) {
#pragma unroll
    for (int j = 0; j < R; ++j) w.b[j] = chunk(pb[j], kb);
#pragma unroll
    for (int i = 0; i < F; ++i) w.a[i] = chunk(pa[i], kb);
    const float s_b = sb[kb * a.sb_col];
#pragma unroll
    for (int i = 0; i < F; ++i) w.s[i] = s_b * sa[i][kb * a.sa_col];
  };
  auto use = [&](const Block& w) {
#pragma unroll
    for (int j = 0; j < R; ++j) {
      if constexpr (WIDE) {
        const Wide n = widened(w.b[j]);
#pragma unroll
        for (int i = 0; i < F; ++i) {
          const Wide m = widened(w.a[i]);
          f32x4 p = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int q = 0; q < 4; ++q) p = __builtin_amdgcn_mfma_f32_16x16x32_bf16(n.k[q], m.k[q], p, 0, 0, 0);
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][j][e] = fmaf(w.s[i], p[e], acc[i][j][e]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < F; ++i) {
          const f32x4 p = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w.b[j], w.a[i], f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0,
                                                                           0, 0, 0, 0);
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][j][e] = fmaf(w.s[i], p[e], acc[i][j][e]);
        }
      }
    }
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
  const int krem = static_cast<int>(a.k - nfull * 128);
  if (krem > 0) {   // the partial block: zeros past K
    auto part = [&](const unsigned char* p) {
      alignas(16) unsigned char b[32];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int c = lgrp * 16 + h * 64;
        const unsigned char* q = p + nfull * 128 + h * 64;
        if (c + 16 <= krem) {
          *reinterpret_cast<u32x4*>(b + h * 16) = *reinterpret_cast<const u32x4*>(q);
        } else {
#pragma unroll
          for (int k = 0; k < 16; ++k) b[h * 16 + k] = c + k < krem ? q[k] : 0;
        }
      }
      i32x8 r;
      __builtin_memcpy(&r, b, 32);
      return r;
    };
    Block w;
#pragma unroll
    for (int j = 0; j < R; ++j) w.b[j] = part(pb[j]);
#pragma unroll
    for (int i = 0; i < F; ++i) {
      w.a[i] = part(pa[i]);
      w.s[i] = sb[nfull * a.sb_col] * sa[i][nfull * a.sa_col];
    }
    use(w);
  }
  OT* const C = static_cast<OT*>(a.c);
  const bool vec = a.ldc % 4 == 0 && reinterpret_cast<uintptr_t>(C) % (4 * sizeof(OT)) == 0;
#pragma unroll
  for (int i = 0; i < F; ++i) {
    const int64_t row = i * 16 + lrow;
    if (row >= a.m) continue;
#pragma unroll
    for (int j = 0; j < R; ++j) {
      const int64_t col = n0 + j * 16 + 4 * lgrp;
      OT* const d = C + row * a.ldc + col;
      const f32x4 v = acc[i][j];
      if (vec && col + 4 <= a.n) {
        if constexpr (sizeof(OT) == 2) *reinterpret_cast<u32x2*>(d) = u32x2{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])};
        else *reinterpret_cast<f32x4*>(d) = v;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (col + e < a.n) d[e] = static_cast<OT>(v[e]);
      }
    }
  }
}

template <typename OT, bool WIDE>
void (*few_kernel(int64_t m))(Fp8MmArgs) {
  return m <= 16 ? fp8_few_kernel<OT, WIDE, 1> : m <= 32 ? fp8_few_kernel<OT, WIDE, 2> : fp8_few_kernel<OT, WIDE, 4>;
}

// Whether the product runs there: always up to 16 rows; up to 64 where reading A in
// every wave costs less than the tiles' rounds. Both sides' us fitted at 32 and 64
// rows of 4096 x 131072 (203 and 211 against 147), 4096 x 32000 (50 and 114, fp32
// 46 and 78, against 51, fp32 111) and 1000 x 11000 (18 against 25 to 48).
bool few_rows(const Fp8MmArgs& a, bool wide) {
  if (a.m <= 16) return true;
  if (a.m > 64) return false;
  const double few = static_cast<double>(a.n) * a.k * (a.m <= 32 ? 3.8e-7 : wide ? 5.9e-7 : 8.7e-7);
  const double blocks = static_cast<double>((a.k + 127) / 128);
  const double tiles = static_cast<double>(((a.n + kTile - 1) / kTile + 255) / 256) * (blocks * (wide ? 3.3 : 1.4) + 8.0);
  return few < tiles;
}

}  // namespace

hipError_t launch_fp8_quant(const Fp8QuantArgs& a, DType t, bool blocks, hipStream_t stream) {
  if (a.rows <= 0 || a.cols <= 0) return hipSuccess;
  if (a.ldc % 8 != 0 || reinterpret_cast<uintptr_t>(a.codes) % 8 != 0) return hipErrorInvalidValue;
  const int64_t each = blocks ? 128 : 16, across = blocks ? (a.cols + 127) / 128 : (a.cols + 511) / 512;
  const int64_t most = most_blocks(256) / across * each;   // rows of a launch
  using K = void (*)(Fp8QuantArgs);
  const int64_t at = reinterpret_cast<uintptr_t>(a.src) | static_cast<uint64_t>(a.lds * dtype_size(t));
  K k;
  if (!blocks) k = t == DType::BF16 ? static_cast<K>(fp8_quant_rows_kernel<__bf16>) : fp8_quant_rows_kernel<float>;
  else if (t == DType::F32) k = at % 16 == 0 ? fp8_quant_blocks_kernel<float, 4, true>
                              : at % 8 == 0  ? fp8_quant_blocks_kernel<float, 2, true>
                                             : fp8_quant_blocks_kernel<float, 1, true>;
  else k = at % 16 == 0  ? fp8_quant_blocks_kernel<__bf16, 8, true>
           : at % 8 == 0 ? fp8_quant_blocks_kernel<__bf16, 4, true>
           : at % 4 == 0 ? fp8_quant_blocks_kernel<__bf16, 2, true>
                         : fp8_quant_blocks_kernel<__bf16, 8, false>;
  for (int64_t r = 0; r < a.rows; r += most) {
    Fp8QuantArgs p = a;
    p.rows = a.rows - r < most ? a.rows - r : most;
    p.src = static_cast<const char*>(a.src) + r * a.lds * dtype_size(t);
    p.codes = a.codes + r * a.ldc;
    p.scales = a.scales + r / (blocks ? 128 : 1) * a.scale_row;
    hipLaunchKernelGGL(k, dim3(static_cast<unsigned>((p.rows + each - 1) / each * across)), dim3(256), 0, stream, p);
  }
  return hipGetLastError();
}

hipError_t launch_fp8_pack(const uint8_t* src, int64_t lds, int64_t rows, int64_t cols, uint8_t* dst, int64_t ldd,
                           hipStream_t stream) {
  if (ldd % 16 != 0 || reinterpret_cast<uintptr_t>(dst) % 16 != 0) return hipErrorInvalidValue;
  const int64_t n = (rows * (ldd / 16) + 255) / 256;
  if (n <= 0) return hipSuccess;
  hipLaunchKernelGGL(fp8_pack_kernel, dim3(static_cast<unsigned>(n < 65536 ? n : 65536)), dim3(256), 0, stream, src, lds,
                     rows, cols, dst, ldd);
  return hipGetLastError();
}

hipError_t launch_fp8_mm(const Fp8MmArgs& a, DType out, hipStream_t stream) {
  if (a.m <= 0 || a.n <= 0) return hipSuccess;
  if (a.lda % 16 != 0 || a.ldb % 16 != 0 || reinterpret_cast<uintptr_t>(a.a) % 16 != 0 ||
      reinterpret_cast<uintptr_t>(a.b) % 16 != 0)
    return hipErrorInvalidValue;
  if (few_rows(a, out == DType::F32)) {
    auto* k = out == DType::BF16 ? few_kernel<__bf16, false>(a.m) : few_kernel<float, true>(a.m);
    constexpr int64_t kMost = most_blocks(256) / 2 * 128;   // columns of a launch, whole blocks of B
    for (int64_t n0 = 0; n0 < a.n; n0 += kMost) {
      Fp8MmArgs p = a;
      p.n = a.n - n0 < kMost ? a.n - n0 : kMost;
      p.b = a.b + n0 * a.ldb;
      p.sb = a.sb + n0 / 128 * a.sb_row;
      p.c = static_cast<char*>(a.c) + n0 * dtype_size(out);
      hipLaunchKernelGGL(k, dim3(static_cast<unsigned>((p.n + 63) / 64)), dim3(256), 0, stream, p);
    }
    return hipGetLastError();
  }
  const int64_t tiles = (a.m + kTile - 1) / kTile * ((a.n + kTile - 1) / kTile);
  if (tiles > most_blocks(kThreads)) return hipErrorInvalidValue;   // 1 TB of outputs
  auto* k = out == DType::BF16 ? fp8_mm_kernel<__bf16, false> : fp8_mm_kernel<float, true>;
  hipLaunchKernelGGL(k, dim3(static_cast<unsigned>(tiles)), dim3(kThreads), 0, stream, a);
  return hipGetLastError();
}

}  // namespace orda
