// wave.h — sums and maxima over a wave's 64 lanes by moves between neighbouring lanes,
// which take neither LDS nor its latency.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace orda {
namespace {

// Each lane's value and those of the lanes before it; of rows of 16 lanes alone.
struct Sum {
  template <typename T>
  __device__ __forceinline__ T operator()(T a, T b) const { return a + b; }
};
struct Most {   // of whole numbers from 0 on
  template <typename T>
  __device__ __forceinline__ T operator()(T a, T b) const { return a > b ? a : b; }
};
template <int MOVE, int ROWS, typename T>
__device__ __forceinline__ T moved(T v) {   // 0 where nothing is moved to
  if constexpr (sizeof(T) == 4) {
    return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), MOVE, ROWS, 0xf, false));
  } else {
    const auto u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(u), MOVE, ROWS, 0xf, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(u >> 32), MOVE, ROWS, 0xf, false);
    return __builtin_bit_cast(T, static_cast<uint64_t>(hi) << 32 | lo);
  }
}
template <typename Op, typename T>
__device__ __forceinline__ T row_scan(T v, Op op) {
  v = op(v, moved<0x111, 0xf>(v));   // from 1, 2, 4 and 8 lanes before
  v = op(v, moved<0x112, 0xf>(v));
  v = op(v, moved<0x114, 0xf>(v));
  return op(v, moved<0x118, 0xf>(v));
}
template <typename Op, typename T>
__device__ __forceinline__ T wave_scan(T v, Op op) {
  v = row_scan(v, op);
  v = op(v, moved<0x142, 0xa>(v));   // a row's last to the row after, then to the two after
  return op(v, moved<0x143, 0xc>(v));
}
// The largest of each LANES (8 or 16) neighbouring lanes, in all of them.
template <int LANES>
__device__ __forceinline__ uint32_t most_of(uint32_t v) {
  const Most op;
  v = op(v, moved<0xb1, 0xf>(v));    // from the lane 1 and then 2 apart,
  v = op(v, moved<0x4e, 0xf>(v));
  v = op(v, moved<0x141, 0xf>(v));   // the mirrored ones of 8 and of 16
  return LANES == 8 ? v : op(v, moved<0x140, 0xf>(v));
}
template <typename T>
__device__ __forceinline__ T lane_of(T v, int lane);
// The wave's largest, given values that each LANES (8 or 16) neighbouring lanes have alike.
template <int LANES>
__device__ __forceinline__ uint32_t most_of_rows(uint32_t v) {
  const Most op;
  if constexpr (LANES == 8) v = op(v, moved<0x118, 0xf>(v));
  v = op(v, moved<0x142, 0xa>(v));
  return lane_of(op(v, moved<0x143, 0xc>(v)), 63);
}
template <typename T>
__device__ __forceinline__ T lane_of(T v, int lane) {
  if constexpr (sizeof(T) == 4) {
    return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
  } else {
    const auto u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(u), lane);
    const uint32_t hi = __builtin_amdgcn_readlane(static_cast<int>(u >> 32), lane);
    return __builtin_bit_cast(T, static_cast<uint64_t>(hi) << 32 | lo);
  }
}
template <typename T>
__device__ __forceinline__ T wave_sum(T x) { return lane_of(wave_scan(x, Sum{}), 63); }

// A value that all lanes have, in scalar registers.
template <typename T>
__device__ __forceinline__ T uniform(T v) {
  if constexpr (sizeof(T) == 4) {
    return __builtin_bit_cast(T, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, v)));
  } else {
    const auto u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(u));
    const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(u >> 32));
    return __builtin_bit_cast(T, static_cast<uint64_t>(hi) << 32 | lo);
  }
}

}  // namespace
}  // namespace orda
