// lds_dma.h — global memory to LDS by DMA, ordered by explicit waits.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace orda {

typedef __attribute__((address_space(3))) void lds_void;

// s_waitcnt encodings (gfx9): vmcnt in bits 3:0 and 15:14, expcnt 6:4,
// lgkmcnt 11:8. Both wait for every LDS operation.
constexpr int kWaitAll = 0x0070;                              // vmcnt(0) lgkmcnt(0)
constexpr int vm_wait(int n) { return 0x0070 | (n & 15) | ((n >> 4) << 14); }
constexpr int kWaitLds = 0xC07F;                              // lgkmcnt(0) only

// One DMA transfer: every active lane copies the 16 bytes at sbase + voff
// into LDS at M0 + 16 * lane (global_load_lds_dwordx4, saddr form). Written as
// inline asm so that the compiler's memory-counter bookkeeping does not see
// the transfers: it would otherwise make every later LDS transpose read wait
// for all of them (vmcnt(0)). The kernel orders DMA and reads itself with
// explicit s_waitcnt + s_barrier. M0 is reserved by the compiler, hence the
// clobber (nothing else in these kernels keeps a value in M0).
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void dma16(const unsigned char* sbase, uint32_t voff, unsigned char* l) {
  // sbase and the LDS destination are wave-uniform; readfirstlane states it
  // to the compiler so that they live in SGPRs also inside divergent code.
  // (readfirstlane returns int: each half goes through uint32_t so that the
  // low half is not sign-extended into the high one.)
  const uint64_t p = reinterpret_cast<uint64_t>(sbase);
  const uint32_t lo = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(p)));
  const uint32_t hi =
      static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(p >> 32)));
  const uint64_t ps = (static_cast<uint64_t>(hi) << 32) | lo;
  const uint32_t m0 = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(
      static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_void*)l))));
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %0"
               :
               : "s"(ps), "v"(voff), "s"(m0)
               : "memory", "m0");
}
// Main-loop form: M0 = m0base + imm in one SALU add (the caller keeps
// m0base = the stage slot's LDS offset + this wave's 1 KB block).
template <int IMM>
__device__ __forceinline__ void dma16_at(uint64_t sbase, uint32_t voff, uint32_t m0base) {
  asm volatile("s_add_u32 m0, %2, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %0"
               :
               : "s"(sbase), "v"(voff), "s"(m0base), "n"(IMM)
               : "memory", "m0", "scc");
}
// 4 bytes a lane, to M0 + 4 * lane.
__device__ __forceinline__ void dma4(uint64_t sbase, uint32_t voff, uint32_t m0) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %1, %0"
               :
               : "s"(sbase), "v"(voff), "s"(m0)
               : "memory", "m0");
}
#pragma clang diagnostic pop
// A wave-uniform 64-bit value in an SGPR pair.
__device__ __forceinline__ uint64_t uniform64(const void* p) {
  const uint64_t v = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v)));
  const uint32_t hi =
      static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v >> 32)));
  return (static_cast<uint64_t>(hi) << 32) | lo;
}

}  // namespace orda
