// mkv_dma.h — loads straight from global memory into LDS, and their completion, shared by
// the decode attention kernels.
#pragma once

#include "mkv_device.h"

namespace mkv {

// Orders this wave's LDS writes before its later LDS reads (other lanes').
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// ---- direct-to-LDS loads and their completion ---------------------------------
//
// The loads are issued from inline assembly, so the compiler neither inserts
// waits for them nor reorders LDS accesses across them ("memory" clobber);
// every wait on them is explicit below. M0 holds the LDS destination of the
// lane-0 bytes (the hardware adds 16 or 4 bytes per lane). The statements do
// not tell the compiler that they write it, so a source that includes this
// file must use nothing else that goes through M0 (LDS DMA builtins, GWS,
// message or movrel instructions). Before a slot is refilled, the wave's
// earlier LDS reads of it must have returned: lgkmcnt(0) first.

__device__ __forceinline__ uint32_t lds_addr(const void* p) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p;
}
// A wave-uniform pointer in scalar registers (the compiler cannot always
// prove uniformity through the index arithmetic).
__device__ __forceinline__ const void* uniform_ptr(const void* p) {
  const uint64_t u = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)u);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(u >> 32));
  return reinterpret_cast<const void*>(((uint64_t)hi << 32) | lo);
}
// 16 bytes per lane from base + voff (saddr form: base scalar, voff per lane)
__device__ __forceinline__ void dma16(const void* base, uint32_t voff, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt"
               :
               : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(voff), "s"(uniform_ptr(base))
               : "memory");
}
// the same through the caches (pages several sequences read: a prefix
// shared through the block manager)
__device__ __forceinline__ void dma16_cached(const void* base, uint32_t voff, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
               :
               : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(voff), "s"(uniform_ptr(base))
               : "memory");
}
// 4 bytes per lane from a per-lane 64-bit address
__device__ __forceinline__ void dma4(const void* addr, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off nt"
               :
               : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(addr)
               : "memory");
}
__device__ __forceinline__ void lds_reads_done() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
template <int N>
__device__ __forceinline__ void vm_wait_n() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

}  // namespace mkv
