// tcgen05 primitives shared by the kernels on the 5th-generation tensor cores
// (tgemm.cu, kv4_prompt.cu).
#pragma once

#include "kcommon.cuh"

namespace swl {

__device__ __forceinline__ uint64_t tg_desc(uint32_t saddr) {
  // K-major operand, 128-byte swizzle: 8-row groups of 128-byte rows 1024
  // bytes apart (SBO), descriptor version 1 (sm_100)
  return uint64_t((saddr >> 4) & 0x3FFFu) | (uint64_t(1) << 16) | (uint64_t(1024 >> 4) << 32) | (uint64_t(1) << 46) |
         (uint64_t(2) << 61);
}
__device__ __forceinline__ void tg_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void tg_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tg_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tg_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// Pipeline wait: polls without sleeping for the first ~4k tries (hand-offs
// between the roles are short), then backs off; gives up after about 2 s.
__device__ __forceinline__ bool tg_wait(uint64_t* b, unsigned parity) {
  if (mbar_try(b, parity)) return true;
  const unsigned long long t0 = gtimer();
  for (int i = 0; i < (1 << 26); ++i) {
    if (mbar_try(b, parity)) return true;
    if (i >= 4096) __nanosleep(128);
    if ((i & 255) == 0 && gtimer() - t0 > kWaitLimitNs) break;
  }
  return false;
}

}  // namespace swl
