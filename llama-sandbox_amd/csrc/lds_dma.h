// lds_dma.h -- loads from global memory straight to LDS, and the waits for them.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#define MOE_LDS_OOB 0xffffff00u  // a lane offset past any buffer: the load returns 0
#define MOE_LDS_RSRC 0x00020000  // raw buffer, 32-bit dwords, no swizzle

// Waits for vmcnt <= n only (gfx9 encoding), then for this wave's LDS reads, then for every wave.
template <int N>
__device__ __forceinline__ void lds_wait_barrier() {
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | 0x70 | 0xF00);
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// 64 lanes' 16 bytes at base + vo + so into the 1 KiB at buf; _once: read by no other
// workgroup (non-temporal).
__device__ __forceinline__ void lds_dma(const void *base, uint32_t bytes, void *buf, uint32_t vo, uint32_t so) {
  typedef __attribute__((address_space(3))) void *lds_t;
  const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void *)base, 0, (int)bytes, MOE_LDS_RSRC);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_t)buf, 16, vo, so, 0, 0);
}
__device__ __forceinline__ void lds_dma_once(const void *base, uint32_t bytes, void *buf, uint32_t vo, uint32_t so) {
  typedef __attribute__((address_space(3))) void *lds_t;
  const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void *)base, 0, (int)bytes, MOE_LDS_RSRC);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_t)buf, 16, vo, so, 0, 2);
}
