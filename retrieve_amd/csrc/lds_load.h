// Loads straight to LDS, and the waits of kernels that keep several stages of them in flight.
#pragma once

#include "rt_common.h"

namespace rt {

// Cache-policy bits of direct-to-LDS loads of data that is read once (nontemporal).
constexpr int kNontemporal = 2;
// Word 3 of a raw buffer descriptor (stride 0, byte offsets; out-of-range loads return zeros).
constexpr int kBufferWord3 = 0x00020000;

// BYTES per lane from base + voffset (out-of-range past base + range: zeros) straight into LDS at
// lds + lane * BYTES (lds wave-uniform); NT: nontemporal. (The builtin's size and cache-policy
// operands must be literals, not template parameters.)
template <int BYTES, bool NT>
__device__ inline void buffer_load_lds(const void* base, int range, int voffset, void* lds) {
  static_assert(BYTES == 4 || BYTES == 16, "load size");
  const __amdgpu_buffer_rsrc_t rs =
      __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, range, kBufferWord3);
  auto* l = (__attribute__((address_space(3))) void*)(lds);
  if constexpr (BYTES == 4) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, l, 4, voffset, 0, 0, 0);
  } else if constexpr (NT) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, l, 16, voffset, 0, 0, kNontemporal);
  } else {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, l, 16, voffset, 0, 0, 0);
  }
}

// s_waitcnt immediate: vmcnt <= N (N < 64), expcnt and lgkmcnt unconstrained (gfx9 encoding).
template <int N>
__device__ inline void wait_vmcnt() {
  static_assert(N >= 0 && N < 64, "vmcnt range");
  __builtin_amdgcn_s_waitcnt((N & 0xf) | ((N >> 4) << 14) | (0x7 << 4) | (0xf << 8));
}

// vmcnt <= later * LOADS for a wave-uniform later in [0, MAXL] (the immediate must be constant).
template <int LOADS, int MAXL>
__device__ inline void wait_later(int later) {
  if constexpr (MAXL > 0) {
    if (later >= MAXL) {
      wait_vmcnt<MAXL * LOADS>();
      return;
    }
    wait_later<LOADS, MAXL - 1>(later);
  } else {
    wait_vmcnt<0>();
  }
}

// Workgroup barrier over the staged tiles: waits for this wave's LDS accesses (lgkmcnt(0)),
// then s_barrier. __syncthreads() would also wait for every outstanding global load (its
// workgroup release fence), draining the tiles still in flight; the direct-to-LDS loads of the
// tile about to be read are covered by the wait_vmcnt before this. The empty asm statements
// keep the compiler from moving memory accesses across the barrier.
__device__ inline void tile_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0), vmcnt and expcnt unconstrained
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

}  // namespace rt
