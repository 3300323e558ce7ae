// pz_lmdev.h -- what the LM heads' kernels (bf16, 8-bit integers) share: loads
// straight to LDS, their waits, and the keys of the fused argmax.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "pz_device.h"

typedef uint32_t lm_u32x4 __attribute__((ext_vector_type(4)));
typedef float lm_f32x4 __attribute__((ext_vector_type(4)));

// Key of logit v of id: the largest key is the first maximum.
__device__ __forceinline__ uint64_t argmax_key(float v, int id) {
  return ((uint64_t)pz_key(v) << 32) | (uint64_t)(0xffffffffu - (uint32_t)id);
}

// Keys of the fused argmax spread over LMM_SLOTS slots per batch row (one
// per workgroup index modulo LMM_SLOTS, each on its own cache line), so the
// workgroups' atomics do not all meet on the batch's few words.
constexpr int LMM_SLOTS = 16;

// 16 bytes per lane from base + off to LDS at byte address lds + 16 lane.
// (Written as asm because for the builtin the compiler orders every later
// LDS read of the workgroup behind all such loads; the stage loop below
// waits for exactly the loads that it needs.  M0, the LDS base, is a clobber:
// a value that the compiler keeps there is not taken for one that survived.)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // (M0 is a reserved register)
template <bool NT>
__device__ __forceinline__ void lm_lds_load16(const void* base, uint32_t off, uint32_t lds) {
  if (NT)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt"
                 :
                 : "s"(lds), "v"(off), "s"(base)
                 : "m0", "memory");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                 :
                 : "s"(lds), "v"(off), "s"(base)
                 : "m0", "memory");
}
#pragma clang diagnostic pop
// At most N of this wave's vector memory operations, and none of its LDS
// operations, still outstanding.
template <int N>
__device__ __forceinline__ void lm_wait() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" : : "n"(N) : "memory");
}
