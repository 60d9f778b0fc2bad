// Direct global-to-LDS loads and the waits and barrier of a ring of LDS slots that they fill.
#pragma once

#include "common.hpp"

namespace frt {

typedef __attribute__((address_space(3))) void* lds_ptr_t;
typedef const __attribute__((address_space(1))) void* gbl_ptr_t;
// direct global -> LDS load of 16 bytes per lane to lds_base + 16 lane (lds_base uniform)
__device__ __forceinline__ void ldsdma16(const void* g, void* lds_base) {
    __builtin_amdgcn_global_load_lds((gbl_ptr_t)g, (lds_ptr_t)lds_base, 16, 0, 0);
}
// the same as a non-temporal (streaming) load, for bytes that are read once
__device__ __forceinline__ void ldsdma16_nt(const void* g, void* lds_base) {
    __builtin_amdgcn_global_load_lds((gbl_ptr_t)g, (lds_ptr_t)lds_base, 16, 0, 2);
}
// the same with 4 bytes per lane, to lds_base + 4 lane
__device__ __forceinline__ void ldsdma4(const void* g, void* lds_base) {
    __builtin_amdgcn_global_load_lds((gbl_ptr_t)g, (lds_ptr_t)lds_base, 4, 0, 0);
}
// A workgroup barrier that does not wait for outstanding global loads (__syncthreads' release fence
// would wait for all of them, the ring's later stages included): this wave's LDS accesses complete,
// then s_barrier. The wait is the builtin (so the compiler's own wait insertion knows the LDS reads
// before it are complete); the empty asm statements keep memory accesses from moving across.
__device__ __forceinline__ void ring_barrier() {
    __builtin_amdgcn_sched_barrier(0);   // nothing is scheduled across (register math included)
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xC07F);   // lgkmcnt(0); vmcnt and expcnt not waited for
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}
// this wave's LDS reads have returned, before anything after this is issued (direct global-to-LDS loads
// may then overwrite what they read)
__device__ __forceinline__ void lds_reads_done() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xC07F);   // lgkmcnt(0)
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}
// s_waitcnt with vmcnt = N (gfx9 encoding; expcnt and lgkmcnt not waited for)
template <int N>
__device__ __forceinline__ void wait_vm() {
    __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | 0x70 | 0xF00);
}
}  // namespace frt
