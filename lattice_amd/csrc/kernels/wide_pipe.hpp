// Pieces of the two products on 256-row tiles (gemm_wide.hip,
// gemm_epi_wide.hip): direct loads into LDS, counted waits, bare barriers, the
// order of tiles over the XCDs.
#pragma once
#include "common.hpp"

namespace kcmm {
namespace {

typedef __attribute__((address_space(3))) void* lds_ptr;

// 16 bytes per lane from global memory straight into LDS at lds + 16 * lane
// (lds is wave-uniform).
__device__ __forceinline__ void load_lds16(const uint8_t* g, uint8_t* lds) {
    __builtin_amdgcn_global_load_lds(g, (lds_ptr)lds, 16, 0, 0);
}

// The same, nontemporal (weights that one token tile reads once).
__device__ __forceinline__ void load_lds16_nt(const uint8_t* g, uint8_t* lds) {
    __builtin_amdgcn_global_load_lds(g, (lds_ptr)lds, 16, 0, 2);
}

// s_waitcnt vmcnt(N) lgkmcnt(0) (gfx9 encoding: vmcnt bits 3:0 and 15:14,
// expcnt 6:4, lgkmcnt 11:8).
template <int N>
__device__ __forceinline__ void wait_vm_lgkm0() {
    static_assert(N >= 0 && N < 64, "vmcnt is 6 bits");
    asm volatile("" ::: "memory");   // the LDS reads before it stay before it
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt((N & 0xF) | ((N >> 4) << 14) | (0x7 << 4));
}

// A bare barrier (a fenced one would wait for the loads in flight), which no
// memory access moves across.
__device__ __forceinline__ void phase_barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
}

// The idx-th tile of a run of n workgroups, so that each XCD (workgroup i of
// a grid runs on XCD i % 8) takes a contiguous piece of the tile list.
__device__ __forceinline__ int xcd_order(int idx, int n) {
    const int x = idx & 7, q = n >> 3, r = n & 7;
    return x * q + min(x, r) + (idx >> 3);
}

}  // namespace
}  // namespace kcmm
