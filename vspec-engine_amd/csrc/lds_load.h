// lds_load.h -- tile loads straight into LDS, for the kernels that stream tiles through an LDS ring
// (decode_mfma_int4.hip, tree_wide.hip).
#pragma once
#include "kv_common.h"

namespace vkv {
namespace {

// ---- tile loads straight into LDS (buffer_load ... lds) ----
//
// A wave's next tiles stream into an LDS ring while it works on the current ones, so the loads
// in flight take no VGPRs.  Each load goes through a buffer
// descriptor bounded to the tile's bytes (out-of-range lanes and descriptors of size 0
// write zeros and read nothing), built on the scalar unit per tile; the per-lane offsets
// are loop invariants.  Lane i of a load writes its bytes at M0 + size * i.
//
// The loads are issued from inline asm (a compiler-visible LDS DMA makes every later LDS
// read wait for all of them), so their waits are explicit: vector memory operations
// complete in issue order, and s_waitcnt vmcnt(n) returns once at most n are in flight,
// so waiting for all loads issued after a tile's lands that tile.  Loads the
// compiler issues itself in between could only make such a wait longer.
typedef int32_t rsrc_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ rsrc_t tile_rsrc(const void* base, uint32_t bytes) {
    const uint64_t a = reinterpret_cast<uint64_t>(base);
    // word 1: base bits 32..47, stride 0 (the host admits pool addresses below 2^47, so
    // bits 48..63 are zero); word 3: 32-bit data format (raw buffer access)
    return rsrc_t{(int32_t)(uint32_t)a, (int32_t)(uint32_t)(a >> 32), (int32_t)bytes, 0x00020000};
}
__device__ __forceinline__ uint32_t lds_addr(const void* p) { return (uint32_t)reinterpret_cast<uintptr_t>(p); }
// 16 (4) bytes per lane from the descriptor's base + voff into LDS at lds + 16 (4) * lane
__device__ __forceinline__ void lds_load16(uint32_t lds, rsrc_t r, uint32_t voff) {
    asm volatile("buffer_load_dwordx4 %0, %1, 0 offen nt lds" ::"v"(voff), "s"(r), "{m0}"(lds) : "memory");
}
__device__ __forceinline__ void lds_load4(uint32_t lds, rsrc_t r, uint32_t voff) {
    asm volatile("buffer_load_dword %0, %1, 0 offen nt lds" ::"v"(voff), "s"(r), "{m0}"(lds) : "memory");
}

template <int N>
__device__ __forceinline__ void wait_loads() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// LDS reads done (before a load overwrites what they read)
__device__ __forceinline__ void wait_lds_reads() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

}  // namespace
}  // namespace vkv
