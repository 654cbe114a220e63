// tree_attn.h -- parameters of the attention of a drafted tree (tree_attn.hip).
#pragma once
#include "kv_common.h"

namespace vkv {

struct TreeParams {
    const uint8_t* k;
    const uint8_t* v;
    const uint16_t* ks;
    const uint16_t* vs;
    const int32_t* block_tables;
    const int32_t* block_used;  // or null
    const int32_t* start_pos;
    const int32_t* tree_lens;   // or null: nodes each
    const uint64_t* tree_mask;  // or null: a chain
    const void* q;
    void* out;
    uint32_t batch, nodes, hq, hkv, group;
    uint32_t block_tokens, max_blocks, num_blocks;
    uint32_t block_magic, block_shift;  // table entry of a tile (tree_block_of)
    float scale;       // softmax scale * log2(e)
    float alpha;       // std-clamp alpha
    float logit_clip;  // 24 * log2(e) in 3-bit mode, +inf otherwise
    float input_clip;  // 16 in 3-bit mode, +inf otherwise
    // work split: an item is (sequence, kv head, group of column tiles); its steps are cut into
    // up to `parts` parts of at least part_steps steps, a workgroup each
    uint32_t parts, part_steps;
    uint32_t col_groups;  // of col_waves * CT tiles of 16 columns
    uint32_t col_waves;   // waves of a workgroup side by side over columns: 1, 2 or 4
    float* part_acc;      // [item][part][column tile][D/16][lane][4]
    float* part_ml;       // [item][part][column tile][16][2]: reference point (log2 units), sum
};

// The table entry of a tile, tile / (tiles of a block), as a product: tiles are below 2^27, and with 2^(s-1) <
// block tiles <= 2^s, block_magic = 16 ceil(2^(27+s) / block tiles) and block_shift = s it is exact.  (A division
// by a number known only at run time is some 30 scalar instructions, four times a step.)
__device__ __forceinline__ int tree_block_of(uint32_t magic, uint32_t shift, int tile) {
    return (int)(__umulhi(2u * (uint32_t)tile, magic) >> shift);
}

// A value that every lane holds alike, in a scalar register: what follows from a division (done on the
// vector unit) would otherwise keep addresses and loop counts in vector registers.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// A sequence's slots: [0, start) are the prefix, start + j is node j, j < len.
struct TreeSpan {
    int start, len, end;  // end: slots that the table holds of both
};
__device__ __forceinline__ TreeSpan tree_span(const TreeParams& p, uint32_t b) {
    const int cap = (int)min((uint64_t)p.max_blocks * p.block_tokens, (uint64_t)0x7fffff00u);
    TreeSpan s;
    s.start = min(max(as_const(p.start_pos)[b], 0), cap);
    s.len = p.tree_lens ? min(max(as_const(p.tree_lens)[b], 0), (int)p.nodes) : (int)p.nodes;
    s.end = min(s.start + s.len, cap);
    s.start = uniform(s.start);
    s.len = uniform(s.len);
    s.end = uniform(s.end);
    return s;
}
// Bits of the nodes that node i of sequence b sees.
__device__ __forceinline__ uint64_t tree_bits(const TreeParams& p, uint32_t b, int i, int len) {
    const uint64_t all = len >= 64 ? ~0ull : (1ull << len) - 1;
    const uint64_t m = p.tree_mask ? p.tree_mask[(size_t)b * p.nodes + i] : (2ull << i) - 1;
    return i < len ? m & all : 0;
}

// Element e of the value row in `slot` of (block, head) bh where it may be other than finite
// (of an int4 pool: else 0, a code times a finite scale is finite).
template <int DT, int D>
__device__ __forceinline__ float tree_value(const uint8_t* values, const uint16_t* scales, uint32_t P, size_t bh, uint32_t slot, uint32_t e) {
    if constexpr (DT == VSPEC_KV_F32) return reinterpret_cast<const float*>(values)[(bh * P + slot) * D + e];
    if constexpr (DT == VSPEC_KV_F16) return half_bits_to_float(reinterpret_cast<const uint16_t*>(values)[f16_v_index(bh, P, D, slot, e)]);
    uint32_t high;
    const uint8_t c = values[int4_v_byte(bh, P, D, slot, e, &high)];
    const uint32_t s = scales[(bh * P + slot) * (D / 32) + e / 32];
    return (s & 0x7fffu) < 0x7C00u ? 0.f : nibble((uint32_t)c, (int)high) * half_bits_to_float(s);
}

// A sequence's steps of NT tiles: first the tiles that hold prefix alone, then those from the first
// node's on.  Part i of them begins at step i * chunk.
struct TreeParts {
    int tiles, prefix_tiles, prefix_steps;
    int steps, count, chunk;
};
template <int NT>
__device__ __forceinline__ TreeParts tree_parts(const TreeParams& p, const TreeSpan& s) {
    TreeParts r;
    r.tiles = s.len ? (s.end + kTile - 1) / kTile : 0;  // (no nodes: nothing to read)
    r.prefix_tiles = min(s.start / kTile, r.tiles);
    r.prefix_steps = (r.prefix_tiles + NT - 1) / NT;
    r.steps = r.prefix_steps + (r.tiles - r.prefix_tiles + NT - 1) / NT;
    const int most = max(1, min((int)p.parts, (r.steps + (int)p.part_steps - 1) / (int)p.part_steps));
    r.chunk = uniform(max(1, (r.steps + most - 1) / most));
    r.count = uniform(max(1, (r.steps + r.chunk - 1) / r.chunk));
    return r;
}

// A scalar of its own.  Arguments are loaded eight or sixteen registers at a time, and short of scalar
// registers the compiler keeps and restores such a tuple whole for one of its members (measured: 16 lane reads
// for each).
template <typename T>
__device__ __forceinline__ T own_scalar(T x) {
    T y;
    if constexpr (sizeof(T) == 8) asm volatile("s_mov_b64 %0, %1" : "=s"(y) : "s"(x));
    else asm volatile("s_mov_b32 %0, %1" : "=s"(y) : "s"(x));
    return y;
}

// The kernel's own arguments, read again where they are needed: kept from the start they would fill the scalar
// registers of the main loop.
typedef const __attribute__((address_space(4))) TreeParams kernel_args;
__device__ __forceinline__ kernel_args* late_args() {
    kernel_args* a = (kernel_args*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(a));
    return a;
}

// Launch the kernels of one pool type and head size (tree_mfma.hip): ct column tiles a wave.
void launch_tree_f32_d64(const TreeParams& p, int32_t io, uint32_t ct, hipStream_t s);
void launch_tree_f32_d128(const TreeParams& p, int32_t io, uint32_t ct, hipStream_t s);
void launch_tree_f16_d64(const TreeParams& p, int32_t io, uint32_t ct, hipStream_t s);
void launch_tree_f16_d128(const TreeParams& p, int32_t io, uint32_t ct, hipStream_t s);
void launch_tree_int4_d64(const TreeParams& p, int32_t io, uint32_t ct, hipStream_t s);
void launch_tree_int4_d128(const TreeParams& p, int32_t io, uint32_t ct, hipStream_t s);
// The same for more than 32 columns (tree_wide.hip): col_waves 4 or 8 waves, ct 1 or 2 tiles each
void launch_tree_wide_f16_d64(const TreeParams& p, int32_t io, uint32_t ct, hipStream_t s);
void launch_tree_wide_f16_d128(const TreeParams& p, int32_t io, uint32_t ct, hipStream_t s);
void launch_tree_wide_int4_d64(const TreeParams& p, int32_t io, uint32_t ct, hipStream_t s);
void launch_tree_wide_int4_d128(const TreeParams& p, int32_t io, uint32_t ct, hipStream_t s);
// 16-token tiles of a step
constexpr int wide_step_tiles(bool f32_rows, int ct) { return f32_rows || ct > 1 ? 2 : 4; }
constexpr int tree_step_tiles(int dtype) { return dtype == VSPEC_KV_F32 ? 1 : 2; }
// Workgroups of tree_mfma.hip that a CU holds.  Two hide each other's waits, where 256 registers a
// lane hold K, V, q and the output without spilling more than a few.
constexpr int tree_cu_groups(int dtype, int d, bool f32_rows, int ct) {
    return ct == 1 || d == 64 || dtype == VSPEC_KV_F32 || (dtype == VSPEC_KV_F16 && !f32_rows) ? 2 : 1;
}

}  // namespace vkv
