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
    float scale;       // softmax scale * log2(e)
    float alpha;       // std-clamp alpha
    float logit_clip;  // 24 * log2(e) in 3-bit mode, +inf otherwise
    float input_clip;  // 16 in 3-bit mode, +inf otherwise
};

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
    return s;
}
// Bits of the nodes that node i of sequence b sees.
__device__ __forceinline__ uint64_t tree_bits(const TreeParams& p, uint32_t b, int i, int len) {
    const uint64_t all = len >= 64 ? ~0ull : (1ull << len) - 1;
    const uint64_t m = p.tree_mask ? p.tree_mask[(size_t)b * p.nodes + i] : (2ull << i) - 1;
    return i < len ? m & all : 0;
}

}  // namespace vkv
