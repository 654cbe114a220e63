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
    // work split (tree_job): a row of the grid is a sequence or a part of one, for every kv head and group of column
    // tiles.  slot_rows: rows that the card holds at once (0: rows are sequences); min_units: least units of a part
    uint32_t rows, slot_rows, min_units;
    uint32_t col_groups;  // of col_waves * CT tiles of 16 columns
    uint32_t col_waves;   // waves of a workgroup side by side over columns: 1, 2 or 4
    int4* plan;           // [0]: x sequences are in parts; [1 + i]: the ith of them, its parts, their first state
    float* part_acc;      // [state][item][column tile][D/16][lane][4]; item: column group, kv head
    float* part_ml;       // [state][item][column tile][16][2]: reference point (log2 units), sum
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
__device__ __forceinline__ TreeSpan make_span(const TreeParams& p, int start, int len) {
    const int cap = (int)min((uint64_t)p.max_blocks * p.block_tokens, (uint64_t)0x7fffff00u);
    TreeSpan s;
    s.start = min(max(start, 0), cap);
    s.len = min(max(len, 0), (int)p.nodes);
    s.end = min(s.start + s.len, cap);
    return s;
}
__device__ __forceinline__ TreeSpan tree_span(const TreeParams& p, uint32_t b) {
    const TreeSpan s = make_span(p, as_const(p.start_pos)[b], p.tree_lens ? as_const(p.tree_lens)[b] : (int)p.nodes);
    return {uniform(s.start), uniform(s.len), uniform(s.end)};
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
// node's on.
struct TreeSteps {
    int tiles, prefix_tiles, prefix_steps, steps;
};
template <int NT>
__device__ __forceinline__ TreeSteps tree_steps(const TreeSpan& s) {
    TreeSteps r;
    r.tiles = s.len ? (s.end + kTile - 1) / kTile : 0;  // (no nodes: nothing to read)
    r.prefix_tiles = min(s.start / kTile, r.tiles);
    r.prefix_steps = (r.prefix_tiles + NT - 1) / NT;
    r.steps = r.prefix_steps + (r.tiles - r.prefix_tiles + NT - 1) / NT;
    return r;
}

// Inclusive prefix sums over the wave.
__device__ __forceinline__ int wave_scan(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr 1, 2, 4, 8
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast 15, 31
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);
    return x;
}

// What a row of the grid does: steps [lo, hi) of sequence b (< 0: nothing).
//
// The lengths are on the device, so the rows are dealt out there, by every wave for itself.  With `units` the steps
// of a sequence in units of `unit`, sequence b gets ceil(units_b / c) rows: c is the mean load of a row that the
// card holds, or, where there are fewer sequences than those, the least c (or one near it) that gives no more rows
// than that, so that the longest row is about as short as it can be.  A division by the longest sequence alone
// took 159 us where this takes 103 (13 sequences of up to 9000 tokens, 27 nodes).
constexpr uint32_t kMaxSlotRows = 256;  // and parts of a sequence
constexpr int kPlanGroups = 4;
constexpr uint32_t kPlanSequences = 64 * kPlanGroups;
struct TreeJob {
    int b, lo, hi;
    int part, count;  // of the sequence's parts
    int state;        // of its first part, where count > 1
    int split;        // sequences before it that are in parts
    TreeSpan span;
};
template <int NT>
__device__ __forceinline__ TreeJob tree_job(const TreeParams& p, int row, int unit) {
    TreeJob r;
    r.b = row;
    r.part = 0;
    r.count = 1;
    r.state = 0;
    r.split = 0;
    r.lo = 0;
    if (p.slot_rows == 0) {
        r.span = tree_span(p, (uint32_t)row);
        r.hi = tree_steps<NT>(r.span).steps;
        return r;
    }
    const int lane = threadIdx.x & 63, batch = (int)p.batch;
    int units[kPlanGroups], steps[kPlanGroups];
    TreeSpan span[kPlanGroups];
    int sum = 0;
#pragma unroll
    for (int k = 0; k < kPlanGroups; ++k) {
        units[k] = 0;
        if (64 * k < batch) {
            const int b = 64 * k + lane, from = min(b, batch - 1);
            span[k] = make_span(p, p.start_pos[from], p.tree_lens ? p.tree_lens[from] : (int)p.nodes);
            steps[k] = tree_steps<NT>(span[k]).steps;
            units[k] = b < batch ? max(1, (steps[k] + unit - 1) / unit) : 0;
            sum += units[k];
        }
    }
    auto parts = [&](const int k, const int c) -> int { return (int)((uint32_t)(units[k] + c - 1) / (uint32_t)c); };
    auto rows_of = [&](const int c) -> int {
        int x = 0;
#pragma unroll
        for (int k = 0; k < kPlanGroups; ++k) {
            if (64 * k < batch) x += parts(k, c);
        }
        return __builtin_amdgcn_readlane(wave_scan(x), 63);
    };
    const int total = __builtin_amdgcn_readlane(wave_scan(sum), 63), most = (int)p.rows;
    auto up = [](const int x, const int by) -> int { return uniform((x + by - 1) / by); };
    int c = max((int)p.min_units, up(total, (int)p.slot_rows));
    if (rows_of(c) > most) {
        int hi = most > batch ? max(c + 1, up(total, most - batch)) : total;  // that many are enough
        while (c + 1 < hi) {
            const int mid = c + (hi - c) / 2;
            if (rows_of(mid) > most) c = mid;
            else hi = mid;
        }
        c = hi;
    }
    int base = 0, state = 0, split = 0;
    r.b = -1;
#pragma unroll
    for (int k = 0; k < kPlanGroups; ++k) {
        if (64 * k >= batch) continue;
        const int mine = parts(k, c), held = mine > 1 ? mine : 0;
        const int rows = wave_scan(mine), states = wave_scan(held);
        const int l = (int)__builtin_popcountll(__builtin_amdgcn_ballot_w64(base + rows <= row));
        const uint64_t in_parts = __builtin_amdgcn_ballot_w64(mine > 1);
        if (l < 64 && r.b < 0) {
            const int n = __builtin_amdgcn_readlane(mine, l), u = __builtin_amdgcn_readlane(units[k], l), all = __builtin_amdgcn_readlane(steps[k], l);
            const int even = up(u, n);  // no part much longer than another
            r.count = up(u, even);
            r.part = row - (base + __builtin_amdgcn_readlane(rows, l) - n);
            r.b = r.part < r.count ? 64 * k + l : batch;  // (batch: a row too many)
            r.state = state + __builtin_amdgcn_readlane(states, l) - (n > 1 ? n : 0);
            r.split = split + (int)__builtin_popcountll(in_parts & ((1ull << l) - 1));
            r.lo = r.part * even * unit;
            r.hi = min(r.lo + even * unit, all);
            r.span = {__builtin_amdgcn_readlane(span[k].start, l), __builtin_amdgcn_readlane(span[k].len, l), __builtin_amdgcn_readlane(span[k].end, l)};
        }
        base += __builtin_amdgcn_readlane(rows, 63);
        state += __builtin_amdgcn_readlane(states, 63);
        split += (int)__builtin_popcountll(in_parts);
    }
    if (r.b >= batch) r.b = -1;
    if (blockIdx.x == 0 && threadIdx.x == 0) {  // for tree_merge
        if (row == 0) p.plan[0].x = split;
        if (r.b >= 0 && r.part == 0 && r.count > 1) p.plan[1 + r.split] = make_int4(r.b, r.count, r.state, 0);
    }
    r.b = uniform(r.b);
    r.lo = uniform(r.lo), r.hi = uniform(r.hi);
    r.part = uniform(r.part), r.count = uniform(r.count), r.state = uniform(r.state);
    r.span = {uniform(r.span.start), uniform(r.span.len), uniform(r.span.end)};
    return r;
}

// A scalar of its own.  Arguments are loaded eight or sixteen registers at a time, and short of scalar
// registers the compiler keeps and restores such a tuple whole for one of its members (measured: 16 lane reads
// for each).
template <typename T>
__device__ __forceinline__ T own_scalar(T x) {
    T y;
    asm volatile("s_mov_b32 %0, %1" : "=s"(y) : "s"(x));
    return y;
}
template <typename T>
__device__ __forceinline__ T* own_scalar(T* x) {
    uint64_t y;
    asm volatile("s_mov_b64 %0, %1" : "=s"(y) : "s"(x));
    return (T*)(__attribute__((address_space(1))) T*)y;  // (device memory: a pointer of unknown origin is read by flat loads, which also wait for LDS)
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
// Workgroups of tree_mfma.hip that a CU holds.  Two hide each other's waits, and 256 registers a lane then hold K, V,
// q and the output, but for up to 39 (int4, two tiles of f16 rows: 64 x 4097 tokens, 8 nodes 187 us with one workgroup,
// 157 with two).  Two tiles of f32 rows would spill 68 and 90 (f16 and int4, 16 x 2049: 36 and 38 us with one, 50 and
// 57 with two).
constexpr int tree_cu_groups(int dtype, int d, bool f32_rows, int ct) {
    return ct == 1 || d == 64 || dtype == VSPEC_KV_F32 || !f32_rows ? 2 : 1;
}

}  // namespace vkv
