// tree_attn.hip -- vspec_rocm_paged_tree_attention: its checks, its plan and its launches (the
// kernels: tree_mfma.hip, tree_wide.hip).
#include <math.h>

#include "host.h"
#include "tree_attn.h"

namespace vkv {
namespace {

int check_tree(const VspecTreeAttnDesc* d) {
    if (!d) {
        host_error("paged_tree_attention: null descriptor");
        return 0;
    }
    if (!host_check_kv(&d->kv, "paged_tree_attention", true)) return 0;
    if (d->num_nodes == 0 || d->num_nodes > 64) {
        host_error("paged_tree_attention: num_nodes must be 1..64");
        return 0;
    }
    if (d->num_q_heads == 0 || d->num_q_heads % d->kv.num_kv_heads != 0) {
        host_error("paged_tree_attention: num_q_heads must be a positive multiple of num_kv_heads");
        return 0;
    }
    if (d->io_dtype != VSPEC_KV_F32 && d->io_dtype != VSPEC_KV_F16) {
        host_error("paged_tree_attention: io_dtype must be f32 or f16");
        return 0;
    }
    if (d->numerics != VSPEC_NUMERICS_PLAIN && d->numerics != VSPEC_NUMERICS_3BIT) {
        host_error("paged_tree_attention: bad numerics mode");
        return 0;
    }
    if (d->batch > 65535u || d->num_q_heads > 65535u) {
        host_error("paged_tree_attention: batch and num_q_heads at most 65535");
        return 0;
    }
    const uint64_t cap = (uint64_t)d->max_blocks_per_seq * d->kv.block_tokens;
    if (cap > 0x7fffff00ull) {
        host_error("paged_tree_attention: block table beyond 2^31 tokens");
        return 0;
    }
    if (d->max_start_pos > cap) {
        host_error("paged_tree_attention: max_start_pos exceeds the block table");
        return 0;
    }
    return 1;
}

struct TreePlan {
    uint32_t ct, col_waves, col_groups, rows, slot_rows, min_units;
    bool wide;  // tree_wide.hip
    size_t plan_bytes, acc_floats, ws_bytes;
};

// Columns first: a workgroup holds as many as K and V can be read once for.  Then rows of the grid
// (tree_job): sequences, and parts of them where that shortens the longest row.
TreePlan plan_tree(const VspecTreeAttnDesc* d) {
    TreePlan pl = {};
    const uint32_t cols = d->num_nodes * (d->num_q_heads / d->kv.num_kv_heads);
    const uint32_t tiles = (cols + 15) / 16;
    // Up to two column tiles a wave keeps to itself (tree_mfma.hip); of more, waves share K and V through LDS
    // (tree_wide.hip).  At 8 nodes of 4 heads, two tiles: 16 x 2049 tokens of an f16 pool 45 and 51 us, 64 x 4097 of
    // an int4 pool 186 and 246; at 16 nodes, four tiles, the first kernel took 136 us where the second takes 49.
    // f32 pools stay with the first: an exact clip of every key and f32 products, no operands
    // in f16 to share.
    pl.wide = d->kv.dtype != VSPEC_KV_F32 && tiles > 2;
    const uint64_t cap = (uint64_t)d->max_blocks_per_seq * d->kv.block_tokens;
    uint64_t bound = (d->max_start_pos ? d->max_start_pos : cap) + d->num_nodes;
    if (bound > cap) bound = cap;
    if (pl.wide) {
        pl.ct = tiles <= 4 ? 1 : 2;  // the least that holds them: a wave without columns reads and waits all the same
        pl.col_waves = tiles <= 8 ? 4 : 8;
    } else {
        // Two tiles to a wave read K and V once, which counts where they are long (64 x 4097 tokens, 8 nodes: f16 208 us,
        // int4 177; by two waves side by side 245 and 226); two waves have less to do in a row each, which counts where
        // a CU gets few tokens (one sequence of 700, 5 nodes: 11 us and 10, by one wave 13 and 12.6; 16 x 500, 250 tokens
        // a CU: 21.6 and 20.7).
        const bool beside = tiles == 2 && bound * d->batch * d->kv.num_kv_heads <= 128ull * host_num_cus();
        pl.ct = tiles == 1 || beside ? 1 : 2;
        pl.col_waves = (tiles + pl.ct - 1) / pl.ct > 2 ? 4 : (tiles + pl.ct - 1) / pl.ct;
    }
    pl.col_groups = (tiles + pl.ct * pl.col_waves - 1) / (pl.ct * pl.col_waves);
    const bool f32_rows = d->io_dtype == VSPEC_KV_F32;
    // a unit: a step, or one of each of the waves that share a row's steps
    const uint32_t per = 16 * (pl.wide ? wide_step_tiles(f32_rows, pl.ct) : tree_step_tiles(d->kv.dtype) * (4 / pl.col_waves));
    // (of 1 and 2 without sharing: one sequence of 700 tokens 13.3 and 14.6 us, 16 of 500 17.6 and 15.9)
    pl.min_units = pl.wide ? 4 : 1;
    const uint64_t batch = d->batch, units = (bound + per - 1) / per;
    const uint64_t items = (uint64_t)d->kv.num_kv_heads * pl.col_groups;
    const uint64_t wgs = (uint64_t)host_num_cus() * (pl.wide ? (pl.col_waves == 8 ? 1 : 2) : tree_cu_groups(d->kv.dtype, d->kv.head_dim, f32_rows, pl.ct));
    uint64_t slots = wgs / items ? wgs / items : 1;
    if (slots > kMaxSlotRows) slots = kMaxSlotRows;
    uint64_t rows = slots > batch ? slots : slots + batch;
    const uint64_t most = batch * ((units + pl.min_units - 1) / pl.min_units);
    if (rows > most) rows = most;
    pl.rows = (uint32_t)batch;
    if (rows > batch && batch <= kPlanSequences && batch * (cap / per + 2) < 1u << 30) {
        pl.rows = (uint32_t)rows;
        pl.slot_rows = (uint32_t)slots;
        // parts of sequences that have more than one: at most a row's mean load each, and one more for each sequence
        const uint64_t states = rows < 2 * slots ? rows : 2 * slots;
        const size_t state_tiles = (size_t)(states * items * pl.col_waves * pl.ct);
        pl.plan_bytes = (1 + slots) * sizeof(int4);
        pl.acc_floats = state_tiles * d->kv.head_dim * 16;
        pl.ws_bytes = pl.plan_bytes + (pl.acc_floats + state_tiles * 32) * sizeof(float);
    }
    return pl;
}

}  // namespace
}  // namespace vkv

using namespace vkv;

extern "C" size_t vspec_rocm_paged_tree_attention_workspace_bytes(const VspecTreeAttnDesc* desc) {
    if (!check_tree(desc)) return 0;
    return plan_tree(desc).ws_bytes;
}

extern "C" int vspec_rocm_paged_tree_attention(const VspecTreeAttnDesc* desc) {
    if (!check_tree(desc)) return 0;
    if (desc->batch == 0) return 1;
    if (!desc->block_tables || !desc->start_pos || !desc->q || !desc->out || desc->max_blocks_per_seq == 0) {
        host_error("paged_tree_attention: null argument");
        return 0;
    }
    if (((uintptr_t)desc->q | (uintptr_t)desc->out) % 16 != 0) {
        host_error("paged_tree_attention: q and out must be 16-byte aligned");
        return 0;
    }
    const VspecPagedKV& kv = desc->kv;
    float scale = desc->scale > 0.f ? desc->scale : 1.0f / sqrtf((float)kv.head_dim);
    const bool three = desc->numerics == VSPEC_NUMERICS_3BIT;
    if (three) scale = fminf(fmaxf(scale, 1e-4f), 32.0f);
    TreeParams p = {};
    p.k = (const uint8_t*)kv.k_data;
    p.v = (const uint8_t*)kv.v_data;
    p.ks = kv.k_scales;
    p.vs = kv.v_scales;
    p.block_tables = desc->block_tables;
    p.block_used = desc->block_used;
    p.start_pos = desc->start_pos;
    p.tree_lens = desc->tree_lens;
    p.tree_mask = desc->tree_mask;
    p.q = desc->q;
    p.out = desc->out;
    p.batch = desc->batch;
    p.nodes = desc->num_nodes;
    p.hq = desc->num_q_heads;
    p.hkv = kv.num_kv_heads;
    p.group = p.hq / p.hkv;
    p.block_tokens = kv.block_tokens;
    p.max_blocks = desc->max_blocks_per_seq;
    p.num_blocks = kv.num_blocks;
    const uint32_t block_tiles = kv.block_tokens / kTile;
    while ((1u << p.block_shift) < block_tiles) ++p.block_shift;
    p.block_magic = (uint32_t)((((1ull << (27 + p.block_shift)) + block_tiles - 1) / block_tiles) << 4);
    p.scale = scale * kLog2e;
    p.alpha = desc->clamp_alpha > 0.f ? desc->clamp_alpha : 4.5f;
    p.logit_clip = three ? 24.0f * kLog2e : INFINITY;
    p.input_clip = three ? 16.0f : INFINITY;
    const TreePlan pl = plan_tree(desc);
    void* ws = nullptr;
    if (pl.ws_bytes) {
        if (desc->workspace) {
            if (desc->workspace_bytes < pl.ws_bytes || (uintptr_t)desc->workspace % 16 != 0) {
                host_error("paged_tree_attention: workspace too small (%zu < %zu) or not 16-byte aligned", desc->workspace_bytes, pl.ws_bytes);
                return 0;
            }
            ws = desc->workspace;
        } else {
            ws = host_workspace(pl.ws_bytes);
            if (!ws) {
                host_error("paged_tree_attention: cannot allocate %zu workspace bytes", pl.ws_bytes);
                return 0;
            }
        }
    }
    p.rows = pl.rows;
    p.slot_rows = pl.slot_rows;
    p.min_units = pl.min_units;
    p.col_groups = pl.col_groups;
    p.col_waves = pl.col_waves;
    p.plan = (int4*)ws;
    p.part_acc = (float*)((uint8_t*)ws + pl.plan_bytes);
    p.part_ml = p.part_acc + pl.acc_floats;
    hipStream_t s = (hipStream_t)desc->stream;
    const bool d128 = kv.head_dim == 128;
    switch (kv.dtype) {
        case VSPEC_KV_F32: (d128 ? launch_tree_f32_d128 : launch_tree_f32_d64)(p, desc->io_dtype, pl.ct, s); break;
        case VSPEC_KV_F16:
            if (pl.wide) (d128 ? launch_tree_wide_f16_d128 : launch_tree_wide_f16_d64)(p, desc->io_dtype, pl.ct, s);
            else (d128 ? launch_tree_f16_d128 : launch_tree_f16_d64)(p, desc->io_dtype, pl.ct, s);
            break;
        default:
            if (pl.wide) (d128 ? launch_tree_wide_int4_d128 : launch_tree_wide_int4_d64)(p, desc->io_dtype, pl.ct, s);
            else (d128 ? launch_tree_int4_d128 : launch_tree_int4_d64)(p, desc->io_dtype, pl.ct, s);
            break;
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) {
        host_error("tree attention launch: %s", hipGetErrorString(e));
        return 0;
    }
    return 1;
}
