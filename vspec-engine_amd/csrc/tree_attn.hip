// tree_attn.hip -- attention of a tree of drafted tokens over the paged cache
// (vspec_rocm_paged_tree_attention): every node of a sequence sees the cached prefix and the
// nodes that its mask names, in one pass over the sequence's tokens.
#include <math.h>

#include "host.h"
#include "tree_attn.h"

namespace vkv {
namespace {

// Element e of the key or value row in `slot` of (block, head) bh.
template <int DT, int D>
__device__ __forceinline__ float key_at(const TreeParams& p, size_t bh, uint32_t slot, uint32_t e) {
    const uint32_t P = p.block_tokens;
    const size_t row = bh * P + slot;
    if constexpr (DT == VSPEC_KV_F32) return reinterpret_cast<const float*>(p.k)[row * D + e];
    if constexpr (DT == VSPEC_KV_F16) return half_bits_to_float(reinterpret_cast<const uint16_t*>(p.k)[row * D + e]);
    return nibble((uint32_t)p.k[row * (D / 2) + e / 2], (int)(e & 1u)) *
           half_bits_to_float(p.ks[int4_ks_index(bh, D / 32, P, slot, e / 32)]);
}
template <int DT, int D>
__device__ __forceinline__ float value_at(const TreeParams& p, size_t bh, uint32_t slot, uint32_t e) {
    const uint32_t P = p.block_tokens;
    if constexpr (DT == VSPEC_KV_F32) return reinterpret_cast<const float*>(p.v)[(bh * P + slot) * D + e];
    if constexpr (DT == VSPEC_KV_F16) return half_bits_to_float(reinterpret_cast<const uint16_t*>(p.v)[f16_v_index(bh, P, D, slot, e)]);
    uint32_t high;
    const uint8_t c = p.v[int4_v_byte(bh, P, D, slot, e, &high)];
    return nibble((uint32_t)c, (int)high) * half_bits_to_float(p.vs[(bh * P + slot) * (D / 32) + e / 32]);
}

// One wave for each (node, query head, sequence): 64 tokens at a time, a lane each for the
// scores, then D / 64 elements of the output a lane.
template <int DT, int D, typename IO>
__global__ __launch_bounds__(64) void tree_rows(TreeParams p) {
    __shared__ float q[D];
    __shared__ float pr[64];
    __shared__ size_t bhs[64];
    const uint32_t i = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
    const int lane = threadIdx.x;
    constexpr int E = D / 64;
    const TreeSpan sp = tree_span(p, b);
    const size_t row = (((size_t)b * p.nodes + i) * p.hq + h) * D;
    const uint64_t bits = tree_bits(p, b, (int)i, sp.len);
    IO* out = reinterpret_cast<IO*>(p.out) + row;

    float x[E], sum = 0.f, var = 0.f;
    for (int e = 0; e < E; ++e) {
        x[e] = (float)(reinterpret_cast<const IO*>(p.q) + row)[lane + 64 * e];
        sum += x[e];
    }
    const float mean = wave_sum(sum) * (1.0f / D);
    for (int e = 0; e < E; ++e) var = fmaf(x[e] - mean, x[e] - mean, var);
    const float th = fminf(fmaxf(1e-6f, p.alpha * sqrtf(wave_sum(var) * (1.0f / D))), p.input_clip);
    for (int e = 0; e < E; ++e) q[lane + 64 * e] = fminf(fmaxf(x[e], -th), th) * p.scale;
    __syncthreads();

    float m = -INFINITY, l = 0.f, acc[E] = {};
    const int end = (int)i < sp.len ? sp.end : 0;
    for (int t0 = 0; t0 < end; t0 += 64) {
        const int t = t0 + lane;
        bool sees = t < end && (t < sp.start || (bits >> (t - sp.start) & 1));
        float s = -INFINITY;
        if (sees) {
            const size_t at = (size_t)b * p.max_blocks + t / p.block_tokens;
            const uint32_t slot = (uint32_t)t % p.block_tokens;
            const int entry = p.block_tables[at];
            sees = entry >= 0 && (uint32_t)entry < p.num_blocks && (!p.block_used || (int)slot < p.block_used[at]);
            if (sees) {
                const size_t bh = (size_t)entry * p.hkv + h / p.group;
                bhs[lane] = bh;
                float sm = 0.f, v2 = 0.f, dot = 0.f;
                for (uint32_t e = 0; e < D; ++e) sm += key_at<DT, D>(p, bh, slot, e);
                sm *= 1.0f / D;
                for (uint32_t e = 0; e < D; ++e) {
                    const float y = key_at<DT, D>(p, bh, slot, e) - sm;
                    v2 = fmaf(y, y, v2);
                }
                const float kth = fminf(fmaxf(1e-6f, p.alpha * sqrtf(v2 * (1.0f / D))), p.input_clip);
                for (uint32_t e = 0; e < D; ++e) dot = fmaf(q[e], fminf(fmaxf(key_at<DT, D>(p, bh, slot, e), -kth), kth), dot);
                s = fminf(fmaxf(dot, -p.logit_clip), p.logit_clip);
            }
        }
        const float mt = fmaxf(m, wave_max(s));
        const float base = mt == -INFINITY ? 0.f : mt;
        const float f = exp2f(m - base);
        m = mt;
        const float w = exp2f(s - base);
        l = l * f + wave_sum(w);
        pr[lane] = sees ? w : -1.f;
        __syncthreads();
        for (int e = 0; e < E; ++e) acc[e] *= f;
        for (int n = 0; n < 64; ++n) {
            if (pr[n] < 0.f) continue;
            for (int e = 0; e < E; ++e) {
                acc[e] = fmaf(pr[n], value_at<DT, D>(p, bhs[n], (uint32_t)(t0 + n) % p.block_tokens, lane + 64 * e), acc[e]);
            }
        }
        __syncthreads();
    }
    for (int e = 0; e < E; ++e) out[lane + 64 * e] = (IO)(m == -INFINITY ? 0.f : acc[e] / l);
}

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

template <int DT, int D>
void launch_rows(const TreeParams& p, int32_t io, hipStream_t s) {
    const dim3 grid(p.nodes, p.hq, p.batch);
    if (io == VSPEC_KV_F32) hipLaunchKernelGGL((tree_rows<DT, D, float>), grid, dim3(64), 0, s, p);
    else hipLaunchKernelGGL((tree_rows<DT, D, _Float16>), grid, dim3(64), 0, s, p);
}

}  // namespace
}  // namespace vkv

using namespace vkv;

extern "C" size_t vspec_rocm_paged_tree_attention_workspace_bytes(const VspecTreeAttnDesc* desc) {
    if (!check_tree(desc)) return 0;
    return 0;
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
    p.scale = scale * kLog2e;
    p.alpha = desc->clamp_alpha > 0.f ? desc->clamp_alpha : 4.5f;
    p.logit_clip = three ? 24.0f * kLog2e : INFINITY;
    p.input_clip = three ? 16.0f : INFINITY;
    hipStream_t s = (hipStream_t)desc->stream;
    const bool wide = kv.head_dim == 128;
    switch (kv.dtype) {
        case VSPEC_KV_F32: wide ? launch_rows<VSPEC_KV_F32, 128>(p, desc->io_dtype, s) : launch_rows<VSPEC_KV_F32, 64>(p, desc->io_dtype, s); break;
        case VSPEC_KV_F16: wide ? launch_rows<VSPEC_KV_F16, 128>(p, desc->io_dtype, s) : launch_rows<VSPEC_KV_F16, 64>(p, desc->io_dtype, s); break;
        default: wide ? launch_rows<VSPEC_KV_INT4, 128>(p, desc->io_dtype, s) : launch_rows<VSPEC_KV_INT4, 64>(p, desc->io_dtype, s); break;
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) {
        host_error("tree attention launch: %s", hipGetErrorString(e));
        return 0;
    }
    return 1;
}
