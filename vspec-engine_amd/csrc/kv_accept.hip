// kv_accept.hip -- keep the accepted path of a drafted tree (vspec_rocm_kv_accept): rows move
// between slots of one sequence, in the pools of all layers.
//
// Sources and destinations of a sequence overlap, so every row is read before any is written.
// Rows move unit by unit: a unit is a column of all rows (16 bytes of K, of V in f32 pools; the
// scattered elements of V in f16 and int4 tiles, kv_common.h; one scale), and units are
// independent of each other.  A workgroup holds one (layer, sequence, kv head) and K or V; its
// threads take (row, unit) pairs, kBatch of them in registers between two barriers.
#include "host.h"
#include "kv_common.h"

namespace vkv {
namespace {

constexpr uint32_t kLayers = 32;  // pools of one launch: their addresses are kernel arguments
constexpr uint32_t kNodes = 64;

struct AcceptPool {
    uint8_t* k;
    uint8_t* v;
    uint16_t* ks;
    uint16_t* vs;
    uint32_t* kf;
};

struct AcceptParams {
    AcceptPool pools[kLayers];
    const int32_t* block_tables;
    const int32_t* start_pos;
    const int32_t* path;
    int32_t* new_lens;  // or null
    uint32_t max_blocks, max_path, num_nodes;
    uint32_t hkv, head_dim, block_tokens, num_blocks;
};

// Where slot `pos` of sequence b lies: its (block, head) index and the slot in the block.
__device__ __forceinline__ bool accept_slot(const AcceptParams& p, uint32_t b, int64_t pos, uint32_t h, size_t* bh,
                                            uint32_t* slot) {
    if (pos < 0 || pos >= (int64_t)p.max_blocks * p.block_tokens) return false;
    const int entry = p.block_tables[(size_t)b * p.max_blocks + (uint32_t)(pos / p.block_tokens)];
    if (entry < 0 || (uint32_t)entry >= p.num_blocks) return false;
    *bh = (size_t)entry * p.hkv + h;
    *slot = (uint32_t)(pos % p.block_tokens);
    return true;
}

template <int DT>
__global__ __launch_bounds__(256) void kv_accept(AcceptParams p) {
    const uint32_t h = blockIdx.x, b = blockIdx.y;
    const bool isv = blockIdx.z & 1u;
    const AcceptPool& pool = p.pools[blockIdx.z >> 1];
    const uint32_t lane = threadIdx.x & 63u;
    // the path's length: lanes before the first entry that names no node
    const int32_t node_l = lane < p.max_path ? p.path[(size_t)b * p.max_path + lane] : -1;
    const uint64_t ends = __builtin_amdgcn_ballot_w64(node_l < 0 || (uint32_t)node_l >= p.num_nodes);
    const uint32_t count = ends ? (uint32_t)__builtin_ctzll(ends) : 64u;
    const int64_t start = max(p.start_pos[b], 0);
    if (h == 0 && blockIdx.z == 0 && threadIdx.x == 0 && p.new_lens) p.new_lens[b] = (int32_t)(start + count);

    // row `lane` of the path
    __shared__ size_t from_bh[kNodes], to_bh[kNodes];
    __shared__ uint32_t from_slot[kNodes], to_slot[kNodes];
    __shared__ bool moves[kNodes];
    if (threadIdx.x < 64) {
        size_t fb = 0, tb = 0;
        uint32_t fs = 0, ts = 0;
        bool ok = lane < count && node_l != (int32_t)lane;
        ok = ok && accept_slot(p, b, start + node_l, h, &fb, &fs);
        ok = ok && accept_slot(p, b, start + lane, h, &tb, &ts);
        from_bh[lane] = fb;
        to_bh[lane] = tb;
        from_slot[lane] = fs;
        to_slot[lane] = ts;
        moves[lane] = ok;
    }
    __syncthreads();
    const uint32_t D = p.head_dim, P = p.block_tokens, G = D / 32;

    // unit u of a row: read(bh, slot, u) and write(bh, slot, u, x)
    auto move = [&](const uint32_t units, auto read, auto write) {
        typedef decltype(read((size_t)0, 0u, 0u)) T;
        constexpr int kBatch = 4;
        const uint32_t wide = (256u / kNodes) * kBatch;  // units between two barriers
        const uint32_t row = threadIdx.x % kNodes, u0 = threadIdx.x / kNodes;
        const bool mine = moves[row];
        for (uint32_t base = 0; base < units; base += wide) {
            T x[kBatch];
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                const uint32_t u = base + u0 + i * (256u / kNodes);
                if (mine && u < units) x[i] = read(from_bh[row], from_slot[row], u);
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                const uint32_t u = base + u0 + i * (256u / kNodes);
                if (mine && u < units) write(to_bh[row], to_slot[row], u, x[i]);
            }
        }
    };

    if constexpr (DT == VSPEC_KV_INT4) {
        if (!isv) {
            const uint32_t rb = D / 2;
            move(rb / 16, [&](size_t bh, uint32_t s, uint32_t u) { return reinterpret_cast<const uint4*>(pool.k + (bh * P + s) * rb)[u]; },
                 [&](size_t bh, uint32_t s, uint32_t u, uint4 x) { reinterpret_cast<uint4*>(pool.k + (bh * P + s) * rb)[u] = x; });
            move(G, [&](size_t bh, uint32_t s, uint32_t u) { return pool.ks[int4_ks_index(bh, G, P, s, u)]; },
                 [&](size_t bh, uint32_t s, uint32_t u, uint16_t x) { pool.ks[int4_ks_index(bh, G, P, s, u)] = x; });
            if (pool.kf) {
                // one bit a row: words are shared between rows, and no other workgroup's
                auto word = [&](size_t bh, uint32_t s) { return pool.kf + bh * (P / 16) + s / 16; };
                uint32_t bit = 0;
                const bool mine = threadIdx.x < 64 && moves[lane];
                if (mine) bit = *word(from_bh[lane], from_slot[lane]) >> (from_slot[lane] % 16) & 1u;
                __syncthreads();
                if (mine) {
                    const uint32_t m = 1u << (to_slot[lane] % 16);
                    if (bit) atomicOr(word(to_bh[lane], to_slot[lane]), m);
                    else atomicAnd(word(to_bh[lane], to_slot[lane]), ~m);
                }
            }
        } else {
            // byte u: a token's codes of two elements
            auto at = [&](size_t bh, uint32_t s, uint32_t u) {
                uint32_t high;
                return pool.v + int4_v_byte(bh, P, D, s, 32u * (u / 16) + u % 16, &high);
            };
            move(D / 2, [&](size_t bh, uint32_t s, uint32_t u) { return *at(bh, s, u); },
                 [&](size_t bh, uint32_t s, uint32_t u, uint8_t x) { *at(bh, s, u) = x; });
            move(G, [&](size_t bh, uint32_t s, uint32_t u) { return pool.vs[(bh * P + s) * G + u]; },
                 [&](size_t bh, uint32_t s, uint32_t u, uint16_t x) { pool.vs[(bh * P + s) * G + u] = x; });
        }
    } else if (DT == VSPEC_KV_F16 && isv) {
        uint16_t* v = reinterpret_cast<uint16_t*>(pool.v);
        move(D, [&](size_t bh, uint32_t s, uint32_t u) { return v[f16_v_index(bh, P, D, s, u)]; },
             [&](size_t bh, uint32_t s, uint32_t u, uint16_t x) { v[f16_v_index(bh, P, D, s, u)] = x; });
    } else {
        const uint32_t rb = D * (DT == VSPEC_KV_F32 ? 4u : 2u);
        uint8_t* base = isv ? pool.v : pool.k;
        move(rb / 16, [&](size_t bh, uint32_t s, uint32_t u) { return reinterpret_cast<const uint4*>(base + (bh * P + s) * rb)[u]; },
             [&](size_t bh, uint32_t s, uint32_t u, uint4 x) { reinterpret_cast<uint4*>(base + (bh * P + s) * rb)[u] = x; });
    }
}

}  // namespace
}  // namespace vkv

using namespace vkv;

extern "C" int vspec_rocm_kv_accept(const VspecPagedKV* kvs, uint32_t num_kvs, uint32_t batch, const int32_t* block_tables,
                                    uint32_t max_blocks_per_seq, const int32_t* start_pos, const int32_t* path,
                                    uint32_t max_path, uint32_t num_nodes, int32_t* new_lens, void* stream) {
    if (!kvs || num_kvs == 0) {
        host_error("kv_accept: no pools");
        return 0;
    }
    for (uint32_t i = 0; i < num_kvs; ++i) {
        if (!host_check_kv(kvs + i, "kv_accept", false)) return 0;
        if (kvs[i].dtype != kvs[0].dtype || kvs[i].num_blocks != kvs[0].num_blocks ||
            kvs[i].block_tokens != kvs[0].block_tokens || kvs[i].num_kv_heads != kvs[0].num_kv_heads ||
            kvs[i].head_dim != kvs[0].head_dim) {
            host_error("kv_accept: pool %u differs from the first in dtype or geometry", i);
            return 0;
        }
        for (uint32_t j = 0; j < i; ++j) {
            if (kvs[j].k_data == kvs[i].k_data || kvs[j].v_data == kvs[i].v_data) {
                host_error("kv_accept: pools %u and %u are the same", j, i);
                return 0;
            }
        }
        if (((uintptr_t)kvs[i].k_data | (uintptr_t)kvs[i].v_data) % 16 != 0) {
            host_error("kv_accept: pool %u is not 16-byte aligned", i);
            return 0;
        }
    }
    if (num_nodes == 0 || num_nodes > kNodes || max_path > kNodes) {
        host_error("kv_accept: num_nodes must be 1..%u and max_path at most %u", kNodes, kNodes);
        return 0;
    }
    if (batch > 65535u) {
        host_error("kv_accept: batch above 65535");
        return 0;
    }
    if (batch == 0) return 1;
    if (!block_tables || !start_pos || (!path && max_path) || max_blocks_per_seq == 0) {
        host_error("kv_accept: null argument");
        return 0;
    }
    AcceptParams p = {};
    p.block_tables = block_tables;
    p.start_pos = start_pos;
    p.path = path;
    p.max_blocks = max_blocks_per_seq;
    p.max_path = max_path;
    p.num_nodes = num_nodes;
    p.hkv = kvs[0].num_kv_heads;
    p.head_dim = kvs[0].head_dim;
    p.block_tokens = kvs[0].block_tokens;
    p.num_blocks = kvs[0].num_blocks;
    hipStream_t s = (hipStream_t)stream;
    for (uint32_t at = 0; at < num_kvs; at += kLayers) {
        const uint32_t n = num_kvs - at < kLayers ? num_kvs - at : kLayers;
        for (uint32_t i = 0; i < n; ++i) {
            const VspecPagedKV& kv = kvs[at + i];
            p.pools[i] = {(uint8_t*)kv.k_data, (uint8_t*)kv.v_data, kv.k_scales, kv.v_scales,
                          kv.dtype == VSPEC_KV_INT4 ? kv.k_flags : nullptr};
        }
        p.new_lens = at == 0 ? new_lens : nullptr;
        const dim3 grid(p.hkv, batch, 2 * n);
        switch (kvs[0].dtype) {
            case VSPEC_KV_F32: hipLaunchKernelGGL((kv_accept<VSPEC_KV_F32>), grid, dim3(256), 0, s, p); break;
            case VSPEC_KV_F16: hipLaunchKernelGGL((kv_accept<VSPEC_KV_F16>), grid, dim3(256), 0, s, p); break;
            default: hipLaunchKernelGGL((kv_accept<VSPEC_KV_INT4>), grid, dim3(256), 0, s, p); break;
        }
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) {
        host_error("kv_accept launch: %s", hipGetErrorString(e));
        return 0;
    }
    return 1;
}
