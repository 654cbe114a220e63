// kv_accept.hip -- keep the accepted path of a drafted tree (vspec_rocm_kv_accept): rows move
// between slots of one sequence, in the pools of all layers.
//
// Sources and destinations of a sequence overlap, so every row is read before any is written.
// Rows move column by column, a column being 16 bytes of every row, and columns are independent
// of each other:
//   K, and V of f32 pools       16 bytes of a token's row
//   V of f16 and int4 pools     16 bytes of a group of 4 tokens, which hold a part of each
//                               (kv_common.h): a destination group is put together from the up to
//                               four groups that its tokens come from and written whole (by
//                               single bytes, 64 x 64 nodes in 16 int4 layers took 71 us)
// A workgroup, one wave, holds one (sequence, kv head) and K or V of some layers; what a row's slots
// are is worked out once for them.  It takes a pass of columns into registers and writes them.
//
// The bytes are few (64 x 64 nodes, 16 int4 layers: 26 MB, 5 us at the rate of a large copy); what
// counts is the chain of waits, path -> table -> row -> write, and how many of them overlap.  So
// workgroups are small and take only as many layers as leave 24 of them to a CU (four waves and
// 8 layers a workgroup: 37 us; this: 22).
#include <type_traits>

#include "host.h"
#include "kv_common.h"

namespace vkv {
namespace {

constexpr uint32_t kLayers = 64;  // pools of one launch: their addresses are kernel arguments
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
    uint32_t layers, share;  // pools of this launch, and of a workgroup
};

// Where slot `pos` of sequence b lies for kv head h: the index of its token, and its slot in the block.
__device__ __forceinline__ bool accept_slot(const AcceptParams& p, uint32_t b, uint32_t pos, uint32_t h, size_t* token, uint32_t* slot) {
    const uint32_t row = pos / p.block_tokens;
    if (row >= p.max_blocks) return false;
    const int entry = p.block_tables[(size_t)b * p.max_blocks + row];
    if (entry < 0 || (uint32_t)entry >= p.num_blocks) return false;
    *slot = pos - row * p.block_tokens;
    *token = ((size_t)entry * p.hkv + h) * p.block_tokens + *slot;
    return true;
}

// 16 bytes of V of a group of 4 tokens: the bits of token r.
template <int DT>
__device__ __forceinline__ uint64_t token_bits(uint64_t w, uint32_t r) {
    if constexpr (DT == VSPEC_KV_F16) return (w >> (16 * r)) & 0xffffull;
    return (w >> (8 * (2 * (r & 1) + (r >> 1)))) & 0x000000ff000000ffull;
}
template <int DT>
__device__ __forceinline__ uint64_t bits_of_token(uint64_t x, uint32_t r) {
    if constexpr (DT == VSPEC_KV_F16) return x << (16 * r);
    return x << (8 * (2 * (r & 1) + (r >> 1)));
}

template <int DT>
__global__ __launch_bounds__(64) void kv_accept(AcceptParams p) {
    constexpr uint32_t kThreads = 64;
    const uint32_t h = blockIdx.x, b = blockIdx.y;
    const bool isv = blockIdx.z & 1u;
    const uint32_t lane = threadIdx.x;
    // the path's length: lanes before the first entry that names no node
    const int32_t node_l = lane < p.max_path ? p.path[(size_t)b * p.max_path + lane] : -1;
    const uint64_t ends = __builtin_amdgcn_ballot_w64(node_l < 0 || (uint32_t)node_l >= p.num_nodes);
    const uint32_t count = ends ? (uint32_t)__builtin_ctzll(ends) : 64u;
    const uint32_t start = (uint32_t)max(p.start_pos[b], 0);
    if (h == 0 && blockIdx.z == 0 && lane == 0 && p.new_lens) p.new_lens[b] = (int32_t)(start + count);

    // row `lane` of the path
    __shared__ size_t from_sh[kNodes], to_sh[kNodes];
    size_t from = 0, to = 0;
    uint32_t fs = 0, ts = 0;
    bool ok = lane < count && node_l != (int32_t)lane;
    ok = ok && accept_slot(p, b, start + node_l, h, &from, &fs);
    ok = ok && accept_slot(p, b, start + lane, h, &to, &ts);
    from_sh[lane] = from;
    to_sh[lane] = to;
    const uint64_t moves = __builtin_amdgcn_ballot_w64(ok);
    if (moves == 0) return;
    __syncthreads();
    const uint32_t D = p.head_dim, P = p.block_tokens, G = D / 32;
    const uint32_t rb = DT == VSPEC_KV_F32 ? 4 * D : DT == VSPEC_KV_F16 ? 2 * D : D / 2;  // bytes of a row
    const uint32_t first = (blockIdx.z >> 1) * p.share, last = min(first + p.share, p.layers);

    // x / d, d <= 4096 and x below 2^20: magic is above 2^32 / d by less than 1
    auto magic_of = [](const uint32_t d) -> uint32_t { return d == 1 ? 0u : 0xffffffffu / d + 1u; };
    auto div = [](const uint32_t x, const uint32_t magic) -> uint32_t { return magic ? __umulhi(x, magic) : x; };
    auto moved = [&](const uint32_t row) -> bool { return row < 64u && (moves >> row) & 1u; };

    // columns of `rows` things, read(row, column) and, if wanted(row), write(row, column, x): up to N a thread and pass
    auto pass = [&](auto batch, const uint32_t rows, const uint32_t columns, auto wanted, auto read, auto write) {
        constexpr int N = decltype(batch)::value;
        typedef decltype(read(0u, 0u)) T;
        const uint32_t most = N * kThreads / rows;
        for (uint32_t c0 = 0; c0 < columns; c0 += most) {
            const uint32_t n = min(most, columns - c0), magic = magic_of(n);
            T x[N];
#pragma unroll
            for (int i = 0; i < N; ++i) {
                // (every lane reads, so that no load waits for the one before it)
                const uint32_t idx = min(lane + kThreads * i, rows * n - 1), row = div(idx, magic);
                if (kThreads * i < rows * n) x[i] = read(row, c0 + idx - row * n);
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const uint32_t idx = lane + kThreads * i, row = div(idx, magic);
                if (row < rows && wanted(row)) write(row, c0 + idx - row * n, x[i]);
            }
        }
    };

    if (DT != VSPEC_KV_F32 && isv) {
        const uint32_t group0 = start / 4, groups = (start + count - 1) / 4 - group0 + 1;  // P is a multiple of 16
        // rows of the path in group i, as bits: token r is row 4 (group0 + i) + r - start
        auto rows_in = [&](const uint32_t i) -> uint32_t {
            const int at = (int)(4 * (group0 + i)) - (int)start;
            return (uint32_t)(at < 0 ? moves << -at : at < 64 ? moves >> at : 0) & 15u;
        };
        for (uint32_t l = first; l < last; ++l) {
            const AcceptPool& pool = p.pools[l];
            uint16_t scale[4] = {0, 0, 0, 0};  // of row `lane`
#pragma unroll
            for (uint32_t c = 0; c < 4; ++c) {
                if (DT == VSPEC_KV_INT4 && ok && c < G) scale[c] = pool.vs[from * G + c];
            }
            pass(std::integral_constant<int, 5>(), groups, rb / 4, [&](uint32_t i) { return rows_in(i) != 0; },
                 [&](uint32_t i, uint32_t u) {
                     const uint32_t in = rows_in(i);
                     const uint32_t any = __builtin_ctz(in | 16u), row0 = 4 * (group0 + i) - start;  // (row0 + r wraps back for r in `in`)
                     const size_t own = in ? to_sh[row0 + any] - any : 0;
                     uint4 w[4];
                     uint32_t r_of[4];
#pragma unroll
                     for (uint32_t r = 0; r < 4; ++r) {
                         const size_t from = (in >> r) & 1u ? from_sh[row0 + r] : own + r;
                         r_of[r] = (uint32_t)from & 3u;
                         w[r] = reinterpret_cast<const uint4*>(pool.v + (from - r_of[r]) * rb)[u];
                     }
                     uint64_t lo = 0, hi = 0;
#pragma unroll
                     for (uint32_t r = 0; r < 4; ++r) {
                         lo |= bits_of_token<DT>(token_bits<DT>((uint64_t)w[r].y << 32 | w[r].x, r_of[r]), r);
                         hi |= bits_of_token<DT>(token_bits<DT>((uint64_t)w[r].w << 32 | w[r].z, r_of[r]), r);
                     }
                     return make_uint4((uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32));
                 },
                 [&](uint32_t i, uint32_t u, uint4 x) {
                     const uint32_t any = __builtin_ctz(rows_in(i)), row0 = 4 * (group0 + i) - start;
                     reinterpret_cast<uint4*>(pool.v + (to_sh[row0 + any] - any) * rb)[u] = x;
                 });
#pragma unroll
            for (uint32_t c = 0; c < 4; ++c) {
                if (DT == VSPEC_KV_INT4 && ok && c < G) pool.vs[to * G + c] = scale[c];
            }
            for (uint32_t c = 4; DT == VSPEC_KV_INT4 && c < G; ++c) {
                if (ok) scale[0] = pool.vs[from * G + c];
                __syncthreads();
                if (ok) pool.vs[to * G + c] = scale[0];
            }
        }
        return;
    }
    for (uint32_t l = first; l < last; ++l) {
        const AcceptPool& pool = p.pools[l];
        uint8_t* const base = isv ? pool.v : pool.k;
        uint16_t scale[4] = {0, 0, 0, 0};  // of row `lane`, and its flag
        uint32_t flag = 0;
        auto scale_at = [&](const size_t token, const uint32_t slot, const uint32_t c) { return pool.ks + (token - slot) * G + (size_t)c * P + slot; };
        auto flag_at = [&](const size_t token) { return pool.kf + token / 16; };  // a bit a row, in words of 16
        const bool scales = DT == VSPEC_KV_INT4 && ok;
#pragma unroll
        for (uint32_t c = 0; c < 4; ++c) {
            if (scales && c < G) scale[c] = *scale_at(from, fs, c);
        }
        if (scales && pool.kf) flag = (*flag_at(from) >> (fs % 16)) & 1u;
        pass(std::integral_constant<int, 8>(), count, rb / 16, moved, [&](uint32_t row, uint32_t u) { return reinterpret_cast<const uint4*>(base + from_sh[row] * rb)[u]; },
             [&](uint32_t row, uint32_t u, uint4 x) { reinterpret_cast<uint4*>(base + to_sh[row] * rb)[u] = x; });
#pragma unroll
        for (uint32_t c = 0; c < 4; ++c) {
            if (scales && c < G) *scale_at(to, ts, c) = scale[c];
        }
        if (scales && pool.kf) {
            const uint32_t m = 1u << (ts % 16);
            if (flag) atomicOr(flag_at(to), m);
            else atomicAnd(flag_at(to), ~m);
        }
        for (uint32_t c = 4; DT == VSPEC_KV_INT4 && c < G; ++c) {
            if (ok) scale[0] = *scale_at(from, fs, c);
            __syncthreads();
            if (ok) *scale_at(to, ts, c) = scale[0];
        }
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
        p.layers = n;
        const uint64_t all = 2ull * n * p.hkv * batch, target = 24ull * host_num_cus();
        p.share = (uint32_t)(all <= target ? 1 : (all + target - 1) / target < n ? (all + target - 1) / target : n);
        const dim3 grid(p.hkv, batch, 2 * ((n + p.share - 1) / p.share));
        switch (kvs[0].dtype) {
            case VSPEC_KV_F32: hipLaunchKernelGGL((kv_accept<VSPEC_KV_F32>), grid, dim3(64), 0, s, p); break;
            case VSPEC_KV_F16: hipLaunchKernelGGL((kv_accept<VSPEC_KV_F16>), grid, dim3(64), 0, s, p); break;
            default: hipLaunchKernelGGL((kv_accept<VSPEC_KV_INT4>), grid, dim3(64), 0, s, p); break;
        }
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) {
        host_error("kv_accept launch: %s", hipGetErrorString(e));
        return 0;
    }
    return 1;
}
