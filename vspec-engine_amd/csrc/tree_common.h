// tree_common.h -- what the kernels of the attention of a drafted tree share: tree_mfma.hip
// (few columns, and f32 pools) and tree_wide.hip (many columns).
#pragma once
#include "tree_attn.h"

namespace vkv {
namespace {

typedef _Float16 h2_t __attribute__((ext_vector_type(2)));
typedef _Float16 h4_t __attribute__((ext_vector_type(4)));
typedef _Float16 h8_t __attribute__((ext_vector_type(8)));
typedef float f4_t __attribute__((ext_vector_type(4)));

// log2 of p at the reference point: p <= 2^(kHeadroom + kThreshold) = 2^11, times 2^4 for int4 values
// beyond one f16
constexpr float kHeadroom = 3.0f;
constexpr float kThreshold = 8.0f;  // growth of the maximum, log2 units, that moves the reference point

__device__ __forceinline__ h8_t join(h4_t a, h4_t b) { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }

// Output element d of accumulator register r of d-tile j in lanes of row group g.
template <int DT>
__device__ __forceinline__ int out_dim(int j, int g, int r) {
    if constexpr (DT == VSPEC_KV_F16) return 32 * (j / 2) + 8 * g + 2 * r + j % 2;
    if constexpr (DT == VSPEC_KV_INT4) return 16 * j + 4 * g + r;
    return 64 * (j / 4) + 16 * g + 4 * r + j % 4;
}

// int4 codes to f16: pairs (nibble k, nibble k + 4) of a dword, exact (a nibble in the mantissa under
// a magic exponent, minus its bias)
__device__ __forceinline__ void codes_to_f16(uint32_t w, h2_t out[4]) {
    const uint32_t w8 = w >> 8;
    const h2_t b0 = {(_Float16)1032.0f, (_Float16)1032.0f}, b1 = {(_Float16)72.0f, (_Float16)72.0f};
    out[0] = __builtin_bit_cast(h2_t, ((w ^ 0x00080008u) & 0x000F000Fu) | 0x64006400u) - b0;
    out[1] = __builtin_bit_cast(h2_t, ((w ^ 0x00800080u) & 0x00F000F0u) | 0x54005400u) - b1;
    out[2] = __builtin_bit_cast(h2_t, ((w8 ^ 0x00080008u) & 0x000F000Fu) | 0x64006400u) - b0;
    out[3] = __builtin_bit_cast(h2_t, ((w8 ^ 0x00800080u) & 0x00F000F0u) | 0x54005400u) - b1;
}

// Between matrix instructions and the first vector instruction that reads their results.  Left to
// itself hipcc 7.2 mixes the two across branches, and one accumulator register of a tile then lost
// part of its sum (rows 4g of every second tile, off by 2^-13; seen in a kernel that added two chains
// behind a branch).
__device__ __forceinline__ void settle() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_nop 15");
    __builtin_amdgcn_sched_barrier(0);
}

constexpr uint32_t kBigScale = 0x6C00u;  // 2^12: a code times it may pass f16's range

// fp16 scales of group c of the lane's tokens 4g + 2e and 4g + 2e + 1 (token r's halves start at word r NQ / 2)
template <int NQ, typename T>
__device__ __forceinline__ uint32_t int4_scale_pair(const T& t, int c, int e) {
    const uint32_t w0 = t.vs[(2 * e) * NQ / 2 + c / 2], w1 = t.vs[(2 * e + 1) * NQ / 2 + c / 2];
    return c % 2 ? (w0 >> 16) | (w1 & 0xffff0000u) : (w0 & 0xffffu) | (w1 << 16);
}
// Values of d-tiles 2c (e) and 2c + 1 (o) from a code dword of group c: rounded, and with LOW the exact rest
template <bool LOW>
__device__ __forceinline__ void int4_values(uint32_t codes, const h2_t (&scale)[2], h4_t& e, h4_t& o, h4_t& el, h4_t& ol) {
    h2_t q[4];  // tokens 0, 1 of e and of o, tokens 2, 3 of e and of o
    codes_to_f16(codes, q);
    const h2_t e0 = q[0] * scale[0], e1 = q[2] * scale[1], o0 = q[1] * scale[0], o1 = q[3] * scale[1];
    e = __builtin_shufflevector(e0, e1, 0, 1, 2, 3);
    o = __builtin_shufflevector(o0, o1, 0, 1, 2, 3);
    if constexpr (LOW) {
        el = __builtin_shufflevector(__builtin_elementwise_fma(q[0], scale[0], -e0), __builtin_elementwise_fma(q[2], scale[1], -e1), 0, 1, 2, 3);
        ol = __builtin_shufflevector(__builtin_elementwise_fma(q[1], scale[0], -o0), __builtin_elementwise_fma(q[3], scale[1], -o1), 0, 1, 2, 3);
    }
}

// After the tokens' loop, and rarely: what is not finite among the nodes' values reaches the rows that see it.  The
// loop took it as zeros, for in its products 0 * inf would have reached the others.  +inf where a visible value is
// +inf or NaN, and -inf where one is -inf or NaN (both: NaN), counted by products of ones over tiles [first, last).
template <int DT, int D, int CT, typename SEES>
__device__ __forceinline__ void add_wild(const int32_t* tables, const int32_t* used, uint32_t num_blocks, uint32_t hkv, uint32_t h, int P, uint32_t magic,
                                         uint32_t shift, const TreeSpan& sp, int lane, int first, int last, SEES sees, f4_t (&acc)[CT][D / 16]) {
    kernel_args* late = late_args();
    const int g = lane >> 4, n = lane & 15;
    for (int tile = first; tile < last; ++tile) {
        const int row = tree_block_of(magic, shift, tile), slot0 = tile * kTile - row * P;
        const int entry = as_const(tables)[row];
        if (entry < 0 || (uint32_t)entry >= num_blocks) continue;
        const size_t bh = (size_t)entry * hkv + h;
        const int valid = min(min(kTile, sp.end - tile * kTile), used ? max(0, as_const(used)[row] - slot0) : kTile);
        uint32_t seen[CT];
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) seen[ct] = sees(ct, tile, valid);
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
            // the element of V operand j in this lane
            const uint32_t d = DT == VSPEC_KV_F16 ? 32 * (j / 2) + 2 * n + j % 2 : DT == VSPEC_KV_INT4 ? 16 * j + n : 64 * (j / 4) + 4 * n + j % 4;
            h4_t plus, minus;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const bool in = 4 * g + r < valid;
                const float v = in ? tree_value<DT, D>(late->v, late->vs, (uint32_t)P, bh, (uint32_t)(slot0 + 4 * g + r), d) : 0.f;
                plus[r] = in && !(v < INFINITY) ? (_Float16)1.f : (_Float16)0.f;
                minus[r] = in && !(v > -INFINITY) ? (_Float16)1.f : (_Float16)0.f;
            }
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) {
                h4_t vis;
#pragma unroll
                for (int r = 0; r < 4; ++r) vis[r] = (seen[ct] >> r) & 1u ? (_Float16)1.f : (_Float16)0.f;
                const f4_t zero = {0.f, 0.f, 0.f, 0.f};
                const f4_t up = __builtin_amdgcn_mfma_f32_16x16x16f16(plus, vis, zero, 0, 0, 0);
                const f4_t dn = __builtin_amdgcn_mfma_f32_16x16x16f16(minus, vis, zero, 0, 0, 0);
                settle();
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    acc[ct][j][r] += up[r] > 0.f ? INFINITY : 0.f;
                    acc[ct][j][r] += dn[r] > 0.f ? -INFINITY : 0.f;
                }
            }
        }
    }
}

// Joins the parts of the sequences that have more than one.  A task is a column tile of an item: the parts' weights
// through LDS, then four of the output's d-tiles, a wave each, or, of many parts, one d-tile that the waves share.
// Each load is 1 KB whole, and what counts is how many are on their way: a workgroup to a column tile, with every
// weight read again for each d-tile, took some 50 us for the 64 parts of 8 items where this takes 4.
constexpr uint32_t kMergeShared = 8;  // parts from which the waves share
template <int DT, int D, typename IO>
__global__ __launch_bounds__(256) void tree_merge(TreeParams p, uint32_t tiles, uint32_t cuts) {
    constexpr int NDT = D / 16;
    extern __shared__ float merge_sh[];  // [2][slot_rows][16]: weights (first: reference points), sums
    __shared__ float red[16][16];
    __shared__ f4_t joined[4][64];
    const uint32_t items = p.hkv * p.col_groups, per = items * tiles * cuts;
    const uint32_t tasks = (uint32_t)as_const(&p.plan->x)[0] * per;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, n = lane & 15;
    const int row = threadIdx.x >> 4;  // parts row, row + 16, ...
    float* const ref_sh = merge_sh + n;
    float* const sum_sh = ref_sh + 16 * p.slot_rows;
    const bool share = cuts == NDT;
    for (uint32_t task = blockIdx.x; task < tasks; task += gridDim.x) {
        const uint32_t split = task / per, rest = task - split * per;
        const uint32_t place = rest / cuts, cut = rest - place * cuts;  // place: item, column tile
        const uint32_t item = place / tiles, tile = place - item * tiles;
        const uint32_t cg = item / p.hkv, h = item - cg * p.hkv;
        const int4 plan = p.plan[1 + split];
        const uint32_t b = (uint32_t)uniform(plan.x);
        const int count = uniform(plan.y);
        const TreeSpan sp = tree_span(p, b);
        const size_t pitch = (size_t)items * tiles, first = (size_t)uniform(plan.z) * pitch + place;  // states of the parts
        float top = -INFINITY, total = 0.f;
        __syncthreads();  // (the task before has read its weights)
        for (int t = row; t < count; t += 16) {
            const float2 ml = reinterpret_cast<const float2*>(p.part_ml)[(first + t * pitch) * 16 + n];
            ref_sh[16 * t] = ml.x;
            sum_sh[16 * t] = ml.y;
            top = fmaxf(top, ml.x);
        }
        red[row][n] = top;
        __syncthreads();
        for (int r = 0; r < 16; ++r) top = fmaxf(top, red[r][n]);
        for (int t = row; t < count; t += 16) {
            const float f = __builtin_amdgcn_exp2f(ref_sh[16 * t] - top);
            ref_sh[16 * t] = f;
            total = fmaf(sum_sh[16 * t], f, total);
        }
        __syncthreads();
        red[row][n] = total;
        __syncthreads();
        total = 0.f;
        for (int r = 0; r < 16; ++r) total += red[r][n];

        const int j = share ? (int)cut : 4 * (int)cut + wave, step = share ? 4 : 1;
        const f4_t* src = reinterpret_cast<const f4_t*>(p.part_acc) + (first * NDT + j) * 64 + lane;
        f4_t a = {0.f, 0.f, 0.f, 0.f};
        int t = share ? wave : 0;
        for (; t + 7 * step < count; t += 8 * step) {
            f4_t x[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) x[u] = src[(size_t)(t + u * step) * pitch * (NDT * 64)];
#pragma unroll
            for (int u = 0; u < 8; ++u) a += x[u] * ref_sh[16 * (t + u * step)];
        }
        for (; t < count; t += step) a += src[(size_t)t * pitch * (NDT * 64)] * ref_sh[16 * t];
        if (share) {
            joined[wave][lane] = a;
            __syncthreads();
            if (wave != 0) continue;
            a = (joined[0][lane] + joined[1][lane]) + (joined[2][lane] + joined[3][lane]);
        }
        const int c = (int)((cg * tiles + tile) * 16) + n;
        if (c >= (int)(p.nodes * p.group)) continue;
        const int i = c / (int)p.group;
        const bool empty = i >= sp.len || total == 0.f;
        IO* dst = reinterpret_cast<IO*>(p.out) + (((size_t)b * p.nodes + i) * p.hq + (size_t)h * p.group + (c - i * (int)p.group)) * D;
#pragma unroll
        for (int r = 0; r < 4; ++r) dst[out_dim<DT>(j, g, r)] = (IO)(empty ? 0.f : a[r] / total);
    }
}

template <int DT, int D, typename IO>
void launch_merge(const TreeParams& p, uint32_t tiles, hipStream_t s) {
    const uint32_t cuts = p.slot_rows >= kMergeShared * p.batch ? D / 16 : D / 64;
    const uint64_t tasks = (uint64_t)min(p.batch, p.slot_rows) * p.hkv * p.col_groups * tiles * cuts;
    hipLaunchKernelGGL((tree_merge<DT, D, IO>), dim3((uint32_t)min(tasks, (uint64_t)1024)), dim3(256), p.slot_rows * 32 * sizeof(float), s, p, tiles, cuts);
}

}  // namespace
}  // namespace vkv
