// tree_wide.hip -- attention of a drafted tree over f16 and int4 pools where many query rows share
// a kv head (more than 32: nodes times GQA group).
//
// The products are those of tree_mfma.hip, S^T = K Q^T and O^T += V^T P^T with 16 columns to a
// tile, but here the W waves of a workgroup are side by side over the columns, CT tiles each, and
// share every K and V tile through LDS in the order in which the matrix instructions take it.
// What is done to a key or value once for all columns is done once by the workgroup:
//   f16   tiles stream into an LDS ring (buffer loads straight into LDS, DEPTH steps).  The wave
//         that loaded a key's row screens it for the clip to its own standard deviation, rewrites a
//         clipped row in place and leaves its low part beside it.
//   int4  codes and scales stream into a ring of each wave; it turns its share of a step into f16
//         rows, keys with their low parts (values for f32 queries), in LDS, clipped on the way.
// A wave's column then costs per 32 tokens its matrix instructions, 8 weights a lane and 16 reads
// of 16 bytes from LDS.  With CT = 2 and 8 waves the LDS reads (128 KB a step, 1024 cycles) are as
// long as the f16 matrix work of 256 columns; with one tile a wave they would be twice that.
//
// What bounds it (GQA 32 / 8, D = 128, 64 x 4097 tokens and 64 nodes, f16 rows): an f16 pool those reads
// and the matrix instructions together, 435 us, 630 TFLOP/s; an int4 pool their low parts besides, 715.
// Few tiles a workgroup: 16 x 2049 tokens, 16 nodes, f32 rows, 45 us (f16), 66 (int4, the conversion).
//
// One barrier a step orders the ring (f16): a wave issues the loads of step s + DEPTH - 1 into the
// slot of step s - 1, which every wave left before the last barrier.
#include "lds_load.h"
#include "tree_common.h"

namespace vkv {
namespace {

// A descriptor in scalar registers, from values that every lane holds alike
__device__ __forceinline__ rsrc_t uniform_rsrc(const void* base, uint32_t bytes) {
    const rsrc_t r = tile_rsrc(base, bytes);
    return rsrc_t{__builtin_amdgcn_readfirstlane(r[0]), __builtin_amdgcn_readfirstlane(r[1]), __builtin_amdgcn_readfirstlane(r[2]),
                  __builtin_amdgcn_readfirstlane(r[3])};
}

__device__ __forceinline__ void barrier_lds() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// The chunk of its row in lane (position) l of a set of TI rows (set m of a tile), and the position's inverse:
// the 16 rows' chunks of one operand then lie in different banks.
template <int D>
__device__ __forceinline__ int chunk_of(int m, int l) {
    constexpr int CPT = D / 8;
    const int t = l / CPT;
    return (l % CPT) ^ (D == 128 ? 4 * m + t : 4 * m + (t >> 1));
}

template <typename IO>
constexpr bool SPLIT_IO = sizeof(IO) == 4;

template <int DT, int D, typename IO, int CT, int W>
__global__ __launch_bounds__(W * 64, 2) void tree_wide(TreeParams p) {
    constexpr bool F16 = DT == VSPEC_KV_F16;
    constexpr bool SPLIT = SPLIT_IO<IO>;      // q in two f16 parts
    constexpr bool KLO = !F16;                // K in two f16 parts
    constexpr bool PLO = SPLIT || !F16;       // p in two f16 parts
    constexpr bool VLO = SPLIT && !F16;       // V in two f16 parts
    constexpr int NQ = D / 32, NDT = D / 16;
    constexpr int KT = wide_step_tiles(SPLIT, CT);  // 16-token tiles of a step
    constexpr int CPT = D / 8;                // 8-element chunks of a row
    constexpr int TI = 64 / CPT;              // rows that a wave takes at a time, a chunk a lane
    constexpr int TPO = 16 * KT / W < TI ? TI : 16 * KT / W;  // rows of a step that a wave looks after: TPO w .., of one tile
    constexpr int SETS = TPO / TI;
    constexpr int OWNERS = 16 * KT / TPO;     // waves that look after rows
    constexpr int kTileB = 32 * D;            // bytes of a tile in f16
    constexpr int kStageB = 2 * KT * kTileB;  // K of all tiles, V of all
    constexpr int DEPTH = F16 ? (KT == 4 ? 2 : W == 8 ? 4 : 3) : 1;
    constexpr int RAW = 3;                    // steps of codes in the ring
    constexpr int kRawB = F16 ? 16 : 512 * SETS + 512;  // of a wave and step: K, V, K scales, V scales
    __shared__ __align__(16) uint8_t stage[DEPTH * kStageB];
    __shared__ __align__(16) uint8_t low[F16 ? (SPLIT ? 2 * KT * kTileB : 16) : (VLO ? kStageB : KT * kTileB)];  // low parts: f16 [mark][K], int4 as a stage
    __shared__ __align__(16) uint8_t raw[F16 ? 16 : RAW * OWNERS * kRawB];
    // a bit for each row of a step, whole bytes of each wave's: clipped or not finite; K (int4) and V (int4) hold a 16th of the
    // value; V held something that is not finite
    __shared__ __align__(8) uint16_t marks[2][4][4];
    __shared__ uint64_t bits_sh[64];

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, n = lane & 15;
    const TreeJob job = tree_job<KT>(p, (int)blockIdx.y, 1);
    if (job.b < 0) return;
    const uint32_t b = (uint32_t)job.b, item = blockIdx.x;
    const uint32_t cg = (uint32_t)uniform((int)(item / p.hkv)), h = item - cg * p.hkv;
    const TreeSpan sp = job.span;
    const TreeSteps tp = tree_steps<KT>(sp);
    const int lo = job.lo, hi = job.hi;
    if (threadIdx.x < 64) bits_sh[threadIdx.x] = threadIdx.x < p.nodes ? tree_bits(p, b, threadIdx.x, sp.len) : 0;

    // q: columns of this wave, on their way before K and V (loads come back in order)
    const int cols = (int)(p.nodes * p.group);
    const int ctile0 = ((int)cg * W + wave) * CT;
    typedef IO raw_t __attribute__((ext_vector_type(8), aligned(16)));
    raw_t rawq[CT][NQ];
    bool live[CT];
    int node[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
        const int c = (ctile0 + ct) * 16 + n;
        const int i = c / (int)p.group;
        node[ct] = min(i, (int)p.nodes - 1);
        live[ct] = c < cols && i < sp.len;
        const IO* src = reinterpret_cast<const IO*>(p.q) + (((size_t)b * p.nodes + (live[ct] ? i : 0)) * p.hq + (size_t)h * p.group + (live[ct] ? c - i * (int)p.group : 0)) * D;
#pragma unroll
        for (int k = 0; k < NQ; ++k) rawq[ct][k] = *reinterpret_cast<const raw_t*>(src + 32 * k + 8 * g);
    }

    const int P = (int)own_scalar(p.block_tokens);
    const int32_t* const tables = own_scalar(p.block_tables + (size_t)b * p.max_blocks);
    const int32_t* const used = own_scalar(p.block_used ? p.block_used + (size_t)b * p.max_blocks : nullptr);
    const uint8_t* const kdata = own_scalar(p.k);
    const uint8_t* const vdata = own_scalar(p.v);
    const uint16_t* const kscales = own_scalar(p.ks);
    const uint16_t* const vscales = own_scalar(p.vs);
    const uint32_t num_blocks = own_scalar(p.num_blocks), hkv = own_scalar(p.hkv);
    const uint32_t magic = own_scalar(p.block_magic), shift = own_scalar(p.block_shift);
    const float alpha = own_scalar(p.alpha), input_clip = own_scalar(p.input_clip);

    // The tiles of the next 64 / KT steps, a lane each: where a tile lies (token index in the pool), its slot in the
    // block and how many tokens it holds (0: it is not read).  Read lane by lane, this costs a step two scalar
    // moves a tile; table look-ups of each step were 170 instructions.
    constexpr int kSpan = 64 / KT;
    size_t t_token = 0;
    int t_info = 0;  // slot0 << 5 | tokens
    auto look_up = [&](const int first) {
        const int step = first + lane / KT, a = lane % KT;
        const int tile = step < tp.prefix_steps ? KT * step + a : tp.prefix_tiles + KT * (step - tp.prefix_steps) + a;
        const bool in = step < hi && tile < (step < tp.prefix_steps ? tp.prefix_tiles : tp.tiles);
        const int row = in ? tree_block_of(magic, shift, tile) : 0;
        const int entry = tables[row];
        const int room = used ? used[row] : P;
        const bool ok = in && entry >= 0 && (uint32_t)entry < num_blocks;
        const int slot0 = ok ? tile * kTile - row * P : 0;
        t_token = ((size_t)(ok ? entry : 0) * hkv + h) * P + slot0;
        t_info = slot0 << 5 | (ok ? min(min(kTile, sp.end - tile * kTile), max(0, room - slot0)) : 0);
    };
    struct Where {
        size_t token;
        int slot0, valid;
    };
    int table0 = lo;  // the first step of the table
    auto where = [&](const int step, const int a) -> Where {
        const int l = uniform((step - table0) * KT + a);
        const uint32_t t0 = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)t_token, l);
        const uint32_t t1 = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(t_token >> 32), l);
        const int info = __builtin_amdgcn_readlane(t_info, l);
        return {(size_t)t1 << 32 | t0, info >> 5, info & 31};
    };
    auto first_tile = [&](const int step) { return step < tp.prefix_steps ? KT * step : tp.prefix_tiles + KT * (step - tp.prefix_steps); };

    // ---- loads of this wave's share of a step ----
    const bool owner = OWNERS == W || wave < OWNERS;
    const int my_tile = owner ? TPO * wave / kTile : 0;  // the tile of its rows
    const int my_part = TPO * wave % kTile / TPO;    // and which TPO rows of it
    uint32_t koff[SETS], voff[SETS];                 // f16: byte offsets of this lane's chunks in the tile
    if constexpr (F16) {
#pragma unroll
        for (int k = 0; k < SETS; ++k) {
            const int m = my_part * SETS + k;  // rows TI m .. of the tile, V operands m
            koff[k] = (uint32_t)((TI * m + lane / CPT) * 2 * D + 16 * chunk_of<D>(m, lane));
            voff[k] = (uint32_t)(g * 8 * D + (32 * m + 2 * n) * 8);
        }
    }
    const uint32_t stage0 = lds_addr(stage), raw0 = lds_addr(raw);
    auto load = [&](const Where& w, const int slot) {
        if (!owner) return;
        if constexpr (F16) {
            const uint32_t bytes = w.valid > 0 ? kTileB : 0;
            const size_t at = w.token * (size_t)(2 * D);
            const rsrc_t kr = uniform_rsrc(kdata + at, bytes), vr = uniform_rsrc(vdata + at, bytes);
            const uint32_t dst = stage0 + slot * kStageB + my_tile * kTileB + my_part * SETS * 1024;
#pragma unroll
            for (int k = 0; k < SETS; ++k) lds_load16(__builtin_amdgcn_readfirstlane(dst + 1024 * k), kr, koff[k]);
#pragma unroll
            for (int k = 0; k < SETS; ++k) lds_load16(__builtin_amdgcn_readfirstlane(dst + KT * kTileB + 1024 * k), vr, voff[k]);
        } else {
            const uint32_t bytes = w.valid > 0 ? 8 * D : 0;
            const size_t at = w.token * (size_t)(D / 2);
            const rsrc_t kr = uniform_rsrc(kdata + at, bytes), vr = uniform_rsrc(vdata + at, bytes);
            const rsrc_t ksr = uniform_rsrc(kscales + (w.token - w.slot0) * NQ + w.slot0, w.valid > 0 ? (uint32_t)((NQ - 1) * P * 2 + 32) : 0u);
            const rsrc_t vsr = uniform_rsrc(vscales + w.token * NQ, w.valid > 0 ? 32 * NQ : 0);
            const uint32_t dst = raw0 + (slot * OWNERS + wave) * kRawB;
            const uint32_t from = my_part * TPO * (D / 2) + 4 * lane;
#pragma unroll
            for (int k = 0; k < SETS; ++k) {
                lds_load4(__builtin_amdgcn_readfirstlane(dst + 256 * k), kr, from + 256 * k);
                lds_load4(__builtin_amdgcn_readfirstlane(dst + 256 * (SETS + k)), vr, from + 256 * k);
            }
            lds_load4(__builtin_amdgcn_readfirstlane(dst + 512 * SETS), ksr, lane < 8 * NQ ? (uint32_t)((lane / 8) * P * 2 + (lane % 8) * 4) : 0x7fffffffu);
            lds_load4(__builtin_amdgcn_readfirstlane(dst + 512 * SETS + 256), vsr, 4 * lane);
        }
    };
    constexpr int kLoads = F16 ? 2 * SETS : 2 * SETS + 2;  // of a step

    // ---- what a wave does to its rows of a step before all waves read them ----
    // (a row's chunks lie in CPT adjacent lanes)
    auto row_sum = [&](float x) { return group_sum<CPT>(x); };
    // the bits of its rows (of set k) from a ballot in which any lane of a row speaks for it
    auto row_bits = [&](uint64_t m) -> uint32_t {
        uint32_t r = 0;
#pragma unroll
        for (int t = 0; t < TI; ++t) r |= (uint32_t)((m >> (CPT * t)) & ((1ull << CPT) - 1)) ? 1u << t : 0u;
        return r;
    };
    auto limit_of = [&](float var) { return fminf(fmaxf(1e-6f, alpha * sqrtf(var * (1.0f / D))), input_clip); };
    auto prepare = [&](const int step, const int valid, const int slot, const int mark, const int raw_slot) {
        if (!owner) return;
        uint32_t clipped = 0, kbig = 0, vbig = 0, odd_v = 0;
        // V of slots without a token may hold any bits and becomes zeros.  In tiles that hold nodes so does
        // what is not finite: in the products 0 * inf would reach the rows that do not see it
        const bool tree = (first_tile(step) + my_tile) * kTile + valid > sp.start;
        if constexpr (F16) {
            uint8_t* mine = stage + slot * kStageB + my_tile * kTileB + my_part * SETS * 1024 + 16 * lane;
            const h2_t ones = {(_Float16)1.0f, (_Float16)1.0f};
#pragma unroll
            for (int k = 0; k < SETS; ++k) {
                const uint4 w = *reinterpret_cast<const uint4*>(mine + 1024 * k);
                const uint32_t w4[4] = {w.x, w.y, w.z, w.w};
                float s1 = 0.f, s2 = 0.f;
                h2_t mx2 = {(_Float16)0.f, (_Float16)0.f};
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const h2_t y = __builtin_bit_cast(h2_t, w4[c]);
                    s1 = __builtin_amdgcn_fdot2(y, ones, s1, false);
                    s2 = __builtin_amdgcn_fdot2(y, y, s2, false);
                    mx2 = __builtin_elementwise_max(mx2, __builtin_elementwise_abs(y));
                }
                const float mx = fmaxf((float)mx2[0], (float)mx2[1]);
                const float mean1 = row_sum(s1) * (1.0f / D), ex2 = row_sum(s2) * (1.0f / D);
                const float var1 = ex2 - mean1 * mean1;
                const float th1 = fminf(fmaxf(1e-6f, alpha * __builtin_amdgcn_sqrtf(fmaxf(var1, 0.f))), input_clip);
                // the margins of the decode's screen; !(<=) also takes what is not finite
                const bool flag = !(mx <= th1 * (1.0f - 0.0009765625f)) || var1 <= ex2 * 0.0009765625f;
                const int row = TI * (my_part * SETS + k) + lane / CPT;
                const uint64_t any = __builtin_amdgcn_ballot_w64(flag && row < valid);
                if (any == 0) continue;
                // exactly, for the rows that it takes: two-pass deviation, the clipped row in two f16 parts.
                // Elements inside the limit stay exact, the limit keeps 22 bits or 2^-25.
                const uint32_t rows = row_bits(any);
                clipped |= rows << (TI * k);
                const h8_t x8 = __builtin_bit_cast(h8_t, w);
                float x[8], sum = 0.f, var = 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    x[e] = (float)x8[e];
                    sum += x[e];
                }
                const float mean = row_sum(sum) * (1.0f / D);
#pragma unroll
                for (int e = 0; e < 8; ++e) var = fmaf(x[e] - mean, x[e] - mean, var);
                const float th = limit_of(row_sum(var));
                h8_t yh, yl;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float y = x[e] != x[e] ? x[e] : __builtin_amdgcn_fmed3f(x[e], -th, th);
                    yh[e] = (_Float16)y;
                    yl[e] = (_Float16)(y - (float)yh[e]);
                }
                if ((rows >> (lane / CPT)) & 1u) {
                    *reinterpret_cast<h8_t*>(mine + 1024 * k) = yh;
                    if constexpr (SPLIT) *reinterpret_cast<h8_t*>(low + mark * KT * kTileB + my_tile * kTileB + (my_part * SETS + k) * 1024 + 16 * lane) = yl;
                }
            }
            if (tree || valid < kTile) {
#pragma unroll
                for (int k = 0; k < SETS; ++k) {
                    h8_t* at = reinterpret_cast<h8_t*>(mine + KT * kTileB + 1024 * k);
                    h8_t v = *at;
                    bool out = false;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const bool held = 4 * g + e % 4 < valid;
                        const bool odd = tree && held && !(fabsf((float)v[e]) < INFINITY);
                        out = out || odd;
                        v[e] = held && !odd ? v[e] : (_Float16)0.f;
                    }
                    *at = v;
                    odd_v |= __builtin_amdgcn_ballot_w64(out) != 0 ? 1u : 0u;
                }
            }
        } else {
            const uint8_t* mine = raw + (raw_slot * OWNERS + wave) * kRawB;
            const uint16_t* kscale = reinterpret_cast<const uint16_t*>(mine + 512 * SETS);
            const uint16_t* vscale = reinterpret_cast<const uint16_t*>(mine + 512 * SETS + 256);
#pragma unroll
            for (int k = 0; k < SETS; ++k) {
                const int row = my_part * TPO + TI * k + lane / CPT, c = lane % CPT;  // row of the tile, chunk
                const uint32_t w = *reinterpret_cast<const uint32_t*>(mine + 256 * k + 4 * lane);
                uint16_t s16 = kscale[(c / 4) * 16 + row];
                const float sc = half_bits_to_float(s16);
                const int c1 = __builtin_amdgcn_sdot8((int)w, 0x11111111, 0, false);
                const int c2 = __builtin_amdgcn_sdot8((int)w, (int)w, 0, false);
                const float mean1 = row_sum(sc * (float)c1) * (1.0f / D), ex2 = row_sum(sc * sc * (float)c2) * (1.0f / D);
                const float var1 = ex2 - mean1 * mean1;
                const float th1 = fminf(fmaxf(1e-6f, alpha * __builtin_amdgcn_sqrtf(fmaxf(var1, 0.f))), input_clip);
                const float mx = 8.0f * fabsf(sc);
                // (a code times a scale past 7500 may pass f16's range)
                const bool flag = !(mx <= th1 * (1.0f - 0.0009765625f)) || var1 <= ex2 * 0.0009765625f || mx > 60000.f;
                h2_t q4[4];
                codes_to_f16(w, q4);
                h8_t yh, yl;
                const h2_t s2v = {__builtin_bit_cast(_Float16, s16), __builtin_bit_cast(_Float16, s16)};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const h2_t y = q4[e] * s2v;
                    yh[2 * e] = y[0], yh[2 * e + 1] = y[1];
                    const h2_t z = __builtin_elementwise_fma(q4[e], s2v, -y);  // exact
                    yl[2 * e] = z[0], yl[2 * e + 1] = z[1];
                }
                const uint64_t any = __builtin_amdgcn_ballot_w64(flag && row < valid);
                if (any != 0) {
                    const uint32_t rows = row_bits(any);
                    clipped |= rows << (TI * k);
                    const uint32_t large = row_bits(__builtin_amdgcn_ballot_w64(mx > 60000.f && row < valid));
                    kbig |= large << (TI * k);
                    float x[8], sum = 0.f, var = 0.f;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        x[e] = (float)q4[e / 2][e % 2] * sc;
                        sum += x[e];
                    }
                    const float mean = row_sum(sum) * (1.0f / D);
#pragma unroll
                    for (int e = 0; e < 8; ++e) var = fmaf(x[e] - mean, x[e] - mean, var);
                    const float th = limit_of(row_sum(var));
                    const float down = (large >> (lane / CPT)) & 1u ? 0.0625f : 1.f;
                    const bool mine_too = (rows >> (lane / CPT)) & 1u;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float y = (x[e] != x[e] ? x[e] : __builtin_amdgcn_fmed3f(x[e], -th, th)) * down;
                        const _Float16 y16 = (_Float16)y, z16 = (_Float16)(y - (float)y16);
                        yh[e] = mine_too ? y16 : yh[e];
                        yl[e] = mine_too ? z16 : yl[e];
                    }
                }
                const int m = row / TI, t = row % TI;
                const int at = my_tile * kTileB + m * 1024 + (CPT * t + chunk_of<D>(m, CPT * t + c)) * 16;
                *reinterpret_cast<h8_t*>(stage + at) = yh;
                *reinterpret_cast<h8_t*>(low + at) = yl;
            }
#pragma unroll
            for (int k = 0; k < SETS; ++k) {
                // V: word c of lane chunk (vg, vn) of the tile, tokens 4 vg .. 4 vg + 3
                const int idx = my_part * (TPO * D / 8) + 64 * k + lane;
                const int c = idx % NQ, chunk = idx / NQ, vg = chunk / 16;
                const uint32_t w = *reinterpret_cast<const uint32_t*>(mine + 256 * (SETS + k) + 4 * lane);
                uint32_t sw[2], top = 0;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    uint32_t a = vscale[(4 * vg + 2 * e) * NQ + c], z = vscale[(4 * vg + 2 * e + 1) * NQ + c];
                    a = 4 * vg + 2 * e < valid ? a : 0u;
                    z = 4 * vg + 2 * e + 1 < valid ? z : 0u;
                    top = max(top, max(a & 0x7fffu, z & 0x7fffu));
                    sw[e] = a | (z << 16);
                }
                if (tree && __builtin_amdgcn_ballot_w64(top >= 0x7C00u) != 0) {
                    odd_v = 1;
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        sw[e] &= ((sw[e] & 0x7fffu) < 0x7C00u ? 0xffffu : 0u) | (((sw[e] >> 16) & 0x7fffu) < 0x7C00u ? 0xffff0000u : 0u);
                    }
                }
                h2_t sp2[2] = {__builtin_bit_cast(h2_t, sw[0]), __builtin_bit_cast(h2_t, sw[1])};
                if (__builtin_amdgcn_ballot_w64(top >= kBigScale) != 0) {
                    // tokens with a scale that large in any group: a 16th of the value, 16 times the weight
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        uint32_t most = (sw[r / 2] >> (16 * (r % 2))) & 0x7fffu;
                        most = max(most, (uint32_t)__shfl_xor((int)most, 1));
                        if constexpr (NQ == 4) most = max(most, (uint32_t)__shfl_xor((int)most, 2));
                        const bool is = most >= kBigScale;
                        sp2[r / 2][r % 2] *= is ? (_Float16)0.0625f : (_Float16)1.f;
                        const uint64_t all = __builtin_amdgcn_ballot_w64(is);
                        // the words of a set belong to 4 tokens (64-element rows: 8, 4 in each half of the wave)
                        if constexpr (NQ == 4) vbig |= all ? 1u << (4 * k + r) : 0u;
                        else vbig |= ((uint32_t)all ? 1u << (8 * k + r) : 0u) | ((uint32_t)(all >> 32) ? 16u << (8 * k + r) : 0u);
                    }
                }
                h4_t ve, vo, vel, vol;
                int4_values<VLO>(w, sp2, ve, vo, vel, vol);
                const int at = KT * kTileB + my_tile * kTileB + c * 1024 + (chunk % 64) * 16;
                *reinterpret_cast<h8_t*>(stage + at) = join(ve, vo);
                if constexpr (VLO) *reinterpret_cast<h8_t*>(low + at) = join(vel, vol);
            }
        }
        if (lane == 0) {
            const uint32_t m[4] = {clipped, kbig, vbig, odd_v};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (TPO == 16) marks[mark][i][wave] = (uint16_t)m[i];
                else reinterpret_cast<uint8_t*>(marks[mark][i])[wave] = (uint8_t)m[i];
            }
        }
    };
    // the marks of a step, and of its tile a alone: 16 bits
    auto marks_of = [&](const int mark, const int which) -> uint64_t {
        const uint2 w = *reinterpret_cast<const uint2*>(marks[mark][which]);
        const uint64_t all = (uint64_t)(uint32_t)uniform((int)w.y) << 32 | (uint32_t)uniform((int)w.x);
        return KT == 4 || TPO == 4 ? all : all & 0xffffffffull;
    };
    auto tile_marks = [](uint64_t m, int a) -> uint32_t {
        if constexpr (TPO == 4) {
            const uint32_t w = (uint32_t)(m >> (32 * a));  // 4 bits in each byte
            return (w & 0xfu) | (w >> 4 & 0xf0u) | (w >> 8 & 0xf00u) | (w >> 12 & 0xf000u);
        } else {
            return (uint32_t)(m >> (16 * a)) & 0xffffu;
        }
    };

    // ---- the first steps on their way, then q ----
    constexpr int AHEAD = F16 ? DEPTH - 1 : RAW - 1;
    int held[AHEAD + 1];  // tokens of the tiles of the step at work and of those on their way, 5 bits each
    look_up(lo);
    auto load_step = [&](const int step, const int slot) -> int {
        if (step == table0 + kSpan) {
            table0 = step;
            look_up(step);
        }
        int tokens = 0;
#pragma unroll
        for (int a = 0; a < KT; ++a) tokens |= (uniform(__builtin_amdgcn_readlane(t_info, (step - table0) * KT + a)) & 31) << (5 * a);
        load(where(step, my_tile), slot);
        return tokens;
    };
#pragma unroll
    for (int s = 0; s < AHEAD; ++s) held[s] = load_step(lo + s, s);

    h8_t qh[CT][NQ], ql[SPLIT ? CT : 1][NQ];
    float fac[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
        float x[8 * NQ], sum = 0.f, var = 0.f, am = 0.f;
#pragma unroll
        for (int e = 0; e < 8 * NQ; ++e) {
            x[e] = live[ct] ? (float)rawq[ct][e / 8][e % 8] : 0.f;
            sum += x[e];
        }
        sum = add_rows(sum);
        const float mean = sum * (1.0f / D);
#pragma unroll
        for (int e = 0; e < 8 * NQ; ++e) var = fmaf(x[e] - mean, x[e] - mean, var);
        const float th = limit_of(add_rows(var));
#pragma unroll
        for (int e = 0; e < 8 * NQ; ++e) {
            x[e] = fminf(fmaxf(x[e], -th), th);
            am = fmaxf(am, fabsf(x[e]));
        }
        int ex = 0;
        if constexpr (SPLIT) ex = qnorm_shift(max_rows(am));
        fac[ct] = sum != sum ? sum : p.scale * pow2i(-ex);  // (a row with NaN gives NaN: the clips would hide it)
        const float up = pow2i(ex);
#pragma unroll
        for (int k = 0; k < NQ; ++k) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                // int4: halves 2m, 2m + 1 are nibbles m, m + 4
                const float y = x[8 * k + (F16 ? e : e / 2 + 4 * (e % 2))] * up;
                const _Float16 y16 = (_Float16)y;
                qh[ct][k][e] = y16;
                if constexpr (SPLIT) ql[ct][k][e] = (_Float16)(y - (float)y16);
            }
        }
    }

    f4_t acc[CT][NDT], total[CT];  // total: sum of the weights, as a row of ones would have it
    float limit[CT], mf[CT], clip[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
        limit[ct] = -INFINITY;
        clip[ct] = p.logit_clip / fac[ct];
        mf[ct] = -1e30f;
        total[ct] = f4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < NDT; ++j) acc[ct][j] = f4_t{0.f, 0.f, 0.f, 0.f};
    }

    // LDS offset of this lane's K operand 0 in a tile; operand i is at kread ^ 64 i
    const int kread = (n / TI) * 1024 + (CPT * (n % TI) + chunk_of<D>(n / TI, CPT * (n % TI) + g)) * 16;

    // bits of the lane's tokens 4g .. 4g + 3 of a tile that column ct sees
    auto sees = [&](const int ct, const int tile, const int valid) -> uint32_t {
        const int j0 = tile * kTile + 4 * g - sp.start;  // the node that the lane's first token is
        const uint64_t mine = bits_sh[node[ct]];
        const uint32_t seen = j0 <= -4 ? 15u
                              : j0 < 0 ? (uint32_t)(mine << -j0) | ((1u << -j0) - 1u)
                              : j0 < 64 ? (uint32_t)(mine >> j0) : 0u;
        const int left = valid - 4 * g;
        return seen & (left >= 4 ? 15u : left > 0 ? (1u << left) - 1u : 0u);
    };
    bool wild = false;  // some step's V held what is not finite, among nodes

    auto compute = [&](const int step, const int slot, const int mark, const int tokens) {
        const uint8_t* st = stage + slot * kStageB;
        f4_t sc[CT][KT];
        const uint64_t fl = marks_of(mark, 0);
        uint64_t kb = 0, vb = 0;
        if constexpr (!F16) kb = marks_of(mark, 1), vb = marks_of(mark, 2);
        // a tile that holds nodes or fewer than 16 tokens
        const bool masked = step >= tp.prefix_steps || tokens != (KT == 4 ? 0x84210 : 0x210);
#pragma unroll
        for (int a = 0; a < KT; ++a) {
            h8_t kh[NQ], kl[KLO ? NQ : 1];
#pragma unroll
            for (int i = 0; i < NQ; ++i) {
                kh[i] = *reinterpret_cast<const h8_t*>(st + a * kTileB + (kread ^ (64 * i)));
                if constexpr (KLO) kl[i] = *reinterpret_cast<const h8_t*>(low + a * kTileB + (kread ^ (64 * i)));
            }
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) {
                f4_t c = {0.f, 0.f, 0.f, 0.f};
                if constexpr (SPLIT) {
#pragma unroll
                    for (int i = 0; i < NQ; ++i) c = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh[i], ql[ct][i], c, 0, 0, 0);
                }
                if constexpr (KLO) {
#pragma unroll
                    for (int i = 0; i < NQ; ++i) c = __builtin_amdgcn_mfma_f32_16x16x32_f16(kl[i], qh[ct][i], c, 0, 0, 0);
                }
#pragma unroll
                for (int i = 0; i < NQ; ++i) c = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh[i], qh[ct][i], c, 0, 0, 0);
                sc[ct][a] = c;
            }
            if constexpr (CT > 1 && SPLIT) __builtin_amdgcn_sched_barrier(0);  // (registers: one tile's operands at a time)
        }
        if constexpr (SPLIT && F16) {
            if (fl != 0) {
#pragma unroll
                for (int a = 0; a < KT; ++a) {
                    if (tile_marks(fl, a) == 0) continue;
                    const bool has = (tile_marks(fl, a) >> n) & 1u;
                    const h8_t zero = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
                    for (int i = 0; i < NQ; ++i) {
                        h8_t kl = *reinterpret_cast<const h8_t*>(low + (mark * KT + a) * kTileB + (kread ^ (64 * i)));
                        kl = has ? kl : zero;
#pragma unroll
                        for (int ct = 0; ct < CT; ++ct) sc[ct][a] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kl, qh[ct][i], sc[ct][a], 0, 0, 0);
                    }
                }
            }
        }
        settle();

        // ---- softmax of column n over the lane's tokens ----
        if (masked || (fl | kb) != 0) {
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) {
#pragma unroll
                for (int a = 0; a < KT; ++a) {
                    const uint32_t seen = sees(ct, first_tile(step) + a, (tokens >> (5 * a)) & 31);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        float x = sc[ct][a][r];
                        if constexpr (!F16) x *= (tile_marks(kb, a) >> (4 * g + r)) & 1u ? 16.f : 1.f;
                        // (a key with NaN is always marked; the median would hide it)
                        x = x != x ? x : __builtin_amdgcn_fmed3f(x, -clip[ct], clip[ct]);
                        sc[ct][a][r] = (seen >> r) & 1u ? x : -INFINITY;
                    }
                }
            }
        } else {
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) {
#pragma unroll
                for (int a = 0; a < KT; ++a) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) sc[ct][a][r] = __builtin_amdgcn_fmed3f(sc[ct][a][r], -clip[ct], clip[ct]);
                }
            }
        }
        float top[CT];
        bool grown = false;
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
            top[ct] = -INFINITY;
#pragma unroll
            for (int a = 0; a < KT; ++a) top[ct] = fmaxf(top[ct], fmaxf(fmaxf(sc[ct][a][0], sc[ct][a][1]), fmaxf(sc[ct][a][2], sc[ct][a][3])));
            grown = grown || top[ct] > limit[ct];
        }
        if (__builtin_amdgcn_ballot_w64(grown) != 0) {
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) {
                const float mt = max_rows(top[ct]);
                const bool need = mt > limit[ct];
                const float nf = fmaf(mt, fac[ct], -kHeadroom);
                const float f = need ? __builtin_amdgcn_exp2f(mf[ct] - nf) : 1.0f;
                limit[ct] = need ? mt + kThreshold / fac[ct] : limit[ct];
                mf[ct] = need ? nf : mf[ct];
                total[ct] *= f;
#pragma unroll
                for (int j = 0; j < NDT; ++j) acc[ct][j] *= f;
            }
        }
        h8_t ph[CT][KT / 2], pl[PLO ? CT : 1][KT / 2];
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
#pragma unroll
            for (int u = 0; u < KT / 2; ++u) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float w = __builtin_amdgcn_exp2f(fmaf(sc[ct][2 * u + e / 4][e % 4], fac[ct], -mf[ct]));
                    const _Float16 w16 = (_Float16)w;
                    ph[ct][u][e] = w16;
                    if constexpr (PLO) pl[ct][u][e] = (_Float16)(w - (float)w16);
                }
                const _Float16 o = (_Float16)1.f;
                const h8_t ones = {o, o, o, o, o, o, o, o};
                total[ct] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, ph[ct][u], total[ct], 0, 0, 0);
                if constexpr (PLO) total[ct] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, pl[ct][u], total[ct], 0, 0, 0);
            }
        }
        if constexpr (!F16) {
            if (vb != 0) {
#pragma unroll
                for (int ct = 0; ct < CT; ++ct) {
#pragma unroll
                    for (int u = 0; u < KT / 2; ++u) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const _Float16 up = (tile_marks(vb, 2 * u + e / 4) >> (4 * g + e % 4)) & 1u ? (_Float16)16.f : (_Float16)1.f;
                            ph[ct][u][e] *= up;
                            if constexpr (PLO) pl[ct][u][e] *= up;
                        }
                    }
                }
            }
        }

        // ---- O^T += V^T P^T ----
#pragma unroll
        for (int u = 0; u < KT / 2; ++u) {
#pragma unroll
            for (int i = 0; i < NQ; ++i) {
                h8_t v[2], vl[VLO ? 2 : 1];  // of tile 2u + a: 4 tokens of d-tile 2i and of 2i + 1
#pragma unroll
                for (int a = 0; a < 2; ++a) {
                    const int at = (KT + 2 * u + a) * kTileB + i * 1024 + lane * 16;
                    v[a] = *reinterpret_cast<const h8_t*>(st + at);
                    if constexpr (VLO) vl[a] = *reinterpret_cast<const h8_t*>(low + at);
                }
#pragma unroll
                for (int o = 0; o < 2; ++o) {
                    const h8_t w = o ? __builtin_shufflevector(v[0], v[1], 4, 5, 6, 7, 12, 13, 14, 15) : __builtin_shufflevector(v[0], v[1], 0, 1, 2, 3, 8, 9, 10, 11);
                    h8_t wl;
                    if constexpr (VLO) wl = o ? __builtin_shufflevector(vl[0], vl[1], 4, 5, 6, 7, 12, 13, 14, 15) : __builtin_shufflevector(vl[0], vl[1], 0, 1, 2, 3, 8, 9, 10, 11);
#pragma unroll
                    for (int ct = 0; ct < CT; ++ct) {
                        f4_t& c = acc[ct][2 * i + o];
                        c = __builtin_amdgcn_mfma_f32_16x16x32_f16(w, ph[ct][u], c, 0, 0, 0);
                        if constexpr (PLO) c = __builtin_amdgcn_mfma_f32_16x16x32_f16(w, pl[ct][u], c, 0, 0, 0);
                        if constexpr (VLO) c = __builtin_amdgcn_mfma_f32_16x16x32_f16(wl, ph[ct][u], c, 0, 0, 0);
                    }
                }
                if constexpr (CT > 1 && SPLIT) __builtin_amdgcn_sched_barrier(0);
            }
        }
        settle();
        if (masked && marks_of(mark, 3) != 0) wild = true;
    };

    // Step s's loads are in slot (s - lo) % (AHEAD + 1); those of its wave have landed once no more than
    // the loads of the AHEAD - 1 steps after it are on their way.
    auto mine = [&](const int tokens) { return (tokens >> (5 * my_tile)) & 31; };
    wait_loads<(AHEAD - 1) * kLoads>();
    prepare(lo, mine(held[0]), 0, 0, 0);
    barrier_lds();
    int slot = 0, mark = 0;
    for (int step = lo; step < hi; ++step) {
        const int next = slot == AHEAD ? 0 : slot + 1;
        held[AHEAD] = load_step(step + AHEAD, slot == 0 ? AHEAD : slot - 1);
        compute(step, F16 ? slot : 0, mark, held[0]);
#pragma unroll
        for (int s = 0; s < AHEAD; ++s) held[s] = held[s + 1];
        wait_loads<(AHEAD - 1) * kLoads>();
        if constexpr (F16) {
            mark ^= 1;
            prepare(step + 1, mine(held[0]), next, mark, 0);
        } else {
            barrier_lds();  // (every wave has read this step's rows)
            prepare(step + 1, mine(held[0]), 0, 0, next);
        }
        barrier_lds();
        slot = next;
    }
    wait_loads<0>();
    settle();

    kernel_args* late = late_args();
    const int group = (int)late->group;
    if (wild) add_wild<DT, D, CT>(tables, used, num_blocks, hkv, h, P, magic, shift, sp, lane, first_tile(max(lo, tp.prefix_steps)), min(first_tile(hi), tp.tiles), sees, acc);
    const bool whole = job.count == 1;
    const size_t state = (size_t)(job.state + job.part) * (late->hkv * late->col_groups) + item;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
        const int tile = wave * CT + ct;
        const float sum = total[ct][0];
        if (!whole) {
#pragma unroll
            for (int j = 0; j < NDT; ++j) reinterpret_cast<f4_t*>(late->part_acc)[((state * (W * CT) + tile) * NDT + j) * 64 + lane] = acc[ct][j];
            if (g == 0) {
                float* ml = late->part_ml + ((state * (W * CT) + tile) * 16 + n) * 2;
                ml[0] = mf[ct];
                ml[1] = sum;
            }
            continue;
        }
        const int c = (ctile0 + ct) * 16 + n;
        if (c >= cols) continue;
        const int i = c / group;
        IO* dst = reinterpret_cast<IO*>(late->out) + (((size_t)b * late->nodes + i) * late->hq + (size_t)h * group + (c - i * group)) * D;
        const bool empty = i >= sp.len || sum == 0.f;
#pragma unroll
        for (int j = 0; j < NDT; ++j) {
#pragma unroll
            for (int r = 0; r < 4; ++r) dst[out_dim<DT>(j, g, r)] = (IO)(empty ? 0.f : acc[ct][j][r] / sum);
        }
    }
}

template <int DT, int D, typename IO, int CT, int W>
void launch(const TreeParams& p, hipStream_t s) {
    hipLaunchKernelGGL((tree_wide<DT, D, IO, CT, W>), dim3(p.hkv * p.col_groups, p.rows), dim3(W * 64), 0, s, p);
    if (p.slot_rows) launch_merge<DT, D, IO>(p, W * CT, s);
}

template <int DT, int D, typename IO>
void launch_any(const TreeParams& p, uint32_t ct, hipStream_t s) {
    if (p.col_waves == 8) launch<DT, D, IO, 2, 8>(p, s);
    else if (ct == 2) launch<DT, D, IO, 2, 4>(p, s);
    else launch<DT, D, IO, 1, 4>(p, s);
}

}  // namespace

#define TREE_LAUNCH_(name, dt, d)                                            \
    void name(const TreeParams& p, int32_t io, uint32_t ct, hipStream_t s) { \
        if (io == VSPEC_KV_F32) launch_any<dt, d, float>(p, ct, s);          \
        else launch_any<dt, d, _Float16>(p, ct, s);                          \
    }
#if VSPEC_HEAD_DIM == 64
TREE_LAUNCH_(launch_tree_wide_f16_d64, VSPEC_KV_F16, 64)
TREE_LAUNCH_(launch_tree_wide_int4_d64, VSPEC_KV_INT4, 64)
#else
TREE_LAUNCH_(launch_tree_wide_f16_d128, VSPEC_KV_F16, 128)
TREE_LAUNCH_(launch_tree_wide_int4_d128, VSPEC_KV_INT4, 128)
#endif
#undef TREE_LAUNCH_

}  // namespace vkv
