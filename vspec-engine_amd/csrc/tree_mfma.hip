// tree_mfma.hip -- attention of a drafted tree over the paged cache on the matrix cores.
//
// The C = nodes * group query rows that share a kv head are columns; 16 of them are a column
// tile.  A wave holds CT column tiles and goes over its share of the tokens once, a step of 32
// (f32 pools 16) tokens at a time, with the running maximum and sum of an online softmax:
//   S^T[16 tok][16 col] = K[16 tok][D] x Q^T     A = K rows as loaded, B = q
//   O^T[d][16 col]     += V^T[d][tok] x P^T      A = V as loaded, B = p, straight from the S^T
//                                                accumulators: lane (g, n) holds tokens 4g..4g+3
//                                                of column n in both
// so neither scores nor weights pass through LDS.  f16 and int4 pools use 16x16x32 f16 MFMAs
// (the 8 tokens of a lane in a step are tokens 4g..4g+3 of two tiles), f32 pools 16x16x4 f32.
//
// Precision.  f32 rows (IO = float) keep 22 bits of q, p and an int4 pool's keys and values, each
// split in two f16 (hi + lo).  f16 rows are exact in f16 and come out rounded to it, 2.1e-4 of the
// output's norm; one more rounding of each weight (f16 pools) makes that 2.5e-4 to 2.9e-4.  Of int4
// pools, rounding weights, keys (a code times a scale has 15 bits) and values once each would make
// it 3.7e-4, so there keys and weights keep their low parts, 2.7e-4, for 10 % of the time of few
// nodes and 30 % of 64 nodes' (64 x 4097 tokens: 4 nodes 118 -> 134, 8 160 -> 177, 64 550 -> 715
// us).  Sums are f32.  p is
// scaled by 2^kHeadroom against the reference point of the softmax, which follows the maximum
// only when that has grown by 2^8, so p <= 2^11 fits f16 and weights down to 2^-27 of the
// largest count.
//
// The clip of every key to its own standard deviation is screened as in the decode
// (decode_mfma.hip); the keys of a tile that it may reach are multiplied again, clipped, in two
// f16 parts.
//
// Work: a row of the grid is a sequence or a part of one (tree_job), a workgroup takes it for one
// kv head and group of column tiles.  Its waves are col_waves side by side over columns, times
// 4 / col_waves over steps, joined through LDS; a second launch joins the parts of a sequence.
//
// Waits.  K's registers take the next step's rows as soon as the scores are there, V's at the end
// of the step, and a second workgroup on the CU fills what is left (tree_cu_groups).  With a whole
// step ahead in registers and one workgroup, 64 x 4097 tokens of an int4 pool, 4 nodes of 4 query
// heads, took 154 us; this took 115 (134 now that their weights and keys have low parts).
//
// What bounds it (GQA 32 / 8, D = 128).  f16 pools: reading them, 64 x 4097 tokens and 4 nodes in
// 190 us, 5.7 TB/s.  int4 pools: the vector instructions that turn codes into f16 and screen the
// keys, 2.3 TB/s there (134 us).  Short sequences: the chain of lengths, table, tile and join, and the
// fetch of the code itself, 11 to 13 us for one sequence of 100 to 3000 tokens.
#include <type_traits>

#include "tree_common.h"

namespace vkv {
namespace {

// A 16-token tile as loaded: lane (g, n) holds K elements of token n and V elements of tokens
// 4g..4g+3.
template <int DT, int D>
struct Tile;
template <int D>
struct Tile<VSPEC_KV_F16, D> {
    uint4 k[D / 32];  // d = 32i + 8g .. +7
    uint4 v[D / 32];  // d = 32i + 2n (first 8 bytes, 4 tokens) and d + 1
};
template <int D>
struct Tile<VSPEC_KV_INT4, D> {
    uint32_t k[D / 32];       // code dwords g*D/32 + i: one group's
    uint32_t v[D / 32];       // lane chunk (g, n)
    uint32_t vs[D / 16];      // scales of tokens 4g..4g+3, D/32 halves each
    uint32_t ks;              // scale of token n and the lane's group
};
template <int D>
struct Tile<VSPEC_KV_F32, D> {
    float k[D / 4];           // d = 16i + 4g .. +3
    float v[4][D / 16];       // token 4g + r, d = 64i + 4n .. +3
};

template <int DT, int D, typename IO, int CT>
__global__ __launch_bounds__(256, tree_cu_groups(DT, D, sizeof(IO) == 4, CT)) void tree_attention(TreeParams p) {
    constexpr bool F32 = DT == VSPEC_KV_F32;
    constexpr bool SPLIT = sizeof(IO) == 4 && !F32;      // q in two f16 parts
    constexpr bool KLO = DT == VSPEC_KV_INT4;            // K in two f16 parts
    constexpr bool PLO = SPLIT || DT == VSPEC_KV_INT4;   // p in two f16 parts
    constexpr bool VLO = SPLIT && DT == VSPEC_KV_INT4;   // V in two f16 parts
    constexpr int NT = tree_step_tiles(DT);
    constexpr int NQ = D / 32;   // f16 score MFMAs of a tile
    constexpr int NDT = D / 16;  // d-tiles of the output
    typedef Tile<DT, D> T;
    __shared__ uint64_t bits_sh[64];
    __shared__ f4_t red[CT][4][NDT][64];
    __shared__ float red_ml[CT][4][16][2];

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, n = lane & 15;
    const int token_waves = 4 / (int)p.col_waves;
    const int cw = wave / token_waves, tw = wave - cw * token_waves;

    const TreeJob job = tree_job<NT>(p, (int)blockIdx.y, token_waves);
    if (job.b < 0) return;
    const uint32_t b = (uint32_t)job.b, item = blockIdx.x;
    const uint32_t cg = (uint32_t)uniform((int)(item / p.hkv)), h = item - cg * p.hkv;
    const TreeSpan sp = job.span;
    const TreeSteps tp = tree_steps<NT>(sp);
    const int lo = job.lo, hi = job.hi;

    if (threadIdx.x < p.nodes) bits_sh[threadIdx.x] = tree_bits(p, b, threadIdx.x, sp.len);

    // ---- q: columns of this wave, on their way before K and V (loads come back in order) ----
    // Column c is node c / group, head c % group of the kv head's.
    const int cols = (int)(p.nodes * p.group);
    const int ctile0 = ((int)cg * (int)p.col_waves + cw) * CT;
    typedef IO raw_t __attribute__((ext_vector_type(4)));
    raw_t raw[CT][D / 16];
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
        for (int u = 0; u < D / 16; ++u) {
            // four adjacent elements: of the lane's 8 of k-step u / 2 (f16: 32i + 8g, int4: 8 (g NQ + i)), or f32's 16u + 4g
            const int d = F32 ? 16 * u + 4 * g : (DT == VSPEC_KV_F16 ? 32 * (u / 2) + 8 * g : 8 * (g * NQ + u / 2)) + 4 * (u % 2);
            raw[ct][u] = *reinterpret_cast<const raw_t*>(src + d);
        }
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

    // ---- tiles ----
    // The tiles of this wave's next 64 / NT steps, a lane each: where a tile lies (token index in the pool), its
    // slot in the block and how many tokens it holds (0: its loads read block 0).
    auto first_tile = [&](const int step) { return step < tp.prefix_steps ? NT * step : tp.prefix_tiles + NT * (step - tp.prefix_steps); };
    size_t t_token = 0;
    int t_info = 0;  // slot0 << 5 | tokens
    auto look_up = [&](const int first) {
        const int step = first + lane / NT * token_waves, tile = first_tile(step) + lane % NT;
        const bool in = step < hi && tile < (step < tp.prefix_steps ? tp.prefix_tiles : tp.tiles);
        const int row = in ? tree_block_of(magic, shift, tile) : 0;
        const int entry = tables[row];
        const int room = used ? used[row] : P;
        const bool ok = in && entry >= 0 && (uint32_t)entry < num_blocks;
        const int slot0 = ok ? tile * kTile - row * P : 0;
        t_token = ((size_t)(ok ? entry : 0) * hkv + h) * P + slot0;
        t_info = slot0 << 5 | (ok ? min(min(kTile, sp.end - tile * kTile), max(0, room - slot0)) : 0);
    };
    auto load_k = [&](const size_t token, const int slot0, T& f) {
        if constexpr (DT == VSPEC_KV_F16) {
            const uint4* kr = reinterpret_cast<const uint4*>(reinterpret_cast<const _Float16*>(kdata) + (token + n) * D + 8 * g);
#pragma unroll
            for (int i = 0; i < D / 32; ++i) f.k[i] = kr[4 * i];
        } else if constexpr (DT == VSPEC_KV_INT4) {
            const uint32_t* kr = reinterpret_cast<const uint32_t*>(kdata + (token + n) * (D / 2)) + g * NQ;
            if constexpr (NQ == 4) {
                const uint4 a = *reinterpret_cast<const uint4*>(kr);
                f.k[0] = a.x, f.k[1] = a.y, f.k[2] = a.z, f.k[3] = a.w;
            } else {
                const uint2 a = *reinterpret_cast<const uint2*>(kr);
                f.k[0] = a.x, f.k[1] = a.y;
            }
            f.ks = kscales[(token - slot0) * NQ + (size_t)((g * NQ) / 4) * P + slot0 + n];
        } else {
            const float* kr = reinterpret_cast<const float*>(kdata) + (token + n) * D + 4 * g;
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
                const float4 w = *reinterpret_cast<const float4*>(kr + 16 * i);
                f.k[4 * i] = w.x, f.k[4 * i + 1] = w.y, f.k[4 * i + 2] = w.z, f.k[4 * i + 3] = w.w;
            }
        }
    };
    auto load_v = [&](const size_t token, T& f) {
        if constexpr (DT == VSPEC_KV_F16) {
            const uint4* vr = reinterpret_cast<const uint4*>(reinterpret_cast<const _Float16*>(vdata) + token * D + g * 4 * D + 8 * n);
#pragma unroll
            for (int i = 0; i < D / 32; ++i) f.v[i] = vr[16 * i];
        } else if constexpr (DT == VSPEC_KV_INT4) {
            const uint32_t* vr = reinterpret_cast<const uint32_t*>(vdata + token * (D / 2)) + (16 * g + n) * NQ;
            const uint4* vs = reinterpret_cast<const uint4*>(vscales + (token + 4 * g) * NQ);
            if constexpr (NQ == 4) {
                const uint4 c = *reinterpret_cast<const uint4*>(vr);
                f.v[0] = c.x, f.v[1] = c.y, f.v[2] = c.z, f.v[3] = c.w;
            } else {
                const uint2 c = *reinterpret_cast<const uint2*>(vr);
                f.v[0] = c.x, f.v[1] = c.y;
            }
#pragma unroll
            for (int i = 0; i < D / 64; ++i) {
                const uint4 w = vs[i];
                f.vs[4 * i] = w.x, f.vs[4 * i + 1] = w.y, f.vs[4 * i + 2] = w.z, f.vs[4 * i + 3] = w.w;
            }
        } else {
            const float* vr = reinterpret_cast<const float*>(vdata) + (token + 4 * g) * D + 4 * n;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
#pragma unroll
                for (int i = 0; i < D / 64; ++i) {
                    const float4 w = *reinterpret_cast<const float4*>(vr + (size_t)r * D + 64 * i);
                    f.v[r][4 * i] = w.x, f.v[r][4 * i + 1] = w.y, f.v[r][4 * i + 2] = w.z, f.v[r][4 * i + 3] = w.w;
                }
            }
        }
    };
    struct Where {
        size_t token[NT];
        int slot0[NT], valid[NT];
    };
    int at_lane = 0;  // of the next step's first tile in the table
    auto where = [&](const int step, Where& w) {
        if (at_lane == 64) {
            look_up(step);
            at_lane = 0;
        }
#pragma unroll
        for (int a = 0; a < NT; ++a) {
            const uint32_t t0 = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)t_token, at_lane + a);
            const uint32_t t1 = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(t_token >> 32), at_lane + a);
            const int info = __builtin_amdgcn_readlane(t_info, at_lane + a);
            w.token[a] = (size_t)t1 << 32 | t0;
            w.slot0[a] = info >> 5;
            w.valid[a] = info & 31;
        }
        at_lane += NT;
    };

    Where now;
    T tile[NT];
    int step = lo + tw;
    look_up(step);
    where(step, now);
#pragma unroll
    for (int a = 0; a < NT; ++a) {
        load_k(now.token[a], now.slot0[a], tile[a]);
        load_v(now.token[a], tile[a]);
    }

    // The operands of q hold clip(q) 2^e (e != 0 only for f32 rows outside f16's range,
    // qnorm_shift); scores come out in that unit and fac takes them to log2 units.
    h8_t qh[F32 ? 1 : CT][NQ], ql[SPLIT ? CT : 1][NQ];
    float qf[F32 ? CT : 1][F32 ? D / 4 : 1];
    float fac[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
        constexpr int E = D / 4;
        float x[E];
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = (float)raw[ct][e / 4][e % 4];
        float sum = 0.f, var = 0.f, am = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            x[e] = live[ct] ? x[e] : 0.f;
            sum += x[e];
        }
        sum = add_rows(sum);
        const float mean = sum * (1.0f / D);
#pragma unroll
        for (int e = 0; e < E; ++e) var = fmaf(x[e] - mean, x[e] - mean, var);
        const float th = fminf(fmaxf(1e-6f, alpha * sqrtf(add_rows(var) * (1.0f / D))), input_clip);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            x[e] = fminf(fmaxf(x[e], -th), th);
            am = fmaxf(am, fabsf(x[e]));
        }
        int ex = 0;
        if constexpr (SPLIT) ex = qnorm_shift(max_rows(am));
        fac[ct] = sum != sum ? sum : p.scale * pow2i(-ex);  // (a row with NaN gives NaN: the clips would hide it)
        const float up = pow2i(ex);
        if constexpr (F32) {
#pragma unroll
            for (int e = 0; e < E; ++e) qf[ct][e] = x[e];
        } else {
#pragma unroll
            for (int k = 0; k < NQ; ++k) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    // int4: halves 2m, 2m + 1 are nibbles m, m + 4
                    const float y = x[8 * k + (DT == VSPEC_KV_INT4 ? e / 2 + 4 * (e % 2) : e)] * up;
                    const _Float16 hi16 = (_Float16)y;
                    qh[ct][k][e] = hi16;
                    if constexpr (SPLIT) ql[ct][k][e] = (_Float16)(y - (float)hi16);
                }
            }
        }
    }

    // ---- state of every column: reference point mf (log2 units), the score that moves it, sum, output ----
    f4_t acc[CT][NDT];
    float limit[CT], mf[CT], l[CT];
    float clip[CT];  // of scores
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
        limit[ct] = -INFINITY;
        clip[ct] = p.logit_clip / fac[ct];
        mf[ct] = -1e30f;
        l[ct] = 0.f;
#pragma unroll
        for (int j = 0; j < NDT; ++j) acc[ct][j] = f4_t{0.f, 0.f, 0.f, 0.f};
    }

    auto sees = [&](const int ct, const int tile, const int valid) -> uint32_t {
        const int j0 = tile * kTile + 4 * g - sp.start;  // the node that the lane's first token is
        const uint64_t mine = bits_sh[node[ct]];
        const uint32_t seen = j0 <= -4 ? 15u
                              : j0 < 0 ? (uint32_t)(mine << -j0) | ((1u << -j0) - 1u)
                              : j0 < 64 ? (uint32_t)(mine >> j0) : 0u;
        const int left = valid - 4 * g;
        return seen & (left >= 4 ? 15u : left > 0 ? (1u << left) - 1u : 0u);
    };
    bool wild = false;  // V held what is not finite, among nodes
    __syncthreads();    // (bits_sh)

    // K's registers take the next step's as soon as the scores are there, V's at the end.
    auto process = [&](const int step, const Where& s, const Where& next) {
        // a tile that holds nodes or fewer than 16 tokens
        const bool masked = step >= tp.prefix_steps || s.valid[0] < kTile || s.valid[NT - 1] < kTile;
        const int tile0 = first_tile(step);
        // ---- K operands, each key held to its own limit ----
        h8_t kh[F32 ? 1 : NT][NQ], kl[SPLIT || KLO ? NT : 1][NQ];
        bool low[NT];    // kl holds something
        float kunit[NT]; // scores come out divided by this
        bool nans[NT];   // a key may be NaN
#pragma unroll
        for (int a = 0; a < NT; ++a) {
            T& t = tile[a];
            low[a] = KLO;
            kunit[a] = 1.f;
            nans[a] = F32;
            if constexpr (F32) {
                // two passes over the row in registers, and the clip itself
                float sum = 0.f, var = 0.f;
#pragma unroll
                for (int e = 0; e < D / 4; ++e) sum += t.k[e];
                const float mean = add_rows(sum) * (1.0f / D);
#pragma unroll
                for (int e = 0; e < D / 4; ++e) var = fmaf(t.k[e] - mean, t.k[e] - mean, var);
                const float th = fminf(fmaxf(1e-6f, alpha * sqrtf(add_rows(var) * (1.0f / D))), input_clip);
#pragma unroll
                for (int e = 0; e < D / 4; ++e) t.k[e] = t.k[e] != t.k[e] ? t.k[e] : __builtin_amdgcn_fmed3f(t.k[e], -th, th);
            } else {
                float s1 = 0.f, s2 = 0.f, mx;
                bool large = false;
                if constexpr (DT == VSPEC_KV_F16) {
                    const h2_t ones = {(_Float16)1.0f, (_Float16)1.0f};
                    h2_t mx2 = {(_Float16)0.f, (_Float16)0.f};
#pragma unroll
                    for (int i = 0; i < NQ; ++i) {
                        kh[a][i] = __builtin_bit_cast(h8_t, t.k[i]);
                        const uint32_t w4[4] = {t.k[i].x, t.k[i].y, t.k[i].z, t.k[i].w};
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            const h2_t y = __builtin_bit_cast(h2_t, w4[c]);
                            s1 = __builtin_amdgcn_fdot2(y, ones, s1, false);
                            s2 = __builtin_amdgcn_fdot2(y, y, s2, false);
                            mx2 = __builtin_elementwise_max(mx2, __builtin_elementwise_abs(y));
                        }
                    }
                    mx = fmaxf((float)mx2[0], (float)mx2[1]);
                } else {
                    const float sc = half_bits_to_float(t.ks);
                    // a code times a scale past 7500 may pass f16's range: the tile's scales drop by 2^4
                    large = __builtin_amdgcn_ballot_w64(n < s.valid[a] && fabsf(sc) > 7500.f) != 0;
                    _Float16 s16 = __builtin_bit_cast(_Float16, (uint16_t)t.ks);
                    if (large) {
                        s16 *= (_Float16)0.0625f;
                        kunit[a] = 16.f;
                    }
                    const h2_t s2v = {s16, s16};
                    int c1 = 0, c2 = 0;
#pragma unroll
                    for (int i = 0; i < NQ; ++i) {
                        c1 = __builtin_amdgcn_sdot8((int)t.k[i], 0x11111111, c1, false);
                        c2 = __builtin_amdgcn_sdot8((int)t.k[i], (int)t.k[i], c2, false);
                        h2_t q4[4];
                        codes_to_f16(t.k[i], q4);
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            const h2_t y = q4[c] * s2v;
                            kh[a][i][2 * c] = y[0];
                            kh[a][i][2 * c + 1] = y[1];
                            if constexpr (KLO) {
                                const h2_t z = __builtin_elementwise_fma(q4[c], s2v, -y);  // exact
                                kl[a][i][2 * c] = z[0];
                                kl[a][i][2 * c + 1] = z[1];
                            }
                        }
                    }
                    s1 = sc * (float)c1;
                    s2 = sc * sc * (float)c2;
                    mx = 8.0f * fabsf(sc);
                }
                s1 = add_rows(s1);
                s2 = add_rows(s2);
                const float mean1 = s1 * (1.0f / D), ex2 = s2 * (1.0f / D);
                const float var1 = ex2 - mean1 * mean1;
                const float th1 = fminf(fmaxf(1e-6f, alpha * __builtin_amdgcn_sqrtf(fmaxf(var1, 0.f))), input_clip);
                // the margins of the decode's screen; !(<=) also takes what is not finite
                const bool flag = !(mx <= th1 * (1.0f - 0.0009765625f)) || var1 <= ex2 * 0.0009765625f;
                const uint64_t any = __builtin_amdgcn_ballot_w64(flag && n < s.valid[a]);
                if (any != 0) {
                    // the flagged keys (any lane of token n flags it), exactly: two-pass deviation, and the clipped row
                    // in two f16 parts.  Elements inside the limit stay exact, the limit keeps 22 bits or 2^-25.
                    nans[a] = true;
                    low[a] = SPLIT || KLO;
                    const bool mine = ((any | (any >> 16) | (any >> 32) | (any >> 48)) >> n) & 1u;
                    float x[8 * NQ], sum = 0.f, var = 0.f;
#pragma unroll
                    for (int i = 0; i < NQ; ++i) {
                        if constexpr (DT == VSPEC_KV_F16) {
                            const h8_t w = __builtin_bit_cast(h8_t, t.k[i]);
#pragma unroll
                            for (int e = 0; e < 8; ++e) x[8 * i + e] = (float)w[e];
                        } else {
                            h2_t q4[4];
                            codes_to_f16(t.k[i], q4);
#pragma unroll
                            for (int e = 0; e < 8; ++e) x[8 * i + e] = (float)q4[e / 2][e % 2] * half_bits_to_float(t.ks);
                        }
#pragma unroll
                        for (int e = 0; e < 8; ++e) sum += x[8 * i + e];
                    }
                    const float mean = add_rows(sum) * (1.0f / D);
#pragma unroll
                    for (int e = 0; e < 8 * NQ; ++e) var = fmaf(x[e] - mean, x[e] - mean, var);
                    const float th = fminf(fmaxf(1e-6f, alpha * sqrtf(add_rows(var) * (1.0f / D))), input_clip);
                    const float down = large ? 0.0625f : 1.f;
#pragma unroll
                    for (int i = 0; i < NQ; ++i) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            float y = x[8 * i + e];
                            y = (y != y ? y : __builtin_amdgcn_fmed3f(y, -th, th)) * down;
                            const _Float16 y16 = (_Float16)y;
                            kh[a][i][e] = mine ? y16 : kh[a][i][e];
                            if constexpr (SPLIT || KLO) {
                                const _Float16 z16 = (_Float16)(y - (float)y16);
                                kl[a][i][e] = mine ? z16 : KLO ? kl[a][i][e] : (_Float16)0.f;
                            }
                        }
                    }
                }
            }
        }

        // ---- scores ----
        f4_t sc[CT][NT];
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
#pragma unroll
            for (int a = 0; a < NT; ++a) {
                f4_t c = {0.f, 0.f, 0.f, 0.f};
                if constexpr (F32) {
#pragma unroll
                    for (int e = 0; e < D / 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(tile[a].k[e], qf[ct][e], c, 0, 0, 0);
                } else {
                    if constexpr (SPLIT) {
#pragma unroll
                        for (int i = 0; i < NQ; ++i) c = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh[a][i], ql[ct][i], c, 0, 0, 0);
                    }
                    if constexpr (KLO) {
#pragma unroll
                        for (int i = 0; i < NQ; ++i) c = __builtin_amdgcn_mfma_f32_16x16x32_f16(kl[a][i], qh[ct][i], c, 0, 0, 0);
                    }
#pragma unroll
                    for (int i = 0; i < NQ; ++i) c = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh[a][i], qh[ct][i], c, 0, 0, 0);
                }
                sc[ct][a] = c;
            }
        }
        if constexpr (SPLIT && !KLO) {
#pragma unroll
            for (int a = 0; a < NT; ++a) {
                if (!low[a]) continue;
#pragma unroll
                for (int ct = 0; ct < CT; ++ct) {
#pragma unroll
                    for (int i = 0; i < NQ; ++i) sc[ct][a] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kl[a][i], qh[ct][i], sc[ct][a], 0, 0, 0);
                }
            }
        }
        settle();
#pragma unroll
        for (int a = 0; a < NT; ++a) load_k(next.token[a], next.slot0[a], tile[a]);
        if constexpr (DT == VSPEC_KV_INT4) {
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) {
#pragma unroll
                for (int a = 0; a < NT; ++a) sc[ct][a] *= kunit[a];
            }
        }

        // ---- softmax of column n over the lane's tokens ----
        if (masked || nans[0] || nans[NT - 1]) {
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) {
#pragma unroll
                for (int a = 0; a < NT; ++a) {
                    const uint32_t seen = sees(ct, tile0 + a, s.valid[a]);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        float x = sc[ct][a][r];
                        // (a key with NaN is always flagged; the median would hide it)
                        x = x != x ? x : __builtin_amdgcn_fmed3f(x, -clip[ct], clip[ct]);
                        sc[ct][a][r] = (seen >> r) & 1u ? x : -INFINITY;
                    }
                }
            }
        } else {
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) {
#pragma unroll
                for (int a = 0; a < NT; ++a) {
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
            for (int a = 0; a < NT; ++a) top[ct] = fmaxf(top[ct], fmaxf(fmaxf(sc[ct][a][0], sc[ct][a][1]), fmaxf(sc[ct][a][2], sc[ct][a][3])));
            grown = grown || top[ct] > limit[ct];
        }
        if (__builtin_amdgcn_ballot_w64(grown) != 0) {
            settle();  // (the outputs of the step before)
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) {
                const float mt = max_rows(top[ct]);
                const bool need = mt > limit[ct];
                const float nf = fmaf(mt, fac[ct], -kHeadroom);
                const float f = need ? __builtin_amdgcn_exp2f(mf[ct] - nf) : 1.0f;
                limit[ct] = need ? mt + kThreshold / fac[ct] : limit[ct];
                mf[ct] = need ? nf : mf[ct];
                l[ct] *= f;
#pragma unroll
                for (int j = 0; j < NDT; ++j) acc[ct][j] *= f;
            }
        }
        h8_t ph[F32 ? 1 : CT], pl[PLO ? CT : 1];
        float pf[F32 ? CT : 1][4];
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
#pragma unroll
            for (int e = 0; e < 4 * NT; ++e) {
                const float w = __builtin_amdgcn_exp2f(fmaf(sc[ct][e / 4][e % 4], fac[ct], -mf[ct]));
                l[ct] += w;
                if constexpr (F32) {
                    pf[ct][e] = w;
                } else {
                    const _Float16 w16 = (_Float16)w;
                    ph[ct][e] = w16;
                    if constexpr (PLO) pl[ct][e] = (_Float16)(w - (float)w16);
                }
            }
        }

        // ---- V operands, O^T += V^T P^T ----
        // Slots without a token may hold any bits and become zeros.  In tiles that hold nodes so do values
        // that are not finite: in the products 0 * inf would reach the rows that do not see them.
        bool tree[NT];
#pragma unroll
        for (int a = 0; a < NT; ++a) tree[a] = (tile0 + a) * kTile + s.valid[a] > sp.start;
        if constexpr (F32) {
            if (masked) {
                bool mine = false;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const bool held = 4 * g + r < s.valid[0];
#pragma unroll
                    for (int j = 0; j < NDT; ++j) {
                        const bool out = tree[0] && !(fabsf(tile[0].v[r][j]) < INFINITY);
                        mine = mine || (held && out);
                        tile[0].v[r][j] = held && !out ? tile[0].v[r][j] : 0.f;
                    }
                }
                wild = wild || __builtin_amdgcn_ballot_w64(mine) != 0;
            }
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) {
#pragma unroll
                for (int j = 0; j < NDT; ++j) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[ct][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(tile[0].v[r][j], pf[ct][r], acc[ct][j], 0, 0, 0);
                }
            }
        } else {
            // acc += V^T p of d-tile j
            auto add_values = [&](const int j, const h8_t v, const h8_t vl, const h8_t (&ph)[CT], const h8_t (&pl)[PLO ? CT : 1]) {
#pragma unroll
                for (int ct = 0; ct < CT; ++ct) {
                    acc[ct][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, ph[ct], acc[ct][j], 0, 0, 0);
                    if constexpr (PLO) acc[ct][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pl[ct], acc[ct][j], 0, 0, 0);
                    if constexpr (VLO) acc[ct][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vl, ph[ct], acc[ct][j], 0, 0, 0);
                }
            };
            if constexpr (DT == VSPEC_KV_INT4) {
                // word c of the lane's chunks at a time: values of d-tiles 2c and 2c + 1.  In the products of scales of 2^12
                // and more (LARGE: of no others) a code may pass f16's range: they are left for a pass of their own, over 2^4,
                // with p 2^4 (p <= 2^11).
                auto values = [&](auto large_tag, const h8_t (&ph)[CT], const h8_t (&pl)[PLO ? CT : 1]) -> bool {
                    constexpr bool LARGE = decltype(large_tag)::value;
                    bool mine_big = false, mine = false;
#pragma unroll
                    for (int c = 0; c < NQ; ++c) {
                        h4_t vh[NT][2], vl[NT][2];
#pragma unroll
                        for (int a = 0; a < NT; ++a) {
                            h2_t sp2[2];
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                uint32_t w = int4_scale_pair<NQ>(tile[a], c, e);
                                if (s.valid[a] < kTile) {
                                    w &= (4 * g + 2 * e < s.valid[a] ? 0xffffu : 0u) | (4 * g + 2 * e + 1 < s.valid[a] ? 0xffff0000u : 0u);
                                }
                                const uint32_t lo16 = w & 0x7fffu, hi16 = (w >> 16) & 0x7fffu;
                                if constexpr (LARGE) {
                                    const bool l_in = lo16 >= kBigScale && (!tree[a] || lo16 < 0x7C00u), h_in = hi16 >= kBigScale && (!tree[a] || hi16 < 0x7C00u);
                                    w &= (l_in ? 0xffffu : 0u) | (h_in ? 0xffff0000u : 0u);
                                    const h2_t down = {(_Float16)0.0625f, (_Float16)0.0625f};
                                    sp2[e] = __builtin_bit_cast(h2_t, w) * down;
                                } else {
                                    mine_big = mine_big || max(lo16, hi16) >= kBigScale;
                                    mine = mine || (tree[a] && max(lo16, hi16) >= 0x7C00u);
                                    w &= (lo16 < kBigScale ? 0xffffu : 0u) | (hi16 < kBigScale ? 0xffff0000u : 0u);
                                    sp2[e] = __builtin_bit_cast(h2_t, w);
                                }
                            }
                            int4_values<VLO>(tile[a].v[c], sp2, vh[a][0], vh[a][1], vl[a][0], vl[a][1]);
                        }
#pragma unroll
                        for (int o = 0; o < 2; ++o) add_values(2 * c + o, join(vh[0][o], vh[NT - 1][o]), join(vl[0][o], vl[NT - 1][o]), ph, pl);
                    }
                    wild = wild || __builtin_amdgcn_ballot_w64(mine) != 0;
                    return __builtin_amdgcn_ballot_w64(mine_big) != 0;
                };
                if (values(std::false_type(), ph, pl)) {
                    const _Float16 up = (_Float16)16.f;
                    const h8_t up8 = {up, up, up, up, up, up, up, up};
                    h8_t ph16[CT], pl16[CT];
#pragma unroll
                    for (int ct = 0; ct < CT; ++ct) {
                        ph16[ct] = ph[ct] * up8;
                        pl16[ct] = pl[ct] * up8;
                    }
                    values(std::true_type(), ph16, pl16);
                }
            } else {
                h4_t vh[NT][NDT];
#pragma unroll
                for (int a = 0; a < NT; ++a) {
#pragma unroll
                    for (int i = 0; i < D / 32; ++i) {
                        vh[a][2 * i] = __builtin_bit_cast(h4_t, make_uint2(tile[a].v[i].x, tile[a].v[i].y));
                        vh[a][2 * i + 1] = __builtin_bit_cast(h4_t, make_uint2(tile[a].v[i].z, tile[a].v[i].w));
                    }
                    if (masked) {
                        bool mine = false;
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const bool held = 4 * g + r < s.valid[a];
#pragma unroll
                            for (int j = 0; j < NDT; ++j) {
                                const bool out = tree[a] && !(fabsf((float)vh[a][j][r]) < INFINITY);
                                mine = mine || (held && out);
                                vh[a][j][r] = held && !out ? vh[a][j][r] : (_Float16)0.f;
                            }
                        }
                        wild = wild || __builtin_amdgcn_ballot_w64(mine) != 0;
                    }
                }
#pragma unroll
                for (int j = 0; j < NDT; ++j) {
                    const h8_t v = join(vh[0][j], vh[NT - 1][j]);
                    add_values(j, v, v, ph, pl);
                }
            }
        }
#pragma unroll
        for (int a = 0; a < NT; ++a) load_v(next.token[a], tile[a]);
    };

    for (; step < hi; step += token_waves) {
        Where next;
        where(step + token_waves, next);
        process(step, now, next);
        now = next;
    }
    settle();
    if (wild) add_wild<DT, D, CT>(tables, used, num_blocks, hkv, h, P, magic, shift, sp, lane, first_tile(max(lo, tp.prefix_steps)), min(first_tile(hi), tp.tiles), sees, acc);

    // ---- join the token waves; the output, or the part's state ----
    const bool whole = job.count == 1;
    const int tiles = (int)p.col_waves * CT;
    const size_t slot = (size_t)(job.state + job.part) * (p.hkv * p.col_groups) + item;
    auto finish = [&](const int ct, const int j, f4_t a, const float sum, const float ref) {
        const int tile = cw * CT + ct;
        if (!whole) {
            reinterpret_cast<f4_t*>(p.part_acc)[((slot * tiles + tile) * NDT + j) * 64 + lane] = a;
            if (j == 0 && g == 0) {
                float* ml = p.part_ml + ((slot * tiles + tile) * 16 + n) * 2;
                ml[0] = ref;
                ml[1] = sum;
            }
            return;
        }
        const int c = (ctile0 + ct) * 16 + n;
        if (c >= cols) return;
        const int i = c / (int)p.group;
        IO* dst = reinterpret_cast<IO*>(p.out) + (((size_t)b * p.nodes + i) * p.hq + (size_t)h * p.group + (c - i * (int)p.group)) * D;
        const bool empty = i >= sp.len || sum == 0.f;
#pragma unroll
        for (int r = 0; r < 4; ++r) dst[out_dim<DT>(j, g, r)] = (IO)(empty ? 0.f : a[r] / sum);
    };
    float sum[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) sum[ct] = add_rows(l[ct]);
    if (token_waves == 1) {
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
#pragma unroll
            for (int j = 0; j < NDT; ++j) finish(ct, j, acc[ct][j], sum[ct], mf[ct]);
        }
        return;
    }
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
        if (g == 0) {
            red_ml[ct][wave][n][0] = mf[ct];
            red_ml[ct][wave][n][1] = sum[ct];
        }
#pragma unroll
        for (int j = 0; j < NDT; ++j) red[ct][wave][j][lane] = acc[ct][j];
    }
    __syncthreads();
#pragma unroll 1
    for (int k = tw; k < CT * NDT; k += token_waves) {
        const int ct = k / NDT, j = k - ct * NDT;
        float top = -INFINITY, total = 0.f;
        f4_t a = {0.f, 0.f, 0.f, 0.f};
        for (int t = 0; t < token_waves; ++t) top = fmaxf(top, red_ml[ct][cw * token_waves + t][n][0]);
        for (int t = 0; t < token_waves; ++t) {
            const float* ml = red_ml[ct][cw * token_waves + t][n];
            const float f = __builtin_amdgcn_exp2f(ml[0] - top);
            total = fmaf(ml[1], f, total);
            a += red[ct][cw * token_waves + t][j][lane] * f;
        }
        finish(ct, j, a, total, top);
    }
}

template <int DT, int D, typename IO>
void launch(const TreeParams& p, uint32_t ct, hipStream_t s) {
    const dim3 grid(p.hkv * p.col_groups, p.rows);
    switch (ct) {
        case 1: hipLaunchKernelGGL((tree_attention<DT, D, IO, 1>), grid, dim3(256), 0, s, p); break;
        default: hipLaunchKernelGGL((tree_attention<DT, D, IO, 2>), grid, dim3(256), 0, s, p); break;
    }
    if (p.slot_rows) launch_merge<DT, D, IO>(p, p.col_waves * ct, s);
}

}  // namespace

#define TREE_LAUNCH_(name, dt, d)                                                      \
    void name(const TreeParams& p, int32_t io, uint32_t ct, hipStream_t s) {           \
        if (io == VSPEC_KV_F32) launch<dt, d, float>(p, ct, s);                        \
        else launch<dt, d, _Float16>(p, ct, s);                                        \
    }
#if VSPEC_HEAD_DIM == 64
TREE_LAUNCH_(launch_tree_f32_d64, VSPEC_KV_F32, 64)
TREE_LAUNCH_(launch_tree_f16_d64, VSPEC_KV_F16, 64)
TREE_LAUNCH_(launch_tree_int4_d64, VSPEC_KV_INT4, 64)
#else
TREE_LAUNCH_(launch_tree_f32_d128, VSPEC_KV_F32, 128)
TREE_LAUNCH_(launch_tree_f16_d128, VSPEC_KV_F16, 128)
TREE_LAUNCH_(launch_tree_int4_d128, VSPEC_KV_INT4, 128)
#endif
#undef TREE_LAUNCH_

}  // namespace vkv
