// rope.hip -- rotary positions given for each token (vspec_rocm_rope).
//
// A pair (x1, x2) at position t turns by a = t f: (x1 cos a - x2 sin a, x1 sin a + x2 cos a).
// The angle is reduced in 64 bits: with f in turns a position, t f is off by 2^-53 of itself,
// 2^-33 turns at a million positions, and only its fraction goes on to the f32 sine and cosine
// (in half turns, sincospif, so that no multiple of pi has to be taken away).  Every angle of a
// token serves all its heads.
//
// What bounds it: reading and writing the rows, 16384 tokens of 40 heads, f16, D = 128, in 67 us,
// 5.0 TB/s, the rate of a large copy; 256 tokens 6 us, launch and waits.
#include <math.h>

#include "host.h"
#include "kv_common.h"

namespace vkv {
namespace {

constexpr uint32_t kMaxPairs = 128;

struct RopeOperand {
    const uint8_t* in;
    uint8_t* out;
    int64_t in_token, in_head, out_token, out_head;  // strides in elements
    uint32_t heads;
};

struct RopeParams {
    RopeOperand q, k;  // an absent operand has no heads
    const int32_t* positions;
    uint32_t tokens;
    uint32_t head_dim;
    uint32_t rope_dim;
    float magnitude;  // of cos and sin
    float sign;       // of sin
    double turns[kMaxPairs];  // turns a position
};

// The pair turned by t = (cos, sin), alike on every path: the sums are held in f32 (left to the compiler, some calls
// round them to f16 within the multiply-add and some after it).
__device__ __forceinline__ float2 turned(float x1, float x2, float2 t) {
    float y1 = fmaf(x1, t.x, -(x2 * t.y)), y2 = fmaf(x1, t.y, x2 * t.x);
    asm("" : "+v"(y1), "+v"(y2));
    return make_float2(y1, y2);
}

// Element by element: any alignment, strides and rope_dim.
template <typename T>
__global__ __launch_bounds__(256) void rope_rows(RopeParams p, bool interleaved) {
    __shared__ float2 cs[kMaxPairs];
    const uint32_t token = blockIdx.x;
    const uint32_t half = p.rope_dim / 2, rest = p.head_dim - p.rope_dim;
    if (threadIdx.x < half) {
        const double t = (double)p.positions[token] * p.turns[threadIdx.x];
        float s, c;
        sincospif(2.0f * (float)(t - rint(t)), &s, &c);
        cs[threadIdx.x] = make_float2(p.magnitude * c, p.sign * p.magnitude * s);
    }
    __syncthreads();
    const uint32_t units = half + rest;  // a row's pairs and its other elements
    for (uint32_t i = threadIdx.x; i < (p.q.heads + p.k.heads) * units; i += 256) {
        uint32_t h = i / units;
        const uint32_t u = i - h * units;
        const bool isk = h >= p.q.heads;
        h -= isk ? p.q.heads : 0u;
        const RopeOperand& o = isk ? p.k : p.q;
        const T* in = reinterpret_cast<const T*>(o.in) + (int64_t)token * o.in_token + (int64_t)h * o.in_head;
        T* out = reinterpret_cast<T*>(o.out) + (int64_t)token * o.out_token + (int64_t)h * o.out_head;
        if (u >= half) {
            out[half + u] = in[half + u];
            continue;
        }
        const uint32_t e1 = interleaved ? 2 * u : u, e2 = interleaved ? 2 * u + 1 : u + half;
        const float x1 = (float)in[e1], x2 = (float)in[e2];
        const float2 t = cs[u];
        const float2 y = turned(x1, x2, t);
        out[e1] = (T)y.x;
        out[e2] = (T)y.y;
    }
}

// The same where every row is whole 16-byte chunks of V elements: a unit is the two chunks whose elements pair up (half
// layout), the chunk that holds its pairs (interleaved), or a chunk past rope_dim, which is copied.
struct RopeSplit {
    uint32_t tokens;                  // of a workgroup
    uint32_t turning, units;          // units of a row that turn, all of them
    uint32_t half_magic, units_magic, rows_magic;  // chunk_div of rope_dim / 2, units, heads of q and k
};
constexpr uint32_t kChunkTokens = 4, kChunkHeads = 8192;  // (as many rows as chunk_div divides)

// x / d for x below 2^32 / d, with magic = ceil(2^32 / d) (0 for d = 1): x magic is above x 2^32 / d by less than x,
// that is, less than the 2^32 / d that the fraction leaves.
__device__ __forceinline__ uint32_t chunk_div(uint32_t x, uint32_t magic) { return magic ? __umulhi(x, magic) : x; }
uint32_t chunk_magic(uint32_t d) { return d == 1 ? 0u : (uint32_t)(((1ull << 32) + d - 1) / d); }

template <typename T, bool INTER>
__global__ __launch_bounds__(256) void rope_chunks(RopeParams p, RopeSplit w) {
    constexpr int V = 16 / sizeof(T);
    struct __align__(16) Chunk {
        T x[V];
    };
    __shared__ __align__(16) float2 cs[kChunkTokens][kMaxPairs];
    const uint32_t token0 = blockIdx.x * w.tokens, tokens = min(w.tokens, p.tokens - token0);
    const uint32_t half = p.rope_dim / 2;
    for (uint32_t i = threadIdx.x; i < tokens * half; i += 256) {
        const uint32_t at = chunk_div(i, w.half_magic), u = i - at * half;
        const double t = (double)p.positions[token0 + at] * p.turns[u];
        float s, c;
        sincospif(2.0f * (float)(t - rint(t)), &s, &c);
        cs[at][u] = make_float2(p.magnitude * c, p.sign * p.magnitude * s);
    }
    __syncthreads();
    const uint32_t rows = p.q.heads + p.k.heads, all = tokens * rows * w.units;
    constexpr int kBatch = 4;  // units of a thread whose loads are on their way
    for (uint32_t base = threadIdx.x; base < all; base += 256 * kBatch) {
        Chunk a[kBatch], b[INTER ? 1 : kBatch];
        T* out[kBatch];
        uint32_t at[kBatch], unit[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const uint32_t idx = min(base + 256 * i, all - 1);
            const uint32_t r = chunk_div(idx, w.units_magic), u = idx - r * w.units;
            at[i] = chunk_div(r, w.rows_magic);
            unit[i] = u;
            uint32_t h = r - at[i] * rows;
            const bool isk = h >= p.q.heads;
            h -= isk ? p.q.heads : 0u;
            const RopeOperand& o = isk ? p.k : p.q;
            const int64_t token = token0 + at[i];
            const uint32_t e = u < w.turning ? V * u : p.rope_dim + V * (u - w.turning);
            const T* in = reinterpret_cast<const T*>(o.in) + token * o.in_token + (int64_t)h * o.in_head + e;
            out[i] = reinterpret_cast<T*>(o.out) + token * o.out_token + (int64_t)h * o.out_head + e;
            a[i] = *reinterpret_cast<const Chunk*>(in);
            if constexpr (!INTER) b[i] = u < w.turning ? *reinterpret_cast<const Chunk*>(in + half) : a[i];
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            if (base + 256 * i >= all) continue;
            if (unit[i] < w.turning) {
                if constexpr (INTER) {
                    const float2* t = cs[at[i]] + V / 2 * unit[i];
#pragma unroll
                    for (int e = 0; e < V; e += 2) {
                        const float x1 = (float)a[i].x[e], x2 = (float)a[i].x[e + 1];
                        const float2 y = turned(x1, x2, t[e / 2]);
                        a[i].x[e] = (T)y.x;
                        a[i].x[e + 1] = (T)y.y;
                    }
                } else {
                    const float2* t = cs[at[i]] + V * unit[i];
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        const float x1 = (float)a[i].x[e], x2 = (float)b[i].x[e];
                        const float2 y = turned(x1, x2, t[e]);
                        a[i].x[e] = (T)y.x;
                        b[i].x[e] = (T)y.y;
                    }
                    *reinterpret_cast<Chunk*>(out[i] + half) = b[i];
                }
            }
            *reinterpret_cast<Chunk*>(out[i]) = a[i];
        }
    }
}

// Turns a position of every pair, and the factor on cosine and sine; 0 with an error.
int rope_turns(const VspecRopeDesc* d, double* turns, float* magnitude) {
    const double r = d->rope_dim;
    double base = d->base, m = 1.0;
    if (!(base > 1.0) || !isfinite(base)) {
        host_error("rope: base must be above 1");
        return 0;
    }
    if (d->scaling < VSPEC_ROPE_SCALE_NONE || d->scaling > VSPEC_ROPE_SCALE_YARN) {
        host_error("rope: bad scaling %d", (int)d->scaling);
        return 0;
    }
    const bool ranged = d->scaling == VSPEC_ROPE_SCALE_BANDS || d->scaling == VSPEC_ROPE_SCALE_YARN;
    if (d->scaling != VSPEC_ROPE_SCALE_NONE && (!(d->factor >= 1.0) || !isfinite(d->factor))) {
        host_error("rope: factor must be at least 1");
        return 0;
    }
    if (ranged && (d->trained_len == 0 || !(d->low > 0.0) || !(d->high > d->low) || !isfinite(d->high))) {
        host_error("rope: bands and yarn need trained_len and 0 < low < high");
        return 0;
    }
    if (d->scaling == VSPEC_ROPE_SCALE_BASE && d->rope_dim > 2) base *= pow(d->factor, r / (r - 2.0));
    const double two_pi = 6.283185307179586476925286766559;
    double first = 0.0, span = 1.0;
    if (d->scaling == VSPEC_ROPE_SCALE_YARN) {
        const double per = r / (2.0 * log(base));
        first = fmax(floor(per * log(d->trained_len / (two_pi * d->high))), 0.0);
        const double last = fmin(ceil(per * log(d->trained_len / (two_pi * d->low))), r - 1.0);
        span = fmax(last - first, 0.001);
        m = 0.1 * log(d->factor) + 1.0;
    }
    for (uint32_t i = 0; i < d->rope_dim / 2; ++i) {
        const double f = pow(base, -2.0 * i / r) / two_pi;
        double keep = 1.0;  // share of the pair's own frequency, the rest is stretched
        if (d->scaling == VSPEC_ROPE_SCALE_LINEAR) keep = 0.0;
        if (d->scaling == VSPEC_ROPE_SCALE_BANDS) {
            keep = fmin(fmax((d->trained_len * f - d->low) / (d->high - d->low), 0.0), 1.0);
        }
        if (d->scaling == VSPEC_ROPE_SCALE_YARN) keep = 1.0 - fmin(fmax((i - first) / span, 0.0), 1.0);
        turns[i] = keep == 1.0 ? f : keep * f + (1.0 - keep) * f / d->factor;
    }
    *magnitude = (float)(d->magnitude > 0.0 ? d->magnitude : m);
    return 1;
}

int rope_operand(const VspecRopeRows* r, const VspecRopeDesc* d, const char* which, RopeOperand* o) {
    if (!r->in && !r->out && r->num_heads == 0) return 1;
    if (!r->in || !r->out || r->num_heads == 0) {
        host_error("rope: %s needs in, out and num_heads", which);
        return 0;
    }
    const size_t size = d->dtype == VSPEC_KV_F32 ? 4 : 2;
    if (((uintptr_t)r->in | (uintptr_t)r->out) % size != 0) {
        host_error("rope: %s is not aligned to its element", which);
        return 0;
    }
    o->in = (const uint8_t*)r->in;
    o->out = (uint8_t*)r->out;
    o->heads = r->num_heads;
    o->in_head = r->in_head_stride ? r->in_head_stride : (int64_t)d->head_dim;
    o->out_head = r->out_head_stride ? r->out_head_stride : (int64_t)d->head_dim;
    o->in_token = r->in_token_stride ? r->in_token_stride : (int64_t)d->head_dim * r->num_heads;
    o->out_token = r->out_token_stride ? r->out_token_stride : (int64_t)d->head_dim * r->num_heads;
    if (r->in == r->out && (o->in_head != o->out_head || o->in_token != o->out_token)) {
        host_error("rope: %s in place needs the same strides in and out", which);
        return 0;
    }
    return 1;
}

// Whether an operand's rows start at whole 16-byte chunks of v elements.
bool whole_chunks(const RopeOperand& o, uint32_t v) {
    return o.heads == 0 || ((((uintptr_t)o.in | (uintptr_t)o.out) % 16) == 0 &&
                            ((o.in_token | o.in_head | o.out_token | o.out_head) & (int64_t)(v - 1)) == 0);
}

}  // namespace
}  // namespace vkv

using namespace vkv;

extern "C" int vspec_rocm_rope(const VspecRopeDesc* d) {
    if (!d) {
        host_error("rope: null descriptor");
        return 0;
    }
    if (d->dtype != VSPEC_KV_F32 && d->dtype != VSPEC_KV_F16) {
        host_error("rope: dtype must be f32 or f16");
        return 0;
    }
    if (d->layout != VSPEC_ROPE_HALF && d->layout != VSPEC_ROPE_INTERLEAVED) {
        host_error("rope: bad layout %d", (int)d->layout);
        return 0;
    }
    if (d->head_dim > 2 * kMaxPairs || d->rope_dim == 0 || d->rope_dim % 2 != 0 || d->rope_dim > d->head_dim) {
        host_error("rope: need an even rope_dim of 2..head_dim and a head_dim of at most %u", 2 * kMaxPairs);
        return 0;
    }
    RopeParams p = {};
    if (!rope_turns(d, p.turns, &p.magnitude)) return 0;
    if (d->num_tokens == 0) return 1;  // (empty tensors have no address)
    if (!rope_operand(&d->q, d, "q", &p.q) || !rope_operand(&d->k, d, "k", &p.k)) return 0;
    const uint64_t heads = (uint64_t)p.q.heads + p.k.heads;
    if (heads > 65536u || d->num_tokens > 0x7fffffffu) {
        host_error("rope: at most 65536 heads and 2^31 - 1 tokens");
        return 0;
    }
    if (heads == 0) return 1;
    if (!d->positions) {
        host_error("rope: null positions");
        return 0;
    }
    p.positions = d->positions;
    p.tokens = d->num_tokens;
    p.head_dim = d->head_dim;
    p.rope_dim = d->rope_dim;
    p.sign = d->inverse ? -1.0f : 1.0f;
    const bool inter = d->layout == VSPEC_ROPE_INTERLEAVED, f32 = d->dtype == VSPEC_KV_F32;
    hipStream_t s = (hipStream_t)d->stream;
    // By chunks where rows, strides and the turned part are whole ones (16384 tokens of 40 heads: 215 us by
    // elements, 70 by chunks).  Tokens share a workgroup where that still leaves 4 to a CU.
    const uint32_t v = f32 ? 4 : 8, turned = inter ? d->rope_dim : d->rope_dim / 2;
    if (heads <= kChunkHeads && d->head_dim % v == 0 && turned % v == 0 && whole_chunks(p.q, v) && whole_chunks(p.k, v)) {
        RopeSplit w = {};
        w.tokens = kChunkTokens;
        while (w.tokens > 1 && d->num_tokens / w.tokens < 4u * host_num_cus()) w.tokens /= 2;
        w.turning = turned / v;
        w.units = w.turning + (d->head_dim - d->rope_dim) / v;
        w.half_magic = chunk_magic(d->rope_dim / 2);
        w.units_magic = chunk_magic(w.units);
        w.rows_magic = chunk_magic((uint32_t)heads);
        const dim3 grid((p.tokens + w.tokens - 1) / w.tokens);
        if (f32 && inter) hipLaunchKernelGGL((rope_chunks<float, true>), grid, dim3(256), 0, s, p, w);
        else if (f32) hipLaunchKernelGGL((rope_chunks<float, false>), grid, dim3(256), 0, s, p, w);
        else if (inter) hipLaunchKernelGGL((rope_chunks<_Float16, true>), grid, dim3(256), 0, s, p, w);
        else hipLaunchKernelGGL((rope_chunks<_Float16, false>), grid, dim3(256), 0, s, p, w);
    } else if (f32) {
        hipLaunchKernelGGL((rope_rows<float>), dim3(p.tokens), dim3(256), 0, s, p, inter);
    } else {
        hipLaunchKernelGGL((rope_rows<_Float16>), dim3(p.tokens), dim3(256), 0, s, p, inter);
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) {
        host_error("rope launch: %s", hipGetErrorString(e));
        return 0;
    }
    return 1;
}
