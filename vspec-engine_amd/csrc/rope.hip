// rope.hip -- rotary positions given for each token (vspec_rocm_rope).
//
// A pair (x1, x2) at position t turns by a = t f: (x1 cos a - x2 sin a, x1 sin a + x2 cos a).
// The angle is reduced in 64 bits: with f in turns a position, t f is off by 2^-53 of itself,
// 2^-33 turns at a million positions, and only its fraction goes on to the f32 sine and cosine
// (in half turns, sincospif, so that no multiple of pi has to be taken away).  Every angle of a
// token serves all its heads.
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
        out[e1] = (T)(x1 * t.x - x2 * t.y);
        out[e2] = (T)(x1 * t.y + x2 * t.x);
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
    if (!rope_operand(&d->q, d, "q", &p.q) || !rope_operand(&d->k, d, "k", &p.k)) return 0;
    const uint64_t heads = (uint64_t)p.q.heads + p.k.heads;
    if (heads > 65536u || d->num_tokens > 0x7fffffffu) {
        host_error("rope: at most 65536 heads and 2^31 - 1 tokens");
        return 0;
    }
    if (d->num_tokens == 0 || heads == 0) return 1;
    if (!d->positions) {
        host_error("rope: null positions");
        return 0;
    }
    p.positions = d->positions;
    p.tokens = d->num_tokens;
    p.head_dim = d->head_dim;
    p.rope_dim = d->rope_dim;
    p.sign = d->inverse ? -1.0f : 1.0f;
    const bool inter = d->layout == VSPEC_ROPE_INTERLEAVED;
    hipStream_t s = (hipStream_t)d->stream;
    if (d->dtype == VSPEC_KV_F32) {
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
