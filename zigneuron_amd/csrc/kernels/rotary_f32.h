// Rotary positions, and the keys and values of new tokens into a paged cache.
//
//   a = p f_i;  (x1, x2) -> s (x1 cos a - x2 sin a, x1 sin a + x2 cos a)
//
// for pair i of a head's first `rot` dims: dims i and i + rot / 2 (layout 0) or
// 2 i and 2 i + 1 (layout 1); the other dims are copied.  The gradient turns
// back (-a).
//
// The angle: p f_i is a product of at most 55 bits, taken as a 64-bit float and
// the rest of its rounding, and reduced to a quarter turn in 64 bits (2 / pi in
// two parts): a turn of a far position is as exact as that of a near one, where
// an angle rounded to 32 bits is off by 2^-24 of itself, 0.06 of a turn's radius
// at 10^6.  The 107 bits of 2 / pi do for angles up to 2^80 (beyond, the turn is
// by any angle).  Sine and cosine of what is left, |y| <= pi / 4, are their Taylor
// polynomials to y^11 and y^10 (the next terms are below 2^-27 of 1).
#ifndef ZN_ROTARY_F32_H
#define ZN_ROTARY_F32_H

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "zn_paged.h"

namespace {

typedef float zn_f32x4_any __attribute__((ext_vector_type(4), aligned(4)));  // at any float
typedef __bf16 zn_bf16x4_any __attribute__((ext_vector_type(4), aligned(2)));

// FAR: an angle past kRotaryNear, where the roundings of a and t are quarter turns of their own.
constexpr float kRotaryNear = 0x1p50f;
template <bool FAR>
__device__ __forceinline__ void rotary_sincos(int position, float freq, float &s, float &c) {
    constexpr double kHi = 0.63661977236758138, kLo = -3.9357353350364972e-17;  // 2 / pi
    const double p = position, f = freq, a = p * f, rest = __builtin_fma(p, f, -a), t = a * kHi, q = __builtin_rint(t);
    double r = (t - q) + __builtin_fma(rest, kHi, __builtin_fma(a, kLo, __builtin_fma(a, kHi, -t)));
    int n = (int)__builtin_fma(__builtin_floor(q * 0.25), -4.0, q);  // of 0..3: q itself may pass 32 bits
    if (FAR) {
        const double k = __builtin_rint(r);
        r -= k;
        n += (int)__builtin_fma(__builtin_floor(k * 0.25), -4.0, k);
    }
    const float y = (float)r * 1.57079632679489662f, z = y * y;
    float u = __builtin_fmaf(z, -1.0f / 39916800.0f, 1.0f / 362880.0f);
    u = __builtin_fmaf(z, u, -1.0f / 5040.0f);
    u = __builtin_fmaf(z, u, 1.0f / 120.0f);
    u = __builtin_fmaf(z, u, -1.0f / 6.0f);
    const float sy = __builtin_fmaf(y * z, u, y);
    float w = __builtin_fmaf(z, -1.0f / 3628800.0f, 1.0f / 40320.0f);
    w = __builtin_fmaf(z, w, -1.0f / 720.0f);
    w = __builtin_fmaf(z, w, 1.0f / 24.0f);
    w = __builtin_fmaf(z, w, -0.5f);
    const float cy = __builtin_fmaf(z, w, 1.0f);
    s = n & 1 ? cy : sy;
    c = n & 1 ? sy : cy;
    if (n & 2) s = -s;
    if ((n + 1) & 2) c = -c;
}

// Four values or the first n of them; the rest are 0.
__device__ __forceinline__ void rotary_load(const float *p, int n, float (&x)[4]) {
    if (n >= 4) {
        const zn_f32x4_any v = *reinterpret_cast<const zn_f32x4_any *>(p);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = v[e];
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = e < n ? p[e] : 0.0f;
    }
}
__device__ __forceinline__ void rotary_store(float *p, int n, const float (&x)[4]) {
    if (n >= 4) {
        *reinterpret_cast<zn_f32x4_any *>(p) = zn_f32x4_any{x[0], x[1], x[2], x[3]};
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (e < n) p[e] = x[e];
    }
}
// ... rounded to bf16, to the nearest, ties to even: the cache's own precision, once for each value that enters it.
__device__ __forceinline__ void rotary_store(__bf16 *p, int n, const float (&x)[4]) {
    if (n >= 4) {
        *reinterpret_cast<zn_bf16x4_any *>(p) = __builtin_convertvector((zn_f32x4_any{x[0], x[1], x[2], x[3]}), zn_bf16x4_any);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (e < n) p[e] = (__bf16)x[e];
    }
}

// A thread's share of a head: 8 dims, four of them at da and four at db (na, nb: how many there are).  Units [0, turns) are pairs.
struct RotaryUnit {
    int da, db, na, nb;
    bool turns, half;
    __device__ __forceinline__ RotaryUnit(int unit, int dim, int rot, int layout) {
        const int n = (rot / 2 + 3) / 4;
        turns = unit < n;
        half = turns && layout == 0;
        if (half) {
            da = 4 * unit;
            db = rot / 2 + da;
            na = nb = min(4, rot / 2 - da);
        } else {
            da = turns ? 8 * unit : rot + 8 * (unit - n);
            db = da + 4;
            na = min(4, (turns ? rot : dim) - da);
            nb = min(4, (turns ? rot : dim) - db);
        }
    }
};

// The unit's sines and cosines at one position.
struct RotaryTurn {
    float s[4], c[4];
    __device__ __forceinline__ RotaryTurn(const RotaryUnit &u, const float *freq, int rot, int position, float scale, float sign) {
        if (fill<false>(u, freq, rot, position, scale, sign) > kRotaryNear) fill<true>(u, freq, rot, position, scale, sign);
    }
    // Returns the largest angle.
    template <bool FAR>
    __device__ __forceinline__ float fill(const RotaryUnit &u, const float *freq, int rot, int position, float scale, float sign) {
        float most = 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            s[e] = 0.0f;
            c[e] = 1.0f;
            const int i = (u.half ? u.da : u.da / 2) + e;
            if (u.turns && i < rot / 2) {
                const float f = freq[i];
                most = fmaxf(most, __builtin_fabsf((float)position * f));
                rotary_sincos<FAR>(position, f, s[e], c[e]);
                s[e] *= sign * scale;
                c[e] *= scale;
            }
        }
        return most;
    }
    __device__ __forceinline__ static void turn(float &x, float &y, float s, float c) {
        const float a = x, b = y;
        x = __builtin_fmaf(a, c, -(b * s));
        y = __builtin_fmaf(a, s, b * c);
    }
    __device__ __forceinline__ void apply(const RotaryUnit &u, float (&a)[4], float (&b)[4]) const {
        if (!u.turns) return;
        if (u.half) {
#pragma unroll
            for (int e = 0; e < 4; ++e) turn(a[e], b[e], s[e], c[e]);
        } else {
            turn(a[0], a[1], s[0], c[0]);
            turn(a[2], a[3], s[1], c[1]);
            turn(b[0], b[1], s[2], c[2]);
            turn(b[2], b[3], s[3], c[3]);
        }
    }
};

}  // namespace

// A thread has the same 8 dims of one token in every head it turns, and takes
// their sines and cosines once: a few dozen 64-bit instructions a pair, beside 16
// bytes a head read and written.  Bound by those, or by the launch.  Neighbouring
// threads have neighbouring dims, then heads or tokens, whichever lie together.
// MI355X, alone in a row: 2 x 40 heads of 4096 x 128 (336 MB moved) 56 us, 6.0 TB/s,
// where the last-level cache helps (67 among other kernels; a large copy 4.9); 3 x 12
// heads of 2777 x 76, half turned (61 MB), 13 us; 8 x 20 heads of one token of 64 3.7
// us, two round trips to memory behind a launch of 1.6.
extern "C" __global__ __launch_bounds__(256) void zn_rotary(ZnRotaryArgs p) {
    const int per = p.slots * p.units, tl = threadIdx.x / per, in = threadIdx.x - tl * per, slot = in / p.units;
    const int64_t token = (int64_t)blockIdx.x * p.tokens + tl;
    if (tl >= p.tokens || token >= (int64_t)p.batch * p.len) return;
    const int b = (int)token / p.len, i = (int)token - b * p.len;
    const RotaryUnit u(in - slot * p.units, p.dim, p.rot, p.layout);
    const RotaryTurn t(u, p.freq, p.rot, p.positions ? p.positions[b * p.position_stride + i] : i, p.scale, p.sign);
    const float *x = p.x + b * p.xs[0] + i * p.xs[2];
    float *y = p.y + b * p.ys[0] + i * p.ys[2];
    for (int h = blockIdx.y * p.slots + slot; h < p.heads; h += gridDim.y * p.slots) {
        float v[2][4];
        rotary_load(x + h * p.xs[1] + u.da, u.na, v[0]);
        rotary_load(x + h * p.xs[1] + u.db, u.nb, v[1]);
        t.apply(u, v[0], v[1]);
        rotary_store(y + h * p.ys[1] + u.da, u.na, v[0]);
        rotary_store(y + h * p.ys[1] + u.db, u.nb, v[1]);
    }
}

namespace {

// Queries, keys and values of new tokens: q turned to q_out, k turned to its page, v to its page.  One launch, as zn_rotary's but for
// the tokens' sequences (64 starts at a time by the whole wave) and pages.  Bound by its bytes, or by the launch.  MI355X: 8192 tokens
// of 32 + 2 x 8 heads of 128 into bf16 (369 MB moved) 73 us, 5.1 TB/s; 6654 tokens of 10 + 2 x 5 heads of 76 19 us (25 among other
// kernels); 64 tokens of 16 + 2 x 4 heads of 64 4.2 us, the third of three dependent loads (start, page, row).
template <typename T>
__device__ __forceinline__ void paged_append(const ZnAppendArgs &p) {
    const ZnPagedCache &c = p.c;
    const int per = p.slots * p.units, tl = threadIdx.x / per, in = threadIdx.x - tl * per, slot = in / p.units;
    const int t0 = (int)blockIdx.x * p.per_wg, t = t0 + tl;
    int b = paged_find(c, t0);
    if (tl >= p.per_wg || t >= c.tokens) return;
    while (b < c.batch && c.starts[b + 1] <= t) ++b;
    if (b < 0 || b >= c.batch) return;  // a row before the first sequence or behind the last
    const PagedSeq seq(c, b);
    const int j = seq.first + t - seq.t0;
    if (t < seq.t0 || t >= seq.t0 + seq.ql) return;
    const RotaryUnit u(in - slot * p.units, c.dim, p.rot, p.layout);
    const RotaryTurn turn(u, p.freq, p.rot, p.positions ? p.positions[t] : j, p.scale, 1.0f);
    const int64_t at = j < 0 ? -1 : paged_at(c, b, 0, j);
    for (int h = blockIdx.y * p.slots + slot; h < p.q_heads + 2 * c.kv_heads; h += gridDim.y * p.slots) {
        const int kh = h - p.q_heads, vh = kh - c.kv_heads;
        const float *x = kh < 0 ? p.q + t * p.qs[0] + h * p.qs[1] : (vh < 0 ? p.k + kh * p.kvs[1] : p.v + vh * p.kvs[1]) + t * p.kvs[0];
        float v[2][4];
        rotary_load(x + u.da, u.na, v[0]);
        rotary_load(x + u.db, u.nb, v[1]);
        if (vh < 0) turn.apply(u, v[0], v[1]);
        if (kh < 0) {
            float *y = p.q_out + t * p.os[0] + h * p.os[1];
            rotary_store(y + u.da, u.na, v[0]);
            rotary_store(y + u.db, u.nb, v[1]);
        } else if (at >= 0) {
            T *y = reinterpret_cast<T *>(vh < 0 ? c.k : c.v) + at + (vh < 0 ? kh : vh) * c.stride[1];
            rotary_store(y + u.da, u.na, v[0]);
            rotary_store(y + u.db, u.nb, v[1]);
        }
    }
}

}  // namespace

extern "C" __global__ __launch_bounds__(256) void zn_paged_append_f32(ZnAppendArgs p) { paged_append<float>(p); }
extern "C" __global__ __launch_bounds__(256) void zn_paged_append_bf16(ZnAppendArgs p) { paged_append<__bf16>(p); }

#endif
