// Multi-head attention for training: shared key/value heads, causal and
// length masks, any strides; forward with the log-sum-exp of every row, and
// the backward pass, which recomputes the probabilities from it.
//
//   S = scale Q K^T over the visible pairs, lse = log sum exp S
//   P = exp(S - lse), O = P V
//   delta = sum_d dO O
//   dV = P^T dO, dS = P (dO V^T - delta), dQ = scale dS K, dK = scale dS^T Q
//
// Sequence b has ql = q_lens[b] queries and kl = kv_lens[b] keys (clamped to
// the tensors' extents).  Query i sees key j when i < ql, j < kl and, under the
// causal mask, j <= i + kl - ql (the last query sees every key).  A masked pair
// takes no part, whatever its values are.  A query that sees nothing has O = 0
// and lse = -inf, and no gradient comes from or to it; rows of padding (i >= ql,
// j >= kl) get zeros the same way.
//
// Everything is fp32 (sums and softmax statistics too); scores are kept in
// the log2 domain (Q times scale * log2 e).
#ifndef ZN_MHA_F32_H
#define ZN_MHA_F32_H

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../zn_kernel_args.h"
#include "zn_mfma_stage.h"
#include "zn_split.h"

namespace {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;

// One sequence's extents.
struct MhaSeq {
    int ql, kl, edge;  // edge: query i sees keys j <= i + edge
    __device__ __forceinline__ MhaSeq(const ZnMhaArgs &p, int b) {
        ql = p.q_lens ? min(max(p.q_lens[b], 0), p.q_len) : p.q_len;
        kl = p.kv_lens ? min(max(p.kv_lens[b], 0), p.kv_len) : p.kv_len;
        edge = p.causal ? kl - ql : kl;
    }
    // keys that query i sees: [0, seen(i))
    __device__ __forceinline__ int seen(int i) const { return i < ql ? max(0, min(kl, i + 1 + edge)) : 0; }
    // the first query that sees key j < kl: [first(j), ql)
    __device__ __forceinline__ int first(int j) const { return max(0, j - edge); }
};

__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
    for (int s = 32; s > 0; s >>= 1) x += __shfl_xor(x, s);
    return x;
}

// A wave to a row, lane l its dims l and l + 64: two values of a row of `dim`.
struct MhaRow {
    float a, b;
    __device__ __forceinline__ MhaRow(const float *row, int dim, int lane) {
        a = lane < dim ? row[lane] : 0.0f;
        b = lane + 64 < dim ? row[lane + 64] : 0.0f;
    }
    __device__ __forceinline__ float dot(const MhaRow &o) const { return wave_sum(a * o.a + b * o.b); }
    __device__ __forceinline__ static void store(float *row, int dim, int lane, float a, float b) {
        if (lane < dim) row[lane] = a;
        if (lane + 64 < dim) row[lane + 64] = b;
    }
};

// The rows one at a time, a wave each: the definition, key by key.  A masked
// pair is never touched, so nothing that it holds can reach a sum.
__device__ __forceinline__ void mha_row_forward(const ZnMhaArgs &p, int b, int h, int i, int lane) {
    const MhaSeq seq(p, b);
    const int n = seq.seen(i);
    const float *k = p.k + b * p.ks[0] + (h / p.group) * p.ks[1], *v = p.v + b * p.ks[0] + (h / p.group) * p.ks[1];
    MhaRow q(p.q + b * p.qs[0] + h * p.qs[1] + i * p.qs[2], n ? p.dim : 0, lane);
    q.a *= p.scale_log2;
    q.b *= p.scale_log2;
    float m = -INFINITY, l = 0.0f, oa = 0.0f, ob = 0.0f;
    for (int j = 0; j < n; ++j) {
        const MhaRow kr(k + j * p.ks[2], p.dim, lane), vr(v + j * p.ks[2], p.dim, lane);
        const float s = q.dot(kr);
        const float mn = fmaxf(m, s), ref = mn == -INFINITY ? 0.0f : mn;
        const float alpha = __builtin_amdgcn_exp2f(m - ref), e = __builtin_amdgcn_exp2f(s - ref);
        l = l * alpha + e;
        oa = oa * alpha + e * vr.a;
        ob = ob * alpha + e * vr.b;
        m = mn;
    }
    const float r = l == 0.0f ? 1.0f : l;
    MhaRow::store(p.out + b * p.os[0] + h * p.os[1] + i * p.os[2], p.dim, lane, oa / r, ob / r);
    if (p.lse && lane == 0)
        p.lse[((int64_t)b * p.q_heads + h) * p.q_len + i] = l == 0.0f ? -INFINITY : (m + __log2f(l)) * kLn2;
}

// grad_q of a row; writes delta too.
__device__ __forceinline__ void mha_row_grad_q(const ZnMhaArgs &p, int b, int h, int i, int lane) {
    const MhaSeq seq(p, b);
    const int64_t at = ((int64_t)b * p.q_heads + h) * p.q_len + i;
    int n = seq.seen(i);
    const float lse = n ? p.lse[at] : -INFINITY;
    if (lse == -INFINITY) n = 0;
    const float *k = p.k + b * p.ks[0] + (h / p.group) * p.ks[1], *v = p.v + b * p.ks[0] + (h / p.group) * p.ks[1];
    const int64_t oat = b * p.os[0] + h * p.os[1] + i * p.os[2], qat = b * p.qs[0] + h * p.qs[1] + i * p.qs[2];
    MhaRow q(p.q + qat, n ? p.dim : 0, lane);
    const MhaRow g(p.grad_out + oat, n ? p.dim : 0, lane), o(p.out + oat, n ? p.dim : 0, lane);
    const float delta = g.dot(o);
    q.a *= p.scale_log2;
    q.b *= p.scale_log2;
    float ga = 0.0f, gb = 0.0f;
    for (int j = 0; j < n; ++j) {
        const MhaRow kr(k + j * p.ks[2], p.dim, lane), vr(v + j * p.ks[2], p.dim, lane);
        const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(lse, -kLog2e, q.dot(kr)));
        const float ds = e * (g.dot(vr) - delta);
        ga += ds * kr.a;
        gb += ds * kr.b;
    }
    MhaRow::store(p.grad_q + qat, p.dim, lane, ga * p.scale, gb * p.scale);
    if (lane == 0) p.delta[at] = delta;
}

// grad_k and grad_v of a row: the query heads of the group in order, their queries ascending.
__device__ __forceinline__ void mha_row_grad_kv(const ZnMhaArgs &p, int b, int kh, int j, int lane) {
    const MhaSeq seq(p, b);
    const bool in = j < seq.kl;
    const int64_t kat = b * p.ks[0] + kh * p.ks[1] + j * p.ks[2];
    const MhaRow kr(p.k + kat, in ? p.dim : 0, lane), vr(p.v + kat, in ? p.dim : 0, lane);
    float ka = 0.0f, kb = 0.0f, va = 0.0f, vb = 0.0f;
    for (int h = kh * p.group; in && h < (kh + 1) * p.group; ++h)
        for (int i = seq.first(j); i < seq.ql; ++i) {
            const int64_t at = ((int64_t)b * p.q_heads + h) * p.q_len + i;
            const float lse = p.lse[at];
            if (lse == -INFINITY) continue;
            const MhaRow q(p.q + b * p.qs[0] + h * p.qs[1] + i * p.qs[2], p.dim, lane);
            const MhaRow g(p.grad_out + b * p.os[0] + h * p.os[1] + i * p.os[2], p.dim, lane);
            const float s = wave_sum((q.a * p.scale_log2) * kr.a + (q.b * p.scale_log2) * kr.b);
            const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(lse, -kLog2e, s));
            const float ds = e * (g.dot(vr) - p.delta[at]);
            va += e * g.a;
            vb += e * g.b;
            ka += ds * q.a;
            kb += ds * q.b;
        }
    MhaRow::store(p.grad_k + kat, p.dim, lane, ka * p.scale, kb * p.scale);
    MhaRow::store(p.grad_v + kat, p.dim, lane, va, vb);
}

}  // namespace

// Grid: x = sequence and head, y = blocks of 4 rows (strided over where there are more than the grid holds).
extern "C" __global__ __launch_bounds__(256) void zn_mha_forward_rows(ZnMhaArgs p) {
    for (int i = blockIdx.y * 4 + threadIdx.x / kWave; i < p.q_len; i += gridDim.y * 4)
        mha_row_forward(p, blockIdx.x / p.q_heads, blockIdx.x % p.q_heads, i, threadIdx.x & (kWave - 1));
}
extern "C" __global__ __launch_bounds__(256) void zn_mha_grad_q_rows(ZnMhaArgs p) {
    for (int i = blockIdx.y * 4 + threadIdx.x / kWave; i < p.q_len; i += gridDim.y * 4)
        mha_row_grad_q(p, blockIdx.x / p.q_heads, blockIdx.x % p.q_heads, i, threadIdx.x & (kWave - 1));
}
extern "C" __global__ __launch_bounds__(256) void zn_mha_grad_kv_rows(ZnMhaArgs p) {
    for (int j = blockIdx.y * 4 + threadIdx.x / kWave; j < p.kv_len; j += gridDim.y * 4)
        mha_row_grad_kv(p, blockIdx.x / p.kv_heads, blockIdx.x % p.kv_heads, j, threadIdx.x & (kWave - 1));
}

#endif
