// Attention of new tokens over a paged cache: each sequence's tokens against
// all that its pages hold, its new keys among it.
//
//   S = scale Q K^T over the visible pairs, lse = log sum exp S, O = exp(S - lse) V
//
// Sequence b has ql new tokens and kl positions (PagedSeq).  Its token i sees
// position j < kl whose page is one of the cache's and, under the causal mask,
// j <= i + kl - ql (the last token sees every position).  A masked pair takes no
// part, whatever its values are.  A query that sees nothing has O = 0 and
// lse = -inf.  Rows of no sequence are not written.
//
// K and V are fp32 or bf16; everything else is fp32 (sums and softmax
// statistics too), scores in the log2 domain (Q times scale * log2 e).
#ifndef ZN_PAGED_F32_H
#define ZN_PAGED_F32_H

#include "mha_f32.h"
#include "zn_paged.h"

namespace {

// A wave to a row, lane l its dims l and l + 64.
template <typename T>
__device__ __forceinline__ MhaRow paged_row(const T *row, int dim, int lane) {
    MhaRow r(nullptr, 0, lane);
    if (lane < dim) r.a = (float)row[lane];
    if (lane + 64 < dim) r.b = (float)row[lane + 64];
    return r;
}

// The definition, key by key: a row's walk over positions [from, to).
template <typename T>
__device__ __forceinline__ void paged_walk(const ZnPagedArgs &p, int b, int t, int h, int from, int to, int lane, MhaRowState &w) {
    const T *k = reinterpret_cast<const T *>(p.c.k), *v = reinterpret_cast<const T *>(p.c.v);
    MhaRow q(p.q + t * p.qs[0] + h * p.qs[1], from < to ? p.c.dim : 0, lane);
    q.a *= p.scale_log2;
    q.b *= p.scale_log2;
    for (int j = from; j < to && w.l == w.l; ++j) {  // a NaN sum stays one, and all of O with it
        const int64_t at = paged_at(p.c, b, h / p.group, j);
        if (at < 0) continue;
        const MhaRow kr = paged_row(k + at, p.c.dim, lane), vr = paged_row(v + at, p.c.dim, lane);
        const float s = q.dot(kr);
        const float mn = fmaxf(w.m, s), ref = mn == -INFINITY ? 0.0f : mn;
        const float alpha = __builtin_amdgcn_exp2f(w.m - ref), e = __builtin_amdgcn_exp2f(s - ref);
        w.l = w.l * alpha + e;
        w.oa = w.oa * alpha + e * vr.a;
        w.ob = w.ob * alpha + e * vr.b;
        w.m = mn;
    }
}

__device__ __forceinline__ void paged_store(const ZnPagedArgs &p, int t, int h, int lane, float m, float l, float oa, float ob) {
    const float r = l == 0.0f ? 1.0f : l;
    MhaRow::store(p.out + t * p.os[0] + h * p.os[1], p.c.dim, lane, oa / r, ob / r);
    if (p.lse && lane == 0) p.lse[(int64_t)t * p.q_heads + h] = mha_lse(m, l);
}

// Rows one at a time, a wave each: grid x the tokens, y four heads.
template <typename T>
__device__ __forceinline__ void paged_rows(const ZnPagedArgs &p) {
    const int lane = threadIdx.x & (kWave - 1), h = blockIdx.y * 4 + threadIdx.x / kWave, t = blockIdx.x;
    if (h >= p.q_heads) return;
    const int b = paged_find(p.c, t);
    if (b < 0 || b >= p.c.batch) return;
    const PagedSeq seq(p.c, b);
    const int i = t - seq.t0;
    if (i < 0 || i >= min(seq.ql, p.max_q)) return;
    MhaRowState w;
    paged_walk<T>(p, b, t, h, 0, p.causal ? max(0, min(seq.kl, seq.first + i + 1)) : seq.kl, lane, w);
    paged_store(p, t, h, lane, w.m, w.l, w.oa, w.ob);
}

}  // namespace

extern "C" __global__ __launch_bounds__(256) void zn_paged_rows_f32(ZnPagedArgs p) { paged_rows<float>(p); }
extern "C" __global__ __launch_bounds__(256) void zn_paged_rows_bf16(ZnPagedArgs p) { paged_rows<__bf16>(p); }

#endif
