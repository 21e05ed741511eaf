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
#include <limits.h>
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
// pair is never touched, so nothing that it holds can reach a sum.  The tiles
// below take these rows where a value or a sum is not finite.

// A row's walk over keys [from, to): running maximum (log2 domain), sum and O.
struct MhaRowState {
    float m = -INFINITY, l = 0.0f, oa = 0.0f, ob = 0.0f;
    __device__ __forceinline__ void walk(const ZnMhaArgs &p, int b, int h, int i, int from, int to, int lane) {
        const float *k = p.k + b * p.ks[0] + (h / p.group) * p.ks[1], *v = p.v + b * p.ks[0] + (h / p.group) * p.ks[1];
        MhaRow q(p.q + b * p.qs[0] + h * p.qs[1] + i * p.qs[2], from < to ? p.dim : 0, lane);
        q.a *= p.scale_log2;
        q.b *= p.scale_log2;
        for (int j = from; j < to; ++j) {
            const MhaRow kr(k + j * p.ks[2], p.dim, lane), vr(v + j * p.ks[2], p.dim, lane);
            const float s = q.dot(kr);
            const float mn = fmaxf(m, s), ref = mn == -INFINITY ? 0.0f : mn;
            const float alpha = __builtin_amdgcn_exp2f(m - ref), e = __builtin_amdgcn_exp2f(s - ref);
            l = l * alpha + e;
            oa = oa * alpha + e * vr.a;
            ob = ob * alpha + e * vr.b;
            m = mn;
        }
    }
};

__device__ __forceinline__ float mha_lse(float m, float l) { return l == 0.0f ? -INFINITY : (m + __log2f(l)) * kLn2; }

__device__ __forceinline__ void mha_row_forward(const ZnMhaArgs &p, int b, int h, int i, int lane) {
    MhaRowState s;
    s.walk(p, b, h, i, 0, MhaSeq(p, b).seen(i), lane);
    const float r = s.l == 0.0f ? 1.0f : s.l;
    MhaRow::store(p.out + b * p.os[0] + h * p.os[1] + i * p.os[2], p.dim, lane, s.oa / r, s.ob / r);
    if (p.lse && lane == 0) p.lse[((int64_t)b * p.q_heads + h) * p.q_len + i] = mha_lse(s.m, s.l);
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

// ------------------------------------------------------------------- tiles
// The same on the bf16 matrix cores, every operand value split into three bf16
// parts (zn_split.h).  One side of the products stays in a wave's registers
// (queries for O and dQ, keys for dK and dV); the other side's two tensors
// (K and V, or Q and dO) come past in blocks of 32 rows, split by the thread
// that loads them and staged in LDS, two stages.
//
// A staged tensor serves products over its dims and over its rows: rows lie
// in slices of 32 dims, a row's 64 bytes as four 16-byte chunks, chunk c the
// dims 4c .. 4c + 3 and 16 + 4c .. 16 + 4c + 3 of the slice.  A fragment over
// dims is one ds_read_b128; one over rows comes from two transposing reads
// (ds_read_b64_tr_b16), whose 4 x 16 blocks are the halves of the chunks.  The
// same chunk order over rows is that of the accumulators: the two 16-row
// blocks of S that a lane holds are its fragment of the next product.
template <int DP, int NT>
struct MhaStage {
    static constexpr int BR = 32, SL = DP / 32, DB = DP / 16;
    static constexpr int kPart = BR * DP * 2;  // bytes of one bf16 part of a tensor's block
    static constexpr int kStage = 6 * kPart;
    static constexpr int kUnits = BR * DP / 4;  // staging units of 8 values: the first tensor's, then the second's
    static constexpr int UPT = (kUnits + NT - 1) / NT;
    static_assert(kUnits / 2 % kWave == 0, "a wave's units are all of one tensor");

    char *lds;
    const float *base[2];
    int64_t stride[2];
    int dim, tid;
    int frag, tr;      // this lane's place in a fragment over dims, over rows
    uint32_t off[UPT];
    int pos[UPT];
    bool second[UPT];
    float g[UPT][8];

    __device__ static __forceinline__ int slot(int r, int c) { return r * 64 + ((c ^ (-(r >> 2) & 3)) << 4); }

    __device__ __forceinline__ MhaStage(char *lds, int tid, int dim, const float *x, int64_t sx, const float *y, int64_t sy)
        : lds(lds), dim(dim), tid(tid) {
        base[0] = x;
        base[1] = y;
        stride[0] = sx;
        stride[1] = sy;
        const int lane = tid & (kWave - 1), li = lane & 15, lh = lane >> 4;
        frag = slot(li, lh);
        tr = slot(4 * lh + li / 4, li % 4);
#pragma unroll
        for (int j = 0; j < UPT; ++j) {
            const int u = j * NT + tid;
            second[j] = __builtin_amdgcn_readfirstlane(u) >= kUnits / 2;
            const int v = second[j] ? u - kUnits / 2 : u;
            const int row = v / (DP / 8), dc = v % (DP / 8), d = 32 * (dc / 4) + 4 * (dc % 4);
            off[j] = (uint32_t)(row * (int)(second[j] ? sy : sx) + d) * 4u;
            pos[j] = (second[j] ? 3 * kPart : 0) + (dc / 4) * (BR * 64) + slot(row, dc % 4);
            if (u >= kUnits) off[j] = kOutOfRange;
        }
    }
    // Rows r0 .. r0 + 31 of the two tensors, zeros from row `end` on (and in every row where r0 >= end).
    __device__ __forceinline__ void load(int r0, int end) {
        const int n = min(BR, end - r0);
        __amdgpu_buffer_rsrc_t r[2];
#pragma unroll
        for (int t = 0; t < 2; ++t)
            r[t] = make_rsrc(base[t] + (n > 0 ? (int64_t)r0 * stride[t] : 0), n > 0 ? (uint32_t)((n - 1) * (int)stride[t] + dim) * 4u : 0u);
#pragma unroll
        for (int j = 0; j < UPT; ++j) {
            if (j * NT + tid >= kUnits) continue;  // whole waves
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int d = (pos_dim(j) + 16 * h);
                const uint32_t o = d < dim ? off[j] + 64u * h : kOutOfRange;
                const zn_f32x4 v = __builtin_bit_cast(zn_f32x4, __builtin_amdgcn_raw_buffer_load_b128(second[j] ? r[1] : r[0], o, 0, 0));
#pragma unroll
                for (int e = 0; e < 4; ++e) g[j][4 * h + e] = v[e];
            }
        }
    }
    // the first dim of unit j's first four
    __device__ __forceinline__ int pos_dim(int j) const {
        const int u = j * NT + tid, v = second[j] ? u - kUnits / 2 : u, dc = v % (DP / 8);
        return 32 * (dc / 4) + 4 * (dc % 4);
    }
    // Unit j's values, the first tensor's times `scale`, to stage st.
    __device__ __forceinline__ void stage(int st, int j, float scale) {
        if (j * NT + tid >= kUnits) return;
        if (dim & 3) {  // the last four of a row end inside it
            const int d = pos_dim(j);
#pragma unroll
            for (int e = 0; e < 8; ++e) g[j][e] = d + (e < 4 ? e : 12 + e) < dim ? g[j][e] : 0.0f;
        }
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = second[j] ? g[j][e] : g[j][e] * scale;
        zn_u32x4 w[3];
        split8(x, w);
#pragma unroll
        for (int q = 0; q < 3; ++q) *reinterpret_cast<zn_u32x4 *>(lds + st * kStage + pos[j] + q * kPart) = w[q];
    }
    // Part q of tensor t: rows 16 rb + li, chunk lh of slice sl
    __device__ __forceinline__ zn_bf16x8 dims(int st, int t, int q, int sl, int rb) const {
        return __builtin_bit_cast(
            zn_bf16x8, *reinterpret_cast<const zn_u32x4 *>(lds + st * kStage + (3 * t + q) * kPart + sl * (BR * 64) + rb * (16 * 64) + frag));
    }
    // ... dims 16 db + li, rows 4 lh .. 4 lh + 3 and 16 + 4 lh .. 16 + 4 lh + 3
    __device__ __forceinline__ zn_bf16x8 rows(int st, int t, int q, int db) const {
        typedef short s4 __attribute__((ext_vector_type(4)));
        typedef short s8 __attribute__((ext_vector_type(8)));
        typedef __attribute__((address_space(3))) s4 ls4;
        char *at = lds + st * kStage + (3 * t + q) * kPart + (db / 2) * (BR * 64) + 8 * (db & 1) + tr;
        const s4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ls4 *)at), b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ls4 *)(at + 16 * 64));
        return __builtin_bit_cast(zn_bf16x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
    }
};

// The six products of two split operands, largest last.
constexpr int kMhaPA[6] = {2, 1, 0, 1, 0, 0}, kMhaPB[6] = {0, 1, 2, 0, 1, 0};

// Dims 32 sl + 4 lh .. + 3 and + 16 of a row (null: zeros) times `scale`, split.
template <int SL>
__device__ __forceinline__ void mha_row_frags(const float *row, int dim, int lh, float scale, zn_bf16x8 (&f)[SL][3]) {
#pragma unroll
    for (int sl = 0; sl < SL; ++sl) {
        float x[8];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int d = 32 * sl + 4 * lh + 16 * h;
            zn_f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
            if (row && d + 4 <= dim) {
                v = *reinterpret_cast<const zn_f32x4u *>(row + d);
            } else if (row) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (d + e < dim) v[e] = row[d + e];
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) x[4 * h + e] = v[e] * scale;
        }
        zn_u32x4 w[3];
        split8(x, w);
#pragma unroll
        for (int q = 0; q < 3; ++q) f[sl][q] = __builtin_bit_cast(zn_bf16x8, w[q]);
    }
}

// The accumulators' value of dims 16 db + 4 lh .. + 3, stored to a row.
__device__ __forceinline__ void mha_store4(float *row, int d, int dim, zn_f32x4 v) {
    if (d + 4 <= dim) {
        *reinterpret_cast<zn_f32x4u *>(row + d) = v;
    } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (d + r < dim) row[d + r] = v[r];
    }
}

__device__ __forceinline__ float max_over_rows(float x) {
    // the 4 lanes of a column: li, li + 16, li + 32, li + 48
    const auto a = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
    x = fmaxf(__builtin_bit_cast(float, a[0]), __builtin_bit_cast(float, a[1]));
    const auto b = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
    return fmaxf(__builtin_bit_cast(float, b[0]), __builtin_bit_cast(float, b[1]));
}

// The query rows of a workgroup: those of the query heads that share a
// key/value head follow each other, row r = g * q_len + i, so that a few
// queries of many heads fill a block.
struct MhaQuery {
    int h, i;
    bool in;
    __device__ __forceinline__ MhaQuery(const ZnMhaArgs &p, int kh, int r) {
        const int g = r / p.q_len;
        i = r - g * p.q_len;
        h = kh * p.group + g;
        in = g < p.group;
    }
};

// O and lse (BACK false) or dQ and delta (BACK true) of NW x FQ x 16 query rows.
template <int DP, int NW, int FQ, bool BACK>
struct MhaQueryTile {
    typedef MhaStage<DP, NW * kWave> Stage;
    static constexpr int SL = Stage::SL, DB = Stage::DB;

    __device__ static __forceinline__ void run(const ZnMhaArgs &p, char *lds) {
        const int tid = threadIdx.x, lane = tid & (kWave - 1);
        const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
        const int li = lane & 15, lh = lane >> 4;
        const int b = blockIdx.x / p.kv_heads, kh = blockIdx.x - b * p.kv_heads;
        const int rows = p.group * p.q_len;
        // causal rows see more the later they come: the long tiles first
        const int r0 = (int)(gridDim.y - 1 - blockIdx.y) * (NW * FQ * 16), w0 = r0 + wave * FQ * 16;
        const MhaSeq seq(p, b);
        const float *k = p.k + b * p.ks[0] + kh * p.ks[1], *v = p.v + b * p.ks[0] + kh * p.ks[1];

        // keys that the tile's rows see: none past `last`; the wave's rows all see those before `all`
        int lim[FQ], all = INT_MAX, any = 0;
        zn_bf16x8 qf[FQ][SL][3], gf[BACK ? FQ : 1][SL][3];
        float lse2[FQ], delta[FQ];
#pragma unroll
        for (int f = 0; f < FQ; ++f) {
            const MhaQuery r(p, kh, w0 + 16 * f + li);
            lim[f] = r.in ? seq.seen(r.i) : 0;
            const float *q = p.q + b * p.qs[0] + r.h * p.qs[1] + r.i * p.qs[2];
            if constexpr (BACK) {
                const int64_t at = ((int64_t)b * p.q_heads + r.h) * p.q_len + r.i;
                const float lse = lim[f] ? p.lse[at] : -INFINITY;
                if (lse == -INFINITY) lim[f] = 0;
                lse2[f] = lse;
                const int64_t oat = b * p.os[0] + r.h * p.os[1] + r.i * p.os[2];
                const float *g = lim[f] ? p.grad_out + oat : nullptr, *o = lim[f] ? p.out + oat : nullptr;
                mha_row_frags<SL>(g, p.dim, lh, 1.0f, gf[f]);
                float sum = 0.0f;
#pragma unroll
                for (int c = 0; c < 2 * SL; ++c)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int d = 16 * c + 4 * lh + e;
                        if (lim[f] && d < p.dim) sum = __builtin_fmaf(g[d], o[d], sum);
                    }
                sum += __shfl_xor(sum, 16);
                sum += __shfl_xor(sum, 32);
                delta[f] = sum;
                if (r.in && lh == 0) p.delta[at] = sum;
            }
            mha_row_frags<SL>(lim[f] ? q : nullptr, p.dim, lh, p.scale_log2, qf[f]);
            all = min(all, lim[f]);
            any = max(any, lim[f]);
        }
#pragma unroll
        for (int s = 1; s < 16; s <<= 1) {
            all = min(all, __shfl_xor(all, s));
            any = max(any, __shfl_xor(any, s));
        }
        all = __builtin_amdgcn_readfirstlane(all);
        any = __builtin_amdgcn_readfirstlane(any);
        // keys that any row of the workgroup sees: its last row's, or all of them where it spans heads
        const int rl = min(r0 + NW * FQ * 16, rows) - 1, i0 = r0 % p.q_len;
        int last = seq.ql ? seq.kl : 0;
        if (r0 - i0 + p.q_len > rl) last = i0 < seq.ql ? seq.seen(min(rl - r0 + i0, seq.ql - 1)) : 0;

        zn_f32x4 o[FQ][DB];
        float m[FQ], l[FQ];
#pragma unroll
        for (int f = 0; f < FQ; ++f) {
            m[f] = -INFINITY;
            l[f] = 0.0f;
#pragma unroll
            for (int d = 0; d < DB; ++d) o[f][d] = zn_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }

        Stage sg(lds, tid, p.dim, k, p.ks[2], v, p.ks[2]);
        const int nblk = (last + 31) / 32;
        sg.load(0, seq.kl);
#pragma unroll
        for (int j = 0; j < Stage::UPT; ++j) sg.stage(0, j, 1.0f);
        for (int blk = 0; blk < nblk; ++blk) {
            const int st = blk & 1, k0 = 32 * blk;
            __syncthreads();  // block blk is in LDS; every wave is done with block blk - 1
            sg.load(k0 + 32, blk + 1 < nblk ? seq.kl : 0);
            if (k0 + 32 <= all) block<false>(sg, st, k0, lane, lim, qf, gf, lse2, delta, o, m, l);
            else if (k0 < any) block<true>(sg, st, k0, lane, lim, qf, gf, lse2, delta, o, m, l);
#pragma unroll
            for (int j = 0; j < Stage::UPT; ++j) sg.stage(st ^ 1, j, 1.0f);
        }

        bool bad = false;
#pragma unroll
        for (int f = 0; f < FQ; ++f) {
            bad |= !BACK && !(l[f] < INFINITY);
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    bad |= !(__builtin_fabsf(o[f][d][r]) < INFINITY);
                    o[f][d][r] *= kSplitUnscale;
                }
        }
        if (__builtin_amdgcn_ballot_w64(bad)) {
            for (int x = 0; x < 16 * FQ; ++x) {
                const MhaQuery r(p, kh, w0 + x);
                if (!r.in) break;
                if constexpr (BACK) mha_row_grad_q(p, b, r.h, r.i, lane);
                else mha_row_forward(p, b, r.h, r.i, lane);
            }
            return;
        }
#pragma unroll
        for (int f = 0; f < FQ; ++f) {
            const MhaQuery r(p, kh, w0 + 16 * f + li);
            float sum = 0.0f;
            if constexpr (!BACK) {
                sum = l[f] + __shfl_xor(l[f], 16);
                sum += __shfl_xor(sum, 32);
            }
            if (!r.in) continue;
            float *row = BACK ? p.grad_q + b * p.qs[0] + r.h * p.qs[1] + r.i * p.qs[2]
                              : p.out + b * p.os[0] + r.h * p.os[1] + r.i * p.os[2];
            if (!BACK && p.lse && lh == 0) p.lse[((int64_t)b * p.q_heads + r.h) * p.q_len + r.i] = mha_lse(m[f], sum);
            const float div = BACK ? 1.0f : (sum == 0.0f ? 1.0f : sum);
#pragma unroll
            for (int d = 0; d < DB; ++d) {
                const zn_f32x4 x = BACK ? o[f][d] * p.scale : o[f][d] / div;
                mha_store4(row, 16 * d + 4 * lh, p.dim, x);
            }
        }
    }

    // One block of 32 keys: S^T = K (cQ)^T (and dP^T = V dO^T), then O^T += V^T P^T or dQ^T += K^T dS^T.
    template <bool MASK>
    __device__ static __forceinline__ void block(const Stage &sg, int st, int k0, int lane, const int (&lim)[FQ],
                                                 const zn_bf16x8 (&qf)[FQ][SL][3], const zn_bf16x8 (&gf)[BACK ? FQ : 1][SL][3],
                                                 const float (&lse2)[FQ], const float (&delta)[FQ], zn_f32x4 (&o)[FQ][DB],
                                                 float (&m)[FQ], float (&l)[FQ]) {
        const int lh = lane >> 4;
        zn_f32x4 s[FQ][2], dp[BACK ? FQ : 1][2];
#pragma unroll
        for (int f = 0; f < FQ; ++f)
#pragma unroll
            for (int rb = 0; rb < 2; ++rb) {
                s[f][rb] = zn_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                if constexpr (BACK) dp[f][rb] = zn_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            }
#pragma unroll
        for (int t = 0; t < (BACK ? 2 : 1); ++t)
#pragma unroll
            for (int sl = 0; sl < SL; ++sl) {
                zn_bf16x8 a[2][3];
#pragma unroll
                for (int rb = 0; rb < 2; ++rb)
#pragma unroll
                    for (int q = 0; q < 3; ++q) a[rb][q] = sg.dims(st, t, q, sl, rb);
#pragma unroll
                for (int pr = 0; pr < 6; ++pr)
#pragma unroll
                    for (int rb = 0; rb < 2; ++rb)
#pragma unroll
                        for (int f = 0; f < FQ; ++f) {
                            if (t == 0) s[f][rb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[rb][kMhaPA[pr]], qf[f][sl][kMhaPB[pr]], s[f][rb], 0, 0, 0);
                            else dp[BACK ? f : 0][rb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[rb][kMhaPA[pr]], gf[BACK ? f : 0][sl][kMhaPB[pr]], dp[BACK ? f : 0][rb], 0, 0, 0);
                        }
            }
        zn_bf16x8 pf[FQ][3];
#pragma unroll
        for (int f = 0; f < FQ; ++f) {
            float x[8];
            if constexpr (BACK) {
                const float ml = lse2[f] * -kLog2e;  // its rounding moves the whole row by less than its scores' own
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float pe = __builtin_amdgcn_exp2f(__builtin_fmaf(s[f][e / 4][e % 4], kSplitUnscale, ml));
                    const float de = __builtin_fmaf(dp[f][e / 4][e % 4], kSplitUnscale, -delta[f]);
                    x[e] = pe * de;
                    if (MASK && k0 + 16 * (e / 4) + 4 * lh + e % 4 >= lim[f]) x[e] = 0.0f;
                }
            } else {
                float mb = -INFINITY;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if (MASK && k0 + 16 * (e / 4) + 4 * lh + e % 4 >= lim[f]) s[f][e / 4][e % 4] = -INFINITY;
                    mb = fmaxf(mb, s[f][e / 4][e % 4]);
                }
                const float mn = fmaxf(m[f], max_over_rows(mb) * kSplitUnscale);
                const float ref = MASK && mn == -INFINITY ? 0.0f : mn;
                const float alpha = __builtin_amdgcn_exp2f(m[f] - ref);
                float rs = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    x[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[f][e / 4][e % 4], kSplitUnscale, -ref));
                    rs += x[e];
                }
                l[f] = l[f] * alpha + rs;
                m[f] = mn;
                if (__builtin_amdgcn_ballot_w64(alpha != 1.0f)) {
#pragma unroll
                    for (int d = 0; d < DB; ++d) o[f][d] *= alpha;
                }
            }
            zn_u32x4 w[3];
            split8(x, w);
#pragma unroll
            for (int q = 0; q < 3; ++q) pf[f][q] = __builtin_bit_cast(zn_bf16x8, w[q]);
        }
#pragma unroll
        for (int d = 0; d < DB; ++d) {
            zn_bf16x8 a[3];
#pragma unroll
            for (int q = 0; q < 3; ++q) a[q] = sg.rows(st, BACK ? 0 : 1, q, d);
#pragma unroll
            for (int pr = 0; pr < 6; ++pr)
#pragma unroll
                for (int f = 0; f < FQ; ++f)
                    o[f][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[kMhaPA[pr]], pf[f][kMhaPB[pr]], o[f][d], 0, 0, 0);
        }
    }
};

// dK and dV of NW x FK x 16 keys: the group's query heads in order, their
// queries ascending in blocks of 32 (Q scaled, dO, and each row's lse and delta
// in LDS).  S = (cQ) K^T and dP = dO V^T, dV^T += dO^T P and dK^T += Q^T dS.
template <int DP, int NW, int FK>
struct MhaKeyTile {
    typedef MhaStage<DP, NW * kWave> Stage;
    static constexpr int SL = Stage::SL, DB = Stage::DB;
    static constexpr int kRows = 2 * Stage::kStage;     // lse and delta of two stages' rows: [stage][lse, delta][32]
    static constexpr int kBytes = kRows + 2 * 2 * 32 * 4;

    __device__ static __forceinline__ void run(const ZnMhaArgs &p, char *lds) {
        const int tid = threadIdx.x, lane = tid & (kWave - 1);
        const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
        const int li = lane & 15, lh = lane >> 4;
        const int b = blockIdx.x / p.kv_heads, kh = blockIdx.x - b * p.kv_heads;
        const int j0 = (int)blockIdx.y * (NW * FK * 16), w0 = j0 + wave * FK * 16;
        const MhaSeq seq(p, b);
        const int64_t kat = b * p.ks[0] + kh * p.ks[1];

        zn_bf16x8 kf[FK][SL][3], vf[FK][SL][3];
        zn_f32x4 dk[FK][DB], dv[FK][DB];
#pragma unroll
        for (int f = 0; f < FK; ++f) {
            const int j = w0 + 16 * f + li;
            mha_row_frags<SL>(j < seq.kl ? p.k + kat + j * p.ks[2] : nullptr, p.dim, lh, 1.0f, kf[f]);
            mha_row_frags<SL>(j < seq.kl ? p.v + kat + j * p.ks[2] : nullptr, p.dim, lh, 1.0f, vf[f]);
#pragma unroll
            for (int d = 0; d < DB; ++d) dk[f][d] = dv[f][d] = zn_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        // query blocks of a head that see any of the tile's keys
        const int b0 = j0 < seq.kl ? seq.first(j0) / 32 : 0, nb = j0 < seq.kl ? max(0, (seq.ql + 31) / 32 - b0) : 0;
        const int total = nb * p.group;
        float *side = reinterpret_cast<float *>(lds + kRows);
        float mine = 0.0f;
        auto enter = [&](Stage &sg, int t) {  // block t's tensors and, in the first wave, its rows' lse and delta
            const int g = nb ? t / nb : 0, h = kh * p.group + g, i0 = 32 * (b0 + t - g * nb);
            const bool in = t < total;
            sg.base[0] = p.q + b * p.qs[0] + (in ? h : 0) * p.qs[1];
            sg.base[1] = p.grad_out + b * p.os[0] + (in ? h : 0) * p.os[1];
            sg.load(i0, in ? seq.ql : 0);
            if (wave == 0) {
                const int i = i0 + (lane & 31);
                mine = lane < 32 ? -INFINITY : 0.0f;
                if (in && i < seq.ql) mine = (lane < 32 ? p.lse : p.delta)[((int64_t)b * p.q_heads + h) * p.q_len + i];
                // exp2(s - inf) = 0: a row that sees nothing has no probabilities
                if (lane < 32) mine = mine == -INFINITY ? INFINITY : mine * kLog2e;
            }
        };
        auto leave = [&](Stage &sg, int st) {
#pragma unroll
            for (int j = 0; j < Stage::UPT; ++j) sg.stage(st, j, p.scale_log2);
            if (wave == 0) side[st * 64 + lane] = mine;
        };
        Stage sg(lds, tid, p.dim, p.q, p.qs[2], p.grad_out, p.os[2]);
        enter(sg, 0);
        leave(sg, 0);
        for (int t = 0; t < total; ++t) {
            const int st = t & 1, i0 = 32 * (b0 + t % nb);
            __syncthreads();
            enter(sg, t + 1);
            const int hi = w0 + FK * 16;  // keys of this wave: [w0, hi)
            if (i0 + seq.edge >= hi - 1 && hi <= seq.kl) block<false>(sg, st, side + st * 64, i0, w0, seq, lane, kf, vf, dk, dv);
            else if (min(i0 + 31, seq.ql - 1) + seq.edge >= w0 && w0 < seq.kl) block<true>(sg, st, side + st * 64, i0, w0, seq, lane, kf, vf, dk, dv);
            leave(sg, st ^ 1);
        }

        bool bad = false;
#pragma unroll
        for (int f = 0; f < FK; ++f)
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    bad |= !(__builtin_fabsf(dk[f][d][r]) < INFINITY) || !(__builtin_fabsf(dv[f][d][r]) < INFINITY);
                    dk[f][d][r] *= kSplitUnscale * kLn2;  // Q was scaled by scale * log2 e
                    dv[f][d][r] *= kSplitUnscale;
                }
        if (__builtin_amdgcn_ballot_w64(bad)) {
            for (int j = w0; j < min(w0 + FK * 16, p.kv_len); ++j) mha_row_grad_kv(p, b, kh, j, lane);
            return;
        }
#pragma unroll
        for (int f = 0; f < FK; ++f) {
            const int j = w0 + 16 * f + li;
            if (j >= p.kv_len) continue;
#pragma unroll
            for (int d = 0; d < DB; ++d) {
                mha_store4(p.grad_k + kat + j * p.ks[2], 16 * d + 4 * lh, p.dim, dk[f][d]);
                mha_store4(p.grad_v + kat + j * p.ks[2], 16 * d + 4 * lh, p.dim, dv[f][d]);
            }
        }
    }

    template <bool MASK>
    __device__ static __forceinline__ void block(const Stage &sg, int st, const float *side, int i0, int w0, const MhaSeq &seq,
                                                 int lane, const zn_bf16x8 (&kf)[FK][SL][3], const zn_bf16x8 (&vf)[FK][SL][3],
                                                 zn_f32x4 (&dk)[FK][DB], zn_f32x4 (&dv)[FK][DB]) {
        const int li = lane & 15, lh = lane >> 4;
        zn_f32x4 s[FK][2], dp[FK][2];
#pragma unroll
        for (int f = 0; f < FK; ++f)
#pragma unroll
            for (int rb = 0; rb < 2; ++rb) s[f][rb] = dp[f][rb] = zn_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int sl = 0; sl < SL; ++sl) {
                zn_bf16x8 a[2][3];
#pragma unroll
                for (int rb = 0; rb < 2; ++rb)
#pragma unroll
                    for (int q = 0; q < 3; ++q) a[rb][q] = sg.dims(st, t, q, sl, rb);
#pragma unroll
                for (int pr = 0; pr < 6; ++pr)
#pragma unroll
                    for (int rb = 0; rb < 2; ++rb)
#pragma unroll
                        for (int f = 0; f < FK; ++f) {
                            if (t == 0) s[f][rb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[rb][kMhaPA[pr]], kf[f][sl][kMhaPB[pr]], s[f][rb], 0, 0, 0);
                            else dp[f][rb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[rb][kMhaPA[pr]], vf[f][sl][kMhaPB[pr]], dp[f][rb], 0, 0, 0);
                        }
            }
        zn_f32x4 ml[2], dl[2];
#pragma unroll
        for (int rb = 0; rb < 2; ++rb) {
            ml[rb] = *reinterpret_cast<const zn_f32x4 *>(side + 16 * rb + 4 * lh);
            dl[rb] = *reinterpret_cast<const zn_f32x4 *>(side + 32 + 16 * rb + 4 * lh);
        }
        zn_bf16x8 pf[FK][3], df[FK][3];
#pragma unroll
        for (int f = 0; f < FK; ++f) {
            const int j = w0 + 16 * f + li;
            float x[8], y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[f][e / 4][e % 4], kSplitUnscale, -ml[e / 4][e % 4]));
                y[e] = x[e] * __builtin_fmaf(dp[f][e / 4][e % 4], kSplitUnscale, -dl[e / 4][e % 4]);
                if (MASK && (j >= seq.kl || j > i0 + 16 * (e / 4) + 4 * lh + e % 4 + seq.edge)) x[e] = y[e] = 0.0f;
            }
            zn_u32x4 w[3];
            split8(x, w);
#pragma unroll
            for (int q = 0; q < 3; ++q) pf[f][q] = __builtin_bit_cast(zn_bf16x8, w[q]);
            split8(y, w);
#pragma unroll
            for (int q = 0; q < 3; ++q) df[f][q] = __builtin_bit_cast(zn_bf16x8, w[q]);
        }
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int d = 0; d < DB; ++d) {
                zn_bf16x8 a[3];
#pragma unroll
                for (int q = 0; q < 3; ++q) a[q] = sg.rows(st, 1 - t, q, d);
#pragma unroll
                for (int pr = 0; pr < 6; ++pr)
#pragma unroll
                    for (int f = 0; f < FK; ++f) {
                        zn_f32x4 &x = t ? dk[f][d] : dv[f][d];
                        x = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[kMhaPA[pr]], t ? df[f][kMhaPB[pr]] : pf[f][kMhaPB[pr]], x, 0, 0, 0);
                    }
            }
    }
};

}  // namespace

// Grid: x = sequence and key/value head (its tiles share an XCD's L2), y = tiles.
#define ZN_MHA_KERNELS(DP, NW, FQ, FK)                                                                       \
    extern "C" __global__ __launch_bounds__(NW * 64, 2) void zn_mha_forward_##DP(ZnMhaArgs p) {              \
        typedef MhaQueryTile<DP, NW, FQ, false> T;                                                           \
        __shared__ __attribute__((aligned(1024))) char lds[2 * T::Stage::kStage];                            \
        T::run(p, lds);                                                                                      \
    }                                                                                                        \
    extern "C" __global__ __launch_bounds__(NW * 64, 2) void zn_mha_grad_q_##DP(ZnMhaArgs p) {               \
        typedef MhaQueryTile<DP, NW, FQ, true> T;                                                            \
        __shared__ __attribute__((aligned(1024))) char lds[2 * T::Stage::kStage];                            \
        T::run(p, lds);                                                                                      \
    }                                                                                                        \
    extern "C" __global__ __launch_bounds__(NW * 64, 2) void zn_mha_grad_kv_##DP(ZnMhaArgs p) {              \
        typedef MhaKeyTile<DP, NW, FK> T;                                                                    \
        __shared__ __attribute__((aligned(1024))) char lds[T::kBytes];                                       \
        T::run(p, lds);                                                                                      \
    }
ZN_MHA_KERNELS(32, 4, 2, 2)
ZN_MHA_KERNELS(64, 4, 2, 2)
ZN_MHA_KERNELS(96, 8, 1, 1)
ZN_MHA_KERNELS(128, 8, 1, 1)

#endif
