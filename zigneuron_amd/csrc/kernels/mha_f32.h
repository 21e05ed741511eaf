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

#include <type_traits>

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
// below take these rows where a value or a sum is not finite.  That is tens of
// times slower, so a walk whose result is NaN already ends: tensors full of NaN,
// as a diverged step has them, cost little more than others (8 heads (4) of 1500
// x 64, causal, a forward and a backward: 9.4 ms when all was walked, 0.22 so,
// 0.12 without NaN).

// A row's walk over keys [from, to): running maximum (log2 domain), sum and O.
struct MhaRowState {
    float m = -INFINITY, l = 0.0f, oa = 0.0f, ob = 0.0f;
    __device__ __forceinline__ void walk(const ZnMhaArgs &p, int b, int h, int i, int from, int to, int lane) {
        const float *k = p.k + b * p.ks[0] + (h / p.group) * p.ks[1], *v = p.v + b * p.ks[0] + (h / p.group) * p.ks[1];
        MhaRow q(p.q + b * p.qs[0] + h * p.qs[1] + i * p.qs[2], from < to ? p.dim : 0, lane);
        q.a *= p.scale_log2;
        q.b *= p.scale_log2;
        for (int j = from; j < to && l == l; ++j) {  // a NaN sum stays one, and all of O with it
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

// Where sums go: to the tensor's row, or to the row's part z (of the walk that the workgroup takes).
__device__ __forceinline__ float *mha_query_part(const ZnMhaArgs &p, int64_t row, int z) { return p.part + (row * p.splits + z) * p.part_ld; }
__device__ __forceinline__ float *mha_key_part(const ZnMhaArgs &p, int64_t row, int z) { return p.kv_part + (row * p.kv_splits + z) * p.part_ld; }
__device__ __forceinline__ int64_t mha_query_row(const ZnMhaArgs &p, int b, int h, int i) { return ((int64_t)b * p.q_heads + h) * p.q_len + i; }
// ... dK's key rows, then dV's
__device__ __forceinline__ int64_t mha_key_row(const ZnMhaArgs &p, int b, int kh, int j, bool v) {
    return (((int64_t)(v ? p.batch : 0) + b) * p.kv_heads + kh) * p.kv_len + j;
}

// O and lse of a row from its sums, or its part: dims lane and lane + 64.
__device__ __forceinline__ void mha_row_finish(const ZnMhaArgs &p, int b, int h, int i, int z, int lane, float m, float l, float oa, float ob) {
    if (p.splits > 1) {
        float *part = mha_query_part(p, mha_query_row(p, b, h, i), z);
        MhaRow::store(part, p.dim, lane, oa, ob);
        if (lane == 0) {
            part[p.part_ld - 4] = m;
            part[p.part_ld - 3] = l;
        }
        return;
    }
    const float r = l == 0.0f ? 1.0f : l;
    MhaRow::store(p.out + b * p.os[0] + h * p.os[1] + i * p.os[2], p.dim, lane, oa / r, ob / r);
    if (p.lse && lane == 0) p.lse[mha_query_row(p, b, h, i)] = mha_lse(m, l);
}

// A row's walk over keys [from, to), those of them that it sees.
__device__ __forceinline__ void mha_row_forward(const ZnMhaArgs &p, int b, int h, int i, int z, int from, int to, int lane) {
    MhaRowState s;
    s.walk(p, b, h, i, from, min(to, MhaSeq(p, b).seen(i)), lane);
    mha_row_finish(p, b, h, i, z, lane, s.m, s.l, s.oa, s.ob);
}

// What the backward keeps of each query beside Q and dO, 32 values each a block:
//   [0]   lse in the log2 domain, +inf where the query sees nothing, NaN where it is far
//   [32]  delta
//   [64], [96]  a and r of P = exp2(S - a) r: lse and 1 or, of a far query, its maximum and 1 / its sum
// An lse's last bit is a relative error of the whole row's probabilities: from
// 2^16 (log2 domain) on, half of it is past 2^-9, and from 2^24 on nothing is left
// of them.  Such a query is far: the split kernel goes over its scores again, one
// key at a time, and its NaN makes the tiles' sums NaN, so that all that it
// reaches is computed row by row, with scores of the very same bits as its maximum.
constexpr int kMhaSide = 128;  // values a block
constexpr float kMhaFar = 65536.0f;
__device__ __forceinline__ const float *mha_side(const ZnMhaArgs &p, int b, int h, int i) {
    return p.side + (((int64_t)b * p.q_heads + h) * p.q_blocks + i / 32) * kMhaSide + i % 32;
}

// grad_q of a row over keys [from, to).
__device__ __forceinline__ void mha_row_grad_q(const ZnMhaArgs &p, int b, int h, int i, int z, int from, int to, int lane) {
    const MhaSeq seq(p, b);
    int n = min(to, seq.seen(i));
    const float *side = mha_side(p, b, h, i);
    if (from < n && side[0] == INFINITY) n = from;
    const bool some = from < n;
    const float delta = some ? side[32] : 0.0f, a = some ? side[64] : 0.0f, r = some ? side[96] : 0.0f;
    const float *k = p.k + b * p.ks[0] + (h / p.group) * p.ks[1], *v = p.v + b * p.ks[0] + (h / p.group) * p.ks[1];
    const int64_t qat = b * p.qs[0] + h * p.qs[1] + i * p.qs[2];
    MhaRow q(p.q + qat, from < n ? p.dim : 0, lane);
    const MhaRow g(p.grad_out + b * p.os[0] + h * p.os[1] + i * p.os[2], from < n ? p.dim : 0, lane);
    q.a *= p.scale_log2;
    q.b *= p.scale_log2;
    float ga = 0.0f, gb = 0.0f;
    if (r != r || delta != delta) {  // NaN in every product
        ga = gb = __builtin_nanf("");
        n = from;
    }
    for (int j = from; j < n; ++j) {
        const MhaRow kr(k + j * p.ks[2], p.dim, lane), vr(v + j * p.ks[2], p.dim, lane);
        const float ds = __builtin_amdgcn_exp2f(q.dot(kr) - a) * r * (g.dot(vr) - delta);
        ga += ds * kr.a;
        gb += ds * kr.b;
    }
    if (p.splits > 1) MhaRow::store(mha_query_part(p, mha_query_row(p, b, h, i), z), p.dim, lane, ga, gb);
    else MhaRow::store(p.grad_q + qat, p.dim, lane, ga * p.scale, gb * p.scale);
}

// grad_k and grad_v of a row over the query blocks [from, to) of its tile's walk: nb blocks from b0 of each query head of the
// group, the heads in order, the queries ascending.
__device__ __forceinline__ void mha_row_grad_kv(const ZnMhaArgs &p, int b, int kh, int j, int z, int b0, int nb, int from, int to, int lane) {
    const MhaSeq seq(p, b);
    const bool in = j < seq.kl;
    const int64_t kat = b * p.ks[0] + kh * p.ks[1] + j * p.ks[2];
    const MhaRow kr(p.k + kat, in ? p.dim : 0, lane), vr(p.v + kat, in ? p.dim : 0, lane);
    float ka = 0.0f, kb = 0.0f, va = 0.0f, vb = 0.0f;
    // a query whose sum is NaN makes NaN of every dim
    for (int t = from; in && t < to; ++t) {
        const int g = t / nb, i = 32 * (b0 + t - g * nb) + lane % 32;
        const bool nan = i >= seq.first(j) && i < seq.ql && __builtin_isnan(mha_side(p, b, kh * p.group + g, min(i, p.q_len - 1))[96]);
        if (!__builtin_amdgcn_ballot_w64(nan)) continue;
        ka = kb = va = vb = __builtin_nanf("");
        to = from;
    }
    for (int t = from; in && t < to; ++t) {
        const int g = t / nb, h = kh * p.group + g, i0 = 32 * (b0 + t - g * nb);
        for (int i = max(i0, seq.first(j)); i < min(i0 + 32, seq.ql); ++i) {
            const float *side = mha_side(p, b, h, i);
            if (side[0] == INFINITY) continue;
            const MhaRow q(p.q + b * p.qs[0] + h * p.qs[1] + i * p.qs[2], p.dim, lane);
            const MhaRow d(p.grad_out + b * p.os[0] + h * p.os[1] + i * p.os[2], p.dim, lane);
            const float s = wave_sum((q.a * p.scale_log2) * kr.a + (q.b * p.scale_log2) * kr.b);
            const float e = __builtin_amdgcn_exp2f(s - side[64]) * side[96];
            const float ds = e * (d.dot(vr) - side[32]);
            va += e * d.a;
            vb += e * d.b;
            ka += ds * q.a;
            kb += ds * q.b;
        }
    }
    const bool part = p.kv_splits > 1;
    MhaRow::store(part ? mha_key_part(p, mha_key_row(p, b, kh, j, false), z) : p.grad_k + kat, p.dim, lane, ka * p.scale, kb * p.scale);
    MhaRow::store(part ? mha_key_part(p, mha_key_row(p, b, kh, j, true), z) : p.grad_v + kat, p.dim, lane, va, vb);
}

// ------------------------------------------------------------------- tiles
// The same on the bf16 matrix cores, every operand value split into three bf16
// parts (zn_split.h).  One side of the products stays in a wave's registers
// (queries for O and dQ, keys for dK and dV); the other side's two tensors
// (K and V, or Q and dO) come past in blocks of 32 rows, staged in LDS, two
// stages.
//
// A staged tensor serves products over its dims and over its rows: rows lie
// in slices of 32 dims, a row's 64 bytes as four 16-byte chunks, chunk c the
// dims 4c .. 4c + 3 and 16 + 4c .. 16 + 4c + 3 of the slice.  A fragment over
// dims is one ds_read_b128; one over rows comes from two transposing reads
// (ds_read_b64_tr_b16), whose 4 x 16 blocks are the halves of the chunks.  The
// same chunk order over rows is that of the accumulators: the two 16-row
// blocks of S that a lane holds are its fragment of the next product.
//
// The splitting is 6.5 vector instructions a value.  Where a tensor goes past
// many tiles it is split once, by a kernel of its own, into an image of the
// staged blocks (10 bytes of traffic a value), which the tiles then bring to LDS
// by DMA (MhaImageStage).  Where it goes past few, the thread that loads a value
// splits it (MhaRawStage).
//
// What bounds the gradients' tiles is the matrix cores: six bf16 products for one
// fp32 product, at a clock that the power limit holds near 2 GHz while they are
// 68 to 73% busy (the largest split GEMM 74%).  The causal forward's are 56%
// busy: the softmax and the split of P are 1.5 vector instructions a product, and
// the edge's blocks are half masked.  MI355X, forward of 2 x 16 heads (4
// key/value) of 2048 x 128, causal: 171 us with the split, 201 TFLOP/s of fp32
// products; both gradients of 2 x 32 heads (8) of 4096 x 128, causal, 4.23 ms, 162
// TFLOP/s; of 8 x 16 heads of 1024 x 64, 552 us, 156 TFLOP/s.
//
// Sums stand at 2^48 times their value, so that nothing of a split is lost: one
// beyond 2^80 or so, an infinity or a NaN (visible, or masked for some rows
// of a block only, where it meets a probability of 0) makes a sum that is not
// finite, and the wave then takes its rows one at a time.  A score below -2^80
// becomes -inf, which says the same as its probability of 0, unless the row sees
// nothing above it: the forward then finds a maximum of -inf where keys were
// visible, and in the backward the row's lse is far (mha_side).
template <int DP>
struct MhaBlock {
    static constexpr int BR = 32, SL = DP / 32, DB = DP / 16;
    static constexpr int kPart = BR * DP * 2;    // bytes of one bf16 part of a tensor's block
    static constexpr int kImage = 3 * kPart;     // of a block
    static constexpr int kStage = 2 * kImage;    // of two tensors' blocks

    __device__ static __forceinline__ int slot(int r, int c) { return r * 64 + ((c ^ (-(r >> 2) & 3)) << 4); }
    // Where row r of a block has chunk lh of slice sl, part q.
    __device__ static __forceinline__ int place(int r, int lh, int sl, int q) { return q * kPart + sl * (BR * 64) + slot(r, lh); }
};

// Six fragments: over dims rows 0 .. 15 and 16 .. 31, over rows two blocks of 16 dims, three parts each.
typedef zn_bf16x8 MhaSix[2][3];

// Fragments of a staged block.
template <int DP>
struct MhaFrags : MhaBlock<DP> {
    typedef MhaBlock<DP> B;
    const char *lds;
    int frag, tr[2];  // this lane's place in a fragment over dims, over rows (even and odd blocks of dims)
    __device__ __forceinline__ MhaFrags(const char *lds, int lane) : lds(lds) {
        frag = B::slot(lane & 15, lane >> 4);
        tr[0] = B::slot(4 * (lane >> 4) + (lane & 15) / 4, lane % 4 / 2) + lane % 2 * 8;
        tr[1] = tr[0] ^ 32;
    }
    // The first of the 4 dims of block db that a lane of quarter lh has in an accumulator whose rows are dims.
    __device__ static __forceinline__ int dim_of(int db, int lh) { return 32 * (db / 2) + 8 * (db & 1) + 4 * (lh / 2) + 16 * (lh & 1); }
    // Part q of tensor t: rows 16 rb + li, chunk lh of slice sl
    __device__ __forceinline__ zn_bf16x8 dims(int st, int t, int q, int sl, int rb) const {
        return __builtin_bit_cast(zn_bf16x8, *reinterpret_cast<const zn_u32x4 *>(lds + st * B::kStage + t * B::kImage + q * B::kPart +
                                                                                sl * (B::BR * 64) + rb * (16 * 64) + frag));
    }
    __device__ __forceinline__ void dims(int st, int t, int sl, MhaSix &a) const {
#pragma unroll
        for (int q = 2; q >= 0; --q)  // in the order of their use
#pragma unroll
            for (int rb = 0; rb < 2; ++rb) a[rb][q] = dims(st, t, q, sl, rb);
    }
    __device__ __forceinline__ void dims(int st, int t, int sl, int q, MhaSix &a) const {
#pragma unroll
        for (int rb = 0; rb < 2; ++rb) a[rb][q] = dims(st, t, q, sl, rb);
    }
    // ... 16 dims of block db (chunks 0 and 1 of its slice, or 2 and 3), rows 4 lh .. 4 lh + 3 and 16 + 4 lh .. 16 + 4 lh + 3.
    // Whole chunks: the 4 rows of a 16-lane group leave the other half of the banks to the next group's (rotated) chunks; the
    // first or second halves of all four chunks met in half of the banks (a third of the LDS cycles were conflicts).
    __device__ __forceinline__ zn_bf16x8 rows(int st, int t, int q, int db) const {
        typedef short s4 __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) s4 ls4;
        const char *at = lds + st * B::kStage + t * B::kImage + q * B::kPart + (db / 2) * (B::BR * 64) + tr[db & 1];
        const s4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ls4 *)at), b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ls4 *)(at + 16 * 64));
        return __builtin_bit_cast(zn_bf16x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
    }
    __device__ __forceinline__ void rows(int st, int t, int db, MhaSix &a) const {
#pragma unroll
        for (int q = 2; q >= 0; --q)
#pragma unroll
            for (int c = 0; c < 2; ++c) a[c][q] = rows(st, t, q, db + c);
    }
    __device__ __forceinline__ void rows(int st, int t, int db, int q, MhaSix &a) const {
#pragma unroll
        for (int c = 0; c < 2; ++c) a[c][q] = rows(st, t, q, db + c);
    }
};

// A pointer that is the same in the whole wave, in scalar registers, where inline assembly takes its descriptor from.
__device__ __forceinline__ const float *mha_uniform(const void *p) {
    const uint64_t x = reinterpret_cast<uint64_t>(p);
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)x), hi = __builtin_amdgcn_readfirstlane((uint32_t)(x >> 32));
    return reinterpret_cast<const float *>((uint64_t)hi << 32 | lo);
}

// Blocks of two tensors from their images, NW waves.
template <int DP, int NW>
struct MhaImageStage {
    typedef MhaBlock<DP> B;
    static constexpr int kChunks = B::kImage / 1024;  // wave instructions a tensor
    char *lds;
    const char *x, *y;  // the images of the current heads
    int wave;
    uint32_t lane16;
    __device__ __forceinline__ MhaImageStage(char *lds, int tid, const char *x, const char *y) : lds(lds), x(x), y(y) {
        wave = __builtin_amdgcn_readfirstlane(tid / kWave);
        lane16 = (tid & (kWave - 1)) * 16;
    }
    // buffer_load ... lds, as DmaStage issues it: 1 KB at LDS address `to` from byte `at` of r
    __device__ static __forceinline__ void dma(__amdgpu_buffer_rsrc_t r, char *to, uint32_t lane16, uint32_t at) {
        const uint32_t m0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(zn_lds_void *)to);
        asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" : : "s"(m0), "v"(lane16), "s"(r), "s"(at) : "memory");
    }
    __device__ __forceinline__ void fetch(int st, int blk) {
        const __amdgpu_buffer_rsrc_t rx = make_rsrc(mha_uniform(x + (int64_t)blk * B::kImage), B::kImage);
        const __amdgpu_buffer_rsrc_t ry = make_rsrc(mha_uniform(y + (int64_t)blk * B::kImage), B::kImage);
#pragma unroll
        for (int i = 0; i < (2 * kChunks + NW - 1) / NW; ++i) {
            const int c = i * NW + wave;
            char *to = lds + st * B::kStage + c * 1024;
            if (c < kChunks) dma(rx, to, lane16, (uint32_t)c * 1024u);
            else if (c < 2 * kChunks) dma(ry, to, lane16, (uint32_t)(c - kChunks) * 1024u);
        }
    }
    // Wait for the blocks on their way: vmcnt(0) as a builtin, which the compiler counts.  Its own loads before the loop are then
    // known to be done; with the wait in inline assembly it waits for them again inside the loop, and so for the blocks just asked for.
    __device__ __forceinline__ void arrive() {
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(0x0f70);
        asm volatile("" ::: "memory");
    }
    __device__ __forceinline__ void commit(int) {}
};

// Blocks of K and V from the tensors themselves.
template <int DP, int NW>
struct MhaRawStage {
    typedef MhaBlock<DP> B;
    static constexpr int NT = NW * kWave;
    static constexpr int kUnits = B::BR * DP / 4;  // staging units of 8 values: the first tensor's, then the second's
    static constexpr int UPT = (kUnits + NT - 1) / NT;
    static_assert(kUnits / 2 % kWave == 0, "a wave's units are all of one tensor");

    char *lds;
    const float *src[2];
    int64_t stride;
    int dim, tid, end;  // rows from `end` on are zeros
    float g[UPT][8];

    __device__ __forceinline__ MhaRawStage(char *lds, int tid, const float *x, const float *y, int64_t stride, int dim, int end)
        : lds(lds), src{x, y}, stride(stride), dim(dim), tid(tid), end(end) {}
    // Unit j's tensor, row, slice and chunk.
    __device__ __forceinline__ void unit(int j, bool &second, int &row, int &sl, int &c) const {
        const int u = j * NT + tid;
        second = __builtin_amdgcn_readfirstlane(u) >= kUnits / 2;
        const int v = second ? u - kUnits / 2 : u, dc = v % (DP / 8);
        row = v / (DP / 8);
        sl = dc / 4;
        c = dc % 4;
    }
    __device__ __forceinline__ void fetch(int, int blk) {
        const int r0 = blk * B::BR, n = min(B::BR, end - r0);
        const uint32_t bytes = n > 0 ? (uint32_t)((n - 1) * (int)stride + dim) * 4u : 0u;
        __amdgpu_buffer_rsrc_t r[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) r[t] = make_rsrc(src[t] + (n > 0 ? (int64_t)r0 * stride : 0), bytes);
#pragma unroll
        for (int j = 0; j < UPT; ++j) {
            if (j * NT + tid >= kUnits) continue;  // whole waves
            bool second;
            int row, sl, c;
            unit(j, second, row, sl, c);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int d = 32 * sl + 4 * c + 16 * h;
                const uint32_t o = d < dim ? (uint32_t)(row * (int)stride + d) * 4u : kOutOfRange;
                const zn_f32x4 v = __builtin_bit_cast(zn_f32x4, __builtin_amdgcn_raw_buffer_load_b128(second ? r[1] : r[0], o, 0, 0));
#pragma unroll
                for (int e = 0; e < 4; ++e) g[j][4 * h + e] = d + e < dim ? v[e] : 0.0f;
            }
        }
    }
    __device__ __forceinline__ void arrive() {}
    __device__ __forceinline__ void commit(int st) {
#pragma unroll
        for (int j = 0; j < UPT; ++j) {
            if (j * NT + tid >= kUnits) continue;
            bool second;
            int row, sl, c;
            unit(j, second, row, sl, c);
            zn_u32x4 w[3];
            split8(g[j], w);
#pragma unroll
            for (int q = 0; q < 3; ++q)
                *reinterpret_cast<zn_u32x4 *>(lds + st * B::kStage + (second ? B::kImage : 0) + B::place(row, c, sl, q)) = w[q];
        }
    }
};

// The instruction order of a group's M products, the R fragment reads of the
// next group spread between them: left alone the compiler reads a fragment
// right before its use and waits out the whole latency (128 dims, dQ: 1.03e9
// CU cycles, so 0.91e9).
template <int M, int R>
__device__ __forceinline__ void mha_order() {
#pragma unroll
    for (int i = 0; i < R; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x8, M / R, 0);  // MFMA
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);    // LDS read
    }
    __builtin_amdgcn_sched_barrier(0);
}

// The same with one set of fragments: a part's last product frees its
// registers for the next group's (load(part)), requested 6 F to 10 F products
// before their use.  x(c, f) += a[c] . b(f) for c < 2, f < F.  READS: LDS reads
// of a part.  FLUSH: the six products are summed from zero and then added, one
// rounding of a long sum per block instead of six (4 heads of 4096 x 128 on a
// key/value head, against 64 bits: dK 1.9e-6 -> 8e-7).  For the key tiles, which two sets make spill (and a reload from
// scratch waits for the blocks on their way too).
template <int F, int READS, bool FLUSH, typename Acc, typename Operand, typename Load>
__device__ __forceinline__ void mha_group(MhaSix &a, Acc x, Operand b, Load load) {
    zn_f32x4 t[2][F];
    auto products = [&](auto count) {  // part 3 - count of a with parts count - 1 .. 0 of b
        constexpr int N = decltype(count)::value, P = 3 - N;
#pragma unroll
        for (int q = N - 1; q >= 0; --q)
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int f = 0; f < F; ++f) {
                    zn_f32x4 &y = FLUSH ? t[c][f] : x(c, f);
                    y = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[c][P], b(f)[q], FLUSH && N == 1 ? zn_f32x4{0.0f, 0.0f, 0.0f, 0.0f} : y, 0, 0, 0);
                }
        load(P);
        __builtin_amdgcn_sched_group_barrier(0x8, 2 * F * N, 0);                         // MFMA
        if constexpr (READS > 0) __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);  // LDS read
    };
    products(std::integral_constant<int, 1>());
    products(std::integral_constant<int, 2>());
    products(std::integral_constant<int, 3>());
    if constexpr (FLUSH) {
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int f = 0; f < F; ++f) x(c, f) += t[c][f];
    }
    __builtin_amdgcn_sched_barrier(0);
}

// Probabilities (or dS) times kSplitScale to the parts of a fragment.  The factor is a product of its own behind the
// exponential, or another factor's: in the exponent's argument it would round the largest probabilities' near 24, to 2^-20
// (a probability of an even row 6 to 9 half steps off in the mean, 1 to 1.5 so).
__device__ __forceinline__ void mha_split8(const float (&x)[8], zn_bf16x8 (&f)[3]) {
    zn_u32x4 w[3];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        uint32_t hi, mid, lo;
        split_scaled(x[2 * e], x[2 * e + 1], hi, mid, lo);
        w[0][e] = hi;
        w[1][e] = mid;
        w[2][e] = lo;
    }
#pragma unroll
    for (int q = 0; q < 3; ++q) f[q] = __builtin_bit_cast(zn_bf16x8, w[q]);
}

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

// O and lse (BACK false, K and V split here or before) or dQ (BACK true, everything split before) of NW x FQ x 16 query rows.
template <int DP, int NW, int FQ, bool BACK, bool IMAGE>
struct MhaQueryTile {
    typedef MhaFrags<DP> Frags;
    typedef typename std::conditional<IMAGE, MhaImageStage<DP, NW>, MhaRawStage<DP, NW>>::type Stage;
    static constexpr int SL = Frags::SL, DB = Frags::DB;
    static constexpr int kBytes = 2 * Frags::kStage;
    static_assert(IMAGE || !BACK, "the backward's tensors are all split before");

    // Tile y, part z of its walk: causal rows see more the later they come, so the last tiles of each head come first.
    __device__ static __forceinline__ void run(const ZnMhaArgs &p, int y, int z, char *lds) {
        const int tid = threadIdx.x, lane = tid & (kWave - 1);
        const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
        const int li = lane & 15, lh = lane >> 4;
        const int b = blockIdx.x / p.kv_heads, kh = blockIdx.x - b * p.kv_heads;
        const int rows = p.group * p.q_len, per = p.query_tiles / p.group;
        const int r0 = (y % p.group * per + per - 1 - y / p.group) * (NW * FQ * 16), w0 = r0 + wave * FQ * 16;
        if (r0 >= rows) return;
        const MhaSeq seq(p, b);

        // keys that the tile's rows see: none past `last`; the wave's rows all see those before `all`
        int lim[FQ], all = INT_MAX, any = 0;
        zn_bf16x8 qf[FQ][SL][3], gf[BACK ? FQ : 1][SL][3];
        float lse2[FQ], delta[FQ];
#pragma unroll
        for (int f = 0; f < FQ; ++f) {
            const MhaQuery r(p, kh, w0 + 16 * f + li);
            lim[f] = r.in ? seq.seen(r.i) : 0;
            if constexpr (BACK) {
                const float *side = mha_side(p, b, r.h, r.i);
                lse2[f] = lim[f] ? side[0] : INFINITY;
                delta[f] = lim[f] ? side[32] * kSplitScale : 0.0f;
                const int64_t at = (((int64_t)b * p.q_heads + r.h) * p.q_blocks + r.i / 32) * Frags::kImage;
#pragma unroll
                for (int sl = 0; sl < SL; ++sl)
#pragma unroll
                    for (int q = 0; q < 3; ++q) {
                        const int64_t o = at + Frags::place(r.i % 32, lh, sl, q);
                        zn_u32x4 x = {0, 0, 0, 0}, y = {0, 0, 0, 0};
                        if (lim[f]) {
                            x = *reinterpret_cast<const zn_u32x4 *>(p.qi + o);
                            y = *reinterpret_cast<const zn_u32x4 *>(p.gi + o);
                        }
                        qf[f][sl][q] = __builtin_bit_cast(zn_bf16x8, x);
                        gf[f][sl][q] = __builtin_bit_cast(zn_bf16x8, y);
                    }
            } else {
                mha_row_frags<SL>(lim[f] ? p.q + b * p.qs[0] + r.h * p.qs[1] + r.i * p.qs[2] : nullptr, p.dim, lh, p.scale_log2, qf[f]);
            }
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

        const Frags fr(lds, lane);
        // the part's share of the blocks
        const int all_blocks = (last + 31) / 32, share = (all_blocks + p.splits - 1) / p.splits;
        const int blk0 = __builtin_amdgcn_readfirstlane(min(z * share, all_blocks)), nblk = __builtin_amdgcn_readfirstlane(min(blk0 + share, all_blocks));
        auto walk = [&](Stage sg) {
            if (blk0 < nblk) {
                sg.fetch(0, blk0);
                sg.commit(0);
            }
            for (int blk = blk0; blk < nblk; ++blk) {
                const int st = (blk - blk0) & 1, k0 = 32 * blk;
                sg.arrive();
                __syncthreads();  // block blk is in LDS; every wave is done with block blk - 1
                if (blk + 1 < nblk) sg.fetch(st ^ 1, blk + 1);
                if (k0 < any) block(fr, st, k0 + 32 > all, k0, lane, lim, qf, gf, lse2, delta, o, m, l);
                if (blk + 1 < nblk) sg.commit(st ^ 1);
            }
        };
        if constexpr (IMAGE) {
            const int64_t at = ((int64_t)b * p.kv_heads + kh) * p.k_blocks * Frags::kImage;
            walk(Stage(lds, tid, p.ki + at, p.vi + at));
        } else {
            const int64_t at = b * p.ks[0] + kh * p.ks[1];
            walk(Stage(lds, tid, p.k + at, p.v + at, p.ks[2], p.dim, seq.kl));
        }

        bool bad = false;
#pragma unroll
        for (int f = 0; f < FQ; ++f) {
            bad |= !BACK && (!(l[f] < INFINITY) || (m[f] == -INFINITY && blk0 < nblk && lim[f] > 32 * blk0));
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
                if constexpr (BACK) mha_row_grad_q(p, b, r.h, r.i, z, 32 * blk0, 32 * nblk, lane);
                else mha_row_forward(p, b, r.h, r.i, z, 32 * blk0, 32 * nblk, lane);
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
            if (p.splits > 1) {
                float *part = mha_query_part(p, mha_query_row(p, b, r.h, r.i), z);
#pragma unroll
                for (int d = 0; d < DB; ++d) mha_store4(part, Frags::dim_of(d, lh), p.dim, o[f][d]);
                if (!BACK && lh == 0) {
                    part[p.part_ld - 4] = m[f];
                    part[p.part_ld - 3] = sum;
                }
                continue;
            }
            float *row = BACK ? p.grad_q + b * p.qs[0] + r.h * p.qs[1] + r.i * p.qs[2]
                              : p.out + b * p.os[0] + r.h * p.os[1] + r.i * p.os[2];
            if (!BACK && p.lse && lh == 0) p.lse[mha_query_row(p, b, r.h, r.i)] = mha_lse(m[f], sum);
            const float div = BACK ? 1.0f : (sum == 0.0f ? 1.0f : sum);
#pragma unroll
            for (int d = 0; d < DB; ++d) {
                const zn_f32x4 x = BACK ? o[f][d] * p.scale : o[f][d] / div;
                mha_store4(row, Frags::dim_of(d, lh), p.dim, x);
            }
        }
    }

    // One block of 32 keys: S^T = K (cQ)^T (and dP^T = V dO^T), then O^T += V^T P^T or dQ^T += K^T dS^T.
    // `mask` (of the whole wave): some of its pairs are masked.  One code for both, as MhaKeyTile's.
    __device__ static __forceinline__ void block(const Frags &sg, int st, bool mask, int k0, int lane, const int (&lim)[FQ],
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
        MhaSix a[2];
        constexpr int ND = (BACK ? 2 : 1) * SL, NR = DB / 2;  // groups of products over dims, over rows
        sg.dims(st, 0, 0, a[0]);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < ND; ++i) {
            const int t = i / SL, sl = i % SL;
            if (i + 1 < ND) sg.dims(st, (i + 1) / SL, (i + 1) % SL, a[(i + 1) & 1]);
            else sg.rows(st, BACK ? 0 : 1, 0, a[(i + 1) & 1]);
#pragma unroll
            for (int pr = 0; pr < 6; ++pr)
#pragma unroll
                for (int rb = 0; rb < 2; ++rb)
#pragma unroll
                    for (int f = 0; f < FQ; ++f) {
                        zn_f32x4 &x = t ? dp[BACK ? f : 0][rb] : s[f][rb];
                        x = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i & 1][rb][kMhaPA[pr]], t ? gf[BACK ? f : 0][sl][kMhaPB[pr]] : qf[f][sl][kMhaPB[pr]], x, 0, 0, 0);
                    }
            if (i + 1 < ND) mha_order<12 * FQ, 6>();
            else mha_order<12 * FQ, 12>();
        }
        if (mask) {
#pragma unroll
            for (int f = 0; f < FQ; ++f)
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (k0 + 16 * (e / 4) + 4 * lh + e % 4 >= lim[f]) s[f][e / 4][e % 4] = -INFINITY;
        }
        zn_bf16x8 pf[FQ][3];
#pragma unroll
        for (int f = 0; f < FQ; ++f) {
            float x[8];
            if constexpr (BACK) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float pe = __builtin_amdgcn_exp2f(__builtin_fmaf(s[f][e / 4][e % 4], kSplitUnscale, -lse2[f]));
                    const float de = __builtin_fmaf(dp[f][e / 4][e % 4], kSplitUnscale * kSplitScale, -delta[f]);  // times kSplitScale
                    x[e] = pe * de;
                }
            } else {
                float mb = -INFINITY;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    mb = fmaxf(mb, s[f][e / 4][e % 4]);
                }
                const float mn = fmaxf(m[f], max_over_rows(mb) * kSplitUnscale);
                const float ref = mn == -INFINITY ? 0.0f : mn;  // nothing seen so far
                const float alpha = __builtin_amdgcn_exp2f(m[f] - ref);
                float rs = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    x[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[f][e / 4][e % 4], kSplitUnscale, -ref));
                    rs += x[e];
                    x[e] *= kSplitScale;
                }
                l[f] = l[f] * alpha + rs;
                m[f] = mn;
                if (__builtin_amdgcn_ballot_w64(alpha != 1.0f)) {
#pragma unroll
                    for (int d = 0; d < DB; ++d) o[f][d] *= alpha;
                }
            }
            mha_split8(x, pf[f]);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            if (i + 1 < NR) sg.rows(st, BACK ? 0 : 1, 2 * (i + 1), a[(ND + i + 1) & 1]);
#pragma unroll
            for (int pr = 0; pr < 6; ++pr)
#pragma unroll
                for (int c = 0; c < 2; ++c)
#pragma unroll
                    for (int f = 0; f < FQ; ++f)
                        o[f][2 * i + c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[(ND + i) & 1][c][kMhaPA[pr]], pf[f][kMhaPB[pr]], o[f][2 * i + c], 0, 0, 0);
            mha_order<12 * FQ, 12>();
        }
    }
};

// dK and dV of NW x FK x 16 keys: the group's query heads in order, their
// queries ascending in blocks of 32 (Q scaled, dO, and each row's lse and delta
// in LDS).  S = (cQ) K^T and dP = dO V^T, dV^T += dO^T P and dK^T += Q^T dS.
template <int DP, int NW, int FK>
struct MhaKeyTile {
    typedef MhaFrags<DP> Frags;
    static constexpr int SL = Frags::SL, DB = Frags::DB;
    static constexpr int kSide = 2 * Frags::kStage;  // lse and delta of two stages' rows: [stage][lse, delta][32]
    static constexpr int kBytes = kSide + 2 * 64 * 4;

    __device__ static __forceinline__ void run(const ZnMhaArgs &p, int y, int z, char *lds) {
        const int tid = threadIdx.x, lane = tid & (kWave - 1);
        const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
        const int li = lane & 15, lh = lane >> 4;
        const int b = blockIdx.x / p.kv_heads, kh = blockIdx.x - b * p.kv_heads;
        const int j0 = y * (NW * FK * 16), w0 = j0 + wave * FK * 16;
        const MhaSeq seq(p, b);
        const int ql = __builtin_amdgcn_readfirstlane(seq.ql), kl = __builtin_amdgcn_readfirstlane(seq.kl);
        const int edge = __builtin_amdgcn_readfirstlane(seq.edge);
        const int64_t kat = b * p.ks[0] + kh * p.ks[1];

        zn_bf16x8 kf[FK][SL][3], vf[FK][SL][3];
        zn_f32x4 dk[FK][DB], dv[FK][DB];
#pragma unroll
        for (int f = 0; f < FK; ++f) {
            const int j = w0 + 16 * f + li;
            const int64_t at = (((int64_t)b * p.kv_heads + kh) * p.k_blocks + j / 32) * Frags::kImage;
#pragma unroll
            for (int sl = 0; sl < SL; ++sl)
#pragma unroll
                for (int q = 0; q < 3; ++q) {
                    const int64_t o = at + Frags::place(j % 32, lh, sl, q);
                    zn_u32x4 x = {0, 0, 0, 0}, y = {0, 0, 0, 0};
                    if (j < kl) {
                        x = *reinterpret_cast<const zn_u32x4 *>(p.ki + o);
                        y = *reinterpret_cast<const zn_u32x4 *>(p.vi + o);
                    }
                    kf[f][sl][q] = __builtin_bit_cast(zn_bf16x8, x);
                    vf[f][sl][q] = __builtin_bit_cast(zn_bf16x8, y);
                }
#pragma unroll
            for (int d = 0; d < DB; ++d) dk[f][d] = dv[f][d] = zn_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        // query blocks of a head that see any of the tile's keys
        const int b0 = j0 < kl ? max(0, j0 - edge) / 32 : 0, nb = j0 < kl ? max(0, (ql + 31) / 32 - b0) : 0;
        // the part's share of the blocks of all the group's heads
        const int share = (nb * p.group + p.kv_splits - 1) / p.kv_splits;
        const int from = __builtin_amdgcn_readfirstlane(min(z * share, nb * p.group));
        const int total = __builtin_amdgcn_readfirstlane(min(from + share, nb * p.group));
        const float *side = reinterpret_cast<const float *>(lds + kSide);
        const int64_t head0 = ((int64_t)b * p.q_heads + kh * p.group) * p.q_blocks;  // the group's first query block
        const char *const qi = p.qi + head0 * Frags::kImage, *const gi = p.gi + head0 * Frags::kImage;
        const float *const sides = p.side + head0 * kMhaSide;
        const int q_blocks = p.q_blocks;
        MhaImageStage<DP, NW> sg(lds, tid, qi, gi);
        auto fetch = [&](int st, int g, int blk) {
            const int64_t at = (int64_t)g * q_blocks;
            sg.x = qi + at * Frags::kImage;
            sg.y = gi + at * Frags::kImage;
            sg.fetch(st, blk);
            if (wave == NW - 1) {  // lse and delta, 256 bytes: a value to a lane
                const __amdgpu_buffer_rsrc_t r = make_rsrc(mha_uniform(sides + (at + blk) * kMhaSide), 256);
                const uint32_t m0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(zn_lds_void *)(lds + kSide + st * 256));
                asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dword %1, %2, 0 offen lds" : : "s"(m0), "v"(sg.lane16 / 4), "s"(r) : "memory");
            }
        };
        const Frags fr(lds, lane);
        int g = __builtin_amdgcn_readfirstlane(nb ? from / nb : 0), blk = __builtin_amdgcn_readfirstlane(b0 + from - g * nb);
        if (from < total) fetch(0, g, blk);
        for (int t = from; t < total; ++t) {
            const int st = (t - from) & 1, i0 = 32 * blk;
            sg.arrive();
            __syncthreads();
            if (++blk == b0 + nb) {
                blk = b0;
                ++g;
            }
            if (t + 1 < total) fetch(st ^ 1, g, blk);
            const int hi = w0 + FK * 16;  // keys of this wave: [w0, hi)
            if (min(i0 + 31, ql - 1) + edge >= w0 && w0 < kl)
                block(fr, st, i0 + edge < hi - 1 || hi > kl, side + st * 64, i0, w0, kl, edge, lane, kf, vf, dk, dv);
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
            for (int j = w0; j < min(w0 + FK * 16, p.kv_len); ++j) mha_row_grad_kv(p, b, kh, j, z, b0, nb, from, total, lane);
            return;
        }
#pragma unroll
        for (int f = 0; f < FK; ++f) {
            const int j = w0 + 16 * f + li;
            if (j >= p.kv_len) continue;
            const bool part = p.kv_splits > 1;
            float *rk = part ? mha_key_part(p, mha_key_row(p, b, kh, j, false), z) : p.grad_k + kat + j * p.ks[2];
            float *rv = part ? mha_key_part(p, mha_key_row(p, b, kh, j, true), z) : p.grad_v + kat + j * p.ks[2];
#pragma unroll
            for (int d = 0; d < DB; ++d) {
                mha_store4(rk, Frags::dim_of(d, lh), p.dim, dk[f][d]);
                mha_store4(rv, Frags::dim_of(d, lh), p.dim, dv[f][d]);
            }
        }
    }

    // One block of 32 queries.  `mask` (of the whole wave): some of its pairs are masked.  One code for both: with a copy for
    // each, the sums lie in other registers at the end of the copies, and moving them together spills.
    __device__ static __forceinline__ void block(const Frags &sg, int st, bool mask, const float *side, int i0, int w0, int kl, int edge,
                                                 int lane, const zn_bf16x8 (&kf)[FK][SL][3], const zn_bf16x8 (&vf)[FK][SL][3],
                                                 zn_f32x4 (&dk)[FK][DB], zn_f32x4 (&dv)[FK][DB]) {
        const int li = lane & 15, lh = lane >> 4;
        constexpr int NR = DB / 2;
        zn_f32x4 s[FK][2], dp[FK][2];
        MhaSix a;
#pragma unroll
        for (int q = 2; q >= 0; --q) sg.dims(st, 0, 0, q, a);
#pragma unroll
        for (int f = 0; f < FK; ++f)
#pragma unroll
            for (int rb = 0; rb < 2; ++rb) s[f][rb] = dp[f][rb] = zn_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        __builtin_amdgcn_sched_barrier(0);
        // S
#pragma unroll
        for (int i = 0; i < SL; ++i)
            mha_group<FK, 2, false>(a, [&](int rb, int f) -> zn_f32x4 & { return s[f][rb]; }, [&](int f) -> const zn_bf16x8(&)[3] { return kf[f][i]; },
                             [&](int q) { sg.dims(st, i + 1 < SL ? 0 : 1, i + 1 < SL ? i + 1 : 0, q, a); });
        // P times 2^24, in the place of S
        {
            zn_f32x4 ml[2];
#pragma unroll
            for (int rb = 0; rb < 2; ++rb) ml[rb] = *reinterpret_cast<const zn_f32x4 *>(side + 16 * rb + 4 * lh);
#pragma unroll
            for (int f = 0; f < FK; ++f)
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    s[f][e / 4][e % 4] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[f][e / 4][e % 4], kSplitUnscale, -ml[e / 4][e % 4])) * kSplitScale;
        }
        if (mask) {
#pragma unroll
            for (int f = 0; f < FK; ++f) {
                const int j = w0 + 16 * f + li;
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (j >= kl || j > i0 + 16 * (e / 4) + 4 * lh + e % 4 + edge) s[f][e / 4][e % 4] = 0.0f;
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        // dP
#pragma unroll
        for (int i = 0; i < SL; ++i) {
            auto acc = [&](int rb, int f) -> zn_f32x4 & { return dp[f][rb]; };
            auto operand = [&](int f) -> const zn_bf16x8(&)[3] { return vf[f][i]; };
            if (i + 1 < SL) mha_group<FK, 2, false>(a, acc, operand, [&](int q) { sg.dims(st, 1, i + 1, q, a); });
            else mha_group<FK, 4, false>(a, acc, operand, [&](int q) { sg.rows(st, 1, 0, q, a); });
        }
        // dS times 2^24, in the place of P, and P's parts; dS's take their registers once dV is done
        zn_bf16x8 pf[FK][3];
        {
            zn_f32x4 dl[2];
#pragma unroll
            for (int rb = 0; rb < 2; ++rb) dl[rb] = *reinterpret_cast<const zn_f32x4 *>(side + 32 + 16 * rb + 4 * lh);
#pragma unroll
            for (int f = 0; f < FK; ++f) {
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    x[e] = s[f][e / 4][e % 4];
                    s[f][e / 4][e % 4] = x[e] * __builtin_fmaf(dp[f][e / 4][e % 4], kSplitUnscale, -dl[e / 4][e % 4]);
                }
                mha_split8(x, pf[f]);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        // dV^T += dO^T P
#pragma unroll
        for (int i = 0; i < NR; ++i)
            mha_group<FK, 4, true>(a, [&](int c, int f) -> zn_f32x4 & { return dv[f][2 * i + c]; }, [&](int f) -> const zn_bf16x8(&)[3] { return pf[f]; },
                             [&](int q) { sg.rows(st, i + 1 < NR ? 1 : 0, i + 1 < NR ? 2 * (i + 1) : 0, q, a); });
        // dK^T += Q^T dS
#pragma unroll
        for (int f = 0; f < FK; ++f) {
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = s[f][e / 4][e % 4];
            mha_split8(y, pf[f]);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            auto acc = [&](int c, int f) -> zn_f32x4 & { return dk[f][2 * i + c]; };
            auto operand = [&](int f) -> const zn_bf16x8(&)[3] { return pf[f]; };
            if (i + 1 < NR) mha_group<FK, 4, true>(a, acc, operand, [&](int q) { sg.rows(st, 0, 2 * (i + 1), q, a); });
            else mha_group<FK, 0, true>(a, acc, operand, [](int) {});
        }
    }
};

// O and lse of at most 16 query rows of a key/value head: a few new tokens
// against a long cache, bound by reading K and V once.  The fp32 matrix cores
// keep up with that (16 rows, most of them padding, take 4 x 16 of their products
// for 16 keys of 64 dims: 18 TB/s of K and V), so nothing is split and nothing passes
// through LDS: each of the NW waves of each workgroup and split walks its own
// keys, 16 at a time, loaded one step ahead straight into the fragments (K:
// lane li a key, 4 dims of each 16 per quarter; V: lane li G neighbouring
// dims of one key per quarter).  The waves' sums are joined in LDS.  MI355X, 8
// tokens of 16 heads (4) against 2048 x 64: 9.6 us for 33.5 MB (3.5 TB/s; a
// wave has four steps), 12.5 us with the join of the parts.  Four steps in flight
// cost occupancy (12.9 us; 32 x 32 heads of 2048 x 64 207 and 219).
template <int DP, int NW>
struct MhaFew {
    static constexpr int G = DP / 16;  // groups of 16 dims; also the 16-dim blocks of O^T
    // Past 64 dims the loads above take half of each 128-byte line, and the next one waits for the line that is on its way.
    // There a load takes whole lines: K's 32 dims of 8 keys, whose halves change lanes before their use; V's 64 dims of 4 keys.
    // MI355X, 16 x 8 heads of 4096 x 128: 138 and 113 us (4.75 TB/s); at 64 dims whole lines of K cost 0.5 us.
    static constexpr bool WHOLE = DP > 64;
    // The dim of O^T's row i of block c.
    __device__ static constexpr int dim_of(int c, int i) { return !WHOLE ? G * i + c : c < G / 4 * 4 ? 64 * (c / 4) + 4 * i + c % 4 : 16 * c + i; }
    static constexpr int kLd = DP + 4;
    static constexpr int kBytes = NW * 16 * kLd * 4;
    struct Keys {
        float k[G][4], v[4][G];
    };

    __device__ static __forceinline__ void load4(__amdgpu_buffer_rsrc_t r, uint32_t row, int d, int dim, float (&x)[4]) {
        const uint32_t off = d < dim ? row + (uint32_t)d * 4u : kOutOfRange;
        const zn_f32x4 v = __builtin_bit_cast(zn_f32x4, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0));
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = d + e < dim ? v[e] : 0.0f;
    }

    __device__ static __forceinline__ void run(const ZnMhaArgs &p, char *lds) {
        const int tid = threadIdx.x, lane = tid & (kWave - 1);
        const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
        const int li = lane & 15, lh = lane >> 4;
        const int b = blockIdx.x / p.kv_heads, kh = blockIdx.x - b * p.kv_heads;
        const MhaSeq seq(p, b);
        const MhaQuery r(p, kh, li);
        const int lim = r.in ? seq.seen(r.i) : 0;
        int any = lim;
#pragma unroll
        for (int s = 1; s < 16; s <<= 1) any = max(any, __shfl_xor(any, s));
        any = __builtin_amdgcn_readfirstlane(any);
        float q[G][4];
        const float *row = p.q + b * p.qs[0] + r.h * p.qs[1] + r.i * p.qs[2];
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int d = 16 * g + 4 * lh + e;
                q[g][e] = lim && d < p.dim ? row[d] * p.scale_log2 : 0.0f;
            }
        // the wave's share of the keys that any row sees, whole steps of 16
        const int steps = (any + 15) / 16, walks = p.splits * NW, share = (steps + walks - 1) / walks;
        const int s0 = min(((int)blockIdx.z * NW + wave) * share, steps), s1 = min(s0 + share, steps);
        const int64_t at = b * p.ks[0] + kh * p.ks[1];
        const int stride = (int)p.ks[2];
        auto load = [&](int s, Keys &x) {
            const int k0 = 16 * s, n = min(16, any - k0);  // s < s1: at least one
            const uint32_t bytes = (uint32_t)((n - 1) * stride + p.dim) * 4u;
            const __amdgpu_buffer_rsrc_t rk = make_rsrc(p.k + at + (int64_t)k0 * p.ks[2], bytes);
            const __amdgpu_buffer_rsrc_t rv = make_rsrc(p.v + at + (int64_t)k0 * p.ks[2], bytes);
#pragma unroll
            for (int g = 0; g < G; ++g)
                if (WHOLE) load4(rk, (uint32_t)((li % 8 + g % 2 * 8) * stride) * 4u, 32 * (g / 2) + 16 * (li / 8) + 4 * lh, p.dim, x.k[g]);
                else load4(rk, (uint32_t)(li * stride) * 4u, 16 * g + 4 * lh, p.dim, x.k[g]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t off = (uint32_t)((4 * lh + e) * stride) * 4u;
#pragma unroll
                for (int c = 0; c + 4 <= G; c += 4) {
                    float y[4];
                    load4(rv, off, dim_of(c, li), p.dim, y);
#pragma unroll
                    for (int z = 0; z < 4; ++z) x.v[e][c + z] = y[z];
                }
#pragma unroll
                for (int c = G / 4 * 4; c < G; ++c) {
                    const int d = dim_of(c, li);
                    x.v[e][c] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rv, d < p.dim ? off + (uint32_t)d * 4u : kOutOfRange, 0, 0));
                }
            }
        };
        zn_f32x4 o[G];
#pragma unroll
        for (int c = 0; c < G; ++c) o[c] = zn_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        float m = -INFINITY, l = 0.0f;
        Keys x[2];
        auto step = [&](int s, Keys &y) {
#pragma unroll
            for (int g = 0; g < (WHOLE ? G : 0); g += 2)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int a = __builtin_bit_cast(int, y.k[g][e]), b = __builtin_bit_cast(int, y.k[g + 1][e]);
                    y.k[g][e] = __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(a, b, 0x128, 0xf, 0xc, false));  // row_ror:8
                    y.k[g + 1][e] = __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(b, a, 0x128, 0xf, 0x3, false));
                }
            zn_f32x4 t[2] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int e = 0; e < 4; ++e) t[e & 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(y.k[g][e], q[g][e], t[e & 1], 0, 0, 0);
            t[0] += t[1];
            float mb = -INFINITY;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (16 * s + 4 * lh + e >= lim) t[0][e] = -INFINITY;
                mb = fmaxf(mb, t[0][e]);
            }
            const float mn = fmaxf(m, max_over_rows(mb)), ref = mn == -INFINITY ? 0.0f : mn;
            const float alpha = __builtin_amdgcn_exp2f(m - ref);
            float rs = 0.0f;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                t[0][e] = __builtin_amdgcn_exp2f(t[0][e] - ref);
                rs += t[0][e];
            }
            l = l * alpha + rs;
            m = mn;
#pragma unroll
            for (int c = 0; c < G; ++c) o[c] *= alpha;
#pragma unroll
            for (int e = 0; e < 4; ++e)  // key 16 s + 4 lh + e
#pragma unroll
                for (int c = 0; c < G; ++c) o[c] = __builtin_amdgcn_mfma_f32_16x16x4f32(y.v[e][c], t[0][e], o[c], 0, 0, 0);
        };
        if (s0 < s1) load(s0, x[0]);
        for (int s = s0; s < s1; s += 2) {
            if (s + 1 < s1) load(s + 1, x[1]);
            step(s, x[0]);
            if (s + 1 < s1) {
                if (s + 2 < s1) load(s + 2, x[0]);
                step(s + 1, x[1]);
            }
        }
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
        // a value that is not finite in a pair masked for some rows only: the rows one by one
        bool bad = !(l < INFINITY);
#pragma unroll
        for (int c = 0; c < G; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) bad |= !(__builtin_fabsf(o[c][e]) < INFINITY);
        float *mine = reinterpret_cast<float *>(lds) + wave * 16 * kLd;  // [row][dims, maximum, sum]
        if (__builtin_amdgcn_ballot_w64(bad)) {
            for (int y = 0; y < 16; ++y) {
                const MhaQuery w(p, kh, y);
                MhaRowState t;
                if (w.in) t.walk(p, b, w.h, w.i, 16 * s0, min(16 * s1, seq.seen(w.i)), lane);
                MhaRow::store(mine + y * kLd, p.dim, lane, t.oa, t.ob);
                if (lane == 0) {
                    mine[y * kLd + DP] = t.m;
                    mine[y * kLd + DP + 1] = t.l;
                }
            }
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int c = 0; c < G; ++c) mine[li * kLd + dim_of(c, 4 * lh + e)] = o[c][e];
            if (lh == 0) {
                mine[li * kLd + DP] = m;
                mine[li * kLd + DP + 1] = l;
            }
        }
        __syncthreads();
        const float *sums = reinterpret_cast<const float *>(lds);
        for (int y = wave; y < 16; y += NW) {  // a wave to a row, the waves' sums in order
            const MhaQuery w(p, kh, y);
            if (!w.in) break;
            float mx = -INFINITY, sl = 0.0f, oa = 0.0f, ob = 0.0f;
#pragma unroll
            for (int z = 0; z < NW; ++z) mx = fmaxf(mx, sums[(z * 16 + y) * kLd + DP]);
            const float ref = mx == -INFINITY ? 0.0f : mx;
#pragma unroll
            for (int z = 0; z < NW; ++z) {
                const float *t = sums + (z * 16 + y) * kLd;
                const float f = __builtin_amdgcn_exp2f(t[DP] - ref);
                sl += f * t[DP + 1];
                if (lane < p.dim) oa += f * t[lane];
                if (lane + 64 < p.dim) ob += f * t[lane + 64];
            }
            mha_row_finish(p, b, w.h, w.i, blockIdx.z, lane, mx, sl, oa, ob);
        }
    }
};

// Maximum and sum of a far query's row, one key at a time (op[0]: the queries, op[2]: the keys).
__device__ __forceinline__ void mha_row_far(const ZnMhaSplitArgs &a, int b, int h, int i, int ql, int lane, float &m, float &l) {
    const ZnMhaSplitOp &q = a.op[0], &k = a.op[2];
    const int kl = k.lens ? min(max(k.lens[b], 0), k.len) : k.len, n = a.causal ? max(0, min(kl, i + 1 + kl - ql)) : kl;
    MhaRow x(q.src + b * q.stride[0] + h * q.stride[1] + i * q.stride[2], a.dim, lane);
    x.a *= q.scale;
    x.b *= q.scale;
    const float *row = k.src + b * k.stride[0] + h / (q.heads / k.heads) * k.stride[1];
    m = -INFINITY;
    l = 0.0f;
    for (int j = 0; j < n && l == l; ++j) {  // a NaN stays
        const float s = x.dot(MhaRow(row + j * k.stride[2], a.dim, lane)), mn = fmaxf(m, s), ref = mn == -INFINITY ? 0.0f : mn;
        l = l * __builtin_amdgcn_exp2f(m - ref) + __builtin_amdgcn_exp2f(s - ref);
        m = mn;
    }
}

// Tensors to their images: a workgroup to a block of 32 rows, a unit of 8
// values to a thread and step.  Rows past a sequence's length are zeros, and on
// the query side rows that see nothing (lse -inf); blocks past it are not read
// and not written.  10 bytes of traffic a value, and out's 4 for delta (MI355X, the
// four tensors of 8 x 16 heads of 1024 x 64: 66 us, 5.6 TB/s).
template <int DP>
__device__ __forceinline__ void mha_split(const ZnMhaSplitArgs &a) {
    typedef MhaBlock<DP> B;
    int which = 0;
#pragma unroll
    for (int i = 1; i < 4; ++i)
        if (i < a.ops && (int)blockIdx.x >= a.op[i].first) which = i;
    const ZnMhaSplitOp &p = a.op[which];
    const int wg = (int)blockIdx.x - p.first, blk = wg % p.blocks, bh = wg / p.blocks, b = bh / p.heads, h = bh - b * p.heads;
    const int n = p.lens ? min(max(p.lens[b], 0), p.len) : p.len, r0 = 32 * blk;
    if (r0 >= n) return;
    const int64_t at = b * p.stride[0] + h * p.stride[1];
    char *dst = p.dst + ((int64_t)bh * p.blocks + blk) * B::kImage;
    for (int u = threadIdx.x; u < B::SL * 32 * 4; u += 256) {
        const int sl = u / 128, row = u / 4 % 32, c = u % 4, i = r0 + row;
        const bool in = i < n && !(p.lse && p.lse[(int64_t)bh * p.len + i] == -INFINITY);
        const float *src = p.src + at + i * p.stride[2];
        float x[8];
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            const int d = 32 * sl + 4 * c + 16 * g;
            zn_f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
            if (in && d + 4 <= a.dim) {
                v = *reinterpret_cast<const zn_f32x4u *>(src + d);
            } else if (in) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (d + e < a.dim) v[e] = src[d + e];
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) x[4 * g + e] = v[e] * p.scale;
        }
        zn_u32x4 w[3];
        split8(x, w);
#pragma unroll
        for (int q = 0; q < 3; ++q) *reinterpret_cast<zn_u32x4 *>(dst + B::place(row, c, sl, q)) = w[q];
    }
    if (p.side) {  // 8 threads to a row
        const int row = threadIdx.x / 8, i = r0 + row;
        const float lse = i < n ? p.lse[(int64_t)bh * p.len + i] : -INFINITY;
        const float *g = p.src + at + i * p.stride[2], *o = p.out + at + i * p.stride[2];
        float sum = 0.0f;
        if (lse != -INFINITY)
            for (int d = threadIdx.x % 8; d < a.dim; d += 8) sum = __builtin_fmaf(g[d], o[d], sum);
#pragma unroll
        for (int s = 1; s < 8; s <<= 1) sum += __shfl_xor(sum, s);
        float *side = p.side + ((int64_t)bh * p.blocks + blk) * kMhaSide + row;
        const float lse2 = lse == -INFINITY ? INFINITY : lse * kLog2e;
        const bool far = lse != -INFINITY && !(__builtin_fabsf(lse2) < kMhaFar);
        if (threadIdx.x % 8 == 0) {
            side[0] = far ? __builtin_nanf("") : lse2;
            side[32] = sum;
            if (!far) {
                side[64] = lse2;
                side[96] = 1.0f;
            }
        }
        const int lane = threadIdx.x % kWave;
        for (uint64_t left = __builtin_amdgcn_ballot_w64(far && threadIdx.x % 8 == 0); left; left &= left - 1) {
            const int from = __builtin_ctzll(left), r = (int)threadIdx.x / kWave * 8 + from / 8;  // the whole wave, row by row
            float m, l;
            mha_row_far(a, b, h, r0 + r, n, lane, m, l);
            if (lane == from) {
                side[64] = m;
                side[96] = 1.0f / l;
            }
        }
    }
}

}  // namespace

// Rows of partial sums: the parts in order, a wave to a row, lane l its dims l
// and l + 64, eight splits' loads in flight.
extern "C" __global__ __launch_bounds__(256) void zn_mha_join(ZnMhaJoinArgs a) {
    const ZnMhaJoinOp &p = a.op[blockIdx.y];
    const int lane = threadIdx.x & (kWave - 1);
    const int64_t row = (int64_t)blockIdx.x * 4 + threadIdx.x / kWave;
    if (row >= p.rows) return;
    const float *src = p.part + row * p.splits * a.part_ld;
    float mx = -INFINITY, sl = 0.0f, oa = 0.0f, ob = 0.0f;
    for (int z0 = 0; z0 < p.splits; z0 += 8) {
        float x[8], y[8], m[8], l[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const float *t = src + (int64_t)min(z0 + u, p.splits - 1) * a.part_ld;  // any row of parts: no load waits for a condition
            x[u] = t[min(lane, a.dim - 1)];
            y[u] = t[min(lane + 64, a.dim - 1)];
            m[u] = t[a.part_ld - 4];
            l[u] = t[a.part_ld - 3];
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const bool in = z0 + u < p.splits;
            x[u] = in ? x[u] : 0.0f;
            y[u] = in ? y[u] : 0.0f;
            m[u] = in && a.forward ? m[u] : -INFINITY;
            l[u] = in ? l[u] : 0.0f;
        }
        float mn = mx;
#pragma unroll
        for (int u = 0; u < 8; ++u) mn = fmaxf(mn, m[u]);
        const float ref = mn == -INFINITY ? 0.0f : mn, alpha = a.forward ? __builtin_amdgcn_exp2f(mx - ref) : 1.0f;
        mx = mn;
        sl *= alpha;
        oa *= alpha;
        ob *= alpha;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const float f = a.forward ? __builtin_amdgcn_exp2f(m[u] - ref) : 1.0f;
            sl += f * l[u];
            oa += f * x[u];
            ob += f * y[u];
        }
    }
    const int bh = (int)row / p.len, b = bh / p.heads;  // a launch has fewer than 2^31 rows
    float *dst = p.dst + b * p.stride[0] + (bh - b * p.heads) * p.stride[1] + ((int)row - bh * p.len) * p.stride[2];
    if (a.forward) {
        const float r = sl == 0.0f ? 1.0f : sl;
        MhaRow::store(dst, a.dim, lane, oa / r, ob / r);
        if (a.lse && lane == 0) a.lse[row] = mha_lse(mx, sl);
    } else {
        MhaRow::store(dst, a.dim, lane, oa * p.factor, ob * p.factor);
    }
}

// Grid: x = sequence and key/value head (its tiles share an XCD's L2), y = the parts of each tile, the longest walks first (the
// gradients': tiles of keys before those of queries).  zn_mha_few_*: z = the parts.
#define ZN_MHA_KERNEL(NAME, NW, BYTES, ...)                                           \
    extern "C" __global__ __launch_bounds__(NW * 64, 2) void NAME(ZnMhaArgs p) {      \
        __shared__ __attribute__((aligned(1024))) char lds[BYTES];                    \
        __VA_ARGS__;                                                                  \
    }
// NW waves of F blocks of 16 rows, backward BNW waves of BF.  Workgroups of 4 waves
// share a CU by two, as far as LDS allows: up to 96 dims.  There the backward gains (both gradients of 2 x 16 heads (4) of
// 2048 x 96, causal: 809 us with 8 waves, 694 with 4) and the forward loses (137 and 159).
#define ZN_MHA_KERNELS(DP, NW, F, BNW, BF)                                                                         \
    typedef MhaQueryTile<DP, NW, F, false, true> MhaForward##DP;                                                   \
    typedef MhaQueryTile<DP, NW, F, false, false> MhaForwardRaw##DP;                                               \
    typedef MhaQueryTile<DP, BNW, BF, true, true> MhaGradQ##DP;                                                    \
    typedef MhaKeyTile<DP, BNW, BF> MhaGradKv##DP;                                                                 \
    typedef MhaFew<DP, 4> MhaFew##DP;                                                                              \
    ZN_MHA_KERNEL(zn_mha_few_##DP, 4, MhaFew##DP::kBytes, MhaFew##DP::run(p, lds))                                 \
    ZN_MHA_KERNEL(zn_mha_forward_##DP, NW, MhaForward##DP::kBytes,                                                 \
                  MhaForward##DP::run(p, blockIdx.y / p.splits, blockIdx.y % p.splits, lds))                       \
    ZN_MHA_KERNEL(zn_mha_forward_raw_##DP, NW, MhaForwardRaw##DP::kBytes,                                          \
                  MhaForwardRaw##DP::run(p, blockIdx.y / p.splits, blockIdx.y % p.splits, lds))                    \
    ZN_MHA_KERNEL(zn_mha_grad_##DP, BNW, MhaGradKv##DP::kBytes,                                                    \
                  const int y = (int)blockIdx.y - p.key_tiles * p.kv_splits;                                       \
                  if (y < 0) MhaGradKv##DP::run(p, blockIdx.y / p.kv_splits, blockIdx.y % p.kv_splits, lds);       \
                  else MhaGradQ##DP::run(p, y / p.splits, y % p.splits, lds))                                      \
    extern "C" __global__ __launch_bounds__(256) void zn_mha_split_##DP(ZnMhaSplitArgs a) { mha_split<DP>(a); }
ZN_MHA_KERNELS(32, 4, 2, 4, 2)
ZN_MHA_KERNELS(64, 4, 2, 4, 2)
ZN_MHA_KERNELS(96, 8, 1, 4, 1)
ZN_MHA_KERNELS(128, 8, 1, 8, 1)
// Two blocks of rows to a wave past 64 dims too: each fragment read from LDS serves twice the products, and half as many tiles
// are left.  MI355X, forward of 8 x 16 heads of 1024 x 128 411 us, 371 so; 2 x 16 (4) of 4096 x 96, causal, 535, 486;
// but 2 x 16 (4) of 2048 x 128, causal, 171, 232.
#define ZN_MHA_WIDE(DP)                                                                                             \
    typedef MhaQueryTile<DP, 8, 2, false, true> MhaWide##DP;                                                       \
    ZN_MHA_KERNEL(zn_mha_forward_wide_##DP, 8, MhaWide##DP::kBytes,                                                \
                  MhaWide##DP::run(p, blockIdx.y / p.splits, blockIdx.y % p.splits, lds))
ZN_MHA_WIDE(96)
ZN_MHA_WIDE(128)

#endif
