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

// Keys that token i of a sequence sees: positions [0, seen).
__device__ __forceinline__ int paged_seen(const ZnPagedArgs &p, const PagedSeq &s, int i) {
    return p.causal ? max(0, min(s.kl, s.first + i + 1)) : s.kl;
}

__device__ __forceinline__ void paged_store(const ZnPagedArgs &p, int t, int h, int lane, float m, float l, float oa, float ob) {
    const float r = l == 0.0f ? 1.0f : l;
    MhaRow::store(p.out + t * p.os[0] + h * p.os[1], p.c.dim, lane, oa / r, ob / r);
    if (p.lse && lane == 0) p.lse[(int64_t)t * p.q_heads + h] = mha_lse(m, l);
}

// A row's sums: to the tensor, or to its part (another XCD may read that in the same launch: agent-scope stores).
__device__ __forceinline__ void paged_finish(const ZnPagedArgs &p, float *part, int t, int h, int lane, float m, float l, float oa, float ob) {
    if (!part) return paged_store(p, t, h, lane, m, l, oa, ob);
    auto put = [&](int i, float x) { __hip_atomic_store(part + i, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
    if (lane < p.c.dim) put(lane, oa);
    if (lane + 64 < p.c.dim) put(lane + 64, ob);
    if (lane < 2) put(p.part_ld - 4 + lane, lane ? l : m);
}

// A row's parts in order, a wave to a row, lane l its dims l and l + 64, N parts' loads in flight.
template <int N>
__device__ __forceinline__ void paged_join(const ZnPagedArgs &p, const float *src, int parts, int t, int h, int lane) {
    float mx = -INFINITY, sl = 0.0f, oa = 0.0f, ob = 0.0f;
    for (int z0 = 0; z0 < parts; z0 += N) {
        float x[N], y[N], m[N], l[N];
#pragma unroll
        for (int u = 0; u < N; ++u) {
            const float *r = src + (int64_t)min(z0 + u, parts - 1) * p.part_ld;  // any of them: no load waits for a condition
            auto get = [&](int i) { return __hip_atomic_load(r + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
            x[u] = get(min(lane, p.c.dim - 1));
            y[u] = get(min(lane + 64, p.c.dim - 1));
            m[u] = get(p.part_ld - 4);
            l[u] = get(p.part_ld - 3);
        }
        float mn = mx;
#pragma unroll
        for (int u = 0; u < N; ++u) {
            if (z0 + u >= parts) m[u] = -INFINITY, l[u] = x[u] = y[u] = 0.0f;
            mn = fmaxf(mn, m[u]);
        }
        const float ref = mn == -INFINITY ? 0.0f : mn, alpha = __builtin_amdgcn_exp2f(mx - ref);
        mx = mn;
        sl *= alpha;
        oa *= alpha;
        ob *= alpha;
#pragma unroll
        for (int u = 0; u < N; ++u) {
            const float f = __builtin_amdgcn_exp2f(m[u] - ref);
            sl += f * l[u];
            oa += f * x[u];
            ob += f * y[u];
        }
    }
    paged_store(p, t, h, lane, mx, sl, oa, ob);
}

__device__ __forceinline__ void paged_join(const ZnPagedArgs &p, const float *src, int parts, int t, int h, int lane) {
    if (parts <= 4) paged_join<4>(p, src, parts, t, h, lane);
    else paged_join<16>(p, src, parts, t, h, lane);
}

// Parts of a walk over `keys` positions: one at least.
__device__ __forceinline__ int paged_parts(int keys, int len) { return max(1, (keys + len - 1) / len); }
// ... of few rows: as many equal parts as the call has, in multiples of 128 (32 for each of four waves).
__device__ __forceinline__ int paged_few_len(const ZnPagedArgs &p, int keys) { return 128 * max(1, (int)(((uint32_t)keys + 128u * p.few_splits - 1) / (128u * p.few_splits))); }

// Rows one at a time, a wave each: grid x the tokens, y four heads.  For heads of fewer dims than a 16-byte load of bf16 has.
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
    paged_walk<T>(p, b, t, h, 0, paged_seen(p, seq, i), lane, w);
    paged_store(p, t, h, lane, w.m, w.l, w.oa, w.ob);
}

// ------------------------------------------------------------- common parts
// Loads at any address that a cache's strides lead to: 2-byte aligned.
typedef uint32_t zn_u32x4_2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t zn_u32x2_2 __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t zn_u32_2 __attribute__((aligned(2)));
typedef uint32_t zn_u32x2 __attribute__((ext_vector_type(2)));

// Dims.  A load takes W dims of a row at d, a multiple of W, and never passes the row's end: where d + W > dim it takes the last W
// dims.  Those of them before d are another load's too: there Q holds 0 (so that each dim is counted once), and O is not stored.
__device__ __forceinline__ int paged_dim(int d, int w, int dim) { return min(d, dim - w); }

// mha_split8 (eight probabilities times kSplitScale to three bf16 parts of each), bit for bit, in 28 instructions for 44: what is left of
// a value, x - h, is a dot product of a pair of parts with (-1, 0) or (0, -1) on top of x, where h as a float is an instruction of its
// own.  For bf16 pages (4 x 512 tokens of 32 heads (8) of 64 over 4096: 202 us, 197 so; of 128 327, 323); not for fp32 ones, whose
// tiles lose by it (594, 598).
__device__ __forceinline__ void paged_split8(const float (&x)[8], zn_bf16x8 (&f)[3]) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    uint32_t first;  // in a register: as an inline constant it would be the float -1, which is (0, -1)
    asm("s_mov_b32 %0, 0xbf80" : "=s"(first));
    const zn_bf16x2 one = __builtin_bit_cast(zn_bf16x2, first), two = __builtin_bit_cast(zn_bf16x2, 0xbf800000u);
    zn_u32x4 w[3];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        float t0 = x[2 * e], t1 = x[2 * e + 1];
        const zn_bf16x2 h = __builtin_convertvector((f2{t0, t1}), zn_bf16x2);
        t0 = __builtin_amdgcn_fdot2_f32_bf16(h, one, t0, false);
        t1 = __builtin_amdgcn_fdot2_f32_bf16(h, two, t1, false);
        const zn_bf16x2 m = __builtin_convertvector((f2{t0, t1}), zn_bf16x2);
        t0 = __builtin_amdgcn_fdot2_f32_bf16(m, one, t0, false);
        t1 = __builtin_amdgcn_fdot2_f32_bf16(m, two, t1, false);
        w[0][e] = __builtin_bit_cast(uint32_t, h);
        w[1][e] = __builtin_bit_cast(uint32_t, m);
        w[2][e] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{t0, t1}), zn_bf16x2));
    }
#pragma unroll
    for (int q = 0; q < 3; ++q) f[q] = __builtin_bit_cast(zn_bf16x8, w[q]);
}

constexpr float kPagedUnscale = 1.0f / 16777216.0f;  // of sums whose other operand is bf16 already: 2^24 times their value

// W dims (4 or 8) of a query row at d, times `scale`; zeros of a row that is not `in` (row: any one).
template <int W>
__device__ __forceinline__ void paged_query(const float *row, bool in, int d, int dim, float scale, float (&x)[W]) {
    const int at = paged_dim(d, W, dim);
#pragma unroll
    for (int h = 0; h < W; h += 4) {
        const zn_f32x4 v = *reinterpret_cast<const zn_f32x4u *>(row + at + h);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[h + e] = in && at + h + e >= d ? v[e] * scale : 0.0f;
    }
}

// ------------------------------------------------------------- few query rows
// At most 16 RB query rows of a key/value head (a token or a few, of the heads
// that share it) against a long cache: bound by reading K and V once.  K and V do
// not pass through LDS: each of the NW waves walks its own keys, straight into
// fragments; Q's fragments are in LDS, and the waves' sums are joined there.
//  - fp32 pages: the fp32 matrix cores, 16 keys a step (as zn_mha_few_*).
//  - bf16 pages: the bf16 ones, 32 keys a step: K and V are operands as they lie,
//    Q and P are split into three parts, so that three products take one of fp32.
//    V's rows hold one key's dims, its operand one dim's keys: pairs of keys
//    change halves of a register (half an instruction a value).
// One set of registers each for K and V: the next step's K is asked for behind
// the products with K, its V behind those with V.
// Rows are read in whole 128-byte lines where they have them: K's two slices of a
// line go to lanes 8 apart, which then exchange theirs.
// Each walk is cut into parts (paged_few_parts) so that a few sequences fill the
// chip.  MI355X, one new token each: 64 x 32 heads (8) against up to 8192 x 128 bf16
// (1.48 GB) 280 us, 5.3 TB/s, a large copy's rate 4.9; 8 x 16 (4) against 2048 x 64
// fp32 (34 MB) 12 us: parts of 128 positions, so two steps of a wave, the second
// asked for behind the first one's products, then the waves' sums and the join by the
// last workgroup.  Five tokens of 16 x 16 heads (4) against up to 4096 x 128 bf16 (83 MB) 27
// us and the join's 5.
template <typename T, int DP, int NW, int RB, bool PAGES16>
struct PagedFew {
    static constexpr bool BF = sizeof(T) == 2;
    static constexpr int STEP = BF ? 32 : 16;        // keys
    static constexpr int KB = STEP / 16;             // blocks of 16 keys
    static constexpr int KW = BF ? 8 : 4;            // dims of a load of K
    static constexpr int KS = DP / (4 * KW);         // slices: what the four quarters of a wave load together
    static constexpr bool WHOLE = KS >= 2 && DP * sizeof(T) >= 128;  // two slices at a time
    static constexpr int KR = WHOLE ? 2 : 1;         // rows of K that a lane reads of each 16
    static constexpr int VR = STEP / 4;              // ... of V
    static constexpr int G = DP / 16;                // blocks of 16 dims of O^T
    static constexpr int VB = DP == 96 || (DP == 128 && !BF) ? 2 : 1;  // loads of a row of V: of w dims at 64 b + w li
    static constexpr int vw(int b) { return DP == 128 ? (BF ? 8 : 4) : DP == 96 ? (b ? 2 : 4) : DP == 64 ? 4 : 2; }
    static constexpr int ROWS = 16 * RB;
    // Blocks of rows that a sequence does not fill are left out, except with 64 rows of 128 dims in bf16, where the branches spill (33 x 9
    // heads of 42 tokens against up to 2713 x 127 fp32: 258 us, 226 so; 64 rows of 128 dims bf16 104, 155).
    static constexpr bool SKIP = !(BF && DP == 128);
    static constexpr int kLd = DP + 4;
    static constexpr int QP = BF ? 3 : 1;            // parts of Q; a fragment: 16 bytes a lane
    static constexpr int kQuery = RB * KS * QP * 1024, kSums = NW * 16 * kLd * 4;
    static constexpr int kBytes = kQuery > kSums ? kQuery : kSums;
    typedef uint32_t Raw __attribute__((ext_vector_type(4)));

    template <int BYTES>
    __device__ static __forceinline__ void load(const T *at, uint32_t (&x)[4]) {
        if constexpr (BYTES == 16) {
            const zn_u32x4_2 y = *reinterpret_cast<const zn_u32x4_2 *>(at);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = y[e];
        } else if constexpr (BYTES == 8) {
            const zn_u32x2_2 y = *reinterpret_cast<const zn_u32x2_2 *>(at);
            x[0] = y[0];
            x[1] = y[1];
        } else {
            static_assert(BYTES == 4, "2 to 8 dims");
            x[0] = *reinterpret_cast<const zn_u32_2 *>(at);
        }
    }
    // x's upper eight lanes of 16 and y's lower eight change places
    __device__ static __forceinline__ void swap(Raw &x, Raw &y) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int a = (int)x[e], b = (int)y[e];
            x[e] = (uint32_t)__builtin_amdgcn_update_dpp(a, b, 0x128, 0xf, 0xc, false);  // row_ror:8
            y[e] = (uint32_t)__builtin_amdgcn_update_dpp(b, a, 0x128, 0xf, 0x3, false);
        }
    }

    // Where a walk's rows lie.  Pages whose size is a multiple of 16 (PAGES16) hold each block of 16 keys whole: one page of the block
    // for the wave, read by the scalar unit (16 x 16 heads (4) of five tokens against up to 4096 x 128 bf16 with the join 31.9 us, row
    // by row 34.5).  Other pages are looked up row by row.  Either a step ahead of the rows.  Keys past the walk's end are its last.
    struct Place {
        typedef __attribute__((address_space(4))) const int32_t Table;  // constant: for scalar loads
        const ZnPagedCache &c;
        const int32_t *table;
        int from, to, li, lh;
        bool hole = false;
        int kp[KB][PAGES16 ? 1 : KR], vp[PAGES16 ? KB : VR];
        __device__ __forceinline__ Place(const ZnPagedCache &c, int b, int from, int to, int lane)
            : c(c), table(c.table + (int64_t)b * c.max_pages), from(from), to(to), li(lane & 15), lh(lane >> 4) {}
        __device__ __forceinline__ int page_of(int j) const { return (int)(((uint64_t)(uint32_t)j * c.div_mul) >> (31 + c.div_shift)); }
        __device__ __forceinline__ int key_k(int rb, int r) const { return 16 * rb + (WHOLE ? li % 8 + 8 * r : li); }  // of a step
        __device__ __forceinline__ int key_v(int e) const { return 16 * (e / 4) + 4 * lh + e % 4; }
        __device__ __forceinline__ int key(int s, int i) const { return min(from + STEP * s + i, to - 1); }
        __device__ __forceinline__ int page_at(int j) const { return PAGES16 ? ((Table *)(uintptr_t)table)[page_of(j)] : table[page_of(j)]; }
        __device__ __forceinline__ void ask_k(int s) {
#pragma unroll
            for (int rb = 0; rb < KB; ++rb)
#pragma unroll
                for (int r = 0; r < (PAGES16 ? 1 : KR); ++r) kp[rb][r] = page_at(key(s, PAGES16 ? 16 * rb : key_k(rb, r)));
        }
        __device__ __forceinline__ void ask_v(int s) {
#pragma unroll
            for (int e = 0; e < (PAGES16 ? KB : VR); ++e) vp[e] = page_at(key(s, PAGES16 ? 16 * e : key_v(e)));
        }
        // A row's elements from the head's first: key i of step s, in block rb, whose page is `page`.
        __device__ __forceinline__ int64_t at(int s, int rb, int page, int i) {
            const bool in = (uint32_t)page < (uint32_t)c.pages;
            hole |= !in;
            const int j0 = key(s, PAGES16 ? 16 * rb : i);
            const int64_t first = (in ? page : 0) * c.stride[0] + (j0 - page_of(j0) * c.page_size) * c.stride[2];
            return PAGES16 ? first + (int64_t)((uint64_t)(uint32_t)(key(s, i) - j0) * (uint32_t)c.stride[2]) : first;
        }
        __device__ __forceinline__ int64_t at_k(int s, int rb, int r) { return at(s, rb, kp[rb][PAGES16 ? 0 : r], key_k(rb, r)); }
        __device__ __forceinline__ int64_t at_v(int s, int e) { return at(s, e / 4, vp[PAGES16 ? e / 4 : e], key_v(e)); }
    };

    // Sequence and key/value head x, part z of its walk.
    __device__ static __forceinline__ void run(const ZnPagedArgs &p, char *lds, int x_, int z) {
        const int tid = threadIdx.x, lane = tid & (kWave - 1);
        const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
        const int li = lane & 15, lh = lane >> 4;
        const int b = x_ / p.c.kv_heads, kh = x_ - b * p.c.kv_heads, dim = p.c.dim;
        const PagedSeq seq(p.c, b);
        const int rows = min(seq.ql, p.max_q) * p.group;
        if (rows == 0 || rows > ROWS) return;
        const int any = __builtin_amdgcn_readfirstlane(paged_seen(p, seq, (rows - 1) / p.group));
        const int len = paged_few_len(p, any), parts = paged_parts(any, len);
        if (z >= parts) return;
        // the wave's share of the part's keys, whole steps
        const int from = z * len, to = min(from + len, any);
        const int steps = (to - from + STEP - 1) / STEP, share = (steps + NW - 1) / NW;
        const int s0 = min(wave * share, steps), s1 = min(s0 + share, steps), end = min(from + STEP * s1, to);

        const T *const k = reinterpret_cast<const T *>(p.c.k) + kh * p.c.stride[1], *const v = reinterpret_cast<const T *>(p.c.v) + kh * p.c.stride[1];
        Place at(p.c, b, from, end, lane);
        Raw x[KB][KS];
        uint32_t y[VR][VB][4];
        auto load_k = [&](int s) {
#pragma unroll
            for (int rb = 0; rb < KB; ++rb) {
                const T *r[KR];
#pragma unroll
                for (int i = 0; i < KR; ++i) r[i] = k + at.at_k(s, rb, i);
#pragma unroll
                for (int g = 0; g < KS; ++g) {
                    // two slices of a line together, or the last one of an odd number
                    const bool two = WHOLE && (g | 1) < KS;
                    const T *const of = two ? r[KR == 2 ? g & 1 : 0] : KR == 2 ? (li < 8 ? r[0] : r[KR - 1]) : r[0];
                    const int d = two ? 4 * KW * ((g & ~1) + li / 8) + KW * lh : 4 * KW * g + KW * lh;
                    uint32_t u[4];
                    load<16>(of + paged_dim(d, KW, dim), u);
                    x[rb][g] = Raw{u[0], u[1], u[2], u[3]};
                }
            }
        };
        auto load_v = [&](int s) {
#pragma unroll
            for (int e = 0; e < VR; ++e) {
                const T *const r = v + at.at_v(s, e);
#pragma unroll
                for (int c = 0; c < VB; ++c) {
                    if (vw(c) == 8) load<16>(r + paged_dim(64 * c + 8 * li, 8, dim), y[e][c]);
                    else if (vw(c) == 4) load<4 * (int)sizeof(T)>(r + paged_dim(64 * c + 4 * li, 4, dim), y[e][c]);
                    else load<2 * (int)sizeof(T)>(r + paged_dim(64 * c + 2 * li, 2, dim), y[e][c]);
                }
            }
        };
        if (s0 < s1) {
            at.ask_k(s0);
            at.ask_v(s0);
            load_k(s0);
            load_v(s0);
            at.ask_k(s0 + 1);
            at.ask_v(s0 + 1);
        }

        // Q's fragments: those of row block f and slice g by one wave
        for (int i = wave; i < RB * KS; i += NW) {
            const int f = i / KS, g = i - f * KS, r = 16 * f + li;
            const int i0 = min(r, rows - 1) / p.group, h = min(r, rows - 1) - i0 * p.group;
            float q[KW];
            paged_query(p.q + (seq.t0 + i0) * p.qs[0] + (kh * p.group + h) * p.qs[1], r < rows, 4 * KW * g + KW * lh, dim, p.scale_log2, q);
            zn_u32x4 w[3];
            if constexpr (BF) {
                split8(q, w);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) w[0][e] = __builtin_bit_cast(uint32_t, q[e]);
            }
#pragma unroll
            for (int part = 0; part < QP; ++part) *reinterpret_cast<zn_u32x4 *>(lds + (i * QP + part) * 1024 + lane * 16) = w[part];
        }
        int lim[RB];
#pragma unroll
        for (int f = 0; f < RB; ++f) lim[f] = 16 * f + li < rows ? min(paged_seen(p, seq, (16 * f + li) / p.group), to) : 0;
        __syncthreads();

        zn_f32x4 o[RB][G];
        float m[RB], l[RB];
#pragma unroll
        for (int f = 0; f < RB; ++f) {
            m[f] = -INFINITY;
            l[f] = 0.0f;
#pragma unroll
            for (int c = 0; c < G; ++c) o[f][c] = zn_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        for (int s = s0; s < s1; ++s) {
#pragma unroll
            for (int rb = 0; rb < KB; ++rb)
#pragma unroll
                for (int g = 0; g + 1 < KS; g += 2)
                    if (WHOLE) swap(x[rb][g], x[rb][g + 1]);
            uint32_t qat = lane * 16;  // read again in each step: kept in registers, Q would cost a wave of every SIMD
            asm volatile("" : "+v"(qat));
            const char *const query = lds + qat;
            zn_f32x4 t[RB][KB];
#pragma unroll
            for (int f = 0; f < RB; ++f) {
                if (SKIP && f > 1 && 16 * f >= rows) break;
                if constexpr (BF) {
#pragma unroll
                    for (int rb = 0; rb < KB; ++rb) t[f][rb] = zn_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int part = 2; part >= 0; --part)  // the largest last
#pragma unroll
                        for (int g = 0; g < KS; ++g) {
                            const zn_bf16x8 q = __builtin_bit_cast(zn_bf16x8, *reinterpret_cast<const zn_u32x4 *>(query + ((f * KS + g) * 3 + part) * 1024));
#pragma unroll
                            for (int rb = 0; rb < KB; ++rb)
                                t[f][rb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(zn_bf16x8, x[rb][g]), q, t[f][rb], 0, 0, 0);
                        }
#pragma unroll
                    for (int rb = 0; rb < KB; ++rb) t[f][rb] *= kPagedUnscale;
                } else {
                    zn_f32x4 u[2] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
                    for (int g = 0; g < KS; ++g) {
                        const zn_f32x4 q = *reinterpret_cast<const zn_f32x4 *>(query + (f * KS + g) * 1024);
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            u[e & 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, (uint32_t)x[0][g][e]), q[e], u[e & 1], 0, 0, 0);
                    }
                    t[f][0] = u[0] + u[1];
                }
            }
            // Behind the last step: its last key, which no load goes to memory for, and no branch splits the loop's body.  The barriers
            // keep the loads here: left alone the compiler asks for the next step's K and V together at the end.
            __builtin_amdgcn_sched_barrier(0);
            load_k(s + 1);
            at.ask_k(s + 2);
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (BF) {  // the first and the second dim of each pair, of 8 keys
#pragma unroll
                for (int c = 0; c < VB; ++c)
#pragma unroll
                    for (int w = 0; w < vw(c) / 2; ++w)
#pragma unroll
                        for (int e = 0; e < VR; e += 2) {
                            const uint32_t a = y[e][c][w], b = y[e + 1][c][w];
                            y[e][c][w] = __builtin_amdgcn_perm(b, a, 0x05040100u);
                            y[e + 1][c][w] = __builtin_amdgcn_perm(b, a, 0x07060302u);
                        }
            }
            const int k0 = from + STEP * s;
#pragma unroll
            for (int f = 0; f < RB; ++f) {
                if (SKIP && f > 1 && 16 * f >= rows) break;
                float mb = -INFINITY;
#pragma unroll
                for (int e = 0; e < VR; ++e) {
                    if (k0 + 16 * (e / 4) + 4 * lh + e % 4 >= lim[f]) t[f][e / 4][e % 4] = -INFINITY;
                    mb = fmaxf(mb, t[f][e / 4][e % 4]);
                }
                const float mn = fmaxf(m[f], max_over_rows(mb)), ref = mn == -INFINITY ? 0.0f : mn;
                const float alpha = __builtin_amdgcn_exp2f(m[f] - ref);
                float rs = 0.0f, e8[VR];
#pragma unroll
                for (int e = 0; e < VR; ++e) {
                    e8[e] = __builtin_amdgcn_exp2f(t[f][e / 4][e % 4] - ref);
                    rs += e8[e];
                }
                l[f] = l[f] * alpha + rs;
                m[f] = mn;
#pragma unroll
                for (int c = 0; c < G; ++c) o[f][c] *= alpha;
                if constexpr (BF) {
#pragma unroll
                    for (int e = 0; e < VR; ++e) e8[e] *= kSplitScale;
                    zn_bf16x8 pf[3];
                    paged_split8(e8, pf);
#pragma unroll
                    for (int part = 2; part >= 0; --part)
#pragma unroll
                        for (int c = 0; c < VB; ++c)
#pragma unroll
                            for (int w = 0; w < vw(c); ++w) {
                                const zn_u32x4 a = {y[w % 2][c][w / 2], y[2 + w % 2][c][w / 2], y[4 + w % 2][c][w / 2], y[6 + w % 2][c][w / 2]};
                                zn_f32x4 &z = o[f][4 * c + w];
                                z = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(zn_bf16x8, a), pf[part], z, 0, 0, 0);
                            }
                } else {
#pragma unroll
                    for (int e = 0; e < VR; ++e)  // key 4 lh + e
#pragma unroll
                        for (int c = 0; c < VB; ++c)
#pragma unroll
                            for (int w = 0; w < vw(c); ++w)
                                o[f][4 * c + w] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, y[e][c][w]), e8[e], o[f][4 * c + w], 0, 0, 0);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            load_v(s + 1);
            at.ask_v(s + 2);
        }
        // a page that is none of the cache's, a sum that is not finite (also of a value in a pair masked for some rows only), or scores
        // that all fell below the split's range: the rows one by one
        bool bad = at.hole;
#pragma unroll
        for (int f = 0; f < RB; ++f) {
            l[f] += __shfl_xor(l[f], 16);
            l[f] += __shfl_xor(l[f], 32);
            bad |= !(l[f] < INFINITY) || (BF && m[f] == -INFINITY && s0 < s1 && lim[f] > from + STEP * s0);
#pragma unroll
            for (int c = 0; c < G; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    bad |= !(__builtin_fabsf(o[f][c][e]) < INFINITY);
                    if (BF) o[f][c][e] *= kPagedUnscale;
                }
        }
        const bool one_by_one = __builtin_amdgcn_ballot_w64(bad);
        float *mine = reinterpret_cast<float *>(lds) + wave * 16 * kLd;  // [row][dims, maximum, sum]
#pragma unroll
        for (int f = 0; f < RB; ++f) {
            if (16 * f >= rows) break;
            __syncthreads();  // Q, or the last block's sums, are read
            if (one_by_one) {
                for (int i = 0; i < min(16, rows - 16 * f); ++i) {
                    const int r = 16 * f + i;
                    MhaRowState w;
                    paged_walk<T>(p, b, seq.t0 + r / p.group, kh * p.group + r % p.group, from + STEP * s0,
                                  min(end, paged_seen(p, seq, r / p.group)), lane, w);
                    MhaRow::store(mine + i * kLd, dim, lane, w.oa, w.ob);
                    if (lane == 0) {
                        mine[i * kLd + DP] = w.m;
                        mine[i * kLd + DP + 1] = w.l;
                    }
                }
            } else {
#pragma unroll
                for (int c = 0; c < VB; ++c)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int d = 64 * c + vw(c) * (4 * lh + e), to_d = paged_dim(d, vw(c), dim);
#pragma unroll
                        for (int w = 0; w < vw(c); ++w)
                            if (to_d + w >= d) mine[li * kLd + to_d + w] = o[f][4 * c + w][e];
                    }
                if (lh == 0) {
                    mine[li * kLd + DP] = m[f];
                    mine[li * kLd + DP + 1] = l[f];
                }
            }
            __syncthreads();
            const float *sums = reinterpret_cast<const float *>(lds);
            for (int i = wave; i < min(16, rows - 16 * f); i += NW) {  // a wave to a row, the waves' sums in order
                float mx = -INFINITY, sl = 0.0f, oa = 0.0f, ob = 0.0f;
#pragma unroll
                for (int w = 0; w < NW; ++w) mx = fmaxf(mx, sums[(w * 16 + i) * kLd + DP]);
                const float ref = mx == -INFINITY ? 0.0f : mx;
#pragma unroll
                for (int w = 0; w < NW; ++w) {
                    const float *t = sums + (w * 16 + i) * kLd;
                    const float f = __builtin_amdgcn_exp2f(t[DP] - ref);
                    sl += f * t[DP + 1];
                    if (lane < dim) oa += f * t[lane];
                    if (lane + 64 < dim) ob += f * t[lane + 64];
                }
                const int r = 16 * f + i;
                float *part = parts > 1 ? p.few_part + (((int64_t)x_ * p.few + r) * p.few_splits + z) * p.part_ld : nullptr;
                paged_finish(p, part, seq.t0 + r / p.group, kh * p.group + r % p.group, lane, mx, sl, oa, ob);
            }
        }
        if (!p.counters || parts == 1) return;
        // the workgroup that arrives last, whichever it is, joins the parts in their order and sets the counter back
        __shared__ int last;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the wave's rows are written
        __syncthreads();
        if (tid == 0) last = __hip_atomic_fetch_add(p.counters + x_ * kCounterStride, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == parts - 1;
        __syncthreads();
        if (!last) return;
        if (tid == 0) __hip_atomic_store(p.counters + x_ * kCounterStride, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        for (int r = wave; r < rows; r += NW)
            paged_join(p, p.few_part + ((int64_t)x_ * p.few + r) * p.few_splits * p.part_ld, parts, seq.t0 + r / p.group, kh * p.group + r % p.group, lane);
    }
};

// ------------------------------------------------------------- tiles of rows
// NW x FQ x 16 query rows of a key/value head against its keys in blocks of 32,
// staged in LDS, two stages: the products of MhaQueryTile's forward, with rows of
// the heads that share the keys beside each other (row = token * group + head), so
// that a tile's rows see nearly the same keys.
//  - A thread stages 8 dims of a key's K and V: its page is asked for a block
//    before the row, the row a block before its use.  fp32 rows are split there
//    (three parts), bf16 ones are operands as they lie (one part): six products
//    for one of fp32, or three.
//  - Bound by the products and the vector instructions beside them (softmax, P's
//    split, fp32 rows' split: 1.8 a product with fp32 pages, 2.2 with bf16 ones),
//    whose times nearly add up; the matrix cores are busy half of the time.  MI355X:
//    4 x 512 tokens of 32 heads (8) over 2730 to 8192 x 128 fp32 550 us and the
//    join's 14 (201 TFLOP/s), one prompt of 4096 tokens over bf16 pages 349 us (394).
//    Measured and not kept: softmax of one block of rows between the products of the
//    other (K and V's fragments read twice; 4 to 18% slower), a wave's priority raised
//    over its products (within 1%), three workgroups a CU, half of the waves half a
//    block behind the others (5% slower to 4% faster), fp32 rows' split between the
//    products with V (0 to 9% slower).
//  - The parts of all sequences' tiles are one range without gaps, and few rows of
//    other sequences follow it: where each part of each tile had a place of its own,
//    the gaps fell on the same XCDs or shader engines each time and left them idle (4
//    x 32 tokens of 16 (4) x 128 over 2048, in 12 parts: 52 us, 32 so).  The workgroups
//    that the host could not know to be too many come last.
template <int DP, int NP>
struct PagedFrags {
    typedef MhaBlock<DP> B;
    static constexpr int kTensor = NP * B::kPart, kStage = 2 * kTensor;
    const char *lds;
    int frag, tr[2];  // as MhaFrags'
    __device__ __forceinline__ PagedFrags(const char *lds, int lane) : lds(lds) {
        frag = B::slot(lane & 15, lane >> 4);
        tr[0] = B::slot(4 * (lane >> 4) + (lane & 15) / 4, lane % 4 / 2) + lane % 2 * 8;
        tr[1] = tr[0] ^ 32;
    }
    typedef zn_bf16x8 Set[2][NP];
    __device__ __forceinline__ void dims(int st, int t, int sl, Set &a) const {
#pragma unroll
        for (int q = NP - 1; q >= 0; --q)  // in the order of their use
#pragma unroll
            for (int rb = 0; rb < 2; ++rb)
                a[rb][q] = __builtin_bit_cast(zn_bf16x8, *reinterpret_cast<const zn_u32x4 *>(lds + st * kStage + t * kTensor + q * B::kPart +
                                                                                            sl * (B::BR * 64) + rb * (16 * 64) + frag));
    }
    __device__ __forceinline__ void rows(int st, int t, int db, Set &x) const {
        typedef short s4 __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) s4 ls4;
#pragma unroll
        for (int q = NP - 1; q >= 0; --q)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const char *at = lds + st * kStage + t * kTensor + q * B::kPart + ((db + c) / 2) * (B::BR * 64) + tr[(db + c) & 1];
                const s4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ls4 *)at), b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ls4 *)(at + 16 * 64));
                x[c][q] = __builtin_bit_cast(zn_bf16x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
            }
    }
    // The chunk of dims whose values a lane of quarter lh has in the accumulators of block db, and which half of it.
    __device__ static __forceinline__ int chunk_of(int db, int lh) { return 32 * (db / 2) + 8 * (2 * (db & 1) + lh / 2); }
};

template <typename T, int DP, int NW, int FQ, bool PAGES16>
struct PagedTile {
    static constexpr bool BF = sizeof(T) == 2;
    static constexpr int NP = BF ? 1 : 3, PRODUCTS = BF ? 3 : 6;
    typedef PagedFrags<DP, NP> Frags;
    typedef typename Frags::B B;
    static constexpr int SL = B::SL, DB = B::DB, NT = NW * kWave, ROWS = NW * FQ * 16;
    static constexpr int kUnits = B::BR * DP / 8, UPT = (kUnits + NT - 1) / NT;
    static constexpr int kFlag = 2 * Frags::kStage, kBytes = kFlag + 16;
    static constexpr float kUnscale = BF ? kPagedUnscale : kSplitUnscale;

    struct Stage {
        const ZnPagedCache &c;
        char *lds;
        const T *k, *v;
        const int32_t *table;
        int tid, wave, kl, page[UPT];
        bool hole = false;
        zn_u32x4_2 g[UPT][2][BF ? 1 : 2];
        __device__ __forceinline__ Stage(const ZnPagedCache &c, char *lds, int tid, int wave, int b, int kh, int kl)
            : c(c), lds(lds), k(reinterpret_cast<const T *>(c.k) + kh * c.stride[1]), v(reinterpret_cast<const T *>(c.v) + kh * c.stride[1]),
              table(c.table + (int64_t)b * c.max_pages), tid(tid), wave(wave), kl(kl) {}
        __device__ __forceinline__ int page_of(int j) const { return (int)(((uint64_t)(uint32_t)j * c.div_mul) >> (31 + c.div_shift)); }
        __device__ __forceinline__ bool mine(int i) const { return (i + 1) * NT <= kUnits || i * NT + tid < kUnits; }
        // Unit i's row of a block, and the key that its page is looked up for (past the sequence's end: its last): with pages of a
        // multiple of 16 positions the first of its 16 rows, which a wave's rows share (16 rows are a multiple of 64 units).  Against a
        // lookup a row (4 x 512 tokens of 32 heads (8) over 4096, pages of 64): bf16 of 128 dims 317 -> 312 us, of 64 198 -> 190, fp32
        // 601 -> 598 and 337 -> 349; 128 x 7 heads (1) of up to 64 tokens against up to 4096 x 96 bf16 258 -> 277.
        __device__ __forceinline__ int row(int i) const { return (i * NT + tid) / (DP / 8); }
        __device__ __forceinline__ int key(int i, int blk) const {
            return min(32 * blk + (PAGES16 ? (i * NT + wave * kWave) / (2 * DP) * 16 : row(i)), kl - 1);
        }
        __device__ __forceinline__ void pages(int blk) {
            typedef __attribute__((address_space(4))) const int32_t Table;  // constant: for scalar loads
#pragma unroll
            for (int i = 0; i < UPT; ++i) {
                if constexpr (PAGES16) page[i] = ((Table *)(uintptr_t)table)[page_of(key(i, blk))];
                else if (mine(i)) page[i] = table[page_of(key(i, blk))];
            }
        }
        __device__ __forceinline__ void fetch(int blk) {
#pragma unroll
            for (int i = 0; i < UPT; ++i) {
                if (!mine(i)) continue;
                const bool in = (uint32_t)page[i] < (uint32_t)c.pages;
                hole |= !in;
                const int j = key(i, blk);
                int64_t at = (in ? page[i] : 0) * c.stride[0] + (j - page_of(j) * c.page_size) * c.stride[2];
                if constexpr (PAGES16) {
                    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)at), hi = __builtin_amdgcn_readfirstlane((uint32_t)(at >> 32));
                    at = (int64_t)((uint64_t)hi << 32 | lo) + (int64_t)((uint64_t)(uint32_t)min(row(i) % 16, kl - 1 - j) * (uint32_t)c.stride[2]);
                }
                at += paged_dim((i * NT + tid) % (DP / 8) * 8, 8, c.dim);
                const T *const from[2] = {k + at, v + at};
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int h = 0; h < (BF ? 1 : 2); ++h) g[i][t][h] = *reinterpret_cast<const zn_u32x4_2 *>(from[t] + 4 * h);
            }
        }
        __device__ __forceinline__ void commit(int st) {
#pragma unroll
            for (int i = 0; i < UPT; ++i) {
                if (!mine(i)) continue;
                const int u = i * NT + tid, dc = u % (DP / 8);
                char *const to = lds + st * Frags::kStage + dc / 4 * (B::BR * 64) + B::slot(u / (DP / 8), dc % 4);
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    if constexpr (BF) {
                        *reinterpret_cast<zn_u32x4 *>(to + t * Frags::kTensor) = zn_u32x4{g[i][t][0][0], g[i][t][0][1], g[i][t][0][2], g[i][t][0][3]};
                    } else {
                        float x[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) x[e] = __builtin_bit_cast(float, (uint32_t)g[i][t][e / 4][e % 4]);
                        zn_u32x4 w[3];
                        split8(x, w);
#pragma unroll
                        for (int q = 0; q < 3; ++q) *reinterpret_cast<zn_u32x4 *>(to + t * Frags::kTensor + q * B::kPart) = w[q];
                    }
                }
            }
        }
    };

    // The sequence whose tiles' parts hold number `slot`, and which of them it is; or -1 and how many there are.  Those of 64 sequences
    // are summed at a time.
    __device__ static __forceinline__ int find(const ZnPagedArgs &p, int slot, int &at, PagedSeq &seq) {
        const int lane = threadIdx.x & (kWave - 1);
        int before = 0;
        for (int i0 = 0; i0 < p.c.batch; i0 += 64) {
            int own = 0;
            const PagedSeq s(p.c, min(i0 + lane, p.c.batch - 1));
            if (i0 + lane < p.c.batch) {
                const int n = min(s.ql, p.max_q), r = n * p.group;
                if (r > p.few) own = (r + ROWS - 1) / ROWS * paged_parts(paged_seen(p, s, n - 1), p.tile_len);
            }
            int sum = own;
#pragma unroll
            for (int s = 1; s < 64; s <<= 1) {
                const int y = __shfl_up(sum, s);
                if (lane >= s) sum += y;
            }
            const int n = __builtin_popcountll(__builtin_amdgcn_ballot_w64(before + sum <= slot));
            if (n < 64) {
                at = __builtin_amdgcn_readlane(slot - before - sum + own, n);
                seq.t0 = __builtin_amdgcn_readlane(s.t0, n);
                seq.ql = __builtin_amdgcn_readlane(s.ql, n);
                seq.kl = __builtin_amdgcn_readlane(s.kl, n);
                seq.first = seq.kl - seq.ql;
                return i0 + n;
            }
            before += __shfl(sum, 63);
        }
        at = __builtin_amdgcn_readfirstlane(before);
        return -1;
    }

    // Key/value head kh, part `at` of sequence b's tiles.
    __device__ static __forceinline__ void run(const ZnPagedArgs &p, char *lds, int kh, int b, int at, const PagedSeq &seq) {
        const int tid = threadIdx.x, lane = tid & (kWave - 1);
        const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
        const int li = lane & 15, lh = lane >> 4, dim = p.c.dim;
        // part z of the tile; a sequence's last tiles first, which see more keys
        const int rows = min(seq.ql, p.max_q) * p.group, tiles = max(1, (rows + ROWS - 1) / ROWS), z = at / tiles;
        if (rows == 0 || at < 0) return;  // starts that do not ascend
        const int r0 = __builtin_amdgcn_readfirstlane(tiles - 1 - (at - z * tiles)) * ROWS;
        // keys that any row of the workgroup sees, its parts, this one's blocks
        const int last = paged_seen(p, seq, (min(r0 + ROWS, rows) - 1) / p.group);
        const int parts = paged_parts(last, p.tile_len);
        if (z >= parts) return;
        const int blk0 = __builtin_amdgcn_readfirstlane(z * p.tile_len / 32), nblk = __builtin_amdgcn_readfirstlane((min((z + 1) * p.tile_len, last) + 31) / 32);

        // the first block's pages, then Q, then its rows: each on its way while the one before is waited for
        int *const flag = reinterpret_cast<int *>(lds + kFlag);
        if (tid == 0) *flag = 0;
        Stage sg(p.c, lds, tid, wave, b, kh, seq.kl);
        if (blk0 < nblk) sg.pages(blk0);
        __builtin_amdgcn_sched_barrier(0);
        const int w0 = r0 + wave * FQ * 16;
        int lim[FQ], all = INT_MAX, any = 0;
        float q[FQ][SL][8];
#pragma unroll
        for (int f = 0; f < FQ; ++f) {
            const int r = min(w0 + 16 * f + li, rows - 1), i = r / p.group;
            lim[f] = w0 + 16 * f + li < rows ? paged_seen(p, seq, i) : 0;
            const float *const row = p.q + (seq.t0 + i) * p.qs[0] + (kh * p.group + r - i * p.group) * p.qs[1];
#pragma unroll
            for (int sl = 0; sl < SL; ++sl) paged_query(row, lim[f] > 0, 32 * sl + 8 * lh, dim, p.scale_log2, q[f][sl]);
            all = min(all, lim[f]);
            any = max(any, lim[f]);
        }
        if (blk0 < nblk) {
            sg.fetch(blk0);
            sg.pages(blk0 + 1);
        }
        __builtin_amdgcn_sched_barrier(0);
        zn_bf16x8 qf[FQ][SL][3];
#pragma unroll
        for (int f = 0; f < FQ; ++f)
#pragma unroll
            for (int sl = 0; sl < SL; ++sl) {
                zn_u32x4 w[3];
                split8(q[f][sl], w);
#pragma unroll
                for (int part = 0; part < 3; ++part) qf[f][sl][part] = __builtin_bit_cast(zn_bf16x8, w[part]);
            }
#pragma unroll
        for (int s = 1; s < 16; s <<= 1) {
            all = min(all, __shfl_xor(all, s));
            any = max(any, __shfl_xor(any, s));
        }
        all = __builtin_amdgcn_readfirstlane(all);
        any = __builtin_amdgcn_readfirstlane(any);

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
        if (blk0 < nblk) sg.commit(0);
        for (int blk = blk0; blk < nblk; ++blk) {
            const int st = (blk - blk0) & 1, k0 = 32 * blk;
            __syncthreads();  // block blk is in LDS; every wave is done with block blk - 1
            if (blk + 1 < nblk) {
                sg.fetch(blk + 1);
                sg.pages(blk + 2);
            }
            if (k0 < any) block(fr, st, k0 + 32 > all, k0, lane, lim, qf, o, m, l);
            if (blk + 1 < nblk) sg.commit(st ^ 1);
        }
        if (sg.hole) *flag = 1;
        __syncthreads();
        bool bad = *flag;
#pragma unroll
        for (int f = 0; f < FQ; ++f) {
            bad |= !(l[f] < INFINITY) || (m[f] == -INFINITY && blk0 < nblk && lim[f] > 32 * blk0);
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    bad |= !(__builtin_fabsf(o[f][d][r]) < INFINITY);
                    o[f][d][r] *= kUnscale;
                }
        }
        auto part_of = [&](int t, int h) { return parts > 1 ? p.tile_part + (((int64_t)t * p.q_heads + h) * p.tile_splits + z) * p.part_ld : nullptr; };
        if (__builtin_amdgcn_ballot_w64(bad)) {  // as PagedFew's
            for (int r = w0; r < min(w0 + 16 * FQ, rows); ++r) {
                const int i = r / p.group, t = seq.t0 + i, h = kh * p.group + r - i * p.group;
                MhaRowState w;
                paged_walk<T>(p, b, t, h, 32 * blk0, min(32 * nblk, paged_seen(p, seq, i)), lane, w);
                paged_finish(p, part_of(t, h), t, h, lane, w.m, w.l, w.oa, w.ob);
            }
            return;
        }
#pragma unroll
        for (int f = 0; f < FQ; ++f) {
            const int r = w0 + 16 * f + li, i = r / p.group, t = seq.t0 + i, h = kh * p.group + r - i * p.group;
            float sum = l[f] + __shfl_xor(l[f], 16);
            sum += __shfl_xor(sum, 32);
            if (r >= rows) continue;
            float *const part = part_of(t, h), *const to = part ? part : p.out + t * p.os[0] + h * p.os[1];
            const float div = part || sum == 0.0f ? 1.0f : sum;
#pragma unroll
            for (int d = 0; d < DB; ++d) {
                const int at = Frags::chunk_of(d, lh), half = 4 * (lh & 1);
                const zn_f32x4 x = o[f][d] / div;
                if (at + 8 <= dim) {
                    *reinterpret_cast<zn_f32x4u *>(to + at + half) = x;
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (dim - 8 + half + e >= at) to[dim - 8 + half + e] = x[e];
                }
            }
            if (lh != 0) continue;
            if (part) {
                part[p.part_ld - 4] = m[f];
                part[p.part_ld - 3] = sum;
            } else if (p.lse) {
                p.lse[(int64_t)t * p.q_heads + h] = mha_lse(m[f], sum);
            }
        }
    }

    // One block of 32 keys: S^T = K (cQ)^T, then O^T += V^T P^T.  `mask` (of the whole wave): some of its pairs are masked.
    __device__ static __forceinline__ void block(const Frags &sg, int st, bool mask, int k0, int lane, const int (&lim)[FQ],
                                                 const zn_bf16x8 (&qf)[FQ][SL][3], zn_f32x4 (&o)[FQ][DB], float (&m)[FQ], float (&l)[FQ]) {
        const int lh = lane >> 4;
        zn_f32x4 s[FQ][2];
#pragma unroll
        for (int f = 0; f < FQ; ++f) s[f][0] = s[f][1] = zn_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        typename Frags::Set a[2];
        constexpr int NR = DB / 2, M = 2 * FQ * PRODUCTS;
        // The products' parts, the largest last.
        constexpr int PA[6] = {BF ? 0 : 2, BF ? 0 : 1, 0, 1, 0, 0}, PB[6] = {BF ? 2 : 0, 1, BF ? 0 : 2, 0, 1, 0};
        sg.dims(st, 0, 0, a[0]);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < SL; ++i) {
            if (i + 1 < SL) sg.dims(st, 0, i + 1, a[(i + 1) & 1]);
            else sg.rows(st, 1, 0, a[(i + 1) & 1]);
#pragma unroll
            for (int pr = 0; pr < PRODUCTS; ++pr)
#pragma unroll
                for (int rb = 0; rb < 2; ++rb)
#pragma unroll
                    for (int f = 0; f < FQ; ++f)
                        s[f][rb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i & 1][rb][PA[pr]], qf[f][i][PB[pr]], s[f][rb], 0, 0, 0);
            if (i + 1 < SL) mha_order<M, 2 * NP>();
            else mha_order<M, 4 * NP>();
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
            float x[8], mb = -INFINITY;
#pragma unroll
            for (int e = 0; e < 8; ++e) mb = fmaxf(mb, s[f][e / 4][e % 4]);
            // The reference moves where the maximum leaves it by more than 2^8: until then the probabilities are up to 2^8 times what they
            // are relative to the maximum, which no rounding sees, and O is not multiplied (16 vector instructions for every 16 dims; 4 x
            // 512 tokens of 32 heads (8) over 4096, bf16 of 128 dims 318 -> 312 us, of 64 196 -> 190, fp32 of 128 610 -> 598).
            const float top = max_over_rows(mb) * kUnscale, mn = top > m[f] + 8.0f ? top : m[f];
            const float ref = mn == -INFINITY ? 0.0f : mn;  // nothing seen so far
            const float alpha = __builtin_amdgcn_exp2f(m[f] - ref);
            float rs = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[f][e / 4][e % 4], kUnscale, -ref));
                rs += x[e];
                x[e] *= kSplitScale;
            }
            l[f] = l[f] * alpha + rs;
            m[f] = mn;
            if (__builtin_amdgcn_ballot_w64(alpha != 1.0f)) {
#pragma unroll
                for (int d = 0; d < DB; ++d) o[f][d] *= alpha;
            }
            if constexpr (BF) paged_split8(x, pf[f]);
            else mha_split8(x, pf[f]);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            if (i + 1 < NR) sg.rows(st, 1, 2 * (i + 1), a[(SL + i + 1) & 1]);
#pragma unroll
            for (int pr = 0; pr < PRODUCTS; ++pr)
#pragma unroll
                for (int c = 0; c < 2; ++c)
#pragma unroll
                    for (int f = 0; f < FQ; ++f)
                        o[f][2 * i + c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[(SL + i) & 1][c][PA[pr]], pf[f][PB[pr]], o[f][2 * i + c], 0, 0, 0);
            mha_order<M, 4 * NP>();
        }
    }
};

}  // namespace

// The join of rows that are in parts.  Grid x: the tokens, y: groups of four heads, a wave each (one after the other where the call
// has many tokens: a token's place is three dependent loads).
extern "C" __global__ __launch_bounds__(256) void zn_paged_join(ZnPagedArgs p) {
    const int lane = threadIdx.x & (kWave - 1), t = blockIdx.x;
    const int b = paged_find(p.c, t);
    if (b < 0 || b >= p.c.batch) return;
    const PagedSeq seq(p.c, b);
    const int rows = min(seq.ql, p.max_q) * p.group, i = t - seq.t0;
    if (i < 0 || i * p.group >= rows) return;
    const bool few = rows <= p.few;
    const int any = few ? paged_seen(p, seq, (rows - 1) / p.group) : 0, few_parts = few ? paged_parts(any, paged_few_len(p, any)) : 0;
    for (int h = blockIdx.y * 4 + threadIdx.x / kWave; h < p.q_heads; h += gridDim.y * 4) {
        const int kh = h / p.group, r = i * p.group + h - kh * p.group;
        if (few) {
            if (few_parts > 1) paged_join(p, p.few_part + (((int64_t)b * p.c.kv_heads + kh) * p.few + r) * p.few_splits * p.part_ld, few_parts, t, h, lane);
        } else {
            const int parts = paged_parts(paged_seen(p, seq, (min((r / p.tile + 1) * p.tile, rows) - 1) / p.group), p.tile_len);
            if (parts > 1) paged_join(p, p.tile_part + ((int64_t)t * p.q_heads + h) * p.tile_splits * p.part_ld, parts, t, h, lane);
        }
    }
}

extern "C" __global__ __launch_bounds__(256) void zn_paged_rows_f32(ZnPagedArgs p) { paged_rows<float>(p); }
extern "C" __global__ __launch_bounds__(256) void zn_paged_rows_bf16(ZnPagedArgs p) { paged_rows<__bf16>(p); }

#define ZN_PAGED_KERNEL(NAME, NW, BYTES, ...)                                      \
    extern "C" __global__ __launch_bounds__(NW * 64, 2) void NAME(ZnPagedArgs p) { \
        __shared__ __attribute__((aligned(1024))) char lds[BYTES];                 \
        __VA_ARGS__;                                                               \
    }
// Few rows: grid x the sequences' key/value heads, z the parts.  P: pages whose size is a multiple of 16 (_p), any.
#define ZN_PAGED_FEW(NAME, ...)                                                                          \
    typedef PagedFew<__VA_ARGS__> NAME##_k;                                                             \
    ZN_PAGED_KERNEL(NAME, 4, NAME##_k::kBytes, NAME##_k::run(p, lds, blockIdx.x, blockIdx.z))
// NW waves of F blocks of 16 rows: the tiles' parts, then the parts of few rows.
#define ZN_PAGED_TILE(NAME, T, DP, NW, F, P)                                                             \
    typedef PagedTile<T, DP, NW, F, P> NAME##_k;                                                        \
    typedef PagedFew<T, DP, NW, 1, P> NAME##_f;                                                         \
    ZN_PAGED_KERNEL(NAME, NW, (NAME##_k::kBytes > NAME##_f::kBytes ? NAME##_k::kBytes : NAME##_f::kBytes), \
                    const int slot = blockIdx.x / p.c.kv_heads;                                         \
                    int at;                                                                             \
                    PagedSeq seq(p.c);                                                                  \
                    const int b = NAME##_k::find(p, slot, at, seq);                                     \
                    if (b >= 0) return NAME##_k::run(p, lds, blockIdx.x - slot * p.c.kv_heads, b, at, seq); \
                    const int x = (int)blockIdx.x - at * p.c.kv_heads;                                  \
                    if (p.few && x < p.few_heads * p.few_splits) NAME##_f::run(p, lds, x % p.few_heads, x / p.few_heads))
#define ZN_PAGED_KERNELS(DP, S, P)                                        \
    ZN_PAGED_FEW(zn_paged_few_f32_##DP##S, float, DP, 4, 1, P)            \
    ZN_PAGED_FEW(zn_paged_few2_f32_##DP##S, float, DP, 4, 2, P)           \
    ZN_PAGED_FEW(zn_paged_few4_f32_##DP##S, float, DP, 4, 4, P)           \
    ZN_PAGED_FEW(zn_paged_few_bf16_##DP##S, __bf16, DP, 4, 1, P)          \
    ZN_PAGED_FEW(zn_paged_few2_bf16_##DP##S, __bf16, DP, 4, 2, P)         \
    ZN_PAGED_FEW(zn_paged_few4_bf16_##DP##S, __bf16, DP, 4, 4, P)
#define ZN_PAGED_TILES(DP, NW, F, S, P)                                   \
    ZN_PAGED_TILE(zn_paged_tile_f32_##DP##S, float, DP, NW, F, P)         \
    ZN_PAGED_TILE(zn_paged_wide_f32_##DP##S, float, DP, 8, 2, P)          \
    ZN_PAGED_TILE(zn_paged_tile_bf16_##DP##S, __bf16, DP, 4, 2, P)
ZN_PAGED_KERNELS(32, , false)
ZN_PAGED_KERNELS(32, _p, true)
ZN_PAGED_KERNELS(64, , false)
ZN_PAGED_KERNELS(64, _p, true)
ZN_PAGED_KERNELS(96, , false)
ZN_PAGED_KERNELS(96, _p, true)
ZN_PAGED_KERNELS(128, , false)
ZN_PAGED_KERNELS(128, _p, true)
#define ZN_PAGED_TILES2(...) ZN_PAGED_TILES(__VA_ARGS__, , false) ZN_PAGED_TILES(__VA_ARGS__, _p, true)
// dims; fp32 pages: waves and blocks of 16 rows of tiles of 128 rows.  bf16 pages have no tiles of 256: a block of 32 keys of 128 dims
// takes 2.5 us there and 2.6 in two tiles of 128 on the same CU, which cut a call's work finer.
ZN_PAGED_TILES2(32, 4, 2)
ZN_PAGED_TILES2(64, 4, 2)
ZN_PAGED_TILES2(96, 8, 1)
ZN_PAGED_TILES2(128, 8, 1)

#endif
