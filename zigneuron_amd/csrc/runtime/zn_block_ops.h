// Language-model blocks of the C ABI (include/zn_hip.h): grouped attention,
// the gated Dense layer and distillation, forward and backward.  Included by
// zn_hip.cpp, whose helpers it uses.
#ifndef ZN_BLOCK_OPS_H
#define ZN_BLOCK_OPS_H

#include <cmath>

// ------------------------------------------------------- grouped attention
namespace {

constexpr int64_t kMhaMaxDim = 128;
constexpr int64_t kMhaMaxRow = (int64_t)1 << 22;  // position stride: a block of 64 rows stays inside 32-bit offsets

constexpr int64_t kMhaMaxBlocks = ((int64_t)1 << 24) - 1;  // 32-row blocks to split in one launch

// Element strides that a call only reads, or (written) also writes.
bool mha_strides_ok(int64_t sb, int64_t sh, int64_t ss, int64_t batch, int64_t heads, int64_t rows, int64_t dim,
                    bool written) {
    if (ss < dim || ss > kMhaMaxRow || sb < 0 || sh < 0) return false;
    return !written || rows == 0 || heads == 0 || ((sb > 0 || batch <= 1) && (sh > 0 || heads <= 1));
}

// The checks and the argument block that both directions share.  *work: there is something to do.
int mha_args(zn_ctx *ctx, ZnMhaArgs &a, int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t q_len, int64_t kv_len,
             int64_t head_dim, float scale, int causal, const void *q_lens, const void *kv_lens, const int64_t (&qs)[3],
             const int64_t (&ks)[3], const int64_t (&os)[3], bool backward, bool *work) {
    *work = false;
    if (!ctx || batch < 0 || q_heads < 0 || kv_heads < 0 || q_len < 0 || kv_len < 0 || head_dim < 1 ||
        head_dim > kMhaMaxDim || !std::isfinite(scale) || causal < 0 || causal > 1)
        return ZN_ERR_INVALID_ARG;
    if (kv_heads == 0 ? q_heads != 0 : q_heads % kv_heads != 0) return ZN_ERR_INVALID_ARG;
    if (!mha_strides_ok(qs[0], qs[1], qs[2], batch, q_heads, q_len, head_dim, backward) ||
        !mha_strides_ok(ks[0], ks[1], ks[2], batch, kv_heads, kv_len, head_dim, backward) ||
        !mha_strides_ok(os[0], os[1], os[2], batch, q_heads, q_len, head_dim, !backward))
        return ZN_ERR_INVALID_ARG;
    constexpr int64_t kMax = INT_MAX / 2, kMaxHeads = (int64_t)1 << 22;  // heads: a launch has fewer than 2^32 threads
    if (batch > kMax || q_heads > kMax || kv_heads > kMax || q_len > kMax || kv_len > kMax || batch * q_heads > kMax || batch * kv_heads > kMaxHeads)
        return ZN_ERR_OVERFLOW;
    const int64_t tile = kMhaRows[kMhaGrad][(head_dim - 1) / 32], max_rows = 65533 * tile;  // tiles: the grid's second extent
    if (kv_len + (kv_heads ? q_heads / kv_heads * (q_len + tile) : 0) > max_rows) return ZN_ERR_OVERFLOW;
    std::memset(&a, 0, sizeof(a));
    std::memcpy(a.qs, qs, sizeof(a.qs));
    std::memcpy(a.ks, ks, sizeof(a.ks));
    std::memcpy(a.os, os, sizeof(a.os));
    a.q_lens = static_cast<const int32_t *>(q_lens);
    a.kv_lens = static_cast<const int32_t *>(kv_lens);
    a.batch = (int32_t)batch;
    a.q_heads = (int32_t)q_heads;
    a.kv_heads = (int32_t)kv_heads;
    a.group = kv_heads ? (int32_t)(q_heads / kv_heads) : 0;
    a.q_len = (int32_t)q_len;
    a.kv_len = (int32_t)kv_len;
    a.dim = (int32_t)head_dim;
    a.causal = causal;
    a.scale = scale;
    a.scale_log2 = scale * 1.44269504088896340736f;
    *work = batch > 0 && kv_heads > 0;
    return ZN_OK;
}

int64_t mha_rows(MhaKernel kernel, const ZnMhaArgs &a) { return kMhaRows[kernel][(a.dim - 1) / 32]; }

// Query tiles of a key/value head: the same number for each query head of its group.
int64_t mha_query_tiles(MhaKernel kernel, const ZnMhaArgs &a) {
    return a.group * cdiv(cdiv((int64_t)a.group * a.q_len, mha_rows(kernel, a)), std::max(a.group, 1));
}

constexpr double kPartUs = 2.0;  // the way in and out of a walk

// One kind of tile of a call: how many, the blocks that one walks, the times of a
// block, the rows that a part of its walk writes for zn_mha_join.
struct MhaWalks {
    int64_t tiles, blocks;
    double block_us, alone_us;  // of a CU whose workgroups fill it, of a workgroup alone
    int64_t rows;
    int32_t splits;
};

// `factor`: a block's products against the forward's.  A workgroup of 4 waves has half a CU's, and alone does not fill it.
MhaWalks mha_walks(MhaKernel kernel, const ZnMhaArgs &a, int64_t tiles, int64_t blocks, double factor, int64_t rows) {
    const double us = (0.8 + 0.012 * a.dim) * factor * (double)mha_rows(kernel, a) / 128.0;
    return {tiles, blocks, us, us * (kMhaThreads[kernel][(a.dim - 1) / 32] == 256 ? 1.3 : 1.0), rows, 1};
}

// The parts that each kind's walks are cut into: the least of the longest part
// or all parts' time on the chip, whichever is more, and the join, 4 us and each
// part's rows written and read at 2 TB/s.  A walk is long where queries of many
// heads pass the same keys, and few tiles leave most of the chip idle; causal
// tiles average half their walk.  MI355X, us whole (few tiles, both gradients:
// in equal parts) and so: both gradients of 2 x 16 heads (4) of 2048 x 128,
// causal, 1013 and 640, 4 x 28 (4) of 500 x 128 438 and 197, one of 4096 x 128
// 142 and 107; its forward 52 and 46.  But 8 x 16 of 1024 x 128 1252 and 1236.
// Returns the time so found.
double mha_splits(const zn_ctx *ctx, const ZnMhaArgs &a, MhaWalks *w, int kinds) {
    constexpr int kParts[12] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64};
    const double cus = (double)cus_now(ctx), share = a.causal ? 0.5 : 1.0;
    const int64_t heads = (int64_t)a.batch * a.kv_heads;
    double best = INFINITY;
    for (int i = 0; i < (kinds > 1 ? 12 : 1); ++i)
        for (int j = 0; j < 12; ++j) {
            const int s[2] = {kParts[j], kParts[i]};
            double all = 0.0, longest = 0.0, join = 0.0;
            int64_t y = 0;
            for (int k = 0; k < kinds; ++k) {
                const double part = kPartUs + w[k].alone_us * (double)cdiv(w[k].blocks, s[k]);
                all += (double)(w[k].tiles * s[k]) * kPartUs + (double)w[k].tiles * w[k].block_us * (double)w[k].blocks * share;
                longest = std::max(longest, w[k].tiles ? part : 0.0);
                if (s[k] > 1) join = std::max(join, 4.0) + 8.0 * (double)(w[k].rows * s[k]) * a.dim / 2e6;
                y += w[k].tiles / heads * s[k];
                if (s[k] > std::max<int64_t>(1, w[k].blocks)) y = INT_MAX;
            }
            const double us = std::max(longest, all / cus) + join;
            if (us < best && (y <= 65535 || (s[0] == 1 && s[1] == 1))) {
                best = us;
                for (int k = 0; k < kinds; ++k) w[k].splits = s[k];
            }
        }
    return best;
}

int mha_tiles(zn_ctx *ctx, MhaKernel kernel, ZnMhaArgs &a, int64_t y, int parts) {
    const int dim = (a.dim - 1) / 32;
    return launch(ctx, ctx->mha[kernel][dim], (unsigned)(a.batch * a.kv_heads), (unsigned)y, kMhaThreads[kernel][dim], &a, (unsigned)parts);
}

int mha_join(zn_ctx *ctx, const ZnMhaArgs &a, ZnMhaJoinArgs &j, int ops) {
    j.part_ld = a.part_ld;
    j.dim = a.dim;
    int64_t rows = 0;
    for (int i = 0; i < ops; ++i) rows = std::max(rows, j.op[i].rows);
    return launch(ctx, ctx->mha_join, (unsigned)cdiv(rows, 4), (unsigned)ops, 256, &j);
}

void mha_join_op(ZnMhaJoinOp &op, const float *part, float *dst, const int64_t (&stride)[3], int64_t batch, int32_t heads, int32_t len, int32_t splits, float factor) {
    op.part = part;
    op.dst = dst;
    std::memcpy(op.stride, stride, sizeof(op.stride));
    op.rows = batch * heads * len;
    op.heads = heads;
    op.len = len;
    op.splits = splits;
    op.factor = factor;
}

// The images that a call's tiles read (kernels/mha_f32.h), in one leased buffer.
struct MhaImages {
    Lease lease;
    ZnMhaSplitArgs s;
    int64_t bytes = 0, groups = 0;
    explicit MhaImages(zn_ctx *ctx) : lease(ctx) { std::memset(&s, 0, sizeof(s)); }
    // A tensor's image: its offset in the buffer.
    int64_t add(const ZnMhaArgs &a, const float *src, const int64_t (&stride)[3], const int32_t *lens, int heads, int len, float scale) {
        ZnMhaSplitOp &op = s.op[s.ops++];
        op.src = src;
        std::memcpy(op.stride, stride, sizeof(op.stride));
        op.lens = lens;
        op.heads = heads;
        op.len = len;
        op.blocks = (int32_t)cdiv(len, 32);
        op.scale = scale;
        op.first = (int32_t)groups;
        groups += (int64_t)a.batch * heads * op.blocks;
        const int64_t at = bytes;
        bytes += (int64_t)a.batch * heads * op.blocks * (192 * 32) * cdiv(a.dim, 32);
        return at;
    }
    int get(int64_t more) { return lease.get((size_t)((bytes + more) / 4)); }
    char *at(int64_t offset) const { return reinterpret_cast<char *>(lease.ptr) + offset; }
    int run(zn_ctx *ctx, const ZnMhaArgs &a) {
        s.dim = a.dim;
        s.causal = a.causal;
        return groups ? launch(ctx, ctx->mha[kMhaSplit][(a.dim - 1) / 32], (unsigned)groups, 1, 256, &s) : ZN_OK;
    }
};

}  // namespace

int zn_hip_mha_forward(zn_ctx *ctx, const float *q, const float *k, const float *v, float *out, float *lse,
                       int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t q_len, int64_t kv_len,
                       int64_t head_dim, float scale, int causal, const void *q_lens, const void *kv_lens,
                       int64_t q_stride_b, int64_t q_stride_h, int64_t q_stride_s, int64_t kv_stride_b,
                       int64_t kv_stride_h, int64_t kv_stride_s, int64_t out_stride_b, int64_t out_stride_h,
                       int64_t out_stride_s) {
    ZnMhaArgs a;
    bool work = false;
    int rc = mha_args(ctx, a, batch, q_heads, kv_heads, q_len, kv_len, head_dim, scale, causal, q_lens, kv_lens,
                      {q_stride_b, q_stride_h, q_stride_s}, {kv_stride_b, kv_stride_h, kv_stride_s},
                      {out_stride_b, out_stride_h, out_stride_s}, false, &work);
    if (rc || !work || q_heads == 0 || q_len == 0) return rc;
    if (!q || !out || (kv_len > 0 && (!k || !v))) return ZN_ERR_INVALID_ARG;
    if ((rc = select_device(ctx))) return rc;
    a.q = q;
    a.k = k;
    a.v = v;
    a.out = out;
    a.lse = lse;
    // At most 16 rows of a head read K and V as they are.  Each tile splits what it reads: past a few tiles, once for all of
    // them is cheaper.
    const int64_t rows = (int64_t)a.group * q_len, heads = (int64_t)a.batch * a.kv_heads;
    MhaKernel kernel = rows <= mha_rows(kMhaFew, a) ? kMhaFew : rows < 3 * mha_rows(kMhaForwardRaw, a) ? kMhaForwardRaw : kMhaForward;
    if (kernel == kMhaFew) {
        a.query_tiles = 1;
        // parts of about 96 KB of K and V each, at most two workgroups a CU; past 8 a multiple of them, which the join reads at once
        // (MI355X, us in parts of 256 keys and so: 4 x 8 of 700 x 64 14.2 and 11.6, 4 x 8 of 1100 x 128 28.2 and 21.7, 4 of
        // 600 x 120 21.1 and 14.1; 8 x 4 of 2048 x 64 in 8 parts 13.7, in 11 15.7, in 16 14.8)
        a.splits = (int32_t)std::max<int64_t>(1, std::min<int64_t>({64, 2 * cus_now(ctx) / heads, (kv_len * a.dim + 4915) / 12288}));
        if (a.splits > 8) a.splits -= a.splits % 8;
    } else {
        const int64_t q_rows = batch * q_heads * q_len, blocks = cdiv(kv_len, 32);
        MhaWalks w = mha_walks(kernel, a, heads * mha_query_tiles(kernel, a), blocks, 1.0, q_rows);
        const double us = mha_splits(ctx, a, &w, 1);
        if (kernel == kMhaForward && mha_rows(kMhaForwardWide, a)) {
            MhaWalks wide = mha_walks(kMhaForwardWide, a, heads * mha_query_tiles(kMhaForwardWide, a), blocks, 0.9, q_rows);
            if (mha_splits(ctx, a, &wide, 1) < 0.97 * us) {
                kernel = kMhaForwardWide;
                w = wide;
            }
        }
        a.query_tiles = (int32_t)(w.tiles / heads);
        a.splits = w.splits;
    }
    Lease part(ctx);
    if (a.splits > 1) {
        a.part_ld = (a.dim + 3) / 4 * 4 + 4;
        if ((rc = part.get((size_t)(batch * q_heads * q_len) * a.splits * a.part_ld))) return rc;
        a.part = part.ptr;
    }
    MhaImages im(ctx);
    if (kernel != kMhaFew && kernel != kMhaForwardRaw && kv_len > 0) {
        const int64_t ki = im.add(a, k, a.ks, a.kv_lens, a.kv_heads, a.kv_len, 1.0f), vi = im.add(a, v, a.ks, a.kv_lens, a.kv_heads, a.kv_len, 1.0f);
        if (im.groups > kMhaMaxBlocks) return ZN_ERR_OVERFLOW;
        if ((rc = im.get(0))) return rc;
        a.k_blocks = im.s.op[0].blocks;
        a.ki = im.s.op[0].dst = im.at(ki);
        a.vi = im.s.op[1].dst = im.at(vi);
        if ((rc = im.run(ctx, a))) return rc;
    }
    if ((rc = mha_tiles(ctx, kernel, a, kernel == kMhaFew ? 1 : (int64_t)a.query_tiles * a.splits, kernel == kMhaFew ? a.splits : 1)) || a.splits == 1) return rc;
    ZnMhaJoinArgs j;
    std::memset(&j, 0, sizeof(j));
    j.forward = 1;
    j.lse = lse;
    mha_join_op(j.op[0], a.part, out, a.os, a.batch, a.q_heads, a.q_len, a.splits, 1.0f);
    return mha_join(ctx, a, j, 1);
}

int zn_hip_mha_backward(zn_ctx *ctx, const float *q, const float *k, const float *v, const float *out,
                        const float *lse, const float *grad_out, float *grad_q, float *grad_k, float *grad_v,
                        int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t q_len, int64_t kv_len,
                        int64_t head_dim, float scale, int causal, const void *q_lens, const void *kv_lens,
                        int64_t q_stride_b, int64_t q_stride_h, int64_t q_stride_s, int64_t kv_stride_b,
                        int64_t kv_stride_h, int64_t kv_stride_s, int64_t out_stride_b, int64_t out_stride_h,
                        int64_t out_stride_s) {
    ZnMhaArgs a;
    bool work = false;
    int rc = mha_args(ctx, a, batch, q_heads, kv_heads, q_len, kv_len, head_dim, scale, causal, q_lens, kv_lens,
                      {q_stride_b, q_stride_h, q_stride_s}, {kv_stride_b, kv_stride_h, kv_stride_s},
                      {out_stride_b, out_stride_h, out_stride_s}, true, &work);
    const bool queries = q_heads > 0 && q_len > 0;
    if (rc || !work || (!queries && kv_len == 0)) return rc;
    if (queries && (!q || !out || !lse || !grad_out || !grad_q)) return ZN_ERR_INVALID_ARG;
    if (kv_len > 0 && (!k || !v || !grad_k || !grad_v)) return ZN_ERR_INVALID_ARG;
    if ((rc = select_device(ctx))) return rc;
    a.q = q;
    a.k = k;
    a.v = v;
    a.grad_out = grad_out;
    a.grad_q = grad_q;
    a.grad_k = grad_k;
    a.grad_v = grad_v;
    MhaImages im(ctx);
    const int64_t qi = im.add(a, q, a.qs, a.q_lens, a.q_heads, a.q_len, a.scale_log2);
    const int64_t gi = im.add(a, grad_out, a.os, a.q_lens, a.q_heads, a.q_len, 1.0f);
    const int64_t ki = im.add(a, k, a.ks, a.kv_lens, a.kv_heads, a.kv_len, 1.0f);
    const int64_t vi = im.add(a, v, a.ks, a.kv_lens, a.kv_heads, a.kv_len, 1.0f);
    if (im.groups > kMhaMaxBlocks) return ZN_ERR_OVERFLOW;
    a.q_blocks = im.s.op[0].blocks;
    a.k_blocks = im.s.op[2].blocks;
    if ((rc = im.get((int64_t)a.batch * a.q_heads * a.q_blocks * 512))) return rc;  // and the sides
    a.qi = im.s.op[0].dst = im.at(qi);
    a.gi = im.s.op[1].dst = im.at(gi);
    a.ki = im.s.op[2].dst = im.at(ki);
    a.vi = im.s.op[3].dst = im.at(vi);
    im.s.op[0].lse = im.s.op[1].lse = lse;
    im.s.op[1].out = out;
    a.side = im.s.op[1].side = reinterpret_cast<float *>(im.at(im.bytes));
    if ((rc = im.run(ctx, a))) return rc;
    a.key_tiles = (int32_t)cdiv(kv_len, mha_rows(kMhaGrad, a));
    a.query_tiles = queries ? (int32_t)mha_query_tiles(kMhaGrad, a) : 0;
    const int64_t q_rows = batch * q_heads * q_len, k_rows = batch * kv_heads * kv_len, heads = (int64_t)a.batch * a.kv_heads;
    MhaWalks w[2] = {mha_walks(kMhaGrad, a, heads * a.query_tiles, a.k_blocks, 1.35, q_rows),
                     mha_walks(kMhaGrad, a, heads * a.key_tiles, (int64_t)a.group * a.q_blocks, 1.8, 2 * k_rows)};
    mha_splits(ctx, a, w, 2);
    a.splits = w[0].splits;
    a.kv_splits = w[1].splits;
    a.part_ld = (a.dim + 3) / 4 * 4;
    Lease part(ctx);
    const int64_t q_part = a.splits > 1 ? q_rows * a.splits * a.part_ld : 0, k_part = a.kv_splits > 1 ? k_rows * a.kv_splits * a.part_ld : 0;
    if (q_part + k_part > 0) {
        if ((rc = part.get((size_t)(q_part + 2 * k_part)))) return rc;
        a.part = part.ptr;
        a.kv_part = part.ptr + q_part;
    }
    if ((rc = mha_tiles(ctx, kMhaGrad, a, (int64_t)a.key_tiles * a.kv_splits + (int64_t)a.query_tiles * a.splits, 1))) return rc;
    ZnMhaJoinArgs j;
    std::memset(&j, 0, sizeof(j));
    int ops = 0;
    if (q_part > 0) mha_join_op(j.op[ops++], a.part, grad_q, a.qs, a.batch, a.q_heads, a.q_len, a.splits, a.scale);
    if (k_part > 0) {
        mha_join_op(j.op[ops++], a.kv_part, grad_k, a.ks, a.batch, a.kv_heads, a.kv_len, a.kv_splits, 1.0f);
        mha_join_op(j.op[ops++], a.kv_part + k_part, grad_v, a.ks, a.batch, a.kv_heads, a.kv_len, a.kv_splits, 1.0f);
    }
    return ops ? mha_join(ctx, a, j, ops) : ZN_OK;
}

// ----------------------------------------------------------- gated Dense
// One problem's operands stay below 2 GiB, as every GEMM's: x, W and, for the backward, z.
constexpr int64_t kGatedLimit = (int64_t)INT_MAX / 4;

static bool gated_extents_ok(int64_t batch, int64_t in_size, int64_t hidden, bool backward) {
    if (batch > INT_MAX || in_size > INT_MAX || hidden > INT_MAX / 2) return false;
    const int64_t n = 2 * hidden;
    return batch * in_size <= kGatedLimit && in_size * n <= kGatedLimit && (!backward || batch * n <= kGatedLimit);
}

// At most 16 rows: from this many weights on the kernel that reads them once
// (MI355X, us with it and as a product and a pass: 4 x 1024 x 8192 9.4 and 14.6,
// 1 x 4096 x 16384 56 and 81; 4 x 512 x 1024 7.3 and 5.7, 8 x 1024 x 2048 8.2 and 7.7;
// in parts of K, of at least 1024 each: 5 x 4096 x 8192 41 us whole, 32 in two).
constexpr int64_t kFewWeights = (int64_t)3 << 20;

// Whether the two projections, n columns together, run as one launch with the
// gate: by the estimates of the unsplit split tiles, and of the product on its
// own (K slices where they pay, or the fp32 kernels at the 75 TFLOP/s that they
// reach on such sizes) with a pass over z at 4 TB/s behind it.  MI355X, us in one
// launch and in two: 777 x 1023 x 2002 39 and 53, 4096 x 64 x 2048 19 and 42,
// 2048 x 256 x 1024 16 and 20, 4096 x 1024 x 8192 332 and 348; 1024 x 512 x
// 1024 21 and 18, 512 x 2048 x 4096 (K slices) 75 and 65, 256 x 1024 x 2048
// 34 and 27, 64 x 256 x 512 13 and 5.
static bool gated_pays(const zn_ctx *ctx, int64_t m, int64_t n, int64_t k) {
    const double one = estimate_split(ctx, m, n, k, 1, 0).us;
    double two = 2e-6 * (double)m * n * k / 75.0;
    if (split_pays(ctx, ZN_LAYOUT_NN, m, n, k, 1)) two = std::min(two, estimate_split(ctx, m, n, k, 1, (int64_t)kScratchBytes).us);
    return one < two + 2.0 + 6.0 * (double)m * n / 4e6;
}

// A launch has fewer than 2^32 threads.
static bool launchable(int64_t workgroups, int64_t threads) { return workgroups <= (int64_t)UINT_MAX / threads; }

int zn_hip_gated_dense_forward(zn_ctx *ctx, int act, const float *x, const float *w, const float *bias, float *z,
                               float *h, int64_t batch, int64_t in_size, int64_t hidden) {
    if (!ctx || act < ZN_GATE_LINEAR || act > ZN_GATE_GELU || batch < 0 || in_size < 0 || hidden < 0)
        return ZN_ERR_INVALID_ARG;
    if (!gated_extents_ok(batch, in_size, hidden, false)) return ZN_ERR_OVERFLOW;
    if (batch == 0 || hidden == 0) return ZN_OK;
    if (!h || (in_size > 0 && (!x || !w))) return ZN_ERR_INVALID_ARG;
    int rc = select_device(ctx);
    if (rc) return rc;
    const int64_t n = 2 * hidden;
    ZnGatedArgs p;
    std::memset(&p, 0, sizeof(p));
    p.a = x;
    p.b = w;
    p.c = h;
    p.z = z;
    p.bias = bias;
    p.lda = in_size;
    p.ldb = n;
    p.ldc = hidden;
    p.m = (int32_t)batch;
    p.n = (int32_t)n;
    p.k = (int32_t)in_size;
    p.act = act;
    p.group_m = 1;
    p.splits = 1;
    p.batch = 1;
    p.k_chunk = (int32_t)in_size;
    // a forced split tile is the one launch's; any other forced choice takes the product and a pass
    const bool whole = in_size > 0 && ctx->forced_splits == 0 && ctx->forced_wave_split < 0 && ctx->forced_persistent < 0;
    const bool free = whole && ctx->forced_tile < 0, named = whole && ctx->forced_tile >= kTileSW && ctx->forced_tile <= kTileSN;
    const int64_t wgs = cdiv(hidden, 32);
    if (free && batch <= 16 && in_size * n >= kFewWeights && launchable(wgs, 1024)) {
        p.splits = (int32_t)std::max<int64_t>(1, std::min<int64_t>(cus_now(ctx) / wgs, in_size / 1024));
        Lease part(ctx);
        if (p.splits > 1) {
            if ((rc = part.get((size_t)(p.splits * batch * n)))) return rc;
            p.ws = part.ptr;
        }
        if ((rc = launch(ctx, ctx->gated_few, (unsigned)wgs, 1, 1024, &p, (unsigned)p.splits)) || p.splits == 1) return rc;
        return launch(ctx, ctx->gated_few_join, (unsigned)cdiv(hidden, 256), (unsigned)batch, 256, &p);
    }
    const Tile tile = named ? (Tile)ctx->forced_tile : estimate_split(ctx, batch, n, in_size, 1, 0).tile;
    const int64_t tiles = cdiv(batch, kTiles[tile].bm) * cdiv(hidden, kTiles[tile].bn / 2);
    if ((named || (free && gated_pays(ctx, batch, n, in_size))) && launchable(tiles, kTiles[tile].threads)) {
        p.tiles_m = (int32_t)cdiv(batch, kTiles[tile].bm);
        p.tiles_n = (int32_t)cdiv(hidden, kTiles[tile].bn / 2);
        p.xcd_remap = (tile == kTileSR || tile == kTileSN) && tiles % 8 == 0;  // as the plain product's
        return launch(ctx, ctx->gated[tile - kTileSW], (unsigned)tiles, 1, (unsigned)kTiles[tile].threads, &p);
    }
    Lease own(ctx);
    if (!z) {
        if ((rc = own.get((size_t)batch * (size_t)n))) return rc;
        z = own.ptr;
    }
    if ((rc = gemm_launch(ctx, ZN_LAYOUT_NN, batch, n, in_size, x, in_size, 0, w, n, 0, z, n, 0, 1, 0, bias, ZN_ACT_LINEAR)))
        return rc;
    ZnGateArgs g;
    std::memset(&g, 0, sizeof(g));
    g.z = z;
    g.h = h;
    g.rows = batch;
    g.n = hidden;
    g.act = act;
    return launch(ctx, ctx->elt[kGateForward], (unsigned)cdiv(hidden, 256), (unsigned)std::min<int64_t>(batch, 65535), 256, &g);
}

int zn_hip_gated_dense_backward(zn_ctx *ctx, int act, const float *x, const float *w, const float *z,
                                const float *grad_h, float *grad_z, float *grad_x, float *grad_w, float *grad_bias,
                                int64_t batch, int64_t in_size, int64_t hidden) {
    if (!ctx || act < ZN_GATE_LINEAR || act > ZN_GATE_GELU || batch < 0 || in_size < 0 || hidden < 0)
        return ZN_ERR_INVALID_ARG;
    if (!gated_extents_ok(batch, in_size, hidden, true)) return ZN_ERR_OVERFLOW;
    const int64_t n = 2 * hidden;
    if (batch > 0 && hidden > 0 && (!z || !grad_h || !grad_z)) return ZN_ERR_INVALID_ARG;
    if (in_size > 0 && hidden > 0 && (!grad_w || (batch > 0 && (!x || !w)))) return ZN_ERR_INVALID_ARG;
    int rc = select_device(ctx);
    if (rc) return rc;
    if (hidden == 0) return grad_x && batch > 0 && in_size > 0 ? zn_hip_fill_f32(ctx, grad_x, 0.0f, batch * in_size) : ZN_OK;
    if (batch == 0) return in_size > 0 ? zn_hip_fill_f32(ctx, grad_w, 0.0f, in_size * n) : ZN_OK;
    ZnGateArgs g;
    std::memset(&g, 0, sizeof(g));
    g.z = z;
    g.grad_h = grad_h;
    g.grad_z = grad_z;
    g.rows = batch;
    g.n = hidden;
    g.act = act;
    // row splits for about 8 workgroups a CU, at least 8 rows each
    const int64_t cus = cus_now(ctx), groups = cdiv(hidden, 256);
    int64_t splits = std::max<int64_t>(1, std::min<int64_t>({cdiv(batch, 8), 8 * cus / groups, 65535}));
    const int64_t per = cdiv(batch, splits);
    splits = cdiv(batch, per);
    g.rows_per_split = (int32_t)per;
    Lease part(ctx);
    ZnReduceArgs r;
    std::memset(&r, 0, sizeof(r));
    if (grad_bias) {
        if ((rc = part.get((size_t)(splits * n)))) return rc;
        g.partial = part.ptr;
        r.ws = part.ptr;
        r.c = grad_bias;
        r.m = 1;
        r.n = (int32_t)n;
        r.ldc = n;
        r.batch = 1;
        r.splits = (int32_t)splits;
        r.accumulate = 1;
        r.act = ZN_ACT_LINEAR;
        r.vec = n % 4 == 0 && aligned16(grad_bias) && aligned16(part.ptr) ? 1 : 0;
    }
    if ((rc = launch(ctx, ctx->elt[kGateBackward], (unsigned)groups, (unsigned)splits, 256, &g))) return rc;
    if (in_size == 0) return grad_bias ? launch_reduce(ctx, r) : ZN_OK;
    int64_t wg_nt = 0, wg_tn = 0;
    if (const int tile = grouped_tile(ctx, batch, in_size, n, grad_x != nullptr, &wg_nt, &wg_tn)) {
        ZnColSumArgs none;
        std::memset(&none, 0, sizeof(none));
        const int64_t blocks = grad_bias ? std::max<int64_t>(1, std::min<int64_t>(cdiv(n / (r.vec ? 4 : 1), 256), 8 * cus)) : 0;
        return dense_backward_grouped(ctx, x, w, grad_z, grad_x, grad_w, r, (int)blocks, none, batch, in_size, n, (int)wg_nt,
                                      (int)wg_tn, tile, ZN_ACT_LINEAR, nullptr, nullptr);
    }
    if (grad_bias && (rc = launch_reduce(ctx, r))) return rc;
    if (grad_x && (rc = gemm_launch(ctx, ZN_LAYOUT_NT, batch, in_size, n, grad_z, n, 0, w, n, 0, grad_x, in_size, 0, 1, 0,
                                    nullptr, ZN_ACT_LINEAR)))
        return rc;
    return gemm_launch(ctx, ZN_LAYOUT_TN, in_size, n, batch, x, in_size, 0, grad_z, n, 0, grad_w, n, 0, 1, 0, nullptr,
                       ZN_ACT_LINEAR);
}

// ---------------------------------------------------------- distillation
namespace {

constexpr int64_t kDistillMaxK = 1024;

int distill_args(zn_ctx *ctx, ZnDistillArgs &a, const float *logits, int64_t ld, const void *index, const float *top,
                 int64_t rows, int64_t vocab, int64_t k, float temperature) {
    if (!ctx || rows < 0 || vocab < 0 || k < 0 || k > kDistillMaxK || ld < vocab || !(temperature > 0.0f) ||
        !std::isfinite(temperature) || !std::isfinite(1.5f / temperature))
        return ZN_ERR_INVALID_ARG;
    if (vocab > INT_MAX / 2) return ZN_ERR_OVERFLOW;
    std::memset(&a, 0, sizeof(a));
    if (rows == 0) return ZN_OK;
    if (vocab > 0 && k > 0 && (!logits || !index || !top)) return ZN_ERR_INVALID_ARG;
    a.logits = logits;
    a.index = static_cast<const int32_t *>(index);
    a.top = top;
    a.ld = ld;
    a.rows = rows;
    a.vocab = (int32_t)vocab;
    a.k = vocab > 0 ? (int32_t)k : 0;
    a.temperature = temperature;
    a.inv_temperature = 1.0f / temperature;
    a.scale_log2 = 1.44269504088896340736f / temperature;
    // fewer rows than fill the chip twice over: parts of them, of at least 4096 values
    const int64_t parts = std::max<int64_t>(1, std::min<int64_t>({2 * cus_now(ctx) / rows, vocab / 4096, 64}));
    a.part_len = (int32_t)(cdiv(cdiv(vocab, parts), 4) * 4);
    a.parts = vocab > 0 ? (int32_t)cdiv(vocab, a.part_len) : 1;
    return ZN_OK;
}

// Workgroups that rows go over in turn.
unsigned distill_rows(const zn_ctx *ctx, int64_t rows) { return (unsigned)std::min<int64_t>(rows, 16 * cus_now(ctx)); }

}  // namespace

int zn_hip_distill_forward(zn_ctx *ctx, const float *logits, int64_t ld, const void *top_index,
                           const float *top_logits, float *loss, float *lse, int64_t rows, int64_t vocab, int64_t k,
                           float temperature) {
    ZnDistillArgs a;
    int rc = distill_args(ctx, a, logits, ld, top_index, top_logits, rows, vocab, k, temperature);
    if (rc || rows == 0) return rc;
    if (!loss || !lse) return ZN_ERR_INVALID_ARG;
    a.loss = loss;
    a.lse = lse;
    if ((rc = select_device(ctx))) return rc;
    Lease part(ctx);
    if (a.parts > 1) {
        if ((rc = part.get((size_t)(rows * a.parts) * 2))) return rc;
        a.part = part.ptr;
    }
    if ((rc = launch(ctx, ctx->elt[kDistillForward], distill_rows(ctx, rows), (unsigned)a.parts, 256, &a)) || a.parts == 1) return rc;
    return launch(ctx, ctx->elt[kDistillJoin], (unsigned)rows, 1, 256, &a);
}

int zn_hip_distill_backward(zn_ctx *ctx, const float *logits, int64_t ld, const void *top_index,
                            const float *top_logits, const float *lse, const float *grad_loss, float *grad_logits,
                            int64_t grad_ld, int64_t rows, int64_t vocab, int64_t k, float temperature) {
    ZnDistillArgs a;
    int rc = distill_args(ctx, a, logits, ld, top_index, top_logits, rows, vocab, k, temperature);
    if (rc) return rc;
    if (grad_ld < vocab) return ZN_ERR_INVALID_ARG;
    if (rows == 0 || vocab == 0) return ZN_OK;
    if (!grad_logits || (k > 0 && (!lse || !grad_loss))) return ZN_ERR_INVALID_ARG;
    a.lse = const_cast<float *>(lse);
    a.grad_loss = grad_loss;
    a.grad = grad_logits;
    a.grad_ld = grad_ld;
    if ((rc = select_device(ctx))) return rc;
    return launch(ctx, ctx->elt[kDistillBackward], distill_rows(ctx, rows), (unsigned)a.parts, 256, &a);
}

#endif
