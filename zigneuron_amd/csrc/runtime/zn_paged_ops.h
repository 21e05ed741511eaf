// Serving a language model's attention (include/zn_hip.h): rotary positions,
// the paged cache and the attention over it.  Included by zn_hip.cpp behind
// zn_block_ops.h, whose helpers it uses too.
#ifndef ZN_PAGED_OPS_H
#define ZN_PAGED_OPS_H

// -------------------------------------------------------- rotary positions
namespace {

constexpr int64_t kRotaryMaxDim = 1024;  // at most 128 threads to a head

// Threads of a workgroup to tokens, heads and shares of a head.  Where a token's heads lie together (together): as many heads of a token
// at a time as fit, tokens where room is left; where a head's tokens do: neighbouring tokens, one head after the other.
struct RotaryGrid {
    int32_t units, slots, tokens;
    unsigned gx, gy;
    RotaryGrid(const zn_ctx *ctx, int64_t units_, int64_t heads, int64_t all, bool together) {
        units = (int32_t)units_;
        slots = together ? (int32_t)std::min<int64_t>(heads, 256 / units) : 1;
        // Where that leaves many threads without work: the most heads that do not (6654 tokens of 20 heads of 10 shares: 200 threads of
        // 256, or 5 heads of 5 tokens four times; 24 and 18.6 us).
        auto busy = [&](int64_t s) { return (double)heads / (double)cdiv(heads, s) * (double)(256 / (s * units)) * (double)units / 256.0; };
        const int64_t fit = slots;
        for (int64_t s = fit; s > 0 && busy(fit) < 0.85; --s)
            if (busy(s) > busy(slots)) slots = (int32_t)s;
        tokens = (int32_t)std::max<int64_t>(1, std::min<int64_t>(all, 256 / (slots * units)));
        gx = (unsigned)cdiv(all, tokens);
        // few tokens: heads beside each other instead of one after the other
        gy = (unsigned)std::max<int64_t>(1, std::min<int64_t>(cdiv(heads, slots), 4 * cus_now(ctx) / gx));
    }
};

int64_t rotary_units(int64_t dim, int64_t rot, bool rest) { return cdiv(rot / 2, 4) + (rest ? cdiv(dim - rot, 8) : 0); }

bool rotary_ok(int64_t dim, int64_t rot, int layout, float scale, const void *freq) {
    return rot >= 0 && rot <= dim && rot % 2 == 0 && layout >= ZN_ROTARY_HALF && layout <= ZN_ROTARY_INTERLEAVED && std::isfinite(scale) &&
           (rot == 0 || freq);
}

// Element strides of an extent, the largest of which a tensor in memory can have.
constexpr int64_t kMaxStride = (int64_t)1 << 46;
bool stride_ok(int64_t stride, int64_t extent, bool written) { return stride >= 0 && (stride > 0 || extent <= 1 || !written); }
bool stride_far(int64_t stride, int64_t extent) { return extent > 1 && stride > kMaxStride / (extent - 1); }

int rotary(zn_ctx *ctx, const float *x, float *y, const float *freq, const void *positions, int64_t batch, int64_t heads, int64_t len,
           int64_t dim, int64_t rot, int layout, float scale, float sign, int64_t position_stride, const int64_t (&xs)[3],
           const int64_t (&ys)[3]) {
    if (!ctx || batch < 0 || heads < 0 || len < 0 || dim < 1 || dim > kRotaryMaxDim || !rotary_ok(dim, rot, layout, scale, freq) ||
        position_stride < 0)
        return ZN_ERR_INVALID_ARG;
    const int64_t extent[3] = {batch, heads, len};
    const bool work = batch > 0 && heads > 0 && len > 0;
    for (int i = 0; i < 3; ++i)
        if (!stride_ok(xs[i], extent[i], false) || !stride_ok(ys[i], extent[i], work)) return ZN_ERR_INVALID_ARG;
    for (int i = 0; i < 3; ++i)
        if (extent[i] > INT_MAX / 2 || stride_far(xs[i], extent[i]) || stride_far(ys[i], extent[i])) return ZN_ERR_OVERFLOW;
    if (batch * len > (1 << 24) - 1 || stride_far(position_stride, batch)) return ZN_ERR_OVERFLOW;  // tokens: a launch has fewer than 2^32 threads
    if (!work) return ZN_OK;
    if (!x || !y) return ZN_ERR_INVALID_ARG;
    int rc = select_device(ctx);
    if (rc) return rc;
    const bool same = x == y && std::memcmp(xs, ys, sizeof(xs)) == 0;  // what is not turned is there already
    ZnRotaryArgs a;
    std::memset(&a, 0, sizeof(a));
    const int64_t units = rotary_units(dim, rot, !same);
    if (units == 0) return ZN_OK;
    const RotaryGrid g(ctx, units, heads, batch * len, xs[1] <= xs[2] || len == 1);
    a.x = x;
    a.y = y;
    a.freq = freq;
    a.positions = static_cast<const int32_t *>(positions);
    std::memcpy(a.xs, xs, sizeof(a.xs));
    std::memcpy(a.ys, ys, sizeof(a.ys));
    a.position_stride = position_stride;
    a.scale = scale;
    a.sign = sign;
    a.batch = (int32_t)batch;
    a.heads = (int32_t)heads;
    a.len = (int32_t)len;
    a.dim = (int32_t)dim;
    a.rot = (int32_t)rot;
    a.layout = layout;
    a.units = g.units;
    a.slots = g.slots;
    a.tokens = g.tokens;
    return launch(ctx, ctx->elt[kRotary], g.gx, g.gy, 256, &a);
}

}  // namespace

int zn_hip_rotary_frequencies(float *freq, size_t freq_len, int64_t rot_dim, float base, int scaling, float factor,
                              int64_t trained_len, float low, float high) {
    if (!freq || rot_dim < 2 || rot_dim % 2 || rot_dim > kRotaryMaxDim || freq_len < (size_t)rot_dim / 2 || !(base > 0.0f) ||
        !std::isfinite(base) || scaling < ZN_ROTARY_PLAIN || scaling > ZN_ROTARY_PAIRS)
        return ZN_ERR_INVALID_ARG;
    if (scaling != ZN_ROTARY_PLAIN && (!(factor > 0.0f) || !std::isfinite(factor))) return ZN_ERR_INVALID_ARG;
    const bool parts = scaling == ZN_ROTARY_TURNS || scaling == ZN_ROTARY_PAIRS;
    if (parts && (trained_len < 1 || !(low > 0.0f) || !(high > low) || !std::isfinite(high) || (scaling == ZN_ROTARY_PAIRS && !(base > 1.0f))))
        return ZN_ERR_INVALID_ARG;
    if (scaling == ZN_ROTARY_BASE && rot_dim < 4) return ZN_ERR_INVALID_ARG;
    const double n = (double)rot_dim, circle = 6.283185307179586;
    double b = base;
    if (scaling == ZN_ROTARY_BASE) b *= std::pow((double)factor, n / (n - 2.0));
    // the pair that makes `turns` turns over trained_len
    auto pair_of = [&](double turns) { return n * std::log((double)trained_len / (turns * circle)) / (2.0 * std::log(b)); };
    double first = 0.0, last = 0.0;
    if (scaling == ZN_ROTARY_PAIRS) {
        first = std::max(0.0, std::floor(pair_of(high)));
        // not the last pair, n / 2 - 1: past it lies the ramp's end wherever that pair makes more than `low` turns
        last = std::min(n - 1.0, std::ceil(pair_of(low)));
    }
    for (int64_t i = 0; i < rot_dim / 2; ++i) {
        const double f = std::pow(b, -2.0 * (double)i / n);
        double keep = 1.0;  // the share that keeps its speed; the rest is slowed down by factor
        if (scaling == ZN_ROTARY_LINEAR) keep = 0.0;
        else if (scaling == ZN_ROTARY_TURNS) keep = ((double)trained_len * f / circle - low) / ((double)high - low);
        else if (scaling == ZN_ROTARY_PAIRS)  // where even the first pair turns less, last <= first
            keep = (double)i >= last ? 0.0 : (double)i <= first ? 1.0 : 1.0 - ((double)i - first) / (last - first);
        keep = std::min(1.0, std::max(0.0, keep));
        freq[i] = (float)(scaling == ZN_ROTARY_PLAIN || scaling == ZN_ROTARY_BASE ? f : keep * f + (1.0 - keep) * f / factor);
    }
    return ZN_OK;
}

int zn_hip_rotary_forward(zn_ctx *ctx, const float *x, float *y, const float *freq, const void *positions, int64_t batch,
                          int64_t heads, int64_t len, int64_t head_dim, int64_t rot_dim, int layout, float scale,
                          int64_t position_stride, int64_t x_stride_b, int64_t x_stride_h, int64_t x_stride_s,
                          int64_t y_stride_b, int64_t y_stride_h, int64_t y_stride_s) {
    return rotary(ctx, x, y, freq, positions, batch, heads, len, head_dim, rot_dim, layout, scale, 1.0f, position_stride,
                  {x_stride_b, x_stride_h, x_stride_s}, {y_stride_b, y_stride_h, y_stride_s});
}

int zn_hip_rotary_backward(zn_ctx *ctx, const float *grad_y, float *grad_x, const float *freq, const void *positions,
                           int64_t batch, int64_t heads, int64_t len, int64_t head_dim, int64_t rot_dim, int layout,
                           float scale, int64_t position_stride, int64_t y_stride_b, int64_t y_stride_h,
                           int64_t y_stride_s, int64_t x_stride_b, int64_t x_stride_h, int64_t x_stride_s) {
    return rotary(ctx, grad_y, grad_x, freq, positions, batch, heads, len, head_dim, rot_dim, layout, scale, -1.0f, position_stride,
                  {y_stride_b, y_stride_h, y_stride_s}, {x_stride_b, x_stride_h, x_stride_s});
}

// --------------------------------------------------------- the paged cache
namespace {

// The checks that both calls share.  Refusals come before anything is read but the descriptor itself.
int paged_args(const zn_paged_cache *c, ZnPagedCache &a, const void *starts, int64_t tokens, bool written) {
    if (!c || tokens < 0 || c->batch < 0 || c->num_pages < 0 || c->page_size < 1 || c->max_pages < 0 || c->kv_heads < 0 ||
        c->head_dim < 1 || c->head_dim > kMhaMaxDim || c->type < ZN_CACHE_F32 || c->type > ZN_CACHE_BF16)
        return ZN_ERR_INVALID_ARG;
    const int64_t stride[3] = {c->stride_page, c->stride_head, c->stride_position};
    const int64_t extent[3] = {c->num_pages, c->kv_heads, c->page_size};
    for (int i = 0; i < 3; ++i)
        if (!stride_ok(stride[i], extent[i], written)) return ZN_ERR_INVALID_ARG;
    if (c->stride_position < c->head_dim) return ZN_ERR_INVALID_ARG;
    constexpr int64_t kMax = INT_MAX / 2;
    if (tokens > (1 << 24) - 1 || c->batch > kMax || c->num_pages > kMax || c->page_size > kMax || c->max_pages > kMax ||
        c->kv_heads > kMax || c->max_pages * c->page_size > kMax)
        return ZN_ERR_OVERFLOW;
    for (int i = 0; i < 3; ++i)
        if (stride_far(stride[i], extent[i])) return ZN_ERR_OVERFLOW;
    if (c->stride_position > INT_MAX) return ZN_ERR_OVERFLOW;
    std::memset(&a, 0, sizeof(a));
    a.k = static_cast<char *>(c->k);
    a.v = static_cast<char *>(c->v);
    a.table = static_cast<const int32_t *>(c->page_table);
    a.kv_lens = static_cast<const int32_t *>(c->kv_lens);
    a.starts = static_cast<const int32_t *>(starts);
    std::memcpy(a.stride, stride, sizeof(a.stride));
    a.batch = (int32_t)c->batch;
    a.pages = (int32_t)c->num_pages;
    a.page_size = (int32_t)c->page_size;
    a.max_pages = (int32_t)c->max_pages;
    a.kv_heads = (int32_t)c->kv_heads;
    a.dim = (int32_t)c->head_dim;
    a.tokens = (int32_t)tokens;
    a.cap = (int32_t)(c->num_pages ? c->max_pages * c->page_size : 0);
    udiv_magic((uint32_t)c->page_size, a.div_mul, a.div_shift);
    return ZN_OK;
}

// What a call with something to do reads of the descriptor.
bool paged_pointers(const ZnPagedCache &a) { return a.kv_lens && a.starts && (a.cap == 0 || (a.k && a.v && a.table)); }

}  // namespace

int zn_hip_paged_append(zn_ctx *ctx, const void *cache, const void *token_starts, int64_t tokens, const float *k,
                        const float *v, int64_t kv_stride_t, int64_t kv_stride_h, const float *q, float *q_out,
                        int64_t q_heads, int64_t q_stride_t, int64_t q_stride_h, int64_t q_out_stride_t,
                        int64_t q_out_stride_h, const float *freq, int64_t rot_dim, int layout, float scale,
                        const void *positions) {
    if (!ctx) return ZN_ERR_INVALID_ARG;
    const zn_paged_cache *desc = static_cast<const zn_paged_cache *>(cache);
    ZnAppendArgs a;
    std::memset(&a, 0, sizeof(a));
    int rc = paged_args(desc, a.c, token_starts, tokens, true);
    if (rc == ZN_ERR_INVALID_ARG) return rc;
    if (q_heads < 0 || !rotary_ok(desc->head_dim, rot_dim, layout, scale, freq)) return ZN_ERR_INVALID_ARG;
    if (!q) q_heads = 0;
    if (!stride_ok(kv_stride_t, tokens, false) || !stride_ok(kv_stride_h, desc->kv_heads, false)) return ZN_ERR_INVALID_ARG;
    if (q_heads > 0 && (!stride_ok(q_stride_t, tokens, false) || !stride_ok(q_stride_h, q_heads, false) ||
                        !stride_ok(q_out_stride_t, tokens, true) || !stride_ok(q_out_stride_h, q_heads, true)))
        return ZN_ERR_INVALID_ARG;
    if (rc) return rc;
    if (q_heads > INT_MAX / 4) return ZN_ERR_OVERFLOW;
    const int64_t heads = q_heads + 2 * desc->kv_heads;
    if (heads > INT_MAX / 2 || stride_far(kv_stride_t, tokens) || stride_far(kv_stride_h, desc->kv_heads) ||
        (q_heads > 0 && (stride_far(q_stride_t, tokens) || stride_far(q_stride_h, q_heads) || stride_far(q_out_stride_t, tokens) ||
                         stride_far(q_out_stride_h, q_heads))))
        return ZN_ERR_OVERFLOW;
    if (tokens == 0 || desc->batch == 0 || heads == 0) return ZN_OK;
    if (!paged_pointers(a.c) || (desc->kv_heads > 0 && (!k || !v)) || (q_heads > 0 && !q_out)) return ZN_ERR_INVALID_ARG;
    if ((rc = select_device(ctx))) return rc;
    const RotaryGrid g(ctx, rotary_units(desc->head_dim, rot_dim, true), heads, tokens, true);
    a.k = k;
    a.v = v;
    a.q = q;
    a.q_out = q_out;
    a.freq = freq;
    a.positions = static_cast<const int32_t *>(positions);
    a.kvs[0] = kv_stride_t;
    a.kvs[1] = kv_stride_h;
    a.qs[0] = q_stride_t;
    a.qs[1] = q_stride_h;
    a.os[0] = q_out_stride_t;
    a.os[1] = q_out_stride_h;
    a.scale = scale;
    a.q_heads = (int32_t)q_heads;
    a.rot = (int32_t)rot_dim;
    a.layout = layout;
    a.units = g.units;
    a.slots = g.slots;
    a.per_wg = g.tokens;
    return launch(ctx, ctx->elt[desc->type == ZN_CACHE_BF16 ? kPagedAppendBf16 : kPagedAppendF32], g.gx, g.gy, 256, &a);
}

int zn_hip_paged_attention(zn_ctx *ctx, const void *cache, const void *token_starts, int64_t tokens, int64_t max_q_len,
                           int64_t max_kv_len, const float *q, float *out, float *lse, int64_t q_heads, float scale,
                           int causal, int64_t q_stride_t, int64_t q_stride_h, int64_t out_stride_t,
                           int64_t out_stride_h) {
    if (!ctx) return ZN_ERR_INVALID_ARG;
    const zn_paged_cache *desc = static_cast<const zn_paged_cache *>(cache);
    ZnPagedArgs a;
    std::memset(&a, 0, sizeof(a));
    int rc = paged_args(desc, a.c, token_starts, tokens, false);
    if (rc == ZN_ERR_INVALID_ARG) return rc;
    if (q_heads < 0 || max_q_len < 0 || max_kv_len < 0 || causal < 0 || causal > 1 || !std::isfinite(scale)) return ZN_ERR_INVALID_ARG;
    if (desc->kv_heads == 0 ? q_heads != 0 : q_heads % desc->kv_heads != 0) return ZN_ERR_INVALID_ARG;
    if (!stride_ok(q_stride_t, tokens, false) || !stride_ok(q_stride_h, q_heads, false) || !stride_ok(out_stride_t, tokens, true) ||
        !stride_ok(out_stride_h, q_heads, true))
        return ZN_ERR_INVALID_ARG;
    if (rc) return rc;
    if (q_heads > 65535 || tokens * q_heads > INT_MAX / 2 || stride_far(q_stride_t, tokens) || stride_far(q_stride_h, q_heads) ||
        stride_far(out_stride_t, tokens) || stride_far(out_stride_h, q_heads) || desc->batch * desc->kv_heads > (int64_t)1 << 22)
        return ZN_ERR_OVERFLOW;
    if (tokens == 0 || desc->batch == 0 || q_heads == 0 || max_q_len == 0) return ZN_OK;
    if (!q || !out || !paged_pointers(a.c)) return ZN_ERR_INVALID_ARG;
    max_q_len = std::min(max_q_len, tokens);
    const int dims = (int)(desc->head_dim - 1) / 32, type = desc->type;
    const int64_t cap = std::min<int64_t>(a.c.cap, max_kv_len);
    if ((rc = select_device(ctx))) return rc;
    a.c.cap = (int32_t)cap;
    a.q = q;
    a.out = out;
    a.lse = lse;
    a.qs[0] = q_stride_t;
    a.qs[1] = q_stride_h;
    a.os[0] = out_stride_t;
    a.os[1] = out_stride_h;
    a.q_heads = (int32_t)q_heads;
    a.group = (int32_t)(q_heads / desc->kv_heads);
    a.causal = causal;
    a.max_q = (int32_t)max_q_len;
    a.scale_log2 = scale * 1.44269504088896340736f;
    // a 16-byte load of bf16 takes 8 dims
    if (desc->head_dim < 8) return launch(ctx, ctx->paged_rows[type], (unsigned)tokens, (unsigned)cdiv(q_heads, 4), 256, &a);
    const int pages = desc->page_size % 16 == 0;
    a.part_ld = (int32_t)(desc->head_dim + 3) / 4 * 4 + 4;
    const PagedPlan plan = paged_plan(a, type, cus_now(ctx));
    if (!plan.fits()) return ZN_ERR_OVERFLOW;
    Lease few_part(ctx), tile_part(ctx);
    if (a.few && a.few_splits > 1) {
        if ((rc = few_part.get((size_t)a.few_heads * a.few * a.few_splits * a.part_ld))) return rc;
        a.few_part = few_part.ptr;
    }
    if (!plan.all_few && a.tile_splits > 1) {
        if ((rc = tile_part.get((size_t)(tokens * q_heads) * a.tile_splits * a.part_ld))) return rc;
        a.tile_part = tile_part.ptr;
    }
    static_assert(kPagedSplitHeads <= kCounterSlots, "a counter for each walk in parts");
    if (plan.own_join && a.few_splits > 1) a.counters = ctx->counters;
    const hipFunction_t f = ctx->paged[plan.kernel][type][dims][pages];
    if (plan.all_few) rc = launch(ctx, f, (unsigned)a.few_heads, 1, 256, &a, (unsigned)a.few_splits);
    else rc = launch(ctx, f, (unsigned)plan.wgs, 1, plan.threads, &a);
    if (rc || plan.own_join || (a.few_splits <= 1 && a.tile_splits <= 1)) return rc;
    // a token's heads beside each other while there are few tokens, eight workgroups a CU (4 x 512 tokens of 32 heads, a quarter of
    // them in parts: 25 us with eight workgroups a token, 15 with one)
    const int64_t join_heads = std::max<int64_t>(1, std::min<int64_t>(cdiv(q_heads, 4), 8 * cus_now(ctx) / tokens));
    return launch(ctx, ctx->paged_join, (unsigned)tokens, (unsigned)join_heads, 256, &a);
}

#endif
