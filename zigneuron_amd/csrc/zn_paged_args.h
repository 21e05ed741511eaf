// Kernel argument blocks of the rotary positions, the paged cache and the
// attention over it, as those of zn_kernel_args.h.
#ifndef ZN_PAGED_ARGS_H
#define ZN_PAGED_ARGS_H

#include <stdint.h>

// Rotary positions (kernels/rotary_f32.h): element strides {batch, head,
// position} of x and y; freq holds rot / 2 frequencies.  A workgroup takes
// `tokens` tokens, `slots` heads of each at a time, `units` threads a head;
// blockIdx.y: the first heads.
struct ZnRotaryArgs {
    const float *x, *freq;
    float *y;
    const int32_t *positions;     // position_stride apart a sequence, or null: 0, 1, ..
    int64_t xs[3], ys[3], position_stride;
    float scale, sign;            // sign: -1 turns back
    int32_t batch, heads, len, dim, rot, layout, units, slots, tokens;
};

// A paged cache and the new tokens of its sequences (kernels/zn_paged.h):
// k and v hold `pages` pages at element strides {page, head, position} with
// contiguous dims; table [batch x max_pages]; sequence b's new tokens are rows
// starts[b] .. starts[b + 1] - 1 and its last kv_lens[b] - cap at most - positions.
struct ZnPagedCache {
    char *k, *v;
    const int32_t *table, *kv_lens, *starts;
    int64_t stride[3];
    int32_t batch, pages, page_size, max_pages, kv_heads, dim, tokens, cap;
    uint32_t div_mul, div_shift;  // j / page_size, as ZnConvGeom's divisors
};

// zn_paged_append_*: strides {token, head}.  Workgroups as ZnRotaryArgs'; the
// heads are q's, then k's, then v's.
struct ZnAppendArgs {
    ZnPagedCache c;
    const float *k, *v, *q, *freq;
    float *q_out;
    const int32_t *positions;
    int64_t kvs[2], qs[2], os[2];
    float scale;
    int32_t q_heads, rot, layout, units, slots, per_wg;
};

// Attention over a paged cache (kernels/paged_f32.h): strides {token, head};
// lse is contiguous [tokens x q_heads], or null.
struct ZnPagedArgs {
    ZnPagedCache c;
    const float *q;
    float *out, *lse;
    int64_t qs[2], os[2];
    int32_t q_heads, group, causal, max_q;  // max_q: rows of a sequence past it are not written
    float scale_log2;             // scale * log2(e)
    // Sequences of at most `few` query rows of a key/value head (new tokens times group) go to the kernels for few rows, the others
    // in tiles of `tile` rows.  Either kind's positions are cut into parts, at most few_splits (equal ones) and tile_splits (of
    // tile_len), whose sums go to rows of part_ld floats: the dims, then the maximum and the sum.  few_part: part z of row y of sequence and
    // key/value head x < few_heads = batch kv_heads at (few x + y) few_splits + z; tile_part: of token t and head h at (t q_heads + h) tile_splits + z.
    // counters: an arrival counter for each x, zero between launches, where the few
    // rows' parts are joined in their own launch; or null.
    float *few_part, *tile_part;
    int32_t *counters;
    int32_t few, few_heads, few_splits, tile, tile_len, tile_splits, part_ld;
};

#endif
