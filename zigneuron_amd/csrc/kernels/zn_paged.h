// Sequences of a paged cache, shared by the kernels that fill it and that
// read it.
//
// Everything that the device arrays say is held to what the host knows: starts
// to [0, tokens], lengths to [0, cap], page numbers to [0, pages).  Nothing in
// them leads outside the tensors.  (The parts without a wave also compile as
// plain C++, for the tests.)
#ifndef ZN_PAGED_H
#define ZN_PAGED_H

#include <stdint.h>

#include "../zn_paged_args.h"

#ifdef __HIPCC__
#include <hip/hip_runtime.h>
#define ZN_PAGED_FN __device__ __forceinline__
#else
#define ZN_PAGED_FN inline
#endif

namespace {

ZN_PAGED_FN int paged_clamp(int x, int lo, int hi) { return x < lo ? lo : x > hi ? hi : x; }

// One sequence's new tokens and length; its token i has position first + i.
struct PagedSeq {
    int t0, ql, kl, first;
    ZN_PAGED_FN explicit PagedSeq(const ZnPagedCache &) : t0(0), ql(0), kl(0), first(0) {}  // none
    ZN_PAGED_FN PagedSeq(const ZnPagedCache &c, int b) {
        t0 = paged_clamp(c.starts[b], 0, c.tokens);
        ql = paged_clamp(c.starts[b + 1], t0, c.tokens) - t0;
        kl = paged_clamp(c.kv_lens[b], 0, c.cap);
        first = kl - ql;
    }
};

// Where position j (0 <= j < cap) of sequence b lies, head kh, in elements of k and of v; -1 where its page is none of the cache's.
ZN_PAGED_FN int64_t paged_at(const ZnPagedCache &c, int b, int kh, int j) {
    const int n = (int)(((uint64_t)(uint32_t)j * c.div_mul) >> (31 + c.div_shift));
    const int page = c.table[(int64_t)b * c.max_pages + n];
    if ((uint32_t)page >= (uint32_t)c.pages) return -1;
    return page * c.stride[0] + kh * c.stride[1] + (j - n * c.page_size) * c.stride[2];
}

#ifdef __HIPCC__
// The largest b <= batch with starts[b] <= t, or -1; t is the same in the whole wave.  64 of the starts at a time.
__device__ __forceinline__ int paged_find(const ZnPagedCache &c, int t) {
    const int lane = threadIdx.x & 63;
    int n = 0;
    for (int i0 = 0; i0 <= c.batch; i0 += 64) {
        const uint64_t at = __builtin_amdgcn_ballot_w64(c.starts[min(i0 + lane, c.batch)] <= t && i0 + lane <= c.batch);
        n += __builtin_popcountll(at);
        if (~at) break;
    }
    return n - 1;
}
#endif

}  // namespace

#endif
