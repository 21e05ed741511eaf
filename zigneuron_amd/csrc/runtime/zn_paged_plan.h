// How a call of the attention over a paged cache is cut up: which kernel takes
// it, in how many parts and workgroups.  A rule on what the host knows (sizes and
// bounds), plain C++.
#ifndef ZN_PAGED_PLAN_H
#define ZN_PAGED_PLAN_H

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "../../../include/zn_hip.h"
#include "../zn_paged_args.h"

namespace {

// The kernels, in the attention code object: zn_paged_<what>_<cache type>_<padded head dim>.
enum PagedKernel { kPagedFew, kPagedFew2, kPagedFew4, kPagedTile, kPagedWide, kNumPaged };
constexpr const char *kPagedName[kNumPaged] = {"zn_paged_few", "zn_paged_few2", "zn_paged_few4", "zn_paged_tile", "zn_paged_wide"};
constexpr int kPagedRows[kNumPaged] = {16, 32, 64, 128, 256};  // query rows of a workgroup
constexpr const char *kCacheName[2] = {"f32", "bf16"};
// Threads of a tile's workgroup [kPagedTile, kPagedWide][cache type][dims in 32s]; the others have 256.  0: there is none.
constexpr unsigned kPagedThreads[2][2][4] = {{{256, 256, 512, 512}, {256, 256, 256, 256}}, {{512, 512, 512, 512}, {0, 0, 0, 0}}};
constexpr int64_t kPagedSplitHeads = 4096;  // sequences' heads of few rows whose walks are cut into parts

inline int64_t paged_ceil(int64_t a, int64_t b) { return (a + b - 1) / b; }

// How many parts the walk of few query rows is cut into: two workgroups a CU of sequences that are as long as the call allows, of 512 KB
// of K and V at most (sequences differ in length), 128 positions at least (paged_few_len).  MI355X, us in parts of 256, 512, 1024, 2048
// and 4096 positions: 64 x 8 heads of up to 8192 x 128 bf16 311, 285, 275, 279, 291; 16 x 4 of up to 4096 x 128 bf16, five tokens, 41,
// 31, 32, 47, 73; 16 x 8 of 4096 x 128 fp32 112, 108, 108, 107, 126; 8 of 65536 x 128 bf16 64, 54, 49, 47, 52; 8 x 4 of 2048 x 64
// fp32 12, 16, 24, 37.  Beside tiles one of their larger workgroups a CU; never
// more than 32 a CU, which bounds the parts' memory.  Past 4096 heads there is enough to do without.
inline void paged_few_parts(ZnPagedArgs &a, int type, int64_t cus, int per_cu) {
    const int64_t most = 524288 / (2 * a.c.dim * (type == ZN_CACHE_BF16 ? 2 : 4));
    const int64_t all = (int64_t)a.c.cap * a.few_heads;
    const int64_t len = std::max({(int64_t)128, std::min(most, all / (per_cu * cus)), all / (32 * cus)});
    a.few_splits = a.few_heads > kPagedSplitHeads ? 1 : (int32_t)std::max<int64_t>(1, std::min<int64_t>(65535, paged_ceil(a.c.cap, len)));
}

// Parts of the walks of tiles: the least of the times of two batches added up, one whose sequences are all as long as the call allows, one
// where one is and the others make it three quarters of that together.  A workgroup's way in and out is 10 us; times of a block of 32
// keys as measured (dims 64, 96, 128; us): fp32 256 rows 2.3, 3.4, 4.0, 128 rows 2.0 alone and 3.0 where two share a CU, then 2.1, 2.5;
// bf16 (128 dims) 2.5 and 2.6.  Without the second batch 4 x 512 tokens of 32 (8) x 128 over 2730 to 8192 positions stay whole: 1015
// us, 550 in two parts; without the first 4 x 512 of 16 (4) x 64 over 4096 take three: 234, 186 in two.  Returns the time so found.
inline double paged_tile_parts(ZnPagedArgs &a, int kernel, int type, int64_t cus_) {
    const int64_t tokens = a.c.tokens, max_q = a.max_q;
    constexpr int kParts[12] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64};
    constexpr double kWay = 10.0;
    const int rows = kPagedRows[kernel];
    const bool pairs = kPagedThreads[kernel - kPagedTile][type][(a.c.dim - 1) / 32] == 256;  // two workgroups share a CU
    const double cus = (double)cus_ / (a.few ? 2.0 : 1.0), slots = cus * (pairs ? 2 : 1), tiles = (double)(paged_ceil(tokens * a.group, rows) * a.c.kv_heads);
    const double wide = (0.6 + 0.0264 * a.c.dim) * (type == ZN_CACHE_BF16 ? 0.65 : 1.0), tile = type == ZN_CACHE_BF16 ? 1.0 : pairs ? 1.2 : 0.64;
    const double full = kernel == kPagedWide ? wide : wide * tile, alone = pairs ? 0.75 * full : full;
    const double share = a.causal && a.c.cap > 0 ? 1.0 - 0.5 * std::min(1.0, (double)max_q / (double)a.c.cap) : 1.0;  // of a walk, on average
    const int64_t blocks = paged_ceil(a.c.cap, 32);
    double best = INFINITY;
    a.tile_splits = 1;
    for (const int s : kParts) {
        if (s > 1 && s > blocks) break;
        const double n = tiles * s, len = (double)paged_ceil(blocks, s), longest = kWay + alone * len, all = n * (kWay + full * len * share) / slots;
        const double join = s > 1 ? 6.0 + 8.0 * (double)tokens * a.q_heads * s * a.c.dim / 2e6 : 0.0;
        const double even = n <= cus ? longest : share < 0.9 ? std::max(longest, all) : std::ceil(n / slots) * (kWay + full * len);
        const double us = even + join + std::max(longest, 0.75 * all) + 0.75 * join;
        if (us < best) {
            best = us;
            a.tile_splits = s;
        }
    }
    a.tile = rows;
    a.tile_len = (int32_t)(32 * std::max<int64_t>(1, paged_ceil(blocks, a.tile_splits)));
    a.tile_splits = (int32_t)std::max<int64_t>(1, paged_ceil(a.c.cap, a.tile_len));
    return best;
}

struct PagedPlan {
    int kernel = kPagedFew;
    bool all_few = true, own_join = false;  // own_join: the last workgroup to arrive joins a walk's parts
    int64_t wgs = 0;                        // tiles: workgroups of the launch, all kinds
    unsigned threads = 256;
    bool fits() const { return wgs <= (int64_t)(UINT32_MAX / threads); }  // a launch has fewer than 2^32 threads
};

// The kernel and its workgroups, and a's few, few_heads, few_splits, tile, tile_len and tile_splits; the rest of a is given.
inline PagedPlan paged_plan(ZnPagedArgs &a, int type, int64_t cus) {
    PagedPlan p;
    const int dims = (a.c.dim - 1) / 32;
    const int64_t group = a.group, tokens = a.c.tokens, batch = a.c.batch;
    a.few_heads = (int32_t)(batch * a.c.kv_heads);
    // Sequences of few query rows have kernels of their own; where others are in the call too, their workgroups follow the tiles'
    // in one launch.
    const int64_t rows = group * a.max_q;
    // 33 to 64 rows: in tiles where there are few heads, whose walks a workgroup then reads too slowly (MI355X, us as few rows and in
    // tiles of 128: 16 tokens of 16 x 8 heads (4) against 4096 x 128 bf16 107 and 131, of 4 x 8 against 2048 39 and 32; fp32 of 33 x 9
    // heads (1) of 42 tokens against up to 2713 x 127 260 and 367, 16 tokens of 16 x 8 (4) against 2048 x 128 112 and 103, of 16 x 4
    // against 4096 x 64 66 and 98).
    const int64_t enough = type == ZN_CACHE_BF16 || a.c.dim <= 64 ? cus / 4 : cus;
    p.all_few = rows <= kPagedRows[a.few_heads >= enough ? kPagedFew4 : kPagedFew2];
    a.few = 0;
    if (p.all_few) {
        while (kPagedRows[p.kernel] < rows) ++p.kernel;
        a.few = (int32_t)rows;
    } else if (group <= kPagedRows[kPagedFew] && tokens < batch * a.max_q) {
        a.few = kPagedRows[kPagedFew];
    }
    if (a.few) paged_few_parts(a, type, cus, p.all_few ? 2 : 1);
    p.own_join = p.all_few && rows <= 8;  // two rows a wave at most
    if (p.all_few) return p;
    ZnPagedArgs wide = a;
    p.kernel = kPagedTile;
    const double us = paged_tile_parts(a, kPagedTile, type, cus);
    if (type == ZN_CACHE_F32 && paged_tile_parts(wide, kPagedWide, type, cus) < us) {
        p.kernel = kPagedWide;
        a = wide;
    }
    // Each sequence in tiles has an unfilled one at most; with more than `few` rows, a whole token's at least, there are only so many.
    // (Counting every sequence: 2048 of 8 heads (2) of one token, one of 300, against 256 x 64 fp32 356 us, 275 so.)
    const int64_t tiled = std::min(batch, tokens * group / std::max<int64_t>(a.few + 1, group));
    p.wgs = (tokens * group / a.tile + tiled) * a.c.kv_heads * a.tile_splits + (a.few ? (int64_t)a.few_heads * a.few_splits : 0);
    p.threads = kPagedThreads[p.kernel - kPagedTile][type][dims];
    return p;
}

}  // namespace

#endif
