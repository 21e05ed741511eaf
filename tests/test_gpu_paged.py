"""The paged cache on the GPU (zn_hip_paged_append, zn_hip_paged_attention) against 64 bits."""
from __future__ import annotations

import numpy as np
import pytest

from block_ops_ref import Mha, check
from gpu_common import announce
from paged_ref import Ints, Pool, Strided, frequencies, from_bf16, rotary, starts_of, to_bf16

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    from zigneuron_amd import Context
    c = Context(0)
    yield c
    c.close()


def rows(n, h, d, order="thd"):
    """(token, head) strides."""
    return {"thd": (h * d, d), "htd": (d, n * d), "gaps": (h * (d + 5) + 3, d + 5)}[order]


# ------------------------------------------------------------------ append
def run_append(ctx, pool, counts, hq, rot, layout="half", scale=1.0, positions=None, pad=0, order="thd", seed=1, in_place=False, q=True):
    """One call; checks caches and queries against the reference."""
    rng = np.random.default_rng(seed)
    n, hk, d = int(sum(counts)) + pad, pool.kv_heads, pool.dim
    f32 = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    xk, xv, xq = f32(n, hk, d), f32(n, hk, d), f32(n, hq, d)
    cache = pool.place(ctx)
    dk, dv = (Strided(ctx, t, rows(n, hk, d, order)) for t in (xk, xv))
    dq = Strided(ctx, xq, rows(n, hq, d, order))
    dout = dq if in_place else Strided(ctx, np.full(xq.shape, 5.0, np.float32), rows(n, hq, d, "gaps"))
    starts = starts_of(counts)
    freq = frequencies(rot)
    dp = None if positions is None else Ints(ctx, positions)
    ctx.paged_append(cache, Ints(ctx, starts).buf, n, dk.ptr, dv.ptr, dk.strides, dq.ptr if q else None, dout.ptr if q else None, hq,
                     dq.strides, dout.strides, ctx.to_device(freq) if rot else None, rot, layout, scale, None if dp is None else dp.ptr)
    at = np.concatenate([pool.lens[b] - c + np.arange(c) for b, c in enumerate(counts)] + [np.zeros(pad)]).astype(np.int64)
    turn = at if positions is None else np.asarray(positions, np.int64)
    rk, bk = rotary(xk, turn[:, None], freq, rot, layout, scale)
    rq, bq = rotary(xq, turn[:, None], freq, rot, layout, scale)
    want = [pool.k.astype(np.float64), pool.v.astype(np.float64)]
    bound = [np.zeros(pool.k.shape), np.zeros(pool.k.shape)]
    t = 0
    for b, c in enumerate(counts):
        for i in range(c):
            j = pool.lens[b] - c + i
            if j >= 0:
                page = pool.table[b, j // pool.page]
                if 0 <= page < pool.pages:
                    s = (page, slice(None), j % pool.page)
                    want[0][s], bound[0][s] = rk[t], bk[t]
                    want[1][s] = xv[t]
            t += 1
    got = pool.read()
    for name, x, w, e in zip("kv", got, want, bound):
        hole = np.isnan(w)
        assert np.array_equal(np.isnan(x), hole), f"{name}: other slots written"
        if pool.dtype == "bf16":
            new = e > 0 if name == "k" else None
            if name == "v":  # copied: rounded exactly once
                assert np.array_equal(to_bf16(np.where(hole, 0, x)), to_bf16(np.where(hole, 0, w).astype(np.float32)))
                continue
            e = np.where(new, e * (1 + 2.0 ** -8) + 2.0 ** -8 * np.abs(np.where(hole, 0, w)), 0)
            plain = ~new & ~hole  # dims that are not turned, and old slots: rounded exactly once
            assert np.array_equal(to_bf16(x[plain]), to_bf16(w[plain].astype(np.float32)))
        elif name == "v" or rot == 0:
            assert np.array_equal(x[~hole], w[~hole].astype(np.float32))
        check(np.where(hole, 0, x), np.where(hole, 0, w), np.where(pool.dtype == "bf16", e + 2.0 ** -8 * np.abs(np.where(hole, 0, w)), e),
              name)
    out = dout.read()
    total = int(sum(counts))
    if q:
        check(out[:total], rq[:total], bq[:total], "q")
    old = xq if in_place or not q else np.full(xq.shape, 5.0, np.float32)
    if in_place or q:
        assert np.array_equal(out[total:], old[total:]), "rows of no sequence written"
    return got, out


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("case", [
    # lens, counts, q heads, kv heads, page, dim, rot
    ([1], [1], 1, 1, 1, 1, 0), ([5], [5], 2, 1, 16, 2, 2), ([37, 16, 40], [1, 1, 1], 8, 2, 16, 64, 64), ([130, 7], [130, 3], 4, 4, 24, 76, 38),
    ([100, 0, 33, 64], [20, 0, 33, 1], 6, 3, 7, 45, 26), ([300], [299], 3, 3, 64, 128, 128), ([9] * 70, [1] * 70, 4, 1, 8, 32, 16),
    ([50, 60], [0, 60], 40, 8, 256, 127, 126), ([3] * 130, [2] * 65 + [0] * 64 + [3], 2, 2, 2, 16, 16), ([20, 21], [5, 6], 200, 2, 5, 96, 96),
])
def test_append(ctx, case, layout, dtype):
    lens, counts, hq, hk, page, d, rot = case
    announce(f"append {case} {layout} {dtype}")
    run_append(ctx, Pool(sum(lens), lens, hk, page, d, dtype), counts, hq, rot, layout, pad=3)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("order", ["phsd", "pshd", "gaps"])
def test_append_strides(ctx, order, dtype):
    announce(f"append strides {order} {dtype}")
    pool = Pool(4, [30, 41], 3, 11, 36, dtype, order)
    run_append(ctx, pool, [7, 41], 6, 20, scale=1.5, order="htd" if order == "pshd" else "gaps")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_append_in_place_positions_and_without_queries(ctx, dtype):
    announce(f"append in place {dtype}")
    lens, counts = [30, 41, 12], [7, 41, 1]
    pos = np.random.default_rng(0).integers(0, 1 << 20, 49 + 2)
    a = run_append(ctx, Pool(4, lens, 3, 16, 64, dtype), counts, 6, 64, positions=pos, pad=2, in_place=True)
    b = run_append(ctx, Pool(4, lens, 3, 16, 64, dtype), counts, 6, 64, positions=pos, pad=2)
    c = run_append(ctx, Pool(4, lens, 3, 16, 64, dtype), counts, 6, 64, positions=pos, pad=2, q=False)
    for x, y, z in zip(a[0], b[0], c[0]):
        assert np.array_equal(x, y, equal_nan=True) and np.array_equal(x, z, equal_nan=True)
    assert np.array_equal(a[1][:49], b[1][:49])


def test_append_bad_pages_and_lengths(ctx):
    """Pages outside the cache and positions before the first are left out, the other tokens are stored."""
    announce("append bad pages")
    pool = Pool(8, [40, 33, 20], 2, 8, 32)
    pool.table[0, 4] = pool.pages
    pool.table[1, 3] = -1
    pool.table[2, 1] = -(1 << 31)
    run_append(ctx, pool, [40, 20, 18], 4, 32)
    pool = Pool(8, [2, 5], 2, 8, 32)
    run_append(ctx, pool, [6, 2], 4, 32)  # four of the six have no position


def test_append_rounds_to_even_and_keeps_specials(ctx):
    announce("append bf16 rounding")
    d = 8
    pool = Pool(8, [1], 1, 4, d, "bf16")
    cache = pool.place(ctx)
    v = np.array([1 + 2.0 ** -8, 1 + 3 * 2.0 ** -8, np.inf, -np.inf, np.nan, 3.4e38, 1e-41, -0.0], np.float32)
    ctx.paged_append(cache, Ints(ctx, [0, 1]).buf, 1, ctx.to_device(v), ctx.to_device(v))
    k, w = pool.read()
    for t in (k, w):
        x = t[pool.table[0, 0], 0, 0]
        assert x[0] == 1 and x[1] == 1 + 2.0 ** -6 and x[2] == np.inf and x[3] == -np.inf and np.isnan(x[4]) and x[5] == np.inf
        assert x[7] == 0 and np.signbit(x[7])


# --------------------------------------------------------------- attention
def run_attention(ctx, pool, counts, hq, scale=None, causal=True, pad=0, order="thd", seed=2, q=None, lse=True, max_q=None, max_kv=None,
                  cache=None):
    rng = np.random.default_rng(seed)
    n, d = int(sum(counts)) + pad, pool.dim
    scale = 1 / np.sqrt(d) if scale is None else scale
    x = rng.standard_normal((n, hq, d)).astype(np.float32) if q is None else q
    cache = pool.place(ctx) if cache is None else cache
    dq = Strided(ctx, x, rows(n, hq, d, order))
    do = Strided(ctx, np.full(x.shape, 7.0, np.float32), rows(n, hq, d, "gaps" if order != "thd" else "thd"))
    dl = ctx.alloc(max(n * hq, 1)).fill(9.0)
    ctx.paged_attention(cache, Ints(ctx, starts_of(counts)).buf, n, max(counts) if max_q is None else max_q,
                        max(pool.lens) if max_kv is None else max_kv, dq.ptr, do.ptr, dl if lse else None, hq, scale, causal, dq.strides,
                        do.strides)
    out, l = do.read(), dl.download(n * hq).reshape(n, hq)
    pool.read()  # nothing of the cache was written
    return x, out, l


def compare(pool, counts, x, out, lse, scale=None, causal=True, keep=None):
    """Every sequence against the padded form's reference on its own positions (keep: those that are not masked)."""
    scale = 1 / np.sqrt(pool.dim) if scale is None else scale
    at = 0
    for b, c in enumerate(counts):
        if c:
            k, v = pool.dense(b, keep=None if keep is None else keep[b])
            ref = Mha(x[at:at + c].transpose(1, 0, 2)[None], k, v, scale, causal)
            check(out[at:at + c].transpose(1, 0, 2)[None], ref.out, ref.out_bound, f"out of sequence {b}")
            check(lse[at:at + c].T[None], ref.lse, ref.lse_bound, f"lse of sequence {b}")
        at += c
    assert np.all(out[at:] == 7.0) and np.all(lse[at:] == 9.0), "rows of no sequence written"


CASES = [
    # lens, counts, q heads, kv heads, page, dim
    ([1], [1], 1, 1, 1, 1), ([1], [1], 1, 1, 16, 64), ([37, 16], [1, 1], 2, 1, 16, 16), ([5], [3], 2, 2, 2, 7),
    ([40, 33, 64, 2], [1, 1, 1, 1], 8, 2, 16, 64), ([700, 300], [1, 1], 16, 4, 16, 128), ([2049], [1], 8, 1, 64, 96),
    ([513, 90, 128], [2, 2, 2], 8, 2, 24, 40), ([100, 0, 33, 64], [20, 0, 33, 1], 6, 3, 7, 45), ([128], [128], 4, 4, 32, 128),
    ([300, 77], [300, 5], 4, 2, 64, 64), ([257], [129], 3, 1, 100, 127), ([640], [200], 2, 2, 16, 33), ([1200, 40, 9], [70, 1, 1], 10, 5, 24, 76),
    ([90, 91], [17, 16], 1, 1, 8, 80), ([1000], [500], 2, 1, 128, 32), ([9] * 70, [1] * 70, 4, 1, 8, 32),
    ([60] * 3, [5] * 3, 71, 1, 16, 64), ([400], [40], 7, 1, 16, 112), ([3] * 130, [2] * 65 + [0] * 64 + [3], 2, 2, 2, 16),
    ([600, 600], [300, 299], 8, 1, 16, 120),
]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("case", CASES)
def test_attention(ctx, case, causal, dtype):
    lens, counts, hq, hk, page, d = case
    announce(f"paged attention {case} causal {causal} {dtype}")
    pool = Pool(sum(lens) + d, lens, hk, page, d, dtype)
    x, out, lse = run_attention(ctx, pool, counts, hq, causal=causal, pad=3)
    compare(pool, counts, x, out, lse, causal=causal)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("order", ["phsd", "pshd", "gaps"])
@pytest.mark.parametrize("case", [([70, 37], [70, 1], 4, 2, 12, 64), ([200], [1], 4, 2, 16, 30), ([333], [150], 2, 1, 32, 128)])
def test_attention_strides(ctx, case, order, dtype):
    lens, counts, hq, hk, page, d = case
    announce(f"paged attention strides {case} {order} {dtype}")
    pool = Pool(5, lens, hk, page, d, dtype, order)
    x, out, lse = run_attention(ctx, pool, counts, hq, scale=0.2, order="htd" if order == "pshd" else "gaps")
    compare(pool, counts, x, out, lse, scale=0.2)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("counts", [[1, 1, 1], [40, 1, 150]])
def test_attention_bounds_above_the_lengths(ctx, counts, dtype):
    """Bounds of a captured call: far above what the sequences have; lse is not asked for."""
    announce(f"paged attention, wide bounds {counts} {dtype}")
    pool = Pool(6, [200, 31, 150], 2, 16, 64, dtype, max_pages=400)
    x, out, lse = run_attention(ctx, pool, counts, 4, max_q=512, max_kv=6400)
    compare(pool, counts, x, out, lse)
    x, out2, none = run_attention(ctx, pool, counts, 4, max_q=512, max_kv=6400, lse=False)
    assert np.array_equal(out, out2) and np.all(none == 9.0)


@pytest.mark.parametrize("most", [2 ** 31, 2 ** 62, 2 ** 63 - 1])
@pytest.mark.parametrize("counts", [[1, 2, 1], [40, 1, 150]])
def test_attention_bounds_above_everything(ctx, counts, most):
    """Bounds that no sequence can have: products with them pass 64 bits."""
    announce(f"paged attention, bounds of {most} {counts}")
    pool = Pool(16, [200, 31, 150], 2, 16, 64)
    x, out, lse = run_attention(ctx, pool, counts, 8, max_q=most, max_kv=most)
    compare(pool, counts, x, out, lse)


@pytest.mark.parametrize("counts", [[3, 1], [60, 20]])
def test_attention_bounds_below_the_lengths(ctx, counts):
    """A longer sequence is cut to max_kv_len, more new tokens to the first max_q_len."""
    announce(f"paged attention, low bounds {counts}")
    pool = Pool(6, [100, 80], 2, 16, 32)
    most = max(counts) - 1
    x, out, lse = run_attention(ctx, pool, counts, 4, max_q=most, max_kv=90)
    k, v = pool.dense(0, keep=np.arange(90))
    ref = Mha(x[:counts[0]].transpose(1, 0, 2)[None], k, v, 1 / np.sqrt(32), True)
    check(out[:most].transpose(1, 0, 2)[None], ref.out[:, :, :most], ref.out_bound[:, :, :most], "out")
    assert np.all(out[most:counts[0]] == 7.0) and np.all(lse[most:counts[0]] == 9.0)
    k, v = pool.dense(1)
    ref = Mha(x[counts[0]:].transpose(1, 0, 2)[None], k, v, 1 / np.sqrt(32), True)
    check(out[counts[0]:].transpose(1, 0, 2)[None], ref.out, ref.out_bound, "out")


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("counts", [[1, 2], [40, 30]])
def test_attention_nothing_to_see(ctx, counts, causal):
    """No positions at all, and tokens before the first position (more new tokens than positions)."""
    announce(f"paged attention, nothing to see {counts} causal {causal}")
    pool = Pool(6, [0, counts[1] - 1], 2, 16, 48)
    x, out, lse = run_attention(ctx, pool, counts, 4, causal=causal)
    n = counts[0]
    assert np.all(out[:n] == 0) and np.all(lse[:n] == -np.inf)
    if causal:
        assert np.all(out[n] == 0) and np.all(lse[n] == -np.inf)
    compare(pool, [0, counts[1]], x[n:], out[n:], lse[n:], causal=causal)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("counts", [[1, 1], [33, 50]])
def test_attention_bad_pages(ctx, counts, dtype):
    """Positions of pages outside the cache are masked."""
    announce(f"paged attention, bad pages {counts} {dtype}")
    pool = Pool(8, [200, 170], 2, 10, 64, dtype)
    good = [np.arange(n) for n in pool.lens]
    k0, v0 = pool.dense(0), pool.dense(1)
    keep = [good[0][(good[0] // 10 != 3) & (good[0] // 10 != 0)], good[1][good[1] // 10 != 7]]
    dense = [pool.dense(b, keep=keep[b]) for b in range(2)]
    pool.table[0, 3], pool.table[0, 0], pool.table[1, 7] = pool.pages, -5, 1 << 30
    x, out, lse = run_attention(ctx, pool, counts, 4)
    at = 0
    for b, c in enumerate(counts):  # all before the new tokens: as if those positions were not there
        ref = Mha(x[at:at + c].transpose(1, 0, 2)[None], *dense[b], 1 / np.sqrt(64), True)
        check(out[at:at + c].transpose(1, 0, 2)[None], ref.out, ref.out_bound, f"out {b}")
        check(lse[at:at + c].T[None], ref.lse, ref.lse_bound, f"lse {b}")
        at += c
    pool.table[:] = -1
    x, out, lse = run_attention(ctx, pool, counts, 4)
    assert np.all(out == 0) and np.all(lse == -np.inf)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("counts", [[4], [64]])
def test_attention_masked_values_are_not_read(ctx, counts, dtype):
    """Infinities and NaN at positions that some rows see and others do not, and in what pages hold past a sequence's end."""
    announce(f"paged attention, NaN in masked places {counts} {dtype}")
    n = counts[0]
    pool = Pool(8, [150], 2, 16, 64, dtype)
    page = pool.table[0, 149 // 16]
    pool.k[page, 0, 149 % 16, 3], pool.v[page, 0, 149 % 16, 5] = np.nan, np.inf  # seen by the last token only
    x, out, lse = run_attention(ctx, pool, counts, 4)
    k, v = pool.dense(0)
    k, v = np.nan_to_num(k, nan=0.0, posinf=0.0), np.nan_to_num(v, nan=0.0, posinf=0.0)
    ref = Mha(x.transpose(1, 0, 2)[None], k, v, 1 / 8, True)
    check(out[:n - 1].transpose(1, 0, 2)[None], ref.out[:, :, :n - 1], ref.out_bound[:, :, :n - 1], "out")
    check(lse[:n - 1].T[None], ref.lse[:, :, :n - 1], ref.lse_bound[:, :, :n - 1], "lse")
    assert np.all(np.isnan(out[n - 1, :2])) and np.all(np.isnan(lse[n - 1, :2]))  # the heads that read key/value head 0
    check(out[n - 1:, 2:].transpose(1, 0, 2)[None], ref.out[:, 2:, n - 1:], ref.out_bound[:, 2:, n - 1:], "out of the other head")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("counts", [[1], [40]])
def test_attention_far_scores(ctx, counts, dtype):
    """Scores far below zero in a whole row, and values of the type's lowest: the softmax is what it is."""
    announce(f"paged attention, far scores {counts} {dtype}")
    d = 32
    pool = Pool(8, [90], 1, 16, d, dtype)
    rng = np.random.default_rng(3)
    for j in range(90):  # K = -big e_0 + small, Q = big e_0: every score near -2^60
        pool.k[pool.table[0, j // 16], 0, j % 16] = 0
        pool.k[pool.table[0, j // 16], 0, j % 16, 0] = -2.0 ** 30
    x = np.zeros((counts[0], 2, d), np.float32)
    x[..., 0] = 2.0 ** 30
    x, out, lse = run_attention(ctx, pool, counts, 2, scale=1.0, q=x)
    first = 90 - counts[0]
    for i in range(counts[0]):  # equal scores: the mean of what is seen
        v = pool.dense(0)[1][0, 0, :first + i + 1].astype(np.float64)
        check(out[i, 0], v.mean(0), 300 * 2.0 ** -24 * np.abs(v).mean(0), f"row {i}")
    low = np.float32(-3.0e38) if dtype == "bf16" else np.finfo(np.float32).min
    for j in range(0, 80, 3):
        pool.k[pool.table[0, j // 16], 0, j % 16] = from_bf16(to_bf16(np.full(d, low))) if dtype == "bf16" else low
    x, out, lse = run_attention(ctx, pool, counts, 2, scale=1.0, q=np.full((counts[0], 2, d), 1.0, np.float32))
    keep = [j for j in range(90) if j >= 80 or j % 3]  # the others' probability is 0
    for i in range(counts[0]):
        js = [j for j in keep if j <= first + i]
        k, v = pool.dense(0, keep=js)
        s = k[0, 0].astype(np.float64).sum(1)
        assert s.max() == s.min()
        check(out[i, 0], v[0, 0].astype(np.float64).mean(0), 300 * 2.0 ** -24 * np.abs(v[0, 0]).mean(0), f"row {i}")


def test_attention_shared_pages(ctx):
    """Sequences that share their first pages, and one page that stands twice in a table."""
    announce("paged attention, shared pages")
    pool = Pool(8, [100, 90], 2, 16, 64)
    pool.table[1, :3] = pool.table[0, :3]
    pool.table[1, 4] = pool.table[1, 3]
    x, out, lse = run_attention(ctx, pool, [3, 20], 4)
    compare(pool, [3, 20], x, out, lse)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_offsets_past_32_bits(ctx, dtype):
    """Pages further apart than 2^32 bytes: a page of the two ends of a large buffer each."""
    announce(f"paged, far pages {dtype}")
    from zigneuron_amd import PagedCache
    size = 2 if dtype == "bf16" else 4
    hk, page, d, lens = 2, 16, 64, [25, 20]
    small = Pool(8, lens, hk, page, d, dtype, spare=0)  # 4 pages
    stride_page = ((1 << 32) + (1 << 20)) // size // 3  # the last page begins past 2^32 bytes
    total = 3 * stride_page + hk * page * d
    big = [ctx.alloc(total * size // 4 + 1) for _ in range(2)]
    from zigneuron_amd import _lib
    for buf, t in zip(big, (small.k, small.v)):
        for n in range(4):
            raw = t[n] if dtype == "f32" else np.where(np.isnan(t[n]), np.uint16(0x7FC0), to_bf16(np.nan_to_num(t[n])))
            raw = np.ascontiguousarray(raw)
            _lib.check(_lib.load().zn_hip_h2d(ctx.handle, buf.ptr + n * stride_page * size, raw.ctypes.data, raw.nbytes), "h2d")
    table, dl = Ints(ctx, small.table), Ints(ctx, lens)
    cache = PagedCache(big[0], big[1], table.ptr, dl.ptr, 2, 4, page, small.max_pages, hk, d, dtype, (stride_page, page * d, d))
    rng = np.random.default_rng(1)
    for counts in ([1, 1], [20, 18]):
        n = sum(counts)
        x = rng.standard_normal((n, 4, d)).astype(np.float32)
        dq, do, dlse = ctx.to_device(x), ctx.alloc(x.size), ctx.alloc(n * 4)
        starts = Ints(ctx, starts_of(counts))
        ctx.paged_attention(cache, starts.ptr, n, max(counts), 25, dq, do, dlse, 4, 1 / 8)
        compare(small, counts, x, do.download().reshape(x.shape), dlse.download().reshape(n, 4))
    # appending there: the last positions of both sequences
    new = rng.standard_normal((2, hk, d)).astype(np.float32)
    dn = ctx.to_device(new)
    ctx.paged_append(cache, Ints(ctx, [0, 1, 2]).buf, 2, dn, dn)
    for b in range(2):
        j = lens[b] - 1
        got = np.empty((hk, page, d), np.uint16 if dtype == "bf16" else np.float32)
        _lib.check(_lib.load().zn_hip_d2h(ctx.handle, got.ctypes.data, big[1].ptr + int(small.table[b, j // page]) * stride_page * size,
                                          got.nbytes), "d2h")
        assert np.array_equal(got[:, j % page], to_bf16(new[b]) if dtype == "bf16" else new[b])
    for buf in big:
        buf.close()


@pytest.mark.parametrize("counts", [[1, 1, 1], [70, 1, 20]])
def test_same_bits_each_time(ctx, counts):
    announce(f"paged attention, twice {counts}")
    pool = Pool(8, [800, 100, 300], 2, 16, 128, "bf16")
    cache = pool.place(ctx)
    a = run_attention(ctx, pool, counts, 8, cache=cache)
    b = run_attention(ctx, pool, counts, 8, cache=cache)
    assert np.array_equal(a[1], b[1]) and np.array_equal(a[2], b[2])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_served_sequence_is_the_whole_sequence(ctx, dtype):
    """The way they are used: a prompt in chunks, then token by token, each step's keys turned and stored and its queries answered -
    against rotary positions and attention of the whole sequence at once, from a captured step replayed for every token."""
    announce(f"served sequence {dtype}")
    hq, hk, d, page, total = 4, 2, 64, 16, 75
    rng = np.random.default_rng(5)
    x = rng.standard_normal((total, hq + 2 * hk, d)).astype(np.float32)  # one projection's output
    pool = Pool(1, [total], hk, page, d, dtype)
    pool.k[:], pool.v[:] = np.nan, np.nan
    cache = pool.place(ctx)
    pitch = ((hq + 2 * hk) * d, d)
    freq = ctx.to_device(frequencies(d))
    dx, dq, do, dl = ctx.alloc(x.size), ctx.alloc(total * hq * d), ctx.alloc(total * hq * d), ctx.alloc(total * hq)
    starts = Ints(ctx, [0, 0])

    def step(n, most):
        ctx.paged_append(cache, starts.ptr, n, dx.offset(hq * d), dx.offset((hq + hk) * d), pitch, dx, dq, hq, pitch, None, freq, d)
        ctx.paged_attention(cache, starts.ptr, n, n, most, dq, do, dl, hq, 1 / 8)

    q_out, out, lse = (np.zeros(s, np.float32) for s in ((total, hq, d), (total, hq, d), (total, hq)))

    def feed(at, n, go):
        dx.upload(x[at:at + n])
        starts.set([0, n])
        pool.dlens.set([at + n])
        go()
        q_out[at:at + n] = dq.download(n * hq * d).reshape(n, hq, d)
        out[at:at + n] = do.download(n * hq * d).reshape(n, hq, d)
        lse[at:at + n] = dl.download(n * hq).reshape(n, hq)

    at = 0
    for n in (40, 20):
        feed(at, n, lambda: step(n, total))
        at += n
    feed(at, 1, lambda: step(1, total))
    at += 1
    graph = ctx.capture(lambda: step(1, total))
    eager = ctx.to_device(np.zeros(1000, np.float32))
    while at < total:
        feed(at, 1, graph.launch)
        eager.fill(float(at))  # other work between the replays
        at += 1
    pos = np.arange(total)
    rq, bq = rotary(x[:, :hq], pos[:, None], frequencies(d), d, "half")
    rk, bk = rotary(x[:, hq:hq + hk], pos[:, None], frequencies(d), d, "half")
    check(q_out, rq, bq, "q")
    k, v = pool.read()
    pages = pool.table[0, pos // page]
    k, v = k[pages, :, pos % page], v[pages, :, pos % page]  # [total, hk, d]
    half = 2.0 ** -8 if dtype == "bf16" else 0.0
    check(k, rk, bk * (1 + half) + half * np.abs(rk), "k")
    check(v, x[:, hq + hk:].astype(np.float64), half * np.abs(x[:, hq + hk:]), "v")
    ref = Mha(q_out.transpose(1, 0, 2)[None], k.transpose(1, 0, 2)[None], v.transpose(1, 0, 2)[None], 1 / 8, True)
    check(out.transpose(1, 0, 2)[None], ref.out, ref.out_bound, "out")
    check(lse.T[None], ref.lse, ref.lse_bound, "lse")
    # and the padded form gives the same on contiguous keys
    dense = [ctx.to_device(np.ascontiguousarray(t.transpose(1, 0, 2))) for t in (q_out, k, v)]
    whole, wl = ctx.alloc(total * hq * d), ctx.alloc(total * hq)
    ctx.mha_forward(*dense, whole, wl, 1, hq, hk, total, total, d, 1 / 8, True)
    check(whole.download().reshape(1, hq, total, d), ref.out, ref.out_bound, "mha")


def test_two_contexts_at_the_same_time(ctx):
    from zigneuron_amd import Context
    announce("paged attention, two contexts")
    pool = Pool(8, [900, 300], 2, 16, 64)
    with Context(0) as other:
        p2 = Pool(8, [900, 300], 2, 16, 64)
        a, b = run_attention(ctx, pool, [1, 1], 8), run_attention(other, p2, [1, 1], 8)
        # queued on both streams before either is read
        caches = [p.place(c) for p, c in ((pool, ctx), (p2, other))]
        outs = []
        for c, cache in ((ctx, caches[0]), (other, caches[1])):
            dq, do = c.to_device(a[0]), c.alloc(a[0].size)
            starts = Ints(c, [0, 1, 2])
            for _ in range(20):
                c.paged_attention(cache, starts.ptr, 2, 1, 900, dq, do, None, 8, 1 / 8)
            outs.append((dq, do, starts))
        for _, do, _ in outs:
            assert np.array_equal(do.download().reshape(a[1].shape), a[1])
        assert np.array_equal(a[1], b[1])
        del outs, caches
