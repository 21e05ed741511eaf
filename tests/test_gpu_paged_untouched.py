"""What calls on a paged cache leave alone: rows and heads beside special values, and everything that starts in any order cannot mean."""
from __future__ import annotations

import numpy as np
import pytest

from gpu_common import announce
from paged_ref import Ints, Pool, from_bf16, starts_of, to_bf16
from test_gpu_paged import run_attention

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    from zigneuron_amd import Context
    c = Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim,page", [(64, 16), (100, 24)])
@pytest.mark.parametrize("new,hq", [(1, 2), (1, 40), (9, 4), (14, 8), (50, 8), (140, 4)])
def test_rows_beside_special_values(ctx, new, hq, dim, page, dtype):
    """NaN and infinities that one token of one key/value head sees: the other sequence and the other head have the bits of the call
    without them, that token has NaN."""
    announce(f"beside special values new {new} heads {hq} dim {dim} {dtype}")
    lens = [300 + new, 70 + new]
    pool, clean = Pool(8, lens, 2, page, dim, dtype), Pool(8, lens, 2, page, dim, dtype)
    j = lens[0] - 1
    s = (pool.table[0, j // page], 0, j % page)
    pool.k[s], pool.v[s] = np.inf, np.nan
    x, out, lse = run_attention(ctx, pool, [new, new], hq)
    _, want, wlse = run_attention(ctx, clean, [new, new], hq)
    other = np.ones(out.shape[:2], bool)
    other[:new, :hq // 2] = False
    assert other.any() and np.array_equal(out[other], want[other]) and np.array_equal(lse[other], wlse[other])
    assert np.all(np.isnan(out[new - 1, :hq // 2])) and np.all(np.isnan(lse[new - 1, :hq // 2]))
    assert np.isfinite(out[:new - 1]).all() and np.isfinite(lse[:new - 1]).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("new", [1, 40])
def test_starts_in_any_order(ctx, new, dtype):
    """Nothing is promised for the tokens' slots, but no other slot is written: not past a sequence's length, not in pages of no
    sequence; what is written are the new rows' values, dim for dim and head for head."""
    announce(f"starts in any order {new} {dtype}")
    n, hk, d = 3 * new, 2, 32
    rng = np.random.default_rng(2)
    xk, xv = (rng.standard_normal((n, hk, d)).astype(np.float32) for _ in range(2))
    if dtype == "bf16":
        xk, xv = from_bf16(to_bf16(xk)), from_bf16(to_bf16(xv))
    for starts in ([n, 0, 2, n + 7], [3, 3, 2, 1], [-5, 1000, -7, 2], [2 ** 31 - 1, -(2 ** 31), 0, 2 ** 31 - 1], [0, n, 0, n]):
        pool = Pool(8, [90, 60, 45], hk, 16, d, dtype, spare=6)
        cache = pool.place(ctx)
        ds, dk, dv = Ints(ctx, starts), ctx.to_device(xk), ctx.to_device(xv)
        ctx.paged_append(cache, ds.ptr, n, dk, dv)
        for got, old, x in zip(pool.read(), (pool.k, pool.v), (xk, xv)):
            assert np.array_equal(np.isnan(got), np.isnan(old)), starts  # slots of no position stay as they were
            page, head, slot, dim = np.nonzero((got != old) & ~np.isnan(old))
            new_rows = x[:, head, dim] == got[page, head, slot, dim]
            assert np.all(new_rows.any(0)), starts


@pytest.mark.parametrize("new", [1, 40])
def test_ascending_starts_between_odd_rows(ctx, new):
    """Rows before the first start and behind the last are of no sequence, for both calls."""
    announce(f"rows of no sequence {new}")
    n, hq, hk, d = 3 * new + 9, 4, 2, 32
    rng = np.random.default_rng(2)
    starts = np.array([5, 5 + new, 5 + 2 * new, 5 + 3 * new], np.int32)
    x = rng.standard_normal((n, hq, d)).astype(np.float32)
    pool = Pool(8, [90, 60, 45], hk, 16, d)
    cache = pool.place(ctx)
    ds, dx, do = Ints(ctx, starts), ctx.to_device(x), ctx.alloc(x.size).fill(5.0)
    ctx.paged_attention(cache, ds.ptr, n, new, 90, dx, do, None, hq, 0.2)
    got = do.download().reshape(x.shape)
    assert np.all(got[:5] == 5.0) and np.all(got[5 + 3 * new:] == 5.0)
    want = ctx.alloc(x.size)
    d0 = Ints(ctx, starts_of([new] * 3))
    dy = ctx.to_device(np.ascontiguousarray(x[5:5 + 3 * new]))
    ctx.paged_attention(cache, d0.ptr, 3 * new, new, 90, dy, want, None, hq, 0.2)
    # the same rows at another place: a tile's rows and parts are the same, so are the bits
    assert np.array_equal(got[5:5 + 3 * new], want.download(3 * new * hq * d).reshape(3 * new, hq, d))
    dk = ctx.to_device(rng.standard_normal((n, hk, d)).astype(np.float32))
    q_out = ctx.alloc(x.size).fill(5.0)
    ctx.paged_append(cache, ds.ptr, n, dk, dk, q=dx, q_out=q_out, q_heads=hq)
    q = q_out.download().reshape(x.shape)
    assert np.all(q[:5] == 5.0) and np.all(q[5 + 3 * new:] == 5.0) and np.array_equal(q[5:5 + 3 * new], x[5:5 + 3 * new])


@pytest.mark.parametrize("counts,d", [([1, 1], 64), ([40, 3], 64), ([9, 0], 128), ([5, 5], 4)])
@pytest.mark.parametrize("causal", [True, False])
def test_a_cache_of_no_pages(ctx, counts, d, causal):
    """Null pools and table: nothing is stored, every position is masked; queries are turned all the same."""
    from zigneuron_amd import PagedCache
    announce(f"no pages {counts} {d} {causal}")
    n, hq, hk = sum(counts), 4, 2
    lens, starts = Ints(ctx, [50, 60]), Ints(ctx, starts_of(counts))
    cache = PagedCache(None, None, None, lens.ptr, 2, 0, 16, 8, hk, d)
    x = np.random.default_rng(1).standard_normal((n, hq, d)).astype(np.float32)
    dx, do, dl = ctx.to_device(x), ctx.alloc(x.size).fill(7.0), ctx.alloc(n * hq).fill(9.0)
    ctx.paged_attention(cache, starts.ptr, n, max(counts), 60, dx, do, dl, hq, 0.2, causal)
    assert np.all(do.download() == 0) and np.all(dl.download() == -np.inf)
    ctx.paged_append(cache, starts.ptr, n, dx, dx, (hq * d, d), dx, do, hq)
    assert np.array_equal(do.download().reshape(x.shape), x)
