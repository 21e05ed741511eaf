"""Attention over a paged cache, path by path: numbers of query rows on both sides of every kernel's limit, walks in parts and whole,
batches of all kinds in one call, captured calls whose lengths change."""
from __future__ import annotations

import numpy as np
import pytest

from block_ops_ref import Mha, check
from gpu_common import announce
from paged_ref import Ints, Pool, starts_of
from test_gpu_paged import compare, run_attention

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    from zigneuron_amd import Context
    c = Context(0)
    yield c
    c.close()


# new tokens x group of 15 to 260 query rows of a key/value head: around 16, 32, 64, 128 and 256
ROWS = [(1, 15), (1, 16), (1, 17), (4, 4), (17, 1), (16, 2), (33, 1), (8, 4), (11, 3), (16, 4), (13, 5), (1, 64), (1, 65), (32, 4),
        (43, 3), (127, 1), (64, 4), (86, 3), (257, 1), (52, 5)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("new,group", ROWS)
def test_numbers_of_rows(ctx, new, group, dtype):
    announce(f"rows {new} x {group} {dtype}")
    for seed, (dim, page, lens) in enumerate(((128, 16, [new + 411, new]), (61, 13, [new + 95, new + 200]))):
        pool = Pool(new + group + seed, lens, 2, page, dim, dtype)
        x, out, lse = run_attention(ctx, pool, [new, new], 2 * group, pad=1)
        compare(pool, [new, new], x, out, lse)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [8, 9, 31, 32, 33, 48, 64, 65, 95, 96, 97, 100, 128])
@pytest.mark.parametrize("new", [1, 6, 40])
def test_dims(ctx, dim, new, dtype):
    announce(f"dims {dim} new {new} {dtype}")
    pool = Pool(dim + new, [new + 77, new + 130], 2, 16, dim, dtype)
    x, out, lse = run_attention(ctx, pool, [new, new], 8)
    compare(pool, [new, new], x, out, lse)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("new,hq", [(1, 4), (1, 16), (7, 4), (12, 4), (100, 4), (300, 2)])
def test_long_walks_in_parts(ctx, new, hq, dtype):
    """Few sequences against thousands of positions: every walk is cut into parts and joined."""
    announce(f"long walk new {new} heads {hq} {dtype}")
    pool = Pool(3, [6000, 2500 + new], 1, 64, 64, dtype)
    x, out, lse = run_attention(ctx, pool, [new, new], hq)
    compare(pool, [new, new], x, out, lse)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("group,dim", [(1, 64), (4, 128), (2, 76), (20, 64)])
def test_all_kinds_in_one_call(ctx, group, dim, dtype):
    """Single tokens, few, chunks and whole prompts, empty slots between them."""
    announce(f"mixed group {group} dim {dim} {dtype}")
    counts = [1, 300, 0, 5, 1, 1, 0, 130, 16, 1, 2, 65]
    lens = [900, 300, 0, 77, 1, 2300, 50, 1400, 16, 33, 1000, 70]
    pool = Pool(9, lens, 2, 24, dim, dtype)
    x, out, lse = run_attention(ctx, pool, counts, 2 * group, pad=4)
    compare(pool, counts, x, out, lse)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_many_sequences(ctx, dtype):
    """More than the 64 sequences that a wave looks at at once; chunks among the last of them."""
    announce(f"many sequences {dtype}")
    counts = [1] * 70 + [0] * 65 + [40, 1, 0, 150, 1]
    lens = [5 + i % 40 for i in range(70)] + [i % 3 for i in range(65)] + [90, 30, 0, 150, 1]
    pool = Pool(9, lens, 2, 8, 32, dtype)
    x, out, lse = run_attention(ctx, pool, counts, 4, pad=2)
    compare(pool, counts, x, out, lse)


def test_more_heads_than_counters(ctx):
    """Past 4096 sequences' heads no walk is cut."""
    announce("many heads")
    n = 1400
    lens = [1 + (7 * i) % 300 for i in range(n)]
    pool = Pool(9, lens, 3, 32, 16)
    x, out, lse = run_attention(ctx, pool, [1] * n, 3)
    some = [0, 1, 699, 1398, 1399]
    for b in some:
        k, v = pool.dense(b)
        ref = Mha(x[b:b + 1].transpose(1, 0, 2)[None], k, v, 1 / 4, True)
        check(out[b:b + 1].transpose(1, 0, 2)[None], ref.out, ref.out_bound, f"out {b}")
        check(lse[b:b + 1].T[None], ref.lse, ref.lse_bound, f"lse {b}")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("new,hq", [(1, 2), (9, 4), (14, 8), (50, 8), (140, 4)])
def test_special_values(ctx, new, hq, dtype):
    """NaN and infinities where only the last token sees them, in every path; the other rows and heads are as without them."""
    announce(f"special values new {new} heads {hq} {dtype}")
    pool = Pool(8, [300 + new, 70 + new], 2, 16, 64, dtype)
    clean = Pool(8, [300 + new, 70 + new], 2, 16, 64, dtype)
    j = pool.lens[0] - 1
    s = (pool.table[0, j // 16], 0, j % 16)
    pool.k[s], pool.v[s] = np.inf, np.nan
    x, out, lse = run_attention(ctx, pool, [new, new], hq)
    _, want, wlse = run_attention(ctx, clean, [new, new], hq)
    mine = np.zeros(out.shape[:2], bool)
    mine[new - 1, :hq // 2] = True
    assert np.all(np.isnan(out[mine])) and np.array_equal(out[~mine].shape, want[~mine].shape)
    at = 0
    for b in range(2):
        k, v = clean.dense(b)
        ref = Mha(x[at:at + new].transpose(1, 0, 2)[None], k, v, 1 / 8, True)
        keep = ~mine[at:at + new].T[None]
        check(out[at:at + new].transpose(1, 0, 2)[None][keep], ref.out[keep], ref.out_bound[keep], f"out {b}")
        check(lse[at:at + new].T[None][keep], ref.lse[keep], ref.lse_bound[keep], f"lse {b}")
        at += new


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("new,hq", [(1, 2), (9, 4), (14, 8), (140, 4)])
def test_holes(ctx, new, hq, dtype):
    """One page outside the cache, in every path: its positions are masked, whichever wave of a workgroup meets it."""
    announce(f"holes new {new} heads {hq} {dtype}")
    for hole in (0, 4, 17):
        pool = Pool(8, [300 + new], 2, 16, 64, dtype)
        js = np.arange(pool.lens[0])
        k, v = pool.dense(0, keep=js[js // 16 != hole])
        pool.table[0, hole] = pool.pages + hole
        x, out, lse = run_attention(ctx, pool, [new], hq)
        ref = Mha(x.transpose(1, 0, 2)[None], k, v, 1 / 8, True)
        check(out.transpose(1, 0, 2)[None], ref.out, ref.out_bound, f"out {hole}")
        check(lse.T[None], ref.lse, ref.lse_bound, f"lse {hole}")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("max_new", [1, 6, 60])
def test_replays_with_other_lengths(ctx, max_new, dtype):
    """A captured call is replayed as the batch changes (lengths, numbers of new tokens, pages), other work between the replays; each
    replay has the bits of an eager call with the same bounds."""
    announce(f"replays {max_new} {dtype}")
    rng = np.random.default_rng(4)
    batch, tokens, hq, d = 5, 5 * max_new, 8, 64
    pool = Pool(8, [700] * batch, 2, 16, d, dtype)
    cache = pool.place(ctx)
    starts = Ints(ctx, [0] * (batch + 1))
    dq, do, dl = ctx.to_device(rng.standard_normal((tokens, hq, d)).astype(np.float32)), ctx.alloc(tokens * hq * d), ctx.alloc(tokens * hq)
    call = lambda: ctx.paged_attention(cache, starts.ptr, tokens, max_new, 700, dq, do, dl, hq, 1 / 8)  # noqa: E731
    call()
    graph = ctx.capture(call)
    a = rng.standard_normal((256, 256)).astype(np.float32)
    da, db, dc = ctx.to_device(a), ctx.to_device(a), ctx.alloc(a.size)
    for step in range(6):
        counts = rng.integers(0, max_new + 1, batch)
        counts[step % batch] = max_new
        lens = np.maximum(counts, rng.integers(0, 701, batch))
        starts.set(starts_of(counts))
        pool.dlens.set(lens)
        pool.dtable.set(pool.table[rng.permutation(batch)])
        got = []
        for go in (graph.launch, call, graph.launch):
            do.fill(7.0)
            dl.fill(9.0)
            go()
            ctx.sgemm("nn", 256, 256, 256, da, 256, db, 256, dc, 256)  # split over workgroups too
            got.append((do.download(), dl.download()))
        for o, l in got[1:]:
            assert np.array_equal(o, got[0][0]) and np.array_equal(l, got[0][1]), f"replay {step}"
        n = int(sum(counts)) * hq
        assert np.all(got[0][0][n * d:] == 7.0) and np.all(got[0][1][n:] == 9.0)
        assert np.isfinite(got[0][0]).all()
        check(dc.download(a.size).reshape(a.shape), a.astype(np.float64) @ a, 300 * 2.0 ** -24 * (np.abs(a).astype(np.float64) @ np.abs(a)), "product")


def test_two_graphs_of_one_context(ctx):
    """Their calls share the context's counters and run one after the other."""
    announce("two graphs")
    pools = [Pool(8 + i, [1500, 300], 2, 16, 64) for i in range(2)]
    eager = [run_attention(ctx, p, [1, 1], 8) for p in pools]
    caches = [p.place(ctx) for p in pools]
    starts, dq, do = Ints(ctx, [0, 1, 2]), [ctx.to_device(e[0]) for e in eager], [ctx.alloc(e[0].size) for e in eager]
    graphs = [ctx.capture(lambda i=i: ctx.paged_attention(caches[i], starts.ptr, 2, 1, 1500, dq[i], do[i], None, 8, 1 / 8)) for i in range(2)]
    for _ in range(5):
        for g in graphs:
            g.launch()
    for i in range(2):
        assert np.array_equal(do[i].download().reshape(eager[i][1].shape), eager[i][1])


def test_starts_that_do_not_ascend(ctx):
    """Nothing is promised for their rows, but nothing else is touched."""
    announce("odd starts")
    for new in (1, 40):
        pool = Pool(8, [90, 60, 45], 2, 16, 32)
        cache = pool.place(ctx)
        n = 3 * new
        x = np.random.default_rng(1).standard_normal((n, 4, 32)).astype(np.float32)
        dq = ctx.to_device(x)
        guard = ctx.alloc(x.size + 2000).fill(5.0)
        for starts in ([n, 0, 2, n + 7], [3, 3, 2, 1], [-5, 1000, -7, 2], [2 ** 31 - 1, -(2 ** 31), 0, 2 ** 31 - 1]):
            ctx.paged_attention(cache, Ints(ctx, starts).buf, n, new, 90, dq, guard.offset(1000), None, 4, 1 / 6)
            ctx.paged_append(cache, Ints(ctx, starts).buf, n, dq, dq, (128, 32))
        now = guard.download()
        assert np.all(now[:1000] == 5.0) and np.all(now[1000 + x.size:] == 5.0)
        pool.dtable.buf.download()
        k, _ = (t.read() for t in (pool.dk, pool.dv))  # nothing between the cache's rows
        assert k.shape == pool.k.shape


def test_zero_scale_and_broadcast(ctx):
    """scale 0: the mean of what is seen.  One query row and one key/value head for all (strides of 0)."""
    announce("zero scale, broadcast")
    pool = Pool(8, [50], 1, 16, 32)
    x, out, lse = run_attention(ctx, pool, [3], 2, scale=0.0)
    for i in range(3):
        v = pool.dense(0)[1][0, 0, :48 + i].astype(np.float64)
        check(out[i, 0], v.mean(0), 100 * 2.0 ** -24 * np.abs(v).mean(0), "mean")
        assert abs(lse[i, 0] - np.log(48 + i)) < 1e-5
    from zigneuron_amd import PagedCache
    pool.place(ctx)
    cache = PagedCache(pool.dk.ptr, pool.dv.ptr, pool.dtable.ptr, pool.dlens.ptr, 1, pool.pages, 16, pool.max_pages, 4, 32,
                       strides=(16 * 32, 0, 32))
    q = np.random.default_rng(0).standard_normal(32).astype(np.float32)
    dq, do = ctx.to_device(q), ctx.alloc(2 * 8 * 32)
    ctx.paged_attention(cache, Ints(ctx, [0, 2]).buf, 2, 2, 50, dq, do, None, 8, 0.2, True, (0, 0))
    got = do.download().reshape(2, 8, 32)
    k, v = pool.dense(0)
    ref = Mha(np.broadcast_to(q, (1, 1, 2, 32)), k, v, 0.2, True)
    for h in range(8):
        check(got[:, h][None, None], ref.out, ref.out_bound, f"head {h}")


def test_no_new_tokens(ctx):
    """Rows of no sequence only: nothing is written."""
    announce("no new tokens")
    pool = Pool(8, [50, 20], 2, 16, 32)
    x, out, lse = run_attention(ctx, pool, [0, 0], 4, pad=3)
    assert np.all(out == 7.0) and np.all(lse == 9.0)
    x, out, lse = run_attention(ctx, pool, [0, 0], 4, pad=3, max_q=40)
    assert np.all(out == 7.0) and np.all(lse == 9.0)
    x, out, lse = run_attention(ctx, pool, [2, 1], 4, max_kv=0)  # nothing to see
    assert np.all(out == 0) and np.all(lse == -np.inf)
    x, out, lse = run_attention(ctx, pool, [20, 20], 4, max_kv=0)
    assert np.all(out == 0) and np.all(lse == -np.inf)
