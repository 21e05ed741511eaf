"""Grouped attention on tensors full of NaN, as a training step that has diverged has them: NaN, and no slower than that
takes.  Rows whose sums are not finite are computed one key at a time, so a walk whose result is known has to end."""
from __future__ import annotations

import time

import numpy as np
import pytest

from block_ops_ref import Mha, check
from gpu_common import announce
from test_gpu_mha import make, run_backward, run_forward

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    from zigneuron_amd import Context
    c = Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("what", ["q", "k", "all"])
@pytest.mark.parametrize("sq", [8, 200, 1500])
def test_a_step_full_of_nan_takes_little_longer(ctx, sq, what):
    b, hq, hk, sk, d = 1, 8, 4, 1500, 64
    shape = (b, hq, hk, sq, sk, d, 0.125, True)
    q, k, v, g = make(1, *shape[:6])
    dev = {n: ctx.to_device(t) for n, t in zip("qkvg", (q, k, v, g))}
    o, l = ctx.alloc(q.size), ctx.alloc(b * hq * sq)
    grads = [ctx.alloc(t.size) for t in (q, k, v)]

    def step():
        ctx.mha_forward(dev["q"], dev["k"], dev["v"], o, l, *shape)
        ctx.mha_backward(dev["q"], dev["k"], dev["v"], o, l, dev["g"], *grads, *shape)

    def best():
        times = []
        for _ in range(5):
            ctx.sync()
            start = time.perf_counter()
            step()
            ctx.sync()
            times.append(time.perf_counter() - start)
        return min(times)

    usual = best()
    for n in "qkvg" if what == "all" else what:
        dev[n].fill(float("nan"))
    announce(f"mha full of NaN: {what}, {sq} queries, {usual * 1e6:.0f} us without")
    diverged = best()
    print(f"{diverged * 1e6:.0f} us", flush=True)
    assert all(np.isnan(t.download()).all() for t in (o, *grads))
    assert np.isnan(l.download()).all()
    # a row that takes its keys one at a time is tens of times slower
    assert diverged < 6 * usual


def test_one_row_of_nan(ctx):
    """A NaN query: its own row, and every key that it sees."""
    shape = (1, 2, 1, 333, 333, 64)
    q, k, v, g = make(2, *shape)
    q[0, 1, 100, 5] = np.nan
    announce("mha beside a NaN query")
    clean = np.where(np.isnan(q), 0.0, q).astype(np.float32)
    ref = Mha(clean, k, v, 0.125, True)
    out, lse = run_forward(ctx, q, k, v, 0.125, True)
    others = np.delete(np.arange(333), 100)
    for h, rows in ((0, np.arange(333)), (1, others)):
        check(out[0, h, rows], ref.out[0, h, rows], ref.out_bound[0, h, rows], "out")
        check(lse[0, h, rows], ref.lse[0, h, rows], ref.lse_bound[0, h, rows], "lse")
    assert np.isnan(out[0, 1, 100]).all() and np.isnan(lse[0, 1, 100])
    gq, gk, gv = run_backward(ctx, q, k, v, out, lse, g, 0.125, True)
    g2 = g.copy()
    g2[0, 1, 100] = 0.0  # without that query's share: what the keys behind it and the other queries have
    clean_out, clean_lse = run_forward(ctx, clean, k, v, 0.125, True)
    grads, bounds = ref.backward(g2, clean_out, clean_lse)
    for h, rows in ((0, np.arange(333)), (1, others)):
        check(gq[0, h, rows], grads[0][0, h, rows], bounds[0][0, h, rows], "grad_q")
    assert np.isnan(gq[0, 1, 100]).all()
    for name, x, i in (("grad_k", gk, 1), ("grad_v", gv, 2)):
        assert np.isnan(x[0, 0, :101]).all(), name
        check(x[0, 0, 101:], grads[i][0, 0, 101:], bounds[i][0, 0, 101:], name)
