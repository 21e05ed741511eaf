"""Every kernel of the attention over a paged cache against 64 bits (which call reaches which is held by tests/test_paged_plan.py)."""
from __future__ import annotations

import numpy as np
import pytest

from block_ops_ref import Mha, check
from gpu_common import announce
from paged_cases import cases
from paged_ref import Pool
from test_gpu_paged import compare, run_attention

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    from zigneuron_amd import Context
    c = Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("case", cases(), ids=lambda c: f"{c[0]}-{c[5]}-{c[6]}")
def test_each_kernel(ctx, case):
    name, lens, counts, hq, hk, page, dim, dtype = case
    for causal in (True, False):
        announce(f"{name} page {page} dim {dim} causal {causal}")
        pool = Pool(page + dim, lens, hk, page, dim, dtype)
        x, out, lse = run_attention(ctx, pool, counts, hq, causal=causal, pad=2)
        compare(pool, counts, x, out, lse, causal=causal)


@pytest.mark.parametrize("case", [c for c in cases() if "few4" in c[0] or "wide" in c[0]], ids=lambda c: f"{c[0]}-{c[5]}-{c[6]}")
def test_special_values_and_holes(ctx, case):
    """A NaN key and an infinite value that only the last token of one sequence sees, and a page outside the cache in another: the rows
    that meet neither have the bits of the call without them."""
    name, lens, counts, hq, hk, page, dim, dtype = case
    announce(f"{name} page {page} dim {dim} special values")
    group, starts = hq // hk, np.concatenate([[0], np.cumsum(counts)])
    holed = [b for b, c in enumerate(counts) if c and lens[b] - c >= 2 * page][-1]  # new tokens behind the hole
    poisoned = [b for b, c in enumerate(counts) if c and lens[b] > c and b != holed][0]
    pool, clean = Pool(page + dim, lens, hk, page, dim, dtype), Pool(page + dim, lens, hk, page, dim, dtype)
    j = lens[poisoned] - 1
    s = (pool.table[poisoned, j // page], 0, j % page)
    pool.k[s], pool.v[s] = np.nan, np.inf
    pool.table[holed, 1] = pool.pages
    x, out, lse = run_attention(ctx, pool, counts, hq, pad=2)
    _, want, wlse = run_attention(ctx, clean, counts, hq, pad=2)
    other = np.ones(out.shape[:2], bool)
    other[starts[poisoned]:starts[poisoned + 1], :group] = False  # the heads that read what holds them
    other[starts[holed]:starts[holed + 1]] = False
    assert np.array_equal(out[other], want[other]) and np.array_equal(lse[other], wlse[other])
    last = starts[poisoned + 1] - 1
    assert np.all(np.isnan(out[last, :group])) and np.all(np.isnan(lse[last, :group]))

    def against(rows, b, keep):
        k, v = clean.dense(b, keep=keep)
        ref = Mha(x[rows].transpose(1, 0, 2)[None], k, v, 1 / np.sqrt(dim), True)
        check(out[rows].transpose(1, 0, 2)[None], ref.out, ref.out_bound, f"out of sequence {b}")
        check(lse[rows].T[None], ref.lse, ref.lse_bound, f"lse of sequence {b}")

    if counts[poisoned] > 1:  # its earlier tokens: as if the last position was not there
        against(slice(starts[poisoned], last), poisoned, np.arange(j))
    js = np.arange(lens[holed])
    against(slice(starts[holed], starts[holed + 1]), holed, js[js // page != 1])
