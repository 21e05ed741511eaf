"""The gated Dense forward's ways to run, each by name or at a size that only it can take."""
from __future__ import annotations

import numpy as np
import pytest

from block_ops_ref import U, check, gate, gate_err
from gpu_common import announce

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    from zigneuron_amd import Context
    c = Context(0)
    yield c
    c.close()


def test_more_units_than_one_launch_of_the_few_row_kernel(ctx):
    """2^27 units, 32 to a workgroup of 1024 threads, would be 2^32 threads: the product and a pass take them."""
    hidden = (1 << 27) + 5
    x = np.array([1.5], np.float32)
    period = 100003
    w = (np.random.default_rng(1).standard_normal(period)).astype(np.float32)
    dx, dw, h = ctx.to_device(x), ctx.to_device(np.resize(w, 2 * hidden)), ctx.alloc(hidden)
    announce(f"gated forward, 1 x 1 x 2 x {hidden}")
    ctx.gated_dense_forward("silu", dx, dw, None, None, h, 1, 1, hidden)
    got = h.download()
    at = np.concatenate([np.arange(5000), np.arange(0, hidden, 1009), np.arange(hidden - 5000, hidden)])
    z, up = (1.5 * w[(at + o) % period].astype(np.float64) for o in (0, hidden))
    y = gate("silu", z)[0]
    # each projection is one product, rounded; the gate's slope is at most 1.13
    ey = gate_err("silu", z)[0] + 1.13 * U * np.abs(z)
    check(got[at], y * up, ey * np.abs(up) + (np.abs(y) + ey) * U * np.abs(up) + 2 * U * np.abs(y * up), "h")
    for t in (dx, dw, h):
        t.close()
