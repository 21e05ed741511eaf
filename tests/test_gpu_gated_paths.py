"""The gated Dense forward's ways to run, each by name or at a size that only it can take."""
from __future__ import annotations

import contextlib

import numpy as np
import pytest

from block_ops_ref import U, check, gate, gate_err
from gpu_common import announce
from test_gpu_gated import ACTS, forward_ref, make, run_forward

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


# the one launch's tiles: 256, 128, 64 units beside as many of the gate's and 256, 256, 128, 128 rows
TILES = ["256x256s", "256x128s", "128x128s", "128x64s"]


@contextlib.contextmanager
def forced(ctx, tile):
    ctx.set_gemm_tile(tile)
    try:
        yield
    finally:
        ctx.set_gemm_tile("auto")


@pytest.mark.parametrize("tile", TILES)
@pytest.mark.parametrize("size", [(1, 1, 1), (3, 31, 5), (127, 33, 33), (256, 64, 128), (257, 129, 131), (130, 1000, 63), (515, 70, 300)])
def test_tiles(ctx, tile, size):
    x, w, b, _, _ = make(sum(size), *size)
    for bias in (None, b):
        announce(f"gated forward on {tile} {size} bias {bias is not None}")
        z, ez, h, eh = forward_ref("silu", x, w, bias)
        with forced(ctx, tile):
            gz, gh = run_forward(ctx, "silu", x, w, bias)
            alone = run_forward(ctx, "silu", x, w, bias, keep=False)[1]
        check(gz, z, ez, "z")
        check(gh, h, eh, "h")
        assert np.array_equal(alone, gh)


@pytest.mark.parametrize("tile", TILES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("bias", [False, True])
def test_gates(ctx, tile, act, bias):
    x, w, b, _, _ = make(1, 270, 53, 141)
    announce(f"gated forward {act} on {tile} bias {bias}")
    z, ez, h, eh = forward_ref(act, x, w, b if bias else None)
    with forced(ctx, tile):
        gz, gh = run_forward(ctx, act, x, w, b if bias else None)
    check(gz, z, ez, "z")
    check(gh, h, eh, "h")


@pytest.mark.parametrize("tile", TILES)
def test_sums_that_are_not_finite(ctx, tile):
    """A NaN in a row of x, infinities in a gate's and an up projection's column of W and sums past the split's range:
    each stays in its row or column, the rest of the tile is what it was."""
    m, k, n = 300, 100, 141
    x, w, b, _, _ = make(6, m, k, n)
    x[:, 7] *= np.float32(1e15)
    w[7] *= np.float32(1e12)  # sums of 1e27: the split's parts of them overflow
    w[5, 33], w[9, n + 77] = np.inf, -np.inf
    rest = np.delete(np.arange(m), 177)
    x[177, 20] = np.nan
    announce(f"gated forward on {tile}, sums not finite")
    finite = np.where(np.isfinite(w), w, 0.0).astype(np.float32)
    z, ez, h, eh = forward_ref("relu", x[rest], finite, b)
    for col, row in ((33, 5), (n + 77, 9)):
        z[:, col] = x[rest, row].astype(np.float64) * w[row, col]
    with np.errstate(invalid="ignore"):
        h = np.maximum(z[:, :n], 0) * z[:, n:]
    # products past fp32's range are infinities there, and an infinity's sign or NaN takes factors whose sign is certain
    h = np.where(np.abs(h) > 2.0 ** 129, np.copysign(np.inf, h), h)
    certain = (np.abs(z[:, :n]) > ez[:, :n]) & (np.abs(z[:, n:]) > ez[:, n:])
    sure = ~np.isnan(h) & (np.abs(h) < 2.0 ** 127) | np.isinf(h) & certain
    assert sure.mean() > 0.9
    with forced(ctx, tile):
        gz, gh = run_forward(ctx, "relu", x, w, b)
    check(gz[rest], z, ez, "z")
    check(np.where(sure, gh[rest], 0.0), np.where(sure, h, 0.0), eh, "h")
    assert np.isnan(gz[177]).all()


@pytest.mark.parametrize("tile", TILES)
def test_the_same_bits_each_time_and_in_a_graph(ctx, tile):
    m, k, n = 392, 160, 224
    x, w, b, _, _ = make(8, m, k, n)
    d = [ctx.to_device(t) for t in (x, w, b)]
    z, h = ctx.alloc(m * 2 * n), ctx.alloc(m * n)

    def step():
        ctx.gated_dense_forward("gelu", *d, z, h, m, k, n)

    announce(f"gated forward on {tile} in a graph")
    with forced(ctx, tile):
        step()
        first = [t.download() for t in (z, h)]
        graph = ctx.capture(step)
        for _ in range(3):
            for run in (graph.launch, step):
                z.fill(float("nan"))
                h.fill(float("nan"))
                run()
                for t, want in zip((z, h), first):
                    assert np.array_equal(t.download(), want)
        graph.close()


@pytest.mark.parametrize("size", [(2048, 256, 4096), (2047, 259, 4099), (4096, 64, 1024), (4097, 65, 1023), (1024, 1024, 4096),
                                  (777, 1023, 1001)])
def test_large_layers(ctx, size):
    """Sizes that the policy gives to the widest tiles, whatever it makes of them later."""
    x, w, b, _, _ = make(sum(size), *size)
    announce(f"gated forward {size}")
    z, ez, h, eh = forward_ref("gelu", x, w, b)
    gz, gh = run_forward(ctx, "gelu", x, w, b)
    check(gz, z, ez, "z")
    check(gh, h, eh, "h")


def test_a_tile_has_the_bits_of_the_product_on_it(ctx):
    m, k, n = 300, 259, 128
    x, w, b, _, _ = make(12, m, k, n)
    dx, dw, dc = ctx.to_device(x), ctx.to_device(w), ctx.alloc(m * 2 * n)
    announce("gated forward against the product on the same tile")
    for tile in TILES:
        with forced(ctx, tile):
            gz, _ = run_forward(ctx, "linear", x, w, None)
            ctx.sgemm("nn", m, 2 * n, k, dx, k, dw, 2 * n, dc, 2 * n)
        assert np.array_equal(gz, dc.download().reshape(m, 2 * n)), tile
