"""The gated Dense layer on the GPU (zn_hip_gated_dense_forward and _backward) against 64 bits."""
from __future__ import annotations

import numpy as np
import pytest

from block_ops_ref import U, check, dot_err, gate, gate_err
from gpu_common import announce

pytestmark = pytest.mark.gpu
ACTS = ("linear", "relu", "sigmoid", "tanh", "silu", "gelu")


@pytest.fixture(scope="module")
def ctx():
    from zigneuron_amd import Context
    c = Context(0)
    yield c
    c.close()


def make(seed, batch, inp, hidden):
    rng = np.random.default_rng(seed)
    f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    return f(batch, inp), (f(inp, 2 * hidden) / np.float32(np.sqrt(inp))), f(2 * hidden), f(batch, 2 * hidden), f(batch, hidden)


def forward_ref(act, x, w, bias):
    """z, h and their bounds."""
    n = w.shape[1] // 2
    x, w = x.astype(np.float64), w.astype(np.float64)
    b = np.zeros(2 * n) if bias is None else bias.astype(np.float64)
    z = x @ w + b
    ez = dot_err(x.shape[1]) * (np.abs(x) @ np.abs(w)) + 2 * U * (np.abs(z) + np.abs(b))
    y, d = gate(act, z[:, :n])
    # the gate's argument is off by ez: at most the largest slope (1.13: GELU's) times that
    ey = gate_err(act, z[:, :n])[0] + 1.13 * 1.05 * ez[:, :n]
    h = y * z[:, n:]
    eh = ey * np.abs(z[:, n:]) + (np.abs(y) + ey) * ez[:, n:] + 2 * U * np.abs(h)
    return z, ez, h, eh


def run_forward(ctx, act, x, w, bias, keep=True):
    m, n = x.shape[0], w.shape[1] // 2
    dx, dw, db = ctx.to_device(x), ctx.to_device(w), None if bias is None else ctx.to_device(bias)
    z, h = ctx.alloc(m * 2 * n + 3).fill(7.0), ctx.alloc(m * n + 3).fill(7.0)
    ctx.gated_dense_forward(act, dx, dw, db, z if keep else None, h, m, x.shape[1], n)
    z, h = z.download(), h.download()
    assert (z[m * 2 * n if keep else 0:] == 7.0).all() and (h[m * n:] == 7.0).all()
    return z[:m * 2 * n].reshape(m, 2 * n), h[:m * n].reshape(m, n)


def backward_check(ctx, act, x, w, z, gh, bias, want_x=True, alias=False):
    m, k, n = x.shape[0], x.shape[1], w.shape[1] // 2
    d = [ctx.to_device(t) for t in (x, w, z, gh)]
    gz = d[2] if alias else ctx.alloc(z.size).fill(float("nan"))
    gx, gw = ctx.alloc(max(1, x.size)).fill(7.0), ctx.alloc(max(1, w.size)).fill(float("nan"))
    b0 = np.random.default_rng(1).standard_normal(2 * n).astype(np.float32)
    gb = ctx.to_device(b0) if bias else None
    ctx.gated_dense_backward(act, d[0], d[1], d[2], d[3], gz, gx if want_x else None, gw, gb, m, k, n)
    zz, g = z.astype(np.float64), gh.astype(np.float64)
    y, s = gate(act, zz[:, :n])
    ey, es = gate_err(act, zz[:, :n])
    ref = np.concatenate([g * zz[:, n:] * s, g * y], 1)
    err = np.concatenate([np.abs(g * zz[:, n:]) * es, np.abs(g) * ey], 1) + 3 * U * np.abs(ref)
    check(gz.download().reshape(ref.shape), ref, err, "grad_z")
    x8, w8 = x.astype(np.float64), w.astype(np.float64)
    if want_x:
        check(gx.download(x.size).reshape(x.shape), ref @ w8.T, (err + dot_err(2 * n) * np.abs(ref)) @ np.abs(w8).T, "grad_x")
    else:
        assert (gx.download() == 7.0).all()
    check(gw.download(w.size).reshape(w.shape), x8.T @ ref, np.abs(x8).T @ (err + dot_err(m) * np.abs(ref)), "grad_w")
    if bias:
        check(gb.download(), b0 + ref.sum(0), (err + dot_err(m) * np.abs(ref)).sum(0) + 2 * U * np.abs(b0), "grad_bias")


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("bias", [False, True])
def test_gates(ctx, act, bias):
    x, w, b, _, _ = make(1, 37, 53, 41)
    announce(f"gated forward {act} bias {bias}")
    z, ez, h, eh = forward_ref(act, x, w, b if bias else None)
    gz, gh = run_forward(ctx, act, x, w, b if bias else None)
    check(gz, z, ez, "z")
    check(gh, h, eh, "h")
    _, again = run_forward(ctx, act, x, w, b if bias else None, keep=False)
    check(again, h, eh, "h alone")


SIZES = [(1, 1, 1), (1, 64, 64), (1, 1023, 515), (2, 17, 3), (3, 300, 1001), (4, 1024, 4096), (5, 4, 128), (8, 515, 64),
         (9, 96, 130), (16, 1024, 512), (17, 33, 65), (31, 1000, 63), (64, 64, 64), (65, 65, 65), (100, 7, 200), (128, 512, 256),
         (129, 100, 127), (255, 300, 129), (300, 1001, 333), (1000, 64, 1000), (2048, 256, 512),
         (1, 4100, 400), (16, 2049, 1000), (7, 3001, 515), (2048, 1024, 1024), (1025, 130, 1030), (333, 257, 4099)]


@pytest.mark.parametrize("size", SIZES)
def test_forward_sizes(ctx, size):
    x, w, b, _, _ = make(sum(size), *size)
    for bias in (None, b):
        announce(f"gated forward {size} bias {bias is not None}")
        z, ez, h, eh = forward_ref("silu", x, w, bias)
        gz, gh = run_forward(ctx, "silu", x, w, bias)
        check(gz, z, ez, "z")
        check(gh, h, eh, "h")
        check(run_forward(ctx, "silu", x, w, bias, keep=False)[1], h, eh, "h alone")


@pytest.mark.parametrize("act", ACTS)
def test_backward_gates(ctx, act):
    x, w, _, z, gh = make(2, 45, 37, 51)
    z *= 3
    announce(f"gated backward {act}")
    backward_check(ctx, act, x, w, z, gh, True)
    backward_check(ctx, act, x, w, z, gh, False, want_x=False, alias=True)


@pytest.mark.parametrize("size", SIZES)
def test_backward_sizes(ctx, size):
    x, w, _, z, gh = make(sum(size) + 1, *size)
    announce(f"gated backward {size}")
    backward_check(ctx, "silu", x, w, z, gh, True)
    backward_check(ctx, "silu", x, w, z, gh, False)


def test_far_gates(ctx):
    """Gates far from zero, where an exponential or a square overflows: the limits, not NaN."""
    far = np.array([-1e30, -3e19, -200.0, -90.0, -20.0, 0.0, 20.0, 90.0, 200.0, 3e19, 1e30], np.float32)
    n = far.size
    z = np.stack([np.concatenate([far, np.full(n, 0.5, np.float32)])] * 2)
    x, w, gh = np.ones((2, 3), np.float32), np.ones((3, 2 * n), np.float32), np.full((2, n), 0.25, np.float32)
    for act in ("sigmoid", "tanh", "silu", "gelu"):
        announce(f"gated far {act}")
        d = [ctx.to_device(t) for t in (x, w, z, gh)]
        gz = ctx.alloc(z.size)
        ctx.gated_dense_backward(act, *d, gz, None, ctx.alloc(w.size), None, 2, 3, n)
        got = gz.download().reshape(z.shape)
        with np.errstate(over="ignore", invalid="ignore"):
            y, s = gate(act, far)
        s = np.where(np.isfinite(s), s, (far > 0).astype(float))  # 64-bit overflow of the same kind
        y = np.where(np.isfinite(y), y, np.maximum(far, 0))
        check(got[0, :n], 0.125 * s, 0.125 * (40 * U * (1 + np.abs(s)) + 1e-37), "slopes")
        check(got[0, n:], 0.25 * y, 0.25 * (120 * U * np.abs(y) + 1e-37), "values")


def test_infinities_stay_where_they_are(ctx):
    """A row of x with an infinity or NaN spoils its own row of z and h only."""
    x, w, b, _, _ = make(6, 200, 96, 160)
    z, ez, h, eh = forward_ref("silu", np.delete(x, 77, 0), w, b)
    x[77, 5] = np.nan
    gz, gh = run_forward(ctx, "silu", x, w, b)
    check(np.delete(gz, 77, 0), z, ez, "z")
    check(np.delete(gh, 77, 0), h, eh, "h")
    assert np.isnan(gz[77]).all()


def test_the_same_bits_each_time_and_in_a_graph(ctx):
    m, k, n = 192, 160, 224
    x, w, b, _, gh = make(8, m, k, n)
    d = [ctx.to_device(t) for t in (x, w, b, gh)]
    z, h, gz, gx, gw, gb = (ctx.alloc(s) for s in (m * 2 * n, m * n, m * 2 * n, m * k, k * 2 * n, 2 * n))
    zero = ctx.alloc(2 * n).fill(0.0)

    def step():
        ctx.gated_dense_forward("gelu", d[0], d[1], d[2], z, h, m, k, n)
        ctx.copy(gb.ptr, zero.ptr, 2 * n)
        ctx.gated_dense_backward("gelu", d[0], d[1], z, d[3], gz, gx, gw, gb, m, k, n)
        ctx.gated_dense_forward("gelu", d[0], d[1], d[2], None, h, m, k, n)

    announce("gated in a graph")
    step()
    first = [t.download() for t in (z, h, gz, gx, gw, gb)]
    graph = ctx.capture(step)
    for _ in range(3):
        for run in (graph.launch, step):
            for t in (z, h, gz, gx, gw, gb):
                t.fill(float("nan"))
            run()
            for t, want in zip((z, h, gz, gx, gw, gb), first):
                assert np.array_equal(t.download(), want)
    graph.close()


@pytest.mark.parametrize("size", [(5, 2000, 900), (200, 300, 260), (2048, 256, 512)])
def test_forced_launch_choices_hold_for_the_projections(ctx, size):
    """A forced tile or split is the projections' too: the result is the same layer's, within its bound."""
    x, w, b, _, _ = make(12, *size)
    z, ez, h, eh = forward_ref("gelu", x, w, b)
    try:
        for force in (lambda: ctx.set_gemm_tile("64x64"), lambda: ctx.set_gemm_splits(2), lambda: ctx.set_gemm_wave_split(4)):
            force()
            gz, gh = run_forward(ctx, "gelu", x, w, b)
            check(gz, z, ez, "z")
            check(gh, h, eh, "h")
            ctx.set_gemm_tile("auto")
            ctx.set_gemm_splits(0)
            ctx.set_gemm_wave_split(-1)
    finally:
        ctx.set_gemm_tile("auto")
        ctx.set_gemm_splits(0)
        ctx.set_gemm_wave_split(-1)


def test_empty_extents(ctx):
    t = ctx.alloc(64).fill(7.0)
    ctx.gated_dense_forward("silu", t, t, None, None, t, 0, 4, 4)
    ctx.gated_dense_forward("silu", t, t, None, None, t, 4, 4, 0)
    assert (t.download() == 7.0).all()
    x, b = ctx.alloc(1), ctx.to_device(np.array([2.0, 3.0, 5.0, 7.0], np.float32))
    h = ctx.alloc(4)
    ctx.gated_dense_forward("linear", x, x, b, None, h, 2, 0, 2)  # no inputs: the bias alone
    assert np.array_equal(h.download(), [10.0, 21.0, 10.0, 21.0])
    gw = ctx.alloc(24).fill(7.0)
    ctx.gated_dense_backward("silu", t, t, t, t, t, None, gw, None, 0, 3, 4)
    assert (gw.download() == 0.0).all()


def test_bad_calls_leave_an_error(ctx):
    from zigneuron_amd import InvalidArgumentError
    t = ctx.alloc(256)
    for args in (("silu", None, t, None, t, t, 2, 2, 2), ("silu", t, None, None, t, t, 2, 2, 2), ("silu", t, t, None, t, None, 2, 2, 2),
                 (6, t, t, None, t, t, 2, 2, 2), (-1, t, t, None, t, t, 2, 2, 2), ("silu", t, t, None, t, t, -1, 2, 2)):
        with pytest.raises(InvalidArgumentError):
            ctx.gated_dense_forward(*args)
    good = ["silu", t, t, t, t, t, t, t, None, 2, 2, 2]
    for i in (1, 2, 3, 4, 5, 7):
        with pytest.raises(InvalidArgumentError):
            ctx.gated_dense_backward(*good[:i], None, *good[i + 1:])
    with pytest.raises(InvalidArgumentError):
        ctx.gated_dense_forward("swish", t, t, None, t, t, 2, 2, 2)
