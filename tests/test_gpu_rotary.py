"""Rotary positions on the GPU (zn_hip_rotary_forward, zn_hip_rotary_backward) against 64 bits."""
from __future__ import annotations

import numpy as np
import pytest

from block_ops_ref import check
from gpu_common import announce
from paged_ref import Ints, Strided, U, frequencies, rotary

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    from zigneuron_amd import Context
    c = Context(0)
    yield c
    c.close()


def strides_of(shape, memory):
    b, h, s, d = shape
    return {"bhsd": (h * s * d, s * d, d), "bshd": (s * h * d, d, h * d), "gaps": (h * (s * (d + 3) + 5) + 7, s * (d + 3) + 5, d + 3)}[memory]


def run(ctx, x, rot, layout, positions=None, stride=None, scale=1.0, back=False, memory=("bhsd", "bhsd"), in_place=False, freq=None):
    b, h, s, d = x.shape
    f = frequencies(rot) if freq is None else freq
    dx = Strided(ctx, x, strides_of(x.shape, memory[0]))
    dy = dx if in_place else Strided(ctx, np.full(x.shape, np.nan, np.float32), strides_of(x.shape, memory[1]))
    df = ctx.to_device(f) if rot else None
    dp = None if positions is None else Ints(ctx, positions)
    call = ctx.rotary_backward if back else ctx.rotary_forward
    call(dx.ptr, dy.ptr, df, b, h, s, d, rot, layout, None if dp is None else dp.ptr, stride, scale, dx.strides, dy.strides)
    return dy.read()


def expect(x, rot, layout, positions=None, stride=None, scale=1.0, back=False, freq=None):
    b, h, s, d = x.shape
    p = np.broadcast_to(np.arange(s), (b, s)) if positions is None else np.stack(
        [np.ravel(positions)[n * (s if stride is None else stride):][:s] for n in range(b)])
    return rotary(x, p[:, None], frequencies(rot) if freq is None else freq, rot, layout, scale, back)


SHAPES = [  # batch, heads, length, dim, rot
    (1, 1, 1, 1, 0), (1, 1, 1, 2, 2), (1, 1, 1, 64, 64), (2, 3, 5, 7, 6), (1, 2, 3, 9, 2), (3, 5, 17, 76, 38), (2, 4, 33, 64, 32),
    (1, 40, 9, 128, 128), (64, 20, 1, 64, 64), (1, 1, 300, 127, 126), (2, 7, 65, 80, 20), (1, 3, 31, 1024, 1024), (1, 2, 5, 1023, 2),
    (5, 33, 3, 96, 90), (1, 300, 2, 32, 32), (1, 1, 4097, 40, 40),
]


@pytest.mark.parametrize("back", [False, True])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("shape", SHAPES)
def test_against_64_bits(ctx, shape, layout, back):
    announce(f"rotary {shape} {layout} back {back}")
    rng = np.random.default_rng(sum(shape))
    x = rng.standard_normal(shape[:4]).astype(np.float32)
    ref, bound = expect(x, shape[4], layout, back=back)
    check(run(ctx, x, shape[4], layout, back=back), ref, bound, "y")


@pytest.mark.parametrize("memory", [("bshd", "bhsd"), ("gaps", "bshd"), ("bhsd", "gaps")])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_strides_and_scale(ctx, layout, memory):
    announce(f"rotary {layout} {memory}")
    x = np.random.default_rng(3).standard_normal((3, 4, 21, 52)).astype(np.float32)
    ref, bound = expect(x, 44, layout, scale=1.25)
    check(run(ctx, x, 44, layout, scale=1.25, memory=memory), ref, bound, "y")


@pytest.mark.parametrize("memory", ["bshd", "gaps"])
@pytest.mark.parametrize("back", [False, True])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_in_place(ctx, layout, back, memory):
    announce(f"rotary in place {layout} {memory} back {back}")
    x = np.random.default_rng(4).standard_normal((2, 6, 19, 45)).astype(np.float32)
    ref, bound = expect(x, 26, layout, back=back)
    got = run(ctx, x, 26, layout, back=back, memory=(memory, memory), in_place=True)
    check(got, ref, bound, "y")
    assert np.array_equal(got[..., 26:], x[..., 26:])
    assert np.array_equal(got, run(ctx, x, 26, layout, back=back))


@pytest.mark.parametrize("stride", [None, 0, 50])
def test_positions(ctx, stride):
    """Near, far, negative and equal positions; of each sequence, shared, and in rows of a longer array."""
    announce(f"rotary positions, stride {stride}")
    rng = np.random.default_rng(9)
    b, s = 3, 40
    pos = rng.integers(-1000, 2 ** 29, (b, 50 if stride == 50 else s)).astype(np.int32)
    pos[:, :6] = [0, 1, -1, 2 ** 29 - 1, -(2 ** 29), 131072]
    pos[:, 6] = pos[:, 7]
    x = rng.standard_normal((b, 2, s, 32)).astype(np.float32)
    ref, bound = expect(x, 32, "half", pos, stride)
    got = run(ctx, x, 32, "half", pos, stride)
    check(got, ref, bound, "y")
    # the turn keeps a pair's length
    n = np.hypot(x[..., :16].astype(np.float64), x[..., 16:])
    assert np.all(np.abs(np.hypot(got[..., :16].astype(np.float64), got[..., 16:]) - n) <= 16 * U * (np.abs(x[..., :16]) + np.abs(x[..., 16:])))


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_far_and_fast(ctx, layout):
    """Positions to both ends of 32 bits and frequencies far above 1: the angle, a product of 55 bits, passes 2^43, its quarter
    turns pass 32 bits.  The reference has it exactly (80-bit floats), so the bound has no term of the angle: 8 U as for near ones."""
    announce(f"rotary, far and fast {layout}")
    assert np.finfo(np.longdouble).nmant >= 63
    rng = np.random.default_rng(10)
    pos = np.concatenate([[0, 1, -1, 2 ** 31 - 1, -(2 ** 31), 2 ** 31 - 2, 2 ** 30 + 1], rng.integers(-(2 ** 31), 2 ** 31, 57)]).astype(np.int32)
    freq = np.array([1, 0.99999994, 1.5707964, 3.0, 7.7, 100.3, 1e-4, 4097.123], np.float32)
    x = rng.standard_normal((1, 2, pos.size, 16)).astype(np.float32)
    a = pos.astype(np.longdouble)[:, None] * freq.astype(np.longdouble)
    s, c = np.sin(a).astype(np.float64), np.cos(a).astype(np.float64)
    one, two = (slice(0, 8), slice(8, 16)) if layout == "half" else (slice(0, 16, 2), slice(1, 16, 2))
    p, q = x[..., one].astype(np.float64), x[..., two].astype(np.float64)
    ref, bound = np.empty(x.shape), np.empty(x.shape)
    ref[..., one], ref[..., two] = p * c - q * s, p * s + q * c
    bound[..., one] = bound[..., two] = 8 * U * (np.abs(p) + np.abs(q))
    check(run(ctx, x, 16, layout, pos, freq=freq), ref, bound, "y")


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_gradient_against_differences(ctx, layout):
    """The turn is linear: its difference quotient along h is its value at h, and <g, f(h)> = <f'(g), h>."""
    announce(f"rotary gradient {layout}")
    rng = np.random.default_rng(12)
    shape, rot = (2, 3, 50, 64), 48
    pos = rng.integers(0, 100000, (2, 50)).astype(np.int32)
    x, h, g = (rng.standard_normal(shape).astype(np.float32) for _ in range(3))
    fh = run(ctx, h, rot, layout, pos, scale=0.7)
    diff = (run(ctx, x + h, rot, layout, pos, scale=0.7).astype(np.float64) - run(ctx, x, rot, layout, pos, scale=0.7))
    _, b1 = expect(x + h, rot, layout, pos, scale=0.7)
    _, b2 = expect(x, rot, layout, pos, scale=0.7)
    _, b3 = expect(h, rot, layout, pos, scale=0.7)
    exact_h = (x + h).astype(np.float64) - x  # what x + h is in fp32
    d, _ = expect(exact_h, rot, layout, pos, scale=0.7)
    assert np.all(np.abs(diff - d) <= b1 + b2 + 1e-30)
    back = run(ctx, g, rot, layout, pos, scale=0.7, back=True)
    _, b4 = expect(g, rot, layout, pos, scale=0.7, back=True)
    left, right = (g.astype(np.float64) * fh).sum(), (back.astype(np.float64) * h).sum()
    assert abs(left - right) <= (np.abs(g) * b3).sum() + (np.abs(h) * b4).sum()


def test_scaled_frequencies(ctx):
    import zigneuron_amd as zn
    announce("rotary scaled")
    x = np.random.default_rng(2).standard_normal((1, 2, 64, 64)).astype(np.float32)
    pos = np.arange(100000, 100064, dtype=np.int32)
    for kind in ("linear", "base", "turns", "pairs"):
        f = zn.rotary_frequencies(64, 500000.0, kind, 8.0, 8192, 1, 4)
        ref, bound = expect(x, 64, "half", pos, freq=f, scale=1.2)
        check(run(ctx, x, 64, "half", pos, freq=f, scale=1.2), ref, bound, kind)


def test_untouched_dims_keep_their_bits(ctx):
    announce("rotary: dims past rot")
    x = np.random.default_rng(1).standard_normal((1, 2, 3, 20)).astype(np.float32)
    x[..., 8], x[..., 9], x[..., 10] = np.nan, np.inf, -0.0
    got = run(ctx, x, 8, "interleaved", scale=3.0)
    assert np.array_equal(got[..., 8:].view(np.uint32), x[..., 8:].view(np.uint32))


def test_captured_and_replayed(ctx):
    """A replay reads the positions of its time."""
    announce("rotary graph")
    x = np.random.default_rng(6).standard_normal((4, 3, 2, 48)).astype(np.float32)
    dx, dy, df = ctx.to_device(x), ctx.alloc(x.size), ctx.to_device(frequencies(48))
    pos = Ints(ctx, np.zeros((4, 2)))
    call = lambda: ctx.rotary_forward(dx, dy, df, 4, 3, 2, 48, 48, "half", pos.ptr)  # noqa: E731
    call()
    graph = ctx.capture(call)
    for step in range(4):
        p = np.arange(8).reshape(4, 2) * 1000 + step
        pos.set(p)
        dy.fill(float("nan"))
        graph.launch()
        ref, bound = expect(x, 48, "half", p)
        check(dy.download().reshape(x.shape), ref, bound, f"replay {step}")


def test_on_another_stream_of_the_device(ctx):
    """Two contexts, a stream each, at the same time."""
    from zigneuron_amd import Context
    announce("rotary, two contexts")
    x = np.random.default_rng(8).standard_normal((2, 8, 100, 64)).astype(np.float32)
    with Context(0) as other:
        a, b = (run(c, x, 64, "half") for c in (ctx, other))
    assert np.array_equal(a, b)
