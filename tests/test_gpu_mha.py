"""Grouped attention on the GPU (zn_hip_mha_forward, zn_hip_mha_backward) against 64 bits."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from block_ops_ref import Mha, check
from gpu_common import announce

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    from zigneuron_amd import Context
    c = Context(0)
    yield c
    c.close()


class Ints:
    """An int32 device array."""

    def __init__(self, ctx, values):
        v = np.ascontiguousarray(values, np.int32)
        self.buf = ctx.to_device(v.view(np.float32))

    @property
    def ptr(self):
        return self.buf.ptr


class Placed:
    """A [batch, heads, positions, dim] tensor inside a larger device buffer, at the strides of a layout."""

    def __init__(self, ctx, values, layout="bhsd", base=None, at=0):
        b, h, s, d = values.shape
        self.shape, self.values = values.shape, np.asarray(values, np.float32)
        if layout == "bhsd":
            self.strides = (h * s * d, s * d, d)
        elif layout == "bshd":
            self.strides = (s * h * d, d, h * d)
        else:  # gaps: rows of d + 3, heads and sequences further apart than they need
            self.strides = (h * (s * (d + 3) + 5) + 7, s * (d + 3) + 5, d + 3)
        self.size = 1 + (b - 1) * self.strides[0] + (h - 1) * self.strides[1] + (s - 1) * self.strides[2] + d - 1 if b * h * s else 1
        host = np.full(self.size, 777.0, np.float32)
        self.index = (np.arange(b)[:, None, None, None] * self.strides[0] + np.arange(h)[:, None, None] * self.strides[1] +
                      np.arange(s)[:, None] * self.strides[2] + np.arange(d))
        host[self.index] = self.values
        self.host = host
        self.buf = ctx.to_device(host)

    def read(self):
        """The tensor, after checking that nothing between its rows was written."""
        now = self.buf.download()
        keep = np.ones(now.size, bool)
        keep[self.index] = False
        assert np.array_equal(now[keep], self.host[keep]), "written outside the tensor"
        return now[self.index]


def make(seed, b, hq, hk, sq, sk, d):
    rng = np.random.default_rng(seed)
    f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    return f(b, hq, sq, d), f(b, hk, sk, d), f(b, hk, sk, d), f(b, hq, sq, d)


def run_forward(ctx, q, k, v, scale, causal=False, q_lens=None, kv_lens=None, layout="bhsd", lse=True):
    b, hq, sq, d = q.shape
    hk, sk = k.shape[1:3]
    pq, pk, pv = (Placed(ctx, t, layout) for t in (q, k, v))
    po = Placed(ctx, np.full(q.shape, np.nan, np.float32), layout)
    pl = ctx.alloc(b * hq * sq).fill(float("nan"))
    lens = [None if t is None else Ints(ctx, t) for t in (q_lens, kv_lens)]
    ctx.mha_forward(pq.buf, pk.buf, pv.buf, po.buf, pl if lse else None, b, hq, hk, sq, sk, d, scale, causal,
                    *(None if t is None else t.ptr for t in lens), pq.strides, pk.strides, po.strides)
    return po.read(), pl.download(b * hq * sq).reshape(b, hq, sq)


def run_backward(ctx, q, k, v, out, lse, g, scale, causal=False, q_lens=None, kv_lens=None, layout="bhsd"):
    b, hq, sq, d = q.shape
    hk, sk = k.shape[1:3]
    pq, pk, pv, po, pg = (Placed(ctx, t, layout) for t in (q, k, v, out, g))
    pl = ctx.to_device(lse)
    gq, gk, gv = (Placed(ctx, np.full(t.shape, np.nan, np.float32), layout) for t in (q, k, v))
    lens = [None if t is None else Ints(ctx, t) for t in (q_lens, kv_lens)]
    ctx.mha_backward(pq.buf, pk.buf, pv.buf, po.buf, pl, pg.buf, gq.buf, gk.buf, gv.buf, b, hq, hk, sq, sk, d, scale, causal,
                     *(None if t is None else t.ptr for t in lens), pq.strides, pk.strides, po.strides)
    return gq.read(), gk.read(), gv.read()


def both(ctx, q, k, v, g, scale, causal, q_lens=None, kv_lens=None, layout="bhsd", what=""):
    announce(f"mha {what or q.shape} kv {k.shape} causal {causal} lens {q_lens} {kv_lens} {layout}")
    ref = Mha(q, k, v, scale, causal, q_lens, kv_lens)
    out, lse = run_forward(ctx, q, k, v, scale, causal, q_lens, kv_lens, layout)
    check(out, ref.out, ref.out_bound, "out")
    check(lse, ref.lse, ref.lse_bound, "lse")
    # the backward is held to the reference given the forward's own results
    grads, bounds = ref.backward(g, out, lse)
    got = run_backward(ctx, q, k, v, out, lse, g, scale, causal, q_lens, kv_lens, layout)
    for name, x, r, e in zip(("grad_q", "grad_k", "grad_v"), got, grads, bounds):
        check(x, r, e, name)


SHAPES = [
    # batch, q heads, kv heads, q_len, kv_len, dim
    (1, 1, 1, 1, 1, 1), (1, 1, 1, 1, 1, 64), (2, 2, 1, 1, 37, 16), (1, 2, 2, 5, 3, 7), (1, 2, 1, 3, 9, 33),
    (2, 4, 2, 31, 31, 32), (1, 3, 1, 32, 33, 31), (1, 2, 2, 33, 65, 64), (2, 6, 2, 64, 64, 40), (1, 4, 4, 65, 63, 65),
    (1, 2, 1, 127, 129, 96), (1, 2, 2, 128, 128, 128), (1, 7, 1, 100, 100, 76), (1, 1, 1, 257, 300, 127),
    (2, 2, 1, 300, 257, 80), (1, 8, 2, 1, 513, 64), (3, 2, 1, 17, 700, 128), (1, 1, 1, 640, 640, 64), (16, 4, 4, 64, 64, 64),
    # few rows of a long cache, long walks of few tiles, tiles that read split images
    (1, 1, 1, 1, 5000, 96), (2, 8, 1, 2, 2049, 128), (1, 5, 1, 3, 999, 50), (1, 1, 1, 2000, 40, 32), (1, 1, 1, 40, 2000, 96),
    (1, 3, 1, 1000, 1000, 128),
]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_against_64_bits(ctx, shape, causal):
    b, hq, hk, sq, sk, d = shape
    q, k, v, g = make(sum(shape), *shape)
    both(ctx, q, k, v, g, 1 / np.sqrt(d), causal)


@pytest.mark.parametrize("layout", ["bshd", "gaps"])
@pytest.mark.parametrize("shape", [(2, 4, 2, 70, 70, 64), (1, 2, 2, 130, 37, 30), (2, 2, 1, 33, 200, 128)])
def test_strides(ctx, shape, layout):
    q, k, v, g = make(7, *shape)
    both(ctx, q, k, v, g, 0.2, True, layout=layout)


def test_one_projection_holds_all(ctx):
    """q, k, v (and their gradients) as heads of one [batch, positions, heads, dim] tensor."""
    b, hq, hk, s, d = 2, 6, 2, 75, 36
    rng = np.random.default_rng(5)
    x = rng.standard_normal((b, s, hq + 2 * hk, d)).astype(np.float32)
    g = rng.standard_normal((b, s, hq, d)).astype(np.float32)
    q, k, v = (np.ascontiguousarray(t.transpose(0, 2, 1, 3)) for t in (x[:, :, :hq], x[:, :, hq:hq + hk], x[:, :, hq + hk:]))
    n = (hq + 2 * hk) * d
    st, so = (s * n, d, n), (s * hq * d, d, hq * d)
    dx, dg, do, dl = ctx.to_device(x), ctx.to_device(g), ctx.alloc(b * s * hq * d), ctx.alloc(b * hq * s)
    gx = ctx.alloc(x.size).fill(float("nan"))
    at = (0, hq * d, (hq + hk) * d)
    shape = (b, hq, hk, s, s, d, 0.15, True, None, None, st, st, so)
    announce("mha on one projection's output")
    ctx.mha_forward(*(dx.offset(o) for o in at), do, dl, *shape)
    ctx.mha_backward(*(dx.offset(o) for o in at), do, dl, dg, *(gx.offset(o) for o in at), *shape)
    ref = Mha(q, k, v, 0.15, True)
    out = do.download().reshape(b, s, hq, d).transpose(0, 2, 1, 3)
    lse = dl.download().reshape(b, hq, s)
    check(out, ref.out, ref.out_bound, "out")
    grads, bounds = ref.backward(g.transpose(0, 2, 1, 3), out, lse)
    got = gx.download().reshape(x.shape).transpose(0, 2, 1, 3)
    for name, x1, r, e in zip(("grad_q", "grad_k", "grad_v"), (got[:, :hq], got[:, hq:hq + hk], got[:, hq + hk:]), grads, bounds):
        check(x1, r, e, name)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dim", [32, 64, 100])
def test_lengths_and_padding_that_holds_anything(ctx, causal, dim):
    """Lengths of 0, 1 and more, past the tensor and negative ones; infinities and NaN in the padding."""
    q_lens, kv_lens = [0, 1, 50, 90, 1000, -3, 70], [5, 1, 90, 0, 1000, 90, 33]
    shape = (7, 4, 2, 90, 90, dim)
    q, k, v, g = make(11, *shape)
    for n in range(7):
        ql, kl = (min(max(t[n], 0), 90) for t in (q_lens, kv_lens))
        q[n, :, ql:], g[n, :, ql:] = np.nan, np.inf
        k[n, :, kl:], v[n, :, kl:] = -np.inf, np.nan
    both(ctx, q, k, v, g, 1 / np.sqrt(dim), causal, q_lens, kv_lens, what="padding")


@pytest.mark.parametrize("sq,sk", [(40, 8), (200, 130), (70, 1), (64, 0), (3, 64)])
def test_queries_that_see_nothing(ctx, sq, sk):
    q, k, v, g = make(3, 1, 4, 2, sq, sk, 48)
    hidden = max(0, sq - sk)
    g[:, :, :hidden], q[:, :, :hidden] = np.nan, np.inf  # nothing comes from these rows
    both(ctx, q, k, v, g, 0.1, True, what="empty rows")


@pytest.mark.parametrize("s,bad", [(150, 101), (700, 555)])
@pytest.mark.parametrize("dim", [64, 128])
def test_masked_values_reach_nothing(ctx, dim, s, bad):
    """A causal mask beside NaN, infinities and the lowest value: only queries that see them may have them."""
    b, hq, hk = 1, 2, 1
    q, k, v, g = make(13, b, hq, hk, s, s, dim)
    # queries from `bad` on see a NaN key, so they and the gradients that they feed are NaN
    k2, v2 = k.copy(), v.copy()
    k2[:, :, bad:], v2[:, :, bad:] = np.nan, np.inf
    v2[:, :, bad + 1:] = np.finfo(np.float32).min
    ref = Mha(q[:, :, :bad], k[:, :, :bad], v[:, :, :bad], 0.1, True)
    announce(f"mha masked NaN, dim {dim}")
    out, lse = run_forward(ctx, q, k2, v2, 0.1, True)
    check(out[:, :, :bad], ref.out, ref.out_bound, "out")
    check(lse[:, :, :bad], ref.lse, ref.lse_bound, "lse")
    assert np.isnan(out[:, :, bad:]).all()
    grads, _ = ref.backward(g[:, :, :bad], out[:, :, :bad], lse[:, :, :bad])
    _, bounds = ref.backward(g[:, :, :bad], out[:, :, :bad], lse[:, :, :bad])
    gq, gk, gv = run_backward(ctx, q, k2, v2, out, lse, g, 0.1, True)
    check(gq[:, :, :bad], grads[0], bounds[0], "grad_q")
    assert np.isnan(gq[:, :, bad:]).all() and np.isnan(gk).all() and np.isnan(gv).all()


@pytest.mark.parametrize("shape, causal, layout", [((16, 16, 16, 500, 200, 100), True, "bhsd"), ((16, 32, 16, 400, 160, 70), False, "bshd")])
def test_many_heads_past_64_dims(ctx, shape, causal, layout):
    """Enough heads for the widest tiles; lengths from nothing to all, padding that holds anything."""
    b, hq, hk, sq, sk, d = shape
    q, k, v, _ = make(48, *shape)
    q_lens, kv_lens = [sq - 31 * n for n in range(b)], [(17 * n) % (sk + 1) if n else sk for n in range(b)]
    for n in range(b):
        q[n, :, q_lens[n]:], k[n, :, kv_lens[n]:], v[n, :, kv_lens[n]:] = np.nan, np.inf, np.nan
    announce(f"mha {shape} causal {causal} {layout}")
    ref = Mha(q, k, v, d ** -0.5, causal, q_lens, kv_lens)
    if causal:  # an infinity that the last query of one head alone sees, beside others of its tile that do not
        v[0, 3, sk - 1] = np.inf
        ref.out[0, 3, sq - 1] = np.inf
    out, lse = run_forward(ctx, q, k, v, d ** -0.5, causal, q_lens, kv_lens, layout)
    check(out, ref.out, ref.out_bound, "out")
    check(lse, ref.lse, ref.lse_bound, "lse")


@pytest.mark.parametrize("causal", [False, True])
def test_new_tokens_of_sequences_of_all_lengths(ctx, causal):
    """One or two new tokens a sequence, caches from nothing to long, padding that holds anything."""
    q_lens, kv_lens = [1, 2, 0, 2, 1, 2], [5, 0, 7, 900, 1024, 1]
    shape = (6, 6, 2, 2, 1024, 64)
    q, k, v, g = make(47, *shape)
    for n in range(6):
        q[n, :, q_lens[n]:], g[n, :, q_lens[n]:] = np.nan, np.inf
        k[n, :, kv_lens[n]:], v[n, :, kv_lens[n]:] = np.inf, np.nan
        hidden = max(0, q_lens[n] - kv_lens[n]) if causal else (q_lens[n] if kv_lens[n] == 0 else 0)
        g[n, :, :hidden] = np.nan
    both(ctx, q, k, v, g, 0.125, causal, q_lens, kv_lens, what="new tokens")


@pytest.mark.parametrize("dim", [24, 64, 96, 128])
def test_a_few_rows_beside_a_masked_nan(ctx, dim):
    """Four new tokens against a long cache whose last keys only the last of them see."""
    shape = (2, 4, 2, 4, 1500, dim)
    q, k, v, _ = make(43, *shape)
    ref = Mha(q, k, v, 0.1, True)
    v[:, :, -2:] = np.nan  # the last two queries'
    k[:, :, -1:] = np.inf
    announce(f"mha few rows beside NaN, dim {dim}")
    out, lse = run_forward(ctx, q, k, v, 0.1, True)
    check(out[:, :, :2], ref.out[:, :, :2], ref.out_bound[:, :, :2], "out")
    check(lse[:, :, :2], ref.lse[:, :, :2], ref.lse_bound[:, :, :2], "lse")
    assert np.isnan(out[:, :, 2:]).all()


@pytest.mark.parametrize("dim", [16, 64, 128])
def test_large_and_tiny_scores(ctx, dim):
    """Scores so large that one key takes all, values near fp32's ends, a negative and a zero scale."""
    q, k, v, g = make(17, 1, 2, 1, 70, 70, dim)
    both(ctx, q * 30, k * 30, v, g, 1.0, True, what="large scores")
    both(ctx, q, k, v, g, -0.3, False, what="negative scale")
    both(ctx, q, k, v, g, 0.0, False, what="zero scale")
    both(ctx, q * np.float32(1e-20), k, v * np.float32(1e30), g * np.float32(1e-35), 0.1, True, what="tiny and large")


def test_values_past_the_split(ctx):
    """Magnitudes whose scaled parts overflow: the rows are done again in plain fp32."""
    q, k, v, g = make(19, 1, 2, 2, 40, 40, 64)
    v[:, :, 3] *= np.float32(1e33)
    both(ctx, q, k, v, g, 0.1, True, what="past the split")


def test_the_same_bits_each_time_and_in_a_graph(ctx):
    b, hq, hk, s, d = 2, 4, 2, 200, 64
    q, k, v, g = make(23, b, hq, hk, s, s, d)
    dq, dk, dv, dg = (ctx.to_device(t) for t in (q, k, v, g))
    o, l = ctx.alloc(q.size), ctx.alloc(b * hq * s)
    grads = [ctx.alloc(t.size) for t in (q, k, v)]
    shape = (b, hq, hk, s, s, d, 0.125, True)

    def step():
        ctx.mha_forward(dq, dk, dv, o, l, *shape)
        ctx.mha_backward(dq, dk, dv, o, l, dg, *grads, *shape)

    def clear():
        for t in (o, l, *grads):
            t.fill(float("nan"))

    def read():
        return [t.download() for t in (o, l, *grads)]

    announce("mha in a graph")
    step()
    first = read()
    graph, second = ctx.capture(step), ctx.capture(step)  # two graphs of one context
    for turn in range(4):
        clear()
        (graph, second)[turn % 2].launch()
        for x, y in zip(read(), first):
            assert np.array_equal(x, y)
        clear()
        step()  # an eager step between the replays
        for x, y in zip(read(), first):
            assert np.array_equal(x, y)
    graph.close()
    second.close()


def test_two_contexts_at_once(ctx):
    """Two contexts (two streams) at work on the same inputs."""
    from zigneuron_amd import Context
    shape = (2, 4, 4, 300, 300, 64)
    q, k, v, g = make(29, *shape)
    with Context(0) as other:
        res = []
        pair = []
        for c in (ctx, other):
            t = [c.to_device(x) for x in (q, k, v, g)]
            o, l = c.alloc(q.size), c.alloc(2 * 4 * 300)
            pair.append((c, t, o, l, [c.alloc(x.size) for x in (q, k, v)]))
        announce("mha on two contexts")
        for _ in range(3):
            for c, t, o, l, gr in pair:
                c.mha_forward(*t[:3], o, l, *shape, 0.125, True)
                c.mha_backward(*t[:3], o, l, t[3], *gr, *shape, 0.125, True)
        for c, t, o, l, gr in pair:
            res.append([x.download() for x in (o, l, *gr)])
        for x, y in zip(*res):
            assert np.array_equal(x, y)


def test_differences(ctx):
    """The gradient against central differences of the reference's loss."""
    b, hq, hk, sq, sk, d = 1, 2, 1, 6, 9, 8
    q, k, v, g = make(31, b, hq, hk, sq, sk, d)
    out, lse = run_forward(ctx, q, k, v, 0.4, True)
    got = run_backward(ctx, q, k, v, out, lse, g, 0.4, True)
    step = 1e-5

    def loss(a, b_, c):
        return (Mha(a, b_, c, 0.4, True).out * g).sum()

    for which, grad in enumerate(got):
        t = [x.astype(np.float64) for x in (q, k, v)]
        num = np.zeros(grad.shape)
        for at in np.ndindex(grad.shape):
            keep = t[which][at]
            t[which][at] = keep + step
            up = loss(*t)
            t[which][at] = keep - step
            num[at] = (up - loss(*t)) / (2 * step)
            t[which][at] = keep
        # differences: step^2 of a third derivative of order one and 1e-16 / step; fp32: a few hundred of its half steps
        assert np.abs(num - grad).max() < 1e-5 * max(1.0, np.abs(num).max())


def test_no_log_sum_exp_wanted(ctx):
    q, k, v, _ = make(37, 1, 2, 2, 50, 50, 64)
    a, _ = run_forward(ctx, q, k, v, 0.125)
    b, lse = run_forward(ctx, q, k, v, 0.125, lse=False)
    assert np.array_equal(a, b) and np.isnan(lse).all()


def test_far_rows(ctx):
    """Positions a stride of 2^22 apart: offsets past 32 bits."""
    s, d, far = 300, 16, 1 << 22
    rng = np.random.default_rng(41)
    k, v = (rng.standard_normal((1, 1, s, d)).astype(np.float32) for _ in range(2))
    q = rng.standard_normal((1, 1, 1, d)).astype(np.float32)
    big = ctx.alloc((s - 1) * far + 2 * d)  # 5 GB; k and v side by side in each row
    rows = np.concatenate([k, v], -1)[0, 0]
    from zigneuron_amd import _lib
    for i in range(s):
        row = np.ascontiguousarray(rows[i])
        _lib.check(_lib.load().zn_hip_h2d(ctx.handle, big.offset(i * far), row.ctypes.data, row.nbytes), "h2d")
    dq, do = ctx.to_device(q), ctx.alloc(d)
    announce("mha with far rows")
    ctx.mha_forward(dq, big.offset(0), big.offset(d), do, None, 1, 1, 1, 1, s, d, 0.25, kv_strides=(0, 0, far))
    got = do.download().reshape(q.shape)
    big.close()
    ref = Mha(q, k, v, 0.25)
    check(got, ref.out, ref.out_bound, "out")


def test_keys_without_queries_have_no_gradient(ctx):
    t = ctx.to_device(np.ones(2 * 3 * 5 * 8, np.float32))
    for hq, sq in ((0, 4), (2, 0)):
        gk, gv = (ctx.alloc(2 * 2 * 5 * 8).fill(7.0) for _ in range(2))
        ctx.mha_backward(t, t, t, t, t, t, t, gk, gv, 2, hq, 2, sq, 5, 8, 1.0)
        assert (gk.download() == 0).all() and (gv.download() == 0).all()


def test_bad_calls_leave_an_error(ctx):
    from zigneuron_amd import InvalidArgumentError
    t = ctx.alloc(4096)
    call = lambda **kw: ctx.mha_forward(*[kw.pop(x, t) for x in ("q", "k", "v", "out", "lse")],  # noqa: E731
                                        *[kw.pop(x, y) for x, y in (("batch", 1), ("q_heads", 2), ("kv_heads", 2), ("q_len", 4),
                                                                    ("kv_len", 4), ("head_dim", 8), ("scale", 1.0))], **kw)
    for bad in ({"q": None}, {"k": None}, {"v": None}, {"out": None}, {"head_dim": 0}, {"head_dim": 129}, {"q_heads": 3},
                {"kv_heads": 0}, {"scale": float("nan")}, {"causal": 2}, {"batch": -1}, {"kv_strides": (32, 32, 7)},
                {"out_strides": (32, 0, 8)}, {"q_strides": (32, -1, 8)}, {"q_strides": (0, 0, (1 << 22) + 1)}):
        with pytest.raises(InvalidArgumentError):
            call(**bad)
    call(batch=0)
    call(q_len=0)
    call(q_heads=0, kv_heads=0)
