"""Distillation from a teacher's top logits on the GPU (zn_hip_distill_forward and _backward) against 64 bits."""
from __future__ import annotations

import numpy as np
import pytest

from block_ops_ref import Distill, check
from gpu_common import announce

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    from zigneuron_amd import Context
    c = Context(0)
    yield c
    c.close()


def make(seed, rows, vocab, k):
    rng = np.random.default_rng(seed)
    logits = (rng.standard_normal((rows, vocab)) * 3).astype(np.float32)
    index = np.stack([rng.permutation(vocab)[:k] for _ in range(rows)]).astype(np.int32).reshape(rows, k)
    top = (rng.standard_normal((rows, k)) * 3).astype(np.float32)
    return logits, index, top, rng.random(rows).astype(np.float32)


def run(ctx, logits, index, top, grad_loss, t, ld=None, alias=False, grad_ld=None):
    """(loss, lse, grad_logits); the columns past the vocabulary have to stay."""
    rows, vocab = logits.shape
    k = index.shape[1]
    ld = ld or vocab
    gld = grad_ld or ld
    host = np.full((rows, ld), 5.0, np.float32)
    host[:, :vocab] = logits
    dl, dt = ctx.to_device(host), ctx.to_device(np.concatenate([top.ravel(), [0]]))
    di = ctx.to_device(np.concatenate([index.ravel(), [0]]).astype(np.int32).view(np.float32))
    dg = ctx.to_device(grad_loss)
    loss, lse = ctx.alloc(rows + 1).fill(9.0), ctx.alloc(rows + 1).fill(9.0)
    grad = dl if alias else ctx.alloc(rows * gld).fill(5.0)
    ctx.distill_forward(dl, ld, di, dt, loss, lse, rows, vocab, k, t)
    ctx.distill_backward(dl, ld, di, dt, lse, dg, grad, gld, rows, vocab, k, t)
    loss, lse, grad = loss.download(), lse.download(), grad.download(rows * gld).reshape(rows, gld)
    assert loss[rows] == 9.0 and lse[rows] == 9.0 and (grad[:, vocab:] == 5.0).all()
    return loss[:rows], lse[:rows], grad[:, :vocab]


def both(ctx, logits, index, top, grad_loss, t, **kw):
    announce(f"distill {logits.shape} k {index.shape[1]} T {t} {kw}")
    ref = Distill(logits, index, top, t)
    loss, lse, grad = run(ctx, logits, index, top, grad_loss, t, **kw)
    check(loss, ref.loss, ref.loss_bound, "loss")
    check(lse, ref.lse, ref.lse_bound, "lse")
    g, bound = ref.backward(grad_loss, lse)
    check(grad, g, bound, "grad_logits")


@pytest.mark.parametrize("t", [1.0, 2.0, 0.7])
@pytest.mark.parametrize("shape", [(1, 1, 1), (1, 2, 1), (3, 5, 5), (2, 255, 4), (5, 256, 100), (4, 1023, 64), (7, 4097, 3),
                                   (1, 32000, 20), (1, 131072, 64), (2, 50257, 257), (300, 1000, 10), (2, 5000, 1024),
                                   (3, 70001, 1), (2100, 130, 7)])
def test_against_64_bits(ctx, shape, t):
    both(ctx, *make(sum(shape), *shape), t)


@pytest.mark.parametrize("vocab,ld", [(100, 101), (4096, 4099), (9001, 9100)])
def test_row_strides_and_in_place(ctx, vocab, ld):
    a = make(vocab, 6, vocab, 9)
    both(ctx, *a, 2.0, ld=ld)
    both(ctx, *a, 2.0, ld=ld, alias=True)
    both(ctx, *a, 2.0, ld=ld, grad_ld=ld + 2)


@pytest.mark.parametrize("vocab", [300, 40000])
def test_absent_entries_and_empty_rows(ctx, vocab):
    """Indices outside the vocabulary, logits of -inf and the lowest value, rows that have nothing."""
    logits, index, top, g = make(5, 8, vocab, 40)
    index[0] = -1
    index[1, 3:] = vocab
    top[2] = -np.inf
    top[3, ::2] = -np.inf
    top[4, 1:] = np.finfo(np.float32).min
    index[5, :20] = -7
    index[6, 39] = np.iinfo(np.int32).max
    index[7] = np.iinfo(np.int32).min
    logits[0], logits[2], logits[7] = np.nan, np.inf, -np.inf  # never read
    ref = Distill(np.nan_to_num(logits, posinf=0, neginf=0), index, top, 1.5)
    announce("distill absent entries")
    loss, lse, grad = run(ctx, logits, index, top, g, 1.5)
    check(loss, ref.loss, ref.loss_bound, "loss")
    check(lse, ref.lse, ref.lse_bound, "lse")
    want, bound = ref.backward(g, lse)
    check(grad, want, bound, "grad_logits")
    assert (grad[[0, 2, 7]] == 0).all() and (loss[[0, 2, 7]] == 0).all()


@pytest.mark.parametrize("vocab", [50, 33333])
def test_the_same_index_twice(ctx, vocab):
    logits, index, top, g = make(6, 4, vocab, 48)
    index[0] = index[0, 0]
    index[1, 1::2] = index[1, ::2]
    index[2, 40:] = index[2, 0]
    both(ctx, logits, index, top, g, 1.0)


def test_no_entries_at_all(ctx):
    logits, _, _, g = make(7, 3, 20, 1)
    loss, lse, grad = run(ctx, logits, np.zeros((3, 0), np.int32), np.zeros((3, 0), np.float32), g, 1.0)
    assert (loss == 0).all() and (lse == 0).all() and (grad == 0).all()


def test_far_logits(ctx):
    """One logit far above the others, masked logits of -inf and the lowest value."""
    logits, index, top, g = make(8, 4, 3000, 5)
    logits[0, 17] = 500.0
    logits[1] = np.finfo(np.float32).min
    logits[1, index[1]] = [1.0, 2.0, 3.0, 4.0, 5.0]
    logits[2, 100:] = -np.inf
    index[2] = [0, 1, 2, 3, 4]
    top[3] = [80.0, -80.0, 0.0, 1.0, 2.0]
    both(ctx, logits, index, top, g, 1.0)


def test_a_probability_of_zero(ctx):
    """The student rules out what the teacher holds likely: the loss is infinite, the gradient is not."""
    logits, index, top, g = make(9, 1, 100, 3)
    logits[0, index[0, 1]] = -np.inf
    loss, _, grad = run(ctx, logits, index, top, g, 1.0)
    assert loss[0] == np.inf and np.isfinite(grad).all()


def test_differences(ctx):
    logits, index, top, g = make(10, 2, 30, 6)
    _, _, grad = run(ctx, logits, index, top, g, 2.0)
    x = logits.astype(np.float64)
    num = np.zeros_like(x)
    for at in np.ndindex(x.shape):
        keep = x[at]
        x[at] = keep + 1e-5
        up = (Distill(x, index, top, 2.0).loss * g).sum()
        x[at] = keep - 1e-5
        num[at] = (up - (Distill(x, index, top, 2.0).loss * g).sum()) / 2e-5
        x[at] = keep
    assert np.abs(num - grad).max() < 1e-5


def test_the_same_bits_each_time_and_in_a_graph(ctx):
    rows, vocab, k = 5, 60000, 33
    logits, index, top, g = make(11, rows, vocab, k)
    dl, dt, dg = ctx.to_device(logits), ctx.to_device(top), ctx.to_device(g)
    di = ctx.to_device(index.view(np.float32))
    loss, lse, grad = ctx.alloc(rows), ctx.alloc(rows), ctx.alloc(rows * vocab)

    def step():
        ctx.distill_forward(dl, vocab, di, dt, loss, lse, rows, vocab, k, 2.0)
        ctx.distill_backward(dl, vocab, di, dt, lse, dg, grad, vocab, rows, vocab, k, 2.0)

    announce("distill in a graph")
    step()
    first = [t.download() for t in (loss, lse, grad)]
    graph = ctx.capture(step)
    for _ in range(3):
        for go in (graph.launch, step):
            for t in (loss, lse, grad):
                t.fill(float("nan"))
            go()
            for t, want in zip((loss, lse, grad), first):
                assert np.array_equal(t.download(), want)
    graph.close()


def test_bad_calls_leave_an_error(ctx):
    from zigneuron_amd import InvalidArgumentError
    t = ctx.alloc(4096)
    good = [t, 100, t, t, t, t, 2, 100, 5, 1.0]
    for i, bad in ((0, None), (1, 99), (2, None), (3, None), (4, None), (5, None), (6, -1), (7, -1), (8, -1), (8, 1025), (9, 0.0),
                   (9, -1.0), (9, float("nan")), (9, float("inf")), (9, 1e-45)):
        with pytest.raises(InvalidArgumentError):
            ctx.distill_forward(*good[:i], bad, *good[i + 1:])
    good = [t, 100, t, t, t, t, t, 100, 2, 100, 5, 1.0]
    for i, bad in ((0, None), (2, None), (3, None), (4, None), (5, None), (6, None), (7, 99), (10, 1025), (11, 0.0)):
        with pytest.raises(InvalidArgumentError):
            ctx.distill_backward(*good[:i], bad, *good[i + 1:])
    ctx.distill_forward(None, 5, None, None, None, None, 0, 5, 3, 1.0)
