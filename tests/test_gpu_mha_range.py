"""Grouped attention on scores far from zero: sums that leave the range of the split operands, and log-sum-exps whose
last bit is larger than a probability can bear.

Every dim of a query (or the first alone, the others zero) is the same power of two, every dim of a key that times 1, 2
or 4.  All keys of one level then have the same score to the last bit, whatever the order of the sum, and two levels
differ by a factor of two: the softmax is uniform over the visible keys of the highest score, exactly, at any magnitude."""
from __future__ import annotations

import numpy as np
import pytest

from block_ops_ref import Mha, U, check, dot_err
from gpu_common import announce
from test_gpu_mha import run_backward, run_forward

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    from zigneuron_amd import Context
    c = Context(0)
    yield c
    c.close()


class Levels(Mha):
    """The reference, with probabilities that are exact but for an exponential of 0 and a quotient."""

    def _probs(self, n, h):
        p, lse, err, s = super()._probs(n, h)
        return p, lse, np.full_like(err, 8 * U), s


def make(seed, shape, exponent, sign, dims):
    b, hq, hk, sq, sk, d = shape
    rng = np.random.default_rng(seed)
    q = np.full((b, hq, sq, d), sign * 2.0 ** exponent, np.float32)
    level = np.array([4.0, 1.0, 2.0], np.float32)[np.arange(sk) % 3]
    k = np.broadcast_to((level * np.float32(2.0 ** exponent))[:, None], (b, hk, sk, d)).copy()
    if dims == "one":
        q[..., 1:] = 0.0
    v, g = (rng.standard_normal(s).astype(np.float32) for s in ((b, hk, sk, d), (b, hq, sq, d)))
    return q, k, v, g


# rows a key/value head: at most 16, fewer than 384, more
SHAPES = [(1, 2, 1, 8, 70, 64), (2, 2, 1, 100, 130, 40), (1, 2, 2, 30, 1500, 128), (1, 4, 2, 200, 200, 64),
          (1, 2, 1, 300, 300, 128), (1, 1, 1, 400, 100, 96)]


@pytest.mark.parametrize("exponent", [9, 22, 41])
@pytest.mark.parametrize("sign", [-1, 1])
@pytest.mark.parametrize("dims", ["one", "all"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_far_scores(ctx, shape, causal, dims, sign, exponent):
    q, k, v, g = make(sum(shape), shape, exponent, sign, dims)
    announce(f"mha far scores {shape} causal {causal} sign {sign} 2^{exponent} {dims}")
    ref = Levels(q, k, v, 1.0, causal)
    out, lse = run_forward(ctx, q, k, v, 1.0, causal)
    check(out, ref.out, ref.out_bound, "out")
    finite = np.where(np.isfinite(ref.lse), ref.lse, 0.0)
    check(lse, ref.lse, ref.lse_bound + dot_err(shape[5]) * np.abs(finite), "lse")
    # the reference takes its own log-sum-exp: the rounding of one this large is no part of what the result may be off by
    grads, bounds = ref.backward(g, out, ref.lse)
    got = run_backward(ctx, q, k, v, out, lse, g, 1.0, causal)
    for name, x, r, e in zip(("grad_q", "grad_k", "grad_v"), got, grads, bounds):
        check(x, r, e, name)


@pytest.mark.parametrize("dims", ["one", "all"])
@pytest.mark.parametrize("sign", [-1, 1])
def test_far_scores_of_many_heads(ctx, sign, dims):
    """Enough heads for the widest tiles, with lengths."""
    shape = (16, 16, 16, 500, 200, 100)
    q, k, v, _ = make(3, shape, 41, sign, dims)
    q_lens, kv_lens = [500 - 31 * n for n in range(16)], [200 - 12 * n for n in range(16)]
    announce(f"mha far scores {shape} sign {sign} {dims}")
    ref = Levels(q, k, v, 1.0, True, q_lens, kv_lens)
    out, _ = run_forward(ctx, q, k, v, 1.0, True, q_lens, kv_lens)
    check(out, ref.out, ref.out_bound, "out")


def test_far_scores_beside_near_ones(ctx):
    """A key whose scores are far below all others, and queries that see nothing else."""
    shape = (1, 2, 1, 300, 300, 64)
    rng = np.random.default_rng(5)
    q, k, v, g = (rng.standard_normal((1, h, 300, 64)).astype(np.float32) for h in (2, 1, 1, 2))
    q[..., 0], k[..., 0] = np.float32(2.0 ** 41), 0.0
    k[:, :, 0, 0] = np.float32(-(2.0 ** 45))  # the first query sees this key alone, the others find nothing of it
    announce("mha far scores beside near ones")
    ref = Mha(q, k, v, 0.125, True)
    plain = Mha(np.where(np.arange(64) == 0, 0.0, q), np.where(np.arange(64) == 0, 0.0, k), v, 0.125, True)
    out, lse = run_forward(ctx, q, k, v, 0.125, True)
    # what the far key's magnitude adds to a bound is not allowed: the other scores do not contain it
    check(out, ref.out, plain.out_bound, "out")
    near = slice(1, None)
    check(lse[:, :, near], ref.lse[:, :, near], plain.lse_bound[:, :, near], "lse")
    gq, gk, gv = run_backward(ctx, q, k, v, out, lse, g, 0.125, True)
    assert all(np.isfinite(t).all() for t in (gq, gk, gv))
    # the far key's value has the first query's gradient and no other's
    want = g[0, :, 0].astype(np.float64).sum(0)
    check(gv[0, 0, 0], want, 8 * U * np.abs(g[0, :, 0]).sum(0), "grad_v of the far key")


@pytest.mark.parametrize("layout", ["bshd", "gaps"])
@pytest.mark.parametrize("causal", [False, True])
def test_far_scores_with_lengths_and_strides(ctx, causal, layout):
    """Sequences of all lengths at other strides, padding that holds NaN."""
    shape = (5, 4, 2, 90, 120, 64)
    q, k, v, g = make(11, shape, 20, -1, "all")
    q_lens, kv_lens = [0, 1, 50, 90, 90], [120, 5, 0, 77, 120]
    for n in range(5):
        q[n, :, q_lens[n]:], g[n, :, q_lens[n]:] = np.nan, np.inf
        k[n, :, kv_lens[n]:], v[n, :, kv_lens[n]:] = -np.inf, np.nan
        hidden = max(0, q_lens[n] - kv_lens[n]) if causal else (q_lens[n] if kv_lens[n] == 0 else 0)
        g[n, :, :hidden] = np.nan
    announce(f"mha far scores with lengths, causal {causal} {layout}")
    ref = Levels(q, k, v, 1.0, causal, q_lens, kv_lens)
    out, lse = run_forward(ctx, q, k, v, 1.0, causal, q_lens, kv_lens, layout)
    check(out, ref.out, ref.out_bound, "out")
    grads, bounds = ref.backward(g, out, ref.lse)
    got = run_backward(ctx, q, k, v, out, lse, g, 1.0, causal, q_lens, kv_lens, layout)
    for name, x, r, e in zip(("grad_q", "grad_k", "grad_v"), got, grads, bounds):
        check(x, r, e, name)
