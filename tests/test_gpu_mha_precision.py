"""What grouped attention's probabilities lose: their 2-norm error, on inputs that show one probability a value.

K and V are rows of the identity, so scores are values of Q and out is P itself; grad_out, Q's other dims and V's first
column are chosen so that grad_v is P, and grad_q and grad_k are dS, with one product a value.  Nothing averages out, and
bounds of whole sums, in which a probability's few half steps vanish, are not needed.

The bound, in u = 2^-24 (half a step relative to a value of 1).  Scores lie within 1 of zero.  Roundings on the way to a
probability, each at most so far: the scale times log2 e, and that times Q (1.45 of the score, ln 2 of it each: 1 u and
1 u); the exponent's argument, below 4 in magnitude in the forward and mostly so in the backward (half a step of [2, 4)
times ln 2: 1.4 u; of [4, 8): 2.8 u); log2 e times the log-sum-exp (1.4 u); the exponential (2 u); a rescale of earlier
blocks (2 u) and its product (1 u); the sum's rounding (1 u) and the quotient (1 u).  Independent and evenly spread, a
rounding of at most e has a root mean square of e / sqrt(3): 2.2 u in the forward and 2.4 u in the backward, 2.6 u with
dP - delta.  4 u leaves room for what they have in common.  An argument rounded near 24 alone would be off by 11 u, 6.4 u
in the mean."""
from __future__ import annotations

import numpy as np
import pytest

from block_ops_ref import U
from gpu_common import announce
from test_gpu_mha import run_backward, run_forward

pytestmark = pytest.mark.gpu
BOUND = 4 * U


@pytest.fixture(scope="module")
def ctx():
    from zigneuron_amd import Context
    c = Context(0)
    yield c
    c.close()


def eye(b, h, rows, d):
    return np.broadcast_to(np.eye(rows, d, dtype=np.float32), (b, h, rows, d)).copy()


def off(got, want):
    return np.linalg.norm(got.astype(np.float64) - want) / np.linalg.norm(want)


def softmax(s):
    e = np.exp(s.astype(np.float64) - s.max(-1, keepdims=True))
    return e / e.sum(-1, keepdims=True)


@pytest.mark.parametrize("b,h,sq,d", [(4, 4, 12, 64), (2, 4, 100, 32), (2, 4, 100, 64), (2, 2, 100, 96), (2, 2, 100, 128),
                                      (1, 4, 500, 32), (1, 4, 500, 64), (1, 2, 500, 96), (1, 2, 500, 128), (16, 16, 500, 96),
                                      (16, 16, 500, 128)])
def test_forward(ctx, b, h, sq, d):
    n = min(d, 96 if b == 16 else 40)  # keys; the many heads take the widest tiles
    q = np.zeros((b, h, sq, d), np.float32)
    q[..., :n] = np.random.default_rng(sq + d).uniform(-1, 1, (b, h, sq, n))
    announce(f"mha precision forward {b} {h} {sq} {d}")
    out, _ = run_forward(ctx, q, eye(b, h, n, d), eye(b, h, n, d), 1.0)
    assert (out[..., n:] == 0).all()
    error = off(out[..., :n], softmax(q[..., :n]))
    print(f"out {error / U:.2f} u", flush=True)
    assert error <= BOUND


@pytest.mark.parametrize("sq", [60, 300, 1500])
@pytest.mark.parametrize("d", [32, 64, 96, 128])
def test_backward(ctx, sq, d):
    n, shown = 8, min(sq, d - 8)
    rng = np.random.default_rng(sq + d)
    q, g = np.zeros((1, 1, sq, d), np.float32), np.zeros((1, 1, sq, d), np.float32)
    k, v = eye(1, 1, n, d), np.zeros((1, 1, n, d), np.float32)
    s = rng.uniform(-1, 1, (sq, n)).astype(np.float32)
    q[0, 0, :, :n] = s
    i = np.arange(shown)
    q[0, 0, i, n + i] = 1.0  # these dims of K are zero
    announce(f"mha precision backward {sq} {d}")
    # grad_v shows P: query i has the i-th unit
    g[0, 0, i, i] = 1.0
    out, lse = run_forward(ctx, q, k, v, 1.0)
    _, _, gv = run_backward(ctx, q, k, v, out, lse, g, 1.0)
    p = np.exp(s.astype(np.float64) - lse[0, 0, :, None].astype(np.float64))
    errors = {"grad_v": off(gv[0, 0, :, :shown], p[:shown].T)}
    # grad_q and grad_k show dS: dP is 1 or -1
    a = np.where(np.arange(n) % 2, 1.0, -1.0)
    v[0, 0, :, 0] = a
    g[:] = 0.0
    g[..., 0] = 1.0
    out, lse = run_forward(ctx, q, k, v, 1.0)
    gq, gk, _ = run_backward(ctx, q, k, v, out, lse, g, 1.0)
    ds = p * (a - out[0, 0, :, :1].astype(np.float64))
    errors["grad_q"] = off(gq[0, 0, :, :n], ds)
    errors["grad_k"] = off(gk[0, 0, :, n:n + shown], ds[:shown].T)
    print({x: f"{e / U:.2f} u" for x, e in errors.items()}, flush=True)
    assert max(errors.values()) <= BOUND, errors
