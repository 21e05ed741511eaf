"""Rotary positions whose angles pass what 64-bit floats count in quarter turns (2^53 and more)."""
from __future__ import annotations

import numpy as np
import pytest

from block_ops_ref import check
from gpu_common import announce
from paged_ref import U
from test_gpu_rotary import run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    from zigneuron_amd import Context
    c = Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("back", [False, True])
@pytest.mark.parametrize("first", [2.0 ** 10, 2.0 ** 18, 2.0 ** 21, 2.0 ** 25, 2.0 ** 30, 2.0 ** 36])
def test_angles_past_a_quarter_turns_rounding(ctx, first, back):
    """Frequencies from `first` on at positions to both ends of 32 bits: angles from 2^41 to 2^70.  Position times frequency is exact
    in 80-bit floats (55 bits), whose sine and cosine reduce it exactly; 8 U is the bound of near positions."""
    announce(f"rotary, angles from {first} back {back}")
    assert np.finfo(np.longdouble).nmant >= 63
    rng = np.random.default_rng(11)
    pos = np.concatenate([[0, 1, -1, 2 ** 31 - 1, -(2 ** 31), 2 ** 31 - 2], rng.integers(-(2 ** 31), 2 ** 31, 58)]).astype(np.int32)
    freq = (first * np.array([1, 1.1, 1.5707964, 3.0, 3.9, 7.7, 0.99999994, 5.123])).astype(np.float32)
    x = rng.standard_normal((1, 2, pos.size, 16)).astype(np.float32)
    a = pos.astype(np.longdouble)[:, None] * freq.astype(np.longdouble)
    s, c = np.sin(a).astype(np.float64) * (-1 if back else 1), np.cos(a).astype(np.float64)
    p, q = x[..., :8].astype(np.float64), x[..., 8:].astype(np.float64)
    ref, bound = np.concatenate([p * c - q * s, p * s + q * c], -1), np.tile(8 * U * (np.abs(p) + np.abs(q)), 2)
    check(run(ctx, x, 16, "half", pos, freq=freq, back=back), ref, bound, "y")


def test_no_angle_makes_a_pair_longer(ctx):
    """Past 2^80 the angle is any: the pair keeps its length all the same."""
    announce("rotary, any angle")
    pos = np.array([2 ** 31 - 1, -(2 ** 31), 1, 0, 123456789], np.int32)
    freq = np.array([3e38, 1e30, 2.0 ** 60, 1e25], np.float32)
    x = np.random.default_rng(3).standard_normal((1, 3, 5, 8)).astype(np.float32)
    got = run(ctx, x, 8, "half", pos, freq=freq).astype(np.float64)
    n, m = np.hypot(x[..., :4].astype(np.float64), x[..., 4:]), np.hypot(got[..., :4], got[..., 4:])
    assert np.all(np.abs(m - n) <= 16 * U * (np.abs(x[..., :4]) + np.abs(x[..., 4:])))
