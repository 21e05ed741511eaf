"""Scaled rotary frequencies over the whole range of context lengths (zn_hip_rotary_frequencies), against 64 bits.

A frequency is rounded once, by 2^-24 of it; the 64-bit powers, logarithms and mixtures before that lose far less than another 2^-24."""
from __future__ import annotations

import math

import numpy as np
import pytest


def pairs(rot, base, factor, trained, low, high):
    """The "pairs" ramp from its definition: from the rounded down number of the pair of `high` turns to the rounded up one of `low`
    turns, both held to 0 .. rot - 1; pairs before the ramp keep their speed."""
    def pair_of(turns):  # f_i trained = 2 pi turns
        return rot / 2 * math.log(trained / (2 * math.pi * turns)) / math.log(base)

    i = np.arange(rot // 2)
    f = base ** (-2.0 * i / rot)
    first, last = max(math.floor(pair_of(high)), 0), min(math.ceil(pair_of(low)), rot - 1)
    keep = np.clip((last - i) / (last - first), 0, 1) if last > first else (i < first).astype(float)
    return keep * f + (1 - keep) * f / factor, trained * f / (2 * math.pi)


@pytest.mark.parametrize("trained", [512, 2048, 8192, 50000, 65536, 131072, 1 << 20, 1 << 24, 1 << 33])
@pytest.mark.parametrize("rot,base", [(64, 10000.0), (128, 10000.0), (16, 10000.0), (64, 500000.0), (2, 10000.0), (38, 100.0)])
@pytest.mark.parametrize("factor", [2.0, 4.0, 8.0])
def test_pairs_at_all_lengths(rot, base, trained, factor):
    """Lengths at which the slowest pair makes fewer than `low` turns, more, and more than `high`."""
    import zigneuron_amd as zn
    got = zn.rotary_frequencies(rot, base, "pairs", factor, trained, 1, 32).astype(np.float64)
    f = base ** (-2.0 * np.arange(rot // 2) / rot)
    want, turns = pairs(rot, base, factor, trained, 1, 32)
    assert np.all(np.abs(got - want) <= 2.0 ** -23 * want), (got / want)
    # whatever the ramp: pairs of `high` turns and more keep their speed, none of more than `low` turns loses all of it
    assert np.all(np.abs(got - f)[turns >= 32 * base ** (2 / rot)] <= 2.0 ** -23 * f[turns >= 32 * base ** (2 / rot)])
    assert np.all(got[turns > 1] > f[turns > 1] / factor * (1 + 2.0 ** -20))


@pytest.mark.parametrize("trained,low", [(1, 1.0), (6, 1.0), (100, 16.0), (2048, 326.0), (128, 1000.0)])
@pytest.mark.parametrize("rot", [2, 8, 64])
def test_pairs_that_all_turn_less_than_low(rot, trained, low):
    """Contexts so short that even the first pair makes `low` turns or fewer: all are slowed down, as "turns" does."""
    import zigneuron_amd as zn
    f = 10000.0 ** (-2.0 * np.arange(rot // 2) / rot)
    assert trained / (2 * math.pi) <= low  # the first pair's frequency is 1
    for kind in ("pairs", "turns"):
        got = zn.rotary_frequencies(rot, 10000.0, kind, 4.0, trained, low, 4 * low).astype(np.float64)
        assert np.all(np.abs(got - f / 4) <= 2.0 ** -23 * f), (kind, got / f)
