"""What enters a bf16 cache is rounded once, to the nearest: a turned key lies between the roundings of the two ends of its fp32 bound.

With y the turn in 64 bits and e the bound of the fp32 turn, the value that is rounded lies in [y - e, y + e], and rounding keeps order."""
from __future__ import annotations

import numpy as np
import pytest

from gpu_common import announce
from paged_ref import Ints, Pool, Strided, frequencies, from_bf16, rotary, starts_of, to_bf16


def ends(y, e):
    """The bf16 values that y - e and y + e round to (their 32-bit neighbours outwards first)."""
    lo, hi = (y - e).astype(np.float32), (y + e).astype(np.float32)
    lo = np.where(lo > y - e, np.nextafter(lo, np.float32(-np.inf)), lo)
    hi = np.where(hi < y + e, np.nextafter(hi, np.float32(np.inf)), hi)
    return from_bf16(to_bf16(lo)), from_bf16(to_bf16(hi))


def test_the_bound_tells_roundings_apart():
    """On the CPU: values rounded to the nearest are inside, truncated or rounded twice upwards ones are not."""
    rng = np.random.default_rng(0)
    x = rng.standard_normal((500, 1, 64)).astype(np.float32)
    y, e = rotary(x, np.arange(500)[:, None], frequencies(64), 64, "half")
    lo, hi = ends(y, e)
    near = from_bf16(to_bf16(y.astype(np.float32)))
    assert np.all((lo <= near) & (near <= hi))
    assert np.mean(lo < hi) < 0.01  # nearly always one value
    cut = from_bf16((y.astype(np.float32).view(np.uint32) >> 16).astype(np.uint16))
    assert np.mean((lo <= cut) & (cut <= hi)) < 0.6


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("case", [
    # lens, counts, kv heads, page, dim, rot, scale, strides of the cache
    ([37, 16, 40], [1, 1, 1], 2, 16, 64, 64, 1.0, "phsd"), ([130, 7], [130, 3], 4, 24, 76, 38, 1.0, "pshd"),
    ([100, 0, 33, 64], [20, 0, 33, 1], 3, 7, 45, 26, 1.3, "gaps"), ([300], [299], 3, 64, 128, 128, 0.7, "phsd"),
    ([50, 60], [0, 60], 8, 256, 127, 126, 1.0, "pshd"), ([5], [5], 1, 16, 2, 2, 1.0, "phsd"), ([9] * 70, [1] * 70, 1, 8, 32, 16, 1.0, "gaps"),
])
def test_turned_keys_are_rounded_once(case, layout):
    from zigneuron_amd import Context
    lens, counts, hk, page, dim, rot, scale, order = case
    announce(f"append, rounding {case} {layout}")
    with Context(0) as ctx:
        pool = Pool(sum(lens), lens, hk, page, dim, "bf16", order)
        cache = pool.place(ctx)
        n = sum(counts)
        rng = np.random.default_rng(n)
        xk, xv = (rng.standard_normal((n, hk, dim)).astype(np.float32) for _ in range(2))
        dk, dv = Strided(ctx, xk), Strided(ctx, xv)
        starts, freq = Ints(ctx, starts_of(counts)), ctx.to_device(frequencies(rot))
        ctx.paged_append(cache, starts.ptr, n, dk.ptr, dv.ptr, freq=freq, rot_dim=rot, layout=layout, scale=scale)
        k, v = pool.read()
    t = 0
    for b, c in enumerate(counts):
        js = np.arange(lens[b] - c, lens[b])
        pages = pool.table[b, js // page]
        got_k, got_v = k[pages, :, js % page], v[pages, :, js % page]
        y, e = rotary(xk[t:t + c], js[:, None], frequencies(rot), rot, layout, scale)
        lo, hi = ends(y, e)
        assert np.all((lo <= got_k) & (got_k <= hi)), f"k of sequence {b}"
        assert np.array_equal(got_v, from_bf16(to_bf16(xv[t:t + c]))), f"v of sequence {b}"
        t += c
