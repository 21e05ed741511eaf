"""Rotary positions and appending queued on two contexts of a device, a stream each, before either is waited for."""
from __future__ import annotations

import numpy as np
import pytest

from gpu_common import announce
from paged_ref import Ints, Pool, frequencies, starts_of
from test_gpu_rotary import expect
from block_ops_ref import check

pytestmark = pytest.mark.gpu


def test_two_contexts_at_once():
    from zigneuron_amd import Context
    announce("rotary and append, two contexts at once")
    rng = np.random.default_rng(8)
    shape, d = (4, 16, 500, 64), 64
    with Context(0) as a, Context(0) as b:
        work = []
        for c in (a, b):
            x = rng.standard_normal(shape).astype(np.float32)
            pos = rng.integers(0, 100000, (4, 500)).astype(np.int32)
            pool = Pool(8, [300] * 4, 2, 16, d)
            work.append(dict(c=c, x=x, pos=pos, dx=c.to_device(x), out=[c.alloc(x.size) for _ in range(6)], p=Ints(c, pos),
                             f=c.to_device(frequencies(d)), pool=pool, cache=pool.place(c), s=Ints(c, starts_of([250] * 4)),
                             kv=rng.standard_normal((1000, 2, d)).astype(np.float32)))
            work[-1]["dkv"] = c.to_device(work[-1]["kv"])
        for w in work:
            w["c"].sync()
        for i in range(6):  # in turn, nothing read in between
            for w in work:
                w["c"].rotary_forward(w["dx"], w["out"][i], w["f"], *shape, d, "half", w["p"].ptr)
                w["c"].paged_append(w["cache"], w["s"].ptr, 1000, w["dkv"], w["dkv"], freq=w["f"], rot_dim=d)
        for w in work:
            ref, bound = expect(w["x"], d, "half", w["pos"])
            first = w["out"][0].download()
            check(first.reshape(shape), ref, bound, "y")
            for o in w["out"][1:]:
                assert np.array_equal(o.download(), first)
            _, v = w["pool"].read()
            js = np.arange(50, 300)
            for b_ in range(4):
                assert np.array_equal(v[w["pool"].table[b_, js // 16], :, js % 16], w["kv"][250 * b_:250 * b_ + 250])
        del work
