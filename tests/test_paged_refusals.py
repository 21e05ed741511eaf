"""What the calls of rotary positions and the paged cache refuse, on the CPU.

Their checks come before anything of the context is used or a device is
selected, so a blank context will do: a call that passed them would report
the missing device (another status) instead."""
from __future__ import annotations

import ctypes
import os

import numpy as np
import pytest

INVALID, OVERFLOW = -4, -8
BIG = 1 << 40
P = 4096  # any address: a refused call reads nothing
no_gpu = pytest.mark.skipif(os.path.exists("/dev/kfd"), reason="a GPU is present: the GPU tests make these calls")


@pytest.fixture(scope="module")
def lib():
    from zigneuron_amd import _lib
    return _lib.load()


@pytest.fixture(scope="module")
def blank():
    memory = ctypes.create_string_buffer(1 << 16)
    yield ctypes.addressof(memory)
    del memory


def rotary(lib, ctx, back=False, **kw):
    a = dict(x=P, y=2 * P, freq=P, positions=None, batch=2, heads=4, len=8, head_dim=16, rot_dim=16, layout=0, scale=1.0, ps=8,
             xb=512, xh=128, xs=16, yb=512, yh=128, ys=16)
    assert set(kw) <= set(a)
    a.update(kw)
    return (lib.zn_hip_rotary_backward if back else lib.zn_hip_rotary_forward)(ctx, *a.values())


def desc(**kw):
    from zigneuron_amd import PagedCache
    a = dict(k=P, v=P, page_table=P, kv_lens=P, batch=2, num_pages=8, page_size=16, max_pages=4, kv_heads=2, head_dim=16, dtype="f32",
             strides=(512, 256, 16))
    assert set(kw) <= set(a)
    a.update(kw)
    return PagedCache(**a)


def append(lib, ctx, cache=None, **kw):
    a = dict(starts=P, tokens=6, k=P, v=P, kt=32, kh=16, q=P, q_out=2 * P, q_heads=4, qt=64, qh=16, ot=64, oh=16, freq=P, rot_dim=16,
             layout=0, scale=1.0, positions=None)
    assert set(kw) <= set(a)
    a.update(kw)
    c = desc() if cache is None else cache
    return lib.zn_hip_paged_append(ctx, c.address if c != 0 else None, *a.values())


def attention(lib, ctx, cache=None, **kw):
    a = dict(starts=P, tokens=6, max_q=4, max_kv=64, q=P, out=2 * P, lse=None, q_heads=4, scale=0.25, causal=1, qt=64, qh=16, ot=64,
             oh=16)
    assert set(kw) <= set(a)
    a.update(kw)
    c = desc() if cache is None else cache
    return lib.zn_hip_paged_attention(ctx, c.address if c != 0 else None, *a.values())


@no_gpu
@pytest.mark.parametrize("back", [False, True])
def test_rotary(lib, blank, back):
    assert rotary(lib, None, back) == INVALID
    assert rotary(lib, blank, back) not in (0, INVALID, OVERFLOW)  # a good call gets to the device
    for good in ({"rot_dim": 0, "freq": None}, {"xb": 0}, {"xh": 0}, {"xs": 0}, {"ps": 0}, {"layout": 1}, {"y": P}, {"scale": 0.0}):
        assert rotary(lib, blank, back, **good) not in (0, INVALID, OVERFLOW), good
    for bad in ({"x": None}, {"y": None}, {"freq": None}, {"batch": -1}, {"heads": -1}, {"len": -1}, {"head_dim": 0}, {"head_dim": 1025},
                {"rot_dim": -2}, {"rot_dim": 15}, {"rot_dim": 18}, {"layout": 2}, {"layout": -1}, {"scale": float("nan")},
                {"scale": float("inf")}, {"ps": -1}, {"xb": -1}, {"xs": -1}, {"yb": 0}, {"yh": 0}, {"ys": 0}, {"yh": -1}):
        assert rotary(lib, blank, back, **bad) == INVALID, bad
    for big in ({"batch": BIG}, {"heads": BIG}, {"len": BIG}, {"batch": 1 << 20, "len": 1 << 20}, {"xb": 1 << 50}, {"ys": 1 << 45},
                {"ps": 1 << 62}):
        assert rotary(lib, blank, back, **big) == OVERFLOW, big
    for nothing in ({"batch": 0}, {"heads": 0}, {"len": 0}, {"len": 0, "x": None, "y": None, "ys": 0}):
        assert rotary(lib, blank, back, **nothing) == 0, nothing


@no_gpu
def test_append(lib, blank):
    assert append(lib, None) == INVALID and append(lib, blank, 0) == INVALID
    assert append(lib, blank) not in (0, INVALID, OVERFLOW)
    for good in ({"q": None, "q_out": None, "q_heads": 0}, {"rot_dim": 0, "freq": None}, {"kt": 0}, {"kh": 0}, {"qt": 0}, {"positions": P}):
        assert append(lib, blank, **good) not in (0, INVALID, OVERFLOW), good
    for bad in ({"starts": None}, {"tokens": -1}, {"k": None}, {"v": None}, {"q_out": None}, {"q_heads": -1}, {"freq": None},
                {"rot_dim": 3}, {"rot_dim": 18}, {"layout": 5}, {"scale": float("inf")}, {"kt": -1}, {"kh": -1}, {"qt": -1}, {"ot": 0},
                {"oh": 0}, {"oh": -1}):
        assert append(lib, blank, **bad) == INVALID, bad
    for bad in ({"k": None}, {"v": None}, {"page_table": None}, {"kv_lens": None}, {"batch": -1}, {"num_pages": -1}, {"page_size": 0},
                {"max_pages": -1}, {"kv_heads": -1}, {"head_dim": 0}, {"head_dim": 129}, {"strides": (512, 256, 15)},
                {"strides": (0, 256, 16)}, {"strides": (512, 0, 16)}, {"strides": (-1, 256, 16)}, {"dtype": 2}, {"dtype": -1}):
        assert append(lib, blank, desc(**bad), rot_dim=0) == INVALID, bad
    for big in ({"batch": BIG}, {"num_pages": BIG}, {"page_size": BIG}, {"max_pages": BIG}, {"kv_heads": BIG},
                {"max_pages": 1 << 20, "page_size": 1 << 20}, {"strides": (1 << 50, 256, 16)}, {"strides": (512, 256, 1 << 45)}):
        assert append(lib, blank, desc(**big)) == OVERFLOW, big
    for big in ({"tokens": 1 << 24}, {"q_heads": BIG}, {"kt": 1 << 50}, {"ot": 1 << 50}):
        assert append(lib, blank, **big) == OVERFLOW, big
    assert append(lib, blank, tokens=0) == 0
    assert append(lib, blank, desc(batch=0)) == 0
    assert append(lib, blank, desc(kv_heads=0), q=None) == 0


@no_gpu
def test_attention(lib, blank):
    assert attention(lib, None) == INVALID and attention(lib, blank, 0) == INVALID
    assert attention(lib, blank) not in (0, INVALID, OVERFLOW)
    for good in ({"causal": 0}, {"lse": P}, {"qt": 0}, {"qh": 0}, {"max_kv": 0}, {"scale": -1.0}):
        assert attention(lib, blank, **good) not in (0, INVALID, OVERFLOW), good
    assert attention(lib, blank, desc(strides=(0, 0, 16))) not in (0, INVALID, OVERFLOW)  # read only: broadcast
    assert attention(lib, blank, desc(k=None, v=None, page_table=None, num_pages=0)) not in (0, INVALID, OVERFLOW)  # no pages: all masked
    for bad in ({"starts": None}, {"tokens": -1}, {"max_q": -1}, {"max_kv": -1}, {"q": None}, {"out": None}, {"q_heads": 5},
                {"q_heads": -4}, {"scale": float("nan")}, {"causal": 2}, {"causal": -1}, {"qt": -1}, {"qh": -1}, {"ot": 0}, {"oh": 0}):
        assert attention(lib, blank, **bad) == INVALID, bad
    for bad in ({"k": None}, {"v": None}, {"page_table": None}, {"kv_lens": None}, {"page_size": 0}, {"kv_heads": 0}, {"head_dim": 129},
                {"dtype": 2}, {"strides": (512, 256, 8)}):
        assert attention(lib, blank, desc(**bad)) == INVALID, bad
    for big in ({"tokens": 1 << 24}, {"q_heads": 1 << 20}, {"qt": 1 << 50}, {"oh": 1 << 50}):
        assert attention(lib, blank, **big) == OVERFLOW, big
    assert attention(lib, blank, desc(max_pages=1 << 20, page_size=1 << 20)) == OVERFLOW
    assert attention(lib, blank, tokens=0) == 0
    assert attention(lib, blank, max_q=0) == 0  # no sequence has a new token
    assert attention(lib, blank, desc(batch=0)) == 0
    assert attention(lib, blank, desc(kv_heads=0), q_heads=0) == 0


def test_names():
    import zigneuron_amd as zn
    with pytest.raises(zn.InvalidArgumentError):
        zn.PagedCache(P, P, P, P, 1, 1, 1, 1, 1, 1, "fp64")
    with pytest.raises(zn.InvalidArgumentError):
        zn.rotary_frequencies(8, scaling="other")


def test_frequencies():
    import zigneuron_amd as zn
    n, base, factor, trained = 64, 10000.0, 4.0, 2048
    i = np.arange(n // 2)
    f = base ** (-2.0 * i / n)

    def near(got, want):
        assert got.dtype == np.float32 and np.all(np.abs(got - want) <= 2.0 ** -23 * want), (got, want)  # a rounding, and pow's last bits

    near(zn.rotary_frequencies(n), f)
    near(zn.rotary_frequencies(n, base, "linear", factor), f / factor)
    near(zn.rotary_frequencies(n, base, "base", factor), (base * factor ** (n / (n - 2))) ** (-2.0 * i / n))
    turns = trained * f / (2 * np.pi)
    keep = np.clip((turns - 1) / (32 - 1), 0, 1)
    near(zn.rotary_frequencies(n, base, "turns", factor, trained, 1, 32), keep * f + (1 - keep) * f / factor)
    first, last = np.nonzero(turns >= 32)[0][-1], np.nonzero(turns <= 1)[0][0]
    keep = np.clip(1 - (i - first) / (last - first), 0, 1)
    near(zn.rotary_frequencies(n, base, "pairs", factor, trained, 1, 32), keep * f + (1 - keep) * f / factor)
    # all pairs of a short context turn less than `low`: all slowed down
    near(zn.rotary_frequencies(8, 100.0, "turns", 2.0, 1, 1, 4), 100.0 ** (-2.0 * np.arange(4) / 8) / 2)


def test_frequencies_refusals(lib):
    buf = (ctypes.c_float * 64)()

    def f(freq=buf, n=64, rot=16, base=1e4, scaling=0, factor=1.0, trained=128, low=1.0, high=4.0):
        return lib.zn_hip_rotary_frequencies(freq, n, rot, base, scaling, factor, trained, low, high)

    for s in range(5):
        assert f(scaling=s) == 0, s
    for bad in ({"freq": None}, {"n": 7}, {"rot": 0}, {"rot": 15}, {"rot": -2}, {"rot": 1026}, {"base": 0.0}, {"base": float("inf")},
                {"base": float("nan")}, {"scaling": 5}, {"scaling": -1}, {"scaling": 1, "factor": 0.0}, {"scaling": 2, "rot": 2},
                {"scaling": 3, "trained": 0}, {"scaling": 3, "low": 0.0}, {"scaling": 4, "high": 1.0}, {"scaling": 4, "base": 1.0},
                {"scaling": 1, "factor": float("nan")}, {"scaling": 3, "high": float("inf")}):
        assert f(**bad) == INVALID, bad
