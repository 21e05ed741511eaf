"""What the language-model entry points refuse, on the CPU.

Their checks come before anything of the context is used or a device is
selected, so a blank context will do: a call that passed them would report
the missing device (another status) instead."""
from __future__ import annotations

import ctypes
import os

import pytest

pytestmark = pytest.mark.skipif(os.path.exists("/dev/kfd"), reason="a GPU is present: the GPU tests make these calls")

INVALID, OVERFLOW = -4, -8
BIG = 1 << 40


@pytest.fixture(scope="module")
def lib():
    from zigneuron_amd import _lib
    return _lib.load()


@pytest.fixture(scope="module")
def blank():
    memory = ctypes.create_string_buffer(1 << 16)
    yield ctypes.addressof(memory)
    del memory


P = 4096  # any address: a refused call reads nothing


def mha(lib, ctx, back=False, **kw):
    names = ["q", "k", "v", "out", "lse"] + (["grad_out", "grad_q", "grad_k", "grad_v"] if back else [])
    a = {n: P for n in names}
    a.update(batch=2, q_heads=4, kv_heads=2, q_len=8, kv_len=8, head_dim=16, scale=0.25, causal=1, q_lens=None, kv_lens=None,
             qb=512, qh=128, qs=16, kb=256, kh=128, ks=16, ob=512, oh=128, os=16)
    assert set(kw) <= set(a)
    a.update(kw)
    return (lib.zn_hip_mha_backward if back else lib.zn_hip_mha_forward)(ctx, *a.values())


@pytest.mark.parametrize("back", [False, True])
def test_mha(lib, blank, back):
    assert mha(lib, None, back) == INVALID
    assert mha(lib, blank, back) not in (0, INVALID, OVERFLOW)  # a good call gets to the device
    for bad in ({"q": None}, {"k": None}, {"v": None}, {"out": None}, {"batch": -1}, {"q_heads": -4}, {"kv_heads": -2}, {"q_len": -1},
                {"kv_len": -1}, {"head_dim": 0}, {"head_dim": 129, "qs": 200, "ks": 200, "os": 200}, {"q_heads": 5}, {"kv_heads": 0},
                {"scale": float("inf")}, {"scale": float("nan")}, {"causal": 2}, {"causal": -1}, {"qs": 15}, {"ks": 15}, {"os": 15},
                {"qs": (1 << 22) + 1}, {"ks": (1 << 22) + 1}, {"os": (1 << 22) + 1}, {"qb": -1}, {"kh": -1}, {"ob": -1}):
        assert mha(lib, blank, back, **bad) == INVALID, bad
    for big in ({"batch": BIG}, {"q_len": BIG}, {"kv_len": BIG}, {"q_heads": BIG}, {"batch": 1 << 29, "q_heads": 8}, {"batch": 1 << 23}):
        assert mha(lib, blank, back, **big) == OVERFLOW, big
    for nothing in ({"batch": 0}, {"q_heads": 0, "kv_heads": 0}, {"q_len": 0, "kv_len": 0}):
        assert mha(lib, blank, back, **nothing) == 0, nothing
    # strides of zero: broadcast what is read, never what is written
    for zero in ({"kb": 0}, {"kh": 0}, {"qb": 0}, {"qh": 0}):
        assert (mha(lib, blank, back, **zero) == INVALID) == back, zero
    for zero in ({"ob": 0}, {"oh": 0}):
        assert (mha(lib, blank, back, **zero) == INVALID) == (not back), zero
    if back:
        for bad in ("lse", "grad_out", "grad_q", "grad_k", "grad_v"):
            assert mha(lib, blank, True, **{bad: None}) == INVALID, bad


def test_gated(lib, blank):
    def f(ctx=blank, act=4, x=P, w=P, bias=None, z=None, h=P, batch=4, n_in=8, hidden=8):
        return lib.zn_hip_gated_dense_forward(ctx, act, x, w, bias, z, h, batch, n_in, hidden)

    def b(ctx=blank, act=4, x=P, w=P, z=P, gh=P, gz=P, gx=P, gw=P, gb=None, batch=4, n_in=8, hidden=8):
        return lib.zn_hip_gated_dense_backward(ctx, act, x, w, z, gh, gz, gx, gw, gb, batch, n_in, hidden)

    for call, needed in ((f, ("x", "w", "h")), (b, ("x", "w", "z", "gh", "gz", "gw"))):
        assert call(ctx=None) == INVALID
        assert call() not in (0, INVALID, OVERFLOW)
        for bad in ({"act": -1}, {"act": 6}, {"batch": -1}, {"n_in": -1}, {"hidden": -1}, *({n: None} for n in needed)):
            assert call(**bad) == INVALID, bad
        for big in ({"batch": BIG}, {"n_in": BIG}, {"hidden": BIG}, {"batch": 1 << 16, "n_in": 1 << 14}, {"n_in": 1 << 15, "hidden": 1 << 14}):
            assert call(**big) == OVERFLOW, big
    assert f(batch=0) == 0 and f(hidden=0) == 0


def test_distill(lib, blank):
    def f(ctx=blank, logits=P, ld=100, index=P, top=P, loss=P, lse=P, rows=4, vocab=100, k=8, t=1.0):
        return lib.zn_hip_distill_forward(ctx, logits, ld, index, top, loss, lse, rows, vocab, k, t)

    def b(ctx=blank, logits=P, ld=100, index=P, top=P, lse=P, gl=P, grad=P, gld=100, rows=4, vocab=100, k=8, t=1.0):
        return lib.zn_hip_distill_backward(ctx, logits, ld, index, top, lse, gl, grad, gld, rows, vocab, k, t)

    for call, needed in ((f, ("logits", "index", "top", "loss", "lse")), (b, ("logits", "index", "top", "lse", "gl", "grad"))):
        assert call(ctx=None) == INVALID
        assert call() not in (0, INVALID, OVERFLOW)
        for bad in ({"ld": 99}, {"rows": -1}, {"vocab": -1}, {"k": -1}, {"k": 1025}, {"t": 0.0}, {"t": -1.0}, {"t": float("nan")},
                    {"t": float("inf")}, {"t": 1e-45}, *({n: None} for n in needed)):
            assert call(**bad) == INVALID, bad
        assert call(vocab=BIG, ld=BIG, **({"gld": BIG} if call is b else {})) == OVERFLOW
        assert call(rows=0) == 0
    assert b(gld=99) == INVALID


def test_mha_backward_of_no_queries_and_no_keys(lib, blank):
    """Heads without queries against heads without keys: nothing to compute, whatever the other lengths are."""
    for nothing in ({"q_heads": 0, "kv_len": 0}, {"q_len": 0, "kv_len": 0}, {"q_heads": 0, "q_len": 0, "kv_len": 0}):
        assert mha(lib, blank, True, **nothing) == 0, nothing
    assert mha(lib, blank, True, q_heads=0) not in (0, INVALID, OVERFLOW)  # keys: their gradients are zeroed


@pytest.mark.parametrize("back", [False, True])
def test_mha_key_heads_without_query_heads(lib, blank, back):
    """Their number is bounded by itself: its product with the batch must not wrap."""
    for batch, heads in ((1 << 30, 1 << 34), (1 << 24, 1 << 40), (1, 1 << 33), (2, 1 << 62)):
        assert mha(lib, blank, back, batch=batch, q_heads=0, kv_heads=heads) == OVERFLOW, (batch, heads)
