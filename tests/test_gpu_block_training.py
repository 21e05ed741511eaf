"""A training step of one block as a program would run it: the projections of
queries, keys and values (one product), grouped attention, its output
projection, the gated feed-forward layer and its down projection, both with a
residual, the logits, and the distillation loss; then every gradient back to
the block's input.  Losses and gradients against 64-bit automatic
differentiation, eagerly and as replays of a captured graph."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from gpu_common import announce

pytestmark = pytest.mark.gpu

B, S, HQ, HK, D, HIDDEN, VOCAB, K = 3, 70, 4, 2, 24, 200, 501, 12
MODEL, QKV = HQ * D, (HQ + 2 * HK) * D
ROWS, T = B * S, 2.0
LENS = np.array([70, 33, 0], np.int32)


def inputs():
    rng = np.random.default_rng(77)
    f = lambda *s, by=1.0: (rng.standard_normal(s) * by).astype(np.float32)  # noqa: E731
    a = {"x": f(ROWS, MODEL), "wqkv": f(MODEL, QKV, by=MODEL ** -0.5), "wo": f(MODEL, MODEL, by=MODEL ** -0.5),
         "wg": f(MODEL, 2 * HIDDEN, by=MODEL ** -0.5), "bg": f(2 * HIDDEN, by=0.1), "wd": f(HIDDEN, MODEL, by=HIDDEN ** -0.5),
         "wv": f(VOCAB, MODEL, by=MODEL ** -0.5), "top": f(ROWS, K, by=3.0)}
    a["index"] = np.stack([rng.permutation(VOCAB)[:K] for _ in range(ROWS)]).astype(np.int32)
    for n in range(B):
        a["index"].reshape(B, S, K)[n, LENS[n]:] = -1  # no loss from padding
    a["grad_loss"] = np.full(ROWS, 1.0 / max(1, int(LENS.sum())), np.float32)
    return a


def reference(a):
    """(loss per row, gradients by name) in 64 bits."""
    t = {n: torch.tensor(v, dtype=torch.float64, requires_grad=True) for n, v in a.items() if n not in ("index", "top", "grad_loss")}
    qkv = (t["x"] @ t["wqkv"]).reshape(B, S, HQ + 2 * HK, D).transpose(1, 2)
    q, k, v = qkv[:, :HQ], qkv[:, HQ:HQ + HK].repeat_interleave(HQ // HK, 1), qkv[:, HQ + HK:].repeat_interleave(HQ // HK, 1)
    lens = torch.tensor(LENS.astype(np.int64))[:, None, None]
    i, j = torch.arange(S)[:, None], torch.arange(S)[None]
    seen = ((i < lens) & (j < lens) & (j <= i))[:, None]
    p = torch.softmax((q @ k.transpose(-1, -2) / D ** 0.5).masked_fill(~seen, -1e300), -1) * seen
    y = t["x"] + (p @ v).transpose(1, 2).reshape(ROWS, MODEL) @ t["wo"]
    z = y @ t["wg"] + t["bg"]
    h = torch.nn.functional.silu(z[:, :HIDDEN]) * z[:, HIDDEN:]
    logits = (y + h @ t["wd"]) @ t["wv"].T
    there = torch.tensor(a["index"] >= 0)
    some = there.any(1)
    lp = torch.log_softmax((torch.tensor(a["top"], dtype=torch.float64) / T).masked_fill(~there & some[:, None], -1e300), 1)
    lq = torch.log_softmax(logits / T, 1).gather(1, torch.tensor(a["index"].astype(np.int64)).clamp(min=0))
    loss = T * T * torch.where(there, lp.exp() * (lp - lq), 0.0).sum(1) * some
    (loss * torch.tensor(a["grad_loss"], dtype=torch.float64)).sum().backward()
    return loss.detach().numpy(), {n: x.grad.numpy() for n, x in t.items()}


class Step:
    def __init__(self, ctx, a):
        self.ctx, new = ctx, ctx.alloc
        up = lambda v: ctx.to_device(v if v.dtype == np.float32 else v.view(np.float32))  # noqa: E731
        self.d = {n: up(v) for n, v in a.items()}
        self.lens, self.zeros = up(LENS), new(2 * HIDDEN).fill(0.0)
        self.b = {n: new(s) for n, s in dict(
            qkv=ROWS * QKV, att=ROWS * MODEL, lse=B * HQ * S, y=ROWS * MODEL, z=ROWS * 2 * HIDDEN, h=ROWS * HIDDEN, out=ROWS * MODEL,
            logits=ROWS * VOCAB, loss=ROWS, loss_lse=ROWS, g_out=ROWS * MODEL, g_h=ROWS * HIDDEN, g_y=ROWS * MODEL, g_att=ROWS * MODEL,
            g_qkv=ROWS * QKV).items()}
        self.g = {n: new(a[n].size) for n in ("x", "wqkv", "wo", "wg", "bg", "wd", "wv")}

    def attention(self, call, *more):
        b, at = self.b, (0, HQ * D, (HQ + HK) * D)
        tensors = [b["qkv"].offset(o) for o in at] + [b["att"], b["lse"]]
        if more:
            tensors += [b["g_att"]] + [b["g_qkv"].offset(o) for o in at]
        st, so = (S * QKV, D, QKV), (S * MODEL, D, MODEL)
        call(*tensors, B, HQ, HK, S, S, D, D ** -0.5, True, self.lens, self.lens, st, st, so)

    def __call__(self):
        c, d, b, g = self.ctx, self.d, self.b, self.g
        mm = c.sgemm
        mm("nn", ROWS, QKV, MODEL, d["x"], MODEL, d["wqkv"], QKV, b["qkv"], QKV)
        self.attention(c.mha_forward)
        c.copy(b["y"].ptr, d["x"].ptr, ROWS * MODEL)
        mm("nn", ROWS, MODEL, MODEL, b["att"], MODEL, d["wo"], MODEL, b["y"], MODEL, True)
        c.gated_dense_forward("silu", b["y"], d["wg"], d["bg"], b["z"], b["h"], ROWS, MODEL, HIDDEN)
        c.copy(b["out"].ptr, b["y"].ptr, ROWS * MODEL)
        mm("nn", ROWS, MODEL, HIDDEN, b["h"], HIDDEN, d["wd"], MODEL, b["out"], MODEL, True)
        mm("nt", ROWS, VOCAB, MODEL, b["out"], MODEL, d["wv"], MODEL, b["logits"], VOCAB)
        c.distill_forward(b["logits"], VOCAB, d["index"], d["top"], b["loss"], b["loss_lse"], ROWS, VOCAB, K, T)
        # backward; the logits' gradient takes their place
        c.distill_backward(b["logits"], VOCAB, d["index"], d["top"], b["loss_lse"], d["grad_loss"], b["logits"], VOCAB, ROWS, VOCAB, K, T)
        mm("nn", ROWS, MODEL, VOCAB, b["logits"], VOCAB, d["wv"], MODEL, b["g_out"], MODEL)
        mm("tn", VOCAB, MODEL, ROWS, b["logits"], VOCAB, b["out"], MODEL, g["wv"], MODEL)
        mm("nt", ROWS, HIDDEN, MODEL, b["g_out"], MODEL, d["wd"], MODEL, b["g_h"], HIDDEN)
        mm("tn", HIDDEN, MODEL, ROWS, b["h"], HIDDEN, b["g_out"], MODEL, g["wd"], MODEL)
        c.copy(g["bg"].ptr, self.zeros.ptr, 2 * HIDDEN)
        c.gated_dense_backward("silu", b["y"], d["wg"], b["z"], b["g_h"], b["z"], b["g_y"], g["wg"], g["bg"], ROWS, MODEL, HIDDEN)
        c.add_bias(b["g_y"], b["g_out"], 1, ROWS * MODEL)  # the residual
        mm("nt", ROWS, MODEL, MODEL, b["g_y"], MODEL, d["wo"], MODEL, b["g_att"], MODEL)
        mm("tn", MODEL, MODEL, ROWS, b["att"], MODEL, b["g_y"], MODEL, g["wo"], MODEL)
        self.attention(c.mha_backward, True)
        c.copy(g["x"].ptr, b["g_y"].ptr, ROWS * MODEL)
        mm("nt", ROWS, MODEL, QKV, b["g_qkv"], QKV, d["wqkv"], QKV, g["x"], MODEL, True)
        mm("tn", MODEL, QKV, ROWS, d["x"], MODEL, b["g_qkv"], QKV, g["wqkv"], QKV)

    def read(self):
        return self.b["loss"].download(), {n: t.download() for n, t in self.g.items()}

    def spoil(self):
        for t in (*self.b.values(), *self.g.values()):
            t.fill(float("nan"))


def test_a_training_step():
    from zigneuron_amd import Context
    a = inputs()
    loss, grads = reference(a)
    with Context(0) as ctx:
        announce("a block's training step")
        step = Step(ctx, a)
        step.spoil()
        step()
        got_loss, got = step.read()
        # Each value is a chain of sums of at most 501 products, eight deep from the input to a gradient and back: against the
        # norm of the whole tensor an fp32 sum of n products is off by at most n u, and a sum of independent roundings by about
        # sqrt(n) u; 8 links of 501 u would be 2.4e-4.
        bound = 8 * 501 * 2.0 ** -24
        assert np.linalg.norm(got_loss - loss) <= bound * np.linalg.norm(loss)
        for n, want in grads.items():
            off = np.linalg.norm(got[n].reshape(want.shape) - want) / np.linalg.norm(want)
            assert off <= bound, (n, off)
        # padding: no loss, and nothing of it in the input's gradient
        pad = (np.arange(S)[None] >= LENS[:, None]).reshape(-1)
        assert (got_loss[pad] == 0).all() and (got["x"].reshape(ROWS, MODEL)[pad] == 0).all()
        graph = ctx.capture(step)
        for _ in range(3):
            for go in (graph.launch, step):
                step.spoil()
                go()
                again_loss, again = step.read()
                assert np.array_equal(again_loss, got_loss)
                for n in got:
                    assert np.array_equal(again[n], got[n]), n
        graph.close()
