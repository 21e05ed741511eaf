"""64-bit references of the language-model blocks (attention with shared heads,
gated Dense, distillation) and bounds of what fp32 arithmetic may lose.

Bounds.  u = 2^-24 is half a step of fp32.  A sum of n products in fp32, in
any order, each product rounded or split into three bf16 parts with the parts
below 2^-25 of it left out, is off by at most (n + 8) u times the sum of the
products' magnitudes (n - 1 additions, the product's own rounding and the left
out parts, a rounding of each operand where it was scaled, and second-order
terms).  DOT(n) is that factor.  An exponential is off by its argument's error
plus 4 u (two steps of the function and its result's rounding).
"""
import math

import numpy as np

U = 2.0 ** -24


def dot_err(n):
    return (n + 8) * U


class Mha:
    """One case's tensors as [batch, heads, positions, dim] float32 and its reference."""

    def __init__(self, q, k, v, scale, causal=False, q_lens=None, kv_lens=None):
        self.q, self.k, self.v = (np.asarray(t, np.float64) for t in (q, k, v))
        self.scale = float(np.float32(scale))
        b, hq, sq, d = q.shape
        _, hk, sk, _ = k.shape
        self.group = hq // hk
        self.shape = (b, hq, hk, sq, sk, d)
        self.seen = np.ones((b, sq, sk), bool)
        for n in range(b):
            ql = sq if q_lens is None else min(max(int(q_lens[n]), 0), sq)
            kl = sk if kv_lens is None else min(max(int(kv_lens[n]), 0), sk)
            i, j = np.arange(sq)[:, None], np.arange(sk)[None]
            m = (i < ql) & (j < kl)
            if causal:
                m &= j <= i + kl - ql
            self.seen[n] = m
        self.out = np.zeros(q.shape)
        self.lse = np.full((b, hq, sq), -np.inf)
        self.out_bound, self.lse_bound = np.zeros(q.shape), np.zeros((b, hq, sq))
        for n in range(b):
            for h in range(hq):
                p, lse, e, _ = self._probs(n, h)
                v = self._clean(self.v[n, h // self.group], n)
                self.lse[n, h], self.out[n, h] = lse, p @ v
                # each probability's relative error twice (its own and the sum's), and the sum over the keys
                self.out_bound[n, h] = (p * (2 * e + dot_err(sk))) @ np.abs(v) + U * np.abs(p @ v)
                self.lse_bound[n, h] = e[:, 0] + dot_err(sk) + 4 * U * np.abs(np.where(np.isfinite(lse), lse, 0))

    def _clean(self, t, n):
        """Rows that no query of sequence n sees hold anything: zeros for the products here."""
        return np.where(self.seen[n].any(0)[:, None], t, 0.0)

    def _probs(self, n, h):
        """P, lse, the relative error bound of each row's P [sq, 1] and the scores."""
        d = self.shape[5]
        seen = self.seen[n]
        q = np.where(seen.any(1)[:, None], self.q[n, h], 0.0)
        k = self._clean(self.k[n, h // self.group], n)
        s = np.where(seen, self.scale * (q @ k.T), -np.inf)
        mag = np.where(seen, abs(self.scale) * (np.abs(q) @ np.abs(k).T), 0.0)
        top = s.max(1, initial=-np.inf, keepdims=True)
        top = np.where(np.isfinite(top), top, 0.0)
        e = np.exp(s - top)
        total = e.sum(1, keepdims=True)
        with np.errstate(divide="ignore"):
            lse = (top + np.log(total))[:, 0]
        p = e / np.where(total > 0, total, 1.0)
        # the score's products; the scores and the log-sum-exp rounded in base 2 and back; the exponential
        worst = (np.abs(np.where(seen, s, 0.0)) + np.abs(np.where(np.isfinite(lse), lse, 0.0))[:, None]).max(1, initial=0.0)
        err = 1.05 * (dot_err(d) * mag.max(1, initial=0.0) + 4 * U * worst + 8 * U)
        return p, lse, err[:, None], s

    def backward(self, grad_out, out32, lse32):
        """(grad_q, grad_k, grad_v) and their bounds, the fp32 forward's out and lse given."""
        b, hq, hk, sq, sk, d = self.shape
        g_all = np.asarray(grad_out, np.float64)
        res = [np.zeros(s) for s in ((b, hq, sq, d), (b, hk, sk, d), (b, hk, sk, d))]
        bound = [np.zeros_like(t) for t in res]
        for n in range(b):
            for h in range(hq):
                kh = h // self.group
                p, lse, e, _ = self._probs(n, h)
                row = self.seen[n].any(1)[:, None]
                g, q = np.where(row, g_all[n, h], 0.0), np.where(row, self.q[n, h], 0.0)
                k, v = self._clean(self.k[n, kh], n), self._clean(self.v[n, kh], n)
                o = np.where(row, np.asarray(out32[n, h], np.float64), 0.0)
                # the given log-sum-exp stands for the exact one: its rounding moves the whole row
                with np.errstate(invalid="ignore"):
                    e = e + np.where(row[:, 0], np.abs(np.asarray(lse32[n, h], np.float64) - lse), 0.0)[:, None]
                dp, delta = g @ v.T, (g * o).sum(1, keepdims=True)
                true_delta = (g * (p @ v)).sum(1, keepdims=True)
                ds = p * (dp - true_delta)
                dp_err = dot_err(d) * (np.abs(g) @ np.abs(v).T)
                delta_err = dot_err(d) * (np.abs(g) * np.abs(o)).sum(1, keepdims=True) + np.abs(delta - true_delta)
                ds_err = 1.05 * (p * (e * np.abs(dp - true_delta) + dp_err + delta_err) + 4 * U * np.abs(ds))
                s = abs(self.scale)
                res[0][n, h] = self.scale * (ds @ k)
                res[1][n, kh] += self.scale * (ds.T @ q)
                res[2][n, kh] += p.T @ g
                bound[0][n, h] = s * ((ds_err + dot_err(sk) * np.abs(ds)) @ np.abs(k))
                bound[1][n, kh] += s * ((ds_err + dot_err(sq * self.group) * np.abs(ds)).T @ np.abs(q))
                bound[2][n, kh] += (p * (1.05 * e + dot_err(sq * self.group))).T @ np.abs(g)
        return res, bound


def gate(act, g):
    """(act(g), act'(g)) in 64 bits."""
    g = np.asarray(g, np.float64)
    if act == "linear":
        return g, np.ones_like(g)
    if act == "relu":
        return np.maximum(g, 0), (g > 0).astype(np.float64)
    if act == "tanh":
        t = np.tanh(g)
        return t, 1 - t * t
    if act == "gelu":
        a = math.sqrt(2 / math.pi)
        t = np.tanh(a * (g + 0.044715 * g ** 3))
        return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * a * (1 + 3 * 0.044715 * g * g)
    s = 1 / (1 + np.exp(-g))
    return (s, s * (1 - s)) if act == "sigmoid" else (g * s, s * (1 + g * (1 - s)))


def gate_err(act, g):
    """Absolute error bounds of an fp32 (act(g), act'(g)): a few roundings of each term that the formula adds.

    A transcendental is off by 4 u of its value, a quotient or product by u; tanh(x) near its limits and 1 + tanh by 4 u
    absolutely.  The argument of GELU's tanh is off by 5 u of |x|, which its slope 1 - t^2 carries."""
    y, d = gate(act, g)
    g = np.asarray(g, np.float64)
    if act in ("linear", "relu"):
        return np.zeros_like(g), np.zeros_like(g)
    if act == "gelu":
        a = math.sqrt(2 / math.pi)
        x = a * (np.abs(g) + 0.044715 * np.abs(g) ** 3)
        t = np.tanh(x)
        dt = 4 * U + 5 * U * x * (1 - t * t)
        slope = a * (1 + 3 * 0.044715 * g * g)
        return 0.5 * np.abs(g) * dt + 4 * U * np.abs(y), 0.5 * dt + 0.5 * np.abs(g) * slope * (2 * dt + 6 * U) + 4 * U * np.abs(d)
    s = 1 / (1 + np.exp(-g))
    if act == "tanh":
        return 5 * U * np.abs(y), 10 * U * np.ones_like(g)
    rel = (8 + np.abs(g)) * U  # the exponential's argument is exact, its value 4 u off
    return (rel * np.abs(y), rel * (np.abs(d) + s * np.abs(g) * (1 - s) + s))


class Distill:
    def __init__(self, logits, index, top, temperature):
        x = np.asarray(logits, np.float64) / float(np.float32(temperature))
        self.t = float(np.float32(temperature))
        rows, vocab = x.shape
        there = (index >= 0) & (index < vocab) & (top != -np.inf)
        self.some = there.any(1)
        z = np.where(there, np.asarray(top, np.float64) / self.t, -np.inf)
        z = z - np.where(self.some, z.max(1, initial=-np.inf), 0.0)[:, None]
        e = np.exp(z)
        self.p = e / np.where(self.some, e.sum(1), 1.0)[:, None]
        logp = z - np.log(np.where(self.some, e.sum(1), 1.0))[:, None]
        self.full = np.zeros((rows, vocab))
        self.at = np.where(there, index, 0)
        np.add.at(self.full, (np.arange(rows)[:, None], self.at), np.where(there, self.p, 0.0))
        self.top_x = x.max(1)
        self.sum = np.exp(x - self.top_x[:, None]).sum(1)
        lse = self.top_x + np.log(self.sum)
        self.q = np.exp(x - lse[:, None])
        diff = logp - (np.take_along_axis(x, self.at, 1) - lse[:, None])
        used = there & (self.p > 0)
        term = np.where(used, self.p * np.where(used, diff, 0.0), 0.0)
        self.loss = self.t ** 2 * term.sum(1) * self.some
        self.lse = np.where(self.some, lse, 0.0)
        # every logarithm and quotient is off by a few u of its value, the sum of the vocabulary by (n + 8) u of itself
        k = index.shape[1]
        size = np.abs(np.take_along_axis(x, self.at, 1)) + np.abs(lse)[:, None] + np.abs(np.where(used, logp, 0.0)) + \
            np.abs(np.where(there, top, 0.0)) / self.t
        unit = np.where(used, self.p * (8 * U * size + dot_err(vocab) + 8 * U), 0.0)
        self.loss_bound = self.t ** 2 * (unit.sum(1) + dot_err(k) * np.abs(term).sum(1) + (
            np.where(used, np.abs(self.p * np.where(used, diff, 0.0)) * (8 * U * (size + 1) + dot_err(k)), 0.0)).sum(1))
        self.lse_bound = dot_err(vocab) + 6 * U * (np.abs(lse) + np.abs(self.top_x))
        self.x, self.exact_lse = x, lse

    def backward(self, grad_loss, lse32):
        g = np.asarray(grad_loss, np.float64)[:, None] * self.t
        res = np.where(self.some[:, None], g * (self.q - self.full), 0.0)
        off = np.where(self.some, np.abs(np.asarray(lse32, np.float64) - self.exact_lse), 0.0)[:, None]
        x = np.where(np.isfinite(self.x), self.x, 0.0)  # exp(-inf) is 0 without any error
        err = self.q * (off + 6 * U * (np.abs(x) + np.abs(self.exact_lse)[:, None] + 1))
        k = self.at.shape[1]
        err = err + self.full * (dot_err(k) + 16 * U * (1 + np.abs(x)))
        return res, np.where(self.some[:, None], np.abs(g) * (1.05 * err + 4 * U * (self.q + self.full)), 0.0)


def check(got, ref, bound, what):
    """got within bound of ref everywhere (equal where ref is infinite)."""
    got = np.asarray(got, np.float64)
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    fine = np.isfinite(ref)
    assert np.array_equal(got[~fine], ref[~fine]), f"{what}: infinities differ"
    assert np.isfinite(got[fine]).all(), f"{what}: not finite"
    # a value below fp32's normal range may be flushed
    off = np.abs(got[fine] - ref[fine])
    over = off - (np.broadcast_to(bound, ref.shape)[fine] + 2.0 ** -126)
    assert not over.size or over.max() <= 0, f"{what}: {over.max():.3e} over its bound, worst error {off.max():.3e}"
