"""The operators that train one block of a language model, as measurable cases.

Three operators, each forward and backward, float32 throughout:
  mha      multi-head attention with shared key/value heads, causal and
           length masks and strided tensors (``Context.mha_forward``, which
           also writes each row's log-sum-exp, and ``Context.mha_backward``,
           which recomputes the probabilities from it);
  gated    the gated feed-forward projections h = act(gate) * up,
           [gate | up] = x . W + b (``Context.gated_dense_forward`` and
           ``Context.gated_dense_backward``);
  distill  the divergence of a teacher's top logits from a student's
           distribution over the whole vocabulary
           (``Context.distill_forward`` and ``Context.distill_backward``).

With ``own`` false a pass computes the operator with elementary torch
operations; with ``own`` true it makes the framework's calls.
"""
import math

import torch

own = False
_handles = {}

GATES = ("linear", "relu", "sigmoid", "tanh", "silu", "gelu")


def _ctx():
    """The device context a program creates once and keeps."""
    if "ctx" not in _handles:
        from zigneuron_amd import Context
        _handles["ctx"] = Context(0)
    return _handles["ctx"]


# ------------------------------------------------------------------ the cases
def _mha(way, batch, q_heads, kv_heads, q_len, kv_len, dim, causal=False, ragged=False, layout="bhsd"):
    return {"kind": "mha_" + way, "batch": batch, "q_heads": q_heads, "kv_heads": kv_heads, "q_len": q_len,
            "kv_len": kv_len, "dim": dim, "causal": causal, "ragged": ragged, "layout": layout}


def _gated(way, batch, inp, hidden, act="silu", bias=False, keep=True):
    return {"kind": "gated_" + way, "batch": batch, "inp": inp, "hidden": hidden, "act": act, "bias": bias, "keep": keep}


def _distill(way, rows, vocab, k, temperature=2.0):
    return {"kind": "distill_" + way, "rows": rows, "vocab": vocab, "k": k, "temperature": temperature}


def listed():
    return [
        # one new token for each of 8 requests, against what 2048 positions left behind: the call where latency counts
        {"name": "mha_token", **_mha("forward", 8, 16, 4, 1, 2048, 64, causal=True)},
        # a causal training forward, 4 query heads to a key/value head
        {"name": "mha_causal", **_mha("forward", 2, 16, 4, 2048, 2048, 128, causal=True, layout="fused")},
        # the backward of 128 heads of 1024 positions and 64 dimensions, no mask
        {"name": "mha_grad", **_mha("backward", 8, 16, 16, 1024, 1024, 64)},
        # the largest: causal backward of long sequences, 4 query heads to a key/value head
        {"name": "mha_grad_long", **_mha("backward", 2, 32, 8, 4096, 4096, 128, causal=True)},
        # a padded batch of odd lengths in one projection's output, an odd head dimension
        {"name": "mha_grad_ragged", **_mha("backward", 12, 10, 5, 333, 333, 76, causal=True, ragged=True, layout="fused")},
        # one small sequence: few workgroups
        {"name": "mha_grad_small", **_mha("backward", 1, 4, 4, 256, 256, 64, causal=True)},
        # the feed-forward projections of 4 tokens being served: the weights are read once
        {"name": "gated_serve", **_gated("forward", 4, 1024, 4096, keep=False)},
        # the same layer in training
        {"name": "gated_step", **_gated("forward", 4096, 1024, 4096)},
        {"name": "gated_grad", **_gated("backward", 4096, 1024, 4096)},
        # no extent a multiple of 4, with bias
        {"name": "gated_grad_ragged", **_gated("backward", 777, 1023, 1001, act="gelu", bias=True)},
        # the loss over a batch's tokens, 64 teacher logits for each
        {"name": "distill_loss", **_distill("forward", 4096, 32000, 64)},
        # its gradient, an odd vocabulary
        {"name": "distill_grad", **_distill("backward", 1000, 50257, 20)},
    ]


def _log(rng, lo, hi):
    """An integer spread over [lo, hi] on a logarithmic scale."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    way = rng.choice(("forward", "backward", "backward"))
    op = rng.choice(("mha", "mha", "mha", "gated", "gated", "distill"))
    if op == "mha":
        while True:
            kv_heads, length = _log(rng, 1, 16), _log(rng, 1, 4096)
            other = length if rng.random() < 0.6 else _log(rng, 1, 4096)
            c = _mha(way, _log(rng, 1, 16), kv_heads * rng.choice((1, 1, 2, 4, 7)), kv_heads, other, length,
                     _log(rng, 16, 128), rng.random() < 0.6, rng.random() < 0.4, rng.choice(("bhsd", "bshd", "fused")))
            if c["layout"] == "fused" and other != length:
                c["layout"] = "bshd"
            pairs = c["batch"] * c["q_heads"] * c["q_len"] * c["kv_len"]
            if pairs * c["dim"] <= 64 * 4096 * 4096 * 64 and pairs <= 64 * 4096 * 4096:
                return c
    if op == "gated":
        while True:
            c = _gated(way, _log(rng, 1, 8192), _log(rng, 16, 4096), _log(rng, 16, 8192), rng.choice(GATES),
                       rng.random() < 0.4, way == "backward" or rng.random() < 0.6)
            if c["batch"] * c["inp"] * c["hidden"] <= 4096 * 1024 * 4096:
                return c
    while True:
        c = _distill(way, _log(rng, 1, 8192), _log(rng, 100, 131072), _log(rng, 1, 100), rng.choice((1.0, 2.0, 4.0)))
        if c["rows"] * c["vocab"] <= 4096 * 32000 and c["k"] <= c["vocab"]:
            return c


# ------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)


def _zeros(*shape):
    return torch.zeros(shape, device="cuda", dtype=torch.float32)


def _heads(c, make):
    """(q, k, v) as [batch, heads, positions, dim] views of memory in the case's layout."""
    b, hq, hk, sq, sk, d = (c[x] for x in ("batch", "q_heads", "kv_heads", "q_len", "kv_len", "dim"))
    if c["layout"] == "fused":  # one projection's output: [batch, positions, q heads then k heads then v heads, dim]
        x = make(b, sq, hq + 2 * hk, d).transpose(1, 2)
        return x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:]
    if c["layout"] == "bshd":
        return tuple(make(b, s, h, d).transpose(1, 2) for h, s in ((hq, sq), (hk, sk), (hk, sk)))
    return make(b, hq, sq, d), make(b, hk, sk, d), make(b, hk, sk, d)


def _like_out(c, make):
    b, h, s, d = c["batch"], c["q_heads"], c["q_len"], c["dim"]
    return make(b, h, s, d) if c["layout"] == "bhsd" else make(b, s, h, d).transpose(1, 2)


def _lengths(c, gen):
    """Per sequence, the positions that hold tokens (an empty one among them), or None."""
    if not c["ragged"]:
        return None, None
    b, sq, sk = c["batch"], c["q_len"], c["kv_len"]
    kv = torch.randint(sk // 3, sk + 1, (b,), generator=gen, device="cuda", dtype=torch.int32)
    kv[0] = sk
    if b > 2:
        kv[b - 1] = 0
    return (kv if sq == sk else torch.clamp(kv, max=sq)).clone(), kv


def _mha_inputs(c, seed):
    gen = _gen(seed)
    q, k, v = _heads(c, lambda *s: _randn(gen, *s))
    q_lens, kv_lens = _lengths(c, gen)
    return {"q": q, "k": k, "v": v, "grad_out": _like_out(c, lambda *s: _randn(gen, *s)), "q_lens": q_lens, "kv_lens": kv_lens}


def _gated_inputs(c, seed):
    gen = _gen(seed)
    b, i, h = c["batch"], c["inp"], c["hidden"]
    s = {"x": _randn(gen, b, i), "w": _randn(gen, i, 2 * h) * math.sqrt(1.0 / i),
         "bias": _randn(gen, 2 * h) * 0.1 if c["bias"] else None}
    if c["kind"] == "gated_backward":
        s["z"], s["grad_h"] = _randn(gen, b, 2 * h), _randn(gen, b, h)
    return s


def _distill_inputs(c, seed):
    gen = _gen(seed)
    r, n, k = c["rows"], c["vocab"], c["k"]
    logits = _randn(gen, r, n) * 3
    teacher = logits + _randn(gen, r, n)
    top, index = teacher.topk(k, dim=1)
    index = index.to(torch.int32)
    # a teacher that keeps only what makes up most of its probability sends fewer for some tokens
    kept = torch.randint(1, k + 1, (r, 1), generator=gen, device="cuda")
    index[torch.arange(k, device="cuda")[None] >= kept] = -1
    if r > 3:  # tokens of the prompt, which the loss leaves out
        index[torch.rand(r, generator=gen, device="cuda") < 0.2] = -1
    return {"logits": logits, "index": index.contiguous(), "top": top.contiguous(),
            "grad_loss": torch.rand(r, generator=gen, device="cuda") / r}


def prepare(case, seed):
    c = case
    if c["kind"].startswith("mha"):
        s = _mha_inputs(c, seed)
        if c["kind"] == "mha_forward":
            del s["grad_out"]
            s["out"], s["lse"] = _like_out(c, _zeros), _zeros(c["batch"], c["q_heads"], c["q_len"])
        else:
            s["out"], s["lse"] = _like_out(c, _zeros), None
            out, s["lse"] = _mha_forward(c, s)
            s["out"].copy_(out)
            s["grad_q"], s["grad_k"], s["grad_v"] = _heads(c, _zeros)
    elif c["kind"].startswith("gated"):
        s = _gated_inputs(c, seed)
        b, i, h = c["batch"], c["inp"], c["hidden"]
        if c["kind"] == "gated_forward":
            s["z"], s["h"] = _zeros(b, 2 * h) if c["keep"] else None, _zeros(b, h)
        else:
            s.update(grad_z=_zeros(b, 2 * h), grad_x=_zeros(b, i), grad_w=_zeros(i, 2 * h),
                     grad_bias=_zeros(2 * h) if c["bias"] else None, zeros=_zeros(2 * h))
    else:
        s = _distill_inputs(c, seed)
        if c["kind"] == "distill_forward":
            s["loss"], s["lse"] = _zeros(c["rows"]), _zeros(c["rows"])
        else:
            s["lse"] = torch.where((s["index"] >= 0).any(1), torch.logsumexp(s["logits"] / c["temperature"], 1), 0.0)
            s["grad_logits"] = _zeros(c["rows"], c["vocab"])
    s["case"] = dict(c)
    return s


# ------------------------------------------------------------------ the plain forms
def _mask(c, s):
    """[batch or 1, 1, 1, q_len, kv_len]: the pairs that attend, the causal edge at the sequences' ends."""
    i = torch.arange(c["q_len"], device="cuda")[:, None]
    j = torch.arange(c["kv_len"], device="cuda")[None]
    if s["q_lens"] is None:
        m = j <= i + (c["kv_len"] - c["q_len"]) if c["causal"] else torch.ones_like(i + j, dtype=torch.bool)
        return m[None, None, None]
    ql, kl = (s[x].to(torch.int64)[:, None, None] for x in ("q_lens", "kv_lens"))
    m = (i < ql) & (j < kl)
    if c["causal"]:
        m = m & (j <= i + kl - ql)
    return m[:, None, None]


def _grouped(c, t):
    """[batch, q heads, ...] as [batch, kv heads, q heads of each, ...]."""
    return t.reshape(t.shape[0], c["kv_heads"], c["q_heads"] // c["kv_heads"], *t.shape[2:])


def _mha_forward(c, s):
    q, k, v = _grouped(c, s["q"]), s["k"][:, :, None], s["v"][:, :, None]
    score = torch.matmul(q, k.transpose(-1, -2)) * (1 / math.sqrt(c["dim"]))
    score = score.masked_fill(~_mask(c, s), -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v) / torch.where(total > 0, total, 1.0)
    lse = (top + torch.log(total)).squeeze(-1)
    return out.reshape(s["q"].shape), lse.reshape(s["q"].shape[:-1])


def _mha_backward(c, s):
    scale = 1 / math.sqrt(c["dim"])
    q, g, o, lse = (_grouped(c, s[x]) for x in ("q", "grad_out", "out", "lse"))
    k, v = s["k"][:, :, None], s["v"][:, :, None]
    score = torch.matmul(q, k.transpose(-1, -2)) * scale
    p = torch.exp(score - lse[..., None]).masked_fill(~_mask(c, s), 0.0)
    gv = torch.matmul(p.transpose(-1, -2), g).sum(2)
    ds = p * (torch.matmul(g, v.transpose(-1, -2)) - (g * o).sum(-1, keepdim=True))
    gq = torch.matmul(ds, k) * scale
    gk = torch.matmul(ds.transpose(-1, -2), q).sum(2) * scale
    return {"grad_q": gq.reshape(s["q"].shape), "grad_k": gk, "grad_v": gv}


def _gate(act, g):
    """act(g) and its derivative."""
    if act == "linear":
        return g, torch.ones_like(g)
    if act == "relu":
        return g.clamp(min=0), (g > 0).to(g.dtype)
    if act == "tanh":
        t = torch.tanh(g)
        return t, 1 - t * t
    if act == "gelu":  # the tanh form
        a = math.sqrt(2 / math.pi)
        t = torch.tanh(a * (g + 0.044715 * g * g * g))
        return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * a * (1 + 3 * 0.044715 * g * g)
    y = 1 / (1 + torch.exp(-g))
    return (y, y * (1 - y)) if act == "sigmoid" else (g * y, y * (1 + g * (1 - y)))


def _gated_forward(c, s):
    z = torch.matmul(s["x"], s["w"])
    if s["bias"] is not None:
        z = z + s["bias"]
    h = _gate(c["act"], z[:, :c["hidden"]])[0] * z[:, c["hidden"]:]
    return {"h": h, "z": z if c["keep"] else None}


def _gated_backward(c, s):
    y, dy = _gate(c["act"], s["z"][:, :c["hidden"]])
    gz = torch.cat((s["grad_h"] * s["z"][:, c["hidden"]:] * dy, s["grad_h"] * y), 1)
    return {"grad_z": gz, "grad_x": torch.matmul(gz, s["w"].t()), "grad_w": torch.matmul(s["x"].t(), gz),
            "grad_bias": gz.sum(0) if c["bias"] else None}


def _teacher(c, s):
    """The teacher's probabilities of its top entries (0 for absent ones), where they are, and the rows that have any."""
    there = s["index"] >= 0
    t = (s["top"] / c["temperature"]).masked_fill(~there, -math.inf)
    some = there.any(1, keepdim=True)
    t = t.masked_fill(~some, 0.0)
    e = torch.exp(t - t.amax(1, keepdim=True)).masked_fill(~there, 0.0)
    return e / torch.where(some, e.sum(1, keepdim=True), 1.0), s["index"].clamp(min=0).to(torch.int64), there, some


def _distill_forward(c, s):
    p, at, there, some = _teacher(c, s)
    z = s["logits"] / c["temperature"]
    top = z.amax(1, keepdim=True)
    lse = top + torch.log(torch.exp(z - top).sum(1, keepdim=True))
    term = p * (torch.log(torch.where(p > 0, p, 1.0)) - (z.gather(1, at) - lse))
    loss = c["temperature"] ** 2 * torch.where(there & (p > 0), term, 0.0).sum(1)
    return {"loss": loss, "lse": torch.where(some, lse, 0.0).squeeze(1)}


def _distill_backward(c, s):
    p, at, there, some = _teacher(c, s)
    g = torch.exp(s["logits"] / c["temperature"] - s["lse"][:, None]).scatter_add(1, at, -p)
    return {"grad_logits": torch.where(some, c["temperature"] * s["grad_loss"][:, None] * g, 0.0)}


# ------------------------------------------------------------------ one pass
def _p(t):
    return None if t is None else t.data_ptr()


def _strides(t):
    return t.stride(0), t.stride(1), t.stride(2)


def _mha_call(c, s):
    """What both directions take after their tensors."""
    return (c["batch"], c["q_heads"], c["kv_heads"], c["q_len"], c["kv_len"], c["dim"], 1 / math.sqrt(c["dim"]), c["causal"],
            _p(s["q_lens"]), _p(s["kv_lens"]), _strides(s["q"]), _strides(s["k"]), _strides(s["out"]))


def run(state):
    s, c = state, state["case"]
    kind = c["kind"]
    if not own:
        if kind == "mha_forward":
            out, lse = _mha_forward(c, s)
            return {"out": out, "lse": lse}
        return {"mha_backward": _mha_backward, "gated_forward": _gated_forward, "gated_backward": _gated_backward,
                "distill_forward": _distill_forward, "distill_backward": _distill_backward}[kind](c, s)
    ctx = _ctx()
    if kind == "mha_forward":
        ctx.mha_forward(_p(s["q"]), _p(s["k"]), _p(s["v"]), _p(s["out"]), _p(s["lse"]), *_mha_call(c, s))
        return {"out": s["out"], "lse": s["lse"]}
    if kind == "mha_backward":
        ctx.mha_backward(_p(s["q"]), _p(s["k"]), _p(s["v"]), _p(s["out"]), _p(s["lse"]), _p(s["grad_out"]), _p(s["grad_q"]),
                         _p(s["grad_k"]), _p(s["grad_v"]), *_mha_call(c, s))
        return {x: s[x] for x in ("grad_q", "grad_k", "grad_v")}
    if kind == "gated_forward":
        ctx.gated_dense_forward(c["act"], _p(s["x"]), _p(s["w"]), _p(s["bias"]), _p(s["z"]), _p(s["h"]), c["batch"], c["inp"],
                                c["hidden"])
        return {"h": s["h"], "z": s["z"]}
    if kind == "gated_backward":
        if c["bias"]:  # the bias gradient accumulates: a training loop clears it before each step
            ctx.copy(_p(s["grad_bias"]), _p(s["zeros"]), 2 * c["hidden"])
        ctx.gated_dense_backward(c["act"], _p(s["x"]), _p(s["w"]), _p(s["z"]), _p(s["grad_h"]), _p(s["grad_z"]), _p(s["grad_x"]),
                                 _p(s["grad_w"]), _p(s["grad_bias"]), c["batch"], c["inp"], c["hidden"])
        return {x: s[x] for x in ("grad_z", "grad_x", "grad_w", "grad_bias")}
    if kind == "distill_forward":
        ctx.distill_forward(_p(s["logits"]), c["vocab"], _p(s["index"]), _p(s["top"]), _p(s["loss"]), _p(s["lse"]), c["rows"],
                            c["vocab"], c["k"], c["temperature"])
        return {"loss": s["loss"], "lse": s["lse"]}
    ctx.distill_backward(_p(s["logits"]), c["vocab"], _p(s["index"]), _p(s["top"]), _p(s["lse"]), _p(s["grad_loss"]),
                         _p(s["grad_logits"]), c["vocab"], c["rows"], c["vocab"], c["k"], c["temperature"])
    return {"grad_logits": s["grad_logits"]}


def work(case):
    c, kind = case, case["kind"]
    if kind.startswith("mha"):
        b, hq, hk, sq, sk, d = (c[x] for x in ("batch", "q_heads", "kv_heads", "q_len", "kv_len", "dim"))
        if c["causal"]:  # visible pairs of one head: row i sees min(sk, i + 1 + sk - sq) keys
            pairs = sum(max(0, min(sk, i + 1 + sk - sq)) for i in range(sq))
        else:
            pairs = sq * sk
        if c["ragged"]:  # lengths between a third and all: about two thirds on average
            pairs = pairs * 0.48
        q, kv = b * hq * sq * d, b * hk * sk * d
        if kind == "mha_forward":  # two products; q, k, v read, out and the log-sum-exp written
            return {"bytes": 4 * (2 * q + 2 * kv + b * hq * sq), "flops": 4 * b * hq * pairs * d}
        # five products; q, k, v, out, grad_out, log-sum-exp read, three gradients written
        return {"bytes": 4 * (4 * q + 4 * kv + b * hq * sq), "flops": 10 * b * hq * pairs * d}
    if kind.startswith("gated"):
        b, i, h = c["batch"], c["inp"], c["hidden"]
        if kind == "gated_forward":
            return {"bytes": 4 * (b * i + 2 * i * h + b * h * (3 if c["keep"] else 1)), "flops": 4 * b * i * h}
        return {"bytes": 4 * (2 * b * i + 4 * i * h + 5 * b * h), "flops": 8 * b * i * h}
    r, n, k = c["rows"], c["vocab"], c["k"]
    share = 0.8 if r > 3 else 1.0  # a fifth of the rows are left out
    if kind == "distill_forward":
        return {"bytes": 4 * (share * r * n + 2 * r * k + 2 * r), "flops": 4 * share * r * n}
    return {"bytes": 4 * ((share + 1) * r * n + 2 * r * k + 2 * r), "flops": 4 * share * r * n}


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    c, kind = case, case["kind"]
    f8 = torch.float64
    if kind.startswith("mha"):
        s = _mha_inputs(c, seed)
        b, hq, hk, sq, sk, d = (c[x] for x in ("batch", "q_heads", "kv_heads", "q_len", "kv_len", "dim"))
        group = hq // hk
        res = {"out": torch.zeros(b, hq, sq, d, dtype=f8, device="cuda"),
               "lse": torch.full((b, hq, sq), -math.inf, dtype=f8, device="cuda")}
        if kind == "mha_backward":
            res = {x: torch.zeros(b, h, n, d, dtype=f8, device="cuda")
                   for x, h, n in (("grad_q", hq, sq), ("grad_k", hk, sk), ("grad_v", hk, sk))}
        for n in range(b):  # one head at a time, cut to the sequence's own positions
            lq, lk = (sq, sk) if s["q_lens"] is None else (int(s["q_lens"][n]), int(s["kv_lens"][n]))
            if lq == 0 or lk == 0:
                continue
            hidden = None
            if c["causal"]:
                hidden = torch.ones(lq, lk, device="cuda").triu(1 + lk - lq) > 0
            for h in range(hq):
                q, k, v = s["q"][n, h, :lq].to(f8), s["k"][n, h // group, :lk].to(f8), s["v"][n, h // group, :lk].to(f8)
                x = (q @ k.T) / d ** 0.5
                if hidden is not None:
                    x[hidden] = -math.inf
                lse = torch.logsumexp(x, 1)
                seen = lse > -math.inf
                p = torch.exp(x - torch.where(seen, lse, 0.0)[:, None])
                if kind == "mha_forward":
                    res["lse"][n, h, :lq] = lse
                    res["out"][n, h, :lq] = p @ v
                    continue
                g = s["grad_out"][n, h, :lq].to(f8)
                gp = g @ v.T
                gx = p * (gp - (p * gp).sum(1, keepdim=True)) / d ** 0.5
                res["grad_q"][n, h, :lq] = gx @ k
                res["grad_k"][n, h // group, :lk] += gx.T @ q
                res["grad_v"][n, h // group, :lk] += p.T @ g
        return res
    if kind.startswith("gated"):
        s = {x: None if t is None else t.to(f8) for x, t in _gated_inputs(c, seed).items()}
        n = c["hidden"]
        z = s["z"] if kind == "gated_backward" else s["x"] @ s["w"] + (0 if s["bias"] is None else s["bias"])
        gate = z[:, :n].clone().requires_grad_(True)
        act = {"linear": lambda t: t * 1, "relu": torch.relu, "sigmoid": torch.sigmoid, "tanh": torch.tanh,
               "silu": lambda t: t * torch.sigmoid(t),
               "gelu": lambda t: torch.nn.functional.gelu(t, approximate="tanh")}[c["act"]](gate)
        if kind == "gated_forward":
            return {"h": act.detach() * z[:, n:], "z": z if c["keep"] else None}
        slope, = torch.autograd.grad(act.sum(), gate)
        gz = torch.cat([slope * (s["grad_h"] * z[:, n:]), act.detach() * s["grad_h"]], dim=1)
        return {"grad_z": gz, "grad_x": gz @ s["w"].T, "grad_w": s["x"].T @ gz, "grad_bias": gz.sum(0) if c["bias"] else None}
    s, t = _distill_inputs(c, seed), c["temperature"]
    r, n = c["rows"], c["vocab"]
    res = {"grad_logits": torch.zeros(r, n, dtype=f8, device="cuda")}
    if kind == "distill_forward":
        res = {"loss": torch.zeros(r, dtype=f8, device="cuda"), "lse": torch.zeros(r, dtype=f8, device="cuda")}
    for a in range(0, r, 512):  # the teacher as a whole row of probabilities
        index, top = s["index"][a:a + 512].long(), s["top"][a:a + 512].to(f8)
        some = (index >= 0).any(1)
        p = torch.softmax(torch.where(index >= 0, top / t, -math.inf), 1).nan_to_num(0.0)
        full = torch.zeros(index.shape[0], n, dtype=f8, device="cuda").scatter_add_(1, index.clamp(min=0), p)
        logq = torch.log_softmax(s["logits"][a:a + 512].to(f8) / t, 1)
        if kind == "distill_forward":
            res["loss"][a:a + 512] = t * t * (torch.xlogy(full, full) - full * logq).sum(1) * some
            res["lse"][a:a + 512] = torch.logsumexp(s["logits"][a:a + 512].to(f8) / t, 1) * some
        else:
            g = s["grad_loss"][a:a + 512, None].to(f8)
            res["grad_logits"][a:a + 512] = (torch.exp(logq) - full) * g * t * some[:, None]
    return res
