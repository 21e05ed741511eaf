"""The operators that serve a language model's attention, as measurable cases.

Three operators, which follow each other in a served (the first also in a
trained) block:
  rotary   rotary positions, forward and backward: pairs of a head's dims
           turned by the token's position times the pair's frequency
           (``Context.rotary_forward``, ``Context.rotary_backward``);
  append   the keys and values of new tokens into the pages of their
           sequences, keys (and queries) rotated on the way
           (``Context.paged_append``);
  attend   attention of each sequence's new tokens over its pages
           (``Context.paged_attention``).

The cache's pages hold float32 or bfloat16; everything else is float32.  With
``own`` false a pass computes the operator with elementary torch operations;
with ``own`` true it makes the framework's calls.
"""
import math
import random

import torch

own = False
_handles = {}

DIMS = (16, 32, 40, 48, 64, 64, 76, 80, 96, 100, 112, 120, 127, 128, 128)
PAGES = (8, 16, 16, 24, 32, 64, 100, 256)


def _ctx():
    """The device context a program creates once and keeps."""
    if "ctx" not in _handles:
        from zigneuron_amd import Context
        _handles["ctx"] = Context(0)
    return _handles["ctx"]


# ------------------------------------------------------------------ the cases
def _rotary(way, batch, heads, length, dim, rot, layout="half", memory="bshd", far=0):
    """far: the first positions lie up to there (0: every sequence starts at position 0)."""
    return {"kind": "rotary_" + way, "batch": batch, "heads": heads, "length": length, "dim": dim, "rot": rot, "layout": layout,
            "memory": memory, "far": far}


def _paged(kind, batch, q_heads, kv_heads, dim, new, kv_len, chunks="same", ragged=False, page=64, cache="f32", rot=0,
           layout="half", pad=0):
    """new: the most new tokens of a sequence; chunks: "same" for every sequence, "ragged" (any number up to it) or "mixed" (one
    sequence has them, the others a token each); ragged: lengths from a third of kv_len on; pad: rows behind the last sequence."""
    return {"kind": "paged_" + kind, "batch": batch, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "new": new,
            "kv_len": kv_len, "chunks": chunks, "ragged": ragged, "page": page, "cache": cache, "rot": rot, "layout": layout,
            "pad": pad}


def listed():
    return [
        # one new token of 8 requests, query and key heads of one projection's output: the call where latency counts
        {"name": "rotary_token", **_rotary("forward", 8, 20, 1, 64, 64, memory="fused", far=2048)},
        # query and key heads of a training step
        {"name": "rotary_step", **_rotary("forward", 2, 40, 4096, 128, 128, memory="fused")},
        # the gradient of a layer that rotates half of an odd head in pairs of neighbours
        {"name": "rotary_grad", **_rotary("backward", 3, 12, 2777, 76, 38, layout="interleaved", memory="bhsd")},
        # one new token of 64 requests into the cache, queries rotated with the keys
        {"name": "append_token", **_paged("append", 64, 16, 4, 64, 1, 2048, ragged=True, page=16, rot=64)},
        # prompts into a cache of 16-bit values
        {"name": "append_prompt", **_paged("append", 4, 32, 8, 128, 2048, 2048, cache="bf16", rot=128)},
        # chunks of all lengths, pages and heads that are no powers of two, part of the head rotated
        {"name": "append_ragged", **_paged("append", 24, 10, 5, 76, 500, 2000, "ragged", True, 24, rot=38, layout="interleaved", pad=9)},
        # one new token of 8 requests against 2048 positions
        {"name": "attend_token", **_paged("attention", 8, 16, 4, 64, 1, 2048, page=16)},
        # one new token of 64 requests of all lengths, cache in 16 bits
        {"name": "attend_served", **_paged("attention", 64, 32, 8, 128, 1, 8192, ragged=True, cache="bf16")},
        # guessed tokens checked at once: five new tokens of 16 requests
        {"name": "attend_guesses", **_paged("attention", 16, 16, 4, 128, 5, 4096, ragged=True, page=16, cache="bf16")},
        # the next 512 tokens of 4 long prompts
        {"name": "attend_chunk", **_paged("attention", 4, 32, 8, 128, 512, 8192, ragged=True)},
        # a whole prompt, cache in 16 bits
        {"name": "attend_prompt", **_paged("attention", 1, 32, 8, 128, 4096, 4096, cache="bf16")},
        # a prompt's chunk next to 23 requests with one token each, odd heads and pages
        {"name": "attend_mixed", **_paged("attention", 24, 10, 5, 76, 384, 1500, "mixed", True, 24, pad=9)},
    ]


def _log(rng, lo, hi):
    """An integer spread over [lo, hi] on a logarithmic scale."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _rot(rng, dim):
    """How many of a head's dims are rotated: an even number, often all."""
    return dim // 2 * 2 if rng.random() < 0.5 else 2 * rng.randint(1, dim // 2)


def draw(rng):
    op = rng.choice(("rotary", "append", "attention", "attention"))
    layout = rng.choice(("half", "interleaved"))
    dim = rng.choice(DIMS)
    if op == "rotary":
        while True:
            c = _rotary(rng.choice(("forward", "backward")), _log(rng, 1, 64), _log(rng, 1, 64), _log(rng, 1, 8192), dim,
                        _rot(rng, dim), layout, rng.choice(("bhsd", "bshd", "fused")), rng.choice((0, 4096, 1000000)))
            if c["batch"] * c["heads"] * c["length"] * c["dim"] <= 2 * 40 * 4096 * 128:
                return c
    while True:
        kv_heads, kv_len = _log(rng, 1, 16), _log(rng, 1, 8192)
        chunks = rng.choice(("same", "same", "ragged", "mixed"))
        new = 1 if chunks == "same" and rng.random() < 0.5 else _log(rng, 1, min(kv_len, 4096))
        c = _paged(op, _log(rng, 1, 64), kv_heads * rng.choice((1, 2, 4, 7, 8)), kv_heads, dim, new, kv_len, chunks,
                   rng.random() < 0.6, rng.choice(PAGES), rng.choice(("f32", "bf16")),
                   _rot(rng, dim) if op == "append" and rng.random() < 0.8 else 0, layout, rng.choice((0, 0, 5)))
        tokens, held, pairs = _counts(c)
        if held * c["kv_heads"] * c["dim"] <= 64 * 5500 * 8 * 128 and tokens * c["q_heads"] * c["dim"] <= 8192 * 32 * 128 and \
                pairs * c["q_heads"] * c["dim"] <= 4 * 512 * 5000 * 32 * 128:
            return c


# ------------------------------------------------------------------ the plan
def _plan(c):
    """(new tokens, positions held with them) of each sequence, which a serving program knows on the host too."""
    rng = random.Random(repr([c[x] for x in sorted(c) if x != "name"]))
    out = []
    for b in range(c["batch"]):
        if c["ragged"] and b > 1 and b == c["batch"] - 1:
            out.append((0, 0))  # a slot without a request
            continue
        new = {"same": c["new"], "ragged": rng.randint(0, c["new"]), "mixed": c["new"] if b == 0 else 1}[c["chunks"]]
        kv = rng.randint(c["kv_len"] // 3, c["kv_len"]) if c["ragged"] and b > 0 else c["kv_len"]
        out.append((new, max(new, kv)))
    return out


def _pairs(new, kv):
    """Pairs of a sequence's new tokens and the positions that each sees."""
    return new * (kv - new) + new * (new + 1) // 2


def _counts(c):
    """New tokens, positions held and visible pairs of the whole batch."""
    plan = _plan(c)
    return sum(n for n, _ in plan), sum(k for n, k in plan if n), sum(_pairs(n, k) for n, k in plan)


# ------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)


def _zeros(*shape):
    return torch.zeros(shape, device="cuda", dtype=torch.float32)


def _frequencies(rot):
    """The pairs' frequencies: base 10000, the slow half of them at an eighth of their speed for a longer context."""
    i = torch.arange(rot // 2, dtype=torch.float64)
    f = 10000.0 ** (-2 * i / max(rot, 2))
    return torch.where(i < rot // 4, f, f / 8).to(torch.float32).cuda()


def _memory(c, make):
    """A [batch, heads, length, dim] view of memory in the case's layout."""
    b, h, n, d = c["batch"], c["heads"], c["length"], c["dim"]
    if c["memory"] == "bhsd":
        return make(b, h, n, d)
    if c["memory"] == "bshd":
        return make(b, n, h, d).transpose(1, 2)
    return make(b, n, h + (h + 4) // 5, d).transpose(1, 2)[:, :h]  # value heads follow


def _rotary_inputs(c, seed):
    gen = _gen(seed)
    s = {"x": _memory(c, lambda *n: _randn(gen, *n)), "freq": _frequencies(c["rot"]), "positions": None}
    if c["far"]:
        first = torch.randint(0, c["far"], (c["batch"], 1), generator=gen, device="cuda", dtype=torch.int32)
        s["positions"] = (first + torch.arange(c["length"], device="cuda", dtype=torch.int32)).contiguous()
    return s


def _paged_inputs(c, seed):
    gen = _gen(seed)
    plan, ps = _plan(c), c["page"]
    tokens = sum(n for n, _ in plan) + c["pad"]
    need = [-(-k // ps) for _, k in plan]
    pages, most = sum(need) + 3, max(max(need), 1)
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.zeros(c["batch"], most, device="cuda", dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    starts = [0]
    for n, _ in plan:
        starts.append(starts[-1] + n)
    kind = torch.bfloat16 if c["cache"] == "bf16" else torch.float32
    s = {"plan": plan, "tokens": tokens, "total": starts[-1], "pages": pages, "most": most, "table": table,
         "starts": torch.tensor(starts, dtype=torch.int32, device="cuda"),
         "lens": torch.tensor([k for _, k in plan], dtype=torch.int32, device="cuda"),
         "max_new": max(n for n, _ in plan), "max_kv": max(k for _, k in plan)}
    for x in ("k_cache", "v_cache"):
        s[x] = torch.empty(pages, c["kv_heads"], ps, c["dim"], device="cuda", dtype=kind).normal_(generator=gen)
    # the projection's output: query, key and value heads of each token
    x = _randn(gen, tokens, c["q_heads"] + 2 * c["kv_heads"], c["dim"])
    hq, hk = c["q_heads"], c["kv_heads"]
    s["q"], s["k"], s["v"] = x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:]
    s["freq"] = _frequencies(c["rot"]) if c["rot"] else None
    return s


def prepare(case, seed):
    c = case
    if c["kind"].startswith("rotary"):
        s = _rotary_inputs(c, seed)
        s["y"] = _memory(c, _zeros)
    else:
        s = _paged_inputs(c, seed)
        s["out"] = _zeros(s["tokens"], c["q_heads"], c["dim"])
        if c["kind"] == "paged_attention":
            s["lse"] = _zeros(s["tokens"], c["q_heads"])
        s["first"] = torch.arange(s["tokens"], device="cuda")
    s["case"] = dict(c)
    return s


# ------------------------------------------------------------------ the plain forms
def _turn(x, angle, rot, layout, back=False):
    """The first `rot` of the last dim's values turned by `angle` (64 bits, one for each pair)."""
    cos, sin = torch.cos(angle).to(torch.float32), torch.sin(angle).to(torch.float32)
    if back:
        sin = -sin
    y = x.clone()
    if layout == "half":
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y[..., :rot // 2], y[..., rot // 2:rot] = a * cos - b * sin, a * sin + b * cos
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y[..., 0:rot:2], y[..., 1:rot:2] = a * cos - b * sin, a * sin + b * cos
    return y


def _rotary_plain(c, s):
    p = s["positions"] if s["positions"] is not None else torch.arange(c["length"], device="cuda")[None]
    angle = p.to(torch.float64)[:, None, :, None] * s["freq"].to(torch.float64)
    return _turn(s["x"], angle, c["rot"], c["layout"], c["kind"] == "rotary_backward")


def _append_plain(c, s):
    t = s["first"][:s["total"]]
    b = torch.searchsorted(s["starts"][1:], t.to(torch.int32), right=True)
    first, end, held = s["starts"][:-1][b].long(), s["starts"][1:][b].long(), s["lens"][b].long()
    p = held - (end - first) + t - first
    page, slot = s["table"][b, p // c["page"]].long(), p % c["page"]
    q, k, v = (s[x][:s["total"]] for x in ("q", "k", "v"))
    if c["rot"]:
        angle = p.to(torch.float64)[:, None, None] * s["freq"].to(torch.float64)
        q, k = _turn(q, angle, c["rot"], c["layout"]), _turn(k, angle, c["rot"], c["layout"])
    s["k_cache"][page, :, slot] = k.to(s["k_cache"].dtype)
    s["v_cache"][page, :, slot] = v.to(s["v_cache"].dtype)
    s["out"][:s["total"]] = q
    return {"k_cache": s["k_cache"], "v_cache": s["v_cache"], "q": s["out"]}


def _attend(c, q, k, v, kv):
    """q [n, new, q heads, dim], k and v [n, kv heads, positions, dim], kv [n]: the lengths."""
    n, new, hq, d = q.shape
    hk, length = k.shape[1], k.shape[2]
    q = q.reshape(n, new, hk, hq // hk, d).permute(0, 2, 3, 1, 4).reshape(n, hk, hq // hk * new, d)
    i = torch.arange(new, device="cuda")[None, :, None]
    j = torch.arange(length, device="cuda")[None, None]
    seen = (j <= i + (kv[:, None, None] - new))[:, None, None]
    score = torch.matmul(q, k.transpose(-1, -2)).reshape(n, hk, hq // hk, new, length) * (1 / math.sqrt(d))
    score = score.masked_fill(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.reshape(n, hk, hq // hk * new, length), v).reshape(n, hk, hq // hk, new, d) / total
    lse = (top + torch.log(total)).squeeze(-1)
    return out.permute(0, 3, 1, 2, 4).reshape(n * new, hq, d), lse.permute(0, 3, 1, 2).reshape(n * new, hq)


def _attention_plain(c, s):
    some = [b for b, (n, _) in enumerate(s["plan"]) if n]
    same = len({s["plan"][b][0] for b in some}) == 1 and some == list(range(some[0], some[-1] + 1))
    held = torch.as_tensor(s["lens"]).long()
    at = 0
    for group in ([some] if same else [[b] for b in some]):  # sequences with as many new tokens at once
        new, kv = s["plan"][group[0]][0], max(s["plan"][b][1] for b in group)
        table = s["table"][group[0]:group[-1] + 1, :-(-kv // c["page"])].long()
        k, v = (s[x][table].permute(0, 2, 1, 3, 4).reshape(len(group), c["kv_heads"], -1, c["dim"])[:, :, :kv].to(torch.float32)
                for x in ("k_cache", "v_cache"))
        n = len(group) * new
        q = s["q"][at:at + n].reshape(len(group), new, c["q_heads"], c["dim"])
        # positions past a sequence's length hold other sequences' values: masked, and finite
        s["out"][at:at + n], s["lse"][at:at + n] = _attend(c, q, k, v, held[group[0]:group[-1] + 1])
        at += n
    return {"out": s["out"], "lse": s["lse"]}


# ------------------------------------------------------------------ one pass
def _p(t):
    return None if t is None else t.data_ptr()


def _cache(c, s):
    """The framework's view of the pools, made once as a serving program does."""
    if "cache" not in s:
        from zigneuron_amd import PagedCache
        s["cache"] = PagedCache(_p(s["k_cache"]), _p(s["v_cache"]), _p(s["table"]), _p(s["lens"]), c["batch"], s["pages"], c["page"],
                                s["most"], c["kv_heads"], c["dim"], c["cache"])
    return s["cache"]


def run(state):
    s, c = state, state["case"]
    kind = c["kind"]
    if not own:
        if kind.startswith("rotary"):
            return _rotary_plain(c, s)
        return (_append_plain if kind == "paged_append" else _attention_plain)(c, s)
    ctx = _ctx()
    if kind.startswith("rotary"):
        call = ctx.rotary_forward if kind == "rotary_forward" else ctx.rotary_backward
        call(_p(s["x"]), _p(s["y"]), _p(s["freq"]), c["batch"], c["heads"], c["length"], c["dim"], c["rot"], c["layout"],
             positions=_p(s["positions"]), x_strides=s["x"].stride()[:3], y_strides=s["y"].stride()[:3])
        return s["y"]
    heads = (s["q"].stride(0), s["q"].stride(1))  # of one projection's output: the same for q, k and v
    if kind == "paged_append":
        ctx.paged_append(_cache(c, s), _p(s["starts"]), s["tokens"], _p(s["k"]), _p(s["v"]), heads, _p(s["q"]), _p(s["out"]),
                         c["q_heads"], heads, freq=_p(s["freq"]), rot_dim=c["rot"], layout=c["layout"])
        return {"k_cache": s["k_cache"], "v_cache": s["v_cache"], "q": s["out"]}
    ctx.paged_attention(_cache(c, s), _p(s["starts"]), s["tokens"], s["max_new"], s["max_kv"], _p(s["q"]), _p(s["out"]), _p(s["lse"]),
                        c["q_heads"], 1 / math.sqrt(c["dim"]), True, heads)
    return {"out": s["out"], "lse": s["lse"]}


def work(case):
    c = case
    if c["kind"].startswith("rotary"):
        values = c["batch"] * c["heads"] * c["length"] * c["dim"]
        return {"bytes": 8 * values, "flops": 3 * values * c["rot"] // c["dim"]}
    tokens, held, pairs = _counts(c)
    size = 2 if c["cache"] == "bf16" else 4
    q, kv = tokens * c["q_heads"] * c["dim"], c["kv_heads"] * c["dim"]
    if c["kind"] == "paged_append":
        return {"bytes": 8 * q + (8 + 2 * size) * tokens * kv, "flops": 3 * (q + tokens * kv) * c["rot"] // c["dim"]}
    return {"bytes": 8 * q + 4 * tokens * c["q_heads"] + 2 * size * held * kv, "flops": 4 * pairs * c["q_heads"] * c["dim"]}


# ------------------------------------------------------------------ 64 bits
def _complex(x, position, freq, rot, layout, sign=1.0):
    """Pairs as complex numbers times exp(i position freq); position broadcasts over x's dims but the last."""
    x = x.to(torch.float64)
    if not rot:
        return x
    head = x[..., :rot]
    pair = head.unflatten(-1, (2, rot // 2)).transpose(-1, -2) if layout == "half" else head.unflatten(-1, (rot // 2, 2))
    angle = sign * position.to(torch.float64)[..., None] * freq.to(torch.float64)
    z = torch.view_as_real(torch.complex(pair[..., 0], pair[..., 1]) * torch.polar(torch.ones_like(angle), angle))
    turned = (z.transpose(-1, -2) if layout == "half" else z).flatten(-2)
    return torch.cat((turned, x[..., rot:]), -1)


def exact(case, seed):
    c = case
    if c["kind"].startswith("rotary"):
        s = _rotary_inputs(c, seed)
        p = s["positions"]
        if p is None:
            p = torch.arange(c["length"], device="cuda").repeat(c["batch"], 1)
        return _complex(s["x"], p[:, None], s["freq"], c["rot"], c["layout"], -1.0 if c["kind"] == "rotary_backward" else 1.0)
    s = _paged_inputs(c, seed)
    plan, ps = s["plan"], c["page"]
    if c["kind"] == "paged_append":
        res = {"k_cache": s["k_cache"].to(torch.float64), "v_cache": s["v_cache"].to(torch.float64),
               "q": torch.zeros(s["tokens"], c["q_heads"], c["dim"], device="cuda", dtype=torch.float64)}
        at = 0
        for b, (new, kv) in enumerate(plan):
            rows = slice(at, at + new)
            p = torch.arange(kv - new, kv, device="cuda")
            k, q = (_complex(s[x][rows], p[:, None], s["freq"], c["rot"], c["layout"]) for x in ("k", "q"))
            res["q"][rows] = q
            for page in range((kv - new) // ps, -(-kv // ps) if new else 0):  # page by page
                lo, hi = max(kv - new, page * ps), min(kv, (page + 1) * ps)
                there = (int(s["table"][b, page]), slice(None), slice(lo - page * ps, hi - page * ps))
                part = slice(lo - (kv - new), hi - (kv - new))
                res["k_cache"][there] = k[part].transpose(0, 1)
                res["v_cache"][there] = s["v"][rows][part].transpose(0, 1).to(torch.float64)
            at += new
        return res
    out = torch.zeros(s["tokens"], c["q_heads"], c["dim"], device="cuda", dtype=torch.float64)
    lse = torch.zeros(s["tokens"], c["q_heads"], device="cuda", dtype=torch.float64)
    group, at = c["q_heads"] // c["kv_heads"], 0
    for b, (new, kv) in enumerate(plan):
        if not new:
            continue
        pages = s["table"][b, :-(-kv // ps)].long()
        hidden = torch.ones(new, kv, device="cuda").triu(1 + kv - new) > 0
        for h in range(c["kv_heads"]):
            k, v = (s[x][pages, h].reshape(-1, c["dim"])[:kv].to(torch.float64) for x in ("k_cache", "v_cache"))
            for g in range(h * group, (h + 1) * group):
                x = (s["q"][at:at + new, g].to(torch.float64) @ k.T) / c["dim"] ** 0.5
                x[hidden] = -math.inf
                lse[at:at + new, g] = torch.logsumexp(x, 1)
                out[at:at + new, g] = torch.softmax(x, 1) @ v
        at += new
    return {"out": out, "lse": lse}
