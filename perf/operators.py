"""Operators between a trained decoder and its next token: their cases, their plain forms and the framework's calls.

Families (``case["kind"]``); the framework's forms are functions of ``frankentorch_b200.ops.decode``:

* ``rotary``   ``rotary``: rotation of queries and keys by position in training, forward, and backward on their gradients.
* ``append``   ``paged_append``: keys and values of new tokens into a paged cache, rotated on the way, with the queries.
* ``attend``   ``paged_attention``: one new token per sequence over the paged cache, output and log-sum-exp.
* ``logits``   ``logits_process``: penalties for repeated tokens, biases and a grammar mask on the logits of a step.

Formulas.  A token at position ``p`` is turned, in each pair of elements ``(x0, x1)``, by the angle ``a = p w_i``:
``(x0 cos a - x1 sin a, x1 cos a + x0 sin a)``; the backward pass turns by ``-a``.  Position ``p`` of sequence ``b`` is row
``p % page`` of page ``table[b, p // page]``.  ``o = sum_t softmax_t(q k_t / sqrt(hd)) v_t`` over ``t < lengths[b]``; a sequence
of no tokens has ``o = 0`` and a log-sum-exp of ``-inf``.  A logit ``x`` of a token that occurred becomes ``x / r`` if positive and
``x r`` otherwise; then ``x - f n - p [n > 0] + bias`` with ``n`` its count among the generated tokens; what the mask does not
allow is ``-inf``.
"""
import math
import random

import torch

own = False
DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # queries and keys of a tiny model's training step: latency
        {"name": "rotary_tiny", "kind": "rotary", "batch": 2, "seq": 128, "heads": 2, "kv": 2, "hd": 64, "turn": 64,
         "pairs": "halves", "dtype": "bf16"},
        # a layer of a 1.3B decoder in training, micro-batch 4 x 2048
        {"name": "rotary_gpt_1b", "kind": "rotary", "batch": 4, "seq": 2048, "heads": 16, "kv": 16, "hd": 128,
         "turn": 128, "pairs": "halves", "dtype": "bf16"},
        # one conversation of GPT-2 small: one token, learned positions, so nothing is turned; latency
        {"name": "append_one", "kind": "append", "batch": 1, "seq": 1, "heads": 12, "kv": 12, "hd": 64, "turn": 0,
         "pairs": "halves", "page": 16, "longest": 300, "dtype": "bf16"},
        # a step of a full serving batch of the 1.3B decoder
        {"name": "append_step", "kind": "append", "batch": 256, "seq": 1, "heads": 16, "kv": 16, "hd": 128, "turn": 128,
         "pairs": "halves", "page": 64, "longest": 2047, "dtype": "bf16"},
        # ragged prompts in a padded batch, grouped heads, a part of each head turned
        {"name": "append_prompts", "kind": "append", "batch": 16, "seq": 2048, "heads": 16, "kv": 4, "hd": 128,
         "turn": 64, "pairs": "neighbours", "page": 32, "longest": 0, "dtype": "bf16"},
        # one conversation of GPT-2 small: latency
        {"name": "attend_one", "kind": "attend", "batch": 1, "heads": 12, "kv": 12, "hd": 64, "page": 16, "shortest": 301,
         "longest": 301, "idle": 0, "dtype": "bf16"},
        # a ragged batch of the 1.3B decoder with some places not in use
        {"name": "attend_batch", "kind": "attend", "batch": 32, "heads": 16, "kv": 16, "hd": 128, "page": 64,
         "shortest": 20, "longest": 2048, "idle": 3, "dtype": "bf16"},
        # two long documents, grouped heads: little to do side by side but the length
        {"name": "attend_long", "kind": "attend", "batch": 2, "heads": 32, "kv": 4, "hd": 128, "page": 32,
         "shortest": 60001, "longest": 65537, "idle": 0, "dtype": "fp16"},
        # a full serving batch, ragged
        {"name": "attend_full", "kind": "attend", "batch": 128, "heads": 16, "kv": 16, "hd": 128, "page": 64,
         "shortest": 700, "longest": 4096, "idle": 0, "dtype": "bf16"},
        # one conversation over the GPT-2 vocabulary: latency
        {"name": "logits_one", "kind": "logits", "rows": 1, "vocab": 50257, "history": 301, "bias": True, "mask": False,
         "dtype": "bf16", "to": "fp32"},
        # a serving batch over the GPT-2 vocabulary with a grammar
        {"name": "logits_batch", "kind": "logits", "rows": 256, "vocab": 50257, "history": 2048, "bias": False,
         "mask": True, "dtype": "fp32", "to": "fp32"},
        # a full serving batch over a large vocabulary
        {"name": "logits_large", "kind": "logits", "rows": 512, "vocab": 128003, "history": 4096, "bias": True,
         "mask": True, "dtype": "bf16", "to": "bf16"},
    ]


def _log_int(rng, lo, hi, mult=1):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(mult, v // mult * mult)


MAX_BYTES = 1.2e9       # a drawn case stays below the largest listed ones
MAX_PADDED = 4.2e9      # bytes of the cache if all sequences were as long as the longest (the plain form computes on those)


def draw(rng):
    """One more case of the same families."""
    while True:
        kind = rng.choice(["rotary", "append", "attend", "attend", "logits"])
        hd = rng.choice([64, 128])
        group = rng.choice([1, 1, 2, 3, 4, 7, 8, 16])
        kv = _log_int(rng, 1, 16)
        c = {"kind": kind}
        if kind == "logits":
            dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
            c.update(rows=_log_int(rng, 1, 512), vocab=_log_int(rng, 500, 130000), history=_log_int(rng, 1, 8192),
                     bias=rng.random() < 0.5, mask=rng.random() < 0.5, dtype=dtype, to=rng.choice([dtype, "fp32"]))
        elif kind == "attend":
            longest = _log_int(rng, 1, 65536)
            c.update(batch=_log_int(rng, 1, 256), heads=kv * group, kv=kv, hd=hd, page=rng.choice([8, 16, 32, 64, 128]),
                     shortest=_log_int(rng, 1, longest), longest=longest, idle=rng.choice([0, 0, 1]),
                     dtype=rng.choice(["bf16", "bf16", "fp16"]))
            if c["idle"] >= c["batch"] or c["batch"] * longest * kv * hd * 4 > MAX_PADDED:
                continue
        else:
            c.update(batch=_log_int(rng, 1, 64), seq=_log_int(rng, 1, 2048), heads=kv * group, kv=kv, hd=hd,
                     turn=rng.choice([hd, hd, hd // 2]), pairs=rng.choice(["halves", "neighbours"]))
            if kind == "append":
                c.update(turn=rng.choice([0, c["turn"], c["turn"]]), page=rng.choice([8, 16, 32, 64, 128]),
                         longest=rng.choice([0, _log_int(rng, 1, 30000)]))
                if rng.random() < 0.5:
                    c.update(batch=_log_int(rng, 1, 256), seq=1)
            c.update(dtype=rng.choice(["bf16", "bf16", "fp16"]))
        if work(c)["bytes"] <= (MAX_BYTES if kind == "attend" else 3e8):
            return c


# ------------------------------------------------------------------------------------------------ lengths of a case
def _lengths(c):
    """Tokens in the cache of each sequence: a mix that goes by the case alone."""
    rng = random.Random("%s %s %s" % (c["batch"], c["longest"], c["page"]))
    if c["kind"] == "attend":
        n = [rng.randint(c["shortest"], c["longest"]) for _ in range(c["batch"])]
        n[rng.randrange(c["batch"])] = c["longest"]
        for b in rng.sample(range(c["batch"]), c["idle"]):
            n[b] = 0
        return n
    return [rng.randint(0, c["longest"]) for _ in range(c["batch"])]


def _counts(c):
    """New tokens of each sequence of an append: all of them, or ragged prompts."""
    rng = random.Random("%s %s" % (c["batch"], c["seq"]))
    return [rng.randint((c["seq"] + 3) // 4, c["seq"]) for _ in range(c["batch"])]


def _pages(c, ends):
    """(pages of each sequence, columns of the table, pages of the cache)."""
    need = [-(-n // c["page"]) for n in ends]
    return need, max(1, max(need)) + 1, sum(need) + 5


def _history(c):
    """(prompt tokens, tokens in all) of each row."""
    rng = random.Random("%s %s" % (c["rows"], c["history"]))
    total = [rng.randint((c["history"] + 1) // 2, c["history"]) for _ in range(c["rows"])]
    return [rng.randint(0, n) for n in total], total


def work(c):
    e = 4 if c["dtype"] == "fp32" else 2
    if c["kind"] == "rotary":
        n = c["batch"] * c["seq"] * (c["heads"] + c["kv"]) * c["hd"]
        return {"bytes": 4 * n * e + 8 * (c["turn"] // 2), "flops": 6 * n}
    if c["kind"] == "append":
        t = sum(_counts(c)) if c["seq"] > 1 else c["batch"]
        q = c["heads"] if c["turn"] else 0
        n = t * c["hd"] * (q + 2 * c["kv"])
        return {"bytes": 2 * n * e + 4 * t / c["page"] + 12 * c["batch"], "flops": 3 * t * c["turn"] * (q + c["kv"])}
    if c["kind"] == "attend":
        n = sum(_lengths(c))
        q = c["batch"] * c["heads"] * c["hd"]
        return {"bytes": (2 * n * c["kv"] * c["hd"] + 2 * q) * e + 4 * n / c["page"] + 4 * c["batch"] * (c["heads"] + 1),
                "flops": 4 * n * c["heads"] * c["hd"]}
    n = c["rows"] * c["vocab"]
    out = 4 if c["to"] == "fp32" else 2
    return {"bytes": n * (e + out) + (4 * c["vocab"] if c["bias"] else 0) + (n / 8 if c["mask"] else 0) +
            8 * sum(_history(c)[1]) + 20 * c["rows"], "flops": 5 * n}


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _n(g, dtype, *shape):
    return torch.randn(*shape, generator=g, device=DEV).to(dtype)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _frequencies(turn):
    return 10000.0 ** (-torch.arange(0, turn, 2, dtype=torch.float64, device=DEV) / turn)


def _cache(c, g, ends, dtype):
    """Pages in a shuffled order, as a cache has them after some use, and the table of each sequence."""
    need, cols, pages = _pages(c, ends)
    shape = (pages, c["kv"], c["page"], c["hd"])
    k, v = _n(g, dtype, *shape), _n(g, dtype, *shape)
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    first = torch.tensor([0] + need, device=DEV).cumsum(0)[:-1]
    at = torch.arange(cols, device=DEV)
    mine = at[None, :] < torch.tensor(need, device=DEV)[:, None]
    table = torch.where(mine, order[(first[:, None] + at[None, :]).clamp(max=pages - 1)], 0).to(torch.int32)
    return k, v, table


def prepare(c, seed):
    g = _gen(seed)
    dt = TYPES[c["dtype"]]
    if c["kind"] == "rotary":
        B, S, H, Hk, hd = (c[x] for x in ("batch", "seq", "heads", "kv", "hd"))
        return {"c": c, "qkv": _n(g, dt, B, S, H + 2 * Hk, hd), "dqkv": _n(g, dt, B, S, H + 2 * Hk, hd),
                "w": _frequencies(c["turn"])}
    if c["kind"] == "append":
        B, S, H, Hk, hd = (c[x] for x in ("batch", "seq", "heads", "kv", "hd"))
        start = _lengths(c)
        counts = _counts(c) if S > 1 else [1] * B
        k, v, table = _cache(c, g, [n + m for n, m in zip(start, counts)], dt)
        here = torch.arange(S, device=DEV)[None, :] < torch.tensor(counts, device=DEV)[:, None]
        return {"c": c, "qkv": _n(g, dt, B, S, H + 2 * Hk, hd), "k": k, "v": v, "table": table, "start": _i32(start),
                "counts": _i32(counts) if S > 1 else None, "w": _frequencies(c["turn"]) if c["turn"] else None,
                "tokens": here.nonzero(as_tuple=True)}
    if c["kind"] == "attend":
        lengths = _lengths(c)
        k, v, table = _cache(c, g, lengths, dt)
        # the queries of a step are a view into its packed projections
        qkv = _n(g, dt, c["batch"], c["heads"] + 2 * c["kv"], c["hd"])
        return {"c": c, "q": qkv[:, : c["heads"]], "k": k, "v": v, "table": table, "lengths": _i32(lengths)}
    R, V, L = c["rows"], c["vocab"], c["history"]
    prompt, total = _history(c)
    columns = (V + 127) // 128 * 128                      # the head's rows are padded to whole tiles
    logits = (3.0 * torch.randn(R, columns, generator=g, device=DEV)).to(dt)
    # text repeats itself: tokens are drawn from the low ids far more often than from the high ones
    tokens = (torch.rand(R, L, generator=g, device=DEV, dtype=torch.float64) ** 3 * V).long().clamp(max=V - 1)
    words = torch.randint(-2 ** 31, 2 ** 31 - 1, (R, (V + 31) // 32), generator=g, device=DEV, dtype=torch.int64)
    return {"c": c, "logits": logits, "tokens": tokens, "prompt": _i32(prompt), "total": _i32(total),
            "repetition": 1.0 + torch.rand(R, generator=g, device=DEV),
            "frequency": torch.rand(R, generator=g, device=DEV), "presence": torch.rand(R, generator=g, device=DEV),
            "bias": torch.randn(V, generator=g, device=DEV) if c["bias"] else None,
            "allowed": words.to(torch.int32) if c["mask"] else None}


def _split(s):
    """Views of the packed projections: queries, keys, values."""
    H, Hk = s["c"]["heads"], s["c"]["kv"]
    return (t for t in s["qkv"].split([H, Hk, Hk], dim=2))


# ------------------------------------------------------------------------------------------------ plain forms
def _turned(x, start, w, pairs, sign):
    """Elementary form of the rotation: angles in 64 bits, products in 32, one rounding."""
    B, S = x.shape[:2]
    n = w.shape[0]
    p = start.double()[:, None] + torch.arange(S, device=x.device, dtype=torch.float64)
    a = (p[:, :, None] * w)[:, :, None, :]
    cos, sin = a.cos().float(), (sign * a.sin()).float()
    y = x.float()
    part, rest = y[..., : 2 * n], y[..., 2 * n:]
    if pairs == "halves":
        x0, x1 = part[..., :n], part[..., n:]
        part = torch.cat([x0 * cos - x1 * sin, x1 * cos + x0 * sin], -1)
    else:
        x0, x1 = part[..., 0::2], part[..., 1::2]
        part = torch.stack([x0 * cos - x1 * sin, x1 * cos + x0 * sin], -1).flatten(-2)
    return torch.cat([part, rest], -1).to(x.dtype)


def _plain_append(s):
    c = s["c"]
    q, k, v = _split(s)
    b, i = s["tokens"]
    qr = None
    if s["w"] is not None:
        qr = q.clone()
        qr[b, i] = _turned(q, s["start"], s["w"], c["pairs"], 1.0)[b, i]
        k = _turned(k, s["start"], s["w"], c["pairs"], 1.0)
    p = s["start"].long()[b] + i
    page, row = s["table"].long()[b, p // c["page"]], p % c["page"]
    s["k"][page, :, row] = k[b, i]
    s["v"][page, :, row] = v[b, i]
    return {"k": s["k"], "v": s["v"], "q": qr}


def _plain_attend(s):
    c = s["c"]
    B, Hk, hd = c["batch"], c["kv"], c["hd"]
    t = s["table"].long()
    rows = t.shape[1] * c["page"]
    here = torch.arange(rows, device=t.device)[None, :] < s["lengths"][:, None]
    k = s["k"][t].transpose(1, 2).reshape(B, Hk, rows, hd).float()
    x = torch.matmul(s["q"].float().reshape(B, Hk, -1, hd), k.transpose(2, 3)) / math.sqrt(hd)
    del k
    x = torch.where(here[:, None, None, :], x, -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    v = torch.where(here[:, None, :, None], s["v"][t].transpose(1, 2).reshape(B, Hk, rows, hd).float(), 0.0)
    o = torch.matmul(p, v) / torch.where(total == 0, 1.0, total)
    lse = top + torch.log(total)
    return {"o": o.reshape(B, c["heads"], hd).to(s["q"].dtype), "lse": lse.reshape(B, c["heads"])}


def _plain_logits(s):
    c = s["c"]
    V = c["vocab"]
    x = s["logits"][:, :V].float()
    at = torch.arange(s["tokens"].shape[1], device=x.device)[None, :]
    there = (at < s["total"][:, None]).float()
    made = there * (at >= s["prompt"][:, None])
    seen = torch.zeros_like(x).scatter_add_(1, s["tokens"], there) > 0
    n = torch.zeros_like(x).scatter_add_(1, s["tokens"], made)
    r = s["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    x = x - s["frequency"][:, None] * n - s["presence"][:, None] * (n > 0)
    if s["bias"] is not None:
        x = x + s["bias"]
    if s["allowed"] is not None:
        ids = torch.arange(V, device=x.device)
        x = torch.where((s["allowed"][:, ids // 32] >> (ids % 32)) & 1 == 1, x, -math.inf)
    return x.to(TYPES[c["to"]])


def run(s):
    c = s["c"]
    if own:
        return _run_own(s)
    if c["kind"] == "rotary":
        zero = torch.zeros(c["batch"], dtype=torch.int32, device=DEV)
        q, k, _ = _split(s)
        dq, dk, _ = _split({"c": c, "qkv": s["dqkv"]})
        return {"q": _turned(q, zero, s["w"], c["pairs"], 1.0), "k": _turned(k, zero, s["w"], c["pairs"], 1.0),
                "dq": _turned(dq, zero, s["w"], c["pairs"], -1.0), "dk": _turned(dk, zero, s["w"], c["pairs"], -1.0)}
    if c["kind"] == "append":
        return _plain_append(s)
    if c["kind"] == "attend":
        return _plain_attend(s)
    return _plain_logits(s)


# ------------------------------------------------------------------------------------------------ the framework's calls
def _run_own(s):
    from frankentorch_b200.ops import decode as D
    c = s["c"]
    if c["kind"] == "logits":
        return D.logits_process(s["logits"], vocab=c["vocab"], tokens=s["tokens"], lengths=s["total"],
                                prompt_lengths=s["prompt"], repetition=s["repetition"], frequency=s["frequency"],
                                presence=s["presence"], bias=s["bias"], allowed=s["allowed"], out_dtype=TYPES[c["to"]])
    if c["kind"] == "attend":
        o, lse = D.paged_attention(s["q"], s["k"], s["v"], s["table"], s["lengths"])
        return {"o": o, "lse": lse}
    interleaved = c["pairs"] == "neighbours"
    q, k, v = _split(s)
    if c["kind"] == "append":
        turned = None
        if s["w"] is not None:
            turned = D.paged_append(s["k"], s["v"], s["table"], k, v, s["start"], s["counts"], q=q, inv_freq=s["w"],
                                    interleaved=interleaved)
        else:
            D.paged_append(s["k"], s["v"], s["table"], k, v, s["start"], s["counts"])
        return {"k": s["k"], "v": s["v"], "q": turned}
    dq, dk, _ = _split({"c": c, "qkv": s["dqkv"]})
    a, b = D.rotary(q, k, s["w"], interleaved=interleaved)
    da, db = D.rotary(dq, dk, s["w"], interleaved=interleaved, inverse=True)
    return {"q": a, "k": b, "dq": da, "dk": db}


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(c, seed):
    """The outputs from the definitions, in 64 bits; written without the plain forms' code."""
    s = prepare(c, seed)
    if c["kind"] == "logits":
        prompt, total = _history(c)
        rows = []
        for r in range(c["rows"]):
            x = s["logits"][r, : c["vocab"]].double()
            everything = torch.bincount(s["tokens"][r, : total[r]], minlength=c["vocab"])
            n = torch.bincount(s["tokens"][r, min(prompt[r], total[r]): total[r]], minlength=c["vocab"]).double()
            rep = s["repetition"][r].double()
            factor = torch.ones_like(x)
            factor[everything > 0] = rep
            x = torch.where(x > 0, x / factor, x * factor)
            x = x - s["frequency"][r].double() * n
            x[n > 0] -= s["presence"][r].double()
            if s["bias"] is not None:
                x = x + s["bias"].double()
            if s["allowed"] is not None:
                bits = s["allowed"][r][:, None].bitwise_and(
                    torch.tensor([1 << i if i < 31 else -2 ** 31 for i in range(32)], dtype=torch.int32, device=DEV))
                x[bits.flatten()[: c["vocab"]] == 0] = -math.inf
            rows.append(x)
        return torch.stack(rows)
    if c["kind"] == "attend":
        o, lse = [], []
        for b, n in enumerate(_lengths(c)):
            pages = s["table"][b, : -(-n // c["page"])].long()
            k, v = (s[x].index_select(0, pages).movedim(1, 0).flatten(1, 2)[:, :n].double() for x in "kv")
            q = s["q"][b].double().view(c["kv"], -1, c["hd"])
            x = (q @ k.mT) * c["hd"] ** -0.5
            z = torch.logsumexp(x, -1, keepdim=True)
            o.append(((x - z).exp() @ v).reshape(c["heads"], c["hd"]))
            lse.append(z.reshape(c["heads"]))
        return {"o": torch.stack(o), "lse": torch.stack(lse)}

    def turned(x, start, sign):
        """As a product of complex numbers."""
        if not c["turn"]:
            return x.double()
        n = c["turn"] // 2
        p = torch.arange(c["seq"], device=DEV)[None, :] + torch.tensor(start, device=DEV)[:, None]
        f = torch.tensor([10000.0 ** (-2 * i / c["turn"]) for i in range(n)], dtype=torch.float64, device=DEV)
        unit = torch.polar(torch.ones_like(f), sign * p[..., None].double() * f)[:, :, None, :]
        y = x.double()
        order = torch.arange(c["turn"], device=DEV)
        order = order.view(2, n).T if c["pairs"] == "halves" else order.view(n, 2)
        z = torch.view_as_complex(y[..., order].contiguous()) * unit
        y[..., order] = torch.view_as_real(z)
        return y

    H, Hk = c["heads"], c["kv"]
    if c["kind"] == "rotary":
        start = [0] * c["batch"]
        x, d = s["qkv"], s["dqkv"]
        return {"q": turned(x[:, :, :H], start, 1), "k": turned(x[:, :, H: H + Hk], start, 1),
                "dq": turned(d[:, :, :H], start, -1), "dk": turned(d[:, :, H: H + Hk], start, -1)}
    start = _lengths(c)
    counts = _counts(c) if c["seq"] > 1 else [1] * c["batch"]
    k, v, q = s["k"].double(), s["v"].double(), s["qkv"][:, :, :H].double()
    q_new, k_new = turned(s["qkv"][:, :, :H], start, 1), turned(s["qkv"][:, :, H: H + Hk], start, 1)
    for b in range(c["batch"]):
        p = torch.arange(start[b], start[b] + counts[b], device=DEV)
        page, row = s["table"][b, p // c["page"]].long(), p % c["page"]
        k[page, :, row] = k_new[b, : counts[b]]
        v[page, :, row] = s["qkv"][b, : counts[b], H + Hk:].double()
        q[b, : counts[b]] = q_new[b, : counts[b]]
    return {"k": k, "v": v, "q": q if c["turn"] else None}
