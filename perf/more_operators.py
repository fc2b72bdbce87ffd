"""Operators of a served decoder: a key-value cache held in 8 bits, and the choice of the next token.  Their cases, their plain
forms and the framework's calls.

Families (``case["kind"]``); the framework's forms are functions of ``frankentorch_b200.ops.decode``:

* ``append``   ``paged_append`` with ``k_scales`` / ``v_scales``: keys and values of new tokens into a paged cache of 8-bit floating
  point with a scale for each block of tokens and head, rotated on the way, with the queries.
* ``attend``   ``paged_attention`` with the scales: one new token per sequence over that cache, output and log-sum-exp.
* ``sample``   ``sample``: temperature, top-k, top-p and min-p on the logits of a step, and a token from given random numbers.

Formulas.  A block is ``block`` neighbouring rows of a page; with ``s`` its scale an element ``y`` (e4m3) stands for ``s y``.  New tokens
of a block whose largest finite magnitude is ``a`` need ``s = 2^e``, the smallest power of two with ``a <= 448 s``, at least ``2^-100``; a
block whose first rows are there already keeps the larger of ``s`` and its own scale ``s'``, and its rows become ``y s' / s``.  Each
element is rounded once.  ``o = sum_t softmax_t(q k_t / sqrt(hd)) v_t`` over ``t < lengths[b]``; a sequence of no tokens has ``o = 0`` and
a log-sum-exp of ``-inf``.

A token ``i`` weighs ``w_i = round(2^43 exp((x_i - max x) / T))``; tokens are ordered by their logits, equal ones by their ids.  Kept are
the first ``k``, of those the ones before which less than ``p`` of their sum lies, and of those the ones of at least ``min_p`` of the
largest; the choice is the first token, by id, with ``sum_{j <= i} w_j > floor(u sum_j w_j)`` over what is kept, and its log-probability
``log(w_i / sum_j w_j)``.  ``T = 0`` keeps the first alone.
Numbers for all rows count as fp32, as those of a row do.
"""
import math
import random

import torch

own = False
DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
E4M3 = torch.float8_e4m3fn


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # one conversation of GPT-2 small: one token, learned positions, so nothing is turned; latency
        {"name": "append_one", "kind": "append", "batch": 1, "seq": 1, "heads": 12, "kv": 12, "hd": 64, "turn": 0,
         "pairs": "halves", "page": 16, "block": 16, "longest": 300, "dtype": "bf16"},
        # a step of a full serving batch of the 1.3B decoder
        {"name": "append_step", "kind": "append", "batch": 256, "seq": 1, "heads": 16, "kv": 16, "hd": 128, "turn": 128,
         "pairs": "halves", "page": 64, "block": 64, "longest": 2047, "dtype": "bf16"},
        # ragged prompts in a padded batch, grouped heads, a part of each head turned
        {"name": "append_prompts", "kind": "append", "batch": 16, "seq": 2048, "heads": 16, "kv": 4, "hd": 128,
         "turn": 64, "pairs": "neighbours", "page": 32, "block": 16, "longest": 0, "dtype": "bf16"},
        # one conversation of GPT-2 small: latency
        {"name": "attend_one", "kind": "attend", "batch": 1, "heads": 12, "kv": 12, "hd": 64, "page": 16, "block": 16,
         "shortest": 301, "longest": 301, "idle": 0, "dtype": "bf16"},
        # a ragged batch of the 1.3B decoder with some places not in use
        {"name": "attend_batch", "kind": "attend", "batch": 32, "heads": 16, "kv": 16, "hd": 128, "page": 64, "block": 64,
         "shortest": 20, "longest": 2048, "idle": 3, "dtype": "bf16"},
        # two long documents, grouped heads: little to do side by side but the length
        {"name": "attend_long", "kind": "attend", "batch": 2, "heads": 32, "kv": 4, "hd": 128, "page": 32, "block": 32,
         "shortest": 60001, "longest": 65537, "idle": 0, "dtype": "fp16"},
        # a full serving batch, ragged
        {"name": "attend_full", "kind": "attend", "batch": 128, "heads": 16, "kv": 16, "hd": 128, "page": 64, "block": 64,
         "shortest": 700, "longest": 4096, "idle": 0, "dtype": "bf16"},
        # one conversation over the GPT-2 vocabulary with the usual filters: latency
        {"name": "sample_one", "kind": "sample", "rows": 1, "vocab": 50257, "slope": 1.3, "masked": 0.0, "mixed": False,
         "temperature": 0.8, "top_k": 50, "top_p": 0.95, "min_p": 0.0, "dtype": "fp32"},
        # rollouts: the model's own distribution, nothing cut
        {"name": "sample_open", "kind": "sample", "rows": 64, "vocab": 50257, "slope": 1.0, "masked": 0.0, "mixed": False,
         "temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0, "dtype": "fp32"},
        # a serving batch over the GPT-2 vocabulary: every request has its own settings, a grammar has masked some tokens
        {"name": "sample_batch", "kind": "sample", "rows": 256, "vocab": 50257, "slope": 1.2, "masked": 0.3, "mixed": True,
         "temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0, "dtype": "fp32"},
        # a full serving batch over a large vocabulary, nucleus sampling
        {"name": "sample_large", "kind": "sample", "rows": 512, "vocab": 128003, "slope": 1.0, "masked": 0.0, "mixed": False,
         "temperature": 1.0, "top_k": 0, "top_p": 0.9, "min_p": 0.0, "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return max(1, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


MAX_BYTES = 6e8         # a drawn attention stays below the largest listed one
MAX_PADDED = 2.1e9      # elements of the cache if all sequences were as long as the longest (the plain form computes on those)


def draw(rng):
    """One more case of the same families."""
    while True:
        kind = rng.choice(["append", "attend", "sample", "sample"])
        c = {"kind": kind}
        if kind == "sample":
            c.update(rows=_log_int(rng, 1, 512), vocab=_log_int(rng, 500, 130000), slope=round(rng.uniform(0.3, 2.0), 2),
                     masked=rng.choice([0.0, 0.0, 0.3, 0.95]), mixed=rng.random() < 0.4,
                     temperature=rng.choice([0.0, 1.0, round(rng.uniform(0.2, 2.0), 2)]),
                     top_k=rng.choice([0, 0, _log_int(rng, 1, 2000)]),
                     top_p=rng.choice([1.0, round(rng.uniform(0.05, 0.99), 3)]),
                     min_p=rng.choice([0.0, 0.0, round(rng.uniform(0.001, 0.3), 3)]),
                     dtype=rng.choice(["bf16", "fp16", "fp32", "fp32"]))
            if work(c)["bytes"] <= 1.3e8:
                return c
            continue
        hd = rng.choice([64, 128])
        group = rng.choice([1, 1, 2, 3, 4, 7, 8, 16])
        kv = _log_int(rng, 1, 16)
        page = rng.choice([8, 16, 32, 64, 128])
        c.update(heads=kv * group, kv=kv, hd=hd, page=page, block=rng.choice([min(page, 64), min(page, 64), 8, 1]),
                 dtype=rng.choice(["bf16", "bf16", "fp16"]))
        if kind == "attend":
            longest = _log_int(rng, 1, 65536)
            c.update(batch=_log_int(rng, 1, 256), shortest=_log_int(rng, 1, longest), longest=longest,
                     idle=rng.choice([0, 0, 1]))
            if c["idle"] >= c["batch"] or c["batch"] * longest * kv * hd > MAX_PADDED or work(c)["bytes"] > MAX_BYTES:
                continue
            return c
        c.update(batch=_log_int(rng, 1, 64), seq=_log_int(rng, 1, 2048), turn=rng.choice([0, hd, hd, hd // 2]),
                 pairs=rng.choice(["halves", "neighbours"]), longest=rng.choice([0, _log_int(rng, 1, 30000)]))
        if rng.random() < 0.5:
            c.update(batch=_log_int(rng, 1, 256), seq=1)
        if work(c)["bytes"] <= 2e8 and c["batch"] * (c["longest"] + c["seq"]) * kv * hd <= MAX_PADDED:
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
    """New tokens of each sequence of an append: one, or ragged prompts."""
    rng = random.Random("%s %s" % (c["batch"], c["seq"]))
    return [rng.randint((c["seq"] + 3) // 4, c["seq"]) for _ in range(c["batch"])]


def _pages(c, ends):
    """(pages of each sequence, columns of the table, pages of the cache)."""
    need = [-(-n // c["page"]) for n in ends]
    return need, max(1, max(need)) + 1, sum(need) + 5


def work(c):
    e = 4 if c["dtype"] == "fp32" else 2
    if c["kind"] == "append":
        counts, start = _counts(c), _lengths(c)
        t = sum(counts)
        q = c["heads"] if c["turn"] else 0
        blocks = sum((n + m - 1) // c["block"] - n // c["block"] + 1 for n, m in zip(start, counts))
        return {"bytes": t * c["hd"] * (2 * q * e + 2 * c["kv"] * (e + 1)) + 8 * blocks * c["kv"] + 4 * t / c["page"] + 12 * c["batch"],
                "flops": 3 * t * c["turn"] * (q + c["kv"]) + 4 * t * c["kv"] * c["hd"]}
    if c["kind"] == "attend":
        lengths = _lengths(c)
        n = sum(lengths)
        blocks = sum(-(-m // c["block"]) for m in lengths)
        q = c["batch"] * c["heads"] * c["hd"]
        return {"bytes": 2 * n * c["kv"] * c["hd"] + 2 * q * e + 8 * blocks * c["kv"] + 4 * n / c["page"] + 4 * c["batch"] * (c["heads"] + 1),
                "flops": 4 * n * c["heads"] * c["hd"]}
    return {"bytes": c["rows"] * (c["vocab"] * e + 16 + (16 if c["mixed"] else 0)), "flops": 4 * c["rows"] * c["vocab"]}


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _n(g, dtype, *shape):
    return torch.randn(*shape, generator=g, device=DEV).to(dtype)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _frequencies(turn):
    return 10000.0 ** (-torch.arange(0, turn, 2, dtype=torch.float64, device=DEV) / turn)


def _cache(c, g, ends):
    """Pages in a shuffled order, as a cache has them after some use, their scales, and the table of each sequence.  Heads differ in
    size, blocks of a head by a factor of two either way."""
    need, cols, pages = _pages(c, ends)
    made = []
    for _ in range(2):
        data = torch.randn(pages, c["kv"], c["page"], c["hd"], generator=g, device=DEV)
        made.append(data.mul_(64.0).clamp_(-448.0, 448.0).to(E4M3))
        del data
    scales = []
    for _ in range(2):
        of_head = torch.randint(-7, -4, (1, c["kv"], 1), generator=g, device=DEV)
        of_block = torch.randint(-1, 2, (pages, c["kv"], c["page"] // c["block"]), generator=g, device=DEV)
        scales.append(torch.exp2((of_head + of_block).float()))
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    first = torch.tensor([0] + need, device=DEV).cumsum(0)[:-1]
    at = torch.arange(cols, device=DEV)
    mine = at[None, :] < torch.tensor(need, device=DEV)[:, None]
    table = torch.where(mine, order[(first[:, None] + at[None, :]).clamp(max=pages - 1)], 0).to(torch.int32)
    return {"k": made[0], "v": made[1], "ks": scales[0], "vs": scales[1], "table": table}


def prepare(c, seed):
    g = _gen(seed)
    dt = TYPES[c["dtype"]]
    if c["kind"] == "append":
        B, S, H, Hk, hd = (c[x] for x in ("batch", "seq", "heads", "kv", "hd"))
        start, counts = _lengths(c), _counts(c)
        s = _cache(c, g, [n + m for n, m in zip(start, counts)])
        s.update(c=c, qkv=_n(g, dt, B, S, H + 2 * Hk, hd), start=_i32(start), counts=_i32(counts) if S > 1 else None,
                 w=_frequencies(c["turn"]) if c["turn"] else None)
        return s
    if c["kind"] == "attend":
        lengths = _lengths(c)
        s = _cache(c, g, lengths)
        # the queries of a step are a view into its packed projections
        qkv = _n(g, dt, c["batch"], c["heads"] + 2 * c["kv"], c["hd"])
        s.update(c=c, q=qkv[:, : c["heads"]], lengths=_i32(lengths))
        return s
    R, V = c["rows"], c["vocab"]
    columns = (V + 127) // 128 * 128                      # the head's rows are padded to whole tiles
    # a model's probabilities fall with the rank of a token by a power law
    logits = -c["slope"] * torch.log1p(V * torch.rand(R, columns, generator=g, device=DEV))
    logits += 0.3 * torch.randn(R, columns, generator=g, device=DEV)
    if c["masked"]:
        logits.masked_fill_(torch.rand(R, columns, generator=g, device=DEV) < c["masked"], -math.inf)
    s = {"c": c, "logits": logits.to(dt), "uniform": torch.rand(R, generator=g, device=DEV)}
    for name in ("temperature", "top_k", "top_p", "min_p"):
        s[name] = c[name]
    if c["mixed"]:
        def some(share, value, otherwise):
            return torch.where(torch.rand(R, generator=g, device=DEV) < share, value, otherwise)
        r = torch.rand(4, R, generator=g, device=DEV)
        s["temperature"] = some(0.125, 0.0, 0.3 + 1.2 * r[0])
        s["top_k"] = some(0.5, 0.0, torch.exp(5.3 * r[1])).to(torch.int32)
        s["top_p"] = some(0.25, 1.0, 0.5 + 0.49 * r[2])
        s["min_p"] = some(0.5, 0.0, 0.01 + 0.2 * r[3])
    return s


def _split(s):
    """Views of the packed projections: queries, keys, values."""
    H, Hk = s["c"]["heads"], s["c"]["kv"]
    return s["qkv"].split([H, Hk, Hk], dim=2)


# ------------------------------------------------------------------------------------------------ plain forms
def _turned(x, start, w, pairs):
    """Elementary form of the rotation: angles in 64 bits, products in 32."""
    B, S = x.shape[:2]
    n = w.shape[0]
    p = start.double()[:, None] + torch.arange(S, device=x.device, dtype=torch.float64)
    a = (p[:, :, None] * w)[:, :, None, :]
    cos, sin = a.cos().float(), a.sin().float()
    part, rest = x[..., : 2 * n], x[..., 2 * n:]
    if pairs == "halves":
        x0, x1 = part[..., :n], part[..., n:]
        part = torch.cat([x0 * cos - x1 * sin, x1 * cos + x0 * sin], -1)
    else:
        x0, x1 = part[..., 0::2], part[..., 1::2]
        part = torch.stack([x0 * cos - x1 * sin, x1 * cos + x0 * sin], -1).flatten(-2)
    return torch.cat([part, rest], -1)


def _needed(a):
    """The smallest power of two, 2^-100 at least, of which 448 times reaches ``a``."""
    m, e = torch.frexp(a)
    e = torch.where(a > 0, e - 9 + (m > 0.875), -100).clamp(min=-100)
    return torch.ldexp(torch.ones_like(a), e)


def _plain_put(s, pages, scales, x):
    """``x`` (fp32 ``[B, S, Hkv, hd]``) into the 8-bit cache: a grid of the blocks that a sequence can touch, rows by rows."""
    c = s["c"]
    B, S, Hk, hd = x.shape
    n, page, per_page = c["block"], c["page"], c["page"] // c["block"]
    start = s["start"].long()
    counts = s["counts"].long() if s["counts"] is not None else torch.full_like(start, S)
    blocks = (S + n - 2) // n + 1
    first = start // n
    at = first[:, None] * n + torch.arange(blocks * n, device=DEV)                       # positions of the grid
    i = at - start[:, None]
    new, old = (i >= 0) & (i < counts[:, None]), i < 0
    grid = x.gather(1, i.clamp(0, S - 1)[:, :, None, None].expand(-1, -1, Hk, hd))
    grid = torch.where(new[:, :, None, None], grid, 0.0).view(B, blocks, n, Hk, hd)
    touched = new.view(B, blocks, n).any(-1)
    at_block = first[:, None] + torch.arange(blocks, device=DEV)
    page_of = s["table"].long().gather(1, (at_block // per_page).clamp(max=s["table"].shape[1] - 1))
    sub = at_block % per_page
    before = scales[page_of, :, sub]                                                    # [B, blocks, Hkv]
    begun = old.view(B, blocks, n).any(-1) & touched
    scale = _needed(grid.abs().amax((2, 4)))
    scale = torch.where(begun[:, :, None], torch.maximum(scale, before), scale)
    b, j = touched.nonzero(as_tuple=True)
    scales[page_of[b, j], :, sub[b, j]] = scale[b, j]
    b, r = (new | (old & touched.repeat_interleave(n, 1))).nonzero(as_tuple=True)
    j, row = r // n, at[b, r] % page
    raw = pages.view(torch.uint8)
    kept = raw[page_of[b, j], :, row].view(E4M3).float() * (before[b, j] / scale[b, j])[:, :, None]
    y = torch.where(new[b, r][:, None, None], grid.view(B, -1, Hk, hd)[b, r] / scale[b, j][:, :, None], kept)
    raw[page_of[b, j], :, row] = y.to(E4M3).view(torch.uint8)


def _plain_append(s):
    c = s["c"]
    q, k, v = (t.float() for t in _split(s))
    turned = None
    if s["w"] is not None:
        k = _turned(k, s["start"], s["w"], c["pairs"])
        turned = _turned(q, s["start"], s["w"], c["pairs"])
        if s["counts"] is not None:
            here = torch.arange(c["seq"], device=DEV)[None, :] < s["counts"][:, None]
            turned = torch.where(here[:, :, None, None], turned, q)
        turned = turned.to(s["qkv"].dtype)
    _plain_put(s, s["k"], s["ks"], k)
    _plain_put(s, s["v"], s["vs"], v)
    return {"k": s["k"], "v": s["v"], "ks": s["ks"], "vs": s["vs"], "q": turned}


def _plain_attend(s):
    c = s["c"]
    B, Hk, hd = c["batch"], c["kv"], c["hd"]
    t = s["table"].long()
    rows = t.shape[1] * c["page"]
    here = torch.arange(rows, device=t.device)[None, :] < s["lengths"][:, None]

    def whole(pages, scales):
        y = pages.view(torch.uint8)[t].view(E4M3).transpose(1, 2).reshape(B, Hk, rows, hd).float()
        y *= scales[t].transpose(1, 2).reshape(B, Hk, -1, 1).expand(-1, -1, -1, c["block"]).reshape(B, Hk, rows, 1)
        return y
    x = torch.matmul(s["q"].float().reshape(B, Hk, -1, hd), whole(s["k"], s["ks"]).transpose(2, 3)) / math.sqrt(hd)
    x = torch.where(here[:, None, None, :], x, -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    v = torch.where(here[:, None, :, None], whole(s["v"], s["vs"]), 0.0)
    o = torch.matmul(p, v) / torch.where(total == 0, 1.0, total)
    lse = top + torch.log(total)
    return {"o": o.reshape(B, c["heads"], hd).to(s["q"].dtype), "lse": lse.reshape(B, c["heads"])}


def _plain_sample(s):
    V = s["c"]["vocab"]
    x = s["logits"][:, :V].double()

    def per_row(v):
        return (v if isinstance(v, torch.Tensor) else torch.full((x.shape[0],), float(v), device=DEV)).double()[:, None]
    t, p, least = per_row(s["temperature"]), per_row(s["top_p"]), per_row(s["min_p"])
    k = per_row(s["top_k"]).long()
    k = torch.where(t == 0, 1, torch.where(k <= 0, V, k))
    top = x.amax(-1, keepdim=True)
    w = torch.round(torch.exp(torch.where(x == top, 0.0, (x - top) / t)) * 2.0 ** 43)
    w = torch.where(x == -math.inf, 0.0, w).long()
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices
    del x
    w = w.gather(1, order)
    rank = torch.arange(V, device=DEV)
    w = torch.where(rank < k, w, 0)
    before = w.cumsum(-1) - w
    limit = torch.where(p < 1, torch.ceil(p * w.sum(-1, keepdim=True).double()), math.inf)
    w = torch.where(((before < limit) | (rank == 0)) & (w >= least * 2.0 ** 43), w, 0)
    w = torch.zeros_like(w).scatter_(1, order, w)
    sums = w.cumsum(-1)
    total = sums[:, -1:]
    target = torch.floor(s["uniform"].double()[:, None] * total).long()
    token = (sums <= target).sum(-1)
    token = torch.where(total[:, 0] == 0, -1, token)
    chosen = w.gather(1, token.clamp(min=0)[:, None]).double() / total
    return {"token": token, "logprob": torch.where(total == 0, -math.inf, torch.log(chosen))[:, 0].float()}


def run(s):
    c = s["c"]
    if own:
        return _run_own(s)
    if c["kind"] == "append":
        return _plain_append(s)
    if c["kind"] == "attend":
        return _plain_attend(s)
    return _plain_sample(s)


# ------------------------------------------------------------------------------------------------ the framework's calls
def _run_own(s):
    from frankentorch_b200.ops import decode as D
    c = s["c"]
    if c["kind"] == "sample":
        token, logprob = D.sample(s["logits"], s["uniform"], vocab=c["vocab"], temperature=s["temperature"], top_k=s["top_k"],
                                  top_p=s["top_p"], min_p=s["min_p"])
        return {"token": token, "logprob": logprob}
    if c["kind"] == "attend":
        o, lse = D.paged_attention(s["q"], s["k"], s["v"], s["table"], s["lengths"], k_scales=s["ks"], v_scales=s["vs"])
        return {"o": o, "lse": lse}
    q, k, v = _split(s)
    turned = None
    if s["w"] is not None:
        turned = D.paged_append(s["k"], s["v"], s["table"], k, v, s["start"], s["counts"], q=q, inv_freq=s["w"],
                                interleaved=c["pairs"] == "neighbours", k_scales=s["ks"], v_scales=s["vs"])
    else:
        D.paged_append(s["k"], s["v"], s["table"], k, v, s["start"], s["counts"], k_scales=s["ks"], v_scales=s["vs"])
    return {"k": s["k"], "v": s["v"], "ks": s["ks"], "vs": s["vs"], "q": turned}


# ------------------------------------------------------------------------------------------------ in 64 bits
def _exact_sample(c, s):
    tokens, logprobs = [], []
    for r in range(c["rows"]):
        t, k, p, least = (float(v[r]) if isinstance(v, torch.Tensor) else float(torch.tensor(float(v)))
                          for v in (s["temperature"], s["top_k"], s["top_p"], s["min_p"]))
        x = s["logits"][r, : c["vocab"]].double()
        # negated and sorted upwards, equal ones stay in the order of their ids
        y, ids = torch.sort(-x, stable=True)
        here = int((y < math.inf).sum())
        y, ids = y[:here], ids[:here]
        if here == 0:
            tokens.append(-1)
            logprobs.append(-math.inf)
            continue
        y, ids = (y[:1], ids[:1]) if t == 0 else (y[: int(k)], ids[: int(k)]) if k > 0 else (y, ids)
        weight = ((y[0] - y) / (t or 1.0)).exp().mul(2.0 ** 43).round().long()
        if p < 1:
            upto = weight.cumsum(0)
            kept = 1 + int((upto[:-1].double() < p * float(upto[-1])).sum())
            weight, ids = weight[:kept], ids[:kept]
        kept = max(1, int((weight.double() >= least * 2.0 ** 43).sum()))      # weights fall along the order
        weight, ids = weight[:kept], ids[:kept]
        ids, by_id = ids.sort()
        upto = weight[by_id].cumsum(0)
        n, d = float(s["uniform"][r]).as_integer_ratio()
        at = int(torch.searchsorted(upto, n * int(upto[-1]) // d, right=True))
        tokens.append(int(ids[at]))
        logprobs.append(math.log(int(weight[by_id][at]) / int(upto[-1])))
    return {"token": torch.tensor(tokens, device=DEV), "logprob": torch.tensor(logprobs, dtype=torch.float64, device=DEV)}


def exact(c, seed):
    """The outputs from the definitions, in 64 bits; written without the plain forms' code."""
    s = prepare(c, seed)
    if c["kind"] == "sample":
        return _exact_sample(c, s)
    if c["kind"] == "attend":
        o, lse = [], []
        for b, n in enumerate(_lengths(c)):
            pages = s["table"][b, : -(-n // c["page"])].long()
            k, v = (torch.repeat_interleave(s[x + "s"].index_select(0, pages).double(), c["block"], 2)[..., None] *
                    s[x].view(torch.uint8).index_select(0, pages).view(E4M3).double() for x in "kv")
            k, v = (y.movedim(1, 0).flatten(1, 2)[:, :n] for y in (k, v))
            q = s["q"][b].double().view(c["kv"], -1, c["hd"])
            x = (q @ k.mT) * c["hd"] ** -0.5
            z = torch.logsumexp(x, -1, keepdim=True)
            o.append(((x - z).exp() @ v).reshape(c["heads"], c["hd"]))
            lse.append(z.reshape(c["heads"]))
        return {"o": torch.stack(o), "lse": torch.stack(lse)}

    def turned(x):
        """As a product of complex numbers."""
        if not c["turn"]:
            return x.double()
        n = c["turn"] // 2
        p = torch.arange(c["seq"], device=DEV)[None, :] + torch.tensor(_lengths(c), device=DEV)[:, None]
        f = torch.tensor([10000.0 ** (-2 * i / c["turn"]) for i in range(n)], dtype=torch.float64, device=DEV)
        unit = torch.polar(torch.ones_like(f), p[..., None].double() * f)[:, :, None, :]
        y = x.double()
        order = torch.arange(c["turn"], device=DEV)
        order = order.view(2, n).T if c["pairs"] == "halves" else order.view(n, 2)
        z = torch.view_as_complex(y[..., order].contiguous()) * unit
        y[..., order] = torch.view_as_real(z)
        return y

    H, Hk, n = c["heads"], c["kv"], c["block"]
    qkv = s["qkv"]
    start, counts = _lengths(c), _counts(c)
    out = {"q": None}
    if c["turn"]:
        q, t = qkv[:, :, :H].double(), turned(qkv[:, :, :H])
        for b in range(c["batch"]):
            q[b, : counts[b]] = t[b, : counts[b]]
        out["q"] = q
    if sum((m + n - 1) // n + 1 for m in counts) * Hk > 200000:       # a loop over the blocks would take too long
        return None
    for name, x in (("k", turned(qkv[:, :, H: H + Hk])), ("v", qkv[:, :, H + Hk:].double())):
        pages, scales = s[name].float().double(), s[name + "s"].double()
        for b in range(c["batch"]):
            at = start[b]
            while at < start[b] + counts[b]:
                end = min(start[b] + counts[b], at // n * n + n)
                page, row = int(s["table"][b, at // c["page"]]), at % c["page"]
                y = x[b, at - start[b]: end - start[b]]                                # [tokens, heads, hd]
                a = y.abs().amax((0, 2)).clamp(min=1e-300)
                need = torch.exp2(torch.ceil(torch.log2(a / 448)).clamp(min=-100))
                had = scales[page, :, row // n].clone()
                if row % n:
                    need = torch.maximum(need, had)
                    pages[page, :, row // n * n: row] *= (had / need)[:, None, None]
                scales[page, :, row // n] = need
                pages[page, :, row: row + end - at] = (y / need[:, None]).transpose(0, 1)
                at = end
        out[name], out[name + "s"] = pages, scales
    return out
