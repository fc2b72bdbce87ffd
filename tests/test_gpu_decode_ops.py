"""Rotation, paged cache, decoding attention and logits processing against 64-bit arithmetic, at the sizes, layouts and masks
where they can go wrong."""
import math

import pytest
import torch

from _decode_oracle import attention as attention64
from _decode_oracle import close, logits as logits64, rotary as rotary64

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def _rnd(g, *shape, dtype=BF, dev="cuda"):
    return torch.randn(*shape, generator=g, device=dev).to(dtype)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _cache(g, heads, page, hd, ends, dtype=BF, spare=3, layout="pages"):
    """Shuffled pages for sequences of ``ends`` tokens, every row NaN; the table's unused entries are no page at all."""
    need = [-(-n // page) for n in ends]
    P = sum(need) + spare
    if layout == "rows":       # heads innermost: [pages, page, heads, hd] in memory
        mk = lambda: torch.full((P, page, heads, hd), math.nan, dtype=dtype, device="cuda").transpose(1, 2)      # noqa: E731
    else:
        mk = lambda: torch.full((P, heads, page, hd), math.nan, dtype=dtype, device="cuda")                      # noqa: E731
    table = torch.full((len(ends), max(need + [1]) + 1), -7, dtype=torch.int32, device="cuda")
    order = torch.randperm(P, generator=g, device="cuda").to(torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at: at + n]
        at += n
    return mk(), mk(), table


def _fill(g, pages, table, ends):
    """Random values in the rows in use."""
    page = pages.shape[2]
    for b, n in enumerate(ends):
        p = torch.arange(n, device="cuda")
        idx = table[b].long()[p // page]
        pages[idx, :, p % page] = _rnd(g, n, pages.shape[1], pages.shape[3], dtype=pages.dtype)


# ------------------------------------------------------------------------------------------------ rotation
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,S,H,Hk,hd,turned,start", [
    (1, 1, 1, 1, 64, 64, [0]),
    (3, 5, 4, 2, 64, 32, [0, 7, 1000]),
    (2, 9, 3, 1, 128, 128, [131071, 1]),
    (2, 3, 5, 5, 80, 48, [2147483600, -40]),     # the last positions that int32 holds, and ones before the first
    (1, 2, 70, 10, 256, 16, [12345]),
    (2, 33, 1, 1, 16, 16, [3, 0]),
])
def test_rotary(cuda_device, B, S, H, Hk, hd, turned, start, interleaved, dtype):
    from frankentorch_b200.ops import decode as D
    from frankentorch_b200.ops import kernels as K
    g = _gen(S * hd)
    packed = _rnd(g, B, S, H + 2 * Hk, hd, dtype=dtype)
    q, k = packed[:, :, :H], packed[:, :, H: H + Hk]
    w = D.rotary_frequencies(turned)
    before = packed.clone()
    for inverse in (False, True):
        a, b = D.rotary(q, k, w, start=_i32(start), interleaved=interleaved, inverse=inverse)
        close(a, *rotary64(q, w, start, interleaved, inverse), "q")
        close(b, *rotary64(k, w, start, interleaved, inverse), "k")
    assert torch.equal(packed, before)
    # in place, between elements that belong to others; and alone
    out = packed.clone()
    D.rotary(out[:, :, :H], out[:, :, H: H + Hk], w, start=_i32(start), interleaved=interleaved, inverse=True,
             q_out=out[:, :, :H], k_out=out[:, :, H: H + Hk])
    assert torch.equal(out[:, :, :H], a) and torch.equal(out[:, :, H: H + Hk], b)
    assert torch.equal(out[:, :, H + Hk:], packed[:, :, H + Hk:])
    alone, none = D.rotary(q, None, w, start=_i32(start), interleaved=interleaved, inverse=True)
    assert none is None and torch.equal(alone, a)
    K.check_status()


def test_rotary_without_start_and_broadcast_inputs(cuda_device):
    from frankentorch_b200.ops import decode as D
    g = _gen(3)
    w = D.rotary_frequencies(64)
    one = _rnd(g, 1, 6, 1, 64)
    q = one.expand(4, 6, 3, 64)                       # every sequence and head reads the same row
    a, _ = D.rotary(q, None, w)
    assert torch.equal(a, D.rotary(q.contiguous(), None, w)[0])
    close(a[2:3, :, 1:2], *rotary64(one, w, [0]), "q")
    empty, ek = D.rotary(q[:0], q[:0], w)
    assert empty.shape == (0, 6, 3, 64) and ek.shape == (0, 6, 3, 64)
    assert D.rotary(q[:, :0], None, w)[0].shape == (4, 0, 3, 64)


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_backward_is_the_transpose(cuda_device, interleaved):
    """<R x, y> = <x, R' y> for the pair of calls that a training step makes; and the derivative against differences."""
    from frankentorch_b200.ops import decode as D
    g = _gen(8)
    x, y = _rnd(g, 2, 40, 3, 64), _rnd(g, 2, 40, 3, 64)
    w = D.rotary_frequencies(64)
    rx, _ = D.rotary(x, None, w, interleaved=interleaved)
    ry, _ = D.rotary(y, None, w, interleaved=interleaved, inverse=True)
    left, right = (rx.double() * y.double()).sum(), (x.double() * ry.double()).sum()
    # each side has one rounding per element (2^-8 of it), in either sign
    size = (rx.double() * y.double()).abs().sum() + (x.double() * ry.double()).abs().sum()
    assert abs(float(left - right)) <= 2.0 ** -8 * float(size)
    step = torch.zeros_like(x)
    step[1, 17, 2, 5] = 1.0
    diff = (D.rotary(step, None, w, interleaved=interleaved)[0].double() * y.double()).sum()
    # the map is linear: its difference along one element is its value there; two products of rounded factors
    assert abs(float(diff - ry[1, 17, 2, 5].double())) <= 2.0 ** -8 * 3 * float(y[1, 17, 2].abs().max())


# ------------------------------------------------------------------------------------------------ append
@pytest.mark.parametrize("layout", ["pages", "rows"])
@pytest.mark.parametrize("dtype,interleaved", [(BF, False), (HF, True)])
@pytest.mark.parametrize("B,S,H,Hk,hd,turned,page,start,counts", [
    (1, 1, 12, 12, 64, 0, 16, [300], None),
    (4, 1, 8, 2, 128, 128, 64, [63, 64, 0, 1000], None),
    (3, 20, 4, 4, 64, 64, 8, [0, 5, 31], [20, 0, 7]),
    (3, 17, 6, 1, 128, 64, 1, [0, 2, 3], [17, 1, 16]),
    (2, 40, 2, 2, 32, 0, 32, [1, 31], [39, 40]),
    (2, 9, 3, 3, 48, 16, 128, [125, 100000], [9, 5]),
])
def test_append(cuda_device, B, S, H, Hk, hd, turned, page, start, counts, dtype, interleaved, layout):
    from frankentorch_b200.ops import decode as D
    from frankentorch_b200.ops import kernels as K
    g = _gen(S + hd)
    used = counts or [S] * B
    ends = [a + n for a, n in zip(start, used)]
    kp, vp, table = _cache(g, Hk, page, hd, ends, dtype, layout=layout)
    packed = _rnd(g, B, S, H + 2 * Hk, hd, dtype=dtype)
    q, k, v = packed.split([H, Hk, Hk], 2)
    w = D.rotary_frequencies(turned) if turned else None
    ct = None if counts is None else _i32(counts)
    got = D.paged_append(kp, vp, table, k, v, _i32(start), ct, q=q if turned else None, inv_freq=w, interleaved=interleaved)
    K.check_status()
    wk, tk = rotary64(k, w, start, interleaved)
    if turned:
        close(got, *rotary64(q, w, start, interleaved, counts=used), "q")
    else:
        assert got is None
    written = torch.zeros(kp.shape[0], page, dtype=torch.bool)
    for b in range(B):
        p = torch.arange(start[b], ends[b])
        idx, row = table[b].cpu().long()[p // page], p % page
        written[idx, row] = True
        close(kp.cpu()[idx, :, row], wk[b, : used[b]], tk[b, : used[b]], "k")
        assert torch.equal(vp.cpu()[idx, :, row], v[b, : used[b]].cpu())
    assert bool(kp.cpu().transpose(1, 2)[~written].isnan().all()) and bool(vp.cpu().transpose(1, 2)[~written].isnan().all())
    if turned:       # over the queries themselves
        again = packed.clone()
        D.paged_append(kp, vp, table, k, v, _i32(start), ct, q=again[:, :, :H], inv_freq=w, interleaved=interleaved,
                       q_out=again[:, :, :H])
        assert torch.equal(again[:, :, :H], got) and torch.equal(again[:, :, H:], packed[:, :, H:])


def test_append_reports_what_has_no_page(cuda_device):
    """Table entries that are no page, positions behind the table and counts beyond the tokens: reported, not written, and the
    rest of the call is done."""
    from frankentorch_b200.ops import decode as D
    from frankentorch_b200.ops import kernels as K
    g = _gen(1)
    k, v = _rnd(g, 2, 4, 1, 64), _rnd(g, 2, 4, 1, 64)
    for table, start, counts in (([[1, -1], [0, 0]], [6, 0], [4, 1]), ([[1, 3], [0, 0]], [6, 0], [4, 1]),
                                 ([[1, 2], [0, 0]], [14, 0], [4, 1]), ([[1, 2], [0, 0]], [-2, 0], [4, 1])):
        kp, vp = (torch.full((3, 1, 8, 64), math.nan, dtype=BF, device="cuda") for _ in range(2))
        D.paged_append(kp, vp, _i32(table), k, v, _i32(start), _i32(counts))
        with pytest.raises(K.KernelError, match="BAD_INDEX"):
            K.check_status()
        assert torch.equal(kp[0, :, 0], k[1, 0]) and torch.equal(vp[0, :, 0], v[1, 0])
        good = [p for p in range(start[0], start[0] + 4) if 0 <= p < 16 and 0 <= table[0][p // 8] < 3]
        for p in good:
            assert torch.equal(kp[table[0][p // 8], :, p % 8], k[0, p - start[0]])
        assert int((~kp.isnan()).sum()) == 64 * (len(good) + 1) and int((~vp.isnan()).sum()) == 64 * (len(good) + 1)
    for counts, rows in (([5, 1], 5), ([-1, 1], 1)):
        kp, vp = (torch.full((3, 1, 8, 64), math.nan, dtype=BF, device="cuda") for _ in range(2))
        D.paged_append(kp, vp, _i32([[1, 2], [0, 0]]), k, v, _i32([0, 0]), _i32(counts))
        with pytest.raises(K.KernelError, match="BAD_INDEX"):
            K.check_status()
        assert int((~kp.isnan()).sum()) == 64 * rows and torch.equal(kp[0, :, 0], k[1, 0])
    K.check_status()


# ------------------------------------------------------------------------------------------------ attention
def _attend(g, B, H, Hk, hd, page, lengths, dtype, layout="pages"):
    kp, vp, table = _cache(g, Hk, page, hd, lengths, dtype, layout=layout)
    _fill(g, kp, table, lengths)
    _fill(g, vp, table, lengths)
    q = _rnd(g, B, H + 3, hd, dtype=dtype)[:, 1: H + 1]
    return q, kp, vp, table


EDGES = [0, 1, 2, 7, 8, 9, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 255, 257, 300]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("H,Hk,page", [(1, 1, 16), (3, 3, 8), (4, 2, 64), (12, 4, 32), (7, 1, 1), (8, 1, 128), (9, 1, 4),
                                       (32, 2, 16), (17, 1, 2), (48, 1, 16), (40, 2, 256)])
def test_attention(cuda_device, H, Hk, page, hd, dtype):
    from frankentorch_b200.ops import decode as D
    from frankentorch_b200.ops import kernels as K
    g = _gen(H * page + hd)
    q, kp, vp, table = _attend(g, len(EDGES), H, Hk, hd, page, EDGES, dtype, "rows" if page == 32 else "pages")
    o, lse = D.paged_attention(q, kp, vp, table, _i32(EDGES))
    wo, wl, to, tl = attention64(q, kp, vp, table, EDGES)
    close(o, wo, to, "o")
    close(lse, wl, tl, "lse")
    assert bool((o[0] == 0).all())
    # a table for longer sequences: the heads are cut into pieces
    wide = torch.full((len(EDGES), 21 * 64 // page + 1), -7, dtype=torch.int32, device="cuda")
    wide[:, : table.shape[1]] = table[:, : wide.shape[1]]
    o2, lse2 = D.paged_attention(q, kp, vp, wide, _i32(EDGES))
    close(o2, wo, to, "o in pieces")
    close(lse2, wl, tl, "lse in pieces")
    out = torch.full((len(EDGES), H + 2, hd), 7.0, dtype=dtype, device="cuda")
    o2, lse2 = D.paged_attention(q, kp, vp, table, _i32(EDGES), out=out[:, 1:-1])
    assert torch.equal(o2, o) and torch.equal(lse2, lse)
    assert bool((out[:, 0] == 7).all()) and bool((out[:, -1] == 7).all())
    K.check_status()


@pytest.mark.parametrize("B,H,Hk,hd,page,lengths", [
    (1, 1, 1, 64, 16, [1]),
    (1, 1, 1, 128, 32, [5000]),                       # one head: nothing side by side but the length
    (1, 12, 12, 64, 16, [1025]),
    (2, 8, 1, 128, 64, [20011, 3]),
    (3, 16, 4, 64, 8, [0, 9001, 0]),
    (150, 2, 2, 64, 16, [(i * 37) % 90 for i in range(150)]),
    (40, 3, 1, 128, 64, [700 + 13 * i for i in range(40)]),
    (1000, 1, 1, 64, 8, [i % 3 for i in range(1000)]),
    (5, 2, 2, 128, 16, [0, 0, 0, 0, 0]),
])
@pytest.mark.parametrize("scale", [None, 0.3, -0.05])
def test_attention_over_lengths(cuda_device, B, H, Hk, hd, page, lengths, scale):
    from frankentorch_b200.ops import decode as D
    from frankentorch_b200.ops import kernels as K
    g = _gen(sum(lengths) + H)
    q, kp, vp, table = _attend(g, B, H, Hk, hd, page, lengths, BF)
    first = D.paged_attention(q, kp, vp, table, _i32(lengths), scale=scale)
    wo, wl, to, tl = attention64(q, kp, vp, table, lengths, scale)
    close(first[0], wo, to, "o")
    close(first[1], wl, tl, "lse")
    for _ in range(3):       # whatever the order in which parts are done, the same bits
        again = D.paged_attention(q, kp, vp, table, _i32(lengths), scale=scale)
        assert torch.equal(again[0], first[0]) and torch.equal(again[1], first[1])
    K.check_status()


@pytest.mark.parametrize("hd", [64, 128])
def test_attention_of_large_scores(cuda_device, hd):
    """Scores of some hundreds, of one sign at first and of the other later, and equal ones: the running maximum moves far."""
    from frankentorch_b200.ops import decode as D
    g = _gen(hd)
    n = 900
    q, kp, vp, table = _attend(g, 2, 4, 2, hd, 16, [n, n], HF)
    q = q * 8
    for b in range(2):
        p = torch.arange(n, device="cuda")
        idx = table[b].long()[p // 16]
        rows = kp[idx, :, p % 16] * 4
        rows[: n // 3] *= -1
        rows[n // 2:] = rows[n // 2]
        kp[idx, :, p % 16] = rows
    o, lse = D.paged_attention(q, kp, vp, table, _i32([n, n]))
    wo, wl, to, tl = attention64(q, kp, vp, table, [n, n])
    close(o, wo, to, "o")
    close(lse, wl, tl, "lse")


def test_attention_of_infinite_scores(cuda_device):
    """A token whose score is -inf has no weight; a row of nothing else is empty; NaN and +inf are the row's NaN."""
    from frankentorch_b200.ops import decode as D
    q = torch.ones(4, 2, 64, dtype=BF, device="cuda")
    kp = torch.zeros(8, 1, 16, 64, dtype=BF, device="cuda")
    vp = torch.ones(8, 1, 16, 64, dtype=BF, device="cuda")
    table = torch.arange(8, dtype=torch.int32, device="cuda").view(4, 2)
    kp[0, 0, 3, 0] = -math.inf
    vp[0, 0, 3] = 100.0
    kp[2:4, 0, :, 0] = -math.inf
    kp[4, 0, 7, 0] = math.inf
    kp[6, 0, 1, 0] = math.nan
    o, lse = D.paged_attention(q, kp, vp, table, _i32([20, 20, 20, 20]))
    assert bool((o[0] == 1).all()) and torch.allclose(lse[0], torch.full_like(lse[0], math.log(19)), atol=1e-5)
    assert bool((o[1] == 0).all()) and bool((lse[1] == -math.inf).all())
    assert bool(o[2:].isnan().all()) and bool(lse[2:].isnan().all())


def test_attention_reports_what_has_no_page(cuda_device):
    """Entries that are no page count as tokens that are not there; so do tokens behind the table."""
    from frankentorch_b200.ops import decode as D
    from frankentorch_b200.ops import kernels as K
    g = _gen(4)
    q, kp, vp, table = _attend(g, 2, 2, 2, 64, 16, [80, 40], BF)
    for change, lengths, keep in (((0, 1, -3), [80, 40], list(range(16)) + list(range(32, 80))),
                                  ((0, 4, kp.shape[0]), [80, 40], list(range(64)))):
        b, col, val = change
        t = table.clone()
        t[b, col] = val
        o, lse = D.paged_attention(q, kp, vp, t, _i32(lengths))
        with pytest.raises(K.KernelError, match="BAD_INDEX"):
            K.check_status()
        p = torch.tensor(keep, device="cuda")
        k, v = (x[table[0].long()[p // 16], :, p % 16].double() for x in (kp, vp))
        x = torch.einsum("hd,thd->ht", q[0].double(), k) / 8
        want = torch.einsum("ht,thd->hd", torch.softmax(x, -1), v)
        assert float((o[0].double() - want).abs().max()) <= 2.0 ** -7 * float(v.abs().max())
        full, _ = D.paged_attention(q, kp, vp, table, _i32([80, 40]))
        assert torch.equal(o[1], full[1])
    K.check_status()
    o, _ = D.paged_attention(q, kp, vp, table[:, :3].contiguous(), _i32([49, 40]))      # one token behind the table
    with pytest.raises(K.KernelError, match="BAD_INDEX"):
        K.check_status()
    full, _ = D.paged_attention(q, kp, vp, table, _i32([48, 40]))
    assert torch.equal(o, full)
    o, _ = D.paged_attention(q, kp, vp, table, _i32([-1, 40]))
    with pytest.raises(K.KernelError, match="BAD_INDEX"):
        K.check_status()
    assert bool((o[0] == 0).all()) and torch.equal(o[1], full[1])


def test_offsets_beyond_32_bits(cuda_device):
    """The last pages of a cache of more than 2^32 bytes, written and read."""
    from frankentorch_b200.ops import decode as D
    from frankentorch_b200.ops import kernels as K
    g = _gen(9)
    P = 2 ** 31 // (64 * 64) + 40                     # pages of 64 rows of one head: over 2^31 elements in all
    kp = torch.empty(P, 1, 64, 64, dtype=BF, device="cuda")
    vp = torch.empty(P, 1, 64, 64, dtype=BF, device="cuda")
    pages = [P - 1, 3, P - 17, 0, P - 30]
    table = _i32([pages])
    n = 64 * 4 + 11
    k, v, q = _rnd(g, 1, n, 1, 64), _rnd(g, 1, n, 1, 64), _rnd(g, 1, 5, 64)
    D.paged_append(kp, vp, table, k, v, _i32([0]))
    assert torch.equal(kp[P - 1, 0], k[0, :64, 0]) and torch.equal(vp[P - 30, 0, :11], v[0, 256:, 0])
    o, lse = D.paged_attention(q, kp, vp, table, _i32([n]))
    small = _i32([[0, 1, 2, 3, 4]])
    ks, vs = (t[torch.tensor(pages, device="cuda")].clone() for t in (kp, vp))
    want = D.paged_attention(q, ks, vs, small, _i32([n]))
    assert torch.equal(o, want[0]) and torch.equal(lse, want[1])
    K.check_status()


# ------------------------------------------------------------------------------------------------ logits
def _tokens(g, R, L, V):
    return torch.randint(0, max(1, min(V, L // 2 + 1)), (R, L), generator=g, device="cuda")


@pytest.mark.parametrize("dtype,to", [(BF, BF), (BF, torch.float32), (HF, HF), (HF, torch.float32), (torch.float32, torch.float32)])
@pytest.mark.parametrize("R,V,columns,L", [
    (1, 1, 8, 1), (3, 31, 31, 5), (2, 33, 40, 70), (1, 1000, 1024, 300), (4, 501, 512, 0), (2, 8193, 8200, 513),
    (5, 2047, 2047, 40)])
def test_logits(cuda_device, R, V, columns, L, dtype, to):
    from frankentorch_b200.ops import decode as D
    from frankentorch_b200.ops import kernels as K
    g = _gen(V + L)
    x = (3 * torch.randn(R, columns, generator=g, device="cuda")).to(dtype)
    tokens = _tokens(g, R, L, V)
    lengths = torch.randint(0, L + 1, (R,), generator=g, device="cuda", dtype=torch.int32)
    lengths[0] = L
    prompts = (lengths * torch.rand(R, generator=g, device="cuda")).to(torch.int32)
    rep, freq, pres = (s + torch.rand(R, generator=g, device="cuda") for s in (0.6, -0.5, -0.5))
    bias = torch.randn(R, V, generator=g, device="cuda")
    words = torch.randint(-2 ** 31, 2 ** 31 - 1, (R, (V + 31) // 32), generator=g, device="cuda").to(torch.int32)
    words[-1] = 0                                   # a row of which nothing is left
    lists = [t.double().tolist() for t in (rep, freq, pres)]
    pen = dict(repetition=rep, frequency=freq, presence=pres)
    hist = dict(tokens=tokens, lengths=lengths, prompt_lengths=prompts)
    want = (tokens.cpu(), lengths.cpu(), prompts.cpu())
    for kw, args in (
            (dict(**hist, **pen, bias=bias, allowed=words), (*want, *lists, bias, words.cpu())),
            (dict(**hist, **pen), (*want, *lists)),
            (dict(bias=bias[0], allowed=words[0]), (None,) * 6 + (bias[0], words[0].cpu())),
            (dict(tokens=tokens, repetition=1.3, frequency=0.25, presence=-0.5), (want[0], None, None, *([v] * R for v in (1.3, 0.25, -0.5)))),
            (dict(allowed=words[:1]), (None,) * 7 + (words[:1].cpu(),)),
            ({}, ())):
        got = D.logits_process(x, vocab=V, out_dtype=to, **kw)
        assert got.dtype == to
        close(got, *logits64(x, V, to, *args), sorted(kw))
    K.check_status()
    if dtype == to:                                 # over the logits themselves; the padding stays
        y = x.clone()
        D.logits_process(y, vocab=V, bias=bias, allowed=words, out=y[:, :V], **hist, **pen)
        assert torch.equal(y[:, :V], D.logits_process(x, vocab=V, bias=bias, allowed=words, **hist, **pen))
        assert torch.equal(y[:, V:], x[:, V:])


@pytest.mark.parametrize("shift", [0, 1, 3])
def test_logits_of_odd_rows(cuda_device, shift):
    """Rows that start on any element, of logits and results, negative row strides aside; the same values as of aligned ones."""
    from frankentorch_b200.ops import decode as D
    g = _gen(shift)
    R, V = 3, 777
    for dtype in (BF, torch.float32):
        store = torch.randn(R, V + 10 + shift, generator=g, device="cuda").to(dtype)
        x = store[:, shift: shift + V]
        bias = torch.randn(R, V + 5, generator=g, device="cuda")[:, shift: shift + V]
        tokens = _tokens(g, R, 50, V)
        out = torch.full((R, V + 20), 7.0, dtype=dtype, device="cuda")
        kw = dict(tokens=tokens, repetition=1.5, frequency=0.5, bias=bias)
        D.logits_process(x, out=out[:, 3: 3 + V], **kw)
        assert torch.equal(out[:, 3: 3 + V], D.logits_process(x.clone(), **kw))
        assert bool((out[:, :3] == 7).all()) and bool((out[:, 3 + V:] == 7).all())


def test_logits_of_values_that_are_not_finite(cuda_device):
    """What the mask forbids is -inf whatever it was; elsewhere infinities and NaN stay."""
    from frankentorch_b200.ops import decode as D
    x = torch.tensor([[math.nan, math.nan, math.inf, math.inf, -math.inf, -math.inf, 1.0, -3.0e38]], device="cuda")
    words = torch.tensor([0b11101010], dtype=torch.int32, device="cuda")
    got = D.logits_process(x, tokens=torch.tensor([[3, 5, 7]], device="cuda"), repetition=2.0, frequency=1.0, allowed=words)
    inf = math.inf
    assert got[0, [0, 2, 4]].tolist() == [-inf] * 3 and math.isnan(got[0, 1])
    assert got[0, 3] == inf and got[0, 5] == -inf and got[0, 6] == 1.0 and got[0, 7] == -inf


@pytest.mark.parametrize("R,V,L,dtype", [
    (3, 200003, 700, BF),             # a row in several pieces, runs that end inside a row
    (300, 5001, 90, torch.float32),   # a run of several rows
    (37, 70000, 5000, HF),            # more tokens than are requested ahead
    (2, 70001, 40000, BF),            # counts of 32 bits
    (149, 2048, 10, BF),
])
def test_logits_of_many_pieces(cuda_device, R, V, L, dtype):
    from frankentorch_b200.ops import decode as D
    from frankentorch_b200.ops import kernels as K
    g = _gen(R)
    x = (3 * torch.randn(R, V + 5, generator=g, device="cuda")).to(dtype)
    tokens = (torch.rand(R, L, generator=g, device="cuda", dtype=torch.float64) ** 2 * V).long()
    lengths = torch.randint(L // 2, L + 1, (R,), generator=g, device="cuda", dtype=torch.int32)
    prompts = lengths // 3
    rep, freq, pres = (0.5 + torch.rand(R, generator=g, device="cuda") for _ in range(3))
    bias = torch.randn(V, generator=g, device="cuda")
    words = torch.randint(-2 ** 31, 2 ** 31 - 1, (R, (V + 31) // 32), generator=g, device="cuda").to(torch.int32)
    got = D.logits_process(x, vocab=V, tokens=tokens, lengths=lengths, prompt_lengths=prompts, repetition=rep, frequency=freq,
                           presence=pres, bias=bias, allowed=words, out_dtype=torch.float32)
    K.check_status()
    ids = torch.arange(V, device="cuda")
    for r in range(R):
        n, m = int(lengths[r]), int(prompts[r])
        y = x[r, :V].double()
        seen = torch.bincount(tokens[r, :n], minlength=V) > 0
        made = torch.bincount(tokens[r, m:n], minlength=V)
        y = torch.where(seen, torch.where(y > 0, y / rep[r].double(), y * rep[r].double()), y)
        size = y.abs() + freq[r] * made + pres[r] * (made > 0) + bias.abs()
        y = y - freq[r].double() * made - pres[r].double() * (made > 0) + bias.double()
        allowed = words[r][ids // 32] >> (ids % 32) & 1 == 1
        assert torch.equal(got[r].isinf(), ~allowed)
        # six roundings of fp32 on what was added up, as above
        assert bool(((got[r].double() - y).abs() <= 6 * 2.0 ** -24 * size.double())[allowed].all())


def test_logits_count_far(cuda_device):
    """One token a hundred thousand times, and every history's place used."""
    from frankentorch_b200.ops import decode as D
    V, L = 70001, 100000
    x = torch.zeros(1, V, device="cuda")
    tokens = torch.full((1, L), V - 1, device="cuda")
    tokens[0, ::4] = torch.arange(L // 4, device="cuda")
    got = D.logits_process(x, tokens=tokens, frequency=0.5, presence=1.0)
    assert got[0, V - 1] == -0.5 * (L - L // 4) - 1.0
    assert bool((got[0, : L // 4] == -1.5).all()) and bool((got[0, L // 4: V - 1] == 0).all())


def test_logits_report_tokens_outside_the_vocabulary(cuda_device):
    from frankentorch_b200.ops import decode as D
    from frankentorch_b200.ops import kernels as K
    x = torch.zeros(2, 100, device="cuda")
    for bad in (-1, 100, 2 ** 40):
        got = D.logits_process(x, tokens=torch.tensor([[5, bad, 5], [7, 7, 7]], device="cuda"), frequency=1.0)
        with pytest.raises(K.KernelError, match="BAD_INDEX"):
            K.check_status()
        assert got[0, 5] == -2 and got[1, 7] == -3 and int((got != 0).sum()) == 2
    tokens = torch.tensor([[5, -1], [-1, -1]], device="cuda")
    got = D.logits_process(x, tokens=tokens, lengths=_i32([1, 0]), frequency=1.0)       # behind the lengths nothing is read
    K.check_status()
    assert got[0, 5] == -1 and int((got != 0).sum()) == 1
    D.logits_process(x, tokens=tokens, lengths=_i32([1, 3]), frequency=1.0)
    with pytest.raises(K.KernelError, match="BAD_INDEX"):
        K.check_status()


def test_logits_of_no_rows(cuda_device):
    from frankentorch_b200.ops import decode as D
    assert D.logits_process(torch.zeros(0, 50, device="cuda"), vocab=40).shape == (0, 40)


# ------------------------------------------------------------------------------------------------ streams and graphs
def _step(D, s):
    """One step's calls of a layer and the choice, as a program makes them."""
    q, k, v = s["qkv"].split([s["H"], s["Hk"], s["Hk"]], 2)
    q = D.paged_append(s["kp"], s["vp"], s["table"], k, v, s["start"], q=q, inv_freq=s["w"])
    o, lse = D.paged_attention(q[:, 0], s["kp"], s["vp"], s["table"], s["lengths"])
    x = D.logits_process(s["logits"], vocab=5000, tokens=s["tokens"], lengths=s["lengths"], repetition=1.2, frequency=0.1)
    return q, o, lse, x


def _state(D, seed, lengths):
    g = _gen(seed)
    B, H, Hk, hd = len(lengths), 8, 2, 64
    s = {"H": H, "Hk": Hk, "w": D.rotary_frequencies(hd)}
    s["kp"], s["vp"], s["table"] = _cache(g, Hk, 16, hd, [2048] * B, spare=0)
    for n in ("kp", "vp"):
        s[n].copy_(_rnd(g, *s[n].shape))
    s["qkv"] = _rnd(g, B, 1, H + 2 * Hk, hd)
    s["logits"] = _rnd(g, B, 5056)
    s["tokens"] = torch.randint(0, 5000, (B, 2048), generator=g, device="cuda")
    s["lengths"], s["start"] = _i32(lengths), _i32([n - 1 for n in lengths])
    return s


def test_captured_steps_follow_their_lengths(cuda_device):
    """Two graphs captured from calls that interleave, replayed with other lengths, next to each other on two streams."""
    from frankentorch_b200.ops import decode as D
    from frankentorch_b200.ops import kernels as K
    states = [_state(D, 1, [1, 700, 2048]), _state(D, 2, [1500, 3])]
    graphs, held = [], []
    for s in states:
        _step(D, s)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held.append(_step(D, s))
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for lengths in ([[2000, 1, 64], [65, 2048]], [[5, 6, 7], [2, 1]], [[2048, 2048, 2048], [2048, 1]]):
        want = []
        for s, n in zip(states, lengths):
            s["lengths"].copy_(_i32(n))
            s["start"].copy_(_i32([x - 1 for x in n]))
            want.append(_step(D, s))
        torch.cuda.synchronize()
        for _ in range(10):
            for graph, stream in zip(graphs, streams):
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        for got, ref in zip(held, want):
            for a, b in zip(got, ref):
                assert torch.equal(a, b)
    K.check_status()


FIRST_CALLS = """
import sys
sys.path[:0] = ["tests", "."]
import torch
import test_gpu_decode_ops as T
from frankentorch_b200.ops import decode as D
s = T._state(D, 3, [700, 1, 2048])
side = torch.cuda.Stream()
graph = torch.cuda.CUDAGraph()
torch.cuda.synchronize()
with torch.cuda.graph(graph):
    got = T._step(D, s)
graph.replay()
torch.cuda.synchronize()
held = [t.clone() for t in got]
want = T._step(D, s)
from frankentorch_b200.ops import kernels as K
K.check_status()
assert all(torch.equal(a, b) for a, b in zip(held, want))
print("the same")
"""


def test_first_calls_of_a_process_are_captured(cuda_device):
    import subprocess
    import sys
    from pathlib import Path
    out = subprocess.run([sys.executable, "-c", FIRST_CALLS], capture_output=True, text=True, timeout=300,
                         cwd=Path(__file__).resolve().parent.parent)
    assert out.returncode == 0 and "the same" in out.stdout, out.stderr[-2000:]


def test_tables_that_share(cuda_device):
    """Sequences with the same pages, a table that is a view into a wider one, or one row for all sequences."""
    from frankentorch_b200.ops import decode as D
    from frankentorch_b200.ops import kernels as K
    g = _gen(12)
    n = [700, 130, 1, 699]
    q, kp, vp, table = _attend(g, 1, 8, 2, 64, 16, [700], BF)
    q = _rnd(g, 4, 8, 64)
    wide = torch.full((4, table.shape[1] + 9), -1, dtype=torch.int32, device="cuda")
    wide[:, 3: 3 + table.shape[1]] = table
    for t in (table.expand(4, -1), wide[:, 3: 3 + table.shape[1]]):
        o, lse = D.paged_attention(q, kp, vp, t, _i32(n))
        wo, wl, to, tl = attention64(q, kp, vp, t, n)
        close(o, wo, to, "o")
        close(lse, wl, tl, "lse")
    K.check_status()


def test_calls_of_two_streams_and_threads(cuda_device):
    import threading

    from frankentorch_b200.ops import decode as D
    from frankentorch_b200.ops import kernels as K
    states = [_state(D, 5, [2048, 9]), _state(D, 6, [1000, 1001, 40, 2000, 1])]
    want = [_step(D, s) for s in states]
    torch.cuda.synchronize()
    bad = []

    def work(s, ref):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(30):
                got = _step(D, s)
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, ref)):
                    bad.append(1)
    threads = [threading.Thread(target=work, args=x) for x in zip(states, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    K.check_status()
    assert not bad
