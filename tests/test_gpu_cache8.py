"""The key-value cache in 8 bits: appending to it and attending over it, against 64-bit arithmetic, at the sizes, layouts and blocks
where they can go wrong."""
import math

import pytest
import torch

from _decode_oracle import attention as attention64
from _decode_oracle import close, rotary as rotary64
from _served_oracle import E4M3, bytes_of, check_append, turned, whole

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rnd(g, *shape, dtype=BF):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _cache(g, heads, page, block, hd, ends, spare=3, layout="pages"):
    """(k, v, ks, vs, table): shuffled pages for sequences of ``ends`` tokens, every row NaN and every scale NaN; the table's unused
    entries are no page at all."""
    need = [-(-n // page) for n in ends]
    P = sum(need) + spare

    def mk():
        if layout == "rows":       # heads innermost: [pages, page, heads, hd] in memory
            return torch.full((P, page, heads, hd), 0x7f, dtype=torch.uint8, device="cuda").view(E4M3).transpose(1, 2)
        return torch.full((P, heads, page, hd), 0x7f, dtype=torch.uint8, device="cuda").view(E4M3)

    def sc():
        if layout == "rows":
            return torch.full((heads, P, page // block), math.nan, device="cuda").transpose(0, 1)
        return torch.full((P, heads, page // block), math.nan, device="cuda")
    table = torch.full((len(ends), max(need + [1]) + 1), -7, dtype=torch.int32, device="cuda")
    order = torch.randperm(P, generator=g, device="cuda").to(torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at: at + n]
        at += n
    return mk(), mk(), sc(), sc(), table


def _fill(g, pages, scales, table, ends, powers=True):
    """Random values in the rows in use, under scales of a factor of up to 64 between blocks."""
    P, H, page, hd = pages.shape
    block = page // scales.shape[2]
    for b, n in enumerate(ends):
        if n == 0:
            continue
        p = torch.arange(n, device="cuda")
        idx = table[b].long()[p // page]
        y = (torch.randn(n, H, hd, generator=g, device="cuda") * 100).clamp(-448, 448).to(E4M3)
        raw = pages.view(torch.uint8)
        raw[idx, :, p % page] = y.view(torch.uint8)
        e = torch.randint(-9, -3, (n, H), generator=g, device="cuda").float()
        s = torch.exp2(e) if powers else torch.exp2(e) * (1 + torch.rand(n, H, generator=g, device="cuda"))
        first = p % block == 0
        scales[idx[first], :, (p[first] % page) // block] = s[first]


# ------------------------------------------------------------------------------------------------ append
@pytest.mark.parametrize("layout", ["pages", "rows"])
@pytest.mark.parametrize("dtype,interleaved", [(BF, False), (HF, True)])
@pytest.mark.parametrize("B,S,H,Hk,hd,turn,page,block,start,counts", [
    (1, 1, 12, 12, 64, 0, 16, 16, [300], None),
    (4, 1, 8, 2, 128, 128, 64, 64, [63, 64, 0, 1000], None),
    (3, 20, 4, 4, 64, 64, 8, 8, [0, 5, 31], [20, 0, 7]),
    (3, 17, 6, 1, 128, 64, 1, 1, [0, 2, 3], [17, 1, 16]),
    (2, 40, 2, 2, 32, 0, 32, 8, [1, 31], [39, 40]),
    (2, 9, 3, 3, 48, 16, 128, 64, [125, 100000], [9, 5]),
    (2, 150, 2, 1, 128, 128, 64, 64, [37, 0], [150, 129]),
    (1, 70, 4, 2, 256, 256, 64, 32, [3], [70]),
    (2, 5, 1, 1, 1024, 512, 16, 4, [14, 3], [5, 2]),
    (3, 33, 5, 5, 64, 32, 16, 2, [0, 1, 17], [33, 32, 31]),
    (1, 64, 1, 1, 1024, 1024, 64, 64, [0], None),        # more angles than shared memory holds
    (2, 1100, 16, 1, 128, 64, 64, 64, [5, 0], [1100, 900]),      # so many queries that they have a launch of their own
    (40, 3, 30, 10, 64, 64, 16, 16, [i * 7 for i in range(40)], [i % 4 for i in range(40)]),
])
def test_append(cuda_device, B, S, H, Hk, hd, turn, page, block, start, counts, dtype, interleaved, layout):
    from frankentorch_b200.ops import decode as D
    from frankentorch_b200.ops import kernels as K
    g = _gen(S + hd)
    used = counts or [S] * B
    ends = [a + n for a, n in zip(start, used)]
    k8, v8, ks, vs, table = _cache(g, Hk, page, block, hd, ends, layout=layout)
    _fill(g, k8, ks, table, start)
    _fill(g, v8, vs, table, start)
    # tokens of very different sizes, so that scales grow here and stay there
    packed = (_rnd(g, B, S, H + 2 * Hk, hd) * torch.exp2(torch.randint(-4, 5, (B, S, H + 2 * Hk, 1), generator=g, device="cuda").float())).to(dtype)
    q, k, v = packed.split([H, Hk, Hk], 2)
    w = D.rotary_frequencies(turn) if turn else None
    ct = None if counts is None else _i32(counts)
    before = [t.clone() for t in (k8, ks, v8, vs)]
    got = D.paged_append(k8, v8, table, k, v, _i32(start), ct, q=q if turn else None, inv_freq=w, interleaved=interleaved, k_scales=ks,
                         v_scales=vs)
    K.check_status()
    if turn:
        close(got, *rotary64(q, w, start, interleaved, counts=used), "q")
    else:
        assert got is None
    check_append(before[:2], (k8, ks), table, *turned(k, w, start, interleaved, dtype), start, used, "k")
    check_append(before[2:], (v8, vs), table, v.double().cpu(), torch.zeros(v.shape, dtype=torch.float64), start, used, "v")
    after = [t.clone() for t in (k8, ks, v8, vs)]
    again = packed.clone()       # once more, over the queries themselves: the same bits
    D.paged_append(k8, v8, table, k, v, _i32(start), ct, q=again[:, :, :H] if turn else None, inv_freq=w, interleaved=interleaved,
                   q_out=again[:, :, :H] if turn else None, k_scales=ks, v_scales=vs)
    for a, b in zip(after, (k8, ks, v8, vs)):
        assert torch.equal(bytes_of(a.contiguous()), bytes_of(b.contiguous()))
    if turn:
        assert torch.equal(again[:, :, :H], got) and torch.equal(again[:, :, H:], packed[:, :, H:])
    K.check_status()


def test_append_of_odd_values(cuda_device):
    """Zeros, the largest and smallest numbers, infinities and NaN: alone in a block and beside others."""
    from frankentorch_b200.ops import decode as D
    from frankentorch_b200.ops import kernels as K
    g = _gen(5)
    k8, v8, ks, vs, table = _cache(g, 1, 8, 4, 64, [32])
    x = _rnd(g, 1, 32, 1, 64)
    x[0, 0:4] = 0.0
    x[0, 4] = 448.0                                # reaches the scale 1 exactly
    x[0, 5, 0, 3] = -448.0
    x[0, 8, 0, 1] = 3.3895e38                      # the largest bf16
    x[0, 12, 0, 0] = 9.2e-41                       # the smallest
    x[0, 13:16] = 0.0
    x[0, 12, 0, 1:] = 0.0
    x[0, 17, 0, 5] = math.inf
    x[0, 18, 0, 6] = -math.inf
    x[0, 19, 0, 7] = math.nan
    x[0, 20:24] = math.inf                         # nothing finite
    x[0, 24, 0, 9] = 450.0                         # beyond 448
    before = [t.clone() for t in (k8, ks, v8, vs)]
    D.paged_append(k8, v8, table, x, -x, _i32([0]), k_scales=ks, v_scales=vs)
    K.check_status()
    zero = torch.zeros(x.shape, dtype=torch.float64)
    check_append(before[:2], (k8, ks), table, x.double().cpu(), zero, [0], [32], "k")
    check_append(before[2:], (v8, vs), table, -x.double().cpu(), zero, [0], [32], "v")
    at = [float(ks[int(table[0, p // 8]), 0, p % 8 // 4]) for p in range(0, 32, 4)]
    assert at[0] == 2.0 ** -100 and at[1] == 1.0 and at[2] == 2.0 ** 120 and at[3] == 2.0 ** -100 and at[5] == 2.0 ** -100 and at[6] == 2.0


def test_append_token_by_token_is_near_the_prompt(cuda_device):
    """One token after the other, scales growing on the way: every element within the roundings of its block's scales."""
    from frankentorch_b200.ops import decode as D
    g = _gen(6)
    n = 64
    k8, v8, ks, vs, table = _cache(g, 2, 64, 32, 64, [n])
    x = _rnd(g, 1, n, 2, 64) * torch.exp2(torch.linspace(-6, 6, n, device="cuda")).bfloat16()[None, :, None, None]
    for p in range(n):
        D.paged_append(k8, v8, table, x[:, p: p + 1], x[:, p: p + 1], _i32([p]), k_scales=ks, v_scales=vs)
    y = whole(k8, ks)[int(table[0, 0])].transpose(0, 1)
    one = [t.clone() for t in (k8, ks)]
    D.paged_append(k8, v8, table, x, x, _i32([0]), k_scales=ks, v_scales=vs)
    assert torch.equal(one[1][int(table[0, 0])], ks[int(table[0, 0])])      # the same largest elements, so the same scales
    s = ks[int(table[0, 0])].cpu().double().repeat_interleave(32, 1).transpose(0, 1)[..., None]
    want = x[0].double().cpu()
    # half a step of the element, and under the last scale half a step of the smallest numbers for each of the scales before: 2^-10 s
    # (1 + 1/2 + 1/4 ...)
    assert float(((y - want).abs() - (2.0 ** -4 * want.abs() + 2.0 ** -9 * s)).max()) <= 0


def test_append_reports_what_has_no_page(cuda_device):
    from frankentorch_b200.ops import decode as D
    from frankentorch_b200.ops import kernels as K
    g = _gen(1)
    k, v = _rnd(g, 2, 4, 1, 64), _rnd(g, 2, 4, 1, 64)
    for table, start, counts in (([[1, -1], [0, 0]], [6, 0], [4, 1]), ([[1, 3], [0, 0]], [6, 0], [4, 1]),
                                 ([[1, 2], [0, 0]], [14, 0], [4, 1]), ([[1, 2], [0, 0]], [-2, 0], [4, 1])):
        k8, v8 = (torch.full((3, 1, 8, 64), 0x7f, dtype=torch.uint8, device="cuda").view(E4M3) for _ in range(2))
        ks, vs = (torch.full((3, 1, 4), 1.0, device="cuda") for _ in range(2))
        D.paged_append(k8, v8, _i32(table), k, v, _i32(start), _i32(counts), k_scales=ks, v_scales=vs)
        with pytest.raises(K.KernelError, match="BAD_INDEX"):
            K.check_status()
        good = [p for p in range(start[0], start[0] + 4) if 0 <= p < 16 and 0 <= table[0][p // 8] < 3]
        assert int((~k8.float().isnan()).sum()) == 64 * (len(good) + 1) and int((~v8.float().isnan()).sum()) == 64 * (len(good) + 1)
        assert float(ks[0, 0, 0]) != 1.0 and int((ks != 1.0).sum()) <= 1 + len({(table[0][p // 8], p % 8 // 2) for p in good})
    for counts, rows in (([5, 1], 5), ([-1, 1], 1)):
        k8, v8 = (torch.full((3, 1, 8, 64), 0x7f, dtype=torch.uint8, device="cuda").view(E4M3) for _ in range(2))
        ks, vs = (torch.full((3, 1, 4), 1.0, device="cuda") for _ in range(2))
        D.paged_append(k8, v8, _i32([[1, 2], [0, 0]]), k, v, _i32([0, 0]), _i32(counts), k_scales=ks, v_scales=vs)
        with pytest.raises(K.KernelError, match="BAD_INDEX"):
            K.check_status()
        assert int((~k8.float().isnan()).sum()) == 64 * rows
    K.check_status()


# ------------------------------------------------------------------------------------------------ attention
EDGES = [0, 1, 2, 7, 8, 9, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 255, 257, 300]


def _attend(g, B, H, Hk, hd, page, block, lengths, dtype, layout="pages", powers=True):
    k8, v8, ks, vs, table = _cache(g, Hk, page, block, hd, lengths, layout=layout)
    _fill(g, k8, ks, table, lengths, powers)
    _fill(g, v8, vs, table, lengths, powers)
    return _rnd(g, B, H + 3, hd, dtype=dtype)[:, 1: H + 1], k8, v8, ks, vs, table


def _want(q, k8, v8, ks, vs, table, lengths, scale=None):
    return attention64(q, whole(k8, ks), whole(v8, vs), table, lengths, scale)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("H,Hk,page,block", [(1, 1, 16, 16), (3, 3, 8, 4), (4, 2, 64, 64), (12, 4, 32, 16), (7, 1, 1, 1), (8, 1, 128, 64),
                                             (9, 1, 4, 1), (32, 2, 16, 8), (17, 1, 2, 2), (48, 1, 16, 2), (40, 2, 256, 32)])
def test_attention(cuda_device, H, Hk, page, block, hd, dtype):
    from frankentorch_b200.ops import decode as D
    from frankentorch_b200.ops import kernels as K
    g = _gen(H * page + hd)
    q, k8, v8, ks, vs, table = _attend(g, len(EDGES), H, Hk, hd, page, block, EDGES, dtype, "rows" if page == 32 else "pages", page != 4)
    o, lse = D.paged_attention(q, k8, v8, table, _i32(EDGES), k_scales=ks, v_scales=vs)
    wo, wl, to, tl = _want(q, k8, v8, ks, vs, table, EDGES)
    close(o, wo, to, "o")
    close(lse, wl, tl, "lse")
    assert bool((o[0] == 0).all())
    # a table for longer sequences: the heads may be cut into pieces
    wide = torch.full((len(EDGES), 40 * 64 // page + 1), -7, dtype=torch.int32, device="cuda")
    wide[:, : table.shape[1]] = table[:, : wide.shape[1]]
    o2, lse2 = D.paged_attention(q, k8, v8, wide, _i32(EDGES), k_scales=ks, v_scales=vs)
    close(o2, wo, to, "o in pieces")
    close(lse2, wl, tl, "lse in pieces")
    out = torch.full((len(EDGES), H + 2, hd), 7.0, dtype=dtype, device="cuda")
    o2, lse2 = D.paged_attention(q, k8, v8, table, _i32(EDGES), out=out[:, 1:-1], k_scales=ks, v_scales=vs)
    assert torch.equal(o2, o) and torch.equal(lse2, lse)
    assert bool((out[:, 0] == 7).all()) and bool((out[:, -1] == 7).all())
    K.check_status()


@pytest.mark.parametrize("B,H,Hk,hd,page,block,lengths", [
    (1, 1, 1, 64, 16, 16, [1]),
    (1, 1, 1, 128, 32, 32, [5000]),                       # one head: nothing side by side but the length
    (1, 12, 12, 64, 16, 8, [1025]),
    (2, 8, 1, 128, 64, 64, [20011, 3]),
    (3, 16, 4, 64, 8, 8, [0, 9001, 0]),
    (150, 2, 2, 64, 16, 16, [(i * 37) % 90 for i in range(150)]),
    (40, 3, 1, 128, 64, 1, [700 + 13 * i for i in range(40)]),
    (1000, 1, 1, 64, 8, 2, [i % 3 for i in range(1000)]),
    (5, 2, 2, 128, 16, 16, [0, 0, 0, 0, 0]),
    (3, 32, 2, 64, 64, 32, [4000, 1, 2999]),
])
@pytest.mark.parametrize("scale", [None, 0.3, -0.05])
def test_attention_over_lengths(cuda_device, B, H, Hk, hd, page, block, lengths, scale):
    from frankentorch_b200.ops import decode as D
    from frankentorch_b200.ops import kernels as K
    g = _gen(sum(lengths) + H)
    q, k8, v8, ks, vs, table = _attend(g, B, H, Hk, hd, page, block, lengths, BF)
    first = D.paged_attention(q, k8, v8, table, _i32(lengths), scale=scale, k_scales=ks, v_scales=vs)
    wo, wl, to, tl = _want(q, k8, v8, ks, vs, table, lengths, scale)
    close(first[0], wo, to, "o")
    close(first[1], wl, tl, "lse")
    for _ in range(3):       # whatever the order in which parts are done, the same bits
        again = D.paged_attention(q, k8, v8, table, _i32(lengths), scale=scale, k_scales=ks, v_scales=vs)
        assert torch.equal(again[0], first[0]) and torch.equal(again[1], first[1])
    K.check_status()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("dtype,size", [(HF, 8.0), (BF, 8.0), (BF, 2.0 ** 40), (BF, 2.0 ** -60), (HF, 2.0 ** -14)])
def test_attention_of_large_and_small_scores(cuda_device, hd, dtype, size):
    """Scores of some hundreds whatever the size of the queries, of one sign at first and of the other later, and equal ones: the
    running maximum moves far."""
    from frankentorch_b200.ops import decode as D
    g = _gen(hd)
    n = 900
    q, k8, v8, ks, vs, table = _attend(g, 2, 4, 2, hd, 16, 16, [n, n], dtype)
    q = (q.float() * size).to(dtype)
    raw = k8.view(torch.uint8)
    for b in range(2):
        p = torch.arange(n, device="cuda")
        idx = table[b].long()[p // 16]
        rows = raw[idx, :, p % 16]
        rows[: n // 3] ^= 0x80
        rows[n // 2:] = rows[n // 2]
        raw[idx, :, p % 16] = rows
    scale = 32.0 / size / math.sqrt(hd)
    o, lse = D.paged_attention(q, k8, v8, table, _i32([n, n]), scale=scale, k_scales=ks, v_scales=vs)
    wo, wl, to, tl = _want(q, k8, v8, ks, vs, table, [n, n], scale)
    close(o, wo, to, "o")
    close(lse, wl, tl, "lse")


def test_attention_of_scales_far_apart(cuda_device):
    """Values whose scales are 2^90 and 2^-90, scales of 0, and a key's scale of 0: what fp32 holds of the result."""
    from frankentorch_b200.ops import decode as D
    g = _gen(11)
    lengths = [40, 40, 40, 40]
    q, k8, v8, ks, vs, table = _attend(g, 4, 4, 2, 64, 8, 8, lengths, BF)
    ks[:] = 2.0 ** -7
    vs[:] = 2.0 ** -7
    vs[table[0, 2].long()] = 2.0 ** 90
    for c in range(5):
        vs[table[1, c].long()] = 2.0 ** -90
    vs[table[2, 1].long()] = 0.0
    ks[table[2, 3].long()] = 0.0
    for c in range(5):
        vs[table[3, c].long()] = 0.0
    o, lse = D.paged_attention(q, k8, v8, table, _i32(lengths), k_scales=ks, v_scales=vs)
    wo, wl, to, tl = _want(q, k8, v8, ks, vs, table, lengths)
    close(o, wo, to, "o")
    close(lse, wl, tl, "lse")
    assert bool((o[3] == 0).all())


def test_attention_of_nan(cuda_device):
    """NaN behind the length has no influence, nor have its scales; before it a key's is its rows' NaN, a value's its element's."""
    from frankentorch_b200.ops import decode as D
    g = _gen(12)
    lengths = [37, 37, 37]
    q, k8, v8, ks, vs, table = _attend(g, 3, 4, 2, 64, 16, 4, lengths, BF)
    clean = D.paged_attention(q, k8, v8, table, _i32(lengths), k_scales=ks, v_scales=vs)
    assert bool(clean[0].isfinite().all())      # the rest of the last page is NaN
    k8.view(torch.uint8)[int(table[1, 1]), 0, 3, 5] = 0x7f
    v8.view(torch.uint8)[int(table[2, 2]), 1, 2, 9] = 0xff
    o, lse = D.paged_attention(q, k8, v8, table, _i32(lengths), k_scales=ks, v_scales=vs)
    assert torch.equal(o[0], clean[0][0]) and bool(o[1, :2].isnan().all()) and torch.equal(o[1, 2:], clean[0][1, 2:])
    assert bool(lse[1, :2].isnan().all()) and torch.equal(lse[2], clean[1][2])
    want = torch.zeros(4, 64, dtype=torch.bool, device="cuda")
    want[2:, 9] = True
    assert torch.equal(o[2].isnan(), want) and torch.equal(o[2][~want], clean[0][2][~want])


def test_attention_reports_what_has_no_page(cuda_device):
    from frankentorch_b200.ops import decode as D
    from frankentorch_b200.ops import kernels as K
    g = _gen(4)
    q, k8, v8, ks, vs, table = _attend(g, 2, 2, 2, 64, 16, 16, [80, 40], BF)
    kw = dict(k_scales=ks, v_scales=vs)
    for col, val, keep in ((1, -3, list(range(16)) + list(range(32, 80))), (4, k8.shape[0], list(range(64)))):
        t = table.clone()
        t[0, col] = val
        o, lse = D.paged_attention(q, k8, v8, t, _i32([80, 40]), **kw)
        with pytest.raises(K.KernelError, match="BAD_INDEX"):
            K.check_status()
        p = torch.tensor(keep)
        k, v = (whole(x, s)[table[0].cpu().long()[p // 16], :, p % 16] for x, s in ((k8, ks), (v8, vs)))
        x = torch.einsum("hd,thd->ht", q[0].double().cpu(), k) / 8
        want = torch.einsum("ht,thd->hd", torch.softmax(x, -1), v)
        assert float((o[0].double().cpu() - want).abs().max()) <= 2.0 ** -7 * float(v.abs().max())
        full, _ = D.paged_attention(q, k8, v8, table, _i32([80, 40]), **kw)
        assert torch.equal(o[1], full[1])
    K.check_status()
    o, _ = D.paged_attention(q, k8, v8, table[:, :3].contiguous(), _i32([49, 40]), **kw)      # one token behind the table
    with pytest.raises(K.KernelError, match="BAD_INDEX"):
        K.check_status()
    full, _ = D.paged_attention(q, k8, v8, table, _i32([48, 40]), **kw)
    assert torch.equal(o, full)
    o, _ = D.paged_attention(q, k8, v8, table, _i32([-1, 40]), **kw)
    with pytest.raises(K.KernelError, match="BAD_INDEX"):
        K.check_status()
    assert bool((o[0] == 0).all()) and torch.equal(o[1], full[1])


# ------------------------------------------------------------------------------------------------ together
def test_captured_steps_follow_the_device(cuda_device):
    """Appending and attending in one graph, replayed as the sequences grow, against the same calls made one by one; two graphs and an
    eager call of another stream in between."""
    from frankentorch_b200.ops import decode as D
    from frankentorch_b200.ops import kernels as K
    g = _gen(21)
    B, H, Hk, hd, page, block, steps = 3, 4, 2, 64, 16, 8, 20
    start = [0, 13, 30]
    ends = [n + steps for n in start]
    k8, v8, ks, vs, table = _cache(g, Hk, page, block, hd, ends)
    _fill(g, k8, ks, table, start)
    _fill(g, v8, vs, table, start)
    w = D.rotary_frequencies(hd)
    tokens = _rnd(g, steps, B, 1, H + 2 * Hk, hd)

    def step(x, at, c):
        q, k, v = x.split([H, Hk, Hk], 2)
        q = D.paged_append(c[0], c[1], table, k, v, at, q=q, inv_freq=w, k_scales=c[2], v_scales=c[3])
        return D.paged_attention(q[:, 0], c[0], c[1], table, at + 1, k_scales=c[2], v_scales=c[3])
    eager = [t.clone() for t in (k8, v8, ks, vs)]
    want = [step(tokens[i], _i32([n + i for n in start]), eager) for i in range(steps)]
    graphs = []
    for _ in range(2):
        c = [t.clone() for t in (k8, v8, ks, vs)]
        x, at = tokens[0].clone(), _i32(start)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(x, at, c)
        torch.cuda.current_stream().wait_stream(side)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = step(x, at, c)
        graphs.append((gr, x, at, c, out))
    for i in range(steps):
        for gr, x, at, c, out in graphs:
            x.copy_(tokens[i])
            at.copy_(_i32([n + i for n in start]))
            gr.replay()
        with torch.cuda.stream(torch.cuda.Stream()):
            torch.cuda.current_stream().wait_stream(torch.cuda.default_stream())
            other = step(tokens[i], _i32([n + i for n in start]), [t.clone() for t in eager])
        torch.cuda.synchronize()
        for gr, x, at, c, out in graphs:
            assert torch.equal(out[0], want[i][0]) and torch.equal(out[1], want[i][1]), i
        assert bool(other[0].isfinite().all())
    for gr, x, at, c, out in graphs:
        for a, b in zip(c, eager):
            assert torch.equal(bytes_of(a), bytes_of(b))
    K.check_status()


def test_empty_calls(cuda_device):
    from frankentorch_b200.ops import decode as D
    from frankentorch_b200.ops import kernels as K
    g = _gen(2)
    k8, v8, ks, vs, table = _cache(g, 2, 16, 16, 64, [16])
    kw = dict(k_scales=ks, v_scales=vs)
    none = _rnd(g, 0, 1, 2, 64)
    D.paged_append(k8, v8, table[:0], none, none, _i32([]), **kw)
    D.paged_append(k8, v8, table, _rnd(g, 1, 0, 2, 64), _rnd(g, 1, 0, 2, 64), _i32([3]), **kw)
    D.paged_append(k8, v8, table, _rnd(g, 1, 4, 2, 64), _rnd(g, 1, 4, 2, 64), _i32([3]), _i32([0]), **kw)
    assert bool(k8.float().isnan().all()) and bool(ks.isnan().all())
    o, lse = D.paged_attention(_rnd(g, 0, 4, 64), k8, v8, table[:0], _i32([]), **kw)
    assert o.shape == (0, 4, 64) and lse.shape == (0, 4)
    K.check_status()


@pytest.mark.parametrize("hd", [64, 128])
def test_pages_behind_32_bits(cuda_device, hd):
    """Pages whose first byte is more than 2^32 from the cache's: appended to and read where they are."""
    from frankentorch_b200.ops import decode as D
    from frankentorch_b200.ops import kernels as K
    g = _gen(31)
    P, H, page = (1 << 32) // (2 * 64 * hd) + 40, 2, 64
    k8, v8 = (torch.empty(P, H, page, hd, dtype=torch.uint8, device="cuda").view(E4M3) for _ in range(2))
    ks, vs = (torch.ones(P, H, 2, device="cuda") for _ in range(2))
    assert (P - 30) * H * page * hd > 1 << 32
    table = torch.tensor([[P - 1, 3, P - 20, P - 7], [P - 30, P - 2, 0, P - 9]], dtype=torch.int32, device="cuda")
    small = [t[table.flatten().long()].clone() if t.dtype != E4M3 else t.view(torch.uint8)[table.flatten().long()].view(E4M3).clone()
             for t in (k8, ks, v8, vs)]
    near = torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4)
    x, y = _rnd(g, 2, 200, H, hd), _rnd(g, 2, 200, H, hd)
    n = _i32([200, 150])
    D.paged_append(k8, v8, table, x, y, _i32([0, 0]), n, k_scales=ks, v_scales=vs)
    D.paged_append(small[0], small[2], near, x, y, _i32([0, 0]), n, k_scales=small[1], v_scales=small[3])
    q = _rnd(g, 2, 4, hd)
    far = D.paged_attention(q, k8, v8, table, n, k_scales=ks, v_scales=vs)
    want = D.paged_attention(q, small[0], small[2], near, n, k_scales=small[1], v_scales=small[3])
    assert torch.equal(far[0], want[0]) and torch.equal(far[1], want[1]) and bool(far[0].isfinite().all())
    K.check_status()


def test_calls_of_several_threads(cuda_device):
    """Two threads with streams and caches of their own at once: what each has alone."""
    import threading
    from frankentorch_b200.ops import decode as D
    from frankentorch_b200.ops import kernels as K

    def work(seed, out):
        with torch.cuda.stream(torch.cuda.Stream()):
            g = _gen(seed)
            lengths = [300 + seed, 50, 2000]
            q, k8, v8, ks, vs, table = _attend(g, 3, 8, 2, 64, 16, 16, lengths, BF)
            x = _rnd(g, 3, 1, 2, 64)
            for _ in range(20):
                D.paged_append(k8, v8, table, x, x, _i32([n - 1 for n in lengths]), k_scales=ks, v_scales=vs)
                o = D.paged_attention(q, k8, v8, table, _i32(lengths), k_scales=ks, v_scales=vs)
            torch.cuda.current_stream().synchronize()
            out[seed] = (o[0].clone(), o[1].clone(), k8.view(torch.uint8).clone())
    alone, both = {}, {}
    for seed in (1, 2):
        work(seed, alone)
    threads = [threading.Thread(target=work, args=(seed, both)) for seed in (1, 2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    for seed in (1, 2):
        for a, b in zip(alone[seed], both[seed]):
            assert torch.equal(a, b)
    K.check_status()


@pytest.mark.parametrize("group", [1, 3, 9])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("tiles", [16, 17, 60])
def test_more_heads_than_ctas_under_any_width_of_table(cuda_device, tiles, hd, group):
    from frankentorch_b200.ops import decode as D
    from frankentorch_b200.ops import kernels as K
    g = _gen(tiles + hd + group)
    lengths = [(i * 53) % 131 for i in range(96)]
    lengths[5], lengths[94] = 64 * 16, 64 * 15 + 1
    q, k8, v8, ks, vs, table = _attend(g, 96, 16 * group, 16, hd, 16, 8, lengths, BF)
    wide = torch.full((96, 4 * tiles), -7, dtype=torch.int32, device="cuda")
    wide[:, : min(4 * tiles, table.shape[1])] = table[:, : 4 * tiles]
    o, lse = D.paged_attention(q, k8, v8, wide, _i32(lengths), k_scales=ks, v_scales=vs)
    wo, wl, to, tl = _want(q, k8, v8, ks, vs, table, lengths)
    close(o, wo, to, "o")
    close(lse, wl, tl, "lse")
    again = D.paged_attention(q, k8, v8, wide, _i32(lengths), k_scales=ks, v_scales=vs)
    assert torch.equal(o, again[0]) and torch.equal(lse, again[1])
    K.check_status()


def test_many_queries_turned_where_they_are(cuda_device):
    from frankentorch_b200.ops import decode as D
    from frankentorch_b200.ops import kernels as K
    g = _gen(77)
    B, S, H, Hk, hd, page, block = 5, 700, 16, 3, 128, 64, 32
    start, counts = [0, 31, 5, 64, 1], [700, 699, 0, 1, 350]
    x = _rnd(g, B, S, H + 2 * Hk, hd)
    before = x.clone()
    q, k, v = x.split([H, Hk, Hk], 2)
    w = 10000.0 ** (-torch.arange(hd // 2, dtype=torch.float64, device="cuda") / (hd // 2))
    k8, v8, ks, vs, table = _cache(g, Hk, page, block, hd, [s + c for s, c in zip(start, counts)])
    other = tuple(t.clone() for t in (k8.view(torch.uint8), v8.view(torch.uint8), ks, vs))
    apart = D.paged_append(other[0].view(E4M3), other[1].view(E4M3), table, k, v, _i32(start), _i32(counts), q=q, inv_freq=w,
                           q_out=torch.empty(B, S, H, hd, dtype=BF, device="cuda"), k_scales=other[2], v_scales=other[3])
    D.paged_append(k8, v8, table, k, v, _i32(start), _i32(counts), q=q, inv_freq=w, q_out=q, k_scales=ks, v_scales=vs)
    assert torch.equal(q, apart) and torch.equal(x[:, :, H:], before[:, :, H:])
    for b, n in enumerate(counts):
        assert torch.equal(q[b, n:], before[b, n:, :H])
        if n:
            at = start[b] + torch.arange(n, device="cuda")
            angle = at.double()[:, None] * w
            c, s = angle.cos()[:, None], angle.sin()[:, None]
            lo, hi = before[b, :n, :H].double().split(hd // 2, -1)
            want = torch.cat([lo * c - hi * s, hi * c + lo * s], -1)
            size = torch.cat([(lo * c).abs() + (hi * s).abs(), (hi * c).abs() + (lo * s).abs()], -1)
            assert bool(((q[b, :n].double() - want).abs() <= want.abs() * 2.0 ** -8 + size * 2.0 ** -20).all())
    for mine, theirs in ((k8.view(torch.uint8), other[0]), (v8.view(torch.uint8), other[1]), (ks.view(torch.int32), other[2].view(torch.int32)),
                         (vs.view(torch.int32), other[3].view(torch.int32))):
        assert torch.equal(mine, theirs)
    K.check_status()
