"""Every form of the decoding attention and of the logits processing against 64-bit arithmetic: which one a call takes goes by
the number of heads and the width of the table, or by rows, columns and tokens, and each test says which it is about."""
import ctypes as C
import math

import pytest
import torch

from _decode_oracle import attention as attention64
from _decode_oracle import close, logits as logits64
from test_gpu_decode_ops import BF, HF, _attend, _gen, _i32, _tokens

LL, P = C.c_longlong, C.c_void_p


class _AttnDesc(C.Structure):
    """FtkPagedAttnDesc of csrc/ftk_api.h."""
    _fields_ = ([(n, LL) for n in ("type", "B", "Hq", "Hkv", "hd")] + [("scale", C.c_double), ("q", P), ("q_bs", LL), ("q_hs", LL),
                ("o", P), ("o_bs", LL), ("o_hs", LL), ("lse", P), ("k_pages", P), ("kp_ps", LL), ("kp_hs", LL), ("kp_rs", LL),
                ("v_pages", P), ("vp_ps", LL), ("vp_hs", LL), ("vp_rs", LL), ("table", P)] +
                [(n, LL) for n in ("table_stride", "table_cols", "n_pages", "page_shift")] + [("lengths", P)])


def form(B, H, Hk, hd, page, cols, dtype, sms):
    """What a call does, from the scratch that it asks for: "whole", or "heads" / "ctas" for heads cut into pieces with a
    header for each head or for each CTA."""
    from frankentorch_b200.ops import _lib
    fn = _lib.load()["ftk_paged_attn_scratch"]
    fn.argtypes, fn.restype = [C.POINTER(_AttnDesc)], LL
    d = _AttnDesc(type=1 if dtype is HF else 0, B=B, Hq=H, Hkv=Hk, hd=hd, table_cols=cols, n_pages=1,
                  page_shift=page.bit_length() - 1)
    got = fn(C.byref(d))
    group = H // Hk
    subs = -(-group // 16)
    rows = 8 if -(-group // subs) <= 8 else 16
    ctas, heads = (3 if hd == 64 and rows == 8 else 2) * sms, B * Hk * subs
    parts = ctas * 2 * rows * (hd + 2) * 4
    known = {0: "whole", parts + 32 * ctas: "ctas"}
    if heads < ctas:
        known[parts + 32 * heads] = "heads"
    return known[got]


def _sms():
    return torch.cuda.get_device_properties(0).multi_processor_count


def _compare(q, kp, vp, table, lengths):
    from frankentorch_b200.ops import decode as D
    from frankentorch_b200.ops import kernels as K
    o, lse = D.paged_attention(q, kp, vp, table, _i32(lengths))
    wo, wl, to, tl = attention64(q, kp, vp, table, lengths)
    close(o, wo, to, "o")
    close(lse, wl, tl, "lse")
    for _ in range(3):
        again = D.paged_attention(q, kp, vp, table, _i32(lengths))
        assert torch.equal(again[0], o) and torch.equal(again[1], lse)
    K.check_status()
    return o, lse


def _widened(table, tiles, page):
    """The same sequences under a table for ``tiles`` tiles of 64 tokens at least."""
    wide = torch.full((table.shape[0], max(table.shape[1], -(-tiles * 64 // page))), -7, dtype=torch.int32, device="cuda")
    wide[:, : table.shape[1]] = table
    return wide


@pytest.mark.gpu
@pytest.mark.parametrize("B,H,Hk,hd,page,dtype", [
    (40, 12, 12, 64, 16, BF),       # 480 heads, 444 CTAs
    (90, 20, 5, 64, 8, HF),         # groups of 4: 450
    (30, 90, 10, 64, 64, HF),       # groups of 9, sixteen rows: 300 heads, 296 CTAs
    (30, 40, 10, 128, 16, BF),
    (40, 8, 8, 128, 4, HF),
    (38, 128, 8, 128, 32, HF),      # groups of 16
    (50, 51, 3, 128, 64, BF),       # groups of 17, in two parts
    (75, 68, 2, 64, 128, BF),       # groups of 34, in three
])
@pytest.mark.parametrize("most", [1500, 200])
def test_attention_of_more_heads_than_ctas(cuda_device, B, H, Hk, hd, page, dtype, most):
    """Heads cut into pieces where there are more of them than CTAs: a header for each CTA.  Ragged, with empty sequences, the
    first and the last of the list among them; and short sequences under the same table."""
    g = _gen(B * H + most)
    lengths = [0 if b % 7 == 0 or b == B - 1 else 1 + (b * 389 + b * b * 31) % most for b in range(B)]
    lengths[B // 2] = most
    q, kp, vp, table = _attend(g, B, H, Hk, hd, page, lengths, dtype)
    table = _widened(table, 23, page)
    assert form(B, H, Hk, hd, page, table.shape[1], dtype, _sms()) == "ctas"
    o, lse = _compare(q, kp, vp, table, lengths)
    empty = torch.tensor([n == 0 for n in lengths])
    assert bool((o[empty] == 0).all()) and bool((lse[empty] == -math.inf).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("H,Hk,page", [(4, 4, 16), (8, 4, 8), (12, 4, 32), (36, 4, 64), (64, 4, 16), (51, 3, 2)])
def test_attention_of_whole_heads_that_share_an_sm(cuda_device, H, Hk, page, hd, dtype):
    """A short table and more heads than SMs: a CTA of four warps for each."""
    B = 45
    g = _gen(H + page)
    lengths = [(b * 29) % 320 for b in range(B)]
    q, kp, vp, table = _attend(g, B, H, Hk, hd, page, lengths, dtype, "rows" if page == 32 else "pages")
    assert B * Hk * -(-H // Hk // 16) > _sms() and form(B, H, Hk, hd, page, table.shape[1], dtype, _sms()) == "whole"
    _compare(q, kp, vp, table, lengths)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("H,Hk,page", [(12, 4, 32), (40, 2, 256), (7, 1, 1), (48, 1, 16)])
def test_attention_of_few_heads_in_pieces(cuda_device, H, Hk, page, hd, dtype):
    """A table wider than any limit for whole heads, fewer heads than CTAs: a header for each head."""
    lengths = [0, 1, 63, 64, 65, 127, 129, 300, 700, 2500]
    g = _gen(H + hd)
    q, kp, vp, table = _attend(g, len(lengths), H, Hk, hd, page, lengths, dtype)
    table = _widened(table, 40, page)
    assert form(len(lengths), H, Hk, hd, page, table.shape[1], dtype, _sms()) == "heads"
    _compare(q, kp, vp, table, lengths)


def test_forms_of_a_plan():
    """The rule behind the forms, without a GPU (148 SMs are what it counts on there)."""
    if torch.cuda.is_available():
        pytest.skip("the plan follows the GPU's SMs")
    assert form(1, 12, 12, 64, 16, 44, BF, 148) == "whole" and form(1, 12, 12, 64, 16, 45, BF, 148) == "heads"
    assert form(40, 12, 12, 64, 16, 80, BF, 148) == "whole" and form(40, 12, 12, 64, 16, 81, BF, 148) == "ctas"
    assert form(37, 12, 12, 64, 16, 92, BF, 148) == "ctas" and form(30, 12, 12, 64, 16, 92, BF, 148) == "heads"


# ------------------------------------------------------------------------------------------------ logits
def _penalties(g, R, V, L, least=0.5):
    tokens = (torch.rand(R, L, generator=g, device="cuda", dtype=torch.float64) ** 2 * V).long()
    lengths = torch.randint(L // 2, L + 1, (R,), generator=g, device="cuda", dtype=torch.int32)
    rep, freq, pres = (least + torch.rand(R, generator=g, device="cuda") for _ in range(3))
    return dict(tokens=tokens, lengths=lengths, prompt_lengths=lengths // 3, repetition=rep, frequency=freq, presence=pres)


def _check_rows(got, x, V, kw, bias, words):
    """Row by row in 64 bits: six roundings of fp32 on what was added up, as in the oracle, and one of a 16-bit result."""
    half = torch.finfo(got.dtype).eps / 2 if got.dtype != torch.float32 else 0.0
    ids = torch.arange(V, device="cuda")
    for r in range(x.shape[0]):
        n, m = int(kw["lengths"][r]), int(kw["prompt_lengths"][r])
        rep, freq, pres = (kw[p][r].double() for p in ("repetition", "frequency", "presence"))
        y = x[r, :V].double()
        seen = torch.bincount(kw["tokens"][r, :n], minlength=V) > 0
        made = torch.bincount(kw["tokens"][r, m:n], minlength=V)
        y = torch.where(seen, torch.where(y > 0, y / rep, y * rep), y)
        size = y.abs() + freq * made + pres * (made > 0)
        y = y - freq * made - pres * (made > 0)
        if bias is not None:
            size, y = size + bias.abs(), y + bias.double()
        allowed = words[r][ids // 32] >> (ids % 32) & 1 == 1 if words is not None else torch.ones_like(seen)
        assert torch.equal(got[r].isinf(), ~allowed)
        small = 2.0 ** -25 if got.dtype is HF else 0.0
        off = (got[r].double() - y).abs() - 6 * 2.0 ** -24 * size.double() - half * y.abs() - small
        assert float(off[allowed].max()) <= 0, (r, float(off[allowed].max()))


@pytest.mark.gpu
@pytest.mark.parametrize("R,V,columns,L,dtype,to,most", [
    (80, 128003, 128008, 3000, BF, BF, 65536),                 # runs of 69 thousand columns: pieces as long as they get
    (90, 128003, 128016, 500, HF, torch.float32, 65536),
    (220, 50257, 50304, 300, torch.float32, torch.float32, 65536),      # pieces that end with their row
    (40, 128003, 128008, 40000, BF, torch.float32, 32768),     # counts of 32 bits: runs of 34 thousand, cut at 32
    (45, 128003, 128004, 33000, torch.float32, torch.float32, 32768),
    (300, 5001, 5008, 90, BF, torch.float32, 0),               # vectors over runs of several rows
    (149, 2048, 2048, 10, HF, HF, 0),
    (37, 70000, 70000, 5000, torch.float32, torch.float32, 0),
])
def test_logits_of_long_runs(cuda_device, R, V, columns, L, dtype, to, most):
    """Rows on 16 bytes with histories, many per CTA.  ``most``: the piece's limit, which the runs of these sizes pass."""
    from frankentorch_b200.ops import decode as D
    from frankentorch_b200.ops import kernels as K
    run = -(-(-(-V // 64) * R) // _sms()) * 64
    assert run > most and (columns * torch.empty(0, dtype=dtype).element_size()) % 16 == 0
    g = _gen(R + V)
    x = (3 * torch.randn(R, columns, generator=g, device="cuda")).to(dtype)
    kw = _penalties(g, R, V, L)
    bias = torch.randn(V, generator=g, device="cuda")
    words = torch.randint(-2 ** 31, 2 ** 31 - 1, (R, (V + 31) // 32), generator=g, device="cuda").to(torch.int32)
    got = D.logits_process(x, vocab=V, bias=bias, allowed=words, out_dtype=to, **kw)
    _check_rows(got, x, V, kw, bias, words)
    bare = D.logits_process(x, vocab=V, out_dtype=to, **kw)
    _check_rows(bare, x, V, kw, None, None)
    if dtype == to:                  # over the logits themselves
        y = x.clone()
        D.logits_process(y, vocab=V, bias=bias, allowed=words, out=y[:, :V], **kw)
        assert torch.equal(y[:, :V], got) and torch.equal(y[:, V:], x[:, V:])
    K.check_status()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, torch.float32])
@pytest.mark.parametrize("shift", [0, 1, 3])
def test_logits_of_rows_on_and_off_16_bytes(cuda_device, shift, dtype):
    """Logits, results and biases that start on any element, and the same ones on 16 bytes, both against 64 bits."""
    from frankentorch_b200.ops import decode as D
    g = _gen(shift + 20)
    R, V = 3, 777
    x = torch.randn(R, V + 10 + shift, generator=g, device="cuda").to(dtype)[:, shift: shift + V]
    bias = torch.randn(R, V + 5, generator=g, device="cuda")[:, shift: shift + V]
    tokens = _tokens(g, R, 50, V)
    kw = dict(tokens=tokens, repetition=1.5, frequency=0.5)
    want = logits64(x, V, dtype, tokens.cpu(), None, None, [1.5] * R, [0.5] * R, [0.0] * R, bias)
    even = torch.zeros(R, 784, dtype=dtype, device="cuda")
    even[:, :V] = x
    flat = torch.zeros(R, 784, device="cuda")
    flat[:, :V] = bias
    out = torch.full((R, V + 20), 7.0, dtype=dtype, device="cuda")
    D.logits_process(x, out=out[:, 3: 3 + V], bias=bias, **kw)
    close(out[:, 3: 3 + V], *want, "off")
    assert bool((out[:, :3] == 7).all()) and bool((out[:, 3 + V:] == 7).all())
    for a in (even[:, :V], x):
        for b in (flat[:, :V], bias):
            close(D.logits_process(a, bias=b, **kw), *want, "on")
