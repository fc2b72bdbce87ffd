"""Infinities, NaN and extreme numbers in what the decoding operators read, against 64-bit arithmetic."""
import math

import pytest
import torch

from _decode_oracle import attention as attention64, logits as logits64
from test_gpu_decode_forms import _sms, _widened, form
from test_gpu_decode_ops import BF, HF, _attend, _gen, _i32

pytestmark = pytest.mark.gpu
INF = math.inf


def _same(got, want, tol, what):
    """Infinities and NaN where they belong, everything else within its bound."""
    got = got.detach().cpu().double()
    assert torch.equal(got.isnan(), want.isnan()), what
    assert torch.equal(got.isposinf(), want.isposinf()) and torch.equal(got.isneginf(), want.isneginf()), what
    f = want.isfinite()
    assert bool(((got - want).abs() <= tol)[f].all()), what


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("B,H,Hk,hd,page,tiles,kind", [
    (4, 3, 3, 64, 16, 0, "whole"), (4, 12, 2, 128, 64, 0, "whole"), (4, 20, 2, 64, 8, 0, "whole"),        # an SM for each head
    (40, 8, 8, 64, 16, 0, "whole"), (40, 36, 4, 128, 2, 0, "whole"),                                      # four warps
    (4, 3, 3, 64, 16, 40, "heads"), (4, 12, 2, 128, 8, 40, "heads"), (3, 17, 1, 64, 64, 40, "heads"),     # pieces
    (60, 16, 8, 64, 16, 23, "ctas"), (40, 72, 8, 128, 32, 23, "ctas"),
])
def test_attention_of_infinite_values(cuda_device, B, H, Hk, hd, page, tiles, kind, dtype):
    """An infinite value is infinity in its element of the output whatever its weight, two of opposite signs are NaN, and so
    is one whose weight is 0; the other elements are what they are without it."""
    g = _gen(B + H + hd)
    most = 300 if tiles == 0 else 1400
    lengths = [most - (b * 211) % most for b in range(B)]
    q, kp, vp, table = _attend(g, B, H, Hk, hd, page, lengths, dtype)
    table = _widened(table, tiles, page)
    assert form(B, H, Hk, hd, page, table.shape[1], dtype, _sms()) == kind
    q = q.clone()
    q[:, :, 0] = 8.0
    at = lambda b, t: (int(table[b, t // page]), t % page)         # noqa: E731
    for b, n in enumerate(lengths):
        if b % 3 == 2:
            continue                                               # a sequence without
        for col, t, v in ((1, n // 2, INF), (2, n - 1, -INF), (3, 0, INF), (3, n - 1, -INF), (5, n // 3, math.nan),
                          (6, 0, INF), (hd - 1, n // 2, INF), (hd - 1, n // 3, INF)):
            p, r = at(b, t)
            vp[p, b % Hk, r, col] = v
        if n > 40:
            # a token with a weight of e^-60 or less, which fp16 does not hold; and one whose score is -inf, which has none
            for t, k0, col in ((n // 4, -60.0 * math.sqrt(hd) / 8, 7), (n // 4 + 1, -INF, 8)):
                p, r = at(b, t)
                kp[p, b % Hk, r] = 0.0
                kp[p, b % Hk, r, 0] = k0
                vp[p, b % Hk, r, col] = INF
    from frankentorch_b200.ops import decode as D
    from frankentorch_b200.ops import kernels as K
    o, lse = D.paged_attention(q, kp, vp, table, _i32(lengths))
    K.check_status()
    wo, wl, to, tl = attention64(q, kp, vp, table, lengths)
    assert bool(wo.isposinf().any()) and bool(wo.isneginf().any()) and bool(wo.isnan().any())
    _same(o, wo, to, "o")
    _same(lse, wl, tl, "lse")
    again = D.paged_attention(q, kp, vp, table, _i32(lengths))[0]
    assert torch.equal(again.nan_to_num(), o.nan_to_num())


@pytest.mark.parametrize("dtype", [BF, HF, torch.float32])
@pytest.mark.parametrize("columns", [512, 501])
def test_logits_of_extreme_repetitions(cuda_device, columns, dtype):
    """Factors whose reciprocal fp32 does not hold, or holds in fewer bits: per row and as a number."""
    from frankentorch_b200.ops import decode as D
    V, big = 501, torch.finfo(torch.float32).max
    reps = [1e-45, 1e-40, 2.0 ** -128, 2.0 ** -127, 1.17e-38, 2.0 ** -64, 1.0, 1.5, 2.0 ** 64, 2.0 ** 126, 1e38, 3e38, big]
    R = len(reps)
    g = _gen(columns)
    x = torch.randn(R, columns, generator=g, device="cuda")
    # from the smallest numbers of fp32 to the largest, and zeros
    x = x * torch.exp2(torch.rand(R, columns, generator=g, device="cuda") * 250 - 125)
    x[:, ::50] = 0.0
    x = x.to(dtype)
    tokens = torch.arange(V, device="cuda").expand(R, -1)[:, ::2].contiguous()
    rep = torch.tensor(reps, dtype=torch.float32, device="cuda")
    want, tol = logits64(x, V, torch.float32, tokens.cpu(), None, None, rep.double().tolist(), None, None)
    # what leaves fp32's range is infinite there (from half a step above its largest number on)
    want = torch.where(want.abs() >= big * (1 + 2.0 ** -25), want.sign() * INF, want)
    near = want.isfinite() & (want.abs() > big * (1 - 2.0 ** -21))      # what six roundings may carry over the border
    tol = torch.where(want.isfinite(), tol, torch.zeros_like(tol))
    for got in (D.logits_process(x, vocab=V, tokens=tokens, repetition=rep, out_dtype=torch.float32),
                torch.cat([D.logits_process(x[r: r + 1], vocab=V, tokens=tokens[r: r + 1], repetition=float(rep[r]),
                                            out_dtype=torch.float32) for r in range(R)])):
        _same(torch.where(near.cuda(), want.float().cuda(), got), want, tol, "logits")
