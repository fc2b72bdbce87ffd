"""The 8-bit cache and the choice of a token in 64-bit and whole-number arithmetic on the host, block by block and row by row."""
import math

import torch

from _decode_oracle import rotary

E4M3 = torch.float8_e4m3fn


def scale_for(a):
    """The smallest power of two, 2^-100 at least, of which 448 times reaches ``a``."""
    e = -100
    if a > 0:
        m, x = math.frexp(a)                     # 0.5 <= m < 1
        e = max(-100, x - 9 + (m > 0.875))
    return 2.0 ** e


def bytes_of(t):
    return t.detach().cpu().view(torch.uint8)


def check_append(before, after, table, x, tol, start, counts, what):
    """``before`` and ``after``: (pages, scales) of one operand; ``x`` [B, S, Hkv, hd] in 64 bits (turned), off by up to ``tol``."""
    pages0, scales0, pages1, scales1 = (t.detach().cpu() for t in (*before, *after))
    table = table.cpu()
    page = pages0.shape[2]
    n = page // scales0.shape[2]
    left = torch.ones(pages0.shape[:3], dtype=torch.bool)            # rows that the call had nothing to do with
    scales_left = torch.ones(scales0.shape, dtype=torch.bool)
    for b in range(x.shape[0]):
        at, end = start[b], start[b] + counts[b]
        while at < end:
            stop = min(end, at // n * n + n)
            p, row = int(table[b, at // page]), at % page
            first = row // n * n
            for h in range(x.shape[2]):
                y = x[b, at - start[b]: stop - start[b], h]
                t = tol[b, at - start[b]: stop - start[b], h]
                fine = y.isfinite()
                a = float(torch.where(fine, y.abs(), 0.0).max())
                off = float(torch.where(fine, t, 0.0).max())
                s, had = float(scales1[p, h, row // n]), float(scales0[p, h, row // n])
                lo, hi = scale_for(max(0.0, a - off)), scale_for(a + off)
                if first < row:
                    lo, hi = max(lo, had), max(hi, had)
                assert lo <= s <= hi, (what, b, at, h, s, lo, hi, a)
                if first < row:
                    old = pages0[p, h, first:row].float()
                    want = old if s == had else (old * (had / s)).to(E4M3).float()
                    got = pages1[p, h, first:row].float()
                    assert torch.equal(got.nan_to_num(500.0), want.nan_to_num(500.0)), (what, "rows in place", b, at, h)
                got = pages1[p, h, row: row + stop - at].double() * s
                assert bool(got[~fine].isnan().all()), (what, "no number", b, at, h)
                # half a step: 2^-4 of the value, or of the smallest normal one, 2^-6 s
                bound = t + 2.0 ** -4 * (y.abs() + t).clamp(min=2.0 ** -6 * s)
                over = ((got - y).abs() - bound)[fine]
                assert over.numel() == 0 or float(over.max()) <= 0, (what, b, at, h, float(over.max()))
                left[p, h, first: row + stop - at] = False
                scales_left[p, h, row // n] = False
            at = stop
    assert torch.equal(bytes_of(pages1)[left], bytes_of(pages0)[left]), (what, "other rows")
    assert torch.equal(*(t[scales_left].view(torch.int32) for t in (scales1, scales0))), (what, "other scales")      # NaN too


def turned(k, freq, start, interleaved, dtype):
    """Keys turned in 64 bits and how far fp32 may be off (no rounding to 16 bits)."""
    y, tol = rotary(k, freq, start, interleaved)
    if freq is None:
        return y, torch.zeros_like(y)
    return y, tol - (tol > 0) * (torch.finfo(dtype).eps / 2 * y.abs() + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2)


def whole(pages, scales):
    """What the elements of a cache stand for, in fp64."""
    n = pages.shape[2] // scales.shape[2]
    return pages.cpu().double() * scales.cpu().double().repeat_interleave(n, 2)[..., None]


def choose(x, u, t=1.0, k=0, p=1.0, least=0.0):
    """(token, log-probability) of one row of logits: whole numbers and fractions throughout, but for exp."""
    x = [float(v) for v in x]
    if any(math.isnan(v) for v in (*x, u, t, p, least)) or t < 0:
        return -1, math.nan
    top = max(x)
    if top == -math.inf:
        return -1, -math.inf

    def weight(v):
        if v == top:
            return 2 ** 43
        if v == -math.inf or t == 0 or top == math.inf:
            return 0
        return round(math.exp((v - top) / t) * 2.0 ** 43)
    order = sorted(range(len(x)), key=lambda i: (-x[i], i))
    if t == 0:
        order = order[:1]
    elif k > 0:
        order = order[:k]
    w = {i: weight(x[i]) for i in order}
    if p < 1:
        n, d = max(p, 0.0).as_integer_ratio()
        total, before, kept = sum(w.values()), 0, []
        for i in order:
            if kept and before * d >= n * total:
                break
            kept.append(i)
            before += w[i]
        order = kept
    n, d = min(max(least, 0.0), 1.0).as_integer_ratio()
    order = [i for i in order if w[i] * d >= n * 2 ** 43]
    total = sum(w[i] for i in order)
    if u >= 1:
        target = total - 1
    else:
        n, d = max(u, 0.0).as_integer_ratio()
        target = n * total // d
    run = 0
    for i in sorted(order):
        run += w[i]
        if run > target:
            return i, math.log(w[i] / total)
    raise AssertionError("nothing is kept")
