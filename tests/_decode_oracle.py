"""The operators of ``ops.decode`` in 64-bit arithmetic on the host, element by element or row by row, and how far a kernel
with fp32 arithmetic and one rounding may be off."""
import math

import torch


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rotary(x, freq, start, interleaved=False, inverse=False, counts=None):
    """``x`` [B, S, H, hd] turned, and the bound of its error per element."""
    y = x.double().cpu().clone()
    u, dtype = half_step(x.dtype), x.dtype
    B, S, H, hd = x.shape
    n = 0 if freq is None else freq.numel()
    tol = torch.zeros_like(y)
    for b in range(B):
        for s in range(S):
            if n == 0 or (counts is not None and s >= counts[b]):
                continue
            for i in range(n):
                a = (int(start[b]) + s) * float(freq[i])
                c, d = math.cos(a), math.sin(a) * (-1 if inverse else 1)
                j0, j1 = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
                x0, x1 = y[b, s, :, j0].clone(), y[b, s, :, j1].clone()
                y[b, s, :, j0], y[b, s, :, j1] = x0 * c - x1 * d, x1 * c + x0 * d
                # angle: three roundings in 64 bits on up to 2^31 radians, 2^-20 of a radian, and its fraction in fp32; sine and
                # cosine two units of 2^-23; the products two roundings: 2^-18 of |x0| + |x1| covers them
                tol[b, s, :, j0] = tol[b, s, :, j1] = 2.0 ** -18 * (x0.abs() + x1.abs())
    # and the rounding of the output; where nothing is turned there is neither
    turned = tol > 0
    return y, tol + turned * (u * y.abs() + torch.finfo(dtype).smallest_normal * u)


def gather(pages, table, b, n):
    """The first ``n`` rows of sequence ``b``: [heads, n, hd]."""
    p = torch.arange(n)
    return pages[table[b].long()[p // pages.shape[2]], :, p % pages.shape[2]].transpose(0, 1)


def attention(q, k_pages, v_pages, table, lengths, scale=None):
    """``(o, lse, bound of o, bound of lse)``."""
    u = half_step(q.dtype)
    q, table = q.cpu().double(), table.cpu()
    k_pages, v_pages = k_pages.cpu(), v_pages.cpu()
    B, H, hd = q.shape
    Hk = k_pages.shape[1]
    scale = 1.0 / math.sqrt(hd) if scale is None else scale
    o, to = torch.zeros_like(q), torch.zeros_like(q)
    lse, tl = torch.full((B, H), -math.inf, dtype=torch.float64), torch.zeros(B, H, dtype=torch.float64)
    for b in range(B):
        n = int(lengths[b])
        if n == 0:
            continue
        k, v = (gather(t, table, b, n).double() for t in (k_pages, v_pages))
        for h in range(H):
            g = h // (H // Hk)
            x = scale * (k[g] @ q[b, h])
            lse[b, h] = torch.logsumexp(x, 0)
            p = torch.exp(x - lse[b, h])
            o[b, h] = p @ v[g]
            # a score: hd products summed in fp32, in any order; exp of it; a probability carried with 16 bits or more; a sum of
            # n terms.  All of them relative to a probability, which both the numerator and the denominator have once.
            most = float((abs(scale) * (k[g].abs() @ q[b, h].abs())).max())
            e = (hd + 4) * 2.0 ** -24 * most + 2.0 ** -20 + 2.0 ** -17 + n * 2.0 ** -24
            to[b, h] = 2 * e * (p @ v[g].abs()) + u * o[b, h].abs() + torch.finfo(torch.float16).smallest_normal * u
            tl[b, h] = e + 2.0 ** -22 * abs(float(lse[b, h]))
    return o, lse, to, tl


def logits(x, vocab, out_dtype, tokens=None, lengths=None, prompts=None, rep=None, freq=None, pres=None, bias=None,
           allowed=None):
    """``(values, bound)``; penalties are lists per row or None."""
    y = x.cpu().double()[:, :vocab].clone()
    R = y.shape[0]
    size = torch.zeros_like(y)
    for r in range(R):
        count, seen = {}, set()
        if tokens is not None:
            n = tokens.shape[1] if lengths is None else int(lengths[r])
            for j in range(n):
                t = int(tokens[r, j])
                seen.add(t)
                if j >= (0 if prompts is None else int(prompts[r])):
                    count[t] = count.get(t, 0) + 1
        for t in seen:
            if rep is not None:
                y[r, t] = y[r, t] / rep[r] if y[r, t] > 0 else y[r, t] * rep[r]
        size[r] = y[r].abs()
        for t, n in count.items():
            f, p = (0.0 if freq is None else freq[r]), (0.0 if pres is None else pres[r])
            y[r, t] = y[r, t] - f * n - p
            size[r, t] += abs(f * n) + abs(p)
        if bias is not None:
            add = (bias if bias.dim() == 1 else bias[r % bias.shape[0]]).cpu().double()[:vocab]
            y[r] += add
            size[r] += add.abs()
        if allowed is not None:
            words = allowed if allowed.dim() == 1 else allowed[r % allowed.shape[0]]
            for t in range(vocab):
                if not (int(words[t // 32]) >> (t % 32)) & 1:
                    y[r, t] = -math.inf
    # up to six roundings in fp32 of what was added up, one of the result
    tol = 6 * 2.0 ** -24 * size + half_step(out_dtype) * y.abs() + 2.0 ** -149
    if out_dtype is torch.float16:
        tol = tol + 2.0 ** -25
    return y, torch.where(y.isfinite(), tol, torch.zeros_like(tol))


def close(got, want, tol, what):
    got = got.detach().cpu().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.equal(got.isfinite(), want.isfinite()), what
    f = want.isfinite()
    assert torch.equal(got[~f], want[~f]), what
    off = (got - want).abs()[f] - tol[f]
    assert off.numel() == 0 or float(off.max()) <= 0, (what, float(off.max()), float((got - want).abs()[f].max()))
