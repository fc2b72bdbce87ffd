"""The 8-bit cache's attention over values and keys whose scales are as far apart as the append makes them, against 64-bit arithmetic."""
import math

import pytest
import torch

from _decode_oracle import attention as attention64
from _decode_oracle import close
from _served_oracle import E4M3, whole

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _weights_apart(q, k, v, ks, vs, table, lengths, scale=None):
    """What weights held in two halves of fp16 add to the bound: the largest weight of a head, value scale and all, is carried as 2^13 at
    least, and every weight is off by half of 2^-24 at most, so by 2^-38 of the largest; a value is 448 of its scale's unit at most."""
    n = vs.shape[2]
    q, table = q.double().cpu(), table.cpu()
    keys, scales = whole(k, ks), vs.cpu().double().repeat_interleave(k.shape[2] // n, 2)
    H, Hk = q.shape[1], k.shape[1]
    scale = 1.0 / math.sqrt(q.shape[2]) if scale is None else scale
    extra = torch.zeros(q.shape, dtype=torch.float64)
    for b, m in enumerate(lengths):
        if m == 0:
            continue
        p = torch.arange(m)
        at = table[b].long()[p // k.shape[2]], slice(None), p % k.shape[2]
        for h in range(H):
            g = h // (H // Hk)
            w = torch.softmax(scale * (keys[at][:, g] @ q[b, h]), 0) * scales[at][:, g]
            extra[b, h] = m * 448 * 2.0 ** -38 * float(w.max())
    return extra


def _check(q, k, v, table, lengths, ks, vs, scale=None):
    from frankentorch_b200.ops import decode as D
    from frankentorch_b200.ops import kernels as K
    wo, wl, to, tl = attention64(q, whole(k, ks), whole(v, vs), table, lengths, scale)
    to = to + _weights_apart(q, k, v, ks, vs, table, lengths, scale)
    page = k.shape[2]
    for cols in (table.shape[1], 60 * 64 // page + 1):          # left whole, and cut into pieces
        t = torch.full((table.shape[0], max(cols, table.shape[1])), -7, dtype=torch.int32, device="cuda")
        t[:, : table.shape[1]] = table
        o, lse = D.paged_attention(q, k, v, t, _i32(lengths), scale=scale, k_scales=ks, v_scales=vs)
        # The nearest multiple of 2^120 of 1.99 2^127 is 256, and 2^128 is beyond bf16: what passes the type's largest number by the bound,
        # or does not by less, may be infinite
        got = o.cpu().double()
        over = got.isinf() & (got.sign() == wo.sign()) & (wo.abs() + to > torch.finfo(o.dtype).max)
        close(torch.where(over, 0.0, got), torch.where(over, 0.0, wo), to, ("o", cols))
        close(lse, wl, tl, ("lse", cols))
    K.check_status()


# powers of two of the blocks' value scales, over and over: in the same 32 tokens, by 32 tokens (a warp's), by 64 and more (other tiles), and
# from one end to the other; None: a scale of 0
PATTERNS = {
    "low then high": lambda i, n: -100 if i < n // 2 else 40,
    "high then low": lambda i, n: 40 if i < n // 2 else -100,
    "ends, up": lambda i, n: -100 if i < n // 2 else 100,
    "ends, down": lambda i, n: 100 if i < n // 2 else -100,
    "within a warp's tokens": lambda i, n: (-100, 40, 100, None)[i % 4],
    "by warp": lambda i, n: (-100, 60)[i // 4 % 2],
    "by tile": lambda i, n: (60, None, -100)[i // 8 % 3],
    "slowly up": lambda i, n: -100 + 200 * i // max(n - 1, 1),
    "slowly down": lambda i, n: 100 - 200 * i // max(n - 1, 1),
    "one high": lambda i, n: 100 if i == n // 3 else -90,
}


@pytest.mark.parametrize("pattern", PATTERNS, ids=lambda p: p.replace(" ", "_"))
@pytest.mark.parametrize("H,Hk,hd", [(1, 1, 64), (3, 3, 128), (8, 2, 64), (6, 1, 128), (12, 1, 64), (32, 2, 128)])
def test_value_scales_far_apart(cuda_device, H, Hk, hd, pattern):
    """No token is left out of the sum, wherever the scales change."""
    g = _gen(H + hd)
    page, block, lengths = 16, 8, [1900, 61, 200, 9]
    cols = -(-max(lengths) // page)
    need = [-(-n // page) for n in lengths]
    order = torch.randperm(sum(need), generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(lengths), cols), -7, dtype=torch.int32, device="cuda")
    k, v = (torch.randn(sum(need), Hk, page, hd, generator=g, device="cuda").mul(100).clamp(-448, 448).to(E4M3) for _ in range(2))
    ks = torch.full((sum(need), Hk, page // block), 2.0 ** -7, device="cuda")
    vs = torch.ones(sum(need), Hk, page // block, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at: at + n]
        at += n
        blocks = -(-lengths[b] // block)
        for i in range(blocks):
            e = PATTERNS[pattern](i, blocks)
            vs[int(table[b, i // 2]), :, i % 2] = 0.0 if e is None else 2.0 ** e
    # 1.3 of a score on average: tokens of all blocks weigh about the same
    q = torch.randn(len(lengths), H, hd, generator=g, device="cuda").to(BF)
    _check(q, k, v, table, lengths, ks, vs)


def test_equal_scores_under_scales_far_apart(cuda_device):
    """Two tiles of equal scores: each has half of the weight."""
    from frankentorch_b200.ops import decode as D
    for low, high in ((-100, 40), (-100, 100), (None, 30)):
        for first in (0, 1):
            k = torch.zeros(2, 1, 64, 64, dtype=torch.uint8, device="cuda").view(E4M3)
            v = torch.ones(2, 1, 64, 64, device="cuda").to(E4M3)
            ks = torch.ones(2, 1, 1, device="cuda")
            vs = torch.full((2, 1, 1), 2.0 ** high, device="cuda")
            vs[first] = 0.0 if low is None else 2.0 ** low
            for H in (1, 4, 16):
                for cols in (2, 60):
                    table = torch.tensor([[0, 1] + [-1] * (cols - 2)], dtype=torch.int32, device="cuda")
                    o, lse = D.paged_attention(torch.ones(1, H, 64, dtype=BF, device="cuda"), k, v, table, _i32([128]), k_scales=ks, v_scales=vs)
                    assert bool((o.float() == 2.0 ** (high - 1)).all()), (low, high, first, H, cols)
                    assert float((lse - math.log(128)).abs().max()) < 1e-5


@pytest.mark.parametrize("H,Hk", [(2, 2), (8, 2)])
@pytest.mark.parametrize("zero_first", [True, False])
def test_a_zero_block_beside_large_values(cuda_device, H, Hk, zero_first):
    """A block of zeros, which the append gives its smallest scale, beside one of values of 2^90."""
    from frankentorch_b200.ops import decode as D
    g = _gen(3)
    n, page, hd = 256, 64, 64
    x = torch.randn(1, n, Hk, hd, generator=g, device="cuda").to(BF)
    y = (torch.randn(1, n, Hk, hd, generator=g, device="cuda") * 2.0 ** 90).to(BF)
    y[:, : n // 2] = 0
    if not zero_first:
        y = y.flip(1)
    k, v = (torch.zeros(n // page, Hk, page, hd, dtype=torch.uint8, device="cuda").view(E4M3) for _ in range(2))
    ks, vs = (torch.zeros(n // page, Hk, 2, device="cuda") for _ in range(2))
    table = torch.arange(n // page, dtype=torch.int32, device="cuda")[None]
    D.paged_append(k, v, table, x, y, _i32([0]), k_scales=ks, v_scales=vs)
    assert float(vs.min()) == 2.0 ** -100 and float(vs.max()) > 2.0 ** 80
    _check(torch.randn(1, H, hd, generator=g, device="cuda").to(BF), k, v, table, [n], ks, vs)


@pytest.mark.parametrize("H,Hk", [(2, 2), (8, 2), (12, 1)])
@pytest.mark.parametrize("q_size,k_size,v_size,scale", [
    (0, 0, 127, None), (-124, 127, 0, None), (-124, 127, 127, None), (0, 127, 0, 2.0 ** -126), (-20, 127, -99, 2.0 ** -106),
    (98, -95, 0, None), (127, -95, 127, 2.0 ** -31), (-60, 60, -95, None)])
def test_every_scale_that_the_append_makes(cuda_device, H, Hk, q_size, k_size, v_size, scale):
    """Keys and values up to the largest numbers of bf16, whose scales are 2^120, and as small ones; queries of a size that leaves scores of
    about 8."""
    from frankentorch_b200.ops import decode as D
    g = _gen(H + q_size + 200)
    n, page, hd = 300, 64, 64
    # 1 to 1.99, of either sign, times 2^k_size
    x, y = ((torch.rand(1, n, Hk, hd, generator=g, device="cuda").double() * 0.99 + 1) * torch.where(
        torch.rand(1, n, Hk, hd, generator=g, device="cuda") < 0.5, -1, 1) * 2.0 ** e for e in (k_size, v_size))
    x, y = x.to(BF), y.to(BF)
    assert bool(x.isfinite().all()) and bool(y.isfinite().all())
    q = (torch.randn(1, H, hd, generator=g, device="cuda").clamp(-1.9, 1.9).double() * 2.0 ** q_size).to(BF)
    P = -(-n // page)
    k, v = (torch.zeros(P, Hk, page, hd, dtype=torch.uint8, device="cuda").view(E4M3) for _ in range(2))
    ks, vs = (torch.zeros(P, Hk, 1, device="cuda") for _ in range(2))
    table = torch.arange(P, dtype=torch.int32, device="cuda")[None]
    D.paged_append(k, v, table, x, y, _i32([0]), k_scales=ks, v_scales=vs)
    for size, s in ((k_size, ks), (v_size, vs)):
        assert float(s.max()) == float(s.min()) == 2.0 ** max(size - 7, -100)
    _check(q, k, v, table, [n], ks, vs, scale)


@pytest.mark.parametrize("H", [1, 4, 12])
def test_a_page_that_is_none_before_scales_far_apart(cuda_device, H):
    """What is left of the sequence counts in full, however low its scores are."""
    from frankentorch_b200.ops import decode as D
    from frankentorch_b200.ops import kernels as K
    page, n, hd = 32, 600, 64
    P = -(-n // page)
    k = torch.ones(P, 1, page, hd, device="cuda").to(E4M3)
    v = torch.ones(P, 1, page, hd, device="cuda").to(E4M3)
    ks = torch.full((P, 1, 4), 64.0, device="cuda")
    vs = torch.tensor([2.0 ** 40, 2.0 ** -100] * 2, device="cuda").expand(P, 1, 4).contiguous()
    q = torch.full((1, H, hd), -0.5, dtype=BF, device="cuda")            # scores of -256
    for cols in (P, 60):
        table = torch.full((1, cols), -7, dtype=torch.int32, device="cuda")
        table[0, :P] = torch.arange(P, dtype=torch.int32, device="cuda")
        table[0, 0] = -3
        o, lse = D.paged_attention(q, k, v, table, _i32([n]), k_scales=ks, v_scales=vs)
        with pytest.raises(K.KernelError, match="BAD_INDEX"):
            K.check_status()
        assert float((lse.double() - (math.log(n - page) - 256)).abs().max()) < 256 * 68 * 2.0 ** -24
        high = sum(1 for t in range(page, n) if t // 8 % 2 == 0)
        assert float((o.double() / 2.0 ** 40 - high / (n - page)).abs().max()) <= 2.0 ** -8


@pytest.mark.parametrize("B,H,Hk,hd,n", [(2, 16, 1, 64, 2600), (4, 64, 4, 128, 2500), (8, 16, 4, 64, 2400), (8, 32, 4, 128, 1900), (3, 33, 11, 128, 2000)])
def test_few_heads_of_many_queries_in_pieces(cuda_device, B, H, Hk, hd, n):
    """Rows of the join that have an SM each, and more of them than SMs."""
    g = _gen(B * H)
    page, lengths = 64, [n - 37 * b for b in range(B)]
    P = -(-n // page)
    k, v = (torch.randn(B * P, Hk, page, hd, generator=g, device="cuda").mul(100).clamp(-448, 448).to(E4M3) for _ in range(2))
    ks, vs = (torch.exp2(torch.randint(-9, -5, (B * P, Hk, 2), generator=g, device="cuda").float()) for _ in range(2))
    table = torch.randperm(B * P, generator=g, device="cuda").to(torch.int32).view(B, P)
    _check(torch.randn(B, H, hd, generator=g, device="cuda").to(BF), k, v, table, lengths, ks, vs)


@pytest.mark.parametrize("H", [2, 7, 12, 16])
def test_queries_of_a_group_far_apart(cuda_device, H):
    """One head's queries are 2^140 times those of the others, whose scores are next to 0."""
    g = _gen(H)
    n, page, hd = 500, 64, 64
    P = -(-n // page)
    k, v = (torch.randn(P, 1, page, hd, generator=g, device="cuda").mul(100).clamp(-448, 448).to(E4M3) for _ in range(2))
    ks = torch.full((P, 1, 1), 2.0 ** -10, device="cuda")
    vs = torch.full((P, 1, 1), 2.0 ** -7, device="cuda")
    q = torch.randn(1, H, hd, generator=g, device="cuda").clamp(-1.9, 1.9) * 2.0 ** -13
    q[:, H // 2] *= 2.0 ** 70      # (2^140 is no number of fp32)
    q[:, H // 2] *= 2.0 ** 70
    assert bool(q.isfinite().all())
    _check(q.to(BF), k, v, torch.arange(P, dtype=torch.int32, device="cuda")[None], [n], ks, vs)
