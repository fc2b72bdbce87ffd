"""The choice of a token against whole-number arithmetic on the host: settings, ties, masks and odd values."""
import math

import pytest
import torch

from _served_oracle import choose

pytestmark = pytest.mark.gpu
BF, HF, FF = torch.bfloat16, torch.float16, torch.float32


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _values(v, R):
    return [float(torch.tensor(float(v)))] * R if not isinstance(v, torch.Tensor) else [float(x) for x in v.cpu()]


def _check(logits, u, vocab=None, **kw):
    from frankentorch_b200.ops import decode as D
    from frankentorch_b200.ops import kernels as K
    token, logprob = D.sample(logits, u, vocab=vocab, **kw)
    K.check_status()
    R, V = logits.shape[0], vocab or logits.shape[1]
    assert token.shape == logprob.shape == (R,) and token.dtype == torch.int64 and logprob.dtype == torch.float32
    x = logits[:, :V].double().cpu().tolist()
    t, k, p, least = (_values(kw.get(n, o), R) for n, o in (("temperature", 1.0), ("top_k", 0), ("top_p", 1.0), ("min_p", 0.0)))
    for r in range(R):
        want, lp = choose(x[r], float(u[r]), t[r], int(k[r]), p[r], least[r])
        got, glp = int(token[r]), float(logprob[r])
        assert got == want, (r, got, want, t[r], k[r], p[r], least[r])
        if math.isnan(lp) or math.isinf(lp):
            assert glp == lp or (math.isnan(glp) and math.isnan(lp)), (r, glp, lp)
        else:       # a quotient and a logarithm in 64 bits, one rounding
            assert abs(glp - lp) <= 2.0 ** -24 * abs(lp) + 1e-9, (r, glp, lp)
    return token, logprob


SETTINGS = [dict(), dict(temperature=0.0), dict(temperature=0.3), dict(temperature=5.0), dict(top_k=1), dict(top_k=7), dict(top_k=100000),
            dict(top_p=0.5), dict(top_p=1e-6), dict(top_p=0.999), dict(min_p=0.05), dict(min_p=1.0),
            dict(temperature=0.7, top_k=20, top_p=0.8), dict(temperature=1.3, top_p=0.9, min_p=0.02), dict(top_k=5, min_p=0.3),
            dict(temperature=2.0, top_k=50, top_p=0.95, min_p=0.001)]


@pytest.mark.parametrize("kw", SETTINGS, ids=lambda k: "-".join(f"{a}{b}" for a, b in k.items()) or "plain")
@pytest.mark.parametrize("dtype", [FF, BF, HF])
@pytest.mark.parametrize("R,V,columns,first", [(1, 1, 1, 0), (3, 2, 5, 1), (5, 33, 64, 0), (4, 777, 784, 8), (3, 2049, 2100, 3), (2, 20011, 20016, 0)])
def test_sample(cuda_device, R, V, columns, first, dtype, kw):
    g = _gen(V + R)
    # steps of bf16 and fp16 make many equal logits
    x = (3.0 * torch.randn(R, columns + first, generator=g, device="cuda")).to(dtype)[:, first:]
    _check(x, torch.rand(R, generator=g, device="cuda"), vocab=V, **kw)


def test_settings_per_row(cuda_device):
    g = _gen(3)
    R, V = 64, 3000
    x = 2.5 * torch.randn(R, V, generator=g, device="cuda")
    x[torch.rand(R, V, generator=g, device="cuda") < 0.5] = -math.inf
    r = torch.rand(5, R, generator=g, device="cuda")
    t = torch.where(r[0] < 0.2, 0.0, 2 * r[0])
    k = torch.where(r[1] < 0.4, 0, (300 * r[1]).int()).int()
    p = torch.where(r[2] < 0.3, 1.0, r[2])
    least = torch.where(r[3] < 0.4, 0.0, 0.2 * r[3])
    token, logprob = _check(x, r[4], temperature=t, top_k=k, top_p=p, min_p=least)
    # rows alone, in another order, and among others: the same tokens
    from frankentorch_b200.ops import decode as D
    for i in (0, 17, 63):
        a = D.sample(x[i: i + 1], r[4, i: i + 1], temperature=t[i: i + 1], top_k=k[i: i + 1], top_p=p[i: i + 1], min_p=least[i: i + 1])
        assert int(a[0]) == int(token[i]) and float(a[1]) == float(logprob[i])
    o = torch.randperm(R, generator=g, device="cuda")
    a = D.sample(x[o], r[4][o], temperature=t[o], top_k=k[o], top_p=p[o], min_p=least[o])
    assert torch.equal(a[0], token[o]) and torch.equal(a[1], logprob[o])


@pytest.mark.parametrize("kw", [dict(), dict(top_k=100), dict(top_p=0.25), dict(top_p=0.2501), dict(min_p=1.0), dict(temperature=0.0),
                                dict(top_k=100, top_p=0.5), dict(top_k=333, top_p=0.77, min_p=0.5)], ids=str)
@pytest.mark.parametrize("V", [1, 64, 1000, 4096, 30000])
def test_equal_logits(cuda_device, V, kw):
    """The order is that of the ids; sums of equal weights are exact, so the borders are hit."""
    u = torch.tensor([0.0, 0.25, 0.5, 0.75, 1 - 2.0 ** -24, 1e-30], device="cuda")
    _check(torch.full((6, V), -3.25, device="cuda"), u, **kw)
    x = torch.zeros(6, V, device="cuda")
    x[:, 1::2] = -0.0                     # zeros of either sign are equal
    _check(x, u, **kw)
    x = torch.zeros(6, V, device="cuda")
    x[:, ::3] = 1.0
    _check(x.to(BF), u, **kw)


def test_odd_rows(cuda_device):
    inf, nan = math.inf, math.nan
    V = 70
    base = torch.linspace(-2, 2, V, device="cuda")
    rows, u, t, p, least, k = [], [], [], [], [], []

    def row(x, uu=0.4, tt=1.0, pp=1.0, ll=0.0, kk=0):
        rows.append(x), u.append(uu), t.append(tt), p.append(pp), least.append(ll), k.append(kk)

    def put(**at):
        x = base.clone()
        for i, v in at.items():
            x[int(i[1:])] = v
        return x
    row(torch.full_like(base, -inf))                         # nothing allowed
    row(torch.full_like(base, -inf), tt=0.0)
    row(torch.full_like(base, torch.finfo(FF).min))          # the type's lowest value is a number
    row(put(i3=-inf, i69=-inf), uu=0.999999)
    row(put(i5=nan))
    row(put(i69=nan), tt=0.0)
    row(torch.full_like(base, nan))
    row(put(i3=inf, i9=inf), uu=0.7)                         # all the weight on two
    row(put(i3=inf, i9=inf), uu=0.7, pp=0.5)
    row(put(i3=inf, i9=nan))
    row(put(i3=inf, i9=inf), tt=inf, uu=0.7)
    row(put(i3=-inf), tt=inf, uu=0.5)                        # all equal
    row(put(i3=-inf), tt=inf, uu=0.5, kk=4)
    row(base, tt=nan)
    row(base, tt=-1.0)
    row(base, pp=nan)
    row(base, ll=nan)
    row(base, uu=nan)
    row(base, uu=1.0)
    row(base, uu=7.0, kk=10)
    row(base, uu=-3.0)
    row(base, pp=0.0)
    row(base, pp=-1.0, kk=3)
    row(base, pp=2.0)
    row(base, ll=-0.5)
    row(base, ll=1.5)
    row(base, kk=-4)
    row(base, kk=2 ** 31 - 1)
    row(100 * base, uu=0.999)                                # most weights are 0
    row(100 * base, uu=0.0)
    row(1e30 * base, uu=0.5)
    row(1e38 * base, uu=0.5, tt=1e-30)
    row(base, tt=1e-40)
    row(base, tt=1e38, uu=0.123)
    args = {n: torch.tensor(v, dtype=torch.float32, device="cuda") for n, v in (("temperature", t), ("top_p", p), ("min_p", least))}
    token, logprob = _check(torch.stack(rows), torch.tensor(u, device="cuda"), top_k=torch.tensor(k, dtype=torch.int32, device="cuda"), **args)
    assert token[:2].tolist() == [-1, -1] and logprob[:2].tolist() == [-inf, -inf]
    assert int(token[4]) == int(token[13]) == -1 and bool(logprob[4].isnan())


def test_every_token_can_be_drawn(cuda_device):
    """Random numbers on a grid: each token as often as its share, to within one of the grid's points at either end."""
    from frankentorch_b200.ops import decode as D
    g = _gen(9)
    V, n = 50, 4000
    x = torch.randn(1, V, generator=g, device="cuda")
    u = (torch.arange(n, device="cuda", dtype=torch.float64) / n).float()
    token, logprob = D.sample(x.expand(n, V), u, top_p=0.9)
    p = torch.softmax(x[0].double(), 0)
    order = p.argsort(descending=True)
    kept = order[: int((p[order].cumsum(0) < 0.9).sum()) + 1]
    share = torch.zeros(V, dtype=torch.float64, device="cuda")
    share[kept] = p[kept] / p[kept].sum()
    count = torch.bincount(token, minlength=V)
    assert float((count - n * share).abs().max()) <= 1.0
    assert bool((token.diff() >= 0).all())
    assert float((logprob.double() - share.log()[token]).abs().max()) < 1e-6


def test_large_vocabularies(cuda_device):
    """The largest one, and rows behind 2^31 elements of the tensor's start."""
    from frankentorch_b200.ops import decode as D
    from frankentorch_b200.ops import kernels as K
    g = _gen(4)
    V = 1 << 20
    x = torch.zeros(2, V, device="cuda")
    x[1] = torch.randn(V, generator=g, device="cuda")
    u = torch.tensor([1 - 2.0 ** -24, 0.5], device="cuda")
    token, logprob = D.sample(x, u)
    assert int(token[0]) == V - 1 and abs(float(logprob[0]) + math.log(V)) < 1e-5
    w = torch.exp(x[1].double() - x[1].max().double()).cumsum(0)
    assert abs(float(w[int(token[1])] / w[-1]) - 0.5) < 1e-4
    far = torch.empty(1 << 32, dtype=BF, device="cuda").as_strided((2, 1000), ((1 << 32) - 1024, 1))
    far.copy_(torch.randn(2, 1000, generator=g, device="cuda"))
    _check(far, u, top_k=20)
    K.check_status()


def test_streams_and_graphs(cuda_device):
    from frankentorch_b200.ops import decode as D
    g = _gen(5)
    x = torch.randn(6, 9000, generator=g, device="cuda")
    u = torch.rand(6, generator=g, device="cuda")
    k = torch.tensor([0, 1, 5, 50, 900, 9000], dtype=torch.int32, device="cuda")
    want = D.sample(x, u, top_k=k, top_p=0.9)
    with torch.cuda.stream(torch.cuda.Stream()):
        torch.cuda.current_stream().wait_stream(torch.cuda.default_stream())
        a = D.sample(x, u, top_k=k, top_p=0.9)
    torch.cuda.synchronize()
    assert torch.equal(a[0], want[0]) and torch.equal(a[1], want[1])
    gx, gu = torch.zeros_like(x), torch.zeros_like(u)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = D.sample(gx, gu, top_k=k, top_p=0.9)
    for shift in (0, 1, 2):
        gx.copy_(x.roll(shift, 1))
        gu.copy_(u.roll(shift))
        graph.replay()
        want = D.sample(gx, gu, top_k=k, top_p=0.9)
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
    none = D.sample(x[:0], u[:0])
    assert none[0].shape == none[1].shape == (0,)


@pytest.mark.parametrize("kw", [dict(top_k=127), dict(top_k=128), dict(top_k=129), dict(top_k=256), dict(top_k=257), dict(top_k=2000),
                                dict(top_k=400, top_p=0.6), dict(top_k=700, top_p=0.9, min_p=0.01)], ids=str)
@pytest.mark.parametrize("dtype", [FF, BF])
@pytest.mark.parametrize("V", [300, 5000, 40000])
def test_large_k(cuda_device, V, dtype, kw):
    """Around the sizes of a list, where the border is found by counts."""
    g = _gen(V)
    x = (2.0 * torch.randn(3, V, generator=g, device="cuda")).to(dtype)
    _check(x, torch.rand(3, generator=g, device="cuda"), **kw)


def _rows(kind, V, g):
    x = torch.randn(4, V, generator=g, device="cuda")
    if kind == "outlier":            # all others are in one step of the range
        x = 1e-3 * x
        x[:, V // 3] = 50.0
    elif kind == "cluster":          # a spread of a few units of fp32
        x = 100.0 + 2e-5 * x
    elif kind == "lowest":           # masked by the type's lowest value
        x[torch.rand(4, V, generator=g, device="cuda") < 0.7] = torch.finfo(FF).min
    elif kind == "scales":           # clusters within clusters
        x = torch.sign(x) * torch.exp2(-40 * torch.rand(4, V, generator=g, device="cuda"))
    elif kind == "two":              # two values, most of them the lower
        x = torch.where(x > 2.0, 1.0, -1.0)
    elif kind == "few":              # hardly any allowed
        x[torch.rand(4, V, generator=g, device="cuda") < 0.999] = -math.inf
        x[:, V - 1] = 0.0
    elif kind == "huge":
        x = 1e37 * x
    return x


@pytest.mark.parametrize("kw", [dict(temperature=20.0, top_p=0.9), dict(temperature=20.0, top_p=0.3, top_k=3000), dict(top_k=1500),
                                dict(top_k=100, temperature=50.0, top_p=0.99), dict(top_p=0.999, min_p=0.5), dict(temperature=1e38, top_p=0.5),
                                dict(temperature=30.0)], ids=str)
@pytest.mark.parametrize("kind", ["outlier", "cluster", "lowest", "scales", "two", "few", "huge"])
@pytest.mark.parametrize("dtype", [FF, HF, BF])
def test_rows_of_odd_spread(cuda_device, kind, kw, dtype):
    if dtype is HF and kind in ("huge", "lowest"):
        pytest.skip("no such numbers in fp16")
    g = _gen(17)
    _check(_rows(kind, 9001, g).to(dtype), torch.tensor([0.0, 0.3, 0.9, 0.999999], device="cuda"), **kw)


@pytest.mark.parametrize("kw", [dict(), dict(top_k=50, top_p=0.9), dict(top_k=5000), dict(top_p=0.8), dict(temperature=0.0)], ids=str)
@pytest.mark.parametrize("dtype,V", [(FF, 400003), (BF, 800009)])
def test_rows_that_shared_memory_does_not_hold(cuda_device, dtype, V, kw):
    g = _gen(23)
    x = (3.0 * torch.randn(1, V, generator=g, device="cuda")).to(dtype)
    _check(x, torch.tensor([0.6], device="cuda"), **kw)
    odd = torch.empty(V + 1, dtype=dtype, device="cuda")[1:].view(1, V)      # rows that start anywhere
    odd.copy_(x)
    _check(odd, torch.tensor([0.6], device="cuda"), **kw)


def test_many_rows(cuda_device):
    g = _gen(29)
    x = torch.randn(3000, 40, generator=g, device="cuda")
    _check(x, torch.rand(3000, generator=g, device="cuda"), temperature=1.3, top_k=11, top_p=0.9)
