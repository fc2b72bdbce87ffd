"""The sampler at the sizes of serving batches: one, two, four and eight CTAs to a row and the most steps of each, against whole-number arithmetic
for some rows and against the same rows alone for all."""
import math

import pytest
import torch

from _served_oracle import choose

pytestmark = pytest.mark.gpu
BF, HF, FF = torch.bfloat16, torch.float16, torch.float32


def _batch(seed, R, V, dtype):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = -1.2 * torch.log1p(V * torch.rand(R, V, generator=g, device="cuda")) + 0.3 * torch.randn(R, V, generator=g, device="cuda")
    x[R // 3: R // 2, :][torch.rand(R // 2 - R // 3, V, generator=g, device="cuda") < 0.3] = -math.inf
    r = torch.rand(9, R, generator=g, device="cuda")
    kw = dict(temperature=torch.where(r[0] < 0.1, 0.0, 0.3 + 1.2 * r[1]), top_k=torch.where(r[2] < 0.5, 0.0, torch.exp(6.5 * r[3])).int(),
              top_p=torch.where(r[4] < 0.25, 1.0, 0.3 + 0.69 * r[5]), min_p=torch.where(r[6] < 0.6, 0.0, 0.2 * r[7]))
    return x.to(dtype), r[8].contiguous(), kw


@pytest.mark.parametrize("R,V,dtype,some", [
    (256, 50257, FF, 24), (512, 128003, BF, 6), (160, 50257, HF, 8),
    (640, 13312, FF, 24), (640, 13313, FF, 24), (640, 14336, FF, 12), (512, 26624, FF, 12), (512, 27500, FF, 12), (256, 53249, FF, 8),
    (300, 57344, FF, 6), (256, 114688, FF, 4), (620, 26624, BF, 8), (620, 28672, BF, 8), (3000, 1025, HF, 40)])
def test_batches(cuda_device, R, V, dtype, some):
    from frankentorch_b200.ops import decode as D
    from frankentorch_b200.ops import kernels as K
    x, u, kw = _batch(V, R, V, dtype)
    token, logprob = D.sample(x, u, **kw)
    for r in torch.randperm(R, generator=torch.Generator().manual_seed(1))[:some].tolist():
        s = {n: float(v[r]) for n, v in kw.items()}
        want, lp = choose(x[r].double().cpu().tolist(), float(u[r]), s["temperature"], int(s["top_k"]), s["top_p"], s["min_p"])
        assert int(token[r]) == want, (r, s)
        assert abs(float(logprob[r]) - lp) <= 2.0 ** -24 * abs(lp) + 1e-9, (r, s)
    for r in range(0, R, max(1, R // 256)):
        one = D.sample(x[r: r + 1], u[r: r + 1], **{n: v[r: r + 1] for n, v in kw.items()})
        assert int(one[0]) == int(token[r]) and float(one[1]) == float(logprob[r]), r
    K.check_status()
