"""Generation with drawn tokens: rows that end, and rows from which nothing can be drawn."""
import math

import pytest
import torch

from test_gpu_gpt_decode import _build

pytestmark = pytest.mark.gpu


def _decoder(cuda_device, batch=4):
    from frankentorch_b200.models.gpt_decode import GPTDecoder
    cfg, _, model = _build(cuda_device, "rotary", vocab_size=333)
    ids = torch.randint(0, 333, (batch, 20), generator=torch.Generator().manual_seed(6)).to(cuda_device)
    return GPTDecoder(model, batch, 80, page=16), ids, model


def _g(cuda_device):
    return torch.Generator(device=cuda_device).manual_seed(1)


@pytest.mark.parametrize("name,value", [("temperature", math.nan), ("temperature", -1.0), ("top_p", math.nan), ("min_p", math.nan)])
def test_settings_that_are_no_numbers(cuda_device, name, value):
    from frankentorch_b200.ops.kernels import KernelError
    dec, ids, _ = _decoder(cuda_device)
    rows = torch.tensor([0.7, value, 0.9, 0.5], device=cuda_device)
    with pytest.raises(KernelError, match=r"rows \[1\]: NaN"):
        dec.generate(ids, max_new_tokens=5, generator=_g(cuda_device), **{name: rows})
    # the decoder goes on
    tokens, totals = dec.generate(ids, max_new_tokens=5, generator=_g(cuda_device), **{name: rows.nan_to_num(0.5).abs()})
    assert totals.tolist() == [25] * 4


def test_logits_that_are_no_numbers(cuda_device):
    from frankentorch_b200.ops.kernels import KernelError
    dec, ids, model = _decoder(cuda_device)
    bias = torch.zeros(4, 333, device=cuda_device)
    bias[2, 7] = bias[3, 332] = math.nan
    for kw in (dict(temperature=0.0), dict(temperature=1.0), dict(top_k=3), dict(top_p=0.5)):
        with pytest.raises(KernelError, match=r"rows \[2, 3\]"):
            dec.generate(ids, max_new_tokens=3, bias=bias, generator=_g(cuda_device), **kw)
    model.arena.view(model.arena.params, "ln_f.weight")[5] = math.nan
    with pytest.raises(KernelError, match=r"rows \[0, 1, 2, 3\]"):
        dec.generate(ids, max_new_tokens=3, temperature=1.0)


def test_rows_that_end_are_no_errors(cuda_device):
    """A mask without a token ends a row, so does ``eos``; what their logits are afterwards is not looked at."""
    dec, ids, _ = _decoder(cuda_device)
    words = torch.full((4, 11), -1, dtype=torch.int32, device=cuda_device)
    words[1] = 0
    _, totals = dec.generate(ids, max_new_tokens=4, temperature=1.0, allowed=words, generator=_g(cuda_device))
    assert totals.tolist() == [24, 20, 24, 24]
    first = dec.generate(ids, max_new_tokens=1, temperature=0.0)[0][:, 20]
    bias = torch.zeros(4, 333, device=cuda_device)

    def allowed(tokens, totals):      # from the second token on row 0 has a NaN
        bias[0, 3] = math.nan if int(totals.max()) > 20 else 0.0
        return None
    _, totals = dec.generate(ids, max_new_tokens=4, temperature=0.0, bias=bias, allowed=allowed, eos=int(first[0]))
    assert int(totals[0]) == 21
