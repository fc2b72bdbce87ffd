"""Arguments that the 8-bit cache and the sampler refuse, without a GPU: every refusal comes before anything is launched."""
import math

import pytest
import torch

from frankentorch_b200.ops import decode as D
from frankentorch_b200.ops.kernels import KernelError

BF, E4 = torch.bfloat16, torch.float8_e4m3fn


def _z(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype)


def _e(*shape):
    return torch.zeros(*shape, dtype=torch.uint8).view(E4)


def _i(*v):
    return torch.tensor(v, dtype=torch.int32)


def _refused(match, fn, *a, **kw):
    with pytest.raises(KernelError, match=match):
        fn(*a, **kw)


CACHE = dict(k_pages=lambda: _e(5, 2, 16, 64), v_pages=lambda: _e(5, 2, 16, 64), k_scales=lambda: torch.ones(5, 2, 2),
             v_scales=lambda: torch.ones(5, 2, 2), table=lambda: torch.zeros(3, 4, dtype=torch.int32))
APPEND = dict(CACHE, k=lambda: _z(3, 7, 2, 64), v=lambda: _z(3, 7, 2, 64), start=lambda: _i(0, 0, 0))
ATTEND = dict(CACHE, q=lambda: _z(3, 4, 64), lengths=lambda: _i(1, 2, 3))

BOTH = [
    ("CUDA tensors", {}),
    ("need k_scales and v_scales", {"k_scales": lambda: None}),
    ("need k_scales and v_scales", {"v_scales": lambda: None}),
    ("need k_scales and v_scales", {"v_scales": lambda: None, "k_scales": lambda: None}),
    ("belong to pages of torch.float8_e4m3fn", {"k_pages": lambda: _z(5, 2, 16, 64), "v_pages": lambda: _z(5, 2, 16, 64)}),
    ("v_pages is torch.bfloat16", {"v_pages": lambda: _z(5, 2, 16, 64)}),
    ("k_pages is torch type Float8_e5m2", {"k_pages": lambda: _e(5, 2, 16, 64).view(torch.float8_e5m2), "k_scales": lambda: None,
                                           "v_scales": lambda: None}),
    ("v_pages is torch type Byte", {"v_pages": lambda: torch.zeros(5, 2, 16, 64, dtype=torch.uint8)}),
    ("k_scales must be fp32", {"k_scales": lambda: torch.ones(5, 2, 2, dtype=torch.float64)}),
    ("k_scales must be fp32", {"k_scales": lambda: torch.ones(5, 2)}),
    ("k_scales must be fp32", {"k_scales": lambda: torch.ones(4, 2, 2)}),
    ("k_scales must be fp32", {"k_scales": lambda: torch.ones(5, 3, 2)}),
    ("v_scales must be fp32", {"v_scales": lambda: torch.ones(5, 2, 4)[..., ::2]}),
    ("3 blocks for a page", {"k_scales": lambda: torch.ones(5, 2, 3)}),
    ("32 blocks for a page", {"v_scales": lambda: torch.ones(5, 2, 32)}),
    ("0 blocks for a page", {"v_scales": lambda: torch.ones(5, 2, 0)}),
    ("64 at most", {"k_pages": lambda: _e(5, 2, 128, 64), "v_pages": lambda: _e(5, 2, 128, 64), "k_scales": lambda: torch.ones(5, 2, 1),
                    "v_scales": lambda: torch.ones(5, 2, 1)}),
    ("differ", {"k_scales": lambda: torch.ones(5, 2, 4)}),
    ("16 bytes", {"v_pages": lambda: _e(5, 2, 16, 72)[..., :64]}),
    ("16 bytes", {"k_pages": lambda: _e(5 * 2 * 16 * 64 + 8)[8:].view(5, 2, 16, 64)}),
    ("must be a tensor", {"k_scales": lambda: 1.0}),
    ("page table", {"table": lambda: torch.zeros(2, 4, dtype=torch.int32)}),
    ("no pages", {"k_pages": lambda: _e(0, 2, 16, 64), "v_pages": lambda: _e(0, 2, 16, 64)}),
]


@pytest.mark.parametrize("base", [APPEND, ATTEND], ids=["append", "attention"])
@pytest.mark.parametrize("match,change", BOTH)
def test_caches(base, match, change):
    fn = D.paged_append if base is APPEND else D.paged_attention
    _refused(match, fn, **{n: f() for n, f in {**base, **change}.items()})


def test_append():
    def kw(**change):
        return {n: f() for n, f in {**APPEND, **change}.items()}
    _refused("k_scales is written", D.paged_append, **kw(k_scales=lambda: torch.ones(1, 2, 2).expand(5, 2, 2)))
    _refused("v_scales is written", D.paged_append, **kw(v_scales=lambda: torch.ones(5, 1, 2).expand(5, 2, 2)))
    _refused("k_pages is written", D.paged_append, **kw(k_pages=lambda: _e(1, 2, 16, 64).expand(5, 2, 16, 64)))
    _refused("bf16 or fp16", D.paged_append, **kw(k=lambda: _e(3, 7, 2, 64)))
    _refused("inv_freq is missing", D.paged_append, **kw(q=lambda: _z(3, 7, 4, 64)))
    # what is read may be shared
    _refused("CUDA tensors", D.paged_attention, **{n: f() for n, f in {**ATTEND, "k_scales": lambda: torch.ones(1, 1, 2).expand(5, 2, 2)}.items()})


SAMPLE = dict(logits=lambda: _z(2, 40, dtype=torch.float32), uniform=lambda: torch.zeros(2))


@pytest.mark.parametrize("match,change", [
    ("CUDA tensors", {}),
    ("bf16, fp16 or fp32", {"logits": lambda: _z(2, 40, dtype=torch.float64)}),
    ("bf16, fp16 or fp32", {"logits": lambda: _e(2, 40)}),
    ("rows, columns", {"logits": lambda: torch.zeros(2, 2, 40)}),
    ("rows, columns", {"logits": lambda: torch.zeros(40, 2).t()}),
    ("does not fit", {"vocab": lambda: 41}),
    ("does not fit", {"vocab": lambda: 0}),
    ("does not fit", {"vocab": lambda: -3}),
    ("2.20 are the most", {"logits": lambda: torch.empty(1, 2 ** 20 + 1).expand(2, -1)}),
    ("uniform must be", {"uniform": lambda: torch.zeros(3)}),
    ("uniform must be", {"uniform": lambda: torch.zeros(2, dtype=torch.float64)}),
    ("uniform must be", {"uniform": lambda: torch.zeros(2, 1)}),
    ("uniform must be", {"uniform": lambda: torch.zeros(4)[::2]}),
    ("uniform must be a tensor", {"uniform": lambda: 0.5}),
    ("uniform is missing", {"uniform": lambda: None}),
    ("temperature must be 0 or positive", {"temperature": lambda: -0.5}),
    ("temperature must be finite", {"temperature": lambda: math.inf}),
    ("temperature must be 0 or positive", {"temperature": lambda: 1e39}),
    ("temperature must be 0 or positive", {"temperature": lambda: 1e-50}),
    ("temperature must be finite", {"temperature": lambda: math.nan}),
    ("temperature must be a number or", {"temperature": lambda: torch.ones(3)}),
    ("temperature must be a number or", {"temperature": lambda: torch.ones(2, dtype=torch.float64)}),
    ("top_k must not be negative", {"top_k": lambda: -1}),
    ("top_k must not be negative", {"top_k": lambda: -5}),
    ("top_k must be contiguous int32", {"top_k": lambda: torch.ones(2, dtype=torch.int64)}),
    ("top_k must be contiguous int32", {"top_k": lambda: _i(1, 2, 3)}),
    ("top_p must be above 0", {"top_p": lambda: 0.0}),
    ("top_p must be above 0", {"top_p": lambda: 1.01}),
    ("top_p must be a number or", {"top_p": lambda: torch.ones(2, 1)}),
    ("min_p must be from 0 to 1", {"min_p": lambda: -0.1}),
    ("min_p must be from 0 to 1", {"min_p": lambda: 1.5}),
    ("min_p must be finite", {"min_p": lambda: math.nan}),
])
def test_sample(match, change):
    _refused(match, D.sample, **{n: f() for n, f in {**SAMPLE, **change}.items()})


def test_numbers_that_are_none():
    kw = {n: f() for n, f in SAMPLE.items()}
    for name in ("temperature", "top_k", "top_p", "min_p", "vocab"):
        with pytest.raises(TypeError):
            D.sample(**kw, **{name: "x"})
    with pytest.raises(TypeError):
        D.sample(**kw, top_k=2.5)
    with pytest.raises(OverflowError):
        D.sample(**kw, top_k=2 ** 70)
