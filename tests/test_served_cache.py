"""The decoder's cache in 8 bits and the settings of its choice, as far as that goes without a GPU."""
import pytest
import torch

from frankentorch_b200.autograd.tape import TensorTape
from frankentorch_b200.models.gpt import GPT, GPTConfig
from frankentorch_b200.models.gpt_decode import GPTDecoder, PagedKVCache

E4 = torch.float8_e4m3fn


def _cache(**kw):
    return PagedKVCache(2, 3, 64, **{**dict(pages=6, batch=3, max_tokens=40, page=8, device="cpu", dtype=E4), **kw})


def test_pages_and_scales():
    c = _cache()
    assert c.k.shape == c.v.shape == (2, 6, 3, 8, 64) and c.k.dtype == c.v.dtype == E4
    assert c.k_scales.shape == c.v_scales.shape == (2, 6, 3, 1) and c.k_scales.dtype == torch.float32
    s = c.scales(1)
    assert s["k_scales"].data_ptr() == c.k_scales[1].data_ptr() and s["v_scales"].data_ptr() == c.v_scales[1].data_ptr()
    assert _cache(page=128).k_scales.shape == (2, 6, 3, 2) and _cache(block=2).v_scales.shape == (2, 6, 3, 4)
    assert not bool(c.k.view(torch.uint8).any())
    half = _cache(dtype=torch.bfloat16)
    assert half.scales(0) == {} and half.k_scales is None and half.k.dtype == torch.bfloat16


@pytest.mark.parametrize("kw", [dict(block=16), dict(block=0), dict(block=3), dict(page=128, block=128), dict(block=-8),
                                dict(dtype=torch.bfloat16, block=8), dict(dtype=torch.float16, block=1)])
def test_blocks_that_are_refused(kw):
    with pytest.raises(ValueError):
        _cache(**kw)


def _model(**kw):
    cfg = GPTConfig(**{**dict(n_layer=1, d_model=128, n_head=2, d_ff=256, vocab_size=100, max_seq=32, name="t"), **kw})
    return GPT(cfg, TensorTape(grad_dtype=None), device="cpu")


def test_decoder():
    d = GPTDecoder(_model(), 2, 32, page=16, cache_dtype=E4, cache_block=4)
    assert d.cache.k.dtype == E4 and d.cache.k_scales.shape == (1, 4, 2, 4)
    assert GPTDecoder(_model(), 2, 32).cache.k_scales is None
    with pytest.raises(ValueError, match="bfloat16 or float8"):
        GPTDecoder(_model(), 2, 32, cache_dtype=torch.float16)
    with pytest.raises(ValueError, match="no scales"):
        GPTDecoder(_model(), 2, 32, cache_block=4)


def test_choices_that_do_not_go_together():
    d = GPTDecoder(_model(), 2, 32, page=16)
    ids = torch.zeros(2, 4, dtype=torch.int64)
    for kw in (dict(temperature=1.0), dict(top_k=3), dict(top_p=0.5), dict(min_p=0.1), dict(generator=torch.Generator())):
        with pytest.raises(ValueError, match="not both"):
            d.generate(ids, max_new_tokens=2, choose=lambda x: x.argmax(-1), **kw)
    with pytest.raises(ValueError, match="generator is for"):
        d.generate(ids, max_new_tokens=2, generator=torch.Generator())
