"""Page bookkeeping of the decoder's cache and what the decoder refuses, without a GPU."""
import pytest
import torch

from frankentorch_b200.autograd.tape import TensorTape
from frankentorch_b200.models.gpt import GPT, GPTConfig
from frankentorch_b200.models.gpt_decode import CacheFull, GPTDecoder, PagedKVCache


def _cache(**kw):
    return PagedKVCache(2, 3, 64, **{**dict(pages=6, batch=3, max_tokens=40, page=8, device="cpu"), **kw})


def test_pages_are_given_and_taken_back():
    c = _cache()
    assert c.k.shape == (2, 6, 3, 8, 64) and c.v.shape == c.k.shape and c.table.shape == (3, 5)
    c.reserve(0, 1)
    c.reserve(1, 17)
    first = c.table.clone()
    c.reserve(0, 8)                                   # still one page
    assert torch.equal(c.table, first) and c.free_pages == 2
    c.reserve(0, 9)
    held = c.table[0, :2].tolist() + c.table[1, :3].tolist()
    assert len(set(held)) == 5 and all(0 <= p < 6 for p in held)
    assert c.table[0, 0] == first[0, 0]               # what a sequence has stays where it is
    with pytest.raises(CacheFull, match="2 pages, 1 are free"):
        c.reserve(2, 16)
    assert c.free_pages == 1
    c.release(1)
    assert c.free_pages == 4
    c.reserve(2, 32)
    now = c.table[0, :2].tolist() + c.table[2, :4].tolist()
    assert len(set(now)) == 6 and c.free_pages == 0
    c.release(1)                                      # nothing held: nothing given back twice
    assert c.free_pages == 0


@pytest.mark.parametrize("kw", [dict(page=12), dict(page=0), dict(pages=0), dict(batch=0), dict(max_tokens=0)])
def test_cache_refuses(kw):
    with pytest.raises(ValueError):
        _cache(**kw)
    with pytest.raises(ValueError, match="41 tokens"):
        _cache().reserve(0, 41)


def _model(**kw):
    cfg = GPTConfig(**{**dict(n_layer=1, d_model=128, n_head=2, d_ff=256, vocab_size=100, max_seq=32, name="t"), **kw})
    return GPT(cfg, TensorTape(grad_dtype=None), device="cpu")


def test_decoder_refuses():
    with pytest.raises(ValueError, match="learned positions"):
        GPTDecoder(_model(), 2, 33)
    with pytest.raises(ValueError, match="head size"):
        GPTDecoder(_model(n_head=4), 2, 16)
    d = GPTDecoder(_model(), 2, 32, page=16)
    with pytest.raises(ValueError, match="follows a prefill"):
        d.step(torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="one token for each"):
        d.step(torch.zeros(3, dtype=torch.int64))
    with pytest.raises(ValueError, match="for 2 sequences"):
        d.prefill(torch.zeros(3, 4, dtype=torch.int64))
    with pytest.raises(ValueError, match="1 to 4 tokens"):
        d.prefill(torch.zeros(2, 4, dtype=torch.int64), [4, 0])
    with pytest.raises(ValueError, match="positive"):
        d.generate(torch.zeros(2, 4, dtype=torch.int64), max_new_tokens=0)


def test_rotary_model_has_no_position_table():
    learned, rotary = _model(), _model(pos="rotary")
    assert "wpe.weight" in learned.leaf and learned.inv_freq is None and learned.last_embedding == "wpe.weight"
    assert "wpe.weight" not in rotary.leaf and "wpe.weight" not in rotary.state_dict()
    assert rotary.inv_freq.shape == (32,) and rotary.inv_freq.dtype == torch.float64
    assert learned.cfg.param_count() - rotary.cfg.param_count() == 32 * 128
    assert GPTDecoder(rotary, 1, 1000).cache.table.shape == (1, 16)
    with pytest.raises(ValueError, match="'learned' or 'rotary'"):
        _model(pos="none")
    with pytest.raises(ValueError, match="learned positions only"):
        rotary.cfg.require_learned_positions("another model")


class _Seen(Exception):
    pass


@pytest.mark.parametrize("padding", [-1, -100, 100, 2 ** 40])
def test_prompts_are_embedded_without_their_padding(monkeypatch, padding):
    """What stands behind a prompt's tokens need not be a token: the model sees 0 there, the caller's tensor stays."""
    from frankentorch_b200.models import gpt_decode

    def embedding(ids, *a):
        raise _Seen(ids.clone())
    monkeypatch.setattr(gpt_decode.K, "embedding_fwd", embedding)
    ids = torch.tensor([[5, 6, 7, 8], [9, padding, padding, padding], [1, 2, padding, padding]])
    held = ids.clone()
    d = GPTDecoder(_model(), 3, 32, page=16)
    with pytest.raises(_Seen) as e:
        d.prefill(ids, [4, 1, 2])
    assert e.value.args[0].tolist() == [[5, 6, 7, 8], [9, 0, 0, 0], [1, 2, 0, 0]] and torch.equal(ids, held)
    with pytest.raises(_Seen) as e:
        d.prefill(ids.clamp(0, 9).to(torch.int32))                     # no lengths: all of them are tokens
    assert e.value.args[0].tolist() == ids.clamp(0, 9).tolist() and e.value.args[0].dtype == torch.int64


def test_prompts_of_any_layout(monkeypatch):
    """The embedding reads ids one after the other: transposed, strided and broadcast prompts arrive in that order."""
    from frankentorch_b200.models import gpt_decode

    def embedding(ids, *a):
        raise _Seen(ids)
    monkeypatch.setattr(gpt_decode.K, "embedding_fwd", embedding)
    d = GPTDecoder(_model(), 3, 32, page=16)
    for ids in (torch.arange(12).view(4, 3).t(), torch.arange(24).view(3, 8)[:, ::2], torch.arange(4).expand(3, 4)):
        for lengths in (None, [4, 1, 2]):
            with pytest.raises(_Seen) as e:
                d.prefill(ids, lengths)
            got = e.value.args[0]
            assert got.is_contiguous() and [r[:1] for r in got.tolist()] == [r[:1] for r in ids.tolist()]


def _stub_decoder(monkeypatch, logits):
    """A decoder whose model gives the same ``logits`` at every step, and the ids that its steps get."""
    from frankentorch_b200.models import gpt_decode
    B, V = logits.shape
    d = GPTDecoder(_model(vocab_size=V), B, 200, page=16, use_cuda_graph=False) if V > 32 else \
        GPTDecoder(_model(vocab_size=V, pos="rotary"), B, 200, page=16, use_cuda_graph=False)
    steps = []

    def prefill(ids, lengths=None):
        n = [ids.shape[1]] * B if lengths is None else list(lengths)
        d._host_lengths = n
        d.lengths.copy_(torch.tensor(n))
        return logits.clone()

    def step(ids):
        steps.append(ids.clone())
        return logits.clone()

    def process(x, *, vocab, bias=None, allowed=None, **kw):
        x = x[:, :vocab].clone() if bias is None else x[:, :vocab] + bias
        if allowed is not None:
            c = torch.arange(vocab)
            x = x.masked_fill(((allowed.expand(B, -1)[:, c // 32] >> (c % 32)) & 1) == 0, float("-inf"))
        return x
    monkeypatch.setattr(d, "prefill", prefill)
    monkeypatch.setattr(d, "step", step)
    monkeypatch.setattr(gpt_decode.D, "logits_process", process)
    monkeypatch.setattr(gpt_decode.K, "check_status", lambda: None)
    return d, steps


def _sampler(seen):
    def choose(x):
        assert bool(x.isfinite().any(-1).all()) and not bool(x.isnan().any()), "a row without a choice"
        seen.append(x.clone())
        return torch.multinomial(torch.softmax(x, -1), 1)[:, 0]
    return choose


def test_rows_without_a_choice_are_not_sampled(monkeypatch):
    """``choose`` gets rows that have something to choose from: a sampler would turn the others into NaN.  What it returns for a
    row that has ended goes nowhere."""
    V, S = 20, 3
    logits = torch.randn(4, V, generator=torch.Generator().manual_seed(0))
    words = torch.full((4, 1), (1 << V) - 1, dtype=torch.int32)
    words[2] = 0                                           # nothing, from the first token on
    seen = []
    d, steps = _stub_decoder(monkeypatch, logits)
    tokens, totals = d.generate(torch.ones(4, S, dtype=torch.int64), max_new_tokens=5, allowed=words, choose=_sampler(seen))
    assert totals.tolist() == [8, 8, 3, 8] and not bool(tokens[2, S:].any())
    assert len(seen) == 5 and torch.equal(seen[0][[0, 1, 3]], logits[[0, 1, 3]])
    assert all(0 <= int(i) < V for s in steps for i in s) and all(int(s[2]) == 0 for s in steps)
    # a bias that leaves nothing
    bias = torch.zeros(4, V)
    bias[1] = float("-inf")
    d, _ = _stub_decoder(monkeypatch, logits)
    tokens, totals = d.generate(torch.ones(4, S, dtype=torch.int64), max_new_tokens=5, bias=bias, choose=_sampler([]))
    assert totals.tolist() == [8, 3, 8, 8]
    # a function that allows nothing from a row's fifth token on: it ended there, and stays so
    def grammar(tok, tot):
        return torch.where(tot[:, None] < torch.tensor([[9], [5], [9], [4]]), (1 << V) - 1, 0).to(torch.int32)
    d, steps = _stub_decoder(monkeypatch, logits)
    tokens, totals = d.generate(torch.ones(4, S, dtype=torch.int64), max_new_tokens=5, allowed=grammar, choose=_sampler([]))
    assert totals.tolist() == [8, 5, 8, 4]
    # a choice for an ended row that is no token: not fed, not kept
    def wild(x):
        return torch.where(x.abs().sum(-1) == 0, 10 ** 9, 7)
    d, steps = _stub_decoder(monkeypatch, logits)
    tokens, totals = d.generate(torch.ones(4, S, dtype=torch.int64), max_new_tokens=5, allowed=words, choose=wild)
    assert all(s.tolist() == [7, 7, 0, 7] for s in steps) and totals.tolist() == [8, 8, 3, 8]
    # behind the end token as well
    d, steps = _stub_decoder(monkeypatch, logits)
    tokens, totals = d.generate(torch.ones(4, S, dtype=torch.int64), max_new_tokens=5, eos=7, choose=lambda x: torch.tensor([7, 3, 7, 3]))
    assert totals.tolist() == [4, 8, 4, 8] and all(s.tolist()[1::2] == [3, 3] and s[0] in (0, 7) for s in steps)


@pytest.mark.parametrize("how", ["bias", "allowed", "eos"])
def test_generation_stops_when_all_rows_have_ended(monkeypatch, how):
    V = 20
    logits = torch.randn(2, V, generator=torch.Generator().manual_seed(1))
    kw = {"bias": dict(bias=torch.full((V,), float("-inf"))), "allowed": dict(allowed=torch.zeros(1, dtype=torch.int32)),
          "eos": dict(eos=int(logits[0].argmax()), bias=torch.zeros(V).index_fill(0, logits[0].argmax(), 99.0))}[how]
    d, steps = _stub_decoder(monkeypatch, logits)
    _, totals = d.generate(torch.ones(2, 3, dtype=torch.int64), max_new_tokens=150, **kw)
    assert totals.tolist() == ([4, 4] if how == "eos" else [3, 3]) and len(steps) < 40


def test_calls_run_on_the_device_of_the_model(monkeypatch):
    """The kernels take the current device's stream: prefill, step and generate make the model's device current, with its index."""
    import contextlib

    from frankentorch_b200.models import gpt_decode
    d = GPTDecoder(_model(), 2, 32, page=16, use_cuda_graph=False)
    assert d.device == torch.device("cpu")
    inside = []

    @contextlib.contextmanager
    def on():
        inside.append(True)
        try:
            yield
        finally:
            inside.pop()

    def body(*a):
        raise _Seen(bool(inside))
    monkeypatch.setattr(d, "_on", on)
    monkeypatch.setattr(gpt_decode.K, "embedding_fwd", body)
    ids = torch.ones(2, 4, dtype=torch.int64)
    for call in (lambda: d.prefill(ids), lambda: d.generate(ids, max_new_tokens=2)):
        with pytest.raises(_Seen) as e:
            call()
        assert e.value.args[0]
    d._host_lengths = [4, 4]
    with pytest.raises(_Seen) as e:
        d.step(ids[:, 0])
    assert e.value.args[0] and not inside
    monkeypatch.undo()
    asked = []
    monkeypatch.setattr(torch.cuda, "device", lambda dev: asked.append(dev) or contextlib.nullcontext())
    d.device = torch.device("cuda", 1)
    with d._on():
        assert asked == [torch.device("cuda", 1)]
