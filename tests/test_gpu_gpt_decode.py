"""Training with rotary positions, and generation over the paged cache, against the same models in 64-bit arithmetic."""
import math

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu


def _build(dev, pos="rotary", seed=3, **kw):
    from frankentorch_b200.autograd.tape import TensorTape
    from frankentorch_b200.models.gpt import GPT, GPTConfig
    from frankentorch_b200.ops import kernels as K
    cfg = GPTConfig(**{**dict(n_layer=2, d_model=128, n_head=2, d_ff=512, max_seq=128, vocab_size=1000, name="t", pos=pos), **kw})
    tape = TensorTape(grad_dtype=None)
    tape.accumulate_fn = lambda a, b: K.add(a, b) if a.dtype == torch.bfloat16 else a + b
    model = GPT(cfg, tape, device=dev, seed=seed)
    # weights far from their small initial values, so that attention and the head tell positions and tokens apart
    g = torch.Generator(device=dev).manual_seed(seed)
    for n, t in model.named_parameters():
        if n.endswith("weight") and ".ln" not in n and not n.startswith("ln"):
            t.copy_(torch.randn(t.shape, generator=g, device=dev) * (0.5 if n.startswith("w") else 1.5 / math.sqrt(t.shape[-1])))
    model.arena.sync_shadow()
    return cfg, tape, model


def _turn(x, base):
    """[B, H, S, hd] by position."""
    S, hd = x.shape[2:]
    a = torch.arange(S, dtype=torch.float64, device=x.device)[:, None] * base ** (
        -torch.arange(0, hd, 2, dtype=torch.float64, device=x.device) / hd)
    x0, x1 = x[..., : hd // 2], x[..., hd // 2:]
    return torch.cat([x0 * a.cos() - x1 * a.sin(), x1 * a.cos() + x0 * a.sin()], -1)


def _logits64(cfg, P, ids):
    B, S = ids.shape
    d, H = cfg.d_model, cfg.n_head
    x = P["wte.weight"][ids]
    if cfg.pos == "learned":
        x = x + P["wpe.weight"][:S]
    mask = torch.ones(S, S, dtype=torch.bool, device=ids.device).triu(1)
    for l in range(cfg.n_layer):
        p = f"blocks.{l}."
        h = F.layer_norm(x, (d,), P[p + "ln1.weight"], P[p + "ln1.bias"], cfg.ln_eps)
        qkv = h @ P[p + "attn.qkv_proj.weight"].t() + P[p + "attn.qkv_proj.bias"]
        q, k, v = (t.view(B, S, H, d // H).transpose(1, 2) for t in qkv.split(d, dim=-1))
        if cfg.pos == "rotary":
            q, k = _turn(q, cfg.rope_base), _turn(k, cfg.rope_base)
        s = (q @ k.mT / math.sqrt(d // H)).masked_fill(mask, -math.inf)
        x = x + (torch.softmax(s, -1) @ v).transpose(1, 2).reshape(B, S, d) @ P[p + "attn.out_proj.weight"].t() + \
            P[p + "attn.out_proj.bias"]
        h = F.layer_norm(x, (d,), P[p + "ln2.weight"], P[p + "ln2.bias"], cfg.ln_eps)
        u = F.gelu(h @ P[p + "mlp.fc1.weight"].t() + P[p + "mlp.fc1.bias"], approximate="tanh")
        x = x + u @ P[p + "mlp.fc2.weight"].t() + P[p + "mlp.fc2.bias"]
    h = F.layer_norm(x, (d,), P["ln_f.weight"], P["ln_f.bias"], cfg.ln_eps)
    return h @ P["wte.weight"][: cfg.vocab_size].t()


def _params64(cfg, model, grad=False):
    return {n: (t[: cfg.vocab_size] if n == "wte.weight" else t).to(torch.bfloat16).double().requires_grad_(grad)
            for n, t in model.named_parameters()}


# A block rounds to bf16, half a step of 2^-8 each: embedding, norm, projection, two rotations, probabilities, attention, output
# and residual, norm, pre-activation, activation, output and residual: eleven; two blocks, a last norm and the head.  If all
# added up in one direction: 24 * 2^-8 = 9.4e-2 of the 2-norm; a norm over many values sees them as independent, a root of
# 24 times 2^-8 / sqrt(3): 1.1e-2, doubled for what later layers amplify.
FORWARD = 2.3e-2
# Backward once more as many, on top of the forward's
GRADIENT = 6e-2


def test_training_gradients_with_rotary_positions(cuda_device):
    from frankentorch_b200.ops import kernels as K
    cfg, tape, model = _build(cuda_device)
    g = torch.Generator().manual_seed(0)
    tok = torch.randint(0, cfg.vocab_size, (2, 129), generator=g).to(cuda_device)
    ids, tgt = tok[:, :-1].contiguous(), tok[:, 1:].contiguous()
    loss_id = model.forward(ids, tgt)
    report = tape.backward(loss_id)
    K.check_status()
    assert any("rotary" in s.rule for s in report.steps)
    P = _params64(cfg, model, True)
    loss = F.cross_entropy(_logits64(cfg, P, ids).view(-1, cfg.vocab_size), tgt.view(-1))
    loss.backward()
    assert abs(float(tape.value(loss_id).detach()) - float(loss.detach())) <= FORWARD * float(loss.detach())
    for name, _ in model.arena.specs:
        got = model.arena.view(model.arena.grads, name).double()
        got = got[: cfg.vocab_size] if name == "wte.weight" else got
        want = P[name].grad
        part = slice(None)
        if name.endswith("qkv_proj.bias"):
            # a key bias has no gradient but through the rotation: differences of positions leave it small next to the others
            part = torch.cat([torch.arange(cfg.d_model), torch.arange(2 * cfg.d_model, 3 * cfg.d_model)]).to(cuda_device)
        err = float((got[part] - want[part]).norm() / want[part].norm())
        assert err < GRADIENT, (name, err)


def test_attention_gradient_against_differences(cuda_device):
    """Directional derivative of the turned attention, the forward's arithmetic in 64 bits against the kernels' gradient."""
    from frankentorch_b200.autograd.tape import TensorTape
    from frankentorch_b200.ops import decode as D
    from frankentorch_b200.ops import fused as Fu
    B, S, H, hd = 2, 50, 3, 64
    g = torch.Generator(device=cuda_device).manual_seed(2)
    x = torch.randn(B, S, 3 * H * hd, generator=g, device=cuda_device).to(torch.bfloat16)
    gy = torch.randn(B, S, H * hd, generator=g, device=cuda_device).to(torch.bfloat16)
    direction = torch.randn(x.shape, generator=g, device=cuda_device, dtype=torch.float64)
    tape = TensorTape(grad_dtype=None)
    nid = tape.leaf(x.clone(), requires_grad=True)
    out = Fu.attention_packed(tape, nid, H, inv_freq=D.rotary_frequencies(hd))
    assert torch.equal(tape.value(nid), x)
    report = tape.backward(out, seed=gy)
    grad = report.gradients[nid].double()

    def value(t):
        q, k, v = t.view(B, S, 3, H, hd).permute(2, 0, 3, 1, 4)
        s = (_turn(q, 10000.0) @ _turn(k, 10000.0).mT / math.sqrt(hd)).masked_fill(
            torch.ones(S, S, dtype=torch.bool, device=t.device).triu(1), -math.inf)
        return ((torch.softmax(s, -1) @ v).transpose(1, 2).reshape(B, S, H * hd) * gy.double()).sum()
    h = 1e-5                        # the difference's own error is h^2 of third derivatives and 2^-52 / h of the value
    diff = float((value(x.double() + h * direction) - value(x.double() - h * direction)) / (2 * h))
    # probabilities, their gradients, rotations and results are rounded to bf16: as in the attention tests, 1 % of the 2-norm,
    # which a random direction sees through its own norm over the root of the number of elements: four of those
    assert abs(float((grad * direction).sum()) - diff) <= 4 * 1e-2 * float(grad.norm())


def test_rotary_step_in_a_graph_beside_an_eager_one(cuda_device):
    """The engine's captured step and the same step run eagerly give the same weights."""
    from frankentorch_b200.ops import kernels as K
    from frankentorch_b200.training.engine import OptimConfig, TrainEngine
    g = torch.Generator().manual_seed(1)
    tok = torch.randint(0, 1000, (3, 2, 129), generator=g)
    weights = []
    for graph in (True, False):
        cfg, tape, model = _build(cuda_device, seed=5)
        eng = TrainEngine(model, 2, 128, OptimConfig(lr=1e-3), use_cuda_graph=graph)
        for t in tok:
            eng.step(t[:, :-1].contiguous().pin_memory(), t[:, 1:].contiguous().pin_memory())
        K.check_status()
        weights.append(model.arena.master.clone())
    assert torch.equal(*weights)


@pytest.mark.parametrize("graph", [True, False])
@pytest.mark.parametrize("pos,heads,page,lengths", [("learned", 2, 16, [1, 17, 40]), ("rotary", 2, 8, [1, 17, 40]),
                                                    ("rotary", 1, 64, [40, 39, 2]), ("rotary", 2, 32, [40]), ("learned", 1, 4, [1])])
def test_steps_give_the_logits_of_the_whole_sequence(cuda_device, pos, heads, page, lengths, graph):
    """Ragged prompts, then tokens one by one: at every length the logits of the model over all tokens so far."""
    from frankentorch_b200.models.gpt_decode import GPTDecoder
    from frankentorch_b200.ops import kernels as K
    cfg, _, model = _build(cuda_device, pos, n_head=heads)
    P = _params64(cfg, model)
    g = torch.Generator().manual_seed(4)
    new, B = 12, len(lengths)
    tok = torch.randint(0, cfg.vocab_size, (B, 60), generator=g).to(cuda_device)
    dec = GPTDecoder(model, B, 64, page=page, use_cuda_graph=graph)
    for again in range(2):                       # a second batch of prompts takes the pages of the first
        got = [dec.prefill(tok[:, :40], lengths)]
        for i in range(new):
            got.append(dec.step(torch.stack([tok[b, n + i] for b, n in enumerate(lengths)])).clone())
        K.check_status()
        for b, n in enumerate(lengths):
            want = _logits64(cfg, P, tok[b: b + 1, : n + new])[0, n - 1: n + new]
            have = torch.stack([x[b, : cfg.vocab_size] for x in got]).double()
            err = float((have - want).norm() / want.norm())
            assert err < FORWARD, (b, err)
        tok = tok.flip(1)


def test_generation(cuda_device):
    """Greedy choices are the highest logits of a teacher-forced pass; penalties, masks and an end token do what they say; the
    same call gives the same tokens."""
    from frankentorch_b200.models.gpt_decode import GPTDecoder
    cfg, _, model = _build(cuda_device, "rotary", vocab_size=333)
    P = _params64(cfg, model)
    g = torch.Generator().manual_seed(6)
    ids = torch.randint(0, 333, (4, 20), generator=g).to(cuda_device)
    lengths = [20, 3, 11, 1]
    dec = GPTDecoder(model, 4, 80, page=16)
    tokens, totals = dec.generate(ids, lengths, max_new_tokens=30)
    assert totals.tolist() == [n + 30 for n in lengths] and tokens.shape == (4, 50)
    for b, n in enumerate(lengths):
        assert torch.equal(tokens[b, :n], ids[b, :n]) and not bool(tokens[b, n + 30:].any())
        want = _logits64(cfg, P, tokens[b: b + 1, : n + 30])[0, n - 1: n + 29]
        chosen = want.gather(1, tokens[b, n: n + 30, None])[:, 0]
        # a choice may differ from the highest by what the logits may be off: on both sides, relative to the row
        slack = 2 * FORWARD * want.norm(dim=1) / math.sqrt(want.shape[1]) * 4
        assert bool((want.max(1).values - chosen <= slack).all())
    again, _ = dec.generate(ids, lengths, max_new_tokens=30)
    assert torch.equal(again, tokens)
    # only odd ids are allowed, none of them twice (the penalty outweighs every logit), from the first new token on
    words = torch.full((11,), -0x55555556, dtype=torch.int32, device=cuda_device)       # bits 1, 3, 5, ...
    odd, totals = dec.generate(ids, lengths, max_new_tokens=40, frequency=1e6, allowed=words)
    for b, n in enumerate(lengths):
        new = odd[b, n: n + 40].tolist()
        assert all(t % 2 == 1 and t < 333 for t in new) and len(set(new)) == 40
    # an end token: nothing behind it
    eos = int(tokens[0, 25])
    ended, totals = dec.generate(ids, lengths, max_new_tokens=30, eos=eos)
    stop = tokens[0, 20:50].tolist().index(eos) + 20
    assert int(totals[0]) == stop + 1 and torch.equal(ended[0, : stop + 1], tokens[0, : stop + 1])
    assert not bool(ended[0, stop + 1:].any())
    # a function of what is there so far: every row repeats its first token
    def first_only(tok, tot):
        w = torch.zeros(4, 11, dtype=torch.int64, device=tok.device)
        one = tok[:, :1]
        w.scatter_(1, one // 32, torch.ones_like(one) << (one % 32))
        return torch.where(w >= 2 ** 31, w - 2 ** 32, w).to(torch.int32)
    # a mask that leaves a row nothing ends it
    none = words.expand(4, -1).clone()
    none[2] = 0
    stuck, totals = dec.generate(ids, lengths, max_new_tokens=6, allowed=none)
    assert totals.tolist() == [26, 9, 11, 7] and not bool(stuck[2, 11:].any()) and bool((stuck[0, 20:26] % 2 == 1).all())
    same, _ = dec.generate(ids, lengths, max_new_tokens=5, allowed=first_only, bias=torch.zeros(333, device=cuda_device))
    for b, n in enumerate(lengths):
        assert bool((same[b, n: n + 5] == ids[b, 0]).all())


def test_a_cache_that_is_too_small(cuda_device):
    """Pages run out: the call is refused, a smaller one works, and what a refused prefill left is not stepped on."""
    from frankentorch_b200.models.gpt_decode import CacheFull, GPTDecoder
    cfg, _, model = _build(cuda_device)
    ids = torch.zeros(2, 40, dtype=torch.int64, device=cuda_device)
    dec = GPTDecoder(model, 2, 64, page=8, pages=6)
    with pytest.raises(CacheFull):
        dec.prefill(ids)
    with pytest.raises(ValueError, match="follows a prefill"):
        dec.step(ids[:, 0])
    dec.prefill(ids, [16, 20])                   # two and three pages of six
    for _ in range(4):                           # three each, up to 20 and 24 tokens
        dec.step(ids[:, 0])
    with pytest.raises(CacheFull):
        dec.step(ids[:, 0])
    with pytest.raises(ValueError, match="made for 64"):
        dec.generate(ids[:, :8], max_new_tokens=60)
    tokens, totals = dec.generate(ids[:, :8], max_new_tokens=10)
    assert totals.tolist() == [18, 18]


def test_two_decoders_of_one_model(cuda_device):
    """Steps of two decoders taken in turns: their graphs and caches do not meet."""
    from frankentorch_b200.models.gpt_decode import GPTDecoder
    cfg, _, model = _build(cuda_device)
    g = torch.Generator().manual_seed(9)
    tok = torch.randint(0, cfg.vocab_size, (5, 60), generator=g).to(cuda_device)
    alone = []
    for rows in (slice(0, 2), slice(2, 5)):
        dec = GPTDecoder(model, rows.stop - rows.start, 64, page=8)
        seq = [dec.prefill(tok[rows, :30])] + [dec.step(tok[rows, 30 + i]).clone() for i in range(20)]
        alone.append(seq)
    pair = [(GPTDecoder(model, r.stop - r.start, 64, page=8), r) for r in (slice(0, 2), slice(2, 5))]
    both = [[d.prefill(tok[r, :30])] for d, r in pair]
    for i in range(20):
        for (d, r), seq in zip(pair, both):
            seq.append(d.step(tok[r, 30 + i]).clone())
    for a, b in zip(alone, both):
        for x, y in zip(a, b):
            assert torch.equal(x, y)


@pytest.mark.parametrize("pos", ["learned", "rotary"])
@pytest.mark.parametrize("padding", [-1, -100, 10 ** 12])
def test_padding_that_is_no_token(cuda_device, pos, padding):
    """Ragged prompts padded with what is in no vocabulary: the tokens of the same prompts padded with 0, and nothing reported."""
    from frankentorch_b200.models.gpt_decode import GPTDecoder
    from frankentorch_b200.ops import kernels as K
    cfg, _, model = _build(cuda_device, pos)
    g = torch.Generator().manual_seed(11)
    lengths = [9, 1, 4]
    ids = torch.randint(0, cfg.vocab_size, (3, 9), generator=g).to(cuda_device)
    behind = torch.arange(9, device=cuda_device)[None, :] >= torch.tensor(lengths, device=cuda_device)[:, None]
    dec = GPTDecoder(model, 3, 40, page=8)
    want = dec.generate(ids.masked_fill(behind, 0), lengths, max_new_tokens=12, repetition=1.2)
    got = dec.generate(ids.masked_fill(behind, padding), lengths, max_new_tokens=12, repetition=1.2)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    first = dec.prefill(ids.masked_fill(behind, padding), lengths)
    K.check_status()
    assert torch.equal(first, dec.prefill(ids.masked_fill(behind, 0), lengths))


def test_sampling_beside_rows_without_a_choice(cuda_device):
    """A sampler under masks and biases that end some rows early: it gets finite rows only, and the others go on."""
    from frankentorch_b200.models.gpt_decode import GPTDecoder
    cfg, _, model = _build(cuda_device, "rotary", vocab_size=333)
    g = torch.Generator().manual_seed(12)
    ids = torch.randint(0, 333, (4, 6), generator=g).to(cuda_device)
    dec = GPTDecoder(model, 4, 40, page=16)
    draws = torch.Generator(device=cuda_device).manual_seed(0)
    finite = []

    def sample(x):
        finite.append(x.isfinite().any(-1).all() & ~x.isnan().any())
        p = torch.softmax(torch.where(finite[-1], x, torch.zeros_like(x)), -1)       # never NaN in multinomial
        return torch.multinomial(p, 1, generator=draws)[:, 0]
    words = torch.full((4, 11), -0x55555556, dtype=torch.int32, device=cuda_device)
    words[1] = 0
    tokens, totals = dec.generate(ids, [6, 2, 3, 1], max_new_tokens=8, allowed=words, choose=sample)
    assert totals.tolist() == [14, 2, 11, 9] and bool(torch.stack(finite).all())
    assert bool((tokens[0, 6:14] % 2 == 1).all()) and not bool(tokens[1, 2:].any())

    def until(tok, tot):                       # nothing from a length on
        return torch.where(tot[:, None] < torch.tensor([[99], [5], [99], [4]], device=cuda_device), words[:1], 0)
    tokens, totals = dec.generate(ids, [6, 2, 3, 1], max_new_tokens=8, allowed=until, choose=sample, repetition=1.1)
    assert totals.tolist() == [14, 5, 11, 4] and bool(torch.stack(finite).all())
    bias = torch.zeros(4, 333, device=cuda_device)
    bias[3] = -math.inf
    tokens, totals = dec.generate(ids, [6, 2, 3, 1], max_new_tokens=8, bias=bias, choose=sample)
    assert totals.tolist() == [14, 10, 11, 1] and bool(torch.stack(finite).all())
