"""Generation over a cache in 8 bits, and with drawn tokens."""
import math

import pytest
import torch

from test_gpu_gpt_decode import _build, _logits64, _params64

pytestmark = pytest.mark.gpu
E4 = torch.float8_e4m3fn

# Elements of keys and values are off by up to 2^-4 of themselves, 2^-4 / sqrt(3) in the 2-norm: 3.6 %.  That is what values do to an
# attention of few tokens; a score, a sum of 64 or 128 products, is off by 3.6 % of the root of the sum of their squares, which for scores
# that spread by 2 changes probabilities by 7 %.  Two layers, in squares: sqrt(2 (7^2 + 3.6^2)) = 11 %, doubled for what later layers amplify.
EIGHT_BITS = 0.22


@pytest.mark.parametrize("graph", [True, False])
@pytest.mark.parametrize("pos,heads,page,block,lengths", [("learned", 2, 16, None, [1, 17, 40]), ("rotary", 2, 8, 2, [1, 17, 40]),
                                                          ("rotary", 1, 64, 16, [40, 39, 2]), ("rotary", 2, 32, 32, [40]), ("learned", 1, 4, 1, [1])])
def test_steps_give_about_the_logits_of_the_whole_sequence(cuda_device, pos, heads, page, block, lengths, graph):
    from frankentorch_b200.models.gpt_decode import GPTDecoder
    from frankentorch_b200.ops import kernels as K
    cfg, _, model = _build(cuda_device, pos, n_head=heads)
    P = _params64(cfg, model)
    g = torch.Generator().manual_seed(4)
    new, B = 12, len(lengths)
    tok = torch.randint(0, cfg.vocab_size, (B, 60), generator=g).to(cuda_device)
    dec = GPTDecoder(model, B, 64, page=page, use_cuda_graph=graph, cache_dtype=E4, cache_block=block)
    for again in range(2):                       # a second batch of prompts takes the pages and scales of the first
        got = [dec.prefill(tok[:, :40], lengths)]
        for i in range(new):
            got.append(dec.step(torch.stack([tok[b, n + i] for b, n in enumerate(lengths)])).clone())
        K.check_status()
        for b, n in enumerate(lengths):
            want = _logits64(cfg, P, tok[b: b + 1, : n + new])[0, n - 1: n + new]
            have = torch.stack([x[b, : cfg.vocab_size] for x in got]).double()
            err = float((have - want).norm() / want.norm())
            assert err < EIGHT_BITS, (b, err)
        tok = tok.flip(1)


def test_captured_and_eager_steps_are_the_same(cuda_device):
    from frankentorch_b200.models.gpt_decode import GPTDecoder
    cfg, _, model = _build(cuda_device)
    tok = torch.randint(0, cfg.vocab_size, (2, 40), generator=torch.Generator().manual_seed(5)).to(cuda_device)
    runs = []
    for graph in (True, False):
        dec = GPTDecoder(model, 2, 64, page=16, use_cuda_graph=graph, cache_dtype=E4)
        runs.append([dec.prefill(tok[:, :13], [13, 6])] + [dec.step(tok[:, 13 + i]).clone() for i in range(20)] +
                    [dec.cache.k.view(torch.uint8).clone(), dec.cache.v_scales.clone()])
    for a, b in zip(*runs):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4])
def test_drawn_tokens(cuda_device, dtype):
    """The settings do what they say, and the same generator's state gives the same tokens."""
    from frankentorch_b200.models.gpt_decode import GPTDecoder
    cfg, _, model = _build(cuda_device, "rotary", vocab_size=333)
    ids = torch.randint(0, 333, (4, 20), generator=torch.Generator().manual_seed(6)).to(cuda_device)
    lengths = [20, 3, 11, 1]
    dec = GPTDecoder(model, 4, 80, page=16, cache_dtype=dtype)

    def run(seed=None, **kw):
        g = None if seed is None else torch.Generator(device=cuda_device).manual_seed(seed)
        return dec.generate(ids, lengths, max_new_tokens=30, generator=g, **kw)
    best, totals = dec.generate(ids, lengths, max_new_tokens=30)
    for kw in (dict(temperature=0.0), dict(top_k=1), dict(top_p=1e-9), dict(min_p=1.0, temperature=0.7)):
        got, t = run(**kw)
        assert torch.equal(got, best) and torch.equal(t, totals), kw
    a, _ = run(1, temperature=1.5, top_k=40, top_p=0.95)
    b, _ = run(1, temperature=1.5, top_k=40, top_p=0.95)
    c, _ = run(2, temperature=1.5, top_k=40, top_p=0.95)
    assert torch.equal(a, b) and not torch.equal(a, c) and not torch.equal(a, best)
    for row, n in enumerate(lengths):
        assert torch.equal(a[row, :n], ids[row, :n]) and int(a.max()) < 333 and int(a.min()) >= 0
    # settings of each row, a mask, a penalty: only odd ids, none of them twice; a row without any ends
    t = torch.tensor([0.5, 1.0, 2.0, 4.0], device=cuda_device)
    words = torch.full((4, 11), -0x55555556, dtype=torch.int32, device=cuda_device)
    words[2] = 0
    odd, totals = run(3, temperature=t, frequency=1e6, allowed=words)
    assert totals.tolist() == [50, 33, 11, 31] and not bool(odd[2, 11:].any())
    for row in (0, 1, 3):
        new = odd[row, lengths[row]: lengths[row] + 30].tolist()
        assert all(x % 2 == 1 and x < 333 for x in new) and len(set(new)) == 30


def test_drawn_tokens_follow_the_distribution(cuda_device):
    """One step of many sequences of the same prompt: as many of each token as its probability says."""
    from frankentorch_b200.models.gpt_decode import GPTDecoder
    cfg, _, model = _build(cuda_device, "rotary", vocab_size=50)
    B = 512
    ids = torch.randint(0, 50, (1, 8), generator=torch.Generator().manual_seed(7)).to(cuda_device).expand(B, -1)
    dec = GPTDecoder(model, B, 16, page=16)
    logits = dec.prefill(ids)[0, :50].double()
    t = float(logits.std())                         # a spread of 1
    p = torch.softmax(logits / t, 0)
    counts = torch.zeros(50, dtype=torch.float64, device=cuda_device)
    for seed in range(4):
        g = torch.Generator(device=cuda_device).manual_seed(seed)
        tokens, _ = dec.generate(ids, max_new_tokens=1, temperature=t, generator=g)
        counts += torch.bincount(tokens[:, 8], minlength=50)
    n = 4 * B
    # a count of n draws: six standard deviations
    assert bool(((counts - n * p).abs() <= 6 * torch.sqrt(n * p * (1 - p)) + 1).all())
