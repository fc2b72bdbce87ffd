"""Generation with a trained :class:`~frankentorch_b200.models.gpt.GPT`: a paged key-value cache, a prefill pass and a
one-token step.

The reference trains and evaluates its models and has no decoder loop; its nearest parts are the attention and the
embedding of ft-nn.  Here the weights are the model's own bf16 arena.  A prompt runs through the kernels of the training
forward and leaves its keys and values in the cache; a step is, per layer, LayerNorm, the packed projection, the append
(with the rotation of a rotary model), the attention over the cache, and the output and MLP products with their
epilogues.  The step is captured in one CUDA graph: lengths, pages and tokens are device data, so it is replayed as the
sequences grow.
"""
from __future__ import annotations

import contextlib
import functools
from typing import Callable, List, Optional, Sequence, Tuple, Union

import torch

from ..ops import decode as D
from ..ops import kernels as K
from .gpt import GPT

_EPI = {"gelu_tanh": K.EPI_GELU_TANH, "gelu_erf": K.EPI_GELU_ERF, "relu": K.EPI_RELU}


def _on_its_device(method):
    """The kernels of :mod:`..ops.kernels` run on the current device: here that is the model's, whichever the caller's is."""
    @functools.wraps(method)
    def call(self, *args, **kw):
        with self._on():
            return method(self, *args, **kw)
    return call


class CacheFull(RuntimeError):
    """The cache has fewer free pages than a sequence needs."""


class PagedKVCache:
    """Pages of all layers, ``[layers, pages, heads, page, hd]`` for keys and for values, and the page table of ``batch``
    sequences.  A page number means the same page in every layer."""

    def __init__(self, layers: int, heads: int, hd: int, *, pages: int, batch: int, max_tokens: int, page: int = 64,
                 device="cuda", dtype: torch.dtype = torch.bfloat16):
        if page < 1 or page & (page - 1):
            raise ValueError(f"a page holds a power of two of tokens, not {page}")
        if pages < 1 or batch < 1 or max_tokens < 1:
            raise ValueError("pages, batch and max_tokens are positive")
        self.page, self.max_tokens = page, max_tokens
        self.k = torch.zeros((layers, pages, heads, page, hd), dtype=dtype, device=device)
        self.v = torch.zeros_like(self.k)
        self.table = torch.zeros((batch, -(-max_tokens // page)), dtype=torch.int32, device=device)
        self._free: List[int] = list(range(pages - 1, -1, -1))
        self._held: List[List[int]] = [[] for _ in range(batch)]

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def reserve(self, sequence: int, tokens: int) -> None:
        """Give ``sequence`` the pages for its first ``tokens`` positions; it keeps those that it has."""
        if tokens > self.max_tokens:
            raise ValueError(f"{tokens} tokens, the cache was made for {self.max_tokens} per sequence")
        held = self._held[sequence]
        more = -(-tokens // self.page) - len(held)
        if more <= 0:
            return
        if more > len(self._free):
            raise CacheFull(f"sequence {sequence} needs {more} pages, {len(self._free)} are free")
        new = [self._free.pop() for _ in range(more)]
        self.table[sequence, len(held): len(held) + more] = torch.tensor(new, dtype=torch.int32)
        held += new

    def release(self, sequence: int) -> None:
        """Take back all pages of ``sequence``."""
        self._free += reversed(self._held[sequence])
        self._held[sequence] = []


class GPTDecoder:
    """Decoding state of ``batch`` sequences over ``model``; ``pages`` (default: enough for all) bounds the cache."""

    def __init__(self, model: GPT, batch: int, max_tokens: int, *, page: int = 64, pages: Optional[int] = None,
                 use_cuda_graph: bool = True):
        cfg = model.cfg
        if cfg.pos == "learned" and max_tokens > cfg.max_seq:
            raise ValueError(f"{max_tokens} tokens, the model has {cfg.max_seq} learned positions")
        self.model, self.cfg, self.device = model, cfg, model.arena.params.device
        self.batch = batch
        self.hd = cfg.d_model // cfg.n_head
        if self.hd not in D.HEAD_SIZES:
            raise ValueError(f"head size must be one of {D.HEAD_SIZES}, not {self.hd}")
        if pages is None:
            pages = batch * -(-max_tokens // page)
        self.cache = PagedKVCache(cfg.n_layer, cfg.n_head, self.hd, pages=pages, batch=batch, max_tokens=max_tokens,
                                  page=page, device=self.device)
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=self.device)      # tokens in the cache
        self.ids = torch.zeros(batch, dtype=torch.int64, device=self.device)
        self._host_lengths = [0] * batch
        self.use_graph = use_cuda_graph
        self._graph: Optional[torch.cuda.CUDAGraph] = None
        self._logits: Optional[torch.Tensor] = None

    def _on(self):
        return torch.cuda.device(self.device) if self.device.type == "cuda" else contextlib.nullcontext()

    def _w(self, name: str) -> torch.Tensor:
        return self.model.arena.view(self.model.arena.params, name)

    def _layer(self, l: int, x: torch.Tensor, attend: Callable) -> torch.Tensor:
        """One block on ``[rows, d]``; ``attend`` takes the packed projections ``[rows, 3 d]`` to ``[rows, d]``."""
        w, p, cfg = self._w, f"blocks.{l}.", self.cfg
        h = K.layernorm_fwd(x, w(p + "ln1.weight"), w(p + "ln1.bias"), cfg.ln_eps)[0]
        a = attend(K.linear_fwd(h, w(p + "attn.qkv_proj.weight"), w(p + "attn.qkv_proj.bias")))
        x = K.linear_fwd(a, w(p + "attn.out_proj.weight"), w(p + "attn.out_proj.bias"), resid=x)
        h = K.layernorm_fwd(x, w(p + "ln2.weight"), w(p + "ln2.bias"), cfg.ln_eps)[0]
        u = K.linear_fwd(h, w(p + "mlp.fc1.weight"), w(p + "mlp.fc1.bias"), epi=_EPI[cfg.act])
        return K.linear_fwd(u, w(p + "mlp.fc2.weight"), w(p + "mlp.fc2.bias"), resid=x)

    def _head(self, x: torch.Tensor) -> torch.Tensor:
        h = K.layernorm_fwd(x, self._w("ln_f.weight"), self._w("ln_f.bias"), self.cfg.ln_eps)[0]
        return K.gemm(h, self._w("wte.weight" if self.cfg.tie_lm_head else "lm_head.weight"), out_dtype=torch.float32)

    # ------------------------------------------------------------------ prompts
    @_on_its_device
    def prefill(self, ids: torch.Tensor, lengths: Optional[Sequence[int]] = None) -> torch.Tensor:
        """Take the prompts ``ids`` (int64 ``[batch, S]``, the first ``lengths[b]`` of row ``b``; what stands behind them need not be a
        token) into an empty cache; returns the logits behind each prompt's last token, fp32 ``[batch, padded vocabulary]``."""
        cfg, cache = self.cfg, self.cache
        B, S = ids.shape
        lengths = [S] * B if lengths is None else [int(n) for n in lengths]
        if B != self.batch or len(lengths) != B:
            raise ValueError(f"{B} prompts with {len(lengths)} lengths for {self.batch} sequences")
        if not all(1 <= n <= S for n in lengths):
            raise ValueError(f"prompts have 1 to {S} tokens, not {lengths}")
        if S > cfg.max_seq and cfg.pos == "learned":
            raise ValueError(f"{S} tokens, the model has {cfg.max_seq} learned positions")
        self._host_lengths = [0] * B            # until the prompts are in
        for b in range(B):
            cache.release(b)
        for b, n in enumerate(lengths):
            cache.reserve(b, n)
        counts = torch.tensor(lengths, dtype=torch.int32, device=self.device)
        ids = ids.to(self.device, torch.int64)
        ids = torch.where(torch.arange(S, device=self.device)[None, :] < counts[:, None], ids, 0).contiguous()
        start = torch.zeros_like(counts)
        H, hd, d = cfg.n_head, self.hd, cfg.d_model
        x = K.embedding_fwd(ids, self._w("wte.weight"), self._w("wpe.weight") if cfg.pos == "learned" else None, S)
        for l in range(cfg.n_layer):
            def attend(qkv, l=l):
                q, k, v = qkv.view(B, S, 3, H, hd).unbind(2)
                if self.model.inv_freq is not None:
                    q, k = D.rotary(q, k, self.model.inv_freq)
                D.paged_append(cache.k[l], cache.v[l], cache.table, k, v, start, counts)
                return K.attention_fwd(q, k, v, causal=True)[0].view(B * S, d)
            x = self._layer(l, x, attend)
        last = torch.arange(0, B * S, S, device=self.device) + counts - 1
        self.lengths.copy_(counts)
        self._host_lengths = lengths
        return self._head(K.embedding_fwd(last, x, None, 1))

    # ------------------------------------------------------------------ one token
    def _step_body(self) -> torch.Tensor:
        cfg, cache, B = self.cfg, self.cache, self.batch
        H, hd, d = cfg.n_head, self.hd, cfg.d_model
        x = K.embedding_fwd(self.ids, self._w("wte.weight"), None, 1)
        if cfg.pos == "learned":
            x = K.add(x, K.embedding_fwd(self.lengths.to(torch.int64), self._w("wpe.weight"), None, 1))
        reach = self.lengths + 1
        for l in range(cfg.n_layer):
            def attend(qkv, l=l):
                q, k, v = qkv.view(B, 1, 3, H, hd).unbind(2)
                if self.model.inv_freq is None:
                    D.paged_append(cache.k[l], cache.v[l], cache.table, k, v, self.lengths)
                else:
                    q = D.paged_append(cache.k[l], cache.v[l], cache.table, k, v, self.lengths, q=q,
                                       inv_freq=self.model.inv_freq)
                return D.paged_attention(q[:, 0], cache.k[l], cache.v[l], cache.table, reach)[0].view(B, d)
            x = self._layer(l, x, attend)
        out = self._head(x)
        self.lengths.copy_(reach)
        return out

    @_on_its_device
    def step(self, ids: torch.Tensor) -> torch.Tensor:
        """Append one token per sequence (int64 ``[batch]``); returns the logits behind it, fp32 ``[batch, padded vocabulary]``.
        With a CUDA graph the logits are one buffer, which the next step writes again."""
        if ids.shape != (self.batch,):
            raise ValueError(f"one token for each of {self.batch} sequences, got shape {tuple(ids.shape)}")
        if 0 in self._host_lengths:
            raise ValueError("a step follows a prefill")
        for b, n in enumerate(self._host_lengths):
            self.cache.reserve(b, n + 1)
        self.ids.copy_(ids)
        if not self.use_graph:
            out = self._step_body()
        else:
            if self._graph is None:
                self._capture()
            self._graph.replay()
            out = self._logits
        self._host_lengths = [n + 1 for n in self._host_lengths]
        return out

    def _capture(self) -> None:
        held = self.lengths.clone()
        side = torch.cuda.Stream(self.device)
        side.wait_stream(torch.cuda.current_stream(self.device))
        with torch.cuda.stream(side):           # warm-up outside of the capture: what it appends, the replay appends again
            self._step_body()
        torch.cuda.current_stream(self.device).wait_stream(side)
        self.lengths.copy_(held)
        torch.cuda.synchronize(self.device)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):      # (the default capture stream is of the device that captured first)
            self._logits = self._step_body()
        self._graph = graph

    # ------------------------------------------------------------------ generation
    @_on_its_device
    def generate(self, ids: torch.Tensor, lengths: Optional[Sequence[int]] = None, *, max_new_tokens: int,
                 eos: Optional[int] = None, repetition=None, frequency=None, presence=None,
                 bias: Optional[torch.Tensor] = None,
                 allowed: Union[torch.Tensor, Callable[[torch.Tensor, torch.Tensor], torch.Tensor], None] = None,
                 choose: Optional[Callable[[torch.Tensor], torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """Continue the prompts by up to ``max_new_tokens`` tokens; returns ``(tokens [batch, S + max_new_tokens], totals [batch])``.

        Row ``b`` holds its prompt and what was generated behind it, ``totals[b]`` tokens; the rest of the row is 0.  The penalties,
        ``bias`` and ``allowed`` are those of :func:`~frankentorch_b200.ops.decode.logits_process`; ``allowed`` may be a function of the
        tokens and totals so far.  ``choose`` takes the processed logits ``[batch, vocabulary]`` to the next ids (default: the
        highest).  A row ends behind ``eos``, and where mask and bias leave it no token; with a mask or a bias ``choose`` gets
        zeros for the rows that have ended, and what it returns for them is not used."""
        if max_new_tokens < 1:
            raise ValueError("max_new_tokens is positive")
        B, S = ids.shape
        logits = self.prefill(ids, lengths)
        for b, n in enumerate(self._host_lengths):
            self.cache.reserve(b, n + max_new_tokens - 1)        # now rather than in the middle
        prompt = self.lengths.clone()
        totals = prompt.clone()
        at = torch.arange(S, device=self.device)
        tokens = torch.zeros((B, S + max_new_tokens), dtype=torch.int64, device=self.device)
        tokens[:, :S] = torch.where(at[None, :] < prompt[:, None], ids.to(self.device), 0)
        live = torch.ones(B, dtype=torch.bool, device=self.device)
        penalised = not (repetition is None and frequency is None and presence is None)
        for i in range(max_new_tokens):
            words = allowed(tokens, totals) if callable(allowed) else allowed
            x = D.logits_process(logits, vocab=self.cfg.vocab_size, tokens=tokens if penalised else None,
                                 lengths=totals if penalised else None, prompt_lengths=prompt if penalised else None,
                                 repetition=repetition, frequency=frequency, presence=presence, bias=bias, allowed=words)
            if words is not None or bias is not None:
                live &= x.amax(-1) != float("-inf")
                if choose is not None:          # a sampler would make NaN of a row of -inf
                    x = torch.where(live[:, None], x, 0.0)
            new = torch.where(live, x.argmax(-1) if choose is None else choose(x), 0)
            place = totals.to(torch.int64)[:, None]
            tokens.scatter_(1, place, torch.where(live[:, None], new[:, None], tokens.gather(1, place)))
            totals += live
            if eos is not None:
                live &= new != eos
            if i % 32 == 31 and (eos is not None or words is not None or bias is not None) and not bool(live.any()):
                break
            if i + 1 < max_new_tokens:
                logits = self.step(new)
        K.check_status()
        return tokens, totals
