"""Launchers of the operators between a trained decoder and its next token (``torch.Tensor`` in, ``torch.Tensor`` out).

* :func:`rotary`: queries and keys turned by position, forward and backward (training);
* :func:`paged_append`: keys and values of new tokens into a paged cache, turned on the way;
* :func:`paged_attention`: one new token per sequence over the cache;
* :func:`logits_process`: penalties for repeated tokens, biases and a grammar's mask on the logits of a step;
* :func:`sample`: the next token from them and given random numbers (temperature, top-k, top-p, min-p).

The reference composes the rotation from tensor operators (``apply_rotary_pos_emb``) and has no cache, no decoding attention,
no logits processing and no sampling; shapes, masks and empty rows follow its attention (ft-nn/src/lib.rs:5145-5184) where they overlap.

A paged cache is two tensors of pages, ``[pages, heads, page, hd]`` (``page`` a power of two), and a table ``[B, columns]`` of
page numbers (int32): position ``p`` of sequence ``b`` is row ``p % page`` of page ``table[b, p // page]``.  Table entries behind the
last position that a call touches have no meaning for it.  Rows of ``hd`` elements are contiguous and start on 16 bytes; everything else
may be strided.  Lengths, positions and counts are int32 on the device, so a captured graph follows them.

The cache may be held in 8 bits: pages of ``torch.float8_e4m3fn`` with fp32 scales, ``[pages, heads, blocks]`` with unit inner stride,
for keys (``k_scales``) and for values (``v_scales``).  A block is ``page / blocks`` neighbouring rows of a page and head (a power of two,
64 at most), and an element stands for its 8 bits times its block's scale.  :func:`paged_append` makes the scales, powers of two;
:func:`paged_attention` takes those and any other from 2^-100 to 2^120, or 0, in any mixture.  What adds less than 2^-38 of the largest
product of a probability and a value's scale, times 448, to an element of the output does not count.

A call enqueues on the current stream of its tensors' device, also where another device is the current one, and returns.
Arguments that the host can check are refused with :class:`~.kernels.KernelError`; a page, token or length out of range on the
device is reported by that device's :func:`~.kernels.check_status`, and what it leads to is not read and not written.  A call keeps
nothing: its scratch is its own, so calls of several streams, threads and captured graphs do not meet, and the same call gives
the same bits.  (The attention cuts a sequence's heads by the work of the whole call: beside other sequences its last bits may
be others.)  Two tokens of one append must not have the same place (over 8 bits: two sequences no common block), and an output must not
overlap an input other than where the function says so; one whose own rows overlap is refused.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib
from .kernels import KernelError

HEAD_SIZES = (64, 128)          # of paged_attention, as of attention_fwd


def rotary_frequencies(turned: int, base: float = 10000.0, device="cuda") -> torch.Tensor:
    """Angle per position of each pair of the ``turned`` leading elements of a head: ``base ** (-2 i / turned)``, float64."""
    if turned < 16 or turned % 16:
        raise KernelError("the turned elements of a head are a positive multiple of 16")
    return (float(base) ** (-torch.arange(0, turned, 2, dtype=torch.float64) / turned)).to(device)


def rotary(q: torch.Tensor, k: Optional[torch.Tensor], inv_freq: torch.Tensor, *, start: Optional[torch.Tensor] = None,
           interleaved: bool = False, inverse: bool = False, q_out: Optional[torch.Tensor] = None,
           k_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """``(q, k)`` turned by position: pair ``i`` of token ``s`` of sequence ``b`` by ``(start[b] + s) inv_freq[i]``.

    ``q`` is ``[B, S, H, hd]``, ``k`` ``[B, S, Hkv, hd]`` or None; bf16 or fp16, ``hd`` a multiple of 16.  ``inv_freq`` (float64, see
    :func:`rotary_frequencies`) has one entry per pair: pairs are ``(i, i + n)`` with ``n = len(inv_freq)``, or ``(2 i, 2 i + 1)``
    when ``interleaved``; elements from ``2 n`` on are copied.  ``start`` is 0 where it is not given.  ``inverse`` turns back: the
    backward pass of the rotation is its inverse on the gradient.  ``q_out`` / ``k_out`` may be ``q`` / ``k`` themselves."""
    return _lib.bind().rotary(q, k, inv_freq, start, interleaved, inverse, q_out, k_out)


def paged_append(k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                 start: torch.Tensor, counts: Optional[torch.Tensor] = None, *, q: Optional[torch.Tensor] = None,
                 inv_freq: Optional[torch.Tensor] = None, interleaved: bool = False,
                 q_out: Optional[torch.Tensor] = None, k_scales: Optional[torch.Tensor] = None,
                 v_scales: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Put ``k`` and ``v`` (``[B, S, Hkv, hd]``) at positions ``start[b] + s`` of the cache, for ``s < counts[b]`` (all ``S`` tokens
    where ``counts`` is not given); the rest of the cache stays as it was.

    With ``inv_freq`` the keys are turned by position as in :func:`rotary`, and ``q`` (``[B, S, H, hd]``), where given, is
    returned turned; queries behind ``counts[b]`` are copied as they are.  ``q_out`` may be ``q`` itself.

    Into a cache in 8 bits a block's new elements (keys in fp32 behind their rotation) get the smallest power of two, 2^-100 at least, of
    which 448 times reaches the largest finite one, and each is rounded once to a multiple of it; infinities and NaN are held as NaN.
    (From 1.9375 2^127 on the nearest multiple is 2^128, which neither fp32 nor bf16 holds.)
    A block that has rows in front of ``start[b]`` keeps at least its own scale; where it grows, those rows are rounded anew (exact but
    for the smallest ones).  What stands in a block behind the last new token has no meaning any more."""
    return _lib.bind().paged_append(k_pages, v_pages, table, k, v, start, counts, q, inv_freq, interleaved, q_out, k_scales, v_scales)


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor,
                    lengths: torch.Tensor, *, scale: Optional[float] = None,
                    out: Optional[torch.Tensor] = None, k_scales: Optional[torch.Tensor] = None,
                    v_scales: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Attention of one token per sequence over the first ``lengths[b]`` positions of the cache; returns ``(o, lse)``.

    ``q`` is ``[B, H, hd]`` (bf16 or fp16, ``hd`` 64 or 128), ``H`` a multiple of the cache's heads, which groups of ``H / Hkv``
    neighbouring query heads share.  ``o`` is ``[B, H, hd]``, ``lse`` fp32 ``[B, H]`` (natural logarithm).  A sequence of no tokens
    has ``o = 0`` and ``lse = -inf``.  ``scale`` is ``1 / sqrt(hd)`` where it is not given.  What stands in the cache behind
    ``lengths[b]`` has no influence, NaN included; an infinite value before it is infinity in its element of ``o``, NaN beside one of
    the other sign or where its token has no weight (a score of ``-inf``, or so far below the largest that fp32 has 0 for it)."""
    return _lib.bind().paged_attention(q, k_pages, v_pages, table, lengths, scale, out, k_scales, v_scales)


def logits_process(logits: torch.Tensor, *, vocab: Optional[int] = None, tokens: Optional[torch.Tensor] = None,
                   lengths: Optional[torch.Tensor] = None, prompt_lengths: Optional[torch.Tensor] = None,
                   repetition=None, frequency=None, presence=None, bias: Optional[torch.Tensor] = None,
                   allowed: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                   out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """The first ``vocab`` columns of ``logits`` (``[R, columns]``; bf16, fp16 or fp32), ready for a choice, as ``[R, vocab]``.

    ``tokens`` (int64 ``[R, L]``) is the history of each row: ``lengths[r]`` tokens (``L`` where not given), of which the first
    ``prompt_lengths[r]`` (0) are the prompt.  In this order:

    * ``repetition``: a logit of a token anywhere in the history is divided by it if positive, else multiplied (> 0; 1: none);
    * ``frequency``: times the token's count among the generated ones, subtracted;
    * ``presence``: subtracted where that count is not 0;
    * ``bias``: fp32 ``[vocab]`` or ``[R, vocab]``, added;
    * ``allowed``: int32 words, ``[ceil(vocab / 32)]`` or ``[R, ...]``: a column whose bit (``column % 32``, the lowest first) is
      clear becomes ``-inf``, whatever it was.  A row without any allowed column is ``-inf`` throughout.

    The three penalties are numbers, or fp32 ``[R]``.  The result has the type of ``logits`` or ``out_dtype`` (fp32); its rows start
    on 16 bytes, so a new one is a view of wider rows.  ``out`` may be ``logits[:, :vocab]`` itself."""
    return _lib.bind().logits_process(logits, vocab, tokens, lengths, prompt_lengths, repetition, frequency, presence, bias, allowed,
                                      out, out_dtype)


def sample(logits: torch.Tensor, uniform: torch.Tensor, *, vocab: Optional[int] = None, temperature=None, top_k=None, top_p=None,
           min_p=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """A token for each row of ``logits`` (the first ``vocab`` columns, 2^20 at most, of ``[R, columns]``; bf16, fp16 or fp32) from
    ``uniform`` (fp32 ``[R]``, in [0, 1)); returns ``(token int64 [R], logprob fp32 [R])``.

    Token ``i`` weighs ``w_i = round(2^43 exp((x_i - max x) / temperature))`` (formed in 64 bits: within 2^-8 of a half, either neighbour).
    In the order of the logits, equal ones by their ids, are kept

    * ``top_k``: the first ``top_k`` (0: all);
    * ``top_p``: of those the ones before which less than ``top_p`` of their sum lies (1: all; the first always);
    * ``min_p``: of those the ones that weigh at least ``min_p`` of the largest (0: all).

    The token is the first by id with ``sum_{j <= i} w_j > floor(uniform sum_j w_j)`` over what is kept, ``logprob`` is
    ``log(w_i / sum_j w_j)``.  ``temperature`` 0 is the highest logit, the first of equal ones.  Sums are whole numbers: the same row, settings
    and random number give the same token in any batch.

    Settings are numbers, or tensors ``[R]``: fp32, ``top_k`` int32.  Of a tensor's rows, ``top_k`` below 0 is 0, ``top_p`` and ``min_p``
    beyond their range count as its ends, an infinite temperature makes all tokens equal, and ``uniform`` beyond its range takes the first or
    last kept token that weighs anything.  Tokens at ``inf`` leave the others nothing.  A row of nothing but ``-inf`` has token -1 and
    ``logprob`` ``-inf``; one with NaN among its logits, settings or ``uniform``, or with a negative temperature, -1 and NaN."""
    return _lib.bind().sample(logits, uniform, vocab, temperature, top_k, top_p, min_p)
