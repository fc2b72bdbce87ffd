"""Launchers of the operators between a trained decoder and its next token (``torch.Tensor`` in, ``torch.Tensor`` out).

* :func:`rotary`: queries and keys turned by position, forward and backward (training);
* :func:`paged_append`: keys and values of new tokens into a paged cache, turned on the way;
* :func:`paged_attention`: one new token per sequence over the cache;
* :func:`logits_process`: penalties for repeated tokens, biases and a grammar's mask on the logits of a step.

The reference composes the rotation from tensor operators (``apply_rotary_pos_emb``) and has no cache, no decoding attention
and no logits processing; shapes, masks and empty rows follow its attention (ft-nn/src/lib.rs:5145-5184) where they overlap.

A paged cache is two tensors of pages, ``[pages, heads, page, hd]`` (``page`` a power of two), and a table ``[B, columns]`` of
page numbers (int32): position ``p`` of sequence ``b`` is row ``p % page`` of page ``table[b, p // page]``.  Table entries behind the
last position that a call touches are not read.  Rows of ``hd`` elements are contiguous and start on 16 bytes; everything else
may be strided.  Lengths, positions and counts are int32 on the device, so a captured graph follows them.

As everywhere in :mod:`~frankentorch_b200.ops.kernels`, a call enqueues on the current stream of its tensors' device and
returns; arguments that the host can judge are refused with :class:`~.kernels.KernelError`; a page, token or length out of range
on the device is reported by :func:`~.kernels.check_status`, and what it leads to is not read and not written.  A call keeps
nothing: its scratch is its own, so calls of several streams, threads and captured graphs do not meet.  Two tokens of one
append must not have the same place, and an output must not overlap an input other than where the function says so.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from . import _lib
from . import kernels as K
from .kernels import KernelError

_T16 = {torch.bfloat16: 0, torch.float16: 1}
_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
HEAD_SIZES = (64, 128)          # of paged_attention, as of attention_fwd
MAX_HEAD = 1024                 # of rotary and paged_append


def _launch(name: str, fn, dev: torch.device, *args) -> None:
    if dev.index == K._get_device():
        K._chk(fn(*args, K._stream()), name)
    else:
        with torch.cuda.device(dev):
            K._chk(fn(*args, K._stream()), name)


def _on_device(ref: torch.Tensor, **others) -> None:
    if not ref.is_cuda:
        raise KernelError("operands must be CUDA tensors")
    for name, t in others.items():
        if t is not None and t.device != ref.device:
            raise KernelError(f"{name} is on {t.device}, the other operands on {ref.device}")


def _heads(t: torch.Tensor, name: str, ndim: int, dtype: torch.dtype, out: bool = False) -> tuple:
    """Strides of a ``[..., heads, hd]`` operand but the last: rows of whole 16 bytes, every row on a 16-byte boundary."""
    if t.dim() != ndim:
        raise KernelError(f"{name} must have {ndim} dimensions, got shape {tuple(t.shape)}")
    if t.dtype is not dtype:
        raise KernelError(f"{name} is {t.dtype}, expected {dtype}")
    st = t.stride()
    bits = t.data_ptr() >> 1
    for n, x in zip(t.shape[:-1], st):
        if n > 1:
            bits |= x
            if out and x == 0:
                raise KernelError(f"{name} is written: its elements must not share memory")
    if st[-1] != 1 or bits & 7 or t.data_ptr() & 1:
        raise KernelError(f"{name} needs contiguous rows that start on 16 bytes, got strides {st}")
    return st[:-1]


def _ints(t: torch.Tensor, name: str, n: int) -> int:
    if t.dtype is not torch.int32 or t.dim() != 1 or t.shape[0] != n or (n > 1 and t.stride(0) != 1):
        raise KernelError(f"{name} must be contiguous int32 [{n}], got {t.dtype} {tuple(t.shape)}")
    return t.data_ptr()


def _freq(inv_freq: Optional[torch.Tensor], hd: int) -> Tuple[int, int]:
    """(pointer, turned elements) of a table of frequencies."""
    if inv_freq is None:
        return 0, 0
    if inv_freq.dtype is not torch.float64 or inv_freq.dim() != 1 or not inv_freq.is_contiguous():
        raise KernelError("inv_freq must be contiguous float64 [turned elements / 2]")
    n = inv_freq.shape[0]
    if n % 8 or not 0 < 2 * n <= hd:
        raise KernelError(f"inv_freq has {n} entries: a multiple of 8, at most half of the head's {hd} elements, is wanted")
    return inv_freq.data_ptr(), 2 * n


def _table(table: torch.Tensor, B: int) -> None:
    if table.dtype is not torch.int32 or table.dim() != 2 or table.shape[0] != B or table.shape[1] < 1 or \
            (table.shape[1] > 1 and table.stride(1) != 1):
        raise KernelError(f"the page table must be int32 [{B}, columns] with unit inner stride, got {table.dtype} "
                          f"{tuple(table.shape)}")


def _pages(k_pages, v_pages, heads: int, hd: int, dtype: torch.dtype, out: bool) -> tuple:
    ks, vs = _heads(k_pages, "k_pages", 4, dtype, out), _heads(v_pages, "v_pages", 4, dtype, out)
    shape = k_pages.shape
    if v_pages.shape != shape:
        raise KernelError(f"k_pages {tuple(shape)} and v_pages {tuple(v_pages.shape)} differ")
    page = shape[2]
    if shape[1] != heads or shape[3] != hd or page < 1 or page & (page - 1):
        raise KernelError(f"pages must be [pages, {heads}, page, {hd}] with a power of two of rows, got {tuple(shape)}")
    return ks, vs, page.bit_length() - 1


def rotary_frequencies(turned: int, base: float = 10000.0, device="cuda") -> torch.Tensor:
    """Angle per position of each pair of the ``turned`` leading elements of a head: ``base ** (-2 i / turned)``, float64."""
    if turned < 16 or turned % 16:
        raise KernelError("the turned elements of a head are a positive multiple of 16")
    return (float(base) ** (-torch.arange(0, turned, 2, dtype=torch.float64) / turned)).to(device)


_ZEROS3 = (0, 0, 0)


def _rows4(t, name, B, S, hd, dtype):
    st = _heads(t, name, 4, dtype)
    if t.shape[0] != B or t.shape[1] != S or t.shape[3] != hd:
        raise KernelError(f"{name} must be [{B}, {S}, heads, {hd}], got {tuple(t.shape)}")
    return st


def _turned_out(out, like, name, dtype):
    if out is None:
        return like.new_empty(like.shape)
    if out.shape != like.shape:
        raise KernelError(f"{name} must be {tuple(like.shape)}, got {tuple(out.shape)}")
    return out


def rotary(q: torch.Tensor, k: Optional[torch.Tensor], inv_freq: torch.Tensor, *, start: Optional[torch.Tensor] = None,
           interleaved: bool = False, inverse: bool = False, q_out: Optional[torch.Tensor] = None,
           k_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """``(q, k)`` turned by position: pair ``i`` of token ``s`` of sequence ``b`` by ``(start[b] + s) inv_freq[i]``.

    ``q`` is ``[B, S, H, hd]``, ``k`` ``[B, S, Hkv, hd]`` or None; bf16 or fp16, ``hd`` a multiple of 16.  ``inv_freq`` (float64, see
    :func:`rotary_frequencies`) has one entry per pair: pairs are ``(i, i + n)`` with ``n = len(inv_freq)``, or ``(2 i, 2 i + 1)``
    when ``interleaved``; elements from ``2 n`` on are copied.  ``start`` is 0 where it is not given.  ``inverse`` turns back: the
    backward pass of the rotation is its inverse on the gradient.  ``q_out`` / ``k_out`` may be ``q`` / ``k`` themselves."""
    dtype = q.dtype
    if dtype not in _T16:
        raise KernelError(f"rotary takes bf16 or fp16, got {dtype}")
    qs = _heads(q, "q", 4, dtype)
    B, S, H, hd = q.shape
    if hd % 16 or not 0 < hd <= MAX_HEAD:
        raise KernelError(f"head size {hd} is no multiple of 16 up to {MAX_HEAD}")
    if inv_freq is None:
        raise KernelError("rotary needs inv_freq")
    freq, turned = _freq(inv_freq, hd)
    q_out = _turned_out(q_out, q, "q_out", dtype)
    qo = _heads(q_out, "q_out", 4, dtype, True)
    ks = ko = _ZEROS3
    Hk = 0
    if k is not None:
        ks = _rows4(k, "k", B, S, hd, dtype)
        Hk = k.shape[2]
        k_out = _turned_out(k_out, k, "k_out", dtype)
        ko = _heads(k_out, "k_out", 4, dtype, True)
    st = 0 if start is None else _ints(start, "start", B)
    _on_device(q, k=k, inv_freq=inv_freq, start=start, q_out=q_out, k_out=k_out)
    if B * S * (H + Hk) == 0:
        return q_out, k_out
    desc = _lib.ROTARY_DESC.pack(
        _T16[dtype], B, S, H, Hk, hd, turned, interleaved, inverse, q.data_ptr(), *qs,
        0 if k is None else k.data_ptr(), *ks, 0, 0, 0, 0, q_out.data_ptr(), *qo, 0 if k is None else k_out.data_ptr(), *ko,
        freq, st, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0)
    _launch("ftk_rotary", _lib.load().rotary_packed, q.device, desc)
    return q_out, k_out


def paged_append(k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                 start: torch.Tensor, counts: Optional[torch.Tensor] = None, *, q: Optional[torch.Tensor] = None,
                 inv_freq: Optional[torch.Tensor] = None, interleaved: bool = False,
                 q_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Put ``k`` and ``v`` (``[B, S, Hkv, hd]``) at positions ``start[b] + s`` of the cache, for ``s < counts[b]`` (all ``S`` tokens
    where ``counts`` is not given); the rest of the cache stays as it was.

    With ``inv_freq`` the keys are turned by position as in :func:`rotary`, and ``q`` (``[B, S, H, hd]``), where given, is
    returned turned; queries behind ``counts[b]`` are copied as they are.  ``q_out`` may be ``q`` itself."""
    dtype = k.dtype
    if dtype not in _T16:
        raise KernelError(f"paged_append takes bf16 or fp16, got {dtype}")
    ks = _heads(k, "k", 4, dtype)
    B, S, Hk, hd = k.shape
    if hd % 16 or not 0 < hd <= MAX_HEAD:
        raise KernelError(f"head size {hd} is no multiple of 16 up to {MAX_HEAD}")
    vs = _heads(v, "v", 4, dtype)
    if v.shape != k.shape:
        raise KernelError(f"k {tuple(k.shape)} and v {tuple(v.shape)} differ")
    kp, vp, shift = _pages(k_pages, v_pages, Hk, hd, dtype, True)
    _table(table, B)
    st = _ints(start, "start", B)
    ct = 0 if counts is None else _ints(counts, "counts", B)
    freq, turned = _freq(inv_freq, hd)
    qs = qo = _ZEROS3
    H = 0
    if q is not None:
        if inv_freq is None:
            raise KernelError("paged_append takes queries to turn them: inv_freq is missing")
        qs = _rows4(q, "q", B, S, hd, dtype)
        H = q.shape[2]
        q_out = _turned_out(q_out, q, "q_out", dtype)
        qo = _heads(q_out, "q_out", 4, dtype, True)
    elif q_out is not None:
        raise KernelError("q_out without q")
    _on_device(k, v=v, k_pages=k_pages, v_pages=v_pages, table=table, start=start, counts=counts, inv_freq=inv_freq, q=q,
               q_out=q_out)
    if B * S * (H + Hk) == 0:
        return q_out
    if k_pages.shape[0] == 0:
        raise KernelError("the cache has no pages")
    desc = _lib.ROTARY_DESC.pack(
        _T16[dtype], B, S, H, Hk, hd, turned, interleaved, 0, 0 if q is None else q.data_ptr(), *qs, k.data_ptr(), *ks,
        v.data_ptr(), *vs, 0 if q is None else q_out.data_ptr(), *qo, 0, 0, 0, 0, freq, st, ct, k_pages.data_ptr(), *kp,
        v_pages.data_ptr(), *vp, table.data_ptr(), table.stride(0), table.shape[1], k_pages.shape[0], shift)
    _launch("ftk_rotary", _lib.load().rotary_packed, k.device, desc)
    return q_out


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor,
                    lengths: torch.Tensor, *, scale: Optional[float] = None,
                    out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Attention of one token per sequence over the first ``lengths[b]`` positions of the cache; returns ``(o, lse)``.

    ``q`` is ``[B, H, hd]`` (bf16 or fp16, ``hd`` 64 or 128), ``H`` a multiple of the cache's heads, which groups of ``H / Hkv``
    neighbouring query heads share.  ``o`` is ``[B, H, hd]``, ``lse`` fp32 ``[B, H]`` (natural logarithm).  A sequence of no tokens
    has ``o = 0`` and ``lse = -inf``.  ``scale`` is ``1 / sqrt(hd)`` where it is not given.  What stands in the cache behind
    ``lengths[b]`` has no influence, NaN included."""
    dtype = q.dtype
    if dtype not in _T16:
        raise KernelError(f"paged_attention takes bf16 or fp16, got {dtype}")
    qs = _heads(q, "q", 3, dtype)
    B, H, hd = q.shape
    if hd not in HEAD_SIZES:
        raise KernelError(f"head size {hd} is none of {HEAD_SIZES}")
    Hk = k_pages.shape[1] if k_pages.dim() == 4 else 0
    kp, vp, shift = _pages(k_pages, v_pages, Hk, hd, dtype, False)
    if Hk < 1 or H % Hk:
        raise KernelError(f"{H} query heads do not divide into groups over {Hk} heads of the cache")
    _table(table, B)
    ln = _ints(lengths, "lengths", B)
    if out is None:
        out = q.new_empty((B, H, hd))
    elif out.shape != q.shape:
        raise KernelError(f"out must be {tuple(q.shape)}, got {tuple(out.shape)}")
    os_ = _heads(out, "out", 3, dtype, True)
    _on_device(q, k_pages=k_pages, v_pages=v_pages, table=table, lengths=lengths, out=out)
    lse = q.new_empty((B, H), dtype=torch.float32)
    if B * H == 0:
        return out, lse
    desc = _lib.PAGED_ATTN_DESC.pack(
        _T16[dtype], B, H, Hk, hd, 1.0 / math.sqrt(hd) if scale is None else float(scale), q.data_ptr(), *qs[:2],
        out.data_ptr(), *os_[:2], lse.data_ptr(), k_pages.data_ptr(), *kp, v_pages.data_ptr(), *vp, table.data_ptr(),
        table.stride(0), table.shape[1], k_pages.shape[0], shift, ln)
    lib = _lib.load()
    need = lib.paged_attn_scratch(desc)
    scratch = q.new_empty(need, dtype=torch.uint8) if need > 0 else None
    _launch("ftk_paged_attn", lib.paged_attn_packed, q.device, desc, 0 if scratch is None else scratch.data_ptr())
    return out, lse


def _per_row(x, name: str, R: int, default: float) -> Tuple[int, float]:
    if x is None:
        return 0, default
    if isinstance(x, torch.Tensor):
        if x.dtype is not torch.float32 or x.dim() != 1 or x.shape[0] != R or (R > 1 and x.stride(0) != 1):
            raise KernelError(f"{name} must be a number or contiguous fp32 [{R}], got {x.dtype} {tuple(x.shape)}")
        return x.data_ptr(), default
    x = float(x)
    if not math.isfinite(x):
        raise KernelError(f"{name} must be finite, got {x}")
    return 0, x


def _per_column(x, name: str, dtype: torch.dtype, R: int, n: int) -> Tuple[int, int]:
    """(pointer, row stride) of an operand over the vocabulary, one for all rows or one per row."""
    if x is None:
        return 0, 0
    if x.dtype is not dtype or x.dim() not in (1, 2) or x.shape[-1] < n or (x.dim() == 2 and x.shape[0] not in (1, R)) or \
            (x.shape[-1] > 1 and x.stride(-1) != 1):
        raise KernelError(f"{name} must be {dtype} [{n}] or [{R}, {n}] with unit inner stride, got {x.dtype} {tuple(x.shape)}")
    return x.data_ptr(), 0 if x.dim() == 1 or x.shape[0] == 1 else x.stride(0)


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
    dtype = logits.dtype
    if dtype not in _TYPES:
        raise KernelError(f"logits must be bf16, fp16 or fp32, got {dtype}")
    if logits.dim() != 2 or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise KernelError(f"logits must be [rows, columns] with unit inner stride, got {tuple(logits.shape)}")
    R, columns = logits.shape
    V = columns if vocab is None else int(vocab)
    if not 0 < V <= columns:
        raise KernelError(f"vocab {V} does not fit {columns} columns")
    if out is None:
        kind = dtype if out_dtype is None else out_dtype
        if kind is not dtype and kind is not torch.float32:
            raise KernelError(f"logits of {dtype} leave as {dtype} or fp32, not {kind}")
        out = logits.new_empty((R, (V + 7) // 8 * 8), dtype=kind)[:, :V]
    elif out.shape != (R, V) or (V > 1 and out.stride(1) != 1) or (R > 1 and abs(out.stride(0)) < V):
        raise KernelError(f"out must be [{R}, {V}] with unit inner stride, got {tuple(out.shape)}")
    elif (out.dtype is not dtype and out.dtype is not torch.float32) or (out_dtype is not None and out.dtype is not out_dtype):
        raise KernelError(f"logits of {dtype} leave as {dtype} or fp32, not {out.dtype}")
    tk = ldt = L = ln = pl = 0
    if tokens is not None:
        if tokens.dtype is not torch.int64 or tokens.dim() != 2 or tokens.shape[0] != R or \
                (tokens.shape[1] > 1 and tokens.stride(1) != 1):
            raise KernelError(f"tokens must be int64 [{R}, length] with unit inner stride, got {tokens.dtype} "
                              f"{tuple(tokens.shape)}")
        L = tokens.shape[1]
        tk, ldt = (tokens.data_ptr(), tokens.stride(0)) if L else (0, 0)
        ln = 0 if lengths is None else _ints(lengths, "lengths", R)
        pl = 0 if prompt_lengths is None else _ints(prompt_lengths, "prompt_lengths", R)
    elif lengths is not None or prompt_lengths is not None:
        raise KernelError("lengths without tokens")
    elif repetition is not None or frequency is not None or presence is not None:
        raise KernelError("penalties without tokens")
    rep_p, rep = _per_row(repetition, "repetition", R, 1.0)
    if rep <= 0:
        raise KernelError(f"repetition must be positive, got {rep}")
    freq_p, freq = _per_row(frequency, "frequency", R, 0.0)
    pres_p, pres = _per_row(presence, "presence", R, 0.0)
    bias_p, bias_rs = _per_column(bias, "bias", torch.float32, R, V)
    mask_p, mask_rs = _per_column(allowed, "allowed", torch.int32, R, (V + 31) // 32)
    _on_device(logits, tokens=tokens, lengths=lengths, prompt_lengths=prompt_lengths, bias=bias, allowed=allowed, out=out,
               **{n: t for n, t in (("repetition", repetition), ("frequency", frequency), ("presence", presence))
                  if isinstance(t, torch.Tensor)})
    if R == 0:
        return out
    desc = _lib.LOGITS_DESC.pack(_TYPES[dtype], _TYPES[out.dtype], R, V, logits.data_ptr(), logits.stride(0), out.data_ptr(),
                                 out.stride(0), tk, ldt, L, ln, pl, rep_p, freq_p, pres_p, rep, freq, pres, bias_p, bias_rs,
                                 mask_p, mask_rs)
    _launch("ftk_logits", _lib.load().logits_packed, logits.device, desc)
    return out
