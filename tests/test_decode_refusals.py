"""Arguments that the operators between a decoder and its next token refuse, and the page arithmetic that their kernels use,
without a GPU: every refusal comes before anything is launched."""
import subprocess
from pathlib import Path

import pytest
import torch

from frankentorch_b200.ops import decode as D
from frankentorch_b200.ops.kernels import KernelError

CSRC = Path(__file__).resolve().parent.parent / "frankentorch_b200" / "csrc"
BF = torch.bfloat16


def _z(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype)


def _i(*v):
    return torch.tensor(v, dtype=torch.int32)


def _refused(match, fn, *a, **kw):
    with pytest.raises(KernelError, match=match):
        fn(*a, **kw)


ROTARY = dict(q=lambda: _z(2, 3, 4, 64), k=lambda: _z(2, 3, 2, 64), inv_freq=lambda: D.rotary_frequencies(64, device="cpu"))


@pytest.mark.parametrize("match,change", [
    ("CUDA tensors", {}),
    ("bf16 or fp16", {"q": lambda: _z(2, 3, 4, 64, dtype=torch.float32)}),
    ("4 dimensions", {"q": lambda: _z(2, 12, 64)}),
    ("k is torch.float16", {"k": lambda: _z(2, 3, 2, 64, dtype=torch.float16)}),
    (r"k must be \[2, 3", {"k": lambda: _z(2, 4, 2, 64)}),
    ("multiple of 16", {"q": lambda: _z(2, 3, 4, 72), "k": lambda: None}),
    ("16 bytes", {"q": lambda: _z(2, 3, 4, 68)[..., 4:]}),
    ("16 bytes", {"q": lambda: _z(2, 3, 64, 4).transpose(2, 3)}),
    ("16 bytes", {"k": lambda: _z(2, 3, 2, 65)[..., :64]}),
    ("float64", {"inv_freq": lambda: torch.zeros(32)}),
    ("multiple of 8", {"inv_freq": lambda: torch.zeros(12, dtype=torch.float64)}),
    ("half of the head", {"inv_freq": lambda: torch.zeros(40, dtype=torch.float64)}),
    ("needs inv_freq", {"inv_freq": lambda: None}),
    ("start must be", {"start": lambda: torch.zeros(2, dtype=torch.int64)}),
    ("start must be", {"start": lambda: _i(0, 0, 0)}),
    ("q_out must be", {"q_out": lambda: _z(2, 3, 5, 64)}),
    ("must not share memory", {"q_out": lambda: _z(2, 3, 1, 64).expand(2, 3, 4, 64)}),
    ("k_out is torch.float32", {"k_out": lambda: _z(2, 3, 2, 64, dtype=torch.float32)}),
])
def test_rotary(match, change):
    kw = {n: f() for n, f in {**ROTARY, **change}.items()}
    _refused(match, D.rotary, kw.pop("q"), kw.pop("k"), kw.pop("inv_freq"), **kw)


def test_frequencies():
    w = D.rotary_frequencies(64, base=500.0, device="cpu")
    assert w.dtype == torch.float64 and w.shape == (32,)
    assert [float(w[i]) for i in (0, 1, 31)] == pytest.approx([1.0, 500.0 ** (-1 / 32), 500.0 ** (-31 / 32)], rel=1e-15)
    _refused("multiple of 16", D.rotary_frequencies, 24, device="cpu")


APPEND = dict(k_pages=lambda: _z(5, 2, 16, 64), v_pages=lambda: _z(5, 2, 16, 64), table=lambda: torch.zeros(3, 4, dtype=torch.int32),
              k=lambda: _z(3, 7, 2, 64), v=lambda: _z(3, 7, 2, 64), start=lambda: _i(0, 0, 0), counts=lambda: None)


@pytest.mark.parametrize("match,change", [
    ("CUDA tensors", {}),
    ("bf16 or fp16", {"k": lambda: _z(3, 7, 2, 64, dtype=torch.float32)}),
    ("differ", {"v": lambda: _z(3, 7, 1, 64)}),
    ("v is", {"v": lambda: _z(3, 7, 2, 64, dtype=torch.float16)}),
    ("k_pages is", {"k_pages": lambda: _z(5, 2, 16, 64, dtype=torch.float16)}),
    ("differ", {"v_pages": lambda: _z(6, 2, 16, 64)}),
    ("power of two", {"k_pages": lambda: _z(5, 2, 12, 64), "v_pages": lambda: _z(5, 2, 12, 64)}),
    ("pages must be", {"k_pages": lambda: _z(5, 3, 16, 64), "v_pages": lambda: _z(5, 3, 16, 64)}),
    ("pages must be", {"k_pages": lambda: _z(5, 2, 16, 128), "v_pages": lambda: _z(5, 2, 16, 128)}),
    ("must not share memory", {"k_pages": lambda: _z(1, 2, 16, 64).expand(5, 2, 16, 64)}),
    ("16 bytes", {"v_pages": lambda: _z(5, 2, 16, 68)[..., :64]}),
    ("no pages", {"k_pages": lambda: _z(0, 2, 16, 64), "v_pages": lambda: _z(0, 2, 16, 64)}),
    ("page table", {"table": lambda: torch.zeros(3, 4, dtype=torch.int64)}),
    ("page table", {"table": lambda: torch.zeros(2, 4, dtype=torch.int32)}),
    ("page table", {"table": lambda: torch.zeros(3, 0, dtype=torch.int32)}),
    ("page table", {"table": lambda: torch.zeros(4, 3, dtype=torch.int32).t()}),
    ("start must be", {"start": lambda: _i(0, 0)}),
    ("counts must be", {"counts": lambda: torch.zeros(3)}),
    ("inv_freq is missing", {"q": lambda: _z(3, 7, 4, 64)}),
    ("q must be", {"q": lambda: _z(3, 6, 4, 64), "inv_freq": lambda: D.rotary_frequencies(32, device="cpu")}),
    ("q_out without q", {"q_out": lambda: _z(3, 7, 4, 64)}),
])
def test_append(match, change):
    kw = {n: f() for n, f in {**APPEND, **change}.items()}
    _refused(match, D.paged_append, **kw)


ATTEND = dict(q=lambda: _z(3, 4, 64), k_pages=lambda: _z(5, 2, 16, 64), v_pages=lambda: _z(5, 2, 16, 64),
              table=lambda: torch.zeros(3, 4, dtype=torch.int32), lengths=lambda: _i(1, 2, 3))


@pytest.mark.parametrize("match,change", [
    ("CUDA tensors", {}),
    ("bf16 or fp16", {"q": lambda: _z(3, 4, 64, dtype=torch.float32)}),
    ("3 dimensions", {"q": lambda: _z(3, 1, 4, 64)}),
    ("head size", {"q": lambda: _z(3, 4, 32), "k_pages": lambda: _z(5, 2, 16, 32), "v_pages": lambda: _z(5, 2, 16, 32)}),
    ("groups", {"q": lambda: _z(3, 5, 64)}),
    ("groups", {"k_pages": lambda: _z(5, 0, 16, 64), "v_pages": lambda: _z(5, 0, 16, 64)}),
    ("4 dimensions", {"k_pages": lambda: _z(2, 16, 64)}),
    ("k_pages is", {"k_pages": lambda: _z(5, 2, 16, 64, dtype=torch.float16)}),
    ("differ", {"k_pages": lambda: _z(5, 2, 8, 64)}),
    ("power of two", {"k_pages": lambda: _z(5, 2, 24, 64), "v_pages": lambda: _z(5, 2, 24, 64)}),
    ("16 bytes", {"q": lambda: _z(3, 4, 65)[..., :64]}),
    ("no pages", {"k_pages": lambda: _z(0, 2, 16, 64), "v_pages": lambda: _z(0, 2, 16, 64)}),
    ("2.31 - 256 positions", {"table": lambda: torch.empty(1, 2 ** 27, dtype=torch.int32).expand(3, -1)}),
    ("lengths must be", {"lengths": lambda: torch.ones(3, dtype=torch.int64)}),
    ("lengths must be", {"lengths": lambda: _i(1, 1, 1, 1, 1, 1)[::2]}),
    ("page table", {"table": lambda: torch.zeros(12, dtype=torch.int32)}),
    ("out must be", {"out": lambda: _z(3, 4, 128)}),
    ("must not share memory", {"out": lambda: _z(3, 1, 64).expand(3, 4, 64)}),
    ("out is", {"out": lambda: _z(3, 4, 64, dtype=torch.float32)}),
])
def test_attention(match, change):
    _refused(match, D.paged_attention, **{n: f() for n, f in {**ATTEND, **change}.items()})


@pytest.mark.parametrize("match,kw", [
    ("CUDA tensors", {}),
    ("bf16, fp16 or fp32", {"logits": lambda: _z(2, 40, dtype=torch.float64)}),
    ("rows, columns", {"logits": lambda: _z(2, 2, 40)}),
    ("rows, columns", {"logits": lambda: _z(40, 2).t()}),
    ("does not fit", {"vocab": lambda: 41}),
    ("does not fit", {"vocab": lambda: 0}),
    ("leave as", {"out_dtype": lambda: torch.float16}),
    ("leave as", {"out": lambda: _z(2, 40, dtype=torch.float16)}),
    ("out must be", {"out": lambda: _z(2, 39)}),
    ("out must be", {"out": lambda: _z(1, 40).expand(2, 40)}),
    ("tokens must be", {"tokens": lambda: torch.zeros(2, 3, dtype=torch.int32)}),
    ("tokens must be", {"tokens": lambda: torch.zeros(3, 3, dtype=torch.int64)}),
    ("lengths without", {"lengths": lambda: _i(1, 1)}),
    ("penalties without", {"repetition": lambda: 1.2}),
    ("lengths must be", {"tokens": lambda: torch.zeros(2, 3, dtype=torch.int64), "lengths": lambda: _i(1)}),
    ("must be positive", {"tokens": lambda: torch.zeros(2, 3, dtype=torch.int64), "repetition": lambda: 0.0}),
    ("must be finite", {"tokens": lambda: torch.zeros(2, 3, dtype=torch.int64), "presence": lambda: float("nan")}),
    ("frequency must be", {"tokens": lambda: torch.zeros(2, 3, dtype=torch.int64), "frequency": lambda: torch.zeros(3)}),
    ("bias must be", {"bias": lambda: torch.zeros(39)}),
    ("bias must be", {"bias": lambda: torch.zeros(3, 40)}),
    ("bias must be", {"bias": lambda: _z(40)}),
    ("allowed must be", {"allowed": lambda: torch.zeros(1, dtype=torch.int32)}),
    ("allowed must be", {"allowed": lambda: torch.zeros(2, 40, dtype=torch.bool)}),
])
def test_logits(match, kw):
    kw = {n: f() for n, f in kw.items()}
    _refused(match, D.logits_process, kw.pop("logits", _z(2, 40)), **kw)


PROBE = r"""
#include <cassert>
#include "paged_cache.h"
int main() {
  const int table[] = {3, 0, 7, -1, 2, 1, 6, 2147483647};          // two sequences of four pages
  const ftk::PagedTable t = {table, 4, 4, 7, 5};                   // seven pages of 32 rows
  assert(ftk::paged_page(t, 0, 0) == 3 && ftk::paged_page(t, 0, 31) == 3 && ftk::paged_page(t, 0, 32) == 0);
  assert(ftk::paged_page(t, 0, 64) == -1);                         // 7 is no page of the cache
  assert(ftk::paged_page(t, 0, 96) == -1 && ftk::paged_page(t, 0, 127) == -1);
  assert(ftk::paged_page(t, 0, 128) == -1);                        // behind the table: not the next sequence's page
  assert(ftk::paged_page(t, 0, -1) == -1 && ftk::paged_page(t, 1, -128) == -1);
  assert(ftk::paged_page(t, 1, 0) == 2 && ftk::paged_page(t, 1, 95) == 6 && ftk::paged_page(t, 1, 96) == -1);
  assert(ftk::paged_page(t, 0, 1ll << 40) == -1);
  assert(ftk::paged_row(t, 0) == 0 && ftk::paged_row(t, 31) == 31 && ftk::paged_row(t, 33) == 1);
  bool bad;
  assert(ftk::paged_length(t, 0, bad) == 0 && !bad);
  assert(ftk::paged_length(t, 128, bad) == 128 && !bad);
  assert(ftk::paged_length(t, 129, bad) == 128 && bad);
  assert(ftk::paged_length(t, -1, bad) == 0 && bad);
  const ftk::PagedTable wide = {table, 4, 1 << 20, 7, 16};         // more rows than 32 bits count
  assert(ftk::paged_length(wide, 2147483647, bad) == 2147483647 && !bad);
  const ftk::PagedTable one = {table, 4, 4, 7, 0};                 // pages of one row
  assert(ftk::paged_page(one, 1, 2) == 6 && ftk::paged_row(one, 2) == 0);
}
"""


def test_page_arithmetic(tmp_path):
    src = tmp_path / "probe.cpp"
    src.write_text(PROBE)
    exe = tmp_path / "probe"
    subprocess.run(["g++", "-std=c++17", "-I", str(CSRC), str(src), "-o", str(exe)], check=True, timeout=120)
    subprocess.run([str(exe)], check=True, timeout=60)


@pytest.mark.parametrize("bad", [3.5, "x", [1, 2], torch.zeros(3).to_sparse()])
def test_operands_that_are_no_tensors(bad):
    """Refused as every other argument, whatever it is; numbers that are none raise what Python raises."""
    for name, base, fn in (("k", APPEND, D.paged_append), ("lengths", ATTEND, D.paged_attention)):
        kw = {n: f() for n, f in base.items()}
        kw[name] = bad
        _refused("tensor", fn, **kw)
    kw = {n: f() for n, f in ATTEND.items()}
    with pytest.raises(TypeError):
        D.paged_attention(**kw, scale="x")
    _refused("finite", D.paged_attention, **kw, scale=float("inf"))
    _refused("vocab", D.logits_process, _z(2, 40), vocab=-1)
    _refused("out_dtype", D.logits_process, _z(2, 40), out_dtype=7)
    with pytest.raises(TypeError):
        D.logits_process(_z(2, 40), vocab="x")


def test_refusals_leave_the_references_of_their_arguments():
    import sys
    kw = {n: f() for n, f in ATTEND.items()}
    before = {n: sys.getrefcount(t) for n, t in kw.items()}
    for _ in range(50):
        _refused("CUDA tensors", D.paged_attention, **kw)
    assert {n: sys.getrefcount(t) for n, t in kw.items()} == before


@pytest.mark.parametrize("value", [0, -0.0, -1.5, 1e-60, 7e-46, 3.4028236e38, 1e39, 1e300])
def test_repetitions_that_fp32_does_not_hold(value):
    """The factor is handed on in fp32: as 0 it would make infinity of every logit, as infinity NaN of a logit of 0."""
    tokens = torch.zeros(2, 3, dtype=torch.int64)
    _refused("repetition must be positive", D.logits_process, _z(2, 40), tokens=tokens, repetition=value)
    for good in (1e-45, 3.4028234e38):
        _refused("CUDA tensors", D.logits_process, _z(2, 40), tokens=tokens, repetition=good)


def _strided(size, stride, dtype=BF):
    return torch.zeros(1 + sum((n - 1) * s for n, s in zip(size, stride)), dtype=dtype).as_strided(size, stride)


def test_outputs_whose_rows_overlap():
    """Rows, heads or sequences that share elements are written by several threads: refused whatever the stride."""
    def base(kw):
        return {n: f() for n, f in kw.items()}
    for stride in ((128, 32, 1), (64, 64, 1), (64, 128, 1), (8, 64, 1), (256, 56, 1), (192, 64, 1)):
        _refused("must not share memory", D.paged_attention, **base(ATTEND), out=_strided((3, 4, 64), stride))
    for stride in ((256, 64, 1), (64, 192, 1), (264, 64, 1), (1000, 72, 1), (64, 208, 1)):
        _refused("CUDA tensors", D.paged_attention, **base(ATTEND), out=_strided((3, 4, 64), stride))
    size = (5, 2, 16, 64)
    for stride in ((2048, 512, 64, 1), (1024, 1024, 64, 1), (2048, 1024, 32, 1), (2048, 64, 64, 1), (64, 2048, 64, 1), (2048, 32, 128, 1)):
        for name in ("k_pages", "v_pages"):
            _refused("%s is written" % name, D.paged_append, **{**base(APPEND), name: _strided(size, stride)})
        _refused("CUDA tensors", D.paged_attention, **{**base(ATTEND), "k_pages": _strided(size, stride)})      # read, that is well
    for stride in ((2048, 1024, 64, 1), (2048, 64, 128, 1), (1024, 5 * 1024, 64, 1), (64, 320, 640, 1), (4096, 1024, 64, 1)):
        _refused("CUDA tensors", D.paged_append, **{**base(APPEND), "k_pages": _strided(size, stride)})
    kw = base(ROTARY)
    q, k, w = kw.pop("q"), kw.pop("k"), kw.pop("inv_freq")
    for stride in ((768, 128, 64, 1), (768, 256, 48, 1), (256, 256, 64, 1), (0, 256, 64, 1)):
        _refused("q_out is written", D.rotary, q, k, w, q_out=_strided((2, 3, 4, 64), stride))
    _refused("CUDA tensors", D.rotary, q, k, w, q_out=_strided((2, 3, 4, 64), (64, 512, 128, 1)))
    # what has one sequence, page or head may have any stride there
    _refused("CUDA tensors", D.rotary, q[:1], None, w, q_out=_strided((1, 3, 4, 64), (0, 256, 64, 1)))


@pytest.mark.parametrize("scale", [1e39, -1e300, 3e38])
def test_scales_that_fp32_does_not_hold(scale):
    """The kernel multiplies by scale log2(e) in fp32: as infinity it would make NaN of a score of 0."""
    kw = {n: f() for n, f in ATTEND.items()}
    _refused("scale must be finite", D.paged_attention, **kw, scale=scale)
    _refused("CUDA tensors", D.paged_attention, **kw, scale=scale / 1e270)
    _refused("CUDA tensors", D.paged_attention, **kw, scale=2e38)
