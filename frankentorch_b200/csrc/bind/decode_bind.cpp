// Python binding of the operators between a decoder and its next token: one native call per operator.
//
// A step of a small model is a chain of calls of a few microseconds each, and checking eight tensors and packing a descriptor in
// Python takes 11 - 17 us a call, several times what the GPU needs.  Here the same takes about two: arguments are read through
// PyTorch's C++ interface, refused with the package's KernelError, outputs and scratch come from PyTorch's allocator, and the
// launcher of the kernel library is called on the current stream of the tensors' device.  The launchers' addresses, KernelError
// and the launch counter are handed over once, by init().
#include <Python.h>

#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>
#include <string>

#include "ftk_api.h"

namespace {

PyObject* g_error = nullptr;      // KernelError
PyObject* g_launched = nullptr;   // called with (status, name) for every launch
int (*g_rotary)(const FtkRotaryDesc*, void*) = nullptr;
int (*g_attn)(const FtkPagedAttnDesc*, void*, void*) = nullptr;
long long (*g_attn_scratch)(const FtkPagedAttnDesc*) = nullptr;
int (*g_logits)(const FtkLogitsDesc*, void*) = nullptr;

struct Refused {
  std::string why;
};
struct PythonError {};      // the Python error is set
[[noreturn]] void refuse(std::string why) { throw Refused{std::move(why)}; }

std::string text(at::IntArrayRef v) {
  std::string s = "(";
  for (size_t i = 0; i < v.size(); ++i) s += (i ? ", " : "") + std::to_string(v[i]);
  return s + (v.size() == 1 ? ",)" : ")");
}
std::string text(at::ScalarType t) {
  switch (t) {
    case at::kBFloat16: return "torch.bfloat16";
    case at::kHalf: return "torch.float16";
    case at::kFloat: return "torch.float32";
    case at::kDouble: return "torch.float64";
    case at::kInt: return "torch.int32";
    case at::kLong: return "torch.int64";
    default: return std::string("torch type ") + c10::toString(t);
  }
}

// An operand: a tensor, or nothing.
struct Arg {
  const at::Tensor* t = nullptr;
  const char* name;
  explicit operator bool() const { return t != nullptr; }
  const at::Tensor* operator->() const { return t; }
  void* ptr() const { return t ? t->data_ptr() : nullptr; }
};
Arg arg(PyObject* o, const char* name, bool needed) {
  Arg a;
  a.name = name;
  if (o == Py_None) {
    if (needed) refuse(std::string(name) + " is missing");
    return a;
  }
  if (!THPVariable_Check(o)) refuse(std::string(name) + " must be a tensor");
  a.t = &THPVariable_Unpack(o);
  if (a.t->layout() != at::kStrided) refuse(std::string(name) + " must be a dense tensor");
  return a;
}

// Strides of a [..., heads, hd] operand but the last: rows of whole 16 bytes, every row on a 16-byte boundary; rows of an output (`out`)
// one behind the other in some order of the dimensions.
void rows16(const Arg& a, int64_t ndim, at::ScalarType type, bool out, long long* strides) {
  const at::Tensor& t = *a.t;
  if (t.dim() != ndim) refuse(std::string(a.name) + " must have " + std::to_string(ndim) + " dimensions, got shape " + text(t.sizes()));
  if (t.scalar_type() != type) refuse(std::string(a.name) + " is " + text(t.scalar_type()) + ", expected " + text(type));
  const at::IntArrayRef n = t.sizes(), s = t.strides();
  uintptr_t bits = (uintptr_t)t.data_ptr();
  for (int64_t i = 0; i + 1 < ndim; ++i) {
    strides[i] = s[i];
    if (n[i] > 1) {
      bits |= (uintptr_t)(2 * s[i]);
    }
  }
  if (out && t.numel() > 0) {       // each stride passes what the smaller ones span: no element is two rows'
    int64_t order[4], m = 0, span = n[ndim - 1];
    for (int64_t i = 0; i + 1 < ndim; ++i)
      if (n[i] > 1) order[m++] = i;
    std::sort(order, order + m, [&](int64_t x, int64_t y) { return s[x] < s[y]; });
    for (int64_t k = 0; k < m; ++k) {
      if (s[order[k]] < span) refuse(std::string(a.name) + " is written: its elements must not share memory");
      span += s[order[k]] * (n[order[k]] - 1);
    }
  }
  if (s[ndim - 1] != 1 || bits % 16) refuse(std::string(a.name) + " needs contiguous rows that start on 16 bytes, got strides " + text(s));
}
const int* ints(const Arg& a, int64_t n) {
  if (!a) return nullptr;
  if (a->scalar_type() != at::kInt || a->dim() != 1 || a->size(0) != n || (n > 1 && a->stride(0) != 1))
    refuse(std::string(a.name) + " must be contiguous int32 [" + std::to_string(n) + "], got " + text(a->scalar_type()) + " " + text(a->sizes()));
  return (const int*)a.ptr();
}
// Sets the frequencies and the number of turned elements.
void frequencies(const Arg& a, FtkRotaryDesc& d) {
  if (!a) return;
  if (a->scalar_type() != at::kDouble || a->dim() != 1 || !a->is_contiguous()) refuse("inv_freq must be contiguous float64 [turned elements / 2]");
  const int64_t n = a->size(0);
  if (n % 8 || n <= 0 || 2 * n > d.hd)
    refuse("inv_freq has " + std::to_string(n) + " entries: a multiple of 8, at most half of the head's " + std::to_string(d.hd) + " elements, is wanted");
  d.inv_freq = (const double*)a.ptr();
  d.turn = 2 * n;
}
// Positions are counted in 32 bits, which `d`'s pages times the table's columns must not pass.
template <typename D> void page_table(const Arg& a, int64_t B, D& d) {
  if (a->scalar_type() != at::kInt || a->dim() != 2 || a->size(0) != B || a->size(1) < 1 || (a->size(1) > 1 && a->stride(1) != 1))
    refuse("the page table must be int32 [" + std::to_string(B) + ", columns] with unit inner stride, got " + text(a->scalar_type()) + " " + text(a->sizes()));
  d.table = (const int*)a.ptr();
  d.table_stride = a->stride(0), d.table_cols = a->size(1);
  if (d.table_cols > (0x7fffff00ll >> d.page_shift)) refuse("the page table has more than 2^31 - 256 positions");
}
template <typename D> void pages(const Arg& k, const Arg& v, int64_t heads, int64_t hd, at::ScalarType type, bool out, D& d) {
  long long s[3];
  rows16(k, 4, type, out, s);
  d.kp_ps = s[0], d.kp_hs = s[1], d.kp_rs = s[2];
  rows16(v, 4, type, out, s);
  d.vp_ps = s[0], d.vp_hs = s[1], d.vp_rs = s[2];
  const at::IntArrayRef n = k->sizes();
  if (v->sizes() != n) refuse("k_pages " + text(n) + " and v_pages " + text(v->sizes()) + " differ");
  const int64_t page = n[2];
  if (n[1] != heads || n[3] != hd || page < 1 || (page & (page - 1)))
    refuse("pages must be [pages, " + std::to_string(heads) + ", page, " + std::to_string(hd) + "] with a power of two of rows, got " + text(n));
  if (n[0] == 0) refuse("the cache has no pages");
  d.k_pages = k.ptr(), d.v_pages = v.ptr();
  d.n_pages = n[0];
  for (d.page_shift = 0; (int64_t(1) << d.page_shift) < page;) ++d.page_shift;
}
void same_device(const Arg& ref, std::initializer_list<const Arg*> others) {
  if (!ref->is_cuda()) refuse("operands must be CUDA tensors");
  const c10::Device dev = ref->device();
  for (const Arg* a : others)
    if (*a && (*a)->device() != dev) refuse(std::string(a->name) + " is on " + (*a)->device().str() + ", the other operands on " + dev.str());
}

// The tensors' device is current as long as this lives.
struct On {
  c10::cuda::CUDAGuard guard;
  c10::Device dev;
  explicit On(const Arg& a) : guard(a->device()), dev(a->device()) {}
  void* stream() const { return c10::cuda::getCurrentCUDAStream(dev.index()).stream(); }
  at::Tensor empty(at::IntArrayRef n, at::ScalarType type) const { return at::detail::empty_cuda(n, type, dev, std::nullopt); }
};
void launched(int status, const char* name) {
  PyObject* r = PyObject_CallFunction(g_launched, "is", status, name);
  if (!r) throw PythonError{};
  Py_DECREF(r);
}
PyObject* wrapped(const at::Tensor& t) {
  PyObject* o = THPVariable_Wrap(t);
  if (!o) throw PythonError{};
  return o;
}
// A caller's output as it came, or a new tensor.
PyObject* result(PyObject* given, const at::Tensor& made) {
  if (given == Py_None) return wrapped(made);
  Py_INCREF(given);
  return given;
}
PyObject* pair(PyObject* a, PyObject* b) {
  PyObject* t = PyTuple_New(2);
  if (!t) throw PythonError{};
  PyTuple_SET_ITEM(t, 0, a);
  PyTuple_SET_ITEM(t, 1, b);
  return t;
}
bool flag(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw PythonError{};
  return v != 0;
}
// A finite number (`name`), or `absent` for None.
double number(PyObject* o, const char* name, double absent) {
  if (o == Py_None) return absent;
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw PythonError{};
  if (!std::isfinite(v)) refuse(std::string(name) + " must be finite, got " + std::to_string(v));
  return v;
}

// Refusals become KernelError, PyTorch's own errors (out of memory among them) what they are elsewhere.
template <typename F> PyObject* guarded(F&& body) {
  HANDLE_TH_ERRORS
  try {
    return body();
  } catch (const Refused& r) {
    PyErr_SetString(g_error ? g_error : PyExc_RuntimeError, r.why.c_str());
  } catch (const PythonError&) {
  }
  return nullptr;
  END_HANDLE_TH_ERRORS
}
void expect(Py_ssize_t n, Py_ssize_t want, const char* name) {
  if (n != want) refuse(std::string(name) + ": expected " + std::to_string(want) + " arguments, got " + std::to_string(n));
}
int type16(const Arg& a, const char* what) {
  const at::ScalarType t = a->scalar_type();
  if (t != at::kBFloat16 && t != at::kHalf) refuse(std::string(what) + " takes bf16 or fp16, got " + text(t));
  return t == at::kHalf ? FTK_T_FP16 : FTK_T_BF16;
}
void head_size(int64_t hd) {
  if (hd % 16 || hd <= 0 || hd > 1024) refuse("head size " + std::to_string(hd) + " is no multiple of 16 up to 1024");
}
// [B, S, heads, hd] like the others of a call
void tokens4(const Arg& a, int64_t B, int64_t S, int64_t hd, at::ScalarType type, long long* strides) {
  rows16(a, 4, type, false, strides);
  if (a->size(0) != B || a->size(1) != S || a->size(3) != hd)
    refuse(std::string(a.name) + " must be [" + std::to_string(B) + ", " + std::to_string(S) + ", heads, " + std::to_string(hd) + "], got " + text(a->sizes()));
}
void like(const Arg& out, const Arg& in) {
  if (out->sizes() != in->sizes()) refuse(std::string(out.name) + " must be " + text(in->sizes()) + ", got " + text(out->sizes()));
}
void contiguous3(at::IntArrayRef n, long long* s) { s[2] = n[3], s[1] = n[2] * n[3], s[0] = n[1] * n[2] * n[3]; }

// rotary(q, k, inv_freq, start, interleaved, inverse, q_out, k_out) -> (q_out, k_out)
PyObject* rotary(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return guarded([&]() -> PyObject* {
    expect(nargs, 8, "rotary");
    const Arg q = arg(args[0], "q", true), k = arg(args[1], "k", false), w = arg(args[2], "rotary needs inv_freq, which", true);
    const Arg start = arg(args[3], "start", false), qo = arg(args[6], "q_out", false), ko = arg(args[7], "k_out", false);
    FtkRotaryDesc d = {};
    d.type = type16(q, "rotary");
    const at::ScalarType type = q->scalar_type();
    long long s[3];
    rows16(q, 4, type, false, s);
    d.q_bs = s[0], d.q_ss = s[1], d.q_hs = s[2];
    d.B = q->size(0), d.S = q->size(1), d.Hq = q->size(2), d.hd = q->size(3);
    head_size(d.hd);
    frequencies(w, d);
    if (qo) like(qo, q), rows16(qo, 4, type, true, s);
    else contiguous3(q->sizes(), s);
    d.qo_bs = s[0], d.qo_ss = s[1], d.qo_hs = s[2];
    if (k) {
      tokens4(k, d.B, d.S, d.hd, type, s);
      d.k_bs = s[0], d.k_ss = s[1], d.k_hs = s[2];
      d.Hkv = k->size(2);
      if (ko) like(ko, k), rows16(ko, 4, type, true, s);
      else contiguous3(k->sizes(), s);
      d.ko_bs = s[0], d.ko_ss = s[1], d.ko_hs = s[2];
    } else if (ko) {
      refuse("k_out without k");
    }
    d.start = ints(start, d.B);
    d.interleaved = flag(args[4]), d.inverse = flag(args[5]);
    same_device(q, {&k, &w, &start, &qo, &ko});
    const On on(q);
    at::Tensor a, b;
    if (!qo) a = on.empty(q->sizes(), type);
    if (k && !ko) b = on.empty(k->sizes(), type);
    if (d.B * d.S * (d.Hq + d.Hkv) != 0) {
      d.q = q.ptr(), d.q_out = qo ? qo.ptr() : a.data_ptr();
      if (k) d.k = k.ptr(), d.k_out = ko ? ko.ptr() : b.data_ptr();
      launched(g_rotary(&d, on.stream()), "ftk_rotary");
    }
    PyObject* first = result(args[6], a);
    if (!k) {
      Py_INCREF(Py_None);
      return pair(first, Py_None);
    }
    return pair(first, result(args[7], b));
  });
}

// paged_append(k_pages, v_pages, table, k, v, start, counts, q, inv_freq, interleaved, q_out) -> q_out or None
PyObject* paged_append(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return guarded([&]() -> PyObject* {
    expect(nargs, 11, "paged_append");
    const Arg kp = arg(args[0], "k_pages", true), vp = arg(args[1], "v_pages", true), table = arg(args[2], "the page table", true);
    const Arg k = arg(args[3], "k", true), v = arg(args[4], "v", true), start = arg(args[5], "start", true), counts = arg(args[6], "counts", false);
    const Arg q = arg(args[7], "q", false), w = arg(args[8], "inv_freq", false), qo = arg(args[10], "q_out", false);
    FtkRotaryDesc d = {};
    d.type = type16(k, "paged_append");
    const at::ScalarType type = k->scalar_type();
    long long s[3];
    rows16(k, 4, type, false, s);
    d.k_bs = s[0], d.k_ss = s[1], d.k_hs = s[2];
    d.B = k->size(0), d.S = k->size(1), d.Hkv = k->size(2), d.hd = k->size(3);
    head_size(d.hd);
    rows16(v, 4, type, false, s);
    d.v_bs = s[0], d.v_ss = s[1], d.v_hs = s[2];
    if (v->sizes() != k->sizes()) refuse("k " + text(k->sizes()) + " and v " + text(v->sizes()) + " differ");
    pages(kp, vp, d.Hkv, d.hd, type, true, d);
    page_table(table, d.B, d);
    d.start = ints(start, d.B), d.counts = ints(counts, d.B);
    frequencies(w, d);
    d.interleaved = flag(args[9]);
    if (q) {
      if (!w) refuse("paged_append takes queries to turn them: inv_freq is missing");
      tokens4(q, d.B, d.S, d.hd, type, s);
      d.q_bs = s[0], d.q_ss = s[1], d.q_hs = s[2];
      d.Hq = q->size(2);
      if (qo) like(qo, q), rows16(qo, 4, type, true, s);
      else contiguous3(q->sizes(), s);
      d.qo_bs = s[0], d.qo_ss = s[1], d.qo_hs = s[2];
    } else if (qo) {
      refuse("q_out without q");
    }
    same_device(k, {&v, &kp, &vp, &table, &start, &counts, &w, &q, &qo});
    const On on(k);
    at::Tensor a;
    if (q && !qo) a = on.empty(q->sizes(), type);
    if (d.B * d.S * (d.Hq + d.Hkv) != 0) {
      d.k = k.ptr(), d.v = v.ptr();
      if (q) d.q = q.ptr(), d.q_out = qo ? qo.ptr() : a.data_ptr();
      launched(g_rotary(&d, on.stream()), "ftk_rotary");
    }
    if (!q) Py_RETURN_NONE;
    return result(args[10], a);
  });
}

// paged_attention(q, k_pages, v_pages, table, lengths, scale, out) -> (o, lse)
PyObject* paged_attention(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return guarded([&]() -> PyObject* {
    expect(nargs, 7, "paged_attention");
    const Arg q = arg(args[0], "q", true), kp = arg(args[1], "k_pages", true), vp = arg(args[2], "v_pages", true);
    const Arg table = arg(args[3], "the page table", true), lengths = arg(args[4], "lengths", true), out = arg(args[6], "out", false);
    FtkPagedAttnDesc d = {};
    d.type = type16(q, "paged_attention");
    const at::ScalarType type = q->scalar_type();
    long long s[3];
    rows16(q, 3, type, false, s);
    d.q_bs = s[0], d.q_hs = s[1];
    d.B = q->size(0), d.Hq = q->size(1), d.hd = q->size(2);
    if (d.hd != 64 && d.hd != 128) refuse("head size " + std::to_string(d.hd) + " is none of (64, 128)");
    d.Hkv = kp->dim() == 4 ? kp->size(1) : 0;
    pages(kp, vp, d.Hkv, d.hd, type, false, d);
    if (d.Hkv < 1 || d.Hq % d.Hkv)
      refuse(std::to_string(d.Hq) + " query heads do not divide into groups over " + std::to_string(d.Hkv) + " heads of the cache");
    page_table(table, d.B, d);
    d.lengths = ints(lengths, d.B);
    d.scale = number(args[5], "scale", 1.0 / std::sqrt((double)d.hd));
    if (!std::isfinite((float)(d.scale * 1.5))) refuse("scale must be finite in fp32, times log2(e) too, got " + std::to_string(d.scale));
    if (out) like(out, q), rows16(out, 3, type, true, s);
    else s[1] = d.hd, s[0] = d.Hq * d.hd;
    d.o_bs = s[0], d.o_hs = s[1];
    same_device(q, {&kp, &vp, &table, &lengths, &out});
    const On on(q);
    at::Tensor o, scratch;
    if (!out) o = on.empty({d.B, d.Hq, d.hd}, type);
    at::Tensor lse = on.empty({d.B, d.Hq}, at::kFloat);
    if (d.B * d.Hq != 0) {
      d.q = q.ptr(), d.o = out ? out.ptr() : o.data_ptr(), d.lse = (float*)lse.data_ptr();
      const long long need = g_attn_scratch(&d);
      if (need > 0) scratch = on.empty({need}, at::kByte);
      launched(need < 0 ? (int)need : g_attn(&d, need > 0 ? scratch.data_ptr() : nullptr, on.stream()), "ftk_paged_attn");
    }
    PyObject* first = result(args[6], o);
    return pair(first, wrapped(lse));
  });
}

// A number, or fp32 [R]
void per_row(PyObject* o, const char* name, int64_t R, Arg& a, const float*& rows, double& value) {
  a.name = name;
  if (o == Py_None) return;
  if (!THPVariable_Check(o)) {
    value = number(o, name, value);
    return;
  }
  a = arg(o, name, true);
  if (a->scalar_type() != at::kFloat || a->dim() != 1 || a->size(0) != R || (R > 1 && a->stride(0) != 1))
    refuse(std::string(name) + " must be a number or contiguous fp32 [" + std::to_string(R) + "], got " + text(a->scalar_type()) + " " + text(a->sizes()));
  rows = (const float*)a.ptr();
}
// Pointer and row stride of an operand over the vocabulary, one for all rows or one per row
void per_column(const Arg& a, at::ScalarType type, int64_t R, int64_t n, const void*& p, long long& stride) {
  if (!a) return;
  const int64_t dim = a->dim(), last = dim ? a->size(dim - 1) : 0;
  if (a->scalar_type() != type || dim < 1 || dim > 2 || last < n || (dim == 2 && a->size(0) != 1 && a->size(0) != R) || (last > 1 && a->stride(dim - 1) != 1))
    refuse(std::string(a.name) + " must be " + text(type) + " [" + std::to_string(n) + "] or [" + std::to_string(R) + ", " + std::to_string(n) +
           "] with unit inner stride, got " + text(a->scalar_type()) + " " + text(a->sizes()));
  p = a.ptr();
  stride = dim == 1 || a->size(0) == 1 ? 0 : a->stride(0);
}
int type32(at::ScalarType t) { return t == at::kBFloat16 ? FTK_T_BF16 : t == at::kHalf ? FTK_T_FP16 : t == at::kFloat ? FTK_T_FP32 : -1; }

// logits_process(logits, vocab, tokens, lengths, prompt_lengths, repetition, frequency, presence, bias, allowed, out, out_dtype) -> out
PyObject* logits_process(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return guarded([&]() -> PyObject* {
    expect(nargs, 12, "logits_process");
    const Arg x = arg(args[0], "logits", true), tokens = arg(args[2], "tokens", false), lengths = arg(args[3], "lengths", false);
    const Arg prompts = arg(args[4], "prompt_lengths", false), bias = arg(args[8], "bias", false), allowed = arg(args[9], "allowed", false);
    const Arg out = arg(args[10], "out", false);
    const at::ScalarType type = x->scalar_type();
    FtkLogitsDesc d = {};
    d.type = type32(type);
    if (d.type < 0) refuse("logits must be bf16, fp16 or fp32, got " + text(type));
    if (x->dim() != 2 || (x->size(1) > 1 && x->stride(1) != 1)) refuse("logits must be [rows, columns] with unit inner stride, got " + text(x->sizes()));
    d.R = x->size(0);
    const int64_t columns = x->size(1);
    d.V = columns;
    if (args[1] != Py_None) {
      d.V = PyLong_AsLongLong(args[1]);
      if (d.V == -1 && PyErr_Occurred()) throw PythonError{};
    }
    if (d.V <= 0 || d.V > columns) refuse("vocab " + std::to_string(d.V) + " does not fit " + std::to_string(columns) + " columns");
    at::ScalarType kind = type;
    if (args[11] != Py_None) {
      if (!THPDtype_Check(args[11])) refuse("out_dtype must be a type");
      kind = reinterpret_cast<THPDtype*>(args[11])->scalar_type;
    }
    if (out) {
      if (out->dim() != 2 || out->size(0) != d.R || out->size(1) != d.V || (d.V > 1 && out->stride(1) != 1) || (d.R > 1 && std::abs(out->stride(0)) < d.V))
        refuse("out must be [" + std::to_string(d.R) + ", " + std::to_string(d.V) + "] with unit inner stride, got " + text(out->sizes()));
      if (args[11] != Py_None && out->scalar_type() != kind) refuse("out is " + text(out->scalar_type()) + ", out_dtype " + text(kind));
      kind = out->scalar_type();
    }
    if (kind != type && kind != at::kFloat) refuse("logits of " + text(type) + " leave as " + text(type) + " or fp32, not " + text(kind));
    d.out_type = type32(kind);
    if (tokens) {
      if (tokens->scalar_type() != at::kLong || tokens->dim() != 2 || tokens->size(0) != d.R || (tokens->size(1) > 1 && tokens->stride(1) != 1))
        refuse("tokens must be int64 [" + std::to_string(d.R) + ", length] with unit inner stride, got " + text(tokens->scalar_type()) + " " + text(tokens->sizes()));
      d.L = tokens->size(1);
      d.ldt = tokens->stride(0);
      d.lengths = ints(lengths, d.R), d.prompts = ints(prompts, d.R);
    } else if (lengths || prompts) {
      refuse("lengths without tokens");
    } else if (args[5] != Py_None || args[6] != Py_None || args[7] != Py_None) {
      refuse("penalties without tokens");
    }
    Arg rep, freq, pres;
    d.rep = 1.0;
    per_row(args[5], "repetition", d.R, rep, d.rep_rows, d.rep);
    if ((float)d.rep <= 0 || !std::isfinite((float)d.rep)) refuse("repetition must be positive and finite in fp32, got " + std::to_string(d.rep));
    per_row(args[6], "frequency", d.R, freq, d.freq_rows, d.freq);
    per_row(args[7], "presence", d.R, pres, d.pres_rows, d.pres);
    const void* p = nullptr;
    per_column(bias, at::kFloat, d.R, d.V, p, d.bias_rs);
    d.bias = (const float*)p, p = nullptr;
    per_column(allowed, at::kInt, d.R, (d.V + 31) / 32, p, d.allowed_rs);
    d.allowed = (const int*)p;
    same_device(x, {&tokens, &lengths, &prompts, &rep, &freq, &pres, &bias, &allowed, &out});
    const On on(x);
    at::Tensor made;
    d.ldo = out ? out->stride(0) : (d.V + 7) / 8 * 8;
    if (!out) made = on.empty({d.R, d.ldo}, kind);
    if (d.R != 0) {
      d.logits = x.ptr(), d.ld = x->stride(0);
      d.out = out ? out.ptr() : made.data_ptr();
      if (tokens && d.L) d.tokens = (const long long*)tokens.ptr();
      launched(g_logits(&d, on.stream()), "ftk_logits");
    }
    if (!out && d.ldo != d.V) made.unsafeGetTensorImpl()->set_sizes_and_strides(at::IntArrayRef({d.R, d.V}), at::IntArrayRef({d.ldo, 1ll}));
    return result(args[10], made);
  });
}

// init(KernelError, launched, rotary, attention, attention scratch, logits): the last four are addresses
PyObject* init(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  return guarded([&]() -> PyObject* {
    expect(nargs, 6, "init");
    void* p[4];
    for (int i = 0; i < 4; ++i) {
      p[i] = PyLong_AsVoidPtr(args[2 + i]);
      if (!p[i]) {
        if (PyErr_Occurred()) throw PythonError{};
        refuse("init: a launcher has no address");
      }
    }
    Py_INCREF(args[0]);
    Py_INCREF(args[1]);
    Py_XSETREF(g_error, args[0]);
    Py_XSETREF(g_launched, args[1]);
    g_rotary = reinterpret_cast<decltype(g_rotary)>(p[0]);
    g_attn = reinterpret_cast<decltype(g_attn)>(p[1]);
    g_attn_scratch = reinterpret_cast<decltype(g_attn_scratch)>(p[2]);
    g_logits = reinterpret_cast<decltype(g_logits)>(p[3]);
    Py_RETURN_NONE;
  });
}

#define FT_FN(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FT_FN(init), FT_FN(rotary), FT_FN(paged_append), FT_FN(paged_attention), FT_FN(logits_process), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_ft_decode", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__ft_decode(void) { return PyModule_Create(&module); }
