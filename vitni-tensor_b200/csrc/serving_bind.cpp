// serving_bind.cpp -- vtq._serving: the batched serving operators (include/vtq.h) on torch tensors, for
// vtq/serving.py. The checks of tensors, the current stream and the allocation of outputs and scratch are
// here rather than in Python, where they take 20 to 40 us a call: more than most of the kernels.
//
// Errors are C++ exceptions inside and Python exceptions (the package's classes, by status) at the border.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/core/grad_mode.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/full.h>
#include <ATen/ops/zeros.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <c10/util/SmallVector.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>
#include <initializer_list>
#include <limits>
#include <sstream>
#include <string>
#include <utility>

#include "../../include/vtq.h"

namespace {

struct Refused {
  vtq_status status;
  std::string text;
};

template <typename... A>
[[noreturn]] void refuse(vtq_status s, const A&... parts) {
  std::ostringstream o;
  (void)std::initializer_list<int>{(o << parts, 0)...};
  throw Refused{s, o.str()};
}

using at::ScalarType;
using Types = std::initializer_list<ScalarType>;
const Types kFloats = {ScalarType::Float, ScalarType::Half, ScalarType::BFloat16};
const Types kHalves = {ScalarType::Half, ScalarType::BFloat16};
const Types kInt = {ScalarType::Int};

int tag(ScalarType t) {
  return t == ScalarType::Float ? VTQ_F32 : t == ScalarType::Half ? VTQ_F16 : t == ScalarType::BFloat16 ? VTQ_BF16 : VTQ_I8;
}

bool given(PyObject* o) { return o != Py_None; }

// The tensor behind `o`: on `dev` (any CUDA device where that is null), of `dim` dimensions and one of
// `types`, contiguous in its last dimension. A size of -1 in `shape` is any.
const at::Tensor& want(const char* name, PyObject* o, int64_t dim, Types types, const at::Device* dev = nullptr,
                       std::initializer_list<int64_t> shape = {}) {
  if (!THPVariable_Check(o)) refuse(VTQ_ERR_INVALID_ARG, name, ": not a tensor");
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.is_cuda() || (dev && t.device() != *dev)) {
    if (dev) refuse(VTQ_ERR_INVALID_ARG, name, ": on ", t.device(), ", not on ", *dev);
    refuse(VTQ_ERR_INVALID_ARG, name, ": on ", t.device(), ", not on a CUDA device");
  }
  bool ok = false;
  for (ScalarType s : types) ok |= t.scalar_type() == s;
  if (!ok) refuse(VTQ_ERR_NOT_IMPLEMENTED, name, ": not implemented (", t.scalar_type(), ")");
  if (t.dim() != dim) refuse(VTQ_ERR_INTERNAL, name, ": ", t.dim(), " dimensions, not ", dim);
  int i = 0;
  for (int64_t n : shape) {
    if (n >= 0 && t.size(i) != n) refuse(VTQ_ERR_INTERNAL, name, ": size ", t.size(i), " in dimension ", i, ", not ", n);
    i++;
  }
  if (t.size(dim - 1) > 1 && t.stride(dim - 1) != 1) refuse(VTQ_ERR_INTERNAL, name, ": last dimension not contiguous");
  return t;
}

// The operators have no gradient: an input that asks for one would silently lose it.
const at::Tensor& constant(const char* name, const at::Tensor& t) {
  if (t.requires_grad() && at::GradMode::is_enabled())
    refuse(VTQ_ERR_NOT_IMPLEMENTED, name, ": not implemented (its gradient; call under torch.no_grad())");
  return t;
}

// From a tensor's first element's first byte to the last one's end.
int64_t extent(const at::Tensor& t) {
  const auto size = t.sizes(), stride = t.strides();
  int64_t n = 1;
  for (size_t i = 0; i < size.size(); i++) n += (size[i] - 1) * stride[i];
  return n * (int64_t)t.element_size();
}

// Where a tensor's elements lie, in bytes; dimensions of one element left out.
struct Span {
  uintptr_t base;
  int64_t elt;
  c10::SmallVector<std::pair<int64_t, int64_t>, 6> dims;  // (step, size)
  explicit Span(const at::Tensor& t) : base(reinterpret_cast<uintptr_t>(t.data_ptr())), elt((int64_t)t.element_size()) {
    const auto size = t.sizes(), stride = t.strides();
    for (size_t i = 0; i < size.size(); i++)
      if (size[i] > 1) dims.emplace_back(stride[i] * elt, size[i]);
  }
  // The bytes that its elements reach over when those of all steps that are multiples of `period` are laid upon another.
  int64_t within(int64_t period) const {
    int64_t n = elt;
    for (const auto& [step, size] : dims)
      if (step % period) n += (size - 1) * step;
    return n;
  }
};

// Whether two tensors whose extents overlap may have memory in common: no where they are slices of one layout, that is,
// for some step of theirs, lie in different places of each period of that step (the heads, values or tokens of one
// fused tensor).
bool may_share(const Span& a, const Span& b) {
  for (const Span* s : {&a, &b})
    for (const auto& dim : s->dims) {
      const int64_t period = dim.first;
      if (period <= 0) continue;
      const int64_t wa = a.within(period), wb = b.within(period), d = (int64_t)(b.base - a.base) % period, at = d < 0 ? d + period : d;
      if (wa <= at && at + wb <= period) return false;
    }
  return true;
}

// An output: its elements must not share memory. Each step has to pass what all smaller ones reach over.
const at::Tensor& distinct(const char* name, const at::Tensor& t) {
  constant(name, t);
  if (t.is_non_overlapping_and_dense() || !t.numel()) return t;
  Span a(t);
  std::sort(a.dims.begin(), a.dims.end());
  int64_t reach = a.elt;
  for (const auto& [step, size] : a.dims) {
    if (step < reach) refuse(VTQ_ERR_INTERNAL, name, ": written, but its elements share memory");
    reach += (size - 1) * step;
  }
  return t;
}

// An output that is written while `in` is still being read; `same`: unless it is all of it, element for element.
void apart(const char* name, const at::Tensor& t, const char* in_name, const at::Tensor& in, bool same = false) {
  if (!t.numel() || !in.numel()) return;
  const uintptr_t t0 = reinterpret_cast<uintptr_t>(t.data_ptr()), in0 = reinterpret_cast<uintptr_t>(in.data_ptr());
  if (t0 + extent(t) <= in0 || in0 + extent(in) <= t0) return;
  const Span a(t), b(in);
  if (same && a.base == b.base && a.dims == b.dims && t.scalar_type() == in.scalar_type()) return;
  if (may_share(a, b)) refuse(VTQ_ERR_INTERNAL, name, ": shares memory with ", in_name);
}

// What a call wrote into a tensor of the caller's raises its version, as torch's own in-place operations do.
void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
void written(PyObject* o) {
  if (given(o)) written(THPVariable_Unpack(o));
}

void* ptr(const at::Tensor& t) { return t.data_ptr(); }

uint32_t* status_of(PyObject* o, const at::Device& dev) {
  return given(o) ? static_cast<uint32_t*>(ptr(want("status", o, 1, kInt, &dev, {1}))) : nullptr;
}

void check(vtq_status s) {
  if (s != VTQ_OK) throw Refused{s, vtq_device_last_error()};
}

cudaStream_t stream_of(const at::Device& dev) { return c10::cuda::getCurrentCUDAStream(dev.index()).stream(); }

at::Tensor scratch(size_t bytes, const at::Device& dev) {
  return at::empty({(int64_t)bytes}, at::TensorOptions().dtype(at::kByte).device(dev));
}

PyObject* g_errors = nullptr;  // {status: exception class}

// Runs `body` with the border's exceptions: the package's for refusals, torch's for its own failures.
template <typename F>
PyObject* border(F body) {
  try {
    return body();
  } catch (const Refused& r) {
    PyObject* key = PyLong_FromLong(r.status);
    PyObject* cls = key && g_errors ? PyDict_GetItem(g_errors, key) : nullptr;
    Py_XDECREF(key);
    PyErr_SetString(cls ? cls : PyExc_RuntimeError, r.text.c_str());
  } catch (const c10::OutOfMemoryError& e) {
    PyErr_SetString(PyExc_MemoryError, e.what_without_backtrace());
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

PyObject* wrap(const at::Tensor& t) { return THPVariable_Wrap(t); }
PyObject* pair(const at::Tensor& a, const at::Tensor& b) {
  PyObject *x = wrap(a), *y = wrap(b), *r = x && y ? PyTuple_Pack(2, x, y) : nullptr;
  Py_XDECREF(x);
  Py_XDECREF(y);
  return r;
}

#define ARGS(n) \
  if (nargs != n) refuse(VTQ_ERR_INVALID_ARG, "vtq._serving: ", nargs, " arguments, not ", n)

// (x, q, scale)
PyObject* quantize_tokens(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  return border([&]() -> PyObject* {
    ARGS(3);
    const at::Tensor& x = want("x", a[0], 2, kFloats);
    const at::Device dev = x.device();
    const c10::cuda::CUDAGuard guard(dev);
    const int64_t t = x.size(0), n = x.size(1);
    at::Tensor q = given(a[1]) ? distinct("q", want("q", a[1], 2, {ScalarType::Char}, &dev, {t, n}))
                               : at::empty({t, std::max<int64_t>(16, (n + 15) / 16 * 16)}, x.options().dtype(at::kChar)).narrow(1, 0, n);
    at::Tensor s = given(a[2]) ? distinct("scale", want("scale", a[2], 1, {ScalarType::Float}, &dev, {t}))
                               : at::empty({t}, x.options().dtype(at::kFloat));
    if (given(a[1])) apart("q", q, "x", x);
    if (given(a[2])) apart("scale", s, "x", x);
    if (given(a[1]) && given(a[2])) apart("scale", s, "q", q);
    const int64_t ldq = t > 1 ? q.stride(0) : std::max(n, q.stride(0));
    check(vtq_quantize_tokens(tag(x.scalar_type()), ptr(x), x.stride(0), t, n, static_cast<int8_t*>(ptr(q)), ldq,
                              static_cast<float*>(ptr(s)), stream_of(dev)));
    written(a[1]), written(a[2]);
    return pair(q, s);
  });
}

// (x, w, w_scale, bias, out_dtype, x_scale, out, status); w and w_scale were checked when they were laid out
PyObject* linear_i8(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  return border([&]() -> PyObject* {
    ARGS(8);
    const at::Tensor& w = want("w", a[1], 2, {ScalarType::Char});
    const at::Device dev = w.device();
    const int64_t in = w.size(1), n = w.size(0);
    const at::Tensor& ws = want("w_scale", a[2], 1, {ScalarType::Float}, &dev, {n});
    const bool codes = given(a[5]);
    const at::Tensor& x = codes ? want("x", a[0], 2, {ScalarType::Char}, &dev, {-1, in}) : want("x", a[0], 2, kFloats, &dev, {-1, in});
    constant("x", x);
    const c10::cuda::CUDAGuard guard(dev);
    const int64_t t = x.size(0);
    ScalarType type = codes ? ScalarType::Float : x.scalar_type();
    if (given(a[4])) {
      if (!THPDtype_Check(a[4])) refuse(VTQ_ERR_INVALID_ARG, "out_dtype: not a dtype");
      type = reinterpret_cast<THPDtype*>(a[4])->scalar_type;
      if (tag(type) == VTQ_I8) refuse(VTQ_ERR_NOT_IMPLEMENTED, "out_dtype: not implemented (", type, ")");
    }
    at::Tensor out;
    if (given(a[6])) {
      out = distinct("out", want("out", a[6], 2, kFloats, &dev, {t, n}));
      if (given(a[4]) && out.scalar_type() != type) refuse(VTQ_ERR_INTERNAL, "out: not of out_dtype");
    } else {
      out = at::empty({t, n}, x.options().dtype(type));
    }
    vtq_linear_i8_args g = {};
    // (Floating x may be written over: its codes are made before anything of out is.)
    auto read = [&](const char* name, const at::Tensor& r) {
      if (given(a[6])) apart("out", out, name, r);
      return ptr(r);
    };
    g.x = codes ? read("x", x) : ptr(x);
    if (codes) g.x_scale = static_cast<const float*>(read("x_scale", constant("x_scale", want("x_scale", a[5], 1, {ScalarType::Float}, &dev, {t}))));
    g.w = static_cast<const int8_t*>(read("w", w));
    g.w_scale = static_cast<const float*>(read("w_scale", constant("w_scale", ws)));
    if (given(a[3])) g.bias = static_cast<const float*>(read("bias", constant("bias", want("bias", a[3], 1, {ScalarType::Float}, &dev, {n}))));
    g.y = ptr(out);
    g.ldx = x.stride(0);
    g.ldw = w.stride(0);
    g.ldy = out.stride(0);
    g.tokens = t;
    g.in_feat = in;
    g.out_feat = n;
    g.x_dtype = codes ? VTQ_I8 : tag(x.scalar_type());
    g.y_dtype = tag(out.scalar_type());
    g.status = status_of(a[7], dev);
    const size_t need = vtq_linear_i8_workspace_bytes(g.x_dtype, t, in, n);
    at::Tensor s;
    if (need) s = scratch(need, dev);
    check(vtq_linear_i8(&g, need ? ptr(s) : nullptr, need, stream_of(dev)));
    written(a[6]), written(a[7]);
    return wrap(out);
  });
}

vtq_paged_kv paged(PyObject* k_pages, PyObject* v_pages, PyObject* table, at::Device& dev) {
  const at::Tensor& k = want("k_pages", k_pages, 4, kHalves);
  dev = k.device();
  const at::Tensor& v = want("v_pages", v_pages, 4, {k.scalar_type()}, &dev, {k.size(0), k.size(1), k.size(2), k.size(3)});
  const at::Tensor& t = want("page_table", table, 2, kInt, &dev);
  constant("k_pages", k), constant("v_pages", v);
  vtq_paged_kv kv = {};
  kv.k = ptr(k);
  kv.v = ptr(v);
  kv.k_page = k.stride(0), kv.k_slot = k.stride(1), kv.k_head = k.stride(2);
  kv.v_page = v.stride(0), kv.v_slot = v.stride(1), kv.v_head = v.stride(2);
  kv.table = static_cast<const int32_t*>(ptr(t));
  kv.table_ld = t.stride(0);
  kv.table_width = t.size(1);
  kv.seqs = t.size(0);
  kv.pages = k.size(0), kv.page_size = k.size(1), kv.kv_heads = k.size(2), kv.head_dim = k.size(3);
  kv.dtype = tag(k.scalar_type());
  return kv;
}

// (k, v, k_pages, v_pages, table, seq, pos, rope table, half, q, q_out, status)
PyObject* append_kv(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  return border([&]() -> PyObject* {
    ARGS(12);
    at::Device dev(at::kCPU);
    vtq_append_kv_args g = {};
    g.kv = paged(a[2], a[3], a[4], dev);
    const c10::cuda::CUDAGuard guard(dev);
    distinct("k_pages", THPVariable_Unpack(a[2]));
    distinct("v_pages", THPVariable_Unpack(a[3]));
    apart("v_pages", THPVariable_Unpack(a[3]), "k_pages", THPVariable_Unpack(a[2]));
    const at::Tensor& k = want("k", a[0], 3, kFloats, &dev, {-1, g.kv.kv_heads, g.kv.head_dim});
    const int64_t t = k.size(0);
    const at::Tensor& v = want("v", a[1], 3, {k.scalar_type()}, &dev, {t, g.kv.kv_heads, g.kv.head_dim});
    constant("k", k), constant("v", v);
    g.k = ptr(k), g.k_tok = k.stride(0), g.k_head = k.stride(1);
    g.v = ptr(v), g.v_tok = v.stride(0), g.v_head = v.stride(1);
    g.seq = static_cast<const int32_t*>(ptr(want("seq", a[5], 1, kInt, &dev, {t})));
    g.pos = static_cast<const int32_t*>(ptr(want("pos", a[6], 1, kInt, &dev, {t})));
    if (given(a[7])) {
      const at::Tensor& r = want("rope", a[7], 3, {ScalarType::Float}, &dev, {-1, -1, 2});
      if (!r.is_contiguous()) refuse(VTQ_ERR_INTERNAL, "rope: table not contiguous");
      g.rope = static_cast<const float*>(ptr(r));
      g.max_pos = r.size(0);
      g.rot_dim = 2 * r.size(1);
      if (PyObject_IsTrue(a[8])) g.flags |= VTQ_ROPE_HALF;
    }
    at::Tensor out;
    if (given(a[9])) {
      const at::Tensor& q = constant("q", want("q", a[9], 3, {k.scalar_type()}, &dev, {t, -1, g.kv.head_dim}));
      const ScalarType c = THPVariable_Unpack(a[2]).scalar_type();
      out = given(a[10]) ? distinct("q_out", want("q_out", a[10], 3, {c}, &dev, {t, q.size(1), g.kv.head_dim}))
                         : at::zeros(q.sizes(), q.options().dtype(c));
      if (given(a[10])) {
        apart("q_out", out, "q", q, true);
        apart("q_out", out, "k", k);
        apart("q_out", out, "v", v);
      }
      if (q.size(1) > 0) {
        g.q = ptr(q), g.q_tok = q.stride(0), g.q_head = q.stride(1), g.heads = q.size(1);
        g.q_out = ptr(out), g.qo_tok = out.stride(0), g.qo_head = out.stride(1);
      }
    } else if (given(a[10])) {
      refuse(VTQ_ERR_INTERNAL, "q_out: given without q");
    }
    g.tokens = t;
    g.x_dtype = tag(k.scalar_type());
    g.status = status_of(a[11], dev);
    check(vtq_append_kv(&g, stream_of(dev)));
    written(a[2]), written(a[3]), written(a[10]), written(a[11]);
    if (!out.defined()) Py_RETURN_NONE;
    return wrap(out);
  });
}

// (q, k_pages, v_pages, table, kv_len, q_start, shared_len, scale, out, with lse, status)
PyObject* attention_paged(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  return border([&]() -> PyObject* {
    ARGS(11);
    at::Device dev(at::kCPU);
    vtq_attention_args g = {};
    g.kv = paged(a[1], a[2], a[3], dev);
    const c10::cuda::CUDAGuard guard(dev);
    const ScalarType type = THPVariable_Unpack(a[1]).scalar_type();
    const at::Tensor& q = constant("q", want("q", a[0], 3, {type}, &dev, {-1, -1, g.kv.head_dim}));
    const int64_t t = q.size(0), heads = q.size(1);
    g.kv_len = static_cast<const int32_t*>(ptr(want("kv_len", a[4], 1, kInt, &dev, {g.kv.seqs})));
    const bool starts = given(a[5]);
    if (starts) g.q_start = static_cast<const int32_t*>(ptr(want("q_start", a[5], 1, kInt, &dev, {g.kv.seqs + 1})));
    else if (t < g.kv.seqs) refuse(VTQ_ERR_INTERNAL, "q: fewer rows than sequences");
    g.shared_len = PyLong_AsLongLong(a[6]);
    if (g.shared_len == -1 && PyErr_Occurred()) return nullptr;
    g.scale = given(a[7]) ? (float)PyFloat_AsDouble(a[7]) : 1.0f / std::sqrt((float)g.kv.head_dim);
    if (given(a[7]) && PyErr_Occurred()) return nullptr;
    at::Tensor out, lse;
    // Rows that no sequence owns: left alone in the caller's out, zeros (and -inf) in what is allocated here.
    if (given(a[8])) {
      out = distinct("out", want("out", a[8], 3, {type}, &dev, {t, heads, g.kv.head_dim}));
      apart("out", out, "q", q);
    } else {
      out = g.kv.seqs ? at::empty(q.sizes(), q.options()) : at::zeros(q.sizes(), q.options());
      g.clear |= 1;
    }
    if (PyObject_IsTrue(a[9])) {
      g.clear |= 2;
      lse = g.kv.seqs ? at::empty({t, heads}, q.options().dtype(at::kFloat))
                      : at::full({t, heads}, -std::numeric_limits<float>::infinity(), q.options().dtype(at::kFloat));
      g.lse = static_cast<float*>(ptr(lse));
    }
    g.q = ptr(q), g.q_tok = q.stride(0), g.q_head = q.stride(1);
    g.out = ptr(out), g.o_tok = out.stride(0), g.o_head = out.stride(1);
    g.lse_tok = heads;
    g.tokens = t;
    g.heads = heads;
    g.status = status_of(a[10], dev);
    const size_t need = vtq_attention_paged_workspace_bytes(&g);
    at::Tensor s;
    if (need) s = scratch(need, dev);
    check(vtq_attention_paged(&g, need ? ptr(s) : nullptr, need, stream_of(dev)));
    written(a[8]), written(a[10]);
    return lse.defined() ? pair(out, lse) : wrap(out);
  });
}

// (greedy, draft, target, proposal, u, n_draft)
PyObject* verify(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  return border([&]() -> PyObject* {
    ARGS(6);
    const bool greedy = PyObject_IsTrue(a[0]);
    const at::Tensor& d = want("draft", a[1], 2, kInt);
    const at::Device dev = d.device();
    const c10::cuda::CUDAGuard guard(dev);
    const int64_t b = d.size(0), k = d.size(1);
    const at::Tensor& p = want("target", a[2], 3, kFloats, &dev, {b, k + 1});
    vtq_verify_args g = {};
    g.draft = static_cast<const int32_t*>(ptr(d));
    g.target = ptr(p), g.target_seq = p.stride(0), g.target_row = p.stride(1);
    g.vocab = p.size(2);
    if (given(a[3])) {
      const at::Tensor& q = want("proposal", a[3], 3, {p.scalar_type()}, &dev, {b, k, g.vocab});
      g.proposal = ptr(q), g.proposal_seq = q.stride(0), g.proposal_row = q.stride(1);
    }
    if (given(a[4])) {
      const at::Tensor& u = want("u", a[4], 2, {ScalarType::Float}, &dev, {b, k + 1});
      g.u = static_cast<const float*>(ptr(u)), g.ld_u = u.stride(0);
    }
    if (given(a[5])) g.n_draft = static_cast<const int32_t*>(ptr(want("n_draft", a[5], 1, kInt, &dev, {b})));
    at::Tensor tokens = at::empty({b, k + 1}, d.options()), accepted = at::empty({b}, d.options());
    g.tokens = static_cast<int32_t*>(ptr(tokens));
    g.accepted = static_cast<int32_t*>(ptr(accepted));
    g.ld_draft = d.stride(0);
    g.ld_tokens = k + 1;
    g.seqs = b, g.drafts = k;
    g.dtype = tag(p.scalar_type());
    check((greedy ? vtq_verify_greedy : vtq_verify_draft)(&g, stream_of(dev)));
    return pair(tokens, accepted);
  });
}

// ({status: exception class})
PyObject* set_errors(PyObject*, PyObject* errors) {
  Py_INCREF(errors);
  Py_XSETREF(g_errors, errors);
  Py_RETURN_NONE;
}

#define FAST(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FAST(quantize_tokens), FAST(linear_i8), FAST(append_kv), FAST(attention_paged), FAST(verify),
                         {"set_errors", set_errors, METH_O, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_serving", "torch binding of the batched serving operators", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__serving(void) { return PyModule_Create(&module); }
