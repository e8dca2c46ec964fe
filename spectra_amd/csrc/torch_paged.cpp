// The paged KV cache's operators as registered PyTorch operators: torch.ops.spectra_hip.
// paged_rope_append and paged_attend (no counterpart in the reference).
//
// One call each: the checks of shapes, types, strides and devices, the descriptor, the output from
// the caching allocator and the launch on the current HIP stream of the operands' device.  A
// single-token step is launch-bound: the same checks in Python with a ctypes call took 18 us, three
// times the kernel.  Bad arguments raise ValueError; other failures RuntimeError naming the status.
//
// The library is a Python module, too, whose two functions take the same arguments and go past the
// dispatcher (some 2 us a call for this many arguments) where it would only have passed them on:
// plain tensors that nothing is differentiated by, and no mode that wants to see operators.  Otherwise they return
// NotImplemented, and the caller takes the registered operator, which a compiler traces and whose result says, when a
// gradient is asked of it, that there is none.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <c10/hip/HIPStream.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/library.h>

#include <algorithm>
#include <cmath>
#include <vector>

#include "spectra_hip.h"

namespace {

using OptTensor = c10::optional<at::Tensor>;

void check_paged(const char* fn, int st) {
  if (st == SPECTRA_OK) return;
  TORCH_CHECK_VALUE(st != SPECTRA_ERR_INVALID, fn, ": ", spectra_last_error());
  TORCH_CHECK(false, fn, " failed (", st, "): ", spectra_last_error());
}

bool rank1(const at::Tensor& t, at::ScalarType dtype, int64_t n, const at::Device& dev) {
  return t.scalar_type() == dtype && t.dim() == 1 && t.size(0) == n && (n < 2 || t.stride(0) == 1) && t.device() == dev;
}

// Checks a paged cache and its batch for activations x of `heads` query heads and describes it.
spectra_paged_kv_t describe_paged(const at::Tensor& x, int64_t heads, const at::Tensor& kv_lens, const at::Tensor& q_start,
                                  const at::Tensor& block_table, at::TensorList k, at::TensorList v) {
  const bool q4 = k.size() == 3;
  TORCH_CHECK_VALUE((k.size() == 1 || q4) && v.size() == k.size() && k[0].dim() == 4,
                    "k_pages and v_pages must be [pages, kv_heads, page, d], or (codes, scales, zeros) of that");
  const auto dtype = x.scalar_type();
  TORCH_CHECK_VALUE(dtype == at::kHalf || (dtype == at::kBFloat16 && !q4),
                    "activations must be fp16 (or bf16, on bf16 pages), got ", dtype);
  const auto dev = x.device();
  const int64_t pages = k[0].size(0), kv = k[0].size(1), page = k[0].size(2), d = k[0].size(3) * (q4 ? 2 : 1);
  const at::ScalarType types[3] = {q4 ? at::kByte : dtype, at::kHalf, at::kByte};
  const int64_t last[3] = {k[0].size(3), d / 32, d / 32};
  for (size_t i = 0; i < k.size(); ++i)
    for (const at::Tensor* t : {&k[i], &v[i]}) {
      const auto s = t->sizes();
      TORCH_CHECK_VALUE(t->scalar_type() == types[i] && s.size() == 4 && s[0] == pages && s[1] == kv && s[2] == page &&
                            s[3] == last[i] && t->device() == dev,
                        "pages of head size ", d, " must be ", types[i], " [", pages, ", ", kv, ", ", page, ", ", last[i],
                        "] on ", dev, ", got ", t->scalar_type(), " ", s, " on ", t->device());
      const auto st = t->strides();
      TORCH_CHECK_VALUE(st[3] == 1 && st[2] == last[i] && (kv == 1 || st[1] == page * last[i]) &&
                            (pages < 2 || st[0] == k[i].stride(0)),
                        "a page must be contiguous, and k and v equally far from page to page");
    }
  TORCH_CHECK_VALUE(pages > 0 && kv > 0, "the pool has no pages");
  TORCH_CHECK_VALUE(heads > 0 && heads % kv == 0, "heads (", heads, ") must be a multiple of the pages' ", kv, " KV heads");
  const int64_t batch = kv_lens.dim() == 1 ? kv_lens.size(0) : -1;
  TORCH_CHECK_VALUE(batch >= 0 && rank1(kv_lens, at::kInt, batch, dev), "kv_lens must be contiguous int32 [batch] on ", dev);
  TORCH_CHECK_VALUE(rank1(q_start, at::kInt, batch + 1, dev), "q_start must be contiguous int32 [batch + 1 = ", batch + 1,
                    "] on ", dev, ": ", batch, " sequences need that");
  TORCH_CHECK_VALUE(block_table.scalar_type() == at::kInt && block_table.dim() == 2 && block_table.size(0) == batch &&
                        (block_table.size(1) < 2 || block_table.stride(1) == 1) && block_table.device() == dev,
                    "block_table must be int32 [", batch, ", pages a sequence] with contiguous rows on ", dev);
  spectra_paged_kv_t p{};
  p.kind = q4 ? SPECTRA_KV_4BIT : dtype == at::kBFloat16 ? SPECTRA_KV_BF16 : SPECTRA_KV_F16;
  p.kv_heads = (int32_t)kv;
  p.head_dim = (int32_t)d;
  TORCH_CHECK_VALUE(page <= 65536 && kv <= 65536 && d <= 65536 && heads <= (1 << 20) && batch <= (1 << 20) &&
                        block_table.size(1) <= (1 << 30),
                    "sizes out of range");
  p.page_size = (int32_t)page;
  p.num_pages = pages;
  p.k = k[0].data_ptr();
  p.v = v[0].data_ptr();
  p.page_stride = k[0].stride(0);
  if (q4) {
    p.k_scales = k[1].data_ptr();
    p.v_scales = v[1].data_ptr();
    p.scale_stride = k[1].stride(0);
    p.k_zeros = k[2].data_ptr();
    p.v_zeros = v[2].data_ptr();
    p.zero_stride = k[2].stride(0);
  }
  p.batch = (int32_t)batch;
  p.table_width = (int32_t)block_table.size(1);
  p.block_table = static_cast<const int32_t*>(block_table.data_ptr());
  p.table_stride = block_table.stride(0);
  p.kv_lens = static_cast<const int32_t*>(kv_lens.data_ptr());
  p.q_start = static_cast<const int32_t*>(q_start.data_ptr());
  return p;
}

void check_out(const at::Tensor& out, const at::Tensor& x, int64_t tokens, int64_t heads, int64_t d, const char* name) {
  TORCH_CHECK_VALUE(out.scalar_type() == x.scalar_type() && out.dim() == 3 && out.size(0) == tokens &&
                        out.size(1) == heads && out.size(2) == d && out.is_contiguous() && out.device() == x.device(),
                    name, " must be contiguous ", x.scalar_type(), " [", tokens, ", ", heads, ", ", d, "] on ", x.device());
}

// ---- append ----
at::Tensor append(const at::Tensor& qkv_in, const at::Tensor& kv_lens, const at::Tensor& q_start,
                  const at::Tensor& block_table, const OptTensor& cos, const OptTensor& sin, int64_t heads, at::TensorList k,
                  at::TensorList v, const at::Tensor* q_out) {
  at::Tensor qkv = qkv_in;
  TORCH_CHECK_VALUE(qkv.dim() == 2, "qkv must be [T, (heads + 2 kv) * d]");
  const spectra_paged_kv_t p = describe_paged(qkv, heads, kv_lens, q_start, block_table, k, v);
  const int64_t tokens = qkv.size(0), d = p.head_dim, width = (heads + 2 * p.kv_heads) * d;
  TORCH_CHECK_VALUE(qkv.size(1) == width, "qkv rows must hold (heads + 2 kv) * d = ", width, " values, got ", qkv.size(1));
  TORCH_CHECK_VALUE(cos.has_value() == sin.has_value(), "cos and sin must both be given or both be None");
  if (cos.has_value())
    for (const at::Tensor* t : {&*cos, &*sin})
      TORCH_CHECK_VALUE(t->scalar_type() == at::kFloat && t->dim() == 2 && t->size(0) == cos->size(0) &&
                            t->size(0) > 0 && t->size(1) == d / 2 && t->is_contiguous() && t->device() == qkv.device(),
                        "cos and sin must be contiguous fp32 [rows, d / 2], at least a row, on ", qkv.device());
  const c10::DeviceGuard guard(qkv.device());
  // rows are read 16 bytes at a time
  if (qkv.stride(1) != 1 || (tokens > 1 && (qkv.stride(0) < width || qkv.stride(0) % 8 != 0)) ||
      reinterpret_cast<uintptr_t>(qkv.data_ptr()) % 16 != 0)
    qkv = qkv.clone(at::MemoryFormat::Contiguous);
  at::Tensor q;
  if (q_out != nullptr) {
    check_out(*q_out, qkv, tokens, heads, d, "q_out");
    q = *q_out;
  } else {
    q = at::detail::empty_cuda({tokens, heads, d}, qkv.scalar_type(), qkv.device(), c10::nullopt);
  }
  if (tokens == 0) return q;
  check_paged("spectra_paged_rope_append",
              spectra_paged_rope_append(
                  &p, qkv.data_ptr(), tokens > 1 ? qkv.stride(0) : width, tokens,
                  cos.has_value() ? static_cast<const float*>(cos->data_ptr()) : nullptr,
                  sin.has_value() ? static_cast<const float*>(sin->data_ptr()) : nullptr,
                  cos.has_value() ? cos->size(0) : 0, (int32_t)heads, q.data_ptr(),
                  c10::hip::getCurrentHIPStream(qkv.device().index()).stream()));
  return q;
}

at::Tensor paged_rope_append(const at::Tensor& qkv, const at::Tensor& kv_lens, const at::Tensor& q_start,
                             const at::Tensor& block_table, const OptTensor& cos, const OptTensor& sin, int64_t heads,
                             at::TensorList k, at::TensorList v) {
  return append(qkv, kv_lens, q_start, block_table, cos, sin, heads, k, v, nullptr);
}
void paged_rope_append_out(const at::Tensor& qkv, const at::Tensor& kv_lens, const at::Tensor& q_start,
                           const at::Tensor& block_table, const OptTensor& cos, const OptTensor& sin, int64_t heads,
                           at::TensorList k, at::TensorList v, const at::Tensor& q_out) {
  append(qkv, kv_lens, q_start, block_table, cos, sin, heads, k, v, &q_out);
}
// What the results' shapes are made of, for a call without memory.
void check_meta(const at::Tensor& x, int64_t dims, at::TensorList k, at::TensorList v) {
  TORCH_CHECK_VALUE(x.dim() == dims && (k.size() == 1 || k.size() == 3) && v.size() == k.size() && k[0].dim() == 4,
                    "k_pages and v_pages must be [pages, kv_heads, page, d], or (codes, scales, zeros) of that, for ", dims,
                    "-dimensional activations");
}
at::Tensor paged_rope_append_meta(const at::Tensor& qkv, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                                  const OptTensor&, const OptTensor&, int64_t heads, at::TensorList k, at::TensorList v) {
  check_meta(qkv, 2, k, v);
  return at::empty_symint({qkv.sym_size(0), heads, k[0].sym_size(3) * (k.size() == 3 ? 2 : 1)}, qkv.options());
}
void paged_rope_append_out_meta(const at::Tensor& qkv, const at::Tensor&, const at::Tensor&, const at::Tensor&, const OptTensor&,
                                const OptTensor&, int64_t, at::TensorList k, at::TensorList v, const at::Tensor&) {
  check_meta(qkv, 2, k, v);
}

// ---- attention ----
at::Tensor attend(const at::Tensor& q_in, const at::Tensor& kv_lens, const at::Tensor& q_start,
                  const at::Tensor& block_table, at::TensorList k, at::TensorList v, double scale, double cap, int64_t window,
                  const OptTensor& slopes, const OptTensor& prefix, const OptTensor& workspace, const at::Tensor* out_in) {
  at::Tensor q = q_in;
  TORCH_CHECK_VALUE(q.dim() == 3, "q must be [T, heads, d]");
  const int64_t tokens = q.size(0), heads = q.size(1), d = q.size(2);
  const spectra_paged_kv_t p = describe_paged(q, heads, kv_lens, q_start, block_table, k, v);
  TORCH_CHECK_VALUE(d == p.head_dim, "q has head size ", d, ", the pages ", p.head_dim);
  const auto dev = q.device();
  TORCH_CHECK_VALUE(!slopes.has_value() || rank1(*slopes, at::kFloat, heads, dev), "slopes must be contiguous fp32 [", heads,
                    "] on ", dev);
  TORCH_CHECK_VALUE(!prefix.has_value() || rank1(*prefix, at::kInt, p.batch, dev), "prefix must be contiguous int32 [",
                    p.batch, "] on ", dev);
  TORCH_CHECK_VALUE(!workspace.has_value() || (workspace->is_contiguous() && workspace->device() == dev),
                    "workspace must be contiguous on ", dev);
  TORCH_CHECK_VALUE(window >= 0 && cap >= 0.0 && scale > 0.0,
                    "scale must be positive, cap and window 0 (none) or positive, got ", scale, ", ", cap, ", ", window);
  const c10::DeviceGuard guard(dev);
  if (q.stride(2) != 1 || (heads > 1 && q.stride(1) != d) || reinterpret_cast<uintptr_t>(q.data_ptr()) % 16 != 0 ||
      (tokens > 1 && (q.stride(0) % 8 != 0 || q.stride(0) < heads * d)))
    q = q.clone(at::MemoryFormat::Contiguous);
  at::Tensor out;
  if (out_in != nullptr) {
    check_out(*out_in, q, tokens, heads, d, "out");
    out = *out_in;
  } else {
    out = at::detail::empty_cuda({tokens, heads, d}, q.scalar_type(), dev, c10::nullopt);
  }
  if (tokens == 0) return out;
  at::Tensor ws;
  if (workspace.has_value()) {
    ws = *workspace;
  } else {
    ws = at::detail::empty_cuda({(int64_t)spectra_paged_attend_workspace((int32_t)d)}, at::kByte, dev, c10::nullopt);
    if (ws.numel() > 0) ws.narrow(0, 0, SPECTRA_PAGED_COUNTER_BYTES).zero_();
  }
  check_paged("spectra_paged_attend",
              spectra_paged_attend(&p, q.data_ptr(), tokens > 1 ? q.stride(0) : heads * d, tokens, (int32_t)heads,
                                   (float)scale, (float)cap, (int32_t)std::min<int64_t>(window, 1 << 30),
                                   slopes.has_value() ? static_cast<const float*>(slopes->data_ptr()) : nullptr,
                                   prefix.has_value() ? static_cast<const int32_t*>(prefix->data_ptr()) : nullptr,
                                   ws.data_ptr(), (size_t)ws.numel() * ws.element_size(), out.data_ptr(),
                                   c10::hip::getCurrentHIPStream(dev.index()).stream()));
  return out;
}

at::Tensor paged_attend(const at::Tensor& q, const at::Tensor& kv_lens, const at::Tensor& q_start,
                        const at::Tensor& block_table, at::TensorList k, at::TensorList v, double scale, double cap,
                        int64_t window, const OptTensor& slopes, const OptTensor& prefix, const OptTensor& workspace) {
  return attend(q, kv_lens, q_start, block_table, k, v, scale, cap, window, slopes, prefix, workspace, nullptr);
}
void paged_attend_out(const at::Tensor& q, const at::Tensor& kv_lens, const at::Tensor& q_start,
                      const at::Tensor& block_table, at::TensorList k, at::TensorList v, double scale, double cap,
                      int64_t window, const OptTensor& slopes, const OptTensor& prefix, const OptTensor& workspace,
                      const at::Tensor& out) {
  attend(q, kv_lens, q_start, block_table, k, v, scale, cap, window, slopes, prefix, workspace, &out);
}
at::Tensor paged_attend_meta(const at::Tensor& q, const at::Tensor&, const at::Tensor&, const at::Tensor&, at::TensorList k,
                             at::TensorList v, double, double, int64_t, const OptTensor&, const OptTensor&,
                             const OptTensor&) {
  check_meta(q, 3, k, v);
  return at::empty_symint(q.sym_sizes(), q.options());
}
void paged_attend_out_meta(const at::Tensor& q, const at::Tensor&, const at::Tensor&, const at::Tensor&, at::TensorList k,
                           at::TensorList v, double, double, int64_t, const OptTensor&, const OptTensor&, const OptTensor&,
                           const at::Tensor&) {
  check_meta(q, 3, k, v);
}

// ---- the Python functions ----

// A tensor of a device that the dispatcher would do nothing about.
bool plain_tensor(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return false;
  const at::Tensor& t = THPVariable_Unpack(o);
  static const c10::DispatchKeySet views({c10::DispatchKey::Negative, c10::DispatchKey::Conjugate, c10::DispatchKey::ZeroTensor,
                                          c10::DispatchKey::Functionalize, c10::DispatchKey::Python});
  if (!t.is_cuda() || t.key_set().has_any(views)) return false;
  return t.unsafeGetTensorImpl()->autograd_meta() == nullptr ||
         (!(t.requires_grad() && c10::GradMode::is_enabled()) && !t._fw_grad(/*level=*/0).defined());
}

struct Arguments {
  PyObject* const* a;
  bool plain = true;  // nothing but plain tensors where tensors belong

  const at::Tensor* tensor(int i) {
    plain = plain && plain_tensor(a[i]);
    return plain ? &THPVariable_Unpack(a[i]) : nullptr;
  }
  OptTensor optional(int i) {
    if (a[i] == Py_None) return c10::nullopt;
    const at::Tensor* t = tensor(i);
    return t != nullptr ? OptTensor(*t) : c10::nullopt;
  }
  std::vector<at::Tensor> list(int i) {  // a tensor, or a tuple or list of them
    std::vector<at::Tensor> r;
    if (THPVariable_Check(a[i])) {
      if (const at::Tensor* t = tensor(i)) r.push_back(*t);
      return r;
    }
    if (!(plain = plain && (PyTuple_Check(a[i]) || PyList_Check(a[i])))) return r;
    PyObject** items = PySequence_Fast_ITEMS(a[i]);
    for (Py_ssize_t j = 0; j < PySequence_Fast_GET_SIZE(a[i]) && plain; ++j) {
      plain = plain_tensor(items[j]);
      if (plain) r.push_back(THPVariable_Unpack(items[j]));
    }
    plain = plain && !r.empty();
    return r;
  }
  double number(int i) {
    const bool is = PyFloat_Check(a[i]) || PyLong_Check(a[i]);
    const double v = is ? PyFloat_AsDouble(a[i]) : 0.0;
    return whole(is, v);
  }
  int64_t integer(int i) {
    const bool is = PyLong_Check(a[i]);
    return whole(is, is ? (int64_t)PyLong_AsLongLong(a[i]) : 0);
  }

 private:
  template <typename T>
  T whole(bool is, T v) {
    if (PyErr_Occurred() != nullptr) {  // (out of range: the operator says so)
      PyErr_Clear();
      is = false;
    }
    plain = plain && is;
    return v;
  }
};

// Something else wants to see the operators: a mode, or a key that the thread includes.
bool dispatched() {
  return c10::impl::TorchDispatchModeTLS::any_modes_set() ||
         !(c10::impl::tls_local_dispatch_key_set().included_ - c10::default_included_set).empty();
}

PyObject* py_append(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 10, "paged_rope_append takes 10 arguments");
  Arguments a{args};
  const at::Tensor *qkv = a.tensor(0), *lens = a.tensor(1), *starts = a.tensor(2), *table = a.tensor(3);
  const OptTensor cos = a.optional(4), sin = a.optional(5), out = a.optional(9);
  const int64_t heads = a.integer(6);
  const std::vector<at::Tensor> k = a.list(7), v = a.list(8);
  if (!a.plain || dispatched()) Py_RETURN_NOTIMPLEMENTED;
  at::Tensor q;
  {
    pybind11::gil_scoped_release release;
    q = append(*qkv, *lens, *starts, *table, cos, sin, heads, k, v, out.has_value() ? &*out : nullptr);
  }
  return THPVariable_Wrap(q);
  END_HANDLE_TH_ERRORS
}

PyObject* py_attend(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 13, "paged_attend takes 13 arguments");
  Arguments a{args};
  const at::Tensor *q = a.tensor(0), *lens = a.tensor(1), *starts = a.tensor(2), *table = a.tensor(3);
  const std::vector<at::Tensor> k = a.list(4), v = a.list(5);
  const bool usual = args[6] == Py_None;  // 1 / sqrt(d)
  double scale = usual ? 1.0 : a.number(6);
  const double cap = a.number(7);
  const int64_t window = a.integer(8);
  const OptTensor slopes = a.optional(9), prefix = a.optional(10), workspace = a.optional(11), out = a.optional(12);
  if (!a.plain || dispatched()) Py_RETURN_NOTIMPLEMENTED;
  if (usual && q->dim() == 3) scale = 1.0 / std::sqrt((double)q->size(2));
  at::Tensor o;
  {
    pybind11::gil_scoped_release release;
    o = attend(*q, *lens, *starts, *table, k, v, scale, cap, window, slopes, prefix, workspace, out.has_value() ? &*out : nullptr);
  }
  return THPVariable_Wrap(o);
  END_HANDLE_TH_ERRORS
}

PyMethodDef kMethods[] = {
    {"paged_rope_append", (PyCFunction)(void*)py_append, METH_FASTCALL, nullptr},
    {"paged_attend", (PyCFunction)(void*)py_attend, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_spectra_torch", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__spectra_torch(void) { return PyModule_Create(&kModule); }

TORCH_LIBRARY_FRAGMENT(spectra_hip, m) {
  m.def(
      "paged_rope_append(Tensor qkv, Tensor kv_lens, Tensor q_start, Tensor block_table, Tensor? cos, Tensor? sin, "
      "int heads, Tensor(a!)[] k_pages, Tensor(b!)[] v_pages) -> Tensor");
  m.def(
      "paged_rope_append_out(Tensor qkv, Tensor kv_lens, Tensor q_start, Tensor block_table, Tensor? cos, Tensor? sin, "
      "int heads, Tensor(a!)[] k_pages, Tensor(b!)[] v_pages, Tensor(c!) q_out) -> ()");
  m.def(
      "paged_attend(Tensor q, Tensor kv_lens, Tensor q_start, Tensor block_table, Tensor[] k_pages, Tensor[] v_pages, "
      "float scale, float cap, int window, Tensor? slopes, Tensor? prefix, Tensor(a!)? workspace) -> Tensor");
  m.def(
      "paged_attend_out(Tensor q, Tensor kv_lens, Tensor q_start, Tensor block_table, Tensor[] k_pages, Tensor[] v_pages, "
      "float scale, float cap, int window, Tensor? slopes, Tensor? prefix, Tensor(a!)? workspace, Tensor(b!) out) -> ()");
}

TORCH_LIBRARY_IMPL(spectra_hip, CUDA, m) {
  m.impl("paged_rope_append", &paged_rope_append);
  m.impl("paged_rope_append_out", &paged_rope_append_out);
  m.impl("paged_attend", &paged_attend);
  m.impl("paged_attend_out", &paged_attend_out);
}

TORCH_LIBRARY_IMPL(spectra_hip, Meta, m) {
  m.impl("paged_rope_append", &paged_rope_append_meta);
  m.impl("paged_rope_append_out", &paged_rope_append_out_meta);
  m.impl("paged_attend", &paged_attend_meta);
  m.impl("paged_attend_out", &paged_attend_out_meta);
}
