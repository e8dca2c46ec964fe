// The paged KV cache's operators as registered PyTorch operators: torch.ops.spectra_hip.
// paged_rope_append and paged_attend (no counterpart in the reference).
//
// One call each: the checks of shapes, types, strides and devices, the descriptor, the output from
// the caching allocator and the launch on the current HIP stream of the operands' device.  A
// single-token step is launch-bound: the same checks in Python with a ctypes call took 18 us, three
// times the kernel.  Bad arguments raise ValueError; other failures RuntimeError naming the status.
//
// The library is a Python module, too, whose functions take the same arguments and go past the
// dispatcher (some 2 us a call for this many arguments) where it would only have passed them on:
// plain tensors that nothing is differentiated by, and no mode that wants to see operators.  Otherwise they return
// NotImplemented, and the caller takes the registered operator, which a compiler traces and whose result says, when a
// gradient is asked of it, that there is none.
#include "torch_args.h"
#include "torch_batch.h"

using namespace spectra_torch;

namespace {

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
    {"paged_rope_axes_append", (PyCFunction)(void*)py_axes_append, METH_FASTCALL, nullptr},
    {"paged_key_bounds", (PyCFunction)(void*)py_key_bounds, METH_FASTCALL, nullptr},
    {"paged_bounds_values", (PyCFunction)(void*)py_bounds_values, METH_FASTCALL, nullptr},
    {"paged_select", (PyCFunction)(void*)py_select, METH_FASTCALL, nullptr},
    {"paged_attend_blocks", (PyCFunction)(void*)py_attend_blocks, METH_FASTCALL, nullptr},
    {"adjust_logits", (PyCFunction)(void*)py_adjust_logits, METH_FASTCALL, nullptr},
    {"next_tokens", (PyCFunction)(void*)py_next_tokens, METH_FASTCALL, nullptr},
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
