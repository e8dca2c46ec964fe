// What the registered operators of the paged cache and their Python functions share: checks, descriptors, and the test
// for arguments that the dispatcher would only pass on.
#pragma once

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

namespace spectra_torch {

using OptTensor = c10::optional<at::Tensor>;

inline void check_paged(const char* fn, int st) {
  if (st == SPECTRA_OK) return;
  TORCH_CHECK_VALUE(st != SPECTRA_ERR_INVALID, fn, ": ", spectra_last_error());
  TORCH_CHECK(false, fn, " failed (", st, "): ", spectra_last_error());
}

inline bool rank1(const at::Tensor& t, at::ScalarType dtype, int64_t n, const at::Device& dev) {
  return t.scalar_type() == dtype && t.dim() == 1 && t.size(0) == n && (n < 2 || t.stride(0) == 1) && t.device() == dev;
}

// Checks a batch of a pool of `pages` pages (sizes [kv, page, d]) for calls of `heads` query heads and describes it.
inline void describe_batch(spectra_paged_kv_t& p, const at::Device& dev, int64_t heads, int64_t kv, int64_t page, int64_t d,
                           const at::Tensor& kv_lens, const at::Tensor& q_start, const at::Tensor& block_table) {
  TORCH_CHECK_VALUE(heads > 0 && heads % kv == 0, "heads (", heads, ") must be a multiple of the pages' ", kv, " KV heads");
  const int64_t batch = kv_lens.dim() == 1 ? kv_lens.size(0) : -1;
  TORCH_CHECK_VALUE(batch >= 0 && rank1(kv_lens, at::kInt, batch, dev), "kv_lens must be contiguous int32 [batch] on ", dev);
  TORCH_CHECK_VALUE(rank1(q_start, at::kInt, batch + 1, dev), "q_start must be contiguous int32 [batch + 1 = ", batch + 1,
                    "] on ", dev, ": ", batch, " sequences need that");
  TORCH_CHECK_VALUE(block_table.scalar_type() == at::kInt && block_table.dim() == 2 && block_table.size(0) == batch &&
                        (block_table.size(1) < 2 || block_table.stride(1) == 1) && block_table.device() == dev,
                    "block_table must be int32 [", batch, ", pages a sequence] with contiguous rows on ", dev);
  TORCH_CHECK_VALUE(page > 0 && page <= 65536 && kv <= 65536 && d <= 65536 && heads <= (1 << 20) && batch <= (1 << 20) &&
                        block_table.size(1) <= (1 << 30),
                    "sizes out of range");
  p.kv_heads = (int32_t)kv;
  p.head_dim = (int32_t)d;
  p.page_size = (int32_t)page;
  p.batch = (int32_t)batch;
  p.table_width = (int32_t)block_table.size(1);
  p.block_table = static_cast<const int32_t*>(block_table.data_ptr());
  p.table_stride = block_table.stride(0);
  p.kv_lens = static_cast<const int32_t*>(kv_lens.data_ptr());
  p.q_start = static_cast<const int32_t*>(q_start.data_ptr());
}

// Checks a paged cache and its batch for activations of a type and `heads` query heads (0: as many as KV heads) and describes it.
inline spectra_paged_kv_t describe_paged(at::ScalarType dtype, const at::Device& dev, int64_t heads, const at::Tensor& kv_lens,
                                         const at::Tensor& q_start, const at::Tensor& block_table, at::TensorList k,
                                         at::TensorList v) {
  const bool q4 = k.size() == 3;
  TORCH_CHECK_VALUE((k.size() == 1 || q4) && v.size() == k.size() && k[0].dim() == 4,
                    "k_pages and v_pages must be [pages, kv_heads, page, d], or (codes, scales, zeros) of that");
  TORCH_CHECK_VALUE(dtype == at::kHalf || (dtype == at::kBFloat16 && !q4),
                    "activations must be fp16 (or bf16, on bf16 pages), got ", dtype);
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
  spectra_paged_kv_t p{};
  p.kind = q4 ? SPECTRA_KV_4BIT : dtype == at::kBFloat16 ? SPECTRA_KV_BF16 : SPECTRA_KV_F16;
  describe_batch(p, dev, heads == 0 ? kv : heads, kv, page, d, kv_lens, q_start, block_table);
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
  return p;
}
inline spectra_paged_kv_t describe_paged(const at::Tensor& x, int64_t heads, const at::Tensor& kv_lens, const at::Tensor& q_start,
                                         const at::Tensor& block_table, at::TensorList k, at::TensorList v) {
  TORCH_CHECK_VALUE(heads > 0, "heads must be positive, got ", heads);
  return describe_paged(x.scalar_type(), x.device(), heads, kv_lens, q_start, block_table, k, v);
}

inline void check_out(const at::Tensor& out, const at::Tensor& x, int64_t tokens, int64_t heads, int64_t d, const char* name) {
  TORCH_CHECK_VALUE(out.scalar_type() == x.scalar_type() && out.dim() == 3 && out.size(0) == tokens &&
                        out.size(1) == heads && out.size(2) == d && out.is_contiguous() && out.device() == x.device(),
                    name, " must be contiguous ", x.scalar_type(), " [", tokens, ", ", heads, ", ", d, "] on ", x.device());
}

// What the results' shapes are made of, for a call without memory.
inline void check_meta(const at::Tensor& x, int64_t dims, at::TensorList k, at::TensorList v) {
  TORCH_CHECK_VALUE(x.dim() == dims && (k.size() == 1 || k.size() == 3) && v.size() == k.size() && k[0].dim() == 4,
                    "k_pages and v_pages must be [pages, kv_heads, page, d], or (codes, scales, zeros) of that, for ", dims,
                    "-dimensional activations");
}
// A tensor of a device that the dispatcher would do nothing about.
inline bool plain_tensor(PyObject* o) {
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
inline bool dispatched() {
  return c10::impl::TorchDispatchModeTLS::any_modes_set() ||
         !(c10::impl::tls_local_dispatch_key_set().included_ - c10::default_included_set).empty();
}

}  // namespace spectra_torch
