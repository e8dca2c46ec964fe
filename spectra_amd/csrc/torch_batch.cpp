// The operators around the paged cache that a served batch's step is made of, as registered PyTorch operators and as
// Python functions past the dispatcher (torch_paged.cpp says why there are both): appending with rotary positions of
// several axes, bounds of the pages' keys, the selection of pages, attention over them, the adjustment of a batch's
// logits and the choice of its next tokens.
#include "torch_batch.h"

#include <functional>
#include <string>

#include "torch_args.h"

namespace spectra_torch {
namespace {

hipStream_t stream_of(const at::Device& dev) { return c10::hip::getCurrentHIPStream(dev.index()).stream(); }

template <typename T>
const T* ptr(const OptTensor& t) {
  return t.has_value() ? static_cast<const T*>(t->data_ptr()) : nullptr;
}

// ---- append with axes ----
at::Tensor axes_append(const at::Tensor& qkv_in, const at::Tensor& positions_in, const at::Tensor& axis_in,
                       const at::Tensor& kv_lens, const at::Tensor& q_start, const at::Tensor& block_table,
                       const at::Tensor& cos, const at::Tensor& sin, int64_t heads, at::TensorList k, at::TensorList v,
                       const at::Tensor* q_out) {
  at::Tensor qkv = qkv_in, positions = positions_in, axis = axis_in;
  TORCH_CHECK_VALUE(qkv.dim() == 2, "qkv must be [T, (heads + 2 kv) * d]");
  const spectra_paged_kv_t p = describe_paged(qkv, heads, kv_lens, q_start, block_table, k, v);
  const int64_t tokens = qkv.size(0), d = p.head_dim, width = (heads + 2 * p.kv_heads) * d;
  const auto dev = qkv.device();
  TORCH_CHECK_VALUE(qkv.size(1) == width, "qkv rows must hold (heads + 2 kv) * d = ", width, " values, got ", qkv.size(1));
  TORCH_CHECK_VALUE(positions.scalar_type() == at::kInt && positions.dim() == 2 && positions.size(1) == tokens &&
                        positions.size(0) >= 1 && positions.size(0) <= 4 && positions.device() == dev,
                    "positions must be int32 [axes, ", tokens, "] on ", dev, ", one to four axes");
  TORCH_CHECK_VALUE(axis.scalar_type() == at::kByte && axis.dim() == 1 && axis.size(0) == d / 2 && axis.device() == dev,
                    "axis must be uint8 [d / 2 = ", d / 2, "] on ", dev);
  for (const at::Tensor* t : {&cos, &sin})
    TORCH_CHECK_VALUE(t->scalar_type() == at::kFloat && t->dim() == 2 && t->size(0) == cos.size(0) && t->size(0) > 0 &&
                          t->size(1) == d / 2 && t->is_contiguous() && t->device() == dev,
                      "cos and sin must be contiguous fp32 [rows, d / 2], at least a row, on ", dev);
  const c10::DeviceGuard guard(dev);
  // rows are read 16 bytes at a time
  if (qkv.stride(1) != 1 || (tokens > 1 && (qkv.stride(0) < width || qkv.stride(0) % 8 != 0)) ||
      reinterpret_cast<uintptr_t>(qkv.data_ptr()) % 16 != 0)
    qkv = qkv.clone(at::MemoryFormat::Contiguous);
  if ((tokens > 1 && positions.stride(1) != 1) || (positions.size(0) > 1 && positions.stride(0) < tokens))
    positions = positions.clone(at::MemoryFormat::Contiguous);
  if (axis.stride(0) != 1) axis = axis.clone(at::MemoryFormat::Contiguous);
  at::Tensor q;
  if (q_out != nullptr) {
    check_out(*q_out, qkv, tokens, heads, d, "q_out");
    q = *q_out;
  } else {
    q = at::detail::empty_cuda({tokens, heads, d}, qkv.scalar_type(), dev, c10::nullopt);
  }
  if (tokens == 0) return q;
  check_paged("spectra_paged_rope_axes_append",
              spectra_paged_rope_axes_append(&p, qkv.data_ptr(), tokens > 1 ? qkv.stride(0) : width, tokens,
                                             static_cast<const int32_t*>(positions.data_ptr()), positions.stride(0),
                                             (int32_t)positions.size(0), static_cast<const uint8_t*>(axis.data_ptr()),
                                             static_cast<const float*>(cos.data_ptr()),
                                             static_cast<const float*>(sin.data_ptr()), cos.size(0), (int32_t)heads,
                                             q.data_ptr(), stream_of(dev)));
  return q;
}

// ---- bounds ----
// Checks codes and scales of a pool of `pages` pages; -1: of as many as the codes have.
spectra_paged_bounds_t describe_bounds(const at::Tensor& codes, const at::Tensor& scales, int64_t pages, int64_t kv, int64_t d,
                                       const at::Device& dev) {
  TORCH_CHECK_VALUE(codes.scalar_type() == at::kChar && codes.dim() == 4 && (pages < 0 || codes.size(0) == pages) &&
                        (kv < 0 || codes.size(1) == kv) && codes.size(2) == 2 && (d < 0 || codes.size(3) == d) &&
                        codes.device() == dev,
                    "bounds' codes must be int8 [pages, kv_heads, 2, d] of the pool on ", dev);
  pages = codes.size(0), kv = codes.size(1), d = codes.size(3);
  TORCH_CHECK_VALUE(pages > 0 && kv > 0, "the pool has no pages");
  const auto st = codes.strides();
  TORCH_CHECK_VALUE(st[3] == 1 && st[2] == d && (kv == 1 || st[1] == 2 * d), "a page's codes must be contiguous");
  TORCH_CHECK_VALUE(scales.scalar_type() == at::kFloat && scales.dim() == 2 && scales.size(0) == pages && scales.size(1) == kv &&
                        (kv == 1 || scales.stride(1) == 1) && scales.device() == dev,
                    "bounds' scales must be fp32 [", pages, ", ", kv, "] with contiguous rows on ", dev);
  return {static_cast<int8_t*>(codes.data_ptr()), codes.stride(0), static_cast<float*>(scales.data_ptr()), scales.stride(0)};
}

void key_bounds(int64_t tokens, const at::Tensor& kv_lens, const at::Tensor& q_start, const at::Tensor& block_table,
                at::TensorList k, const at::Tensor& codes, const at::Tensor& scales) {
  TORCH_CHECK_VALUE(k.size() == 1 || k.size() == 3, "k_pages must be [pages, kv_heads, page, d], or (codes, scales, zeros) of that");
  const auto dev = k[0].device();
  const spectra_paged_kv_t p =
      describe_paged(k.size() == 3 ? at::kHalf : k[0].scalar_type(), dev, 0, kv_lens, q_start, block_table, k, k);
  const spectra_paged_bounds_t b = describe_bounds(codes, scales, p.num_pages, p.kv_heads, p.head_dim, dev);
  TORCH_CHECK_VALUE(tokens >= 0, "tokens must not be negative, got ", tokens);
  if (tokens == 0) return;
  const c10::DeviceGuard guard(dev);
  check_paged("spectra_paged_key_bounds", spectra_paged_key_bounds(&p, tokens, &b, stream_of(dev)));
}

// dtype: SPECTRA_F16, BF16 or F32
at::ScalarType type_of(int64_t dtype) {
  TORCH_CHECK_VALUE(dtype == SPECTRA_F16 || dtype == SPECTRA_BF16 || dtype == SPECTRA_F32, "unknown dtype ", dtype);
  return dtype == SPECTRA_F16 ? at::kHalf : dtype == SPECTRA_BF16 ? at::kBFloat16 : at::kFloat;
}
at::Tensor bounds_values(const at::Tensor& codes, const at::Tensor& scales, int64_t dtype) {
  const auto dev = codes.device();
  const spectra_paged_bounds_t b = describe_bounds(codes, scales, -1, -1, -1, dev);
  const c10::DeviceGuard guard(dev);
  at::Tensor out = at::detail::empty_cuda(codes.sizes(), type_of(dtype), dev, c10::nullopt);
  TORCH_CHECK_VALUE(codes.size(1) <= 65536 && codes.size(3) <= 65536, "sizes out of range");
  check_paged("spectra_paged_bounds_values",
              spectra_paged_bounds_values(&b, codes.size(0), (int32_t)codes.size(1), (int32_t)codes.size(3), out.data_ptr(),
                                          (int32_t)dtype, stream_of(dev)));
  return out;
}

// ---- selection ----
at::Tensor select(const at::Tensor& q_in, const at::Tensor& kv_lens, const at::Tensor& q_start, const at::Tensor& block_table,
                  const at::Tensor& codes, const at::Tensor& scales, int64_t page, int64_t count, int64_t sink, int64_t local,
                  const OptTensor& workspace, const at::Tensor* out_in) {
  at::Tensor q = q_in;
  TORCH_CHECK_VALUE(q.dim() == 3 && (q.scalar_type() == at::kHalf || q.scalar_type() == at::kBFloat16),
                    "q must be fp16 or bf16 [T, heads, d]");
  const int64_t tokens = q.size(0), heads = q.size(1), d = q.size(2);
  const auto dev = q.device();
  const spectra_paged_bounds_t b = describe_bounds(codes, scales, -1, -1, d, dev);
  const int64_t kv = codes.size(1);
  spectra_paged_kv_t p{};
  describe_batch(p, dev, heads, kv, page, d, kv_lens, q_start, block_table);
  p.num_pages = codes.size(0);
  TORCH_CHECK_VALUE(count >= 1 && count <= 32768 && sink >= 0 && local >= 1 && sink + local <= count && sink <= count,
                    "count must hold the first `sink` and the last `local` (at least one) blocks, got ", count, ", ", sink, ", ",
                    local);
  TORCH_CHECK_VALUE(!workspace.has_value() || (workspace->is_contiguous() && workspace->device() == dev),
                    "workspace must be contiguous on ", dev);
  const c10::DeviceGuard guard(dev);
  if (q.stride(2) != 1 || (heads > 1 && q.stride(1) != d) || reinterpret_cast<uintptr_t>(q.data_ptr()) % 16 != 0 ||
      (tokens > 1 && (q.stride(0) % 8 != 0 || q.stride(0) < heads * d)))
    q = q.clone(at::MemoryFormat::Contiguous);
  at::Tensor out;
  if (out_in != nullptr) {
    TORCH_CHECK_VALUE(out_in->scalar_type() == at::kInt && out_in->dim() == 3 && out_in->size(0) == tokens &&
                          out_in->size(1) == kv && out_in->size(2) == count && out_in->is_contiguous() && out_in->device() == dev,
                      "out must be contiguous int32 [", tokens, ", ", kv, ", ", count, "] on ", dev);
    out = *out_in;
  } else {
    out = at::detail::empty_cuda({tokens, kv, count}, at::kInt, dev, c10::nullopt);
  }
  if (tokens == 0) return out;
  check_paged("spectra_paged_select",
              spectra_paged_select(&p, &b, q.data_ptr(), tokens > 1 ? q.stride(0) : heads * d,
                                   q.scalar_type() == at::kBFloat16 ? SPECTRA_BF16 : SPECTRA_F16, tokens, (int32_t)heads,
                                   (int32_t)count, (int32_t)sink, (int32_t)local,
                                   workspace.has_value() ? workspace->data_ptr() : nullptr,
                                   workspace.has_value() ? (size_t)workspace->numel() * workspace->element_size() : 0,
                                   static_cast<int32_t*>(out.data_ptr()), stream_of(dev)));
  return out;
}

// ---- attention over blocks ----
at::Tensor attend_blocks(const at::Tensor& q_in, const at::Tensor& blocks_in, const at::Tensor& kv_lens, const at::Tensor& q_start,
                         const at::Tensor& block_table, at::TensorList k, at::TensorList v, double scale, double cap,
                         const OptTensor& workspace, const at::Tensor* out_in) {
  at::Tensor q = q_in, blocks = blocks_in;
  TORCH_CHECK_VALUE(q.dim() == 3, "q must be [T, heads, d]");
  const int64_t tokens = q.size(0), heads = q.size(1), d = q.size(2);
  const spectra_paged_kv_t p = describe_paged(q, heads, kv_lens, q_start, block_table, k, v);
  TORCH_CHECK_VALUE(d == p.head_dim, "q has head size ", d, ", the pages ", p.head_dim);
  const auto dev = q.device();
  TORCH_CHECK_VALUE(blocks.scalar_type() == at::kInt && blocks.dim() == 3 && blocks.size(0) == tokens &&
                        blocks.size(1) == p.kv_heads && blocks.size(2) >= 1 && blocks.size(2) <= (1 << 30) && blocks.device() == dev,
                    "blocks must be int32 [", tokens, ", ", p.kv_heads, ", at least one] on ", dev);
  TORCH_CHECK_VALUE(!workspace.has_value() || (workspace->is_contiguous() && workspace->device() == dev),
                    "workspace must be contiguous on ", dev);
  TORCH_CHECK_VALUE(cap >= 0.0 && scale > 0.0, "scale must be positive, cap 0 (none) or positive, got ", scale, ", ", cap);
  const c10::DeviceGuard guard(dev);
  if (q.stride(2) != 1 || (heads > 1 && q.stride(1) != d) || reinterpret_cast<uintptr_t>(q.data_ptr()) % 16 != 0 ||
      (tokens > 1 && (q.stride(0) % 8 != 0 || q.stride(0) < heads * d)))
    q = q.clone(at::MemoryFormat::Contiguous);
  if (!blocks.is_contiguous()) blocks = blocks.clone(at::MemoryFormat::Contiguous);
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
  check_paged("spectra_paged_attend_blocks",
              spectra_paged_attend_blocks(&p, q.data_ptr(), tokens > 1 ? q.stride(0) : heads * d, tokens, (int32_t)heads,
                                          static_cast<const int32_t*>(blocks.data_ptr()), (int32_t)blocks.size(2), (float)scale,
                                          (float)cap, ws.data_ptr(), (size_t)ws.numel() * ws.element_size(), out.data_ptr(),
                                          stream_of(dev)));
  return out;
}

// ---- logits ----
struct Logits {
  spectra_logits_t l{};
  std::vector<at::Tensor> keep;  // copies that the call reads

  // A 2-D operand with contiguous rows.
  const at::Tensor& rows(const at::Tensor& t) {
    if ((t.size(1) < 2 || t.stride(1) == 1) && (t.size(0) < 2 || t.stride(0) >= t.size(1))) return t;
    keep.push_back(t.clone(at::MemoryFormat::Contiguous));
    return keep.back();
  }
};

void describe_logits(Logits& a, const at::Tensor& logits, const OptTensor& history, const OptTensor& lens,
                     const OptTensor& prompt_lens, const OptTensor& repetition, const OptTensor& presence,
                     const OptTensor& frequency, const OptTensor& bias_ids, const OptTensor& bias, const OptTensor& allowed,
                     const OptTensor& allowed_rows) {
  a.keep.reserve(8);
  const auto dtype = logits.scalar_type();
  const auto dev = logits.device();
  TORCH_CHECK_VALUE(logits.dim() == 2 && (dtype == at::kHalf || dtype == at::kBFloat16 || dtype == at::kFloat),
                    "logits must be fp16, bf16 or fp32 [rows, vocab], got ", dtype, " ", logits.sizes());
  const int64_t n = logits.size(0), vocab = logits.size(1);
  TORCH_CHECK_VALUE(n <= 65535 && vocab >= 1 && vocab < (1LL << 31), "rows or vocab out of range: ", logits.sizes());
  spectra_logits_t& l = a.l;
  l.dtype = dtype == at::kHalf ? SPECTRA_F16 : dtype == at::kBFloat16 ? SPECTRA_BF16 : SPECTRA_F32;
  l.rows = (int32_t)n;
  l.vocab = vocab;
  const std::pair<const OptTensor*, const char*> floats[] = {{&repetition, "repetition"}, {&presence, "presence"}, {&frequency, "frequency"}};
  for (const auto& f : floats)
    TORCH_CHECK_VALUE(!f.first->has_value() || rank1(**f.first, at::kFloat, n, dev), f.second, " must be contiguous fp32 [", n, "] on ", dev);
  const std::pair<const OptTensor*, const char*> ints[] = {{&lens, "lens"}, {&prompt_lens, "prompt_lens"}, {&allowed_rows, "allowed_rows"}};
  for (const auto& f : ints)
    TORCH_CHECK_VALUE(!f.first->has_value() || rank1(**f.first, at::kInt, n, dev), f.second, " must be contiguous int32 [", n, "] on ", dev);
  const bool counts = repetition.has_value() || presence.has_value() || frequency.has_value();
  TORCH_CHECK_VALUE(!counts || history.has_value(), "penalties need a history");
  TORCH_CHECK_VALUE(history.has_value() || !(lens.has_value() || prompt_lens.has_value()), "lens and prompt_lens are of a history");
  TORCH_CHECK_VALUE(!history.has_value() || (history->scalar_type() == at::kLong && history->dim() == 2 && history->size(0) == n &&
                                             history->device() == dev && history->size(1) < (1LL << 31) - 4096),
                    "history must be int64 [", n, ", tokens] on ", dev);
  TORCH_CHECK_VALUE(bias_ids.has_value() == bias.has_value(), "bias_ids and bias must both be given or both be None");
  if (bias.has_value())
    TORCH_CHECK_VALUE(bias_ids->scalar_type() == at::kLong && bias_ids->dim() == 2 && bias_ids->size(0) == n &&
                          bias->scalar_type() == at::kFloat && bias->sizes() == bias_ids->sizes() && bias_ids->device() == dev &&
                          bias->device() == dev && bias->size(1) < (1LL << 30),
                      "bias_ids must be int64 and bias fp32 [", n, ", tokens] on ", dev);
  TORCH_CHECK_VALUE(allowed.has_value() || !allowed_rows.has_value(), "allowed_rows name rows of allowed");
  if (allowed.has_value())
    TORCH_CHECK_VALUE(allowed->scalar_type() == at::kInt && allowed->dim() == 2 && allowed->size(1) == (vocab + 31) / 32 &&
                          allowed->size(0) >= 1 && allowed->size(0) < (1LL << 31) &&
                          (allowed_rows.has_value() || allowed->size(0) == n) && allowed->device() == dev,
                      "allowed must be int32 [masks, ", (vocab + 31) / 32, "] on ", dev, ", a mask for each row without allowed_rows");
  if (n == 0) return;
  const c10::DeviceGuard guard(dev);
  const at::Tensor& x = a.rows(logits);
  l.logits = x.data_ptr();
  l.ld = n > 1 ? x.stride(0) : vocab;
  if (counts && history->size(1) > 0) {
    const at::Tensor& h = a.rows(*history);
    l.history = static_cast<const int64_t*>(h.data_ptr());
    l.history_ld = h.stride(0);
    l.history_width = h.size(1);
    l.history_lens = ptr<int32_t>(lens);
    l.prompt_lens = ptr<int32_t>(prompt_lens);
    l.repetition = ptr<float>(repetition);
    l.presence = ptr<float>(presence);
    l.frequency = ptr<float>(frequency);
  }
  if (bias.has_value() && bias->size(1) > 0) {
    const at::Tensor &i = a.rows(*bias_ids), &b = a.rows(*bias);
    l.bias_ids = static_cast<const int64_t*>(i.data_ptr());
    l.bias_ids_ld = i.stride(0);
    l.bias = static_cast<const float*>(b.data_ptr());
    l.bias_ld = b.stride(0);
    l.biases = (int32_t)b.size(1);
  }
  if (allowed.has_value()) {
    const at::Tensor& m = a.rows(*allowed);
    l.allowed = static_cast<const int32_t*>(m.data_ptr());
    l.allowed_ld = m.stride(0);
    l.states = (int32_t)m.size(0);
    l.state = ptr<int32_t>(allowed_rows);
  }
}

at::Tensor adjust(const at::Tensor& logits, const OptTensor& history, const OptTensor& lens, const OptTensor& prompt_lens,
                  const OptTensor& repetition, const OptTensor& presence, const OptTensor& frequency, const OptTensor& bias_ids,
                  const OptTensor& bias, const OptTensor& allowed, const OptTensor& allowed_rows, const at::Tensor* out_in) {
  Logits a;
  describe_logits(a, logits, history, lens, prompt_lens, repetition, presence, frequency, bias_ids, bias, allowed, allowed_rows);
  const auto dev = logits.device();
  const int64_t n = logits.size(0), vocab = logits.size(1);
  const c10::DeviceGuard guard(dev);
  at::Tensor out;
  if (out_in != nullptr) {
    TORCH_CHECK_VALUE(out_in->scalar_type() == logits.scalar_type() && out_in->sizes() == logits.sizes() && out_in->device() == dev &&
                          (vocab == 1 || out_in->stride(1) == 1) && (n < 2 || out_in->stride(0) >= vocab),
                      "out must be ", logits.scalar_type(), " ", logits.sizes(), " with contiguous rows on ", dev);
    out = *out_in;
  } else {
    out = at::detail::empty_cuda({n, vocab}, logits.scalar_type(), dev, c10::nullopt);
  }
  if (n == 0) return out;
  check_paged("spectra_adjust_logits", spectra_adjust_logits(&a.l, out.data_ptr(), n > 1 ? out.stride(0) : vocab, stream_of(dev)));
  return out;
}

at::Tensor next(const at::Tensor& logits, const OptTensor& history, const OptTensor& lens, const OptTensor& prompt_lens,
                const OptTensor& repetition, const OptTensor& presence, const OptTensor& frequency, const OptTensor& bias_ids,
                const OptTensor& bias, const OptTensor& allowed, const OptTensor& allowed_rows, const OptTensor& workspace,
                const at::Tensor* out_in) {
  Logits a;
  describe_logits(a, logits, history, lens, prompt_lens, repetition, presence, frequency, bias_ids, bias, allowed, allowed_rows);
  const auto dev = logits.device();
  const int64_t n = logits.size(0);
  TORCH_CHECK_VALUE(n <= SPECTRA_NEXT_TOKENS_ROWS, "at most ", SPECTRA_NEXT_TOKENS_ROWS, " rows, got ", n);
  TORCH_CHECK_VALUE(!workspace.has_value() || (workspace->is_contiguous() && workspace->device() == dev),
                    "workspace must be contiguous on ", dev);
  const c10::DeviceGuard guard(dev);
  at::Tensor out;
  if (out_in != nullptr) {
    TORCH_CHECK_VALUE(rank1(*out_in, at::kLong, n, dev), "out must be contiguous int64 [", n, "] on ", dev);
    out = *out_in;
  } else {
    out = at::detail::empty_cuda({n}, at::kLong, dev, c10::nullopt);
  }
  if (n == 0) return out;
  at::Tensor ws;
  if (workspace.has_value()) {
    ws = *workspace;
  } else {
    ws = at::detail::empty_cuda({(int64_t)spectra_next_tokens_workspace()}, at::kByte, dev, c10::nullopt);
    ws.zero_();
  }
  check_paged("spectra_next_tokens",
              spectra_next_tokens(&a.l, static_cast<int64_t*>(out.data_ptr()), ws.data_ptr(),
                                  (size_t)ws.numel() * ws.element_size(), stream_of(dev)));
  return out;
}

// ---- the registered operators ----
at::Tensor axes_append_op(const at::Tensor& qkv, const at::Tensor& positions, const at::Tensor& axis, const at::Tensor& kv_lens,
                          const at::Tensor& q_start, const at::Tensor& block_table, const at::Tensor& cos, const at::Tensor& sin,
                          int64_t heads, at::TensorList k, at::TensorList v) {
  return axes_append(qkv, positions, axis, kv_lens, q_start, block_table, cos, sin, heads, k, v, nullptr);
}
void axes_append_out_op(const at::Tensor& qkv, const at::Tensor& positions, const at::Tensor& axis, const at::Tensor& kv_lens,
                        const at::Tensor& q_start, const at::Tensor& block_table, const at::Tensor& cos, const at::Tensor& sin,
                        int64_t heads, at::TensorList k, at::TensorList v, const at::Tensor& q_out) {
  axes_append(qkv, positions, axis, kv_lens, q_start, block_table, cos, sin, heads, k, v, &q_out);
}
at::Tensor axes_append_meta(const at::Tensor& qkv, const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                            const at::Tensor&, const at::Tensor&, const at::Tensor&, int64_t heads, at::TensorList k,
                            at::TensorList v) {
  check_meta(qkv, 2, k, v);
  return at::empty_symint({qkv.sym_size(0), heads, k[0].sym_size(3) * (k.size() == 3 ? 2 : 1)}, qkv.options());
}
void axes_append_out_meta(const at::Tensor& qkv, const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                          const at::Tensor&, const at::Tensor&, const at::Tensor&, int64_t, at::TensorList k, at::TensorList v,
                          const at::Tensor&) {
  check_meta(qkv, 2, k, v);
}

void key_bounds_meta(int64_t, const at::Tensor&, const at::Tensor&, const at::Tensor&, at::TensorList k, const at::Tensor&,
                     const at::Tensor&) {
  TORCH_CHECK_VALUE(k.size() == 1 || k.size() == 3, "k_pages must be [pages, kv_heads, page, d], or (codes, scales, zeros) of that");
}

at::Tensor bounds_values_meta(const at::Tensor& codes, const at::Tensor&, int64_t dtype) {
  return at::empty_symint(codes.sym_sizes(), codes.options().dtype(type_of(dtype)));
}

at::Tensor select_op(const at::Tensor& q, const at::Tensor& kv_lens, const at::Tensor& q_start, const at::Tensor& block_table,
                     const at::Tensor& codes, const at::Tensor& scales, int64_t page, int64_t count, int64_t sink, int64_t local,
                     const OptTensor& workspace) {
  return select(q, kv_lens, q_start, block_table, codes, scales, page, count, sink, local, workspace, nullptr);
}
void select_out_op(const at::Tensor& q, const at::Tensor& kv_lens, const at::Tensor& q_start, const at::Tensor& block_table,
                   const at::Tensor& codes, const at::Tensor& scales, int64_t page, int64_t count, int64_t sink, int64_t local,
                   const OptTensor& workspace, const at::Tensor& out) {
  select(q, kv_lens, q_start, block_table, codes, scales, page, count, sink, local, workspace, &out);
}
at::Tensor select_meta(const at::Tensor& q, const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor& codes,
                       const at::Tensor&, int64_t, int64_t count, int64_t, int64_t, const OptTensor&) {
  TORCH_CHECK_VALUE(q.dim() == 3 && codes.dim() == 4, "q must be [T, heads, d], bounds' codes [pages, kv_heads, 2, d]");
  return at::empty_symint({q.sym_size(0), codes.sym_size(1), count}, q.options().dtype(at::kInt));
}
void select_out_meta(const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                     const at::Tensor&, int64_t, int64_t, int64_t, int64_t, const OptTensor&, const at::Tensor&) {}

at::Tensor attend_blocks_op(const at::Tensor& q, const at::Tensor& blocks, const at::Tensor& kv_lens, const at::Tensor& q_start,
                            const at::Tensor& block_table, at::TensorList k, at::TensorList v, double scale, double cap,
                            const OptTensor& workspace) {
  return attend_blocks(q, blocks, kv_lens, q_start, block_table, k, v, scale, cap, workspace, nullptr);
}
void attend_blocks_out_op(const at::Tensor& q, const at::Tensor& blocks, const at::Tensor& kv_lens, const at::Tensor& q_start,
                          const at::Tensor& block_table, at::TensorList k, at::TensorList v, double scale, double cap,
                          const OptTensor& workspace, const at::Tensor& out) {
  attend_blocks(q, blocks, kv_lens, q_start, block_table, k, v, scale, cap, workspace, &out);
}
at::Tensor attend_blocks_meta(const at::Tensor& q, const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                              at::TensorList k, at::TensorList v, double, double, const OptTensor&) {
  check_meta(q, 3, k, v);
  return at::empty_symint(q.sym_sizes(), q.options());
}
void attend_blocks_out_meta(const at::Tensor& q, const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                            at::TensorList k, at::TensorList v, double, double, const OptTensor&, const at::Tensor&) {
  check_meta(q, 3, k, v);
}

#define SPECTRA_LOGITS_PARAMS                                                                                               \
  const at::Tensor &logits, const OptTensor &history, const OptTensor &lens, const OptTensor &prompt_lens,                 \
      const OptTensor &repetition, const OptTensor &presence, const OptTensor &frequency, const OptTensor &bias_ids,       \
      const OptTensor &bias, const OptTensor &allowed, const OptTensor &allowed_rows
#define SPECTRA_LOGITS_ARGS \
  logits, history, lens, prompt_lens, repetition, presence, frequency, bias_ids, bias, allowed, allowed_rows

at::Tensor adjust_op(SPECTRA_LOGITS_PARAMS) { return adjust(SPECTRA_LOGITS_ARGS, nullptr); }
void adjust_out_op(SPECTRA_LOGITS_PARAMS, const at::Tensor& out) { adjust(SPECTRA_LOGITS_ARGS, &out); }
void adjust_inplace_op(const at::Tensor& logits, const OptTensor& history, const OptTensor& lens, const OptTensor& prompt_lens,
                       const OptTensor& repetition, const OptTensor& presence, const OptTensor& frequency,
                       const OptTensor& bias_ids, const OptTensor& bias, const OptTensor& allowed, const OptTensor& allowed_rows) {
  adjust(SPECTRA_LOGITS_ARGS, &logits);
}
at::Tensor next_op(SPECTRA_LOGITS_PARAMS, const OptTensor& workspace) { return next(SPECTRA_LOGITS_ARGS, workspace, nullptr); }
void next_out_op(SPECTRA_LOGITS_PARAMS, const OptTensor& workspace, const at::Tensor& out) { next(SPECTRA_LOGITS_ARGS, workspace, &out); }

void check_logits_meta(const at::Tensor& logits) { TORCH_CHECK_VALUE(logits.dim() == 2, "logits must be [rows, vocab]"); }
at::Tensor adjust_meta(const at::Tensor& logits, const OptTensor&, const OptTensor&, const OptTensor&, const OptTensor&,
                       const OptTensor&, const OptTensor&, const OptTensor&, const OptTensor&, const OptTensor&, const OptTensor&) {
  check_logits_meta(logits);
  return at::empty_symint(logits.sym_sizes(), logits.options());
}
void adjust_out_meta(const at::Tensor& logits, const OptTensor&, const OptTensor&, const OptTensor&, const OptTensor&,
                     const OptTensor&, const OptTensor&, const OptTensor&, const OptTensor&, const OptTensor&, const OptTensor&,
                     const at::Tensor&) {
  check_logits_meta(logits);
}
void adjust_inplace_meta(const at::Tensor& logits, const OptTensor&, const OptTensor&, const OptTensor&, const OptTensor&,
                         const OptTensor&, const OptTensor&, const OptTensor&, const OptTensor&, const OptTensor&,
                         const OptTensor&) {
  check_logits_meta(logits);
}
at::Tensor next_meta(const at::Tensor& logits, const OptTensor&, const OptTensor&, const OptTensor&, const OptTensor&,
                     const OptTensor&, const OptTensor&, const OptTensor&, const OptTensor&, const OptTensor&, const OptTensor&,
                     const OptTensor&) {
  check_logits_meta(logits);
  return at::empty_symint({logits.sym_size(0)}, logits.options().dtype(at::kLong));
}
void next_out_meta(const at::Tensor& logits, const OptTensor&, const OptTensor&, const OptTensor&, const OptTensor&,
                   const OptTensor&, const OptTensor&, const OptTensor&, const OptTensor&, const OptTensor&, const OptTensor&,
                   const OptTensor&, const at::Tensor&) {
  check_logits_meta(logits);
}

at::Tensor released(const std::function<at::Tensor()>& f) {
  pybind11::gil_scoped_release release;
  return f();
}

}  // namespace

// ---- the Python functions ----
PyObject* py_axes_append(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 12, "paged_rope_axes_append takes 12 arguments");
  Arguments a{args};
  const at::Tensor *qkv = a.tensor(0), *positions = a.tensor(1), *axis = a.tensor(2), *lens = a.tensor(3), *starts = a.tensor(4),
                   *table = a.tensor(5), *cos = a.tensor(6), *sin = a.tensor(7);
  const int64_t heads = a.integer(8);
  const std::vector<at::Tensor> k = a.list(9), v = a.list(10);
  const OptTensor out = a.optional(11);
  if (!a.plain || dispatched()) Py_RETURN_NOTIMPLEMENTED;
  return THPVariable_Wrap(released([&] {
    return axes_append(*qkv, *positions, *axis, *lens, *starts, *table, *cos, *sin, heads, k, v, out.has_value() ? &*out : nullptr);
  }));
  END_HANDLE_TH_ERRORS
}

PyObject* py_key_bounds(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 7, "paged_key_bounds takes 7 arguments");
  Arguments a{args};
  const int64_t tokens = a.integer(0);
  const at::Tensor *lens = a.tensor(1), *starts = a.tensor(2), *table = a.tensor(3);
  const std::vector<at::Tensor> k = a.list(4);
  const at::Tensor *codes = a.tensor(5), *scales = a.tensor(6);
  if (!a.plain || dispatched()) Py_RETURN_NOTIMPLEMENTED;
  {
    pybind11::gil_scoped_release release;
    key_bounds(tokens, *lens, *starts, *table, k, *codes, *scales);
  }
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

PyObject* py_bounds_values(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 3, "paged_bounds_values takes 3 arguments");
  Arguments a{args};
  const at::Tensor *codes = a.tensor(0), *scales = a.tensor(1);
  const int64_t dtype = a.integer(2);
  if (!a.plain || dispatched()) Py_RETURN_NOTIMPLEMENTED;
  return THPVariable_Wrap(released([&] { return bounds_values(*codes, *scales, dtype); }));
  END_HANDLE_TH_ERRORS
}

PyObject* py_select(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 12, "paged_select takes 12 arguments");
  Arguments a{args};
  const at::Tensor *q = a.tensor(0), *lens = a.tensor(1), *starts = a.tensor(2), *table = a.tensor(3), *codes = a.tensor(4),
                   *scales = a.tensor(5);
  const int64_t page = a.integer(6), count = a.integer(7), sink = a.integer(8), local = a.integer(9);
  const OptTensor workspace = a.optional(10), out = a.optional(11);
  if (!a.plain || dispatched()) Py_RETURN_NOTIMPLEMENTED;
  return THPVariable_Wrap(released([&] {
    return select(*q, *lens, *starts, *table, *codes, *scales, page, count, sink, local, workspace, out.has_value() ? &*out : nullptr);
  }));
  END_HANDLE_TH_ERRORS
}

PyObject* py_attend_blocks(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 11, "paged_attend_blocks takes 11 arguments");
  Arguments a{args};
  const at::Tensor *q = a.tensor(0), *blocks = a.tensor(1), *lens = a.tensor(2), *starts = a.tensor(3), *table = a.tensor(4);
  const std::vector<at::Tensor> k = a.list(5), v = a.list(6);
  const bool usual = args[7] == Py_None;  // 1 / sqrt(d)
  double scale = usual ? 1.0 : a.number(7);
  const double cap = a.number(8);
  const OptTensor workspace = a.optional(9), out = a.optional(10);
  if (!a.plain || dispatched()) Py_RETURN_NOTIMPLEMENTED;
  if (usual && q->dim() == 3) scale = 1.0 / std::sqrt((double)q->size(2));
  return THPVariable_Wrap(released([&] {
    return attend_blocks(*q, *blocks, *lens, *starts, *table, k, v, scale, cap, workspace, out.has_value() ? &*out : nullptr);
  }));
  END_HANDLE_TH_ERRORS
}

PyObject* py_adjust_logits(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 12, "adjust_logits takes 12 arguments");
  Arguments a{args};
  const at::Tensor* logits = a.tensor(0);
  OptTensor o[11];
  for (int i = 0; i < 11; ++i) o[i] = a.optional(1 + i);
  if (!a.plain || dispatched()) Py_RETURN_NOTIMPLEMENTED;
  return THPVariable_Wrap(released([&] {
    return adjust(*logits, o[0], o[1], o[2], o[3], o[4], o[5], o[6], o[7], o[8], o[9], o[10].has_value() ? &*o[10] : nullptr);
  }));
  END_HANDLE_TH_ERRORS
}

PyObject* py_next_tokens(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 13, "next_tokens takes 13 arguments");
  Arguments a{args};
  const at::Tensor* logits = a.tensor(0);
  OptTensor o[12];
  for (int i = 0; i < 12; ++i) o[i] = a.optional(1 + i);
  if (!a.plain || dispatched()) Py_RETURN_NOTIMPLEMENTED;
  return THPVariable_Wrap(released([&] {
    return next(*logits, o[0], o[1], o[2], o[3], o[4], o[5], o[6], o[7], o[8], o[9], o[10], o[11].has_value() ? &*o[11] : nullptr);
  }));
  END_HANDLE_TH_ERRORS
}

TORCH_LIBRARY_FRAGMENT(spectra_hip, m) {
  const std::string batch = "Tensor kv_lens, Tensor q_start, Tensor block_table, ";
  const std::string axes = "Tensor qkv, Tensor positions, Tensor axis, " + batch +
                           "Tensor cos, Tensor sin, int heads, Tensor(a!)[] k_pages, Tensor(b!)[] v_pages";
  m.def(("paged_rope_axes_append(" + axes + ") -> Tensor").c_str());
  m.def(("paged_rope_axes_append_out(" + axes + ", Tensor(c!) q_out) -> ()").c_str());
  m.def(("paged_key_bounds(int tokens, " + batch + "Tensor[] k_pages, Tensor(a!) codes, Tensor(b!) scales) -> ()").c_str());
  m.def("paged_bounds_values(Tensor codes, Tensor scales, int dtype) -> Tensor");
  const std::string sel = "Tensor q, " + batch + "Tensor codes, Tensor scales, int page, int count, int sink, int local, Tensor(a!)? workspace";
  m.def(("paged_select(" + sel + ") -> Tensor").c_str());
  m.def(("paged_select_out(" + sel + ", Tensor(b!) out) -> ()").c_str());
  const std::string att = "Tensor q, Tensor blocks, " + batch + "Tensor[] k_pages, Tensor[] v_pages, float scale, float cap, Tensor(a!)? workspace";
  m.def(("paged_attend_blocks(" + att + ") -> Tensor").c_str());
  m.def(("paged_attend_blocks_out(" + att + ", Tensor(b!) out) -> ()").c_str());
  const std::string more =
      "Tensor? history, Tensor? lens, Tensor? prompt_lens, Tensor? repetition, Tensor? presence, Tensor? frequency, "
      "Tensor? bias_ids, Tensor? bias, Tensor? allowed, Tensor? allowed_rows";
  m.def(("adjust_logits(Tensor logits, " + more + ") -> Tensor").c_str());
  m.def(("adjust_logits_out(Tensor logits, " + more + ", Tensor(a!) out) -> ()").c_str());
  m.def(("adjust_logits_(Tensor(a!) logits, " + more + ") -> ()").c_str());
  m.def(("next_tokens(Tensor logits, " + more + ", Tensor(a!)? workspace) -> Tensor").c_str());
  m.def(("next_tokens_out(Tensor logits, " + more + ", Tensor(a!)? workspace, Tensor(b!) out) -> ()").c_str());
}

TORCH_LIBRARY_IMPL(spectra_hip, CUDA, m) {
  m.impl("paged_rope_axes_append", &axes_append_op);
  m.impl("paged_rope_axes_append_out", &axes_append_out_op);
  m.impl("paged_key_bounds", &key_bounds);
  m.impl("paged_bounds_values", &bounds_values);
  m.impl("paged_select", &select_op);
  m.impl("paged_select_out", &select_out_op);
  m.impl("paged_attend_blocks", &attend_blocks_op);
  m.impl("paged_attend_blocks_out", &attend_blocks_out_op);
  m.impl("adjust_logits", &adjust_op);
  m.impl("adjust_logits_out", &adjust_out_op);
  m.impl("adjust_logits_", &adjust_inplace_op);
  m.impl("next_tokens", &next_op);
  m.impl("next_tokens_out", &next_out_op);
}

TORCH_LIBRARY_IMPL(spectra_hip, Meta, m) {
  m.impl("paged_rope_axes_append", &axes_append_meta);
  m.impl("paged_rope_axes_append_out", &axes_append_out_meta);
  m.impl("paged_key_bounds", &key_bounds_meta);
  m.impl("paged_bounds_values", &bounds_values_meta);
  m.impl("paged_select", &select_meta);
  m.impl("paged_select_out", &select_out_meta);
  m.impl("paged_attend_blocks", &attend_blocks_meta);
  m.impl("paged_attend_blocks_out", &attend_blocks_out_meta);
  m.impl("adjust_logits", &adjust_meta);
  m.impl("adjust_logits_out", &adjust_out_meta);
  m.impl("adjust_logits_", &adjust_inplace_meta);
  m.impl("next_tokens", &next_meta);
  m.impl("next_tokens_out", &next_out_meta);
}

}  // namespace spectra_torch
