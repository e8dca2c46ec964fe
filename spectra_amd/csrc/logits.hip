// A batch's logits on their way to the next token: penalties for repeated tokens, biases and grammar masks, and the greedy
// choice from what they leave (the reference's sample_token at temperature 0, engine.py:1690-1697, for one row without them).
//
// For row b and token v, all in fp32, each operation rounded as written:
//   x = logits[b, v]
//   v among the row's tokens so far (prompt or answer):   x = x > 0 ? x / repetition : x * repetition
//   c times in the answer:                                x = x - frequency c,  x = x - presence (c > 0)
//   v among the row's biased tokens (the last wins):       x = x + bias
//   the row's grammar state does not allow v:              x = -inf
// and the choice is the largest x, the lowest v on ties, NaN before all (as torch.argmax); -1 when every x is -inf.
//
// A workgroup takes a slice of a row's vocabulary and keeps the slice's counts in LDS: the row's tokens are read once a
// slice (from L2), those of the slice counted by LDS atomics on whole numbers, whose order changes nothing, and the
// logits pass once, 16 bytes a lane.  So nothing is kept between steps, and the history may change in any way.  The choice
// meets over a row's slices in 64-bit maxima of (value, token) in the workspace, whose last arrival writes the token.
#include <algorithm>

#include "paged.h"

namespace spectra {

constexpr int kLgThreads = 256;
constexpr int kLgRows = SPECTRA_NEXT_TOKENS_ROWS;  // rows whose slices meet in the workspace

struct LogitsArgs {
  const void* x;
  int64_t ldx;
  int64_t vocab;
  const int64_t* history;
  int64_t ldh;
  int hist;            // tokens a row at most
  const int* lens;     // or NULL: hist
  const int* prompts;  // or NULL: 0
  const float *repetition, *presence, *frequency;
  const int64_t* bias_ids;
  const float* bias;
  int64_t ldid, ldbias;
  int biases;
  const uint32_t* allowed;
  int64_t ldallowed;
  int states;
  const int* state;  // or NULL: the row's number
  int slice;         // tokens of a slice, a multiple of 2048
};

// fp32 as an unsigned number of the same order, NaN above all.
__device__ __forceinline__ uint32_t lg_order(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.0f);
  return x != x ? ~0u : u ^ (u >> 31 ? ~0u : 0x80000000u);
}
constexpr uint32_t kLgNothing = 0x007fffffu;  // lg_order(-inf)

typedef uint64_t lg_key_t;
__device__ __forceinline__ lg_key_t lg_most(lg_key_t a, lg_key_t b) { return a > b ? a : b; }
__device__ __forceinline__ int64_t lg_token(lg_key_t k) {
  return (uint32_t)(k >> 32) <= kLgNothing ? -1 : (int64_t)(~(uint32_t)k);
}

// Eight values from any address of their type's alignment.
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) LgEight {
  T v[8];
};
template <int DT>
struct LgType;
template <>
struct LgType<SPECTRA_F16> {
  typedef uint16_t T;
  static __device__ __forceinline__ float get(T v) { return h2f(v); }
  static __device__ __forceinline__ T put(float v) { return f2h(v); }
};
template <>
struct LgType<SPECTRA_BF16> {
  typedef uint16_t T;
  static __device__ __forceinline__ float get(T v) { return bf2f(v); }
  static __device__ __forceinline__ T put(float v) { return f2bf(v); }
};
template <>
struct LgType<SPECTRA_F32> {
  typedef float T;
  static __device__ __forceinline__ float get(T v) { return v; }
  static __device__ __forceinline__ T put(float v) { return v; }
};

template <int DT, bool PICK>
__global__ void __launch_bounds__(kLgThreads) logits_kernel(const LogitsArgs a, void* __restrict__ out, int64_t ldo,
                                                            int64_t* __restrict__ tokens, int slices,
                                                            unsigned long long* __restrict__ best, uint32_t* __restrict__ arrived) {
  typedef typename LgType<DT>::T T;
  extern __shared__ __align__(16) uint32_t seen[];  // [slice]: bit 31 said at all, below it how often in the answer; then
  __shared__ lg_key_t meet[kLgThreads / 64];        // [slice]: 1 + the place of its bias
  const int tid = threadIdx.x, row = blockIdx.y;
  const int64_t begin = (int64_t)blockIdx.x * a.slice;
  const int n = (int)min((int64_t)a.slice, a.vocab - begin);
  const bool counts = a.history != nullptr, biased = a.biases > 0;
  uint32_t* where = seen + (counts ? a.slice : 0);
  if (counts || biased) {
    for (int i = 4 * tid; i < (counts && biased ? 2 : 1) * a.slice; i += 4 * kLgThreads) *(uint4*)(seen + i) = make_uint4(0, 0, 0, 0);
    __syncthreads();
  }
  float rep = 1.0f, pres = 0.0f, freq = 0.0f;
  if (counts) {
    if (a.repetition != nullptr) rep = a.repetition[row];
    if (a.presence != nullptr) pres = a.presence[row];
    if (a.frequency != nullptr) freq = a.frequency[row];
    const int64_t* h = a.history + row * a.ldh;
    const int len = a.lens != nullptr ? min(max(a.lens[row], 0), a.hist) : a.hist;
    const int prompt = a.prompts != nullptr ? a.prompts[row] : 0;
    constexpr int U = 8;
    for (int i0 = tid; i0 < len; i0 += U * kLgThreads) {
      int64_t id[U];
#pragma unroll
      for (int u = 0; u < U; ++u) id[u] = h[min(i0 + u * kLgThreads, len - 1)];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u * kLgThreads;
        const uint64_t at = (uint64_t)(id[u] - begin);
        if (i < len && at < (uint64_t)n) {
          if (i < prompt) atomicOr(&seen[at], 0x80000000u);
          else atomicAdd(&seen[at], 1u);
        }
      }
    }
  }
  if (biased) {
    const int64_t* ids = a.bias_ids + row * a.ldid;
    for (int i = tid; i < a.biases; i += kLgThreads) {
      const uint64_t at = (uint64_t)(ids[i] - begin);
      if (at < (uint64_t)n) atomicMax(&where[at], (uint32_t)i + 1);
    }
  }
  if (counts || biased) __syncthreads();
  const uint8_t* mask = nullptr;
  if (a.allowed != nullptr) {
    const int s = a.state != nullptr ? a.state[row] : row;
    if (s >= 0 && s < a.states) mask = (const uint8_t*)(a.allowed + s * a.ldallowed) + begin / 8;
  }
  const float* bias = a.bias + row * a.ldbias;
  const T* x = (const T*)a.x + row * a.ldx + begin;
  T* y = (T*)out + row * ldo + begin;
  float top = 0.0f;  // the best of this lane, whose tokens come in order
  uint32_t at = 0;
  bool any = false;
  auto adjusted = [&](float v, int i, bool ok) __attribute__((always_inline)) {
    if (counts) {
      const uint32_t s = seen[i];
      if (s != 0) {
        const uint32_t c = s & 0x7fffffffu;
        v = v > 0.0f ? v / rep : v * rep;
        v = v - freq * (float)c;
        if (c != 0) v = v - pres;
      }
    }
    if (biased) {
      const uint32_t p = where[i];
      if (p != 0) v = v + bias[p - 1];
    }
    return ok ? v : -INFINITY;
  };
  auto take = [&](float v, int i) __attribute__((always_inline)) {
    if (!any || (v > top && !(top != top)) || (v != v && !(top != top))) {
      top = v;
      at = (uint32_t)i;
      any = true;
    }
  };
  for (int i = 8 * tid; i < n; i += 8 * kLgThreads) {
    const uint32_t bits = mask != nullptr ? mask[i / 8] : 255u;
    if (i + 8 <= n) {
      const LgEight<T> u = *(const LgEight<T>*)(x + i);
      LgEight<T> w;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float v = adjusted(LgType<DT>::get(u.v[e]), i + e, bits >> e & 1);
        if (PICK) take(v, i + e);
        else w.v[e] = LgType<DT>::put(v);
      }
      if (!PICK) *(LgEight<T>*)(y + i) = w;
    } else {
      for (int e = 0; i + e < n; ++e) {
        const float v = adjusted(LgType<DT>::get(x[i + e]), i + e, bits >> e & 1);
        if (PICK) take(v, i + e);
        else y[i + e] = LgType<DT>::put(v);
      }
    }
  }
  if (PICK) {
    lg_key_t k = any ? (lg_key_t)lg_order(top) << 32 | (uint32_t)~(uint32_t)(begin + at) : 0;
#pragma unroll
    for (int off = 1; off < 64; off *= 2) k = lg_most(k, (lg_key_t)__shfl_xor((unsigned long long)k, off, 64));
    if ((tid & 63) == 0) meet[tid >> 6] = k;
    __syncthreads();
    if (tid == 0) {
#pragma unroll
      for (int w = 1; w < kLgThreads / 64; ++w) k = lg_most(k, meet[w]);
      if (slices > 1) {
        __hip_atomic_fetch_max(best + row, (unsigned long long)k, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __builtin_amdgcn_s_waitcnt(0);
        // (the maximum has happened before the arrival is counted)
        if (__hip_atomic_fetch_add(arrived + row, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) != (uint32_t)slices - 1) return;
        k = __hip_atomic_load(best + row, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(best + row, 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(arrived + row, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
      tokens[row] = lg_token(k);
    }
  }
}

// Slices: of 8192 tokens, whose counts leave room for four workgroups a compute unit; of 2048 while the batch has too few
// of those to fill the card.
int logits_slice(int64_t rows, int64_t vocab) { return rows * ((vocab + 8191) / 8192) >= 512 ? 8192 : 2048; }

int logits_args(const spectra_logits_t* l, LogitsArgs* out, size_t* lds) {
  SPECTRA_REQUIRE(l != nullptr && l->logits, "NULL pointer");
  SPECTRA_REQUIRE(l->dtype == SPECTRA_F16 || l->dtype == SPECTRA_BF16 || l->dtype == SPECTRA_F32, "unknown dtype");
  SPECTRA_REQUIRE(l->rows > 0 && l->rows <= 65535 && l->vocab > 0 && l->vocab < (1LL << 31), "rows or vocab out of range");
  SPECTRA_REQUIRE(l->ld >= l->vocab || l->rows == 1, "logits' row stride too small");
  const bool counts = l->repetition || l->presence || l->frequency;
  SPECTRA_REQUIRE(!counts || (l->history && l->history_width > 0), "penalties need a history");
  SPECTRA_REQUIRE(!counts || l->history_ld >= l->history_width || l->rows == 1, "the history's row stride too small");
  SPECTRA_REQUIRE(l->history_width >= 0 && l->history_width < (1LL << 31) - 4096, "history too wide");
  SPECTRA_REQUIRE(l->biases >= 0 && (l->biases == 0 || (l->bias_ids && l->bias)), "NULL pointer");
  SPECTRA_REQUIRE(l->biases == 0 || l->rows == 1 || (l->bias_ids_ld >= l->biases && l->bias_ld >= l->biases),
                  "biases' row stride too small");
  const int64_t words = (l->vocab + 31) / 32;
  SPECTRA_REQUIRE(!l->allowed || (l->states > 0 && (l->allowed_ld >= words || l->states == 1)), "masks' row stride too small");
  SPECTRA_REQUIRE(!l->allowed || l->state || l->states >= l->rows, "a mask for each row, or states");
  const int es = elem_size(l->dtype);
  auto off = [](const void* p, int to) { return reinterpret_cast<uintptr_t>(p) % to; };
  SPECTRA_REQUIRE(off(l->logits, es) == 0 && off(l->history, 8) == 0 && off(l->history_lens, 4) == 0 && off(l->prompt_lens, 4) == 0 &&
                      off(l->repetition, 4) == 0 && off(l->presence, 4) == 0 && off(l->frequency, 4) == 0 &&
                      off(l->bias_ids, 8) == 0 && off(l->bias, 4) == 0 && off(l->allowed, 4) == 0 && off(l->state, 4) == 0,
                  "operands must be aligned");
  LogitsArgs a{};
  a.x = l->logits;
  a.ldx = l->ld;
  a.vocab = l->vocab;
  if (counts) {
    a.history = l->history;
    a.ldh = l->history_ld;
    a.hist = (int)l->history_width;
    a.lens = l->history_lens;
    a.prompts = l->prompt_lens;
    a.repetition = l->repetition;
    a.presence = l->presence;
    a.frequency = l->frequency;
  }
  a.bias_ids = l->bias_ids;
  a.bias = l->bias;
  a.ldid = l->bias_ids_ld;
  a.ldbias = l->bias_ld;
  a.biases = l->biases;
  a.allowed = (const uint32_t*)l->allowed;
  a.ldallowed = l->allowed_ld;
  a.states = l->states;
  a.state = l->state;
  a.slice = logits_slice(l->rows, l->vocab);
  *lds = (size_t)a.slice * 4 * ((counts ? 1 : 0) + (a.biases > 0 ? 1 : 0));
  *out = a;
  return SPECTRA_OK;
}
// What a call reads, beside what it writes.
int logits_apart(const spectra_logits_t* l, const PagedRegion& written, const PagedRegion& more, bool in_place) {
  const int es = elem_size(l->dtype);
  const PagedRegion x = {"logits", in_place ? nullptr : l->logits, l->vocab * es, l->ld * es, l->rows};
  return paged_apart({written, more},
                     {x,
                      {"history", l->history, 8 * l->history_width, 8 * l->history_ld, l->rows},
                      {"lens", l->history_lens, 4LL * l->rows, 0, 1},
                      {"prompt_lens", l->prompt_lens, 4LL * l->rows, 0, 1},
                      {"repetition", l->repetition, 4LL * l->rows, 0, 1},
                      {"presence", l->presence, 4LL * l->rows, 0, 1},
                      {"frequency", l->frequency, 4LL * l->rows, 0, 1},
                      {"bias_ids", l->bias_ids, 8LL * l->biases, 8 * l->bias_ids_ld, l->rows},
                      {"bias", l->bias, 4LL * l->biases, 4 * l->bias_ld, l->rows},
                      {"allowed", l->allowed, (l->vocab + 31) / 32 * 4, 4 * l->allowed_ld, l->states},
                      {"allowed_rows", l->state, 4LL * l->rows, 0, 1}});
}

template <bool PICK>
static const void* logits_of(int dtype) {
  return dtype == SPECTRA_F16    ? (const void*)logits_kernel<SPECTRA_F16, PICK>
         : dtype == SPECTRA_BF16 ? (const void*)logits_kernel<SPECTRA_BF16, PICK>
                                 : (const void*)logits_kernel<SPECTRA_F32, PICK>;
}

}  // namespace spectra

using namespace spectra;

extern "C" int spectra_adjust_logits(const spectra_logits_t* l, void* out, int64_t ldo, spectra_stream_t stream) {
  LogitsArgs a;
  size_t lds;
  if (int st = logits_args(l, &a, &lds); st != SPECTRA_OK) return st;
  const int es = elem_size(l->dtype);
  SPECTRA_REQUIRE(out != nullptr && reinterpret_cast<uintptr_t>(out) % es == 0, "out missing or not aligned");
  SPECTRA_REQUIRE(ldo >= l->vocab || l->rows == 1, "out's row stride too small");
  const bool in_place = out == l->logits && (ldo == l->ld || l->rows == 1);
  if (int st = logits_apart(l, {"out", out, l->vocab * es, ldo * es, l->rows}, {"", nullptr, 0, 0, 1}, in_place); st != SPECTRA_OK) return st;
  const void* kern = logits_of<false>(l->dtype);
  if (int st = ensure_lds_limit(kern); st != SPECTRA_OK) return st;
  int slices = (int)((l->vocab + a.slice - 1) / a.slice);
  int64_t* tokens = nullptr;
  unsigned long long* best = nullptr;
  uint32_t* arrived = nullptr;
  void* args[] = {(void*)&a, (void*)&out, (void*)&ldo, (void*)&tokens, (void*)&slices, (void*)&best, (void*)&arrived};
  SPECTRA_HIP_CHECK(hipLaunchKernel(kern, dim3((unsigned)slices, (unsigned)l->rows), dim3(kLgThreads), args, lds, (hipStream_t)stream));
  SPECTRA_HIP_CHECK(hipGetLastError());
  return SPECTRA_OK;
}

extern "C" size_t spectra_next_tokens_workspace(void) { return (size_t)kLgRows * 16; }

extern "C" int spectra_next_tokens(const spectra_logits_t* l, int64_t* tokens, void* workspace, size_t workspace_bytes,
                                   spectra_stream_t stream) {
  LogitsArgs a;
  size_t lds;
  if (int st = logits_args(l, &a, &lds); st != SPECTRA_OK) return st;
  SPECTRA_REQUIRE(tokens != nullptr && reinterpret_cast<uintptr_t>(tokens) % 8 == 0, "tokens missing or not aligned");
  SPECTRA_REQUIRE(l->rows <= kLgRows, "too many rows");
  if (workspace == nullptr || workspace_bytes < spectra_next_tokens_workspace())
    return fail(SPECTRA_ERR_WORKSPACE, "workspace missing or smaller than spectra_next_tokens_workspace bytes");
  SPECTRA_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, "workspace must be 16-byte aligned");
  if (int st = logits_apart(l, {"tokens", tokens, 8LL * l->rows, 0, 1},
                            {"the workspace", workspace, (int64_t)spectra_next_tokens_workspace(), 0, 1}, false);
      st != SPECTRA_OK)
    return st;
  const void* kern = logits_of<true>(l->dtype);
  if (int st = ensure_lds_limit(kern); st != SPECTRA_OK) return st;
  int slices = (int)((l->vocab + a.slice - 1) / a.slice);
  unsigned long long* best = (unsigned long long*)workspace;
  uint32_t* arrived = (uint32_t*)(best + kLgRows);
  void* out = nullptr;
  int64_t ldo = 0;
  void* args[] = {(void*)&a, (void*)&out, (void*)&ldo, (void*)&tokens, (void*)&slices, (void*)&best, (void*)&arrived};
  SPECTRA_HIP_CHECK(hipLaunchKernel(kern, dim3((unsigned)slices, (unsigned)l->rows), dim3(kLgThreads), args, lds, (hipStream_t)stream));
  SPECTRA_HIP_CHECK(hipGetLastError());
  return SPECTRA_OK;
}
