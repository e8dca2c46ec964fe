// A batch's logits on their way to the next token: penalties for repeated tokens, biases and grammar masks, and the greedy
// choice from what they leave (the reference's sample_token at temperature 0, engine.py:1690-1697, for one row without them).
//
// For row b and token v, all in fp32, each operation rounded as written:
//   x = logits[b, v]
//   v among the row's tokens so far (prompt or answer):   x = x > 0 ? x / repetition : x * repetition
//   c > 0 times in the answer:                            x = x - frequency c,  x = x - presence
//   v among the row's biased tokens (the last wins):       x = x + bias
//   the row's grammar state does not allow v:              x = -inf
// and the choice is the largest x, the lowest v on ties, NaN before all (as torch.argmax); -1 when every x is -inf.
//
// A workgroup takes a slice of a row's vocabulary, 8 or 16 logits a lane, which are asked for first and stay in registers.
// The row's tokens are read once a slice (from L2); those of the slice are counted in LDS, a word a token, by atomics on
// whole numbers, whose order changes nothing, and a bit each says which words there are to look at: most logits pass
// without.  So nothing is kept between steps, and the history may change in any way.  The choice meets over a row's slices
// in 64-bit maxima of (value, token) in the workspace, whose last arrival writes the token.
//
// Bound by memory and the launch where nothing is adjusted and logits are written (64 rows of 128256 in fp16 9.7 us, 33 MB).
// Choices take as long for fp16 as for fp32 (9.0 us for either; one slice a row 2.8), so not by their bytes but by 4032 small
// workgroups with a read, a reduction and a meeting each.  With long histories by a chain of dependent steps in every slice:
// the tokens, the counts between barriers, each listed token's logit once more, then the rest (4096 tokens a row, 40 biases
// and masks: 14.8, chosen from 13.8).
#include <algorithm>

#include "paged.h"

namespace spectra {

constexpr int kLgRows = SPECTRA_NEXT_TOKENS_ROWS;  // rows whose slices meet in the workspace
constexpr int kLgApart = 256;  // bytes of a row there: the best so far, and from kLgApart / 2 on how many slices have arrived

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

// A token's word: in its lower half how often it is in the answer, the half's top bit for the prompt; in the upper half 1
// + the place of its bias.  Of 32 bits, or of 64 where a history or a list of biases is longer than the halves hold.
template <typename W>
struct LgWord {
  static constexpr int half = 4 * sizeof(W);
  static constexpr W prompt = W(1) << (half - 1), count = prompt - 1, low = (W(1) << half) - 1;
};
// A slice's words, its map of bits and its list of tokens in LDS; of these the first two start at zero.
constexpr size_t lg_zero(int slice, size_t word) { return slice / 8 + slice * word; }

// TH: threads of a workgroup; C: chunks of 8 logits a lane; W: the words' type.
// (out may be the logits themselves: a workgroup reads its slice before it writes it, and no others', and nothing tells the
// compiler that the two lie apart)
template <int DT, bool PICK, int TH, int C, typename W>
__global__ void __launch_bounds__(TH) logits_kernel(const LogitsArgs a, void* out, int64_t ldo, int64_t* __restrict__ tokens,
                                                    int slices, uint8_t* __restrict__ meeting) {
  typedef typename LgType<DT>::T T;
  typedef LgWord<W> Word;
  constexpr int S = 8 * TH * C, U = 2048 / TH > 4 ? 8 : 4;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ lg_key_t meet[TH / 64];
  __shared__ float held[TH];  // the first biases
  __shared__ int listed;
  const int tid = threadIdx.x, row = blockIdx.y;
  const int64_t begin = (int64_t)blockIdx.x * S;
  const int n = (int)min((int64_t)S, a.vocab - begin);
  const bool counts = a.history != nullptr, biased = a.biases > 0;
  const T* x = (const T*)a.x + row * a.ldx + begin;
  T* y = (T*)out + row * ldo + begin;
  // ---- the lane's logits; of a chunk that the row ends in, one by one
  LgEight<T> u[C];
#pragma unroll
  for (int k = 0; k < C; ++k) {
    const int i = 8 * (tid + k * TH);
    if (i + 8 <= n) {
      u[k] = *(const LgEight<T>*)(x + i);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) u[k].v[e] = i + e < n ? x[i + e] : T(0);
    }
  }
  const uint8_t* mask = nullptr;
  if (a.allowed != nullptr) {
    const int s = a.state != nullptr ? a.state[row] : row;
    if (s >= 0 && s < a.states) mask = (const uint8_t*)(a.allowed + s * a.ldallowed) + begin / 8;
  }
  // ---- the tokens that are adjusted
  uint32_t* map = (uint32_t*)smem;
  W* words = (W*)(smem + S / 8);
  uint16_t* list = (uint16_t*)(smem + lg_zero(S, sizeof(W)));
  float rep = 1.0f, pres = 0.0f, freq = 0.0f;
  const float* bias = a.bias + row * a.ldbias;
  if (counts || biased) {
    const int64_t* h = a.history + row * a.ldh;
    const int64_t* ids = a.bias_ids + row * a.ldid;
    // (the first of both are on their way while the words are cleared; a row's history is there beyond its length)
    int64_t id[U], bid = -1;
    int len = 0, prompt = 0;
    if (counts) {
#pragma unroll
      for (int k = 0; k < U; ++k) id[k] = h[min(tid + k * TH, a.hist - 1)];
      len = a.lens != nullptr ? min(max(a.lens[row], 0), a.hist) : a.hist;
      prompt = a.prompts != nullptr ? a.prompts[row] : 0;
      if (a.repetition != nullptr) rep = a.repetition[row];
      if (a.presence != nullptr) pres = a.presence[row];
      if (a.frequency != nullptr) freq = a.frequency[row];
    }
    if (biased && tid < a.biases) {
      bid = ids[tid];
      held[tid] = bias[tid];
    }
    for (int i = tid; i < (int)(lg_zero(S, sizeof(W)) / 16); i += TH) *(uint4*)(smem + 16 * i) = make_uint4(0, 0, 0, 0);
    if (tid == 0) listed = 0;
    __syncthreads();
    auto enlist = [&](uint32_t at) __attribute__((always_inline)) {
      list[atomicAdd(&listed, 1)] = (uint16_t)at;
      atomicOr(&map[at >> 5], 1u << (at & 31));
    };
    for (int i0 = tid; i0 < len; i0 += U * TH) {
      if (i0 >= U * TH) {
#pragma unroll
        for (int k = 0; k < U; ++k) id[k] = h[min(i0 + k * TH, a.hist - 1)];
      }
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int i = i0 + k * TH;
        const uint64_t at = (uint64_t)id[k] - (uint64_t)begin;
        if (i < len && at < (uint64_t)n) {
          const W was = i < prompt ? atomicOr(&words[at], Word::prompt) : atomicAdd(&words[at], W(1));
          if (was == 0) enlist((uint32_t)at);
        }
      }
    }
    if (biased) {
      __syncthreads();  // (lower halves are what they will be)
      for (int i = tid; i < a.biases; i += TH) {
        if (i >= TH) bid = ids[i];
        const uint64_t at = (uint64_t)bid - (uint64_t)begin;
        if (at < (uint64_t)n) {
          if (atomicMax(&words[at], (W)(i + 1) << Word::half | (words[at] & Word::low)) == 0) enlist((uint32_t)at);
        }
      }
    }
    __syncthreads();
    for (int p = tid; p < listed; p += TH) {
      const int at = list[p];
      const W s = words[at], c = s & Word::count;
      float v = LgType<DT>::get(x[at]);
      if ((s & Word::low) != 0) {
        v = v > 0.0f ? v / rep : v * rep;
        if (c != 0) {  // (an infinite penalty forbids what the answer has, and says nothing of the prompt)
          v = v - freq * (float)c;
          v = v - pres;
        }
      }
      const int place = (int)(s >> Word::half);
      if (place != 0) v = v + (place <= TH ? held[place - 1] : bias[place - 1]);
      words[at] = __builtin_bit_cast(uint32_t, v);
    }
    __syncthreads();
  }
  // ---- all of them
  float top = -INFINITY;  // the best of this lane, whose tokens come in order
  int at = -1;
  bool odd = false;       // it is NaN
#pragma unroll
  for (int k = 0; k < C; ++k) {
    const int i = 8 * (tid + k * TH);
    if (i >= n) continue;
    const uint32_t ok = mask != nullptr ? mask[i / 8] : 255u;
    const uint32_t own = counts || biased ? ((const uint8_t*)map)[i / 8] : 0u;
    float z[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) z[e] = LgType<DT>::get(u[k].v[e]);
    if (own != 0) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float v = __builtin_bit_cast(float, (uint32_t)words[i + e]);
        z[e] = own >> e & 1 ? v : z[e];
      }
    }
    LgEight<T> w;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float v = z[e];
      if (!(ok >> e & 1)) v = -INFINITY;
      if (PICK) {
        if (i + e < n && !odd && !(v <= top)) {
          top = v;
          at = i + e;
          odd = v != v;
        }
      } else {
        w.v[e] = LgType<DT>::put(v);
      }
    }
    if (!PICK) {
      if (i + 8 <= n) {
        *(LgEight<T>*)(y + i) = w;
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (i + e < n) y[i + e] = w.v[e];
      }
    }
  }
  if (PICK) {
    lg_key_t k = at >= 0 ? (lg_key_t)lg_order(top) << 32 | (uint32_t)~(uint32_t)(begin + at) : 0;
#pragma unroll
    for (int off = 1; off < 64; off *= 2) k = lg_most(k, (lg_key_t)__shfl_xor((unsigned long long)k, off, 64));
    if ((tid & 63) == 0) meet[tid >> 6] = k;
    __syncthreads();
    if (tid == 0) {
#pragma unroll
      for (int w = 1; w < TH / 64; ++w) k = lg_most(k, meet[w]);
      if (slices > 1) {
        // The maximum has happened before the arrival is counted, both where all of the card sees them.  (An ordered atomic
        // would write back and drop the L2 for it: 53 us, not 16, with 2048 workgroups; rows beside each other in memory
        // have their atomics wait for each other: 64 rows of 128256 took 23 us, not 9.7.)
        unsigned long long* best = (unsigned long long*)(meeting + row * kLgApart);
        uint32_t* arrived = (uint32_t*)(meeting + row * kLgApart + kLgApart / 2);
        __hip_atomic_fetch_max(best, (unsigned long long)k, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        if (__hip_atomic_fetch_add(arrived, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) != (uint32_t)slices - 1) return;
        asm volatile("" ::: "memory");
        k = __hip_atomic_load(best, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(best, 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(arrived, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
      tokens[row] = lg_token(k);
    }
  }
}

// Slices of 16384 logits by 1024 threads, of which two fill a compute unit, or of 2048 by 256, which fill the card with few
// rows and end sooner, but read a row's tokens eight times as often: where that is more than 2^20 tokens or so it costs more.
// (Large and small, us, fp16 rows of 128256: 8 rows with 1000 tokens 7.5 and 6.3, 16 7.5 and 7.2, 24 7.8 and 8.3; 8 rows with
// 4096 8.0 and 8.9, 64 13.2 and 21.0; 64 without 8.8 and 8.8, adjusted 10.0 and 9.6.  Slices of 4096 by 256 or 512 threads took
// 18.5 to 21.7 where large ones took 14.9, of 8192 by 1024 16.2.)
bool logits_large(int64_t rows, int64_t vocab, int64_t ids) { return rows * ((vocab + 2047) / 2048) * ids >= 5 << 18; }

int logits_args(const spectra_logits_t* l, LogitsArgs* out, size_t* lds, int* threads, int* slices, bool* wide) {
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
  *wide = a.hist > (int)LgWord<uint32_t>::count || a.biases >= 65535;
  const bool large = !*wide && logits_large(l->rows, l->vocab, (int64_t)a.hist + a.biases);  // (wide words of such a slice would not fit)
  const int slice = large ? 16384 : 2048;
  *threads = large ? 1024 : 256;
  *slices = (int)((l->vocab + slice - 1) / slice);
  *lds = 0;
  if (counts || a.biases > 0)
    *lds = lg_zero(slice, *wide ? 8 : 4) + 2 * std::min<int64_t>(slice, (int64_t)a.hist + a.biases);
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

template <bool PICK, int TH, int C, typename W>
static const void* logits_of(int dtype) {
  return dtype == SPECTRA_F16    ? (const void*)logits_kernel<SPECTRA_F16, PICK, TH, C, W>
         : dtype == SPECTRA_BF16 ? (const void*)logits_kernel<SPECTRA_BF16, PICK, TH, C, W>
                                 : (const void*)logits_kernel<SPECTRA_F32, PICK, TH, C, W>;
}
template <bool PICK>
static const void* logits_of(int dtype, int threads, bool wide) {
  if (wide) return logits_of<PICK, 256, 1, unsigned long long>(dtype);
  return threads == 256 ? logits_of<PICK, 256, 1, uint32_t>(dtype) : logits_of<PICK, 1024, 2, uint32_t>(dtype);
}

}  // namespace spectra

using namespace spectra;

extern "C" int spectra_adjust_logits(const spectra_logits_t* l, void* out, int64_t ldo, spectra_stream_t stream) {
  LogitsArgs a;
  size_t lds;
  int threads, slices;
  bool wide;
  if (int st = logits_args(l, &a, &lds, &threads, &slices, &wide); st != SPECTRA_OK) return st;
  const int es = elem_size(l->dtype);
  SPECTRA_REQUIRE(out != nullptr && reinterpret_cast<uintptr_t>(out) % es == 0, "out missing or not aligned");
  SPECTRA_REQUIRE(ldo >= l->vocab || l->rows == 1, "out's row stride too small");
  const bool in_place = out == l->logits && (ldo == l->ld || l->rows == 1);
  if (int st = logits_apart(l, {"out", out, l->vocab * es, ldo * es, l->rows}, {"", nullptr, 0, 0, 1}, in_place); st != SPECTRA_OK) return st;
  const void* kern = logits_of<false>(l->dtype, threads, wide);
  if (int st = ensure_lds_limit(kern); st != SPECTRA_OK) return st;
  int64_t* tokens = nullptr;
  uint8_t* meeting = nullptr;
  void* args[] = {(void*)&a, (void*)&out, (void*)&ldo, (void*)&tokens, (void*)&slices, (void*)&meeting};
  SPECTRA_HIP_CHECK(hipLaunchKernel(kern, dim3((unsigned)slices, (unsigned)l->rows), dim3((unsigned)threads), args, lds, (hipStream_t)stream));
  SPECTRA_HIP_CHECK(hipGetLastError());
  return SPECTRA_OK;
}

extern "C" size_t spectra_next_tokens_workspace(void) { return (size_t)kLgRows * kLgApart; }

extern "C" int spectra_next_tokens(const spectra_logits_t* l, int64_t* tokens, void* workspace, size_t workspace_bytes,
                                   spectra_stream_t stream) {
  LogitsArgs a;
  size_t lds;
  int threads, slices;
  bool wide;
  if (int st = logits_args(l, &a, &lds, &threads, &slices, &wide); st != SPECTRA_OK) return st;
  SPECTRA_REQUIRE(tokens != nullptr && reinterpret_cast<uintptr_t>(tokens) % 8 == 0, "tokens missing or not aligned");
  SPECTRA_REQUIRE(l->rows <= kLgRows, "too many rows");
  if (workspace == nullptr || workspace_bytes < spectra_next_tokens_workspace())
    return fail(SPECTRA_ERR_WORKSPACE, "workspace missing or smaller than spectra_next_tokens_workspace bytes");
  SPECTRA_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, "workspace must be 16-byte aligned");
  if (int st = logits_apart(l, {"tokens", tokens, 8LL * l->rows, 0, 1},
                            {"the workspace", workspace, (int64_t)spectra_next_tokens_workspace(), 0, 1}, false);
      st != SPECTRA_OK)
    return st;
  const void* kern = logits_of<true>(l->dtype, threads, wide);
  if (int st = ensure_lds_limit(kern); st != SPECTRA_OK) return st;
  uint8_t* meeting = (uint8_t*)workspace;
  void* out = nullptr;
  int64_t ldo = 0;
  void* args[] = {(void*)&a, (void*)&out, (void*)&ldo, (void*)&tokens, (void*)&slices, (void*)&meeting};
  SPECTRA_HIP_CHECK(hipLaunchKernel(kern, dim3((unsigned)slices, (unsigned)l->rows), dim3((unsigned)threads), args, lds, (hipStream_t)stream));
  SPECTRA_HIP_CHECK(hipGetLastError());
  return SPECTRA_OK;
}
