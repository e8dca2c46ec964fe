// Bounds of a page's keys, in 8 bits: what the selection of pages reads instead of the keys.
//
// For page j and KV head n, over the rows of the page that the sequence has (positions < kv_lens):
//   M_d = max k_d,  m_d = min k_d,  A = max_d max(|M_d|, |m_d|)
//   codes ceil(M_d 127 / A) and floor(m_d 127 / A), clamped to +-127;  scale A / 127
// so that scale (sum_d max(q_d, 0) M_d + min(q_d, 0) m_d) bounds every product of a query with a key of the page, up to
// the last bit of the scale.  Each operation is one fp32 rounding as written (127 / A, its product, A / 127): the codes
// are the same wherever they are worked out.  Maxima know no order, so a page is read once, in any order, and a page is
// always worked out anew from its rows: what it held before, or tokens taken back, leave nothing behind.
// A page with a key that is not finite has codes of 0 and the scale infinity (the selection takes it first, so that the
// attention shows what is wrong); one whose largest magnitude is below 2^-100, codes and scale of 0.
//
// A wave a page and KV head: a row is 16 lanes (head size 128) or 8, so 4 or 8 rows a load of 1 KB, four or eight
// loads in flight; rows meet across the lanes at the end.  Values are compared as pairs of 16-bit integers of the same
// order (five instructions for two; as fp32 values, eighteen), in which infinities and NaN end up at the ends, so that
// the maxima show them.  No LDS, no workspace.
// Bound by its chain of dependent loads (starts and lengths, the id, the rows) for a served batch's tokens: 64 users 4.0 us
// in a graph; by memory for prompts: 55 MB of bf16 keys 12.2 us, 4.6 TB/s; on 4 bits by vector instructions, the expansion's and
// the comparisons', some 520 a wave, which take 71 % of the cycles: 8.9 MB of rows of 64 dims 8.9 us (15.3 with the
// values compared as fp32).  More than one head a wave was slower for tokens (4.2 us with one,
// 5.7, 8.9 and 15.4 with 2, 4 and 8).
#include <algorithm>
#include <type_traits>

#include "paged_attend.h"

namespace spectra {

constexpr int kPbThreads = 256;
constexpr float kPbLeast = 7.8886091e-31f;  // 2^-100

typedef int16_t ps2_t __attribute__((ext_vector_type(2)));

// A pair of fp16 or bf16 values as integers of their order, and back (its own inverse).
__device__ __forceinline__ ps2_t pb_order(uint32_t x) {
  const ps2_t v = __builtin_bit_cast(ps2_t, x);
  return v ^ ((v >> 15) & (ps2_t){0x7fff, 0x7fff});
}

// Eight dims 8 c .. of a row: 16-bit values, or codes with their group's zero point and scale.
struct PbGroup {
  uint32_t zero, scale;
};
template <int HD, int KIND>
__device__ __forceinline__ uint4 pb_load(const PagedKv& kv, int page, int64_t row, int c, PbGroup& g) {
  const uint8_t* p = kv.k + paged_at(page, kv.page_step);
  if constexpr (KIND == kKv4) {
    g.scale = *(const uint16_t*)(kv.ks + paged_at(page, kv.scale_step) + 2 * (row * (HD / 32) + c / 4));
    g.zero = kv.kz[paged_at(page, kv.zero_step) + row * (HD / 32) + c / 4];
    return make_uint4(*(const uint32_t*)(p + row * (HD / 2) + 4 * c), 0, 0, 0);
  } else {
    return *(const uint4*)(p + (row * HD + 8 * c) * 2);
  }
}
// Their bits as pairs: 2 e and 2 e + 1, of 4 bits e and e + 4.  (An infinite or NaN scale gives infinities and NaN.)
template <int KIND>
__device__ __forceinline__ pu4_t pb_values(const uint4& x, const PbGroup& g) {
  if constexpr (KIND == kKv4) return kv4_pairs(x.x, kv4_zero(g.zero | g.zero << 16), __builtin_bit_cast(ph2_t, g.scale | g.scale << 16));
  else return (pu4_t){x.x, x.y, x.z, x.w};
}
template <int LB>
__device__ __forceinline__ void pb_meet(ps2_t& hi, ps2_t& lo, int lane) {
  hi = __builtin_elementwise_max(hi, __builtin_bit_cast(ps2_t, lane_xor<LB>(__builtin_bit_cast(float, hi), lane)));
  lo = __builtin_elementwise_min(lo, __builtin_bit_cast(ps2_t, lane_xor<LB>(__builtin_bit_cast(float, lo), lane)));
}

// Pages that a sequence's tokens of the call lie in: the first, and how many.
struct PagedTouched {
  int first, n;
};
__device__ __forceinline__ PagedTouched paged_touched(const PagedKv& kv, int b) {
  const PagedSeq sq = paged_seq(kv.q_start[b], kv.q_start[b + 1], kv.lens[b], kv.tokens);
  const int first = max(sq.len - sq.n, 0) >> kv.page_shift;
  const int last = min((sq.len - 1) >> kv.page_shift, kv.table_width - 1);
  return {first, sq.n > 0 && sq.len > 0 ? max(last - first + 1, 0) : 0};
}

template <int HD, int KIND>
__global__ void __launch_bounds__(kPbThreads) paged_bounds_kernel(const PagedKv kv, int8_t* __restrict__ codes,
                                                                  int64_t code_step, float* __restrict__ scales,
                                                                  int64_t scale_step, int units) {
  constexpr int CH = HD / 8, G = 64 / CH;  // lanes a row, rows a load
  constexpr bool BF = KIND == kKvBf16;
  const int lane = threadIdx.x & 63, c = lane % CH, rg = lane / CH;
  const int u = sread((int)(blockIdx.x * (kPbThreads / 64) + (threadIdx.x >> 6)));
  if (u >= units) return;
  const int kvh = u % kv.kv_heads, w = u / kv.kv_heads;  // (a page's heads beside each other)
  // the w-th page of the call: the sequences' pages counted, 64 sequences a step
  int base = 0, seq = -1, block = 0;
  for (int c0 = 0; c0 < kv.batch; c0 += 64) {
    const int b = c0 + lane;
    const PagedTouched t = b < kv.batch ? paged_touched(kv, b) : PagedTouched{0, 0};
    const int end = wave_scan(t.n) + base;
    const uint64_t past = __ballot(end > w);
    if (past != 0) {
      const int at = __builtin_ctzll(past);
      seq = c0 + at;
      block = __builtin_amdgcn_readlane(t.first, at) + w - (__builtin_amdgcn_readlane(end - t.n, at));
      break;
    }
    base = __builtin_amdgcn_readlane(end, 63);
  }
  if (seq < 0) return;
  seq = sread(seq);
  block = sread(block);
  const int len = sload(kv.lens + seq), page = sload(kv.table + seq * kv.table_stride + block);
  if ((uint32_t)page >= (uint32_t)kv.num_pages) return;
  const int rows = min(len - (block << kv.page_shift), 1 << kv.page_shift);  // >= 1
  // pairs of 16-bit values as integers of the same order, infinities and NaN at its ends
  ps2_t hi[4], lo[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    hi[e] = (ps2_t){-32768, -32768};
    lo[e] = (ps2_t){32767, 32767};
  }
  const int64_t first = (int64_t)kvh << kv.page_shift;
  auto take = [&](int r0, auto n) __attribute__((always_inline)) {
    constexpr int U = decltype(n)::value;
    uint4 x[U];
    PbGroup z[U];
#pragma unroll
    for (int i = 0; i < U; ++i)  // (past the last row: the last once more)
      x[i] = pb_load<HD, KIND>(kv, page, first + min(r0 + G * i + rg, rows - 1), c, z[i]);
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const pu4_t y = pb_values<KIND>(x[i], z[i]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const ps2_t v = pb_order(y[e]);
        hi[e] = __builtin_elementwise_max(hi[e], v);
        lo[e] = __builtin_elementwise_min(lo[e], v);
      }
    }
  };
  if (rows <= 4 * G) {
    take(0, std::integral_constant<int, 4>());
  } else {
    for (int r0 = 0; r0 < rows; r0 += 8 * G) take(r0, std::integral_constant<int, 8>());
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if constexpr (CH == 8) pb_meet<8>(hi[e], lo[e], lane);
    pb_meet<16>(hi[e], lo[e], lane);
    pb_meet<32>(hi[e], lo[e], lane);
  }
  // back to the values' bits; the largest magnitude
  uint32_t most = 0;
  uint32_t h[4], l[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    h[e] = __builtin_bit_cast(uint32_t, pb_order(__builtin_bit_cast(uint32_t, hi[e])));
    l[e] = __builtin_bit_cast(uint32_t, pb_order(__builtin_bit_cast(uint32_t, lo[e])));
    for (const uint32_t m : {h[e] & 0x7fff7fffu, l[e] & 0x7fff7fffu}) most = max(most, max(m & 0xffffu, m >> 16));
  }
#pragma unroll
  for (int off = 1; off < CH; off *= 2) most = max(most, (uint32_t)__shfl_xor((int)most, off, 64));
  const float a = BF ? bf2f((uint16_t)most) : h2f((uint16_t)most);
  const bool odd = most >= (BF ? 0x7f80u : 0x7c00u), none = odd || a < kPbLeast;
  const float inv = none ? 0.0f : 127.0f / a;
  uint32_t up[2] = {0, 0}, dn[2] = {0, 0};
  if (!none) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int at = KIND == kKv4 ? e & 3 : e >> 1, half = 16 * (KIND == kKv4 ? e >> 2 : e & 1);
      const uint16_t hb = (uint16_t)(h[at] >> half), lb = (uint16_t)(l[at] >> half);
      const float hf = BF ? bf2f(hb) : h2f(hb), lf = BF ? bf2f(lb) : h2f(lb);
      const int m = (int)fminf(fmaxf(__builtin_ceilf(hf * inv), -127.0f), 127.0f);
      const int n = (int)fminf(fmaxf(__builtin_floorf(lf * inv), -127.0f), 127.0f);
      up[e >> 2] |= (uint32_t)(m & 255) << (8 * (e & 3));
      dn[e >> 2] |= (uint32_t)(n & 255) << (8 * (e & 3));
    }
  }
  if (rg == 0) {
    int8_t* to = codes + page * code_step + (int64_t)kvh * 2 * HD + 8 * c;
    *(uint2*)to = make_uint2(up[0], up[1]);
    *(uint2*)(to + HD) = make_uint2(dn[0], dn[1]);
    if (lane == 0) scales[page * scale_step + kvh] = odd ? INFINITY : none ? 0.0f : a / 127.0f;
  }
}

// What the codes stand for: code times scale, rounded once; a page whose scale is infinite has the bounds +-infinity.
template <typename T>
__global__ void __launch_bounds__(256) paged_bounds_values_kernel(const int8_t* __restrict__ codes, int64_t code_step,
                                                                  const float* __restrict__ scales, int64_t scale_step,
                                                                  int kv_heads, int hd, int64_t n16, T* __restrict__ out) {
  const int per = kv_heads * hd / 8;  // 16 codes a lane
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n16; i += (int64_t)gridDim.x * 256) {
    const int64_t page = i / per;
    const int at = (int)(i - page * per), kvh = at / (hd / 8);
    const uint4 w = *(const uint4*)(codes + page * code_step + 16 * at);
    const float s = scales[page * scale_step + kvh];
    const bool low = (16 * at) % (2 * hd) >= hd;
    const uint32_t v[4] = {w.x, w.y, w.z, w.w};
    T y[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const float x = (float)(int8_t)(v[e >> 2] >> (8 * (e & 3)));
      y[e] = (T)(s == INFINITY ? (low ? -INFINITY : INFINITY) : x * s);
    }
#pragma unroll
    for (int p = 0; p < (int)sizeof(T); ++p) *(uint4*)(out + 16 * i + p * (16 / sizeof(T))) = *(const uint4*)(y + p * (16 / sizeof(T)));
  }
}

int paged_bounds_args(const spectra_paged_bounds_t* b, int64_t num_pages, int32_t kv_heads, int32_t hd) {
  SPECTRA_REQUIRE(b != nullptr && b->codes && b->scales, "NULL pointer");
  SPECTRA_REQUIRE(num_pages == 1 || (b->code_stride >= (int64_t)kv_heads * 2 * hd && b->scale_stride >= kv_heads),
                  "bounds' page stride too small");
  SPECTRA_REQUIRE(reinterpret_cast<uintptr_t>(b->codes) % 16 == 0 && (num_pages == 1 || b->code_stride % 16 == 0) &&
                      reinterpret_cast<uintptr_t>(b->scales) % 4 == 0,
                  "bounds' codes must be 16-byte aligned, page by page, their scales aligned");
  SPECTRA_REQUIRE(num_pages == 1 || (b->code_stride < (1LL << 31) && b->scale_stride < (1LL << 31)), "bounds' page stride too large");
  return SPECTRA_OK;
}
PagedRegion paged_bound_codes(const spectra_paged_bounds_t* b, int64_t num_pages, int32_t kv_heads, int32_t hd) {
  return {"the bounds' codes", b->codes, (int64_t)kv_heads * 2 * hd, b->code_stride, num_pages};
}
PagedRegion paged_bound_scales(const spectra_paged_bounds_t* b, int64_t num_pages, int32_t kv_heads) {
  return {"the bounds' scales", b->scales, 4LL * kv_heads, 4 * b->scale_stride, num_pages};
}

template <int HD>
static const void* bounds_of(int kind) {
  return kind == kKv4      ? (const void*)paged_bounds_kernel<HD, kKv4>
         : kind == kKvBf16 ? (const void*)paged_bounds_kernel<HD, kKvBf16>
                           : (const void*)paged_bounds_kernel<HD, kKvF16>;
}

}  // namespace spectra

using namespace spectra;

extern "C" int spectra_paged_key_bounds(const spectra_paged_kv_t* kv, int64_t tokens, const spectra_paged_bounds_t* bounds,
                                        spectra_stream_t stream) {
  SPECTRA_REQUIRE(kv != nullptr, "paged KV descriptor is NULL");
  spectra_paged_kv_t keys = *kv;  // (the values are not read, nor need they be given)
  keys.v = keys.k;
  keys.v_scales = keys.k_scales;
  keys.v_zeros = keys.k_zeros;
  kv = &keys;
  PagedKv p;
  if (int st = paged_args(kv, tokens, kv->kv_heads, &p); st != SPECTRA_OK) return st;
  const int hd = kv->head_dim;
  if (int st = paged_bounds_args(bounds, kv->num_pages, kv->kv_heads, hd); st != SPECTRA_OK) return st;
  const PagedPools pools = paged_pools(kv);
  if (int st = paged_apart({paged_bound_codes(bounds, kv->num_pages, kv->kv_heads, hd),
                            paged_bound_scales(bounds, kv->num_pages, kv->kv_heads)},
                           {pools.k, pools.ks, pools.kz, paged_table(kv), paged_lens(kv), paged_starts(kv)});
      st != SPECTRA_OK)
    return st;
  // a sequence's n tokens lie in at most n pages, and at most n / page + 2
  const int64_t pages = std::min<int64_t>(tokens, (tokens >> p.page_shift) + 2 * std::min<int64_t>(tokens, kv->batch));
  const int64_t all = pages * kv->kv_heads;
  SPECTRA_REQUIRE(all < (1LL << 31) - 256, "tokens out of range");
  int units = (int)all;
  const void* kern = hd == 64 ? bounds_of<64>(kv->kind) : bounds_of<128>(kv->kind);
  int8_t* codes = bounds->codes;
  float* scales = bounds->scales;
  int64_t cs = kv->num_pages == 1 ? 0 : bounds->code_stride, ss = kv->num_pages == 1 ? 0 : bounds->scale_stride;
  void* args[] = {(void*)&p, (void*)&codes, (void*)&cs, (void*)&scales, (void*)&ss, (void*)&units};
  SPECTRA_HIP_CHECK(hipLaunchKernel(kern, dim3((unsigned)((all + 3) / 4)), dim3(kPbThreads), args, 0, (hipStream_t)stream));
  SPECTRA_HIP_CHECK(hipGetLastError());
  return SPECTRA_OK;
}

extern "C" int spectra_paged_bounds_values(const spectra_paged_bounds_t* bounds, int64_t num_pages, int32_t kv_heads,
                                           int32_t head_dim, void* out, int32_t out_dtype, spectra_stream_t stream) {
  SPECTRA_REQUIRE(num_pages > 0 && num_pages < (1LL << 31) && kv_heads > 0 && kv_heads <= (1 << 16), "sizes out of range");
  if (head_dim != 64 && head_dim != 128) return fail(SPECTRA_ERR_UNSUPPORTED, "paged KV head_dim must be 64 or 128");
  if (int st = paged_bounds_args(bounds, num_pages, kv_heads, head_dim); st != SPECTRA_OK) return st;
  SPECTRA_REQUIRE(out != nullptr && reinterpret_cast<uintptr_t>(out) % 16 == 0, "out must be 16-byte aligned");
  SPECTRA_REQUIRE(out_dtype == SPECTRA_F16 || out_dtype == SPECTRA_BF16 || out_dtype == SPECTRA_F32, "unknown dtype");
  const int64_t n = num_pages * kv_heads * 2 * head_dim;
  if (int st = paged_apart({{"out", out, n * elem_size(out_dtype), 0, 1}},
                           {paged_bound_codes(bounds, num_pages, kv_heads, head_dim), paged_bound_scales(bounds, num_pages, kv_heads)});
      st != SPECTRA_OK)
    return st;
  int64_t n16 = n / 16, cs = num_pages == 1 ? 0 : bounds->code_stride, ss = num_pages == 1 ? 0 : bounds->scale_stride;
  const unsigned blocks = (unsigned)std::min<int64_t>((n16 + 255) / 256, 16384);
  const int8_t* codes = bounds->codes;
  const float* scales = bounds->scales;
  int kvh = kv_heads, hd = head_dim;
  const void* kern = out_dtype == SPECTRA_F16    ? (const void*)paged_bounds_values_kernel<_Float16>
                     : out_dtype == SPECTRA_BF16 ? (const void*)paged_bounds_values_kernel<__bf16>
                                                 : (const void*)paged_bounds_values_kernel<float>;
  void* args[] = {(void*)&codes, (void*)&cs, (void*)&scales, (void*)&ss, (void*)&kvh, (void*)&hd, (void*)&n16, (void*)&out};
  SPECTRA_HIP_CHECK(hipLaunchKernel(kern, dim3(blocks), dim3(256), args, 0, (hipStream_t)stream));
  SPECTRA_HIP_CHECK(hipGetLastError());
  return SPECTRA_OK;
}
