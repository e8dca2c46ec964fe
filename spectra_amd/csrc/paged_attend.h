// What the paged attention kernels share: operand types, the joining of a tile's pieces, and the
// row-by-row path.
#pragma once

#include <algorithm>

#include "kv4.h"
#include "paged.h"

namespace spectra {

enum { kKvF16 = SPECTRA_KV_F16, kKvBf16 = SPECTRA_KV_BF16, kKv4 = SPECTRA_KV_4BIT };

typedef _Float16 ph2_t __attribute__((ext_vector_type(2)));
typedef _Float16 ph8_t __attribute__((ext_vector_type(8)));
typedef __bf16 pb2_t __attribute__((ext_vector_type(2)));
typedef __bf16 pb8_t __attribute__((ext_vector_type(8)));
typedef float pf2_t __attribute__((ext_vector_type(2)));
typedef float pf4_t __attribute__((ext_vector_type(4)));
typedef float pf16_t __attribute__((ext_vector_type(16)));
typedef uint32_t pu4_t __attribute__((ext_vector_type(4)));

// D = A B + C of 16 x 16 x 32: lane l holds row (A) or column (B) l % 16, contraction slots
// 8 (l / 16) .. + 7; of D column l % 16, rows 4 (l / 16) .. + 3.
template <bool BF>
__device__ __forceinline__ pf4_t mfma16(pu4_t a, pu4_t b, pf4_t c) {
  if constexpr (BF)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(pb8_t, a), __builtin_bit_cast(pb8_t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(ph8_t, a), __builtin_bit_cast(ph8_t, b), c, 0, 0, 0);
}

// The same of 32 x 32 x 16: row or column l % 32, slots 8 (l / 32) .. + 7; of D column l % 32, element r
// is row 8 (r / 4) + 4 (l / 32) + r % 4.
template <bool BF>
__device__ __forceinline__ pf16_t mfma32(pu4_t a, pu4_t b, pf16_t c) {
  if constexpr (BF)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(pb8_t, a), __builtin_bit_cast(pb8_t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(ph8_t, a), __builtin_bit_cast(ph8_t, b), c, 0, 0, 0);
}

// Two weights rounded to 16 bits (to nearest even), x in the low half.
template <bool BF>
__device__ __forceinline__ uint32_t pack2(float x, float y) {
  if constexpr (BF) {
    const pf2_t v = {x, y};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, pb2_t));
  } else {
    const pf2_t v = {x, y};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, ph2_t));
  }
}

// sum + both of a pair of weights as rounded, in fp32 (one instruction).
template <bool BF>
__device__ __forceinline__ float add2(uint32_t w, float sum) {
  if constexpr (BF)
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(pb2_t, w), __builtin_bit_cast(pb2_t, 0x3f803f80u), sum, false);
  else
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(ph2_t, w), __builtin_bit_cast(ph2_t, 0x3c003c00u), sum, false);
}

// Four pairs of 4-bit codes (nibbles n and n + 4 of w, n = 0 .. 3) as fp16((q - z) * s).  q in the last
// bits of the fp16 1024 is 1024 + q, and in bits 4 .. 7 of 64 it is 64 + q, so a pair takes one
// instruction (three for each shift, mask and merge: 19 a word instead of 13); the differences
// from 1024 + z and 64 + z are exact.
struct Kv4Zero {
  ph2_t n1024, n64;  // -(1024 + z), -(64 + z) of a pair
};
__device__ __forceinline__ Kv4Zero kv4_zero(uint32_t z) {  // z: two zero points, 16 bits each
  const ph2_t n = __builtin_bit_cast(ph2_t, z | 0xe400e400u);
  return {n, n + (ph2_t){(_Float16)960.0f, (_Float16)960.0f}};
}
__device__ __forceinline__ pu4_t kv4_pairs(uint32_t w, const Kv4Zero& z, ph2_t s) {
  auto pair = [](uint32_t x, uint32_t mask, uint32_t one) __attribute__((always_inline)) {
    uint32_t r;
    asm("v_and_or_b32 %0, %1, %2, %3" : "=v"(r) : "v"(x), "s"(mask), "v"(one));
    return __builtin_bit_cast(ph2_t, r);
  };
  const uint32_t w8 = w >> 8;
  return (pu4_t){__builtin_bit_cast(uint32_t, (pair(w, 0x000f000fu, 0x64006400u) + z.n1024) * s),
                 __builtin_bit_cast(uint32_t, (pair(w, 0x00f000f0u, 0x54005400u) + z.n64) * s),
                 __builtin_bit_cast(uint32_t, (pair(w8, 0x000f000fu, 0x64006400u) + z.n1024) * s),
                 __builtin_bit_cast(uint32_t, (pair(w8, 0x00f000f0u, 0x54005400u) + z.n64) * s)};
}

// Loads at a wave's base plus a lane's offset plus a constant: one address register.
template <typename T>
__device__ __forceinline__ T load_from(const void* base, uint32_t lane_off, int imm) {
  typedef const __attribute__((address_space(1))) uint8_t* gbyte_t;
  const gbyte_t p = (gbyte_t)base + (uint64_t)lane_off + imm;
  if constexpr (sizeof(T) == 16) return __builtin_bit_cast(T, *(const __attribute__((address_space(1))) pu4_t*)p);
  else if constexpr (sizeof(T) == 8) return __builtin_bit_cast(T, *(const __attribute__((address_space(1))) uint64_t*)p);
  else return *(const __attribute__((address_space(1))) T*)p;
}

// 64 lanes' 16 bytes at base + off (a lane's own), or 16 or 4 bytes at a lane's address, to LDS at
// `to` + 16 (4) lane, with no register between.  Nothing waits for them but an s_waitcnt vmcnt.
__device__ __forceinline__ void copy_lds(const uint8_t* base, uint32_t off, uint32_t to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(off), "s"(base) : "memory", "m0");
}
__device__ __forceinline__ void copy_lds16(const uint8_t* p, uint32_t to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(p) : "memory", "m0");
}
__device__ __forceinline__ void copy_lds4(const uint8_t* p, uint32_t to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(to), "v"(p) : "memory", "m0");
}
typedef __attribute__((address_space(3))) uint8_t* lds_t;

// Eight dims 8 c .. of a row of the pages (the row-by-row path's reads).
template <int HD, int KIND>
__device__ __forceinline__ void paged_eight(const PagedKv& kv, bool value, int page, int64_t row, int c, float (&x)[8]) {
  const uint8_t* p = (value ? kv.v : kv.k) + paged_at(page, kv.page_step);
  if constexpr (KIND == kKv4) {
    const uint32_t w = *(const uint32_t*)(p + row * (HD / 2) + 4 * c);
    const float s = h2f(*(const uint16_t*)((value ? kv.vs : kv.ks) + paged_at(page, kv.scale_step) + 2 * (row * (HD / 32) + c / 4)));
    const float z = (float)(value ? kv.vz : kv.kz)[paged_at(page, kv.zero_step) + row * (HD / 32) + c / 4];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = h2f(f2h(((float)((w >> (4 * e)) & 15u) - z) * s));
  } else {
    const pu4_t u = *(const pu4_t*)(p + (row * HD + 8 * c) * 2);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint16_t h = (uint16_t)(u[e >> 1] >> (16 * (e & 1)));
      x[e] = KIND == kKvBf16 ? bf2f(h) : h2f(h);
    }
  }
}

// What values that are not finite do to a tile whose rows see different keys: in the product a weight of zero times such
// a value is NaN, so they reach the rows that do not see them.  Those keys lie at the tile's ragged ends, which the wave
// looks over: the first in [klo, alo) and the last in [ahi - 1, khi), and the first in the latter whose values
// are NaN in every dim (rows that see it are NaN in any case).
struct PagedSpoiled {
  int low, high, full;
  // Whether a row that sees [lo, hi) has to be computed by itself.
  __device__ __forceinline__ bool reaches(const PagedRange& r) const {
    return (low < r.lo || high >= r.hi) && !(r.lo <= full && full < r.hi);
  }
};
template <int HD, int KIND, typename U>
__device__ __forceinline__ PagedSpoiled paged_spoiled(const PagedKv& kv, const PagedScore& sc, const U& un, int g, int r0, int nrows) {
  PagedSpoiled sp = {0x7fffffff, -1, 0x7fffffff};
  const int i0 = un.seq.len - un.seq.n, capacity = kv.table_width << kv.page_shift;
  const PagedRange ra = paged_range(i0 + r0 / g, un.seq.len, un.prefix, sc.window);
  const PagedRange rb = paged_range(i0 + (r0 + nrows - 1) / g, un.seq.len, un.prefix, sc.window);
  const int klo = ra.lo, alo = rb.lo, ahi = ra.hi, khi = min(rb.hi, capacity);
  const int lane = __lane_id(), mask = (1 << kv.page_shift) - 1;
#pragma unroll 1
  for (int end = 0; end < 2; ++end) {
    const int from = end ? max(ahi - 1, klo) : klo, to = end ? khi : min(alo, khi);
#pragma unroll 1
    for (int j0 = from; j0 < to; j0 += 64) {
      const int j = min(j0 + lane, to - 1);
      int page = kv.table[un.b * kv.table_stride + (j >> kv.page_shift)];
      if ((uint32_t)page >= (uint32_t)kv.num_pages) page = 0;  // (the rows that stood in for it)
      const int64_t r = ((int64_t)un.kvh << kv.page_shift) + (j & mask);
      uint32_t most = 0, least = ~0u;  // of the magnitudes' bits: infinity's 0x7f800000, NaNs' past it
#pragma unroll 1
      for (int c = 0; c < HD / 8; ++c) {
        float x[8];
        paged_eight<HD, KIND>(kv, true, page, r, c, x);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t bits = __builtin_bit_cast(uint32_t, x[e]) & 0x7fffffffu;
          most = max(most, bits);
          least = min(least, bits);
        }
      }
      const uint64_t some = __ballot(most >= 0x7f800000u), every = __ballot(least > 0x7f800000u);
      if (end == 0 && some != 0) sp.low = min(sp.low, j0 + __builtin_ctzll(some));
      if (end == 1 && some != 0) sp.high = min(j0 + 63 - __builtin_clzll(some), to - 1);
      if (end == 1 && every != 0) sp.full = min(sp.full, j0 + __builtin_ctzll(every));
    }
  }
  return sp;
}

// odd, or NaN where y is infinite or NaN.
__device__ __forceinline__ float paged_odd(float odd, float y) { return __builtin_fmaf(y, 0.0f, odd); }

// The running maximum lags: sums are rescaled only where a score passes the maximum they refer to by
// kPagedSlack (so hardly ever after the first steps).  Weights are 2^(score - maximum + raise): in fp16's range at
// most 2^15, with its subnormals 2^-21 below the largest (values are at most 65504, so 2^30 of them fit fp32's sums);
// in bf16, whose values reach fp32's last power of two, at most 2^-16, so that sums of 65536 of the largest do not pass it.
constexpr float kPagedSlack = 8.0f;
template <bool BF>
constexpr float kPagedRaise = BF ? -24.0f : 7.0f;

// One row by itself, every key that it does not see left out: the path of rows that values reach which they do not
// see (PagedSpoiled), rows of at most the two tiles of a sequence's KV head that such a key lies at an end of.  A wave a row:
// lane = key for the scores; for the sums each lane has 8 dims of every G-th key.  Its loops are not unrolled: four times
// made it 8 % faster, and prompts that never come here 2 % slower (biased 4-bit ones 49.0 to 50.0 us).
template <int HD, int KIND, int MOD, typename U>
__device__ __forceinline__ void paged_row(const PagedKv& kv, const PagedScore& sc, const U& un, int g,
                                       const uint16_t* q, int64_t ldq, int heads, int row, uint16_t* out) {
  constexpr bool BF = KIND == kKvBf16;
  constexpr int CH = HD / 8, G = 64 / CH;
  const int lane = __lane_id(), kc = lane % CH, kg = lane / CH;  // (made anew: the loop before this has no register for it)
  const int tok = row / g, head = un.kvh * g + row % g, i = un.seq.len - un.seq.n + tok;
  const uint16_t* qr = q + (int64_t)(un.seq.q0 + tok) * ldq + head * HD;
  const PagedRange rg = paged_range(i, un.seq.len, un.prefix, sc.window);
  const int capacity = kv.table_width << kv.page_shift, mask = (1 << kv.page_shift) - 1, end = min(rg.hi, capacity);
  const float slope2 = MOD != kModNone && sc.slopes ? sc.slopes[head] * 1.4426950408889634f : 0.0f;
  float m = -INFINITY, l = 0.0f, acc[8] = {};
#pragma unroll 1
  for (int j0 = rg.lo; j0 < end; j0 += 64) {
    const int j = j0 + lane;
    const bool see = j < end;
    const int page = see ? kv.table[un.b * kv.table_stride + (j >> kv.page_shift)] : 0;
    const bool bad = (uint32_t)page >= (uint32_t)kv.num_pages;
    const int64_t r = ((int64_t)un.kvh << kv.page_shift) + (j & mask);
    float x = -INFINITY;
    if (see) {
      x = 0.0f;
#pragma unroll 1
      for (int c = 0; c < CH; ++c) {
        float k[8];
        paged_eight<HD, KIND>(kv, false, bad ? 0 : page, r, c, k);
#pragma unroll
        for (int e = 0; e < 8; ++e) x += (BF ? bf2f(qr[8 * c + e]) : h2f(qr[8 * c + e])) * k[e];
      }
      pf4_t one[1] = {{x, x, x, x}};
      float mul = sc.mul;
      if constexpr (MOD != kModNone) mul = paged_scores<MOD, 1, 4>(one, sc, slope2, (float)(i - j), [](int) { return 0; });
      x = bad ? NAN : one[0][0] * mul;
    }
    const float mn = fmaxf(m, wave_max(x)), mu = mn == -INFINITY ? 0.0f : mn;
    const float corr = __builtin_amdgcn_exp2f(m - mu), e = see ? __builtin_amdgcn_exp2f(x - mu + kPagedRaise<BF>) : 0.0f;
    m = mn;
    l = l * corr + wave_sum(e);
#pragma unroll
    for (int d = 0; d < 8; ++d) acc[d] *= corr;
#pragma unroll 1
    for (int n0 = 0; n0 < 64; n0 += G) {
      const int n = n0 + kg;
      const float p = __shfl(e, n, 64);
      const int pg = __shfl(bad ? 0 : page, n, 64);
      if (j0 + n < end) {
        float v[8];
        paged_eight<HD, KIND>(kv, true, pg, ((int64_t)un.kvh << kv.page_shift) + ((j0 + n) & mask), kc, v);
#pragma unroll
        for (int d = 0; d < 8; ++d) acc[d] += p * v[d];
      }
    }
  }
#pragma unroll
  for (int d = 0; d < 8; ++d)
#pragma unroll
    for (int off = CH; off < 64; off *= 2) acc[d] += __shfl_xor(acc[d], off, 64);
  if (kg == 0) {
    uint32_t w[4];
#pragma unroll
    for (int d = 0; d < 4; ++d)
      w[d] = pack2<BF>(l == 0.0f ? 0.0f : acc[2 * d] / l, l == 0.0f ? 0.0f : acc[2 * d + 1] / l);
    *(uint4*)(out + ((int64_t)(un.seq.q0 + tok) * heads + head) * HD + 8 * kc) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// Arrival of a piece at its tile's counter, its partial sums complete (every thread has waited for
// its stores); true in every thread of the last of `pieces`, which leaves the counter at zero.
__device__ __forceinline__ bool paged_arrive(uint32_t* counter, int pieces, int* flag) {
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  if (threadIdx.x == 0) {
    const uint32_t n = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    *flag = n == (uint32_t)(pieces - 1);
    if (n == (uint32_t)(pieces - 1)) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  return *flag != 0;
}

// The factor that brings sums of maximum m and total l to the maximum mm.  Without keys (-inf and
// 0): 0; a total of NaN (NaN scores do not show in a maximum): 1.
__device__ __forceinline__ float paged_weight(float m, float l, float mm) {
  return m == -INFINITY ? (l == 0.0f ? 0.0f : 1.0f) : __builtin_amdgcn_exp2f(m - mm);
}

// A piece's record in the workspace: [rows][HD] sums of weight times value, [rows] (maximum, total).
template <int HD>
__host__ __device__ constexpr int paged_slot(int rows) {
  return rows * (HD + 2);
}
__device__ __forceinline__ void store_dev2(float* p, float x, float y) {
  __hip_atomic_store((uint64_t*)p, (uint64_t)__builtin_bit_cast(uint32_t, x) | (uint64_t)__builtin_bit_cast(uint32_t, y) << 32,
                     __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 load_dev2(const float* p) {
  const uint64_t v = __hip_atomic_load((const uint64_t*)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return make_float2(__builtin_bit_cast(float, (uint32_t)v), __builtin_bit_cast(float, (uint32_t)(v >> 32)));
}

// A row's pieces (slot_of(p) the p-th's record) joined in their order, whatever order they arrived in:
// NI times four dims of the sum of weight times value (two at `at` in the records, two `next` after them; the
// n-th four n `step` after the first), and the total.  The loads of U pieces are in flight together.
template <int HD, int ROWS, int U, int NI, typename F>
__device__ __forceinline__ float paged_join_by(const float* slots, F slot_of, int pieces, int row, int at, int next, int step,
                                               float (&v)[NI][4]) {
  float mm = -INFINITY, den = 0.0f;
#pragma unroll
  for (int i = 0; i < NI; ++i) v[i][0] = v[i][1] = v[i][2] = v[i][3] = 0.0f;
  for (int p0 = 0; p0 < pieces; p0 += U) {
    float2 ml[U], x[U][NI][2];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float* p = slots + (int64_t)slot_of(min(p0 + u, pieces - 1)) * paged_slot<HD>(ROWS);
      ml[u] = load_dev2(p + ROWS * HD + 2 * row);
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        x[u][i][0] = load_dev2(p + at + i * step);
        x[u][i][1] = load_dev2(p + at + i * step + next);
      }
    }
    float mn = mm;
#pragma unroll
    for (int u = 0; u < U; ++u) mn = fmaxf(mn, ml[u].x);
    const float corr = paged_weight(mm, den, mn);
    den *= corr;
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) v[i][e] *= corr;
    mm = mn;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (p0 + u >= pieces) continue;
      const float f = paged_weight(ml[u].x, ml[u].y, mm);
      den += f * ml[u].y;
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        v[i][0] += f * x[u][i][0].x;
        v[i][1] += f * x[u][i][0].y;
        v[i][2] += f * x[u][i][1].x;
        v[i][3] += f * x[u][i][1].y;
      }
    }
  }
  return den;
}

// The host side of a launch, shared by the kernels' translation units.
struct PagedLaunch {
  PagedKv kv;
  PagedScore sc;
  const uint16_t* q;
  int64_t ldq;
  uint16_t* out;
  int heads, g, kind, hd, units;  // units: the grid
  uint32_t* counters;
  float* slots;
  hipStream_t stream;
  int mod;
  bool wide;  // more key steps than 2^29 are possible
};
// Few rows a sequence (drafted tokens times heads of a KV head): tiles of 16 or 32 rows, as many
// workgroups as are resident at once, and two partial tiles each at most.
constexpr int kFewKeys = 128;
// workgroups a compute unit, by their registers: 4-bit keys of 128 dims fit three in (48 users 121 us; two, from
// registers, 127); those of 64 dims keep more in flight as two (65536 keys 25.7 us, as three, with spills, 31.3); with
// tiles of 32 rows two, but for 16-bit keys of 128 dims, whose tiles in flight take the registers of two
// (48 sequences of 8 drafted tokens on 8192 keys: 4 bits 153 us, one workgroup 199; 16 bits 290, at the memory's rate)
constexpr int few_resident(int kind, int hd, int rows) {
  return rows == 32 ? (hd == 128 && kind != kKv4 ? 1 : 2) : kind == kKv4 && hd == 128 ? 3 : 2;
}
constexpr int few_groups(int kind, int hd, int rows) { return 256 * few_resident(kind, hd, rows); }
constexpr int kFewSlotRows = 2 * 512 * 32;  // the most: two records each, of 512 workgroups of 32 rows
static_assert(2 * few_groups(kKv4, 128, 16) * 16 <= kFewSlotRows && 2 * few_groups(kKv4, 64, 32) * 32 <= kFewSlotRows, "");
int launch_paged_few(const PagedLaunch& a, int rows);
// Many rows a sequence (prompts): tiles of 128 rows, or of 64 up to kManyBig tiles of 128.  Tiles of more
// than 1.5 kManyMinKeys keys may be cut where there are few: into about kManyTarget pieces in all (four times as many,
// when a join cost twice what it does: 1536 tokens 67 us, not 30; twice: 512 tokens on 32768 345, not 279).
constexpr int kManyWaves = 4, kManyKeys = 16 * kManyWaves;  // keys of a step: a wave copies 16
constexpr int kManyBig = 512, kManyMinKeys = 512, kManyTarget = 256, kManySlots = 2 * kManyTarget;
int launch_paged_many(const PagedLaunch& a, int rows);

// The tile and the grid of a call.
struct PagedGrid {
  int rows;       // of a tile
  int64_t tiles;  // at most this many
  int64_t units;  // workgroups
  bool wide;      // the tiles' key steps may be more than 2^29
};
// Rows a sequence has on average pick the tile, the least that holds them: 16 or 32 rows of the few (32
// sequences of 2048 keys, 24 heads of 128 on 8: 18 rows 29.5 us, as two tiles of 16 43; on 4-bit pages 30 rows
// 37.8, of 64 52), or of the many (60 rows 30 us, as two tiles of 32 58).  Tiles of 64, whose key steps two
// pairs of waves share, while 128 would leave compute units idle: up to kManyBig tiles of 128 (777 tokens: 64
// rows 17.4 us, 128 20.2; four such prompts: 39.5 and 33.0).
inline PagedGrid paged_grid(const PagedKv& kv, int64_t tokens, int g, int kind, int hd) {
  PagedGrid grid;
  const int64_t all = tokens * g, seqs = std::min<int64_t>(tokens, kv.batch);
  grid.rows = all <= 16 * seqs ? 16 : all <= 32 * seqs ? 32 : kv.kv_heads * all <= 128 * kManyBig ? 64 : 128;
  const bool many = grid.rows >= 64;
  const int keys = many ? kManyKeys : kFewKeys;
  // each tile of at most as many key steps as its table has
  grid.tiles = kv.kv_heads * (all / grid.rows + seqs);
  const int64_t cuts = (((int64_t)kv.table_width << kv.page_shift) + keys - 1) / keys;
  // the few rows' workgroups: as many a compute unit as are resident, but past one only as long as a tile's join,
  // which is one workgroup's, has no more than some 1024 rows of partial sums (drafts of 24 rows on 8192 4-bit keys: 256
  // workgroups 32 us, 512 48; 48 such sequences: 199 and 153)
  const int64_t joined = grid.tiles * 1024 / std::min<int64_t>(grid.rows, (all + seqs - 1) / seqs);
  const int64_t groups = std::min<int64_t>(few_groups(kind, hd, std::min(grid.rows, 32)), 256 * std::max<int64_t>(1, joined / 256));
  grid.units = std::min(many ? grid.tiles + kManyTarget + 16 : groups, grid.tiles * cuts);
  grid.wide = grid.tiles * cuts >= (1LL << 29);
  return grid;
}

}  // namespace spectra
