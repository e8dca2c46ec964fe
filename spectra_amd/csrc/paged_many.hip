// Attention over a paged KV cache for many rows a sequence: prompts, and chunks of them on their
// context, in tiles of 64 or 128 rows (the tokens' query heads of one KV head beside each other, so the
// heads that share keys share their loads).  The mathematics is the few rows' kernel's: one pass with a running
// maximum, scores transposed, S^T = K Q^T (32 x 32 x 16: K rows as A, the lane's row as B), so a lane holds 16
// scores of one row a tile, maxima cross only to the lane 32 away, and the exponentials are already the B
// operand of O^T = V^T P^T when the contraction takes the keys in the accumulator's order.
//
// Bound by the matrix cores and the exponentials between them (4 head_dim flops and one exponential a score,
// 8 cycles a wave, a quarter of a 32 x 32 x 16 matrix instruction): a prompt of 8192 tokens
// (24 heads of 128) does 412 GFLOP in 403 to 430 us, 960 to 1022 TFLOP/s where a large matrix product reaches
// 1145; there the matrix cores are busy half of the time at a clock that their power lowers.  With a cap (two
// exponentials and a reciprocal a score) 670 to 720 TFLOP/s; 4-bit pages with a bias and heads of 64 250 to 280.  A prompt of
// 777 tokens takes 18 us: 13 key steps one after another for its last rows, and fewer tiles than would
// hide their latencies.
//
// A workgroup is 4 waves of 32 rows each, or for 64 rows two pairs that take the halves of a step's keys; steps
// are 64 keys, in two buffers each of K and V.  16-bit rows go from memory to LDS directly, with no
// register between (8192 tokens: 439 us, 498 through registers), K's and V's chunks turned so that what
// lanes read at once lies on different banks (no conflicts are counted); V is read transposed by the LDS
// itself.  4-bit rows are expanded on the way, once for all rows.  The loop runs one step ahead: the next
// step's Q K^T stands beside this step's exponentials, the copies between them (777 tokens 18.6 us, 19.8 with
// the copies before them).
//
// Roundings: as the few rows' kernel.
#include <cmath>

#include "paged_attend.h"

namespace spectra {

// The buffers of keys, then of values: two each, a row of 16-byte chunks a key.  Chunk c of key r lies
// at c ^ k_turn(r) in K's rows (16 rows' equal chunks, which lanes read at once, on different banks)
// and at c ^ v_turn(r) in V's (four rows' 64 bytes, read transposed, on different banks).
template <int HD>
constexpr int many_lds() {
  return 4 * kManyKeys * HD * 2;
}
template <int HD>
__device__ __forceinline__ int k_turn(int r) {
  return HD == 128 ? r & 15 : (r >> 1) & 7;
}
template <int HD>
__device__ __forceinline__ int v_turn(int r) {
  return HD == 128 ? (r & 3) << 2 : (r & 2) << 1;
}

typedef short ps4_t __attribute__((ext_vector_type(4)));

// Four keys' values of one dim: of each 16 lanes, lanes 4 k .. 4 k + 3 name 4 dims each of key k, and
// lane i gets dim i of the four.
__device__ __forceinline__ uint2 read_turned(const uint8_t* p) {
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) ps4_t*)(lds_t)p));
}

template <int HD, int KIND, int MOD, int QH>
__global__ void __launch_bounds__(64 * kManyWaves, 2)
    paged_many_kernel(const PagedKv kv, const PagedScore sc, const uint16_t* __restrict__ q, int64_t ldq, int g, int heads,
                      uint32_t* __restrict__ counters, float* __restrict__ slots, uint16_t* __restrict__ out) {
  constexpr bool Q4 = KIND == kKv4, BF = KIND == kKvBf16;
  constexpr int CH = HD / 8, KS = HD / 16, DT = HD / 32;  // 8-dim chunks, 16-dim steps, 32-dim tiles
  constexpr int W = kManyWaves, KEYS = kManyKeys, THREADS = 64 * W;
  constexpr int KL = KEYS * CH / THREADS;                 // K chunks a thread copies
  constexpr int KH = W / QH;                              // waves that share a step's keys
  constexpr int ROWS = 32 * QH, TL = KEYS / (32 * KH);    // 32-key tiles of a step that a wave takes
  constexpr int ROWB = Q4 ? HD / 2 : 2 * HD;
  extern __shared__ __align__(16) uint8_t lds[];
  __shared__ int flag;
  __shared__ uint32_t redo[QH];
  const int tid = threadIdx.x, lane = tid & 63, wave = sread(tid >> 6), gh = lane >> 5, ln = lane & 31;
  const int qh = wave % QH, kh = wave / QH;  // the wave's 32 rows, and its share of a step's keys
  PagedUnit un;
  if (!paged_unit<Wave>(kv, g, ROWS, KEYS, kManyMinKeys / KEYS, kManyTarget, kManySlots, sc, blockIdx.x, lane, un)) return;
  const PagedSeq sq = un.seq;
  const int r0 = un.tile * ROWS, nrows = min(ROWS, sq.n * g - r0);
  const int tok0 = sread(r0 / g), tok1 = sread((r0 + nrows - 1) / g), i0 = sq.len - sq.n;
  const int capacity = kv.table_width << kv.page_shift, pmask = (1 << kv.page_shift) - 1;
  // keys that some row of the tile sees
  const PagedRange ra = paged_range(i0 + tok0, sq.len, un.prefix, sc.window);
  const PagedRange rb = paged_range(i0 + tok1, sq.len, un.prefix, sc.window);
  const int klo = ra.lo, khi = min(rb.hi, capacity), kbeg = klo & ~(KEYS - 1);
  const int steps = khi > kbeg ? (khi - kbeg + KEYS - 1) / KEYS : 0;
  const int sbeg = sread((int)((int64_t)steps * un.piece / un.pieces));
  const int send = sread((int)((int64_t)steps * (un.piece + 1) / un.pieces));
  // keys that all of this wave's rows see; the lane's row
  const int wr0 = min(32 * qh, nrows - 1), wr1 = min(32 * qh + 31, nrows - 1);
  const PagedRange wa = paged_range(i0 + (r0 + wr0) / g, sq.len, un.prefix, sc.window);
  const PagedRange wb = paged_range(i0 + (r0 + wr1) / g, sq.len, un.prefix, sc.window);
  const int alo = wb.lo, ahi = min(wa.hi, capacity);
  const bool ok = 32 * qh + ln < nrows;
  const int rr = r0 + min(32 * qh + ln, nrows - 1), tok = rr / g, head = un.kvh * g + (rr - tok * g);
  const PagedRange rg = paged_range(i0 + tok, sq.len, un.prefix, sc.window);
  const float slope2 = MOD != kModNone && sc.slopes ? sc.slopes[head] * 1.4426950408889634f : 0.0f;
  const int pos = i0 + tok - 4 * gh;
  pu4_t qf[KS];
  {
    const uint16_t* qr = q + (int64_t)(sq.q0 + tok) * ldq + head * HD + 8 * gh;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const pu4_t x = *(const pu4_t*)(qr + 16 * s);
      qf[s] = Q4 ? (pu4_t){__builtin_amdgcn_perm(x[2], x[0], 0x05040100u), __builtin_amdgcn_perm(x[2], x[0], 0x07060302u),
                           __builtin_amdgcn_perm(x[3], x[1], 0x05040100u), __builtin_amdgcn_perm(x[3], x[1], 0x07060302u)}
                 : x;
    }
  }

  // ---- staging: a step is a block of 16 keys a wave, in one page: a wave copies its block and needs one
  // page id a step.  16-bit rows go to LDS directly; 4-bit ones through registers, where
  // they are expanded (K's in the order of its codes, as Q is; V's put back in order).
  const int* tab = kv.table + un.b * kv.table_stride;
  auto page_of = [&](int k0) __attribute__((always_inline)) {
    return sread(sload(tab + min((k0 + 16 * wave) >> kv.page_shift, kv.table_width - 1)));
  };
  constexpr int KB = KEYS * HD * 2, RPI = 64 / CH;  // bytes of a buffer, rows of 64 lanes' chunks
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_t)lds;
  const int kc = lane % CH, krow = lane / CH;
  constexpr uint32_t nan2 = BF ? 0x7fc07fc0u : 0x7e007e00u;
  struct Codes {
    uint32_t w[KL], s[KL], z[KL];
  } kcodes, vcodes;
  // where a wave's block of step k0 begins in K (and V, their pages lying alike)
  auto place = [&](int k0, int id) __attribute__((always_inline)) {
    const int row = (un.kvh << kv.page_shift) + ((k0 + 16 * wave) & pmask);
    return paged_at((uint32_t)id < (uint32_t)kv.num_pages ? id : 0, kv.page_step) + row * ROWB;
  };
  auto copy = [&](bool value, uint64_t at, int buf, int i) __attribute__((always_inline)) {
    const int r = krow + i * RPI;
    const uint8_t* base = (value ? kv.v : kv.k) + at;
    const uint32_t off = r * ROWB + 16 * (kc ^ (value ? v_turn<HD>(r) : k_turn<HD>(r)));
    const uint32_t to = lds0 + (value ? 2 * KB : 0) + buf * KB + (16 * wave + i * RPI) * HD * 2;
    copy_lds(base, off, to);
  };
  auto fetch = [&](bool value, int k0, int id, int buf, Codes& cd) __attribute__((always_inline)) {
    if constexpr (Q4) {
      const int pg = (uint32_t)id < (uint32_t)kv.num_pages ? id : 0, row = (un.kvh << kv.page_shift) + ((k0 + 16 * wave) & pmask);
      const uint8_t* base = (value ? kv.v : kv.k) + paged_at(pg, kv.page_step) + row * ROWB;
      const uint8_t* sb = (value ? kv.vs : kv.ks) + paged_at(pg, kv.scale_step) + row * (HD / 16);
      const uint8_t* zb = (value ? kv.vz : kv.kz) + paged_at(pg, kv.zero_step) + row * (HD / 32);
#pragma unroll
      for (int i = 0; i < KL; ++i) {
        cd.w[i] = load_from<uint32_t>(base, krow * ROWB + 4 * kc, i * RPI * ROWB);
        cd.s[i] = load_from<uint16_t>(sb, 2 * (krow * (HD / 32) + kc / 4), i * RPI * (HD / 16));
        cd.z[i] = load_from<uint8_t>(zb, krow * (HD / 32) + kc / 4, i * RPI * (HD / 32));
      }
    } else {
#pragma unroll
      for (int i = 0; i < KL; ++i) copy(value, place(k0, id), buf, i);
    }
  };
  // What was fetched is in place, with NaN for keys of a page that is not there, and zeros for values
  // of keys that no row sees (they must not reach the product).
  auto land = [&](bool value, int k0, int id, int buf, const Codes& cd) __attribute__((always_inline)) {
    uint8_t* to = lds + (value ? 2 * KB : 0) + buf * KB;
    const bool edge = value && (k0 < klo || k0 + KEYS > khi), bad = !value && (uint32_t)id >= (uint32_t)kv.num_pages;
    if (!Q4 && !edge && !bad) return;
#pragma unroll
    for (int i = 0; i < KL; ++i) {
      const int r = krow + i * RPI, key = 16 * wave + r;
      const bool out = edge && (k0 + key < klo || k0 + key >= khi);
      pu4_t x = {0, 0, 0, 0};
      if constexpr (Q4) {
        const uint32_t s = out ? 0 : cd.s[i];
        x = kv4_pairs(cd.w[i], kv4_zero(cd.z[i] | cd.z[i] << 16), __builtin_bit_cast(ph2_t, s | s << 16));
        if (value)
          x = (pu4_t){__builtin_amdgcn_perm(x[1], x[0], 0x05040100u), __builtin_amdgcn_perm(x[3], x[2], 0x05040100u),
                      __builtin_amdgcn_perm(x[1], x[0], 0x07060302u), __builtin_amdgcn_perm(x[3], x[2], 0x07060302u)};
      }
      if (bad) x = (pu4_t){nan2, nan2, nan2, nan2};
      if (Q4 || bad || out) *(pu4_t*)(to + key * HD * 2 + 16 * (kc ^ (value ? v_turn<HD>(key) : k_turn<HD>(key)))) = x;
    }
  };

  pf16_t o[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[d][r] = 0.0f;
  float m = -INFINITY, l = 0.0f;
  // a wave's scores of a step: element r of tile t is key kw + 32 t + 8 (r / 4) + 4 gh + r % 4
  constexpr int NK = TL * KS, NV = 2 * TL * DT;  // matrix instructions of Q K^T and of P V, and operands in flight
  constexpr int RING = 4, RINGV = 8;
  const int kbase = (32 * TL * kh + ln) * HD * 2;
  auto read_k = [&](int buf, int i) __attribute__((always_inline)) {
    const int t = i / KS, st = i % KS;
    return *(const pu4_t*)(lds + buf * KB + kbase + 64 * t * HD + 16 * ((2 * st + gh) ^ k_turn<HD>(ln)));
  };
  const int vi = lane & 15, vbase = (32 * TL * kh + 4 * gh + (vi >> 2)) * HD * 2 + 8 * (vi & 1);
  const int vchunk = 2 * ((lane >> 4) & 1) + ((vi & 3) >> 1);
  auto read_v = [&](int buf, int i) __attribute__((always_inline)) {  // 16 keys i / DT, 32 dims i % DT
    const uint8_t* p = lds + 2 * KB + buf * KB + vbase + 16 * ((4 * (i % DT) + vchunk) ^ v_turn<HD>(vi >> 2)) + 32 * (i / DT) * HD;
    const uint2 x = read_turned(p), y = read_turned(p + 16 * HD);
    return (pu4_t){x.x, x.y, y.x, y.y};
  };
  constexpr pf16_t zero = {};
  auto product = [&](pf16_t (&s)[TL], int buf) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NK; ++i) s[i / KS] = mfma32<BF>(read_k(buf, i), qf[i % KS], i % KS == 0 ? zero : s[i / KS]);
  };
  // One step: softmax of its scores s, their product with its values, and the next step's scores
  // into sn (past the last: of whatever its buffer holds, used by nothing).  The order is written out
  // (the compiler would wait for every operand where it is used): operands are read RING instructions ahead, and the exponentials, and the
  // 2 KL copies `beside`, stand between the matrix instructions of Q K^T, which run beneath them.
  auto step = [&](int k0, pf16_t (&s)[TL], pf16_t (&sn)[TL], int buf, auto beside) __attribute__((always_inline)) {
    const int kw = k0 + 32 * TL * kh;  // this wave's keys
    pu4_t ring[RINGV];
#pragma unroll
    for (int i = 0; i < RING; ++i) ring[i] = read_k(buf ^ 1, i);
    __builtin_amdgcn_sched_barrier(0);
    float mul = sc.mul;
    if constexpr (MOD != kModNone) mul = paged_scores<MOD, TL, 16>(s, sc, slope2, (float)(pos - kw), [](int r) { return 8 * (r >> 2) + (r & 3); });
    if (kw < alo || kw + 32 * TL > ahi) {
      const int from = rg.lo - kw - 4 * gh, to = min(rg.hi, capacity) - kw - 4 * gh;
#pragma unroll
      for (int t = 0; t < TL; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int at = 32 * t + 8 * (r >> 2) + (r & 3);
          if (at < from || at >= to) s[t][r] = -INFINITY;
        }
    }
    float mn = -INFINITY;
#pragma unroll
    for (int t = 0; t < TL; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) mn = fmaxf(mn, s[t][r]);
    mn = fmaxf(mn, lane_xor<32>(mn, lane)) * mul;
    if (__ballot(mn > m + kPagedSlack) != 0) {
      mn = fmaxf(m, mn);
      const float corr = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.0f : mn));
      l *= corr;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] *= corr;
      m = mn;
    }
    const float mu = m == -INFINITY ? 0.0f : m - kPagedRaise<BF>;
    pu4_t pf[TL][2];
    auto weights = [&](int i) __attribute__((always_inline)) {  // the i-th pair
      const int t = i >> 3, r = 2 * (i & 7);
      const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][r], mul, -mu));
      const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][r + 1], mul, -mu));
      const uint32_t w = pack2<BF>(e0, e1);
      l = add2<BF>(w, l);
      pf[t][r >> 3][(r & 7) >> 1] = w;
    };
#pragma unroll
    for (int i = 0; i < NK; ++i) {
      sn[i / KS] = mfma32<BF>(ring[i % RING], qf[i % KS], i % KS == 0 ? zero : sn[i / KS]);
      ring[i % RING] = i + RING < NK ? read_k(buf ^ 1, i + RING) : read_v(buf, i + RING - NK);  // (NK is a multiple of RING)
#pragma unroll
      for (int j = i * 8 * TL / NK; j < (i + 1) * 8 * TL / NK; ++j) weights(j);
#pragma unroll
      for (int j = i * 2 * KL / NK; j < (i + 1) * 2 * KL / NK; ++j) beside(j);
      __builtin_amdgcn_sched_barrier(0);
    }
    // O^T += V^T P^T, 16 keys and 32 dims at a time; keys 16 u + {4 gh + 0 .. 3, 8 + 4 gh + 0 .. 3}
#pragma unroll
    for (int i = RING; i < RINGV; ++i) ring[i] = read_v(buf, i);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int u = i / DT;
      o[i % DT] = mfma32<BF>(ring[i % RINGV], pf[u >> 1][u & 1], o[i % DT]);
      if (i + RINGV < NV) ring[i % RINGV] = read_v(buf, i + RINGV);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  if (sbeg < send) {
    // At step s the buffers hold K of s + 1 and V of s; K of s + 2 and V of s + 1 are on their way.
    int k0 = kbeg + sbeg * KEYS;
    const int kend = kbeg + send * KEYS;
    pf16_t s0[TL], s1[TL];
    int id0 = page_of(k0), id1 = page_of(k0 + KEYS), id2 = page_of(k0 + 2 * KEYS);
    auto wait = [&]() __attribute__((always_inline)) { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); };
    Codes kfirst;
    fetch(false, k0, id0, 0, kfirst);
    fetch(true, k0, id0, 0, vcodes);
    fetch(false, k0 + KEYS, id1, 1, kcodes);
    wait();
    land(false, k0, id0, 0, kfirst);
    land(true, k0, id0, 0, vcodes);
    land(false, k0 + KEYS, id1, 1, kcodes);
    __syncthreads();
    product(s0, 0);
    __syncthreads();  // (K of the first step is read: its buffer is free)
    uint64_t at1 = place(k0 + KEYS, id1);
    auto turn = [&](pf16_t (&s)[TL], pf16_t (&sn)[TL], int buf) __attribute__((always_inline)) {
      const bool more = k0 + KEYS < kend;
      const uint64_t at2 = place(k0 + 2 * KEYS, id2);
      if constexpr (Q4) {
        if (more) {
          fetch(false, k0 + 2 * KEYS, id2, buf, kcodes);
          fetch(true, k0 + KEYS, id1, buf ^ 1, vcodes);
        }
      }
      const int id3 = page_of(k0 + 3 * KEYS);
      step(k0, s, sn, buf, [&](int j) __attribute__((always_inline)) {
        if constexpr (!Q4) copy(j >= KL, j < KL ? at2 : at1, j < KL ? buf : buf ^ 1, j % KL);
      });
      wait();  // (the last step's copies, too, which are of whatever comes next: LDS is used again)
      if (!more) return false;
      land(false, k0 + 2 * KEYS, id2, buf, kcodes);
      land(true, k0 + KEYS, id1, buf ^ 1, vcodes);
      __syncthreads();
      id1 = id2;
      id2 = id3;
      at1 = at2;
      k0 += KEYS;
      return true;
    };
    while (turn(s0, s1, 0) && turn(s1, s0, 1)) {
    }
  }

  l += lane_xor<32>(l, lane);
  if constexpr (KH > 1) {  // the waves that shared the keys meet
    float4* red = (float4*)lds;  // [wave past the first QH][4 DT][lane]
    float2* ml = (float2*)(lds + (W - QH) * 16 * DT * 64 * 4);
    static_assert((W - QH) * (16 * DT * 64 * 4 + 64 * 8) <= many_lds<HD>(), "their sums fit the buffers");
    __syncthreads();
    if (kh > 0) {
      const int at = wave - QH;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          red[(at * 4 * DT + 4 * d + r) * 64 + lane] = make_float4(o[d][4 * r], o[d][4 * r + 1], o[d][4 * r + 2], o[d][4 * r + 3]);
      ml[at * 64 + lane] = make_float2(m, l);
    }
    __syncthreads();
    if (kh == 0) {
      float2 x[KH - 1];
      float mm = m;
#pragma unroll
      for (int k = 0; k < KH - 1; ++k) {
        x[k] = ml[(k * QH + qh) * 64 + lane];
        mm = fmaxf(mm, x[k].x);
      }
      const float c0 = paged_weight(m, l, mm);
      l *= c0;
      m = mm;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] *= c0;
#pragma unroll
      for (int k = 0; k < KH - 1; ++k) {
        const float c = paged_weight(x[k].x, x[k].y, mm);
        l += c * x[k].y;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float4 y = red[((k * QH + qh) * 4 * DT + 4 * d + r) * 64 + lane];
            o[d][4 * r] += c * y.x;
            o[d][4 * r + 1] += c * y.y;
            o[d][4 * r + 2] += c * y.z;
            o[d][4 * r + 3] += c * y.w;
          }
      }
    }
  }
  const bool mixed = tok1 > tok0;  // rows that see different keys
  uint32_t again = 0;              // rows that came out infinite or NaN
  if (un.pieces == 1) {
    const bool past = rg.hi > capacity;
    if (__ballot(l == 0.0f) != 0) {  // rows without keys or scores, whatever the values are
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] = l == 0.0f ? 0.0f : o[d][r];
      l = l == 0.0f ? 1.0f : l;
    }
    const float inv = past ? NAN : 1.0f / l;
    float odd = 0.0f;
    if (ok && kh == 0) {
      uint16_t* orow = out + ((int64_t)(sq.q0 + tok) * heads + head) * HD;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int r = 0; r < 4; ++r) {  // dims 32 d + 8 r + 4 gh + 0 .. 3
          float y[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            y[e] = o[d][4 * r + e] * inv;
            odd = paged_odd(odd, y[e]);
          }
          *(uint2*)(orow + 32 * d + 8 * r + 4 * gh) = make_uint2(pack2<BF>(y[0], y[1]), pack2<BF>(y[2], y[3]));
        }
    }
    const uint64_t b = __ballot(odd != odd && l == l && !past);  // (where the total is NaN the row's own scores are)
    again = (uint32_t)(b | (b >> 32));
  } else {
    const int first = un.slot - un.piece;
    if (tid < QH) redo[tid] = 0;
    if (ok && kh == 0) {  // (a record's sums as the lanes hold them: pairs of dims, a wave's beside each other)
      float* p = slots + (int64_t)un.slot * paged_slot<HD>(ROWS);
      float* at = p + qh * 32 * HD + 2 * lane;
#pragma unroll
      for (int i = 0; i < 4 * DT; ++i) {
        store_dev2(at + 256 * i, o[i >> 2][4 * (i & 3)], o[i >> 2][4 * (i & 3) + 1]);
        store_dev2(at + 256 * i + 128, o[i >> 2][4 * (i & 3) + 2], o[i >> 2][4 * (i & 3) + 3]);
      }
      if (gh == 0) store_dev2(p + ROWS * HD + 2 * (32 * qh + ln), m, l);
    }
    if (!paged_arrive(counters + first, un.pieces, &flag)) return;
    // a wave: NI parts of four dims of each 32 rows, whose loads are in flight together (one part after another
    // would be a round trip past the L2 each)
    constexpr int NI = 4 * DT / W;
    for (int row = ln; row < nrows; row += 32) {
      const int r = r0 + row, t = r / g, h = un.kvh * g + (r - t * g), part = (row >> 5) * 4 * DT + wave;
      float v[NI][4];
      const float den = paged_join_by<HD, ROWS, 4, NI>(slots, [&](int p) { return first + p; }, un.pieces, row, 256 * part + 2 * lane,
                                                       128, 256 * W, v);
      const bool past = paged_range(i0 + t, sq.len, un.prefix, sc.window).hi > capacity;
      float odd = 0.0f;
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        float y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          y[e] = past ? NAN : den == 0.0f ? 0.0f : v[i][e] / den;
          odd = paged_odd(odd, y[e]);
        }
        const int d = 8 * (wave + W * i) + 4 * gh;
        *(uint2*)(out + ((int64_t)(sq.q0 + t) * heads + h) * HD + d) = make_uint2(pack2<BF>(y[0], y[1]), pack2<BF>(y[2], y[3]));
      }
      if (odd != odd && den == den && !past) atomicOr(&redo[row >> 5], 1u << (row & 31));
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < QH; ++h) again |= redo[h];
  }
  again = sread(again);
  if (!mixed || again == 0) return;
  const PagedSpoiled sp = paged_spoiled<HD, KIND>(kv, sc, un, g, r0, nrows);
#pragma unroll 1
  for (int h = 0; h < QH; ++h) {  // (a joined tile's rows by all waves)
    uint32_t r = un.pieces == 1 ? (h == qh ? again : 0) : redo[h] & (0x11111111u << wave);
    for (r = sread(r); r != 0; r &= r - 1) {
      const int row = r0 + 32 * h + __builtin_ctz(r);
      if (sp.reaches(paged_range(i0 + row / g, sq.len, un.prefix, sc.window))) paged_row<HD, KIND, MOD>(kv, sc, un, g, q, ldq, heads, row, out);
    }
  }
}

template <int HD, int KIND, int MOD, int QH>
static int launch_many(const PagedLaunch& a) {
  const void* kern = (const void*)paged_many_kernel<HD, KIND, MOD, QH>;
  if (int st = ensure_lds_limit(kern); st != SPECTRA_OK) return st;
  paged_many_kernel<HD, KIND, MOD, QH><<<dim3((unsigned)a.units), dim3(64 * kManyWaves), many_lds<HD>(), a.stream>>>(
      a.kv, a.sc, a.q, a.ldq, a.g, a.heads, a.counters, a.slots, a.out);
  SPECTRA_HIP_CHECK(hipGetLastError());
  return SPECTRA_OK;
}
template <int HD, int KIND>
static int launch_many_of(const PagedLaunch& a, int rows) {
  if (a.mod == kModLargeCap) return rows == 64 ? launch_many<HD, KIND, kModLargeCap, 2>(a) : launch_many<HD, KIND, kModLargeCap, 4>(a);
  if (rows == 64) return a.mod ? launch_many<HD, KIND, kMod, 2>(a) : launch_many<HD, KIND, kModNone, 2>(a);
  return a.mod ? launch_many<HD, KIND, kMod, 4>(a) : launch_many<HD, KIND, kModNone, 4>(a);
}
int launch_paged_many(const PagedLaunch& a, int rows) {
  if (a.hd == 64)
    return a.kind == kKv4      ? launch_many_of<64, kKv4>(a, rows)
           : a.kind == kKvBf16 ? launch_many_of<64, kKvBf16>(a, rows)
                               : launch_many_of<64, kKvF16>(a, rows);
  return a.kind == kKv4      ? launch_many_of<128, kKv4>(a, rows)
         : a.kind == kKvBf16 ? launch_many_of<128, kKvBf16>(a, rows)
                             : launch_many_of<128, kKvF16>(a, rows);
}

}  // namespace spectra

using namespace spectra;

namespace {
size_t slot_floats(int hd) {
  const size_t few = kFewSlotRows, many = (size_t)kManySlots * 128;
  return (few > many ? few : many) * (hd + 2);
}
}  // namespace

extern "C" size_t spectra_paged_attend_workspace(int32_t head_dim) {
  if (head_dim != 64 && head_dim != 128) return 0;
  return SPECTRA_PAGED_COUNTER_BYTES + slot_floats(head_dim) * sizeof(float);
}

extern "C" int spectra_paged_attend(const spectra_paged_kv_t* kv, const void* q, int64_t ldq, int64_t tokens,
                                    int32_t heads, float scale, float cap, int32_t window, const float* slopes,
                                    const int32_t* prefix, void* workspace, size_t workspace_bytes, void* out,
                                    spectra_stream_t stream) {
  static_assert(8 * few_groups(kKv4, 128, 16) <= SPECTRA_PAGED_COUNTER_BYTES && 4 * kManySlots <= SPECTRA_PAGED_COUNTER_BYTES,
                "a counter for every slot");
  PagedLaunch a;
  if (int st = paged_args(kv, tokens, heads, &a.kv); st != SPECTRA_OK) return st;
  SPECTRA_REQUIRE(q && out, "NULL pointer");
  SPECTRA_REQUIRE(ldq >= (int64_t)heads * kv->head_dim && ldq % 8 == 0, "q token stride too small or not a multiple of 8");
  SPECTRA_REQUIRE((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) % 16 == 0,
                  "q and out must be 16-byte aligned");
  SPECTRA_REQUIRE(reinterpret_cast<uintptr_t>(slopes) % 4 == 0 && reinterpret_cast<uintptr_t>(prefix) % 4 == 0,
                  "slopes and prefix must be aligned");
  SPECTRA_REQUIRE(scale > 0.0f && scale < INFINITY, "scale must be positive");
  SPECTRA_REQUIRE(cap >= 0.0f && cap < INFINITY, "cap must be 0 (none) or positive");
  SPECTRA_REQUIRE(window >= 0, "window must be 0 (none) or positive");
  if (workspace == nullptr || workspace_bytes < spectra_paged_attend_workspace(kv->head_dim))
    return fail(SPECTRA_ERR_WORKSPACE, "workspace missing or smaller than spectra_paged_attend_workspace bytes");
  SPECTRA_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, "workspace must be 16-byte aligned");
  const PagedPools pools = paged_pools(kv);
  if (int st = paged_apart({{"out", out, tokens * heads * kv->head_dim * 2, 0, 1},
                            {"the workspace", workspace, (int64_t)spectra_paged_attend_workspace(kv->head_dim), 0, 1}},
                           {{"q", q, (int64_t)heads * kv->head_dim * 2, ldq * 2, tokens},
                            pools.k, pools.v, pools.ks, pools.vs, pools.kz, pools.vz,
                            paged_table(kv), paged_lens(kv), paged_starts(kv),
                            {"slopes", slopes, 4LL * heads, 0, 1},
                            {"prefix", prefix, 4LL * kv->batch, 0, 1}});
      st != SPECTRA_OK)
    return st;
  constexpr double log2e = 1.4426950408889634;
  a.sc.mul = (float)(cap > 0.0f ? 2.0 * log2e * scale / cap : log2e * scale);
  a.sc.cap2 = (float)(cap * log2e);
  SPECTRA_REQUIRE(a.sc.mul > 0.0f && a.sc.mul < 1e30f && a.sc.cap2 < 1e30f, "scale or cap out of range");
  a.sc.slopes = slopes;
  a.sc.prefix = prefix;
  a.sc.window = window < (1 << 30) ? window : 0;  // (no sequence is longer)
  a.mod = a.sc.cap2 > kPagedCap ? kModLargeCap : cap > 0.0f || slopes != nullptr ? kMod : kModNone;
  a.q = (const uint16_t*)q;
  a.ldq = ldq;
  a.out = (uint16_t*)out;
  a.heads = heads;
  a.g = heads / kv->kv_heads;
  a.kind = kv->kind;
  a.hd = kv->head_dim;
  a.counters = (uint32_t*)workspace;
  a.slots = (float*)((uint8_t*)workspace + SPECTRA_PAGED_COUNTER_BYTES);
  a.stream = (hipStream_t)stream;
  const PagedGrid grid = paged_grid(a.kv, tokens, a.g, a.kind, a.hd);
  SPECTRA_REQUIRE(grid.tiles < (1LL << 28), "tokens out of range");
  a.units = (int)grid.units;
  a.wide = grid.wide;
  return grid.rows >= 64 ? launch_paged_many(a, grid.rows) : launch_paged_few(a, grid.rows);
}
