// Attention over a paged KV cache for few rows a sequence: one token, or a few drafted ones, times
// the query heads of a KV head, in tiles of 16 or 32 rows.
//
//   out = sum_j p_j v_j / sum_j p_j,   p_j = 2^(score_j - m),   scores in log2 units (PagedScore),
// one pass over the keys with the running maximum m of the scores, the sums rescaled when it rises; every wave
// of every workgroup that holds some of a tile's keys ends with such sums of its own, and sums of maxima m and
// m' are brought together by the factors 2^(m - max(m, m')).
//
// Bound by reading the cache once: 64 users with 0 to 8191 keys read 1.11 GB in 200 us, 5.5 TB/s (a copy reaches
// 5.0 both ways), 131071 bf16 keys 537 MB in 109 us, 4.9 TB/s, 48 users on 4-bit pages 455 MB in 110 to 122 us, 3.7 to
// 4.1 TB/s (there the expansion's vector instructions are as much as the loads); 96 keys take 6.7 us, of which an
// empty launch is most.  So 16-bit rows do not go through LDS: a wave takes 32 keys at a
// time straight into the registers that the matrix instructions read, the next 32 in flight
// behind them.  Scores are computed transposed, S^T = K Q^T (16 x 16 x 32): a lane's 16 bytes of a key
// row are the A operand as they lie in memory, and the lane ends with the scores of the keys
// 4 (l / 16) + 0 .. 3 of each 16 for row l % 16 of the tile.  Those are the B operand of O^T = V^T P^T when the
// contraction takes the keys in that order, so the weights never move; V is loaded by the same
// order (a lane: HD / 16 dims of its 8 keys) and turned by byte permutes.  4-bit pages are
// expanded in the registers (codes of a key's row as they lie; Q is put in the codes' order once);
// their codes come through LDS, a wave's own part of it, which costs no registers for what is in flight
// and lets three workgroups be resident, not two (48 users: 121 us, 127 through registers).
//
// As many workgroups as are resident at once share the batch's key steps evenly (PagedWalk); a
// part's 4 waves take 32 keys in turn and meet in LDS at its end, and the parts of a tile that
// several workgroups hold meet in the workspace, where the last to arrive joins them.  (Pieces of a fixed
// length, more of them than fit at once: 131071 keys 125 us, not 113, 64 users 206, not 200.)
//
// Roundings: the weights to the activations' 16 bits, which the product with V takes (half a unit each, in
// sums that stay fp32), the 4-bit values to fp16 (which the products take; three bits more than the bf16 that
// kv4_dequantize and the contiguous 4-bit cache's attention round them to), the output.
#include "paged_attend.h"

namespace spectra {

constexpr int kFewThreads = 256;

// 32 keys of 16-bit K and V as they lie: tile t, register r.
template <int HD>
struct FewTile {
  pu4_t k[2][HD / 32];
  uint32_t v[2][4][HD / 32];
  bool bad[2];  // a page that is not there
};
// 32 keys of 4-bit K and V in LDS, a wave's own: codes, scales and zero points of both.
template <int HD>
struct FewCodes {
  static constexpr int kCodes = 16 * HD, kScales = 2 * HD, kZeros = HD;  // bytes of 32 keys
  static constexpr int kV = kCodes, kS = 2 * kCodes, kZ = kS + 2 * kScales, kBytes = kZ + 2 * kZeros;
  static constexpr int kCopies = HD == 128 ? 7 : 4;  // instructions that bring them
  static constexpr int kDepth = 2;                   // tiles in LDS
};
template <int HD, int KIND>
constexpr int few_lds() {
  const int red = 4 * 16 * (HD + 4) * 4, ring = KIND == kKv4 ? 4 * FewCodes<HD>::kDepth * FewCodes<HD>::kBytes : 0;
  return red > ring ? red : ring;
}

template <int HD, int KIND, int NT, int MOD>
__global__ void __launch_bounds__(kFewThreads, few_resident(KIND, HD, 16 * NT))
    paged_few_kernel(const PagedKv kv, const PagedScore sc, const uint16_t* __restrict__ q, int64_t ldq, int g, int tokens,
                     int heads, bool wide, uint32_t* __restrict__ counters, float* __restrict__ slots, uint16_t* __restrict__ out) {
  constexpr bool Q4 = KIND == kKv4, BF = KIND == kKvBf16;
  constexpr int ROWS = 16 * NT, KS = HD / 32, DPL = HD / 16, RS = HD + 4;
  constexpr int ROWB = Q4 ? HD / 2 : 2 * HD;  // bytes of a row of a page
  __shared__ __align__(16) uint8_t pool[few_lds<HD, KIND>()];  // 4-bit keys on their way; at the end the waves' sums
  float* red = (float*)pool;
  __shared__ float wm[4][ROWS], wl[4][ROWS];
  __shared__ int flag;
  __shared__ uint32_t redo[2];
  const int tid = threadIdx.x, lane = tid & 63, wave = sread(tid >> 6), c = lane & 15, q4 = lane >> 4;
  PagedWalk<Wave> walk(kv, g, ROWS, tokens, kFewKeys, sc, blockIdx.x, gridDim.x, wide, lane);
  PagedPart un;
  if (tid == 0) redo[0] = 0;
  int turn = 1;
  for (int x = walk.line.begin; x < walk.line.end && walk.part(x, un); x = un.t0 + un.to) {
    turn ^= 1;
    const PagedSeq sq = un.seq;
    const int r0 = un.tile * ROWS, nrows = min(ROWS, sq.n * g - r0);
    const bool one = sq.n == 1;  // (its rows are token 0's)
    // the tile's tokens, position of token 0
    const int tok0 = one ? 0 : sread(r0 / g), tok1 = one ? 0 : sread((r0 + nrows - 1) / g), i0 = sq.len - sq.n;
    const int capacity = kv.table_width << kv.page_shift, pmask = (1 << kv.page_shift) - 1;
    // keys that some row of the tile sees, and those that every row does
    const PagedRange ra = paged_range(i0 + tok0, sq.len, un.prefix, sc.window);
    const PagedRange rb = paged_range(i0 + tok1, sq.len, un.prefix, sc.window);
    const int klo = ra.lo, khi = min(rb.hi, capacity), alo = rb.lo, ahi = ra.hi;
    const int kbeg = klo & ~31;
    const int steps = khi > kbeg ? (khi - kbeg + kFewKeys - 1) / kFewKeys : 0;
    const bool whole = un.from == 0 && un.to == un.steps;
    int sbeg = un.from, send = un.to;
    if (steps != un.steps) {  // (fewer than the line counted: a window, or the causal end)
      sbeg = sread((int)((uint64_t)(uint32_t)steps * (uint32_t)un.from / (uint32_t)un.steps));
      send = sread((int)((uint64_t)(uint32_t)steps * (uint32_t)un.to / (uint32_t)un.steps));
    }

    // the lane's rows (column c of each 16): their queries, B operands
    PagedRange rg[NT];
    float slope2[NT];
    int pos[NT];
    pu4_t qf[NT][KS];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = r0 + 16 * nt + c;
      const bool ok = 16 * nt + c < nrows;
      const int tok = one ? 0 : ok ? r / g : tok0, head = un.kvh * g + (ok ? r - tok * g : 0);
      rg[nt] = paged_range(i0 + tok, sq.len, un.prefix, sc.window);
      slope2[nt] = MOD != kModNone && sc.slopes ? sc.slopes[head] * 1.4426950408889634f : 0.0f;
      pos[nt] = i0 + tok;
      const uint16_t* qr = q + (int64_t)(sq.q0 + tok) * ldq + head * HD;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        pu4_t x = {0, 0, 0, 0};
        if (ok) x = *(const pu4_t*)(qr + (Q4 ? (HD / 4) * q4 + 8 * s : 32 * s + 8 * q4));
        if (Q4)  // pairs in the order of the expanded codes: dims n, n + 4
          x = (pu4_t){__builtin_amdgcn_perm(x[2], x[0], 0x05040100u), __builtin_amdgcn_perm(x[2], x[0], 0x07060302u),
                      __builtin_amdgcn_perm(x[3], x[1], 0x05040100u), __builtin_amdgcn_perm(x[3], x[1], 0x07060302u)};
        qf[nt][s] = x;
      }
    }

    // ---- loads: page ids a tile ahead of its rows, rows a tile ahead of their use
    const int* tab = kv.table + un.b * kv.table_stride;
    auto page_of = [&](int key) __attribute__((always_inline)) {
      return sread(sload(tab + min(key >> kv.page_shift, kv.table_width - 1)));
    };
    typedef FewTile<HD> Tile;
    const uint32_t koff = (uint32_t)(c * ROWB + 16 * q4), voff = (uint32_t)(4 * q4 * ROWB + c * (ROWB / 16));
    auto load = [&](Tile& t, int key0, int p0, int p1) __attribute__((always_inline)) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int id = h ? p1 : p0;
        t.bad[h] = (uint32_t)id >= (uint32_t)kv.num_pages;
        const int row = (un.kvh << kv.page_shift) + ((key0 + 16 * h) & pmask);
        const uint64_t at = paged_at(t.bad[h] ? 0 : id, kv.page_step) + row * ROWB;
        const uint8_t *kb = kv.k + at, *vb = kv.v + at;
#pragma unroll
        for (int s = 0; s < KS; ++s) t.k[h][s] = __builtin_bit_cast(pu4_t, load_from<uint4>(kb, koff, 64 * s));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (HD == 128) {
            const uint4 x = load_from<uint4>(vb, voff, i * ROWB);
            t.v[h][i][0] = x.x;
            t.v[h][i][1] = x.y;
            t.v[h][i][2] = x.z;
            t.v[h][i][3] = x.w;
          } else {
            const uint2 x = load_from<uint2>(vb, voff, i * ROWB);
            t.v[h][i][0] = x.x;
            t.v[h][i][1] = x.y;
          }
        }
      }
    };
    // 4 bits: to LDS at `to`, whose last reads are complete; bit h: the page of half h is not there
    typedef FewCodes<HD> C;
    auto fetch = [&](uint32_t to, int key0, int p0, int p1) __attribute__((always_inline)) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      const bool b0 = (uint32_t)p0 >= (uint32_t)kv.num_pages, b1 = (uint32_t)p1 >= (uint32_t)kv.num_pages;
      p0 = b0 ? 0 : p0;
      p1 = b1 ? 0 : p1;
      const int row0 = (un.kvh << kv.page_shift) + (key0 & pmask), row1 = (un.kvh << kv.page_shift) + ((key0 + 16) & pmask);
      const uint64_t a0 = paged_at(p0, kv.page_step) + row0 * ROWB, a1 = paged_at(p1, kv.page_step) + row1 * ROWB;
      const uint64_t s0 = paged_at(p0, kv.scale_step) + row0 * (HD / 16), s1 = paged_at(p1, kv.scale_step) + row1 * (HD / 16);
      const uint64_t z0 = paged_at(p0, kv.zero_step) + row0 * (HD / 32), z1 = paged_at(p1, kv.zero_step) + row1 * (HD / 32);
      if constexpr (HD == 128) {
        const uint32_t off = 16 * lane;
        copy_lds(kv.k + a0, off, to);
        copy_lds(kv.k + a1, off, to + 1024);
        copy_lds(kv.v + a0, off, to + C::kV);
        copy_lds(kv.v + a1, off, to + C::kV + 1024);
        const uint64_t s = (lane < 32 ? s0 : s1) + 4 * (lane & 31);
        copy_lds4(kv.ks + s, to + C::kS);
        copy_lds4(kv.vs + s, to + C::kS + C::kScales);
        copy_lds4((lane < 32 ? kv.kz : kv.vz) + ((lane & 16) == 0 ? z0 : z1) + 4 * (lane & 15), to + C::kZ);
      } else {
        const uint64_t a = (lane < 32 ? a0 : a1) + 16 * (lane & 31);
        copy_lds16(kv.k + a, to);
        copy_lds16(kv.v + a, to + C::kV);
        copy_lds4((lane < 32 ? kv.ks : kv.vs) + ((lane & 16) == 0 ? s0 : s1) + 4 * (lane & 15), to + C::kS);
        if (lane < 32) copy_lds4((lane < 16 ? kv.kz : kv.vz) + ((lane & 8) == 0 ? z0 : z1) + 4 * (lane & 7), to + C::kZ);
      }
      return (b0 ? 1 : 0) | (b1 ? 2 : 0);
    };

    float m[NT], l[NT];
    pf4_t o[NT][DPL];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt] = -INFINITY;
      l[nt] = 0.0f;
#pragma unroll
      for (int j = 0; j < DPL; ++j) o[nt][j] = (pf4_t){0.0f, 0.0f, 0.0f, 0.0f};
    }
    // t: the tile's registers, or its place in LDS
    auto compute = [&](const auto& t, int key0, bool bad0, bool bad1) __attribute__((always_inline)) {
      const bool edge = key0 < klo || key0 + 32 > khi;  // keys that no row sees: their values must not reach the product
      pf4_t s[NT][2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) s[nt][h] = (pf4_t){0.0f, 0.0f, 0.0f, 0.0f};
        if constexpr (Q4) {
          const int key = 16 * h + c, kg = HD == 128 ? q4 : q4 >> 1;  // group of the lane's dims
          const uint32_t zb = t[C::kZ + key * (HD / 32) + kg], sb = *(const uint16_t*)(t + C::kS + 2 * (key * (HD / 32) + kg));
          const Kv4Zero z = kv4_zero(zb | zb << 16);
          const ph2_t sf = __builtin_bit_cast(ph2_t, sb | sb << 16);
          uint32_t w[KS];
          if constexpr (HD == 128) {
            const pu4_t x = *(const pu4_t*)(t + key * ROWB + 16 * q4);
#pragma unroll
            for (int st = 0; st < KS; ++st) w[st] = x[st];
          } else {
            const uint2 x = *(const uint2*)(t + key * ROWB + 8 * q4);
            w[0] = x.x;
            w[1] = x.y;
          }
#pragma unroll
          for (int st = 0; st < KS; ++st) {
            const pu4_t a = kv4_pairs(w[st], z, sf);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) s[nt][h] = mfma16<BF>(a, qf[nt][st], s[nt][h]);
          }
        } else {
#pragma unroll
          for (int st = 0; st < KS; ++st)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) s[nt][h] = mfma16<BF>(t.k[h][st], qf[nt][st], s[nt][h]);
        }
      }
      const bool part = key0 < alo || key0 + 32 > ahi || bad0 || bad1;
      pu4_t pf[NT];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        // scores of the keys key0 + 16 (e / 4) + 4 q4 + e % 4
        float x[8], mn = m[nt], mul = sc.mul;
        if constexpr (MOD != kModNone)
          mul = paged_scores<MOD, 2, 4>(s[nt], sc, slope2[nt], (float)(pos[nt] - (key0 + 4 * q4)), [](int n) { return n; });
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = s[nt][e >> 2][e & 3] * mul;
        if (part) {
          const int from = rg[nt].lo - key0 - 4 * q4, to = min(rg[nt].hi, capacity) - key0 - 4 * q4;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int at = 16 * (e >> 2) + (e & 3);
            if ((e >> 2) ? bad1 : bad0) x[e] = NAN;
            if (at < from || at >= to) x[e] = -INFINITY;
          }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) mn = fmaxf(mn, x[e]);
        mn = fmaxf(mn, lane_xor<16>(mn, lane));
        mn = fmaxf(mn, lane_xor<32>(mn, lane));
        if (__ballot(mn > m[nt] + kPagedSlack) != 0) {
          const float corr = __builtin_amdgcn_exp2f(m[nt] - (mn == -INFINITY ? 0.0f : mn));
          l[nt] *= corr;
#pragma unroll
          for (int j = 0; j < DPL; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[nt][j][i] *= corr;
          m[nt] = mn;
        }
        const float mu = m[nt] == -INFINITY ? 0.0f : m[nt] - kPagedRaise<BF>;
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = __builtin_amdgcn_exp2f(x[e] - mu);
#pragma unroll
        for (int e = 0; e < 4; ++e) {  // (the total is of the weights as rounded, so that a mean of values lies among them)
          pf[nt][e] = pack2<BF>(x[2 * e], x[2 * e + 1]);
          l[nt] = add2<BF>(pf[nt][e], l[nt]);
        }
      }
      // O^T += V^T P^T, dims DPL (l % 16) + j at step j: the 8 keys' values of a dim, in pairs of keys
      uint32_t keep[4] = {~0u, ~0u, ~0u, ~0u};
      if (edge) {
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          const int key = key0 + 16 * (p >> 1) + 4 * q4 + 2 * (p & 1);
          keep[p] = (key >= klo && key < khi ? 0xffffu : 0u) | (key + 1 >= klo && key + 1 < khi ? 0xffff0000u : 0u);
        }
      }
      if constexpr (Q4) {
        constexpr int HALF = HD / 64;  // codes of 4 dims each
        const int vg = c * DPL / 32;   // group of the lane's dims
        Kv4Zero z2[4];
        ph2_t s2[4];
        uint32_t v0[4], v1[4];
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          const int key = 16 * (p >> 1) + 4 * q4 + 2 * (p & 1);  // and the next
          const uint8_t* zp = t + C::kZ + C::kZeros + key * (HD / 32) + vg;
          z2[p] = kv4_zero((uint32_t)zp[0] | (uint32_t)zp[HD / 32] << 16);
          const uint8_t* sp = t + C::kS + C::kScales + 2 * (key * (HD / 32) + vg);
          s2[p] = __builtin_bit_cast(ph2_t, ((uint32_t)*(const uint16_t*)sp | (uint32_t)*(const uint16_t*)(sp + HD / 16) << 16) & keep[p]);
          const uint8_t* vp = t + C::kV + key * ROWB + c * (ROWB / 16);
          if constexpr (HD == 128) {
            v0[p] = *(const uint32_t*)vp;
            v1[p] = *(const uint32_t*)(vp + ROWB);
          } else {
            v0[p] = *(const uint16_t*)vp;
            v1[p] = *(const uint16_t*)(vp + ROWB);
          }
        }
#pragma unroll
        for (int u = 0; u < HALF; ++u) {
          pu4_t a[4];
#pragma unroll
          for (int p = 0; p < 4; ++p) {
            const pu4_t x = kv4_pairs(__builtin_amdgcn_perm(v1[p], v0[p], u ? 0x07060302u : 0x05040100u), z2[p], s2[p]);
#pragma unroll
            for (int n = 0; n < 4; ++n) a[n][p] = x[n];
          }
#pragma unroll
          for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) o[nt][4 * u + n] = mfma16<BF>(a[n], pf[nt], o[nt][4 * u + n]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < DPL; ++j) {
          pu4_t a;
#pragma unroll
          for (int p = 0; p < 4; ++p) {
            a[p] = __builtin_amdgcn_perm(t.v[p >> 1][2 * (p & 1) + 1][j >> 1], t.v[p >> 1][2 * (p & 1)][j >> 1],
                                         (j & 1) ? 0x07060302u : 0x05040100u);
            if (edge) a[p] &= keep[p];
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) o[nt][j] = mfma16<BF>(a, pf[nt], o[nt][j]);
        }
      }
    };

    const int kend = min(khi, kbeg + send * kFewKeys);
    int key = kbeg + sbeg * kFewKeys + 32 * wave;
    if constexpr (Q4) {
      // page ids a tile ahead of the copies, copies kDepth - 1 tiles ahead of their use
      constexpr int D = C::kDepth;
      uint8_t* mine = pool + wave * D * C::kBytes;
      const uint32_t at0 = (uint32_t)(uintptr_t)(lds_t)mine;
      int p0 = page_of(key), p1 = page_of(key + 16), put = 0, ahead = key;
      uint32_t bad = 0;  // two bits a tile on its way, the next one's last
      int n = 0;         // tiles on their way
      auto send_one = [&]() __attribute__((always_inline)) {
        bad |= (uint32_t)fetch(at0 + put * C::kBytes, ahead, p0, p1) << (2 * n);
        ++n;
        put = put == D - 1 ? 0 : put + 1;
        ahead += kFewKeys;
        p0 = page_of(ahead);
        p1 = page_of(ahead + 16);
      };
#pragma unroll
      for (int i = 0; i < D - 1; ++i)
        if (ahead < kend) send_one();
      for (int get = 0; key < kend; key += kFewKeys) {
        if (ahead < kend) {
          send_one();
          asm volatile("s_waitcnt vmcnt(%0)" ::"n"((D - 1) * C::kCopies) : "memory");  // all but the later tiles'
        } else {
          asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
        compute(mine + get * C::kBytes, key, (bad & 1) != 0, (bad & 2) != 0);
        bad >>= 2;
        --n;
        get = get == D - 1 ? 0 : get + 1;
      }
      __syncthreads();  // (the waves' sums go where the codes were)
    } else if (key < kend) {
      Tile ta, tb;
      load(ta, key, page_of(key), page_of(key + 16));
      int b0 = page_of(key + kFewKeys), b1 = page_of(key + kFewKeys + 16);
      while (true) {
        if (key + kFewKeys < kend) load(tb, key + kFewKeys, b0, b1);
        int n0 = page_of(key + 2 * kFewKeys), n1 = page_of(key + 2 * kFewKeys + 16);
        compute(ta, key, ta.bad[0], ta.bad[1]);
        key += kFewKeys;
        if (key >= kend) break;
        if (key + kFewKeys < kend) load(ta, key + kFewKeys, n0, n1);
        n0 = page_of(key + 2 * kFewKeys);
        n1 = page_of(key + 2 * kFewKeys + 16);
        compute(tb, key, tb.bad[0], tb.bad[1]);
        b0 = n0;
        b1 = n1;
        key += kFewKeys;
        if (key >= kend) break;
      }
    }

    // ---- the waves meet: sums of a 16-row half at a time, in LDS
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      l[nt] += lane_xor<16>(l[nt], lane);
      l[nt] += lane_xor<32>(l[nt], lane);
      if (q4 == 0) {
        wm[wave][16 * nt + c] = m[nt];
        wl[wave][16 * nt + c] = l[nt];
      }
    }
    const bool mixed = tok1 > tok0;  // rows that see different keys
    // this share's parts of tiles that others hold the rest of: one may come first, one last
    float* part = slots + (int64_t)walk.line.record((int)blockIdx.x, x) * paged_slot<HD>(ROWS);
    auto write = [&](int row, int d, const float (&v)[4], float den) __attribute__((always_inline)) {
      const int r = r0 + row, tok = one ? 0 : r / g, head = un.kvh * g + (r - tok * g);
      const bool past = paged_range(i0 + tok, sq.len, un.prefix, sc.window).hi > capacity;
      const float inv = past ? NAN : 1.0f / den;
      float y[4];
      float odd = 0.0f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        y[e] = den == 0.0f && !past ? 0.0f : v[e] * inv;
        odd = paged_odd(odd, y[e]);
      }
      // (where the total is NaN the row's own scores are)
      if (mixed && odd != odd && den == den && !past) atomicOr(&redo[turn], 1u << row);
      const uint2 w = make_uint2(pack2<BF>(y[0], y[1]), pack2<BF>(y[2], y[3]));
      *(uint2*)(out + ((int64_t)(sq.q0 + tok) * heads + head) * HD + d) = w;
    };
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      if (16 * nt >= nrows) break;
      if (nt > 0) __syncthreads();
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < DPL; j += 4)
          *(float4*)(red + (wave * 16 + c) * RS + DPL * (4 * q4 + i) + j) =
              make_float4(o[nt][j][i], o[nt][j + 1][i], o[nt][j + 2][i], o[nt][j + 3][i]);
      __syncthreads();
      if (nt == 0 && tid == 0) redo[turn ^ 1] = 0;  // (every wave is past the last part's)
      for (int it = tid; it < 16 * HD / 4; it += kFewThreads) {
        const int r = it / (HD / 4), row = 16 * nt + r, d = 4 * (it % (HD / 4));
        if (row >= nrows) break;
        float mm = -INFINITY, den = 0.0f, v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < 4; ++w) mm = fmaxf(mm, wm[w][row]);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float f = paged_weight(wm[w][row], wl[w][row], mm);
          const float4 x = *(const float4*)(red + (w * 16 + r) * RS + d);
          den += f * wl[w][row];
          v[0] += f * x.x;
          v[1] += f * x.y;
          v[2] += f * x.z;
          v[3] += f * x.w;
        }
        if (whole) {
          write(row, d, v, den);
        } else {
          store_dev2(part + row * HD + d, v[0], v[1]);
          store_dev2(part + row * HD + d + 2, v[2], v[3]);
          if (d == 0) store_dev2(part + ROWS * HD + 2 * row, mm, den);
        }
      }
    }
    if (!whole) {
      const PagedCut cut(walk.line, un.t0, un.steps);
      const int pieces = cut.pieces;
      auto slot_of = [&](int p) __attribute__((always_inline)) { return cut.record(p); };
      if (paged_arrive(counters + cut.first, pieces, &flag)) {  // the last to arrive joins them
        for (int it = tid; it < nrows * (HD / 4); it += kFewThreads) {
          const int row = it / (HD / 4), d = 4 * (it % (HD / 4));
          float v[1][4];
          const float den = pieces <= 4 ? paged_join_by<HD, ROWS, 4, 1>(slots, slot_of, pieces, row, row * HD + d, 2, 0, v)
                                        : paged_join_by<HD, ROWS, 16, 1>(slots, slot_of, pieces, row, row * HD + d, 2, 0, v);
          write(row, d, v[0], den);
        }
      }
    }
    __syncthreads();  // (rows to be done over are known, and LDS is free for the next part)
    if (mixed && redo[turn] != 0) {
      const PagedSpoiled sp = paged_spoiled<HD, KIND>(kv, sc, un, g, r0, nrows);
      for (uint32_t r = redo[turn]; r != 0; r &= r - 1) {
        const int row = __builtin_ctz(r);
        if ((row & 3) != wave || !sp.reaches(paged_range(i0 + (r0 + row) / g, sq.len, un.prefix, sc.window))) continue;
        paged_row<HD, KIND, MOD>(kv, sc, un, g, q, ldq, heads, r0 + row, out);
      }
    }
  }
}

template <int HD, int KIND, int NT, int MOD>
static int launch_few(const PagedLaunch& a) {
  paged_few_kernel<HD, KIND, NT, MOD><<<dim3((unsigned)a.units), dim3(kFewThreads), 0, a.stream>>>(
      a.kv, a.sc, a.q, a.ldq, a.g, 16 * NT / a.g, a.heads, a.wide, a.counters, a.slots, a.out);
  SPECTRA_HIP_CHECK(hipGetLastError());
  return SPECTRA_OK;
}
template <int HD, int KIND>
static int launch_few_of(const PagedLaunch& a, int rows) {
  if (a.mod == kModLargeCap) return rows == 16 ? launch_few<HD, KIND, 1, kModLargeCap>(a) : launch_few<HD, KIND, 2, kModLargeCap>(a);
  if (rows == 16) return a.mod ? launch_few<HD, KIND, 1, kMod>(a) : launch_few<HD, KIND, 1, kModNone>(a);
  return a.mod ? launch_few<HD, KIND, 2, kMod>(a) : launch_few<HD, KIND, 2, kModNone>(a);
}
int launch_paged_few(const PagedLaunch& a, int rows) {
  if (a.hd == 64)
    return a.kind == kKv4      ? launch_few_of<64, kKv4>(a, rows)
           : a.kind == kKvBf16 ? launch_few_of<64, kKvBf16>(a, rows)
                               : launch_few_of<64, kKvF16>(a, rows);
  return a.kind == kKv4      ? launch_few_of<128, kKv4>(a, rows)
         : a.kind == kKvBf16 ? launch_few_of<128, kKvBf16>(a, rows)
                             : launch_few_of<128, kKvF16>(a, rows);
}

}  // namespace spectra
