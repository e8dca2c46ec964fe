// Attention over listed pages of a paged KV cache: each token and KV head has pages of its own (as paged_select.hip chooses
// them), of which it sees the keys up to its position.
//
//   out = sum_j p_j v_j / sum_j p_j,   p_j = 2^(score_j - m),   scores in log2 units (PagedScore),
// one pass over the listed keys with the running maximum m, the sums rescaled where it rises (paged_few.hip, whose
// operand layouts these are: scores transposed, S^T = K Q^T, so that the weights are the next product's operand where
// they lie; V turned by byte permutes; 4-bit pages through LDS).  All rows of a tile, up to 16 query heads of one token
// and KV head, see the same keys, so none has to be computed by itself.
//
// As many workgroups as are resident at once share the tiles' key steps (of 128 keys) evenly (PagedWalk, by the sequences'
// lengths and `count`): whole tiles and at most two parts each; the parts of a tile meet in the workspace, where the last
// to arrive joins them in the order of their keys.  (Shares by `count` alone: 64 users of 100 to 2000 keys with room for
// 4096 took 105 us, not 73.)
//
// Bound by reading the listed pages for a served batch: 64 users of 4096 keys, 1.05 GB, 180 to 188 us, 5.8 to 5.6 TB/s; 4-bit
// pages 81 us, 3.8 TB/s.  60 drafted tokens of 1536 keys of 64 dims on 4-bit pages with a cap take 22.0 us: the vector unit issues
// 57 % of the cycles (the expansion, anew for each token, and the cap), by two waves a SIMD that wait 38 % of theirs.  A
// single token is a chain of the launch, starts, list, ids, rows and the join: 2048 keys in 64 pages 9.4 us.  Roundings: the
// weights to the activations' 16 bits for the product with V, 4-bit values to fp16, the output.
#include "paged_attend.h"

namespace spectra {

constexpr int kBlkThreads = 256, kBlkKeys = 128;

// Workgroups a compute unit.  (Three fit the registers of the 64-dim kernels and, with spills, of the 4-bit ones: drafts on 4
// bits 33.0 us, not 28.3, 64 users of 64 dims 116, not 110.)
constexpr int kBlkResident = 2;
static_assert(2 * 256 * kBlkResident * 16 <= kFewSlotRows && 8 * 256 * kBlkResident <= SPECTRA_PAGED_COUNTER_BYTES, "two records and counters a workgroup");

// 32 keys of 16-bit K and V as they lie.
template <int HD>
struct BlkTile {
  pu4_t k[2][HD / 32];
  uint32_t v[2][4][HD / 32];
};
// 32 keys of 4-bit K and V in LDS, a wave's own: codes (K's, then V's), scales, zero points.  A half's 16 keys are brought
// by half of the lanes, so that a lane has one page: of 64 dims scales, and of both sizes zero points, lie as K's and V's of
// the first 16 keys, then of the others.
template <int HD>
struct BlkCodes {
  static constexpr int kV = 16 * HD, kS = 2 * kV, kZ = kS + 4 * HD;
  static constexpr int kBytes = kZ + (HD == 128 ? 256 : 192);
  static constexpr int kCopies = HD == 128 ? 7 : 4;  // instructions that bring them
  // of a key of a half, and group of 32 dims
  static __device__ __forceinline__ int scale(int v, int half, int key, int group) {
    return kS + (HD == 128 ? 256 * v + 128 * half : 128 * half + 64 * v) + 2 * (key * (HD / 32) + group);
  }
  static __device__ __forceinline__ int zero(int v, int half, int key, int group) {
    return kZ + 128 * half + (HD / 2) * v + key * (HD / 32) + group;
  }
};
// GP: columns that a tile takes of 16 (its rows, at most as many).
template <int HD, int KIND, int GP>
constexpr int blk_lds() {
  const int red = 4 * 16 * (HD + 4) * 4, ring = KIND == kKv4 ? 4 * 2 * (16 / GP) * BlkCodes<HD>::kBytes : 0;
  return red > ring ? red : ring;
}
// Sixteen keys of one page: the position of the first, and how many of them the row sees; where they lie (page 0 for a
// page that is not there, or for nothing).
struct BlkHalf {
  int page, seen;
  bool bad;
};

// The larger of the values of lanes LB apart.
template <int LB>
__device__ __forceinline__ float lane_most(float v) {
  const int iv = __builtin_bit_cast(int, v);
  const auto r = LB == 16 ? __builtin_amdgcn_permlane16_swap(iv, iv, false, false) : __builtin_amdgcn_permlane32_swap(iv, iv, false, false);
  return fmaxf(__builtin_bit_cast(float, (int)r[0]), __builtin_bit_cast(float, (int)r[1]));
}

template <int HD, int KIND, int MOD, int GP>
__global__ void __launch_bounds__(kBlkThreads, kBlkResident)
    paged_blocks_kernel(const PagedKv kv, float mul, float cap2, const uint16_t* __restrict__ q, int64_t ldq, int g, int heads,
                        const int* __restrict__ blocks, int count, bool wide, int apart,
                         uint32_t* __restrict__ counters, float* __restrict__ slots, uint16_t* __restrict__ out) {
  constexpr bool Q4 = KIND == kKv4, BF = KIND == kKvBf16;
  constexpr int ROWS = 16, KS = HD / 32, DPL = HD / 16, RS = HD + 4, PACK = 16 / GP;
  constexpr int ROWB = Q4 ? HD / 2 : 2 * HD;  // bytes of a row of a page
  __shared__ __align__(16) uint8_t pool[blk_lds<HD, KIND, GP>()];  // 4-bit keys on their way; at the end the waves' sums
  float* red = (float*)pool;
  __shared__ float wm[4][ROWS], wl[4][ROWS];
  __shared__ int flag;
  const int tid = threadIdx.x, lane = tid & 63, wave = sread(tid >> 6), c = lane & 15, q4 = lane >> 4;
  const int pmask = (1 << kv.page_shift) - 1, groups = (g + 15) / 16;
  // neighbouring workgroups go to different XCDs: an eighth of the line each, so that the tokens of a sequence and KV head,
  // whose lists have pages in common, meet in one L2
  const int share = (gridDim.x & 7) != 0 ? blockIdx.x : (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
  const PagedScore sc = {mul, cap2, nullptr, nullptr, 0};
  PagedKv line = kv;  // (for the walk: rows are tokens, heads their tiles)
  line.kv_heads = kv.kv_heads * groups;
  PagedScore most{};
  most.window = count << kv.page_shift;
  PagedWalk<Wave> walk(line, 1, 1, -16, kBlkKeys, most, share, gridDim.x, wide, lane);
  PagedPart un;
  for (int x = walk.line.begin; x < walk.line.end && walk.part(x, un); x = un.t0 + un.to) {
    const int tok = un.seq.q0 + un.tile, kvh = sread(un.kvh / groups), h0 = sread(kvh * g + 16 * (un.kvh - kvh * groups));
    const int nrows = min(16, (kvh + 1) * g - h0);
    const int pos = un.seq.len - un.seq.n + un.tile;  // the row's position: it sees the keys up to that
    const bool past = pos >= kv.table_width << kv.page_shift;
    const bool whole = un.from == 0 && un.to == un.steps;
    // the list up to its last entry, and this part of it (a round trip for each 64 entries, in every workgroup that has a
    // part: lists of 32 pages of 16 rows 8.0 us, of 128 9.9, of 1024 28.6, of 8192 158)
    const int* list = blocks + ((int64_t)tok * kv.kv_heads + kvh) * count;
    int extent = 0;
    for (int s0 = 0; s0 < count; s0 += 64) {
      const uint64_t some = __ballot(s0 + lane < count && list[min(s0 + lane, count - 1)] >= 0);
      if (some != 0) extent = s0 + 64 - __builtin_clzll(some);
    }
    const int keys = extent << kv.page_shift, steps = (keys + kBlkKeys - 1) / kBlkKeys;
    int sbeg = un.from, send = un.to;
    if (steps != un.steps) {  // (the line counted by the length)
      sbeg = sread((int)((uint64_t)(uint32_t)steps * (uint32_t)un.from / (uint32_t)un.steps));
      send = sread((int)((uint64_t)(uint32_t)steps * (uint32_t)un.to / (uint32_t)un.steps));
    }

    // the lane's row (column c): its queries, B operands
    pu4_t qf[KS];
    {
      const uint16_t* qr = q + (int64_t)tok * ldq + (int64_t)(h0 + min(c % GP, nrows - 1)) * HD;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        pu4_t y = *(const pu4_t*)(qr + (Q4 ? (HD / 4) * q4 + 8 * s : 32 * s + 8 * q4));
        if (Q4)  // pairs in the order of the expanded codes: dims n, n + 4
          y = (pu4_t){__builtin_amdgcn_perm(y[2], y[0], 0x05040100u), __builtin_amdgcn_perm(y[2], y[0], 0x07060302u),
                      __builtin_amdgcn_perm(y[3], y[1], 0x05040100u), __builtin_amdgcn_perm(y[3], y[1], 0x07060302u)};
        qf[s] = y;
      }
    }

    pu4_t qn[PACK][KS];  // 4 bits: the queries in tile n's columns
#pragma unroll
    for (int n = 0; n < PACK; ++n)
#pragma unroll
      for (int st = 0; st < KS; ++st)
#pragma unroll
        for (int e = 0; e < 4; ++e) qn[n][st][e] = c / GP == n ? qf[st][e] : 0u;

    // ---- loads: rows a tile ahead of their use, the pages' ids two, the list's entries three
    const int* tab = kv.table + un.b * kv.table_stride;
    const int last = extent - 1;
    auto listed = [&](int key) __attribute__((always_inline)) { return sload(list + max(min(key >> kv.page_shift, last), 0)); };
    auto page_of = [&](int b) __attribute__((always_inline)) {
      return sload(tab + ((uint32_t)b < (uint32_t)kv.table_width ? b : 0));
    };
    // the 16 keys from `key` of the list on, in block b of the sequence, whose page has this id
    auto half_of = [&](int key, int b, int id) __attribute__((always_inline)) {
      BlkHalf h;
      const bool there = (key >> kv.page_shift) <= last && (uint32_t)b < (uint32_t)kv.table_width;
      h.seen = there ? min(max(pos + 1 - ((b << kv.page_shift) + (key & pmask)), 0), 16) : 0;
      h.bad = (uint32_t)id >= (uint32_t)kv.num_pages;
      h.page = h.bad || !there ? 0 : id;
      return h;
    };
    typedef BlkTile<HD> Tile;
    const uint32_t koff = (uint32_t)(c * ROWB + 16 * q4), voff = (uint32_t)(4 * q4 * ROWB + c * (ROWB / 16));
    auto load = [&](Tile& t, int key0, const BlkHalf (&hf)[2]) __attribute__((always_inline)) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int row = (kvh << kv.page_shift) + ((key0 + 16 * h) & pmask);
        const uint64_t at = paged_at(hf[h].page, kv.page_step) + row * ROWB;
        const uint8_t *kb = kv.k + at, *vb = kv.v + at;
#pragma unroll
        for (int s = 0; s < KS; ++s) t.k[h][s] = __builtin_bit_cast(pu4_t, load_from<uint4>(kb, koff, 64 * s));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (HD == 128) {
            const uint4 y = load_from<uint4>(vb, voff, i * ROWB);
            t.v[h][i][0] = y.x;
            t.v[h][i][1] = y.y;
            t.v[h][i][2] = y.z;
            t.v[h][i][3] = y.w;
          } else {
            const uint2 y = load_from<uint2>(vb, voff, i * ROWB);
            t.v[h][i][0] = y.x;
            t.v[h][i][1] = y.y;
          }
        }
      }
    };
    // 4 bits: to LDS at `at`, whose last reads are complete.  Addresses are a lane's own: its half's page and 16 rows in
    // units of 16 bytes, one product, and the arrays' bases (a wave's, they took half of the loop's scalar registers).
    typedef BlkCodes<HD> C;
    const int hl = lane >> 5, group0 = kvh << (kv.page_shift - 4);
    const bool zv = (lane & (HD / 8)) != 0;
    const uint8_t* sbase = Q4 ? (HD == 128 || lane % 32 < 16 ? kv.ks : kv.vs) + 4 * (lane % (HD / 4)) : nullptr;
    const uint8_t* zbase = Q4 ? (zv ? kv.vz : kv.kz) + 4 * (lane % (HD / 8)) : nullptr;
    auto fetch = [&](uint32_t at, int key0, int p0, int p1) __attribute__((always_inline)) {
      const uint32_t page = hl ? p1 : p0, row = group0 + (((key0 >> 4) + hl) & (pmask >> 4));  // (16 rows each)
      auto place = [&](uint32_t step, uint32_t each, uint32_t more) __attribute__((always_inline)) {
        return ((uint64_t)page * step + (row * each + more)) << 4;
      };
      const uint64_t sc0 = place(kv.scale_step, HD / 16, 0), ze0 = place(kv.zero_step, HD / 32, 0);
      if constexpr (HD == 128) {
        const uint32_t off = 16 * lane;
        const int row0 = (kvh << kv.page_shift) + (key0 & pmask), row1 = (kvh << kv.page_shift) + ((key0 + 16) & pmask);
        const uint64_t a0 = paged_at(p0, kv.page_step) + row0 * ROWB, a1 = paged_at(p1, kv.page_step) + row1 * ROWB;
        copy_lds(kv.k + a0, off, at);
        copy_lds(kv.k + a1, off, at + 1024);
        copy_lds(kv.v + a0, off, at + C::kV);
        copy_lds(kv.v + a1, off, at + C::kV + 1024);
        copy_lds4(sbase + sc0, at + C::kS);
        copy_lds4(sbase + (kv.vs - kv.ks) + sc0, at + C::kS + 256);
        copy_lds4(zbase + ze0, at + C::kZ);
      } else {
        const uint64_t a = place(kv.page_step, HD / 2, lane & 31);
        copy_lds16(kv.k + a, at);
        copy_lds16(kv.v + a, at + C::kV);
        copy_lds4(sbase + sc0, at + C::kS);
        if ((lane & 16) == 0) copy_lds4(zbase + ze0, at + C::kZ);
      }
    };

    float m = -INFINITY, l = 0.0f;
    pf4_t o[DPL];
#pragma unroll
    for (int j = 0; j < DPL; ++j) o[j] = (pf4_t){0.0f, 0.0f, 0.0f, 0.0f};
    // the weights of scores (but for a positive factor `by`), the running maximum and total
    auto weights = [&](float (&y)[8], float by) __attribute__((always_inline)) {
      float mn = y[0];
#pragma unroll
      for (int e = 1; e < 8; ++e) mn = fmaxf(mn, y[e]);
      mn = lane_most<16>(mn);
      mn = fmaxf(m, lane_most<32>(mn) * by);
      if (__ballot(mn > m + kPagedSlack) != 0) {
        const float corr = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.0f : mn));
        l *= corr;
#pragma unroll
        for (int j = 0; j < DPL; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[j][i] *= corr;
        m = mn;
      }
      const float mu = m == -INFINITY ? 0.0f : m - kPagedRaise<BF>;
      pu4_t pf;
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(y[e], by, -mu));
#pragma unroll
      for (int e = 0; e < 4; ++e) {  // (the total is of the weights as rounded, so that a mean of values lies among them)
        pf[e] = pack2<BF>(y[2 * e], y[2 * e + 1]);
        l = add2<BF>(pf[e], l);
      }
      return pf;
    };
    // which of a pair's keys 16 (p / 2) + 4 q4 + 2 (p % 2) and the next the row sees, of two halves
    auto kept = [&](uint32_t (&keep)[4], int s0, int s1) __attribute__((always_inline)) {
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        const int key = 4 * q4 + 2 * (p & 1), n = p < 2 ? s0 : s1;
        keep[p] = (key < n ? 0xffffu : 0u) | (key + 1 < n ? 0xffff0000u : 0u);
      }
    };
    // 16 bits: a tile in registers
    auto compute = [&](const Tile& t, const BlkHalf (&hf)[2]) __attribute__((always_inline)) {
      pf4_t s[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        s[h] = (pf4_t){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int st = 0; st < KS; ++st) s[h] = mfma16<BF>(t.k[h][st], qf[st], s[h]);
      }
      const bool part = hf[0].seen < 16 || hf[1].seen < 16;  // keys that the row does not see: their values must not reach the product
      // scores of the keys 16 (e / 4) + 4 q4 + e % 4
      float y[8], by = sc.mul;
      if constexpr (MOD != kModNone) by = paged_scores<MOD, 2, 4>(s, sc, 0.0f, 0.0f, [](int n) { return n; });
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = s[e >> 2][e & 3];
      if (part || hf[0].bad || hf[1].bad) {
        int seen[2] = {hf[0].seen, hf[1].seen};
        asm volatile("" : "+v"(seen[0]), "+v"(seen[1]));  // (or the comparisons are made for every tile, ahead of the branch)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (hf[e >> 2].bad) y[e] = NAN;
          if (4 * q4 + (e & 3) >= seen[e >> 2]) y[e] = -INFINITY;
        }
      }
      const pu4_t pf = weights(y, by);
      // O^T += V^T P^T, dims DPL (l % 16) + j at step j: the 8 keys' values of a dim, in pairs of keys
      uint32_t keep[4] = {~0u, ~0u, ~0u, ~0u};
      if (part) kept(keep, hf[0].seen, hf[1].seen);
#pragma unroll
      for (int j = 0; j < DPL; ++j) {
        pu4_t a;
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          a[p] = __builtin_amdgcn_perm(t.v[p >> 1][2 * (p & 1) + 1][j >> 1], t.v[p >> 1][2 * (p & 1)][j >> 1],
                                       (j & 1) ? 0x07060302u : 0x05040100u);
          if (part) a[p] &= keep[p];
        }
        o[j] = mfma16<BF>(a, pf, o[j]);
      }
    };
    // 4 bits: up to PACK tiles, kBlkKeys keys apart, in LDS from `t` on, whose scores take columns of their own: tile n's
    // products are those of queries that are zero in the other's columns, and its weights are zero there.  So a row's 8
    // columns, not 16, are exponentiated for a tile.  (Zero times what is not finite is NaN in the other tile's columns: sums
    // that come out so are made again, a tile at a time.)  half(x): tile x / 2's half x % 2; odd: not all keys are seen, or
    // a page is not there.
    auto packed = [&](const uint8_t* t, int tiles, bool odd, auto half) __attribute__((always_inline)) {
      const int mine = c / GP;  // the tile of the lane's column
      pf4_t s[2] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
      for (int n = 0; n < PACK; ++n) {
        if (n >= tiles) break;
        const uint8_t* tn = t + n * C::kBytes;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int kg = HD == 128 ? q4 : q4 >> 1;  // group of the lane's dims
          const uint32_t zb = tn[C::zero(0, h, c, kg)];
          uint32_t sb = *(const uint16_t*)(tn + C::scale(0, h, c, kg));
          if (PACK > 1 && odd) sb = c < half(2 * n + h).seen ? sb : 0u;  // (NaN of no key would reach the other tile's columns)
          const Kv4Zero z = kv4_zero(zb | zb << 16);
          const ph2_t sf = __builtin_bit_cast(ph2_t, sb | sb << 16);
          uint32_t w[KS];
          if constexpr (HD == 128) {
            const pu4_t y = *(const pu4_t*)(tn + (16 * h + c) * ROWB + 16 * q4);
#pragma unroll
            for (int st = 0; st < KS; ++st) w[st] = y[st];
          } else {
            const uint2 y = *(const uint2*)(tn + (16 * h + c) * ROWB + 8 * q4);
            w[0] = y.x;
            w[1] = y.y;
          }
#pragma unroll
          for (int st = 0; st < KS; ++st) s[h] = mfma16<BF>(kv4_pairs(w[st], z, sf), qn[n][st], s[h]);
        }
      }
      float y[8], by = sc.mul;
      if constexpr (MOD != kModNone) by = paged_scores<MOD, 2, 4>(s, sc, 0.0f, 0.0f, [](int n) { return n; });
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = s[e >> 2][e & 3];
      if (odd) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          int seen = 0;
          bool bad = false;
#pragma unroll
          for (int n = 0; n < PACK; ++n) {
            seen = PACK == 1 || mine == n ? half(2 * n + h).seen : seen;
            bad = PACK == 1 || mine == n ? half(2 * n + h).bad : bad;
          }
          asm volatile("" : "+v"(seen));  // (or the comparisons are made for every tile, ahead of the branch)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (bad) y[4 * h + e] = NAN;
            if (4 * q4 + e >= seen) y[4 * h + e] = -INFINITY;
          }
        }
      }
      const pu4_t pf = weights(y, by);
      constexpr int HALF = HD / 64;  // codes of 4 dims each
      const int vg = c * DPL / 32;   // group of the lane's dims
#pragma unroll
      for (int n = 0; n < PACK; ++n) {
        if (n >= tiles) break;
        const uint8_t* tn = t + n * C::kBytes;
        uint32_t keep[4] = {~0u, ~0u, ~0u, ~0u};
        if (odd) kept(keep, half(2 * n).seen, half(2 * n + 1).seen);
        pu4_t pn = pf;
        if constexpr (PACK > 1) {
#pragma unroll
          for (int e = 0; e < 4; ++e) pn[e] = mine == n ? pf[e] : 0u;
        }
        Kv4Zero z2[4];
        ph2_t s2[4];
        uint32_t v0[4], v1[4];
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          const int key = 4 * q4 + 2 * (p & 1);  // of the half, and the next
          const uint8_t* zp = tn + C::zero(1, p >> 1, key, vg);
          z2[p] = kv4_zero((uint32_t)zp[0] | (uint32_t)zp[HD / 32] << 16);
          const uint8_t* sp = tn + C::scale(1, p >> 1, key, vg);
          s2[p] = __builtin_bit_cast(ph2_t, ((uint32_t)*(const uint16_t*)sp | (uint32_t)*(const uint16_t*)(sp + HD / 16) << 16) & keep[p]);
          const uint8_t* vp = tn + C::kV + (16 * (p >> 1) + key) * ROWB + c * (ROWB / 16);
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
            const pu4_t w = kv4_pairs(__builtin_amdgcn_perm(v1[p], v0[p], u ? 0x07060302u : 0x05040100u), z2[p], s2[p]);
#pragma unroll
            for (int i = 0; i < 4; ++i) a[i][p] = w[i];
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) o[4 * u + i] = mfma16<BF>(a[i], pn, o[4 * u + i]);
        }
      }
    };

    const int kend = min(send * kBlkKeys, keys);  // (of the list's keys)
    int key = sbeg * kBlkKeys + 32 * wave;
    if (key < kend) {
      // blocks and ids of the next tile's halves, blocks of the one after it
      int b0 = 0, b1 = 0, m0 = 0, m1 = 0, id0 = 0, id1 = 0;
      auto first = [&]() __attribute__((always_inline)) {
        b0 = listed(key);
        b1 = listed(key + 16);
        m0 = listed(key + kBlkKeys);
        m1 = listed(key + kBlkKeys + 16);
        id0 = page_of(b0);
        id1 = page_of(b1);
      };
      auto next = [&](BlkHalf (&hf)[2], int k) __attribute__((always_inline)) {
        hf[0] = half_of(k, b0, id0);
        hf[1] = half_of(k + 16, b1, id1);
      };
      auto ahead = [&](int k) __attribute__((always_inline)) {  // k: the tile after the next
        b0 = m0;
        b1 = m1;
        id0 = page_of(b0);
        id1 = page_of(b1);
        m0 = listed(k + kBlkKeys);
        m1 = listed(k + kBlkKeys + 16);
      };
      uint8_t* mine = pool + wave * 2 * PACK * C::kBytes;  // (4 bits)
      const uint32_t at0 = (uint32_t)(uintptr_t)(lds_t)mine;
      if constexpr (Q4 && HD == 64) {
        // PACK tiles at a time in LDS, and the next PACK on their way.  A lane looks up one of their halves (for the wave they
        // would take more scalar registers than there are; of 128 dims a lane's lookups lost more than the packing gained, 64
        // users 26 us, not 24), by loads that go before the tiles' copies, which are counted below.
        constexpr int STEP = PACK * kBlkKeys;
        const int tile = (lane % (2 * PACK)) >> 1, apart = tile * kBlkKeys + 16 * (lane & 1);
        auto entry = [&](int k) __attribute__((always_inline)) { return list[max(min((k + apart) >> kv.page_shift, last), 0)]; };
        auto id_of = [&](int b) __attribute__((always_inline)) { return tab[(uint32_t)b < (uint32_t)kv.table_width ? b : 0]; };
        auto lane_of = [&](int k, int b, int id) __attribute__((always_inline)) {
          BlkHalf h = half_of(k + apart, b, id);
          if (k + tile * kBlkKeys >= kend) h.seen = 0;
          return h;
        };
        auto bring = [&](int turn, int k, const BlkHalf& in) __attribute__((always_inline)) {
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
          for (int n = 0; n < PACK; ++n)
            if (k + n * kBlkKeys < kend)
              fetch(at0 + (turn * PACK + n) * C::kBytes, k + n * kBlkKeys, __builtin_amdgcn_readlane(in.page, 2 * n),
                    __builtin_amdgcn_readlane(in.page, 2 * n + 1));
        };
        int b = entry(key), m = entry(key + STEP), id = id_of(b);
        BlkHalf now = lane_of(key, b, id), then = now;
        b = m;
        id = id_of(b);
        m = entry(key + 2 * STEP);
        bring(0, key, now);
        for (int turn = 0;; turn ^= 1) {
          if (key + STEP < kend) {
            then = lane_of(key + STEP, b, id);
            b = m;
            id = id_of(b);
            m = entry(key + 3 * STEP);
            bring(turn ^ 1, key + STEP, then);
          }
          const int left = (kend - key + kBlkKeys - 1) / kBlkKeys;  // tiles; the copies of those after PACK may be on their way
          if (left >= 2 * PACK) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(PACK * C::kCopies) : "memory");
          else if (left > PACK) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(C::kCopies) : "memory");
          else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
          packed(mine + turn * PACK * C::kBytes, min(PACK, left), __ballot(now.seen < 16 || now.bad) != 0, [&](int x) __attribute__((always_inline)) {
            return BlkHalf{0, __builtin_amdgcn_readlane(now.seen, x), __builtin_amdgcn_readlane((int)now.bad, x) != 0};
          });
          key += STEP;
          if (key >= kend) break;
          now = then;
        }
        if constexpr (PACK > 1) {
          // Sums that are not finite, as a scale that is infinite leaves them: again, in the first tile's columns alone, so that
          // they are what they are without another tile beside (values of some dims infinite, a score of -inf without weight).
          float odd = l * 0.0f;
#pragma unroll
          for (int j = 0; j < DPL; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) odd = __builtin_fmaf(o[j][i], 0.0f, odd);
          if (__ballot(odd != 0.0f) != 0) {
            m = -INFINITY;
            l = 0.0f;
#pragma unroll
            for (int j = 0; j < DPL; ++j) o[j] = (pf4_t){0.0f, 0.0f, 0.0f, 0.0f};
            for (key = sbeg * kBlkKeys + 32 * wave; key < kend; key += kBlkKeys) {
              BlkHalf ha[2];
              b0 = listed(key);
              b1 = listed(key + 16);
              id0 = page_of(b0);
              id1 = page_of(b1);
              next(ha, key);
              asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
              fetch(at0, key, ha[0].page, ha[1].page);
              asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
              packed(mine, 1, true, [&](int x) __attribute__((always_inline)) { return x < 2 ? ha[x] : BlkHalf{0, 0, false}; });
            }
#pragma unroll
            for (int j = 0; j < DPL; ++j)
#pragma unroll
              for (int i = 0; i < 4; ++i) o[j][i] = c < GP ? o[j][i] : 0.0f;
          }
        }
      } else if constexpr (Q4) {
        BlkHalf ha[2], hb[2];
        first();
        next(ha, key);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        fetch(at0, key, ha[0].page, ha[1].page);
        ahead(key + kBlkKeys);
        for (int turn = 0;; turn ^= 1) {
          if (key + kBlkKeys < kend) {
            next(hb, key + kBlkKeys);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            fetch(at0 + (turn ^ 1) * C::kBytes, key + kBlkKeys, hb[0].page, hb[1].page);
            ahead(key + 2 * kBlkKeys);
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(C::kCopies) : "memory");  // all but the next tile's
          } else {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
          }
          packed(mine + turn * C::kBytes, 1, ha[0].seen < 16 || ha[1].seen < 16 || ha[0].bad || ha[1].bad,
                 [&](int x) __attribute__((always_inline)) { return ha[x]; });
          key += kBlkKeys;
          if (key >= kend) break;
          ha[0] = hb[0];
          ha[1] = hb[1];
        }
      } else {
        BlkHalf ha[2], hb[2];
        first();
        next(ha, key);
        // (the next tile is asked for behind the last one, too, whose rows it then has again: a branch around the loads would
        // have the rows before them waited for as if they were the newest, 1.05 GB in 188 us, not 180)
        Tile ta, tb;
        load(ta, key, ha);
        ahead(key + kBlkKeys);
        auto beside = [&](BlkHalf (&hf)[2], const BlkHalf (&now)[2], Tile& t) __attribute__((always_inline)) {
          const bool more = key + kBlkKeys < kend;
          next(hf, key + kBlkKeys);
          hf[0].page = more ? hf[0].page : now[0].page;
          hf[1].page = more ? hf[1].page : now[1].page;
          load(t, key + kBlkKeys, hf);
          ahead(key + 2 * kBlkKeys);
        };
        while (true) {
          beside(hb, ha, tb);
          compute(ta, ha);
          key += kBlkKeys;
          if (key >= kend) break;
          beside(ha, hb, ta);
          compute(tb, hb);
          key += kBlkKeys;
          if (key >= kend) break;
        }
      }
    }
    if constexpr (Q4) __syncthreads();  // (the waves' sums go where the codes were)

    // ---- the waves meet, in LDS
    l += lane_xor<16>(l, lane);
    l += lane_xor<32>(l, lane);
    if (q4 == 0) {
      wm[wave][c] = m;
      wl[wave][c] = l;
    }
    float* part = slots + (int64_t)walk.line.record(share, x) * paged_slot<HD>(ROWS);
    auto write = [&](int row, int d, const float (&v)[4], float den) __attribute__((always_inline)) {
      const float inv = past ? NAN : 1.0f / den;
      float y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = den == 0.0f && !past ? 0.0f : v[e] * inv;
      const uint2 w = make_uint2(pack2<BF>(y[0], y[1]), pack2<BF>(y[2], y[3]));
      *(uint2*)(out + ((int64_t)tok * heads + h0 + row) * HD + d) = w;
    };
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < DPL; j += 4)
        *(float4*)(red + (wave * 16 + c) * RS + DPL * (4 * q4 + i) + j) =
            make_float4(o[j][i], o[j + 1][i], o[j + 2][i], o[j + 3][i]);
    __syncthreads();
    for (int it = tid; it < nrows * (HD / 4); it += kBlkThreads) {
      const int row = it / (HD / 4), d = 4 * (it % (HD / 4));
      // (all reads ahead: one behind the other they took a microsecond)
      float mm = -INFINITY, den = 0.0f, v[4] = {0.0f, 0.0f, 0.0f, 0.0f}, ms[4 * PACK], ls[4 * PACK];
      float4 y[4 * PACK];
#pragma unroll
      for (int w = 0; w < 4 * PACK; ++w) {
        const int col = row + GP * (w % PACK);
        ms[w] = wm[w / PACK][col];
        ls[w] = wl[w / PACK][col];
        y[w] = *(const float4*)(red + (w / PACK * 16 + col) * RS + d);
      }
#pragma unroll
      for (int w = 0; w < 4 * PACK; ++w) mm = fmaxf(mm, ms[w]);
#pragma unroll
      for (int w = 0; w < 4 * PACK; ++w) {
        const float f = paged_weight(ms[w], ls[w], mm);
        den += f * ls[w];
        v[0] += f * y[w].x;
        v[1] += f * y[w].y;
        v[2] += f * y[w].z;
        v[3] += f * y[w].w;
      }
      if (whole) {
        write(row, d, v, den);
      } else {
        store_dev2(part + row * HD + d, v[0], v[1]);
        store_dev2(part + row * HD + d + 2, v[2], v[3]);
        if (d == 0) store_dev2(part + ROWS * HD + 2 * row, mm, den);
      }
    }
    if (!whole) {
      const PagedCut cut(walk.line, un.t0, un.steps);
      const int pieces = cut.pieces;
      auto slot_of = [&](int p) __attribute__((always_inline)) { return cut.record(p); };
      if (paged_arrive(counters + cut.first * apart, pieces, &flag)) {  // the last to arrive joins them
        for (int it = tid; it < nrows * (HD / 4); it += kBlkThreads) {
          const int row = it / (HD / 4), d = 4 * (it % (HD / 4));
          float v[1][4];
          const float den = pieces <= 4 ? paged_join_by<HD, ROWS, 4, 1>(slots, slot_of, pieces, row, row * HD + d, 2, 0, v)
                                        : paged_join_by<HD, ROWS, 16, 1>(slots, slot_of, pieces, row, row * HD + d, 2, 0, v);
          write(row, d, v[0], den);
        }
      }
    }
    __syncthreads();  // (LDS is free for the next part)
  }
}

template <int HD, int KIND, int GP>
static const void* blocks_of(int mod) {
  return mod == kModNone ? (const void*)paged_blocks_kernel<HD, KIND, kModNone, GP>
         : mod == kMod   ? (const void*)paged_blocks_kernel<HD, KIND, kMod, GP>
                         : (const void*)paged_blocks_kernel<HD, KIND, kModLargeCap, GP>;
}
// pack: two tiles at a time.
template <int HD>
static const void* blocks_of(int kind, int mod, bool pack) {
  if (kind == kKvBf16) return blocks_of<HD, kKvBf16, 16>(mod);
  if (kind == kKvF16) return blocks_of<HD, kKvF16, 16>(mod);
  if constexpr (HD == 64) {
    if (pack) return blocks_of<HD, kKv4, 8>(mod);
  }
  return blocks_of<HD, kKv4, 16>(mod);
}

}  // namespace spectra

using namespace spectra;

extern "C" int spectra_paged_attend_blocks(const spectra_paged_kv_t* kv, const void* q, int64_t ldq, int64_t tokens,
                                           int32_t heads, const int32_t* blocks, int32_t count, float scale, float cap,
                                           void* workspace, size_t workspace_bytes, void* out, spectra_stream_t stream) {
  PagedKv p;
  if (int st = paged_args(kv, tokens, heads, &p); st != SPECTRA_OK) return st;
  const int hd = kv->head_dim, g = heads / kv->kv_heads;
  SPECTRA_REQUIRE(q && out && blocks, "NULL pointer");
  SPECTRA_REQUIRE(ldq >= (int64_t)heads * hd && ldq % 8 == 0, "q token stride too small or not a multiple of 8");
  SPECTRA_REQUIRE((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) % 16 == 0 &&
                      reinterpret_cast<uintptr_t>(blocks) % 4 == 0,
                  "q and out must be 16-byte aligned, blocks aligned");
  SPECTRA_REQUIRE(count >= 1 && (int64_t)count * kv->page_size < (1LL << 30), "count out of range");
  SPECTRA_REQUIRE(scale > 0.0f && scale < INFINITY, "scale must be positive");
  SPECTRA_REQUIRE(cap >= 0.0f && cap < INFINITY, "cap must be 0 (none) or positive");
  if (workspace == nullptr || workspace_bytes < spectra_paged_attend_workspace(hd))
    return fail(SPECTRA_ERR_WORKSPACE, "workspace missing or smaller than spectra_paged_attend_workspace bytes");
  SPECTRA_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, "workspace must be 16-byte aligned");
  const int64_t tiles = tokens * kv->kv_heads * ((g + 15) / 16);
  SPECTRA_REQUIRE(tiles < (1LL << 28), "tokens out of range");
  const PagedPools pools = paged_pools(kv);
  if (int st = paged_apart({{"out", out, tokens * heads * hd * 2, 0, 1},
                            {"the workspace", workspace, (int64_t)spectra_paged_attend_workspace(hd), 0, 1}},
                           {{"q", q, (int64_t)heads * hd * 2, ldq * 2, tokens},
                            {"blocks", blocks, tokens * kv->kv_heads * count * 4, 0, 1},
                            pools.k, pools.v, pools.ks, pools.vs, pools.kz, pools.vz,
                            paged_table(kv), paged_lens(kv), paged_starts(kv)});
      st != SPECTRA_OK)
    return st;
  constexpr double log2e = 1.4426950408889634;
  PagedScore sc{};
  sc.mul = (float)(cap > 0.0f ? 2.0 * log2e * scale / cap : log2e * scale);
  sc.cap2 = (float)(cap * log2e);
  SPECTRA_REQUIRE(sc.mul > 0.0f && sc.mul < 1e30f && sc.cap2 < 1e30f, "scale or cap out of range");
  const int mod = sc.cap2 > kPagedCap ? kModLargeCap : cap > 0.0f ? kMod : kModNone;
  // at most as many steps as the lists have
  const int64_t total = tiles * (((int64_t)count * kv->page_size + kBlkKeys - 1) / kBlkKeys);
  const int64_t groups = std::min<int64_t>(total, 256 * kBlkResident);
  bool wide = total >= (1LL << 29);
  // (counters as far apart as there is room: atomics on one line wait for each other)
  int apart = 1;
  while (2 * apart * 2 * groups <= SPECTRA_PAGED_COUNTER_BYTES / 4 && apart < 64) apart *= 2;
  uint32_t* counters = (uint32_t*)workspace;
  float* slots = (float*)((uint8_t*)workspace + SPECTRA_PAGED_COUNTER_BYTES);
  int gv = g, hv = heads, cv = count;
  // 4 bits, 64 dims, 8 heads a KV head at most: two tiles at a time where a workgroup has as many (60 tokens of 1536 keys 21.9
  // us, not 25.0, of 256 keys 8.2 and 8.6; of 128 keys 7.1 and 6.3, one of 8192 14.6 and 14.1)
  const void* kern = hd == 64 ? blocks_of<64>(kv->kind, mod, g <= 8 && total >= 2 * groups) : blocks_of<128>(kv->kind, mod, false);
  void* args[] = {(void*)&p, (void*)&sc.mul, (void*)&sc.cap2, (void*)&q, (void*)&ldq, (void*)&gv, (void*)&hv, (void*)&blocks, (void*)&cv,
                  (void*)&wide, (void*)&apart, (void*)&counters, (void*)&slots, (void*)&out};
  SPECTRA_HIP_CHECK(hipLaunchKernel(kern, dim3((unsigned)groups), dim3(kBlkThreads), args, 0, (hipStream_t)stream));
  SPECTRA_HIP_CHECK(hipGetLastError());
  return SPECTRA_OK;
}
