// Selection of pages for sparse attention: for each token and KV head the pages whose bounds allow the largest products with
// the queries as rounded to 8 bits.
//
// The token's g query heads of the KV head become whole numbers of one scale, A = max |q|, c = rint(q 127 / A) (both
// operations fp32 as written), and page j scores
//   s_j = scale_j max_h sum_d (max(c_hd, 0) M_jd + min(c_hd, 0) m_jd)
// (M, m, scale: paged_bounds.hip): whole numbers below 2^23 summed exactly, one rounding by the product with the scale.  It
// bounds the products of c, not of q: a dim below half a step of A counts nothing.
// So a score is the same whatever order it is summed in, and the choice among near scores, too: the largest scores,
// the lowest page on ties.  A scale of infinity, or a page that is not in the pool, is taken before all scores: the
// attention then shows what is wrong.  The first `sink` and the last `local` pages of the visible are always taken.
//
// Scores are matrix products (16 x 16 x 64 of bytes): rows are query heads, padded to 4, 8 or 16 a token by copies of the
// last one, so that a token's maximum lies in a lane's registers and at most two exchanges; columns are 16 pages, whose
// 2 d bytes a lane reads as they lie.  Scores are kept in LDS as 32-bit keys in the scores' order; the `count`-th largest
// bounds the choice, ties go by the order of the pages, and the chosen are written in that order (sel_pick).
// A workgroup has one token (drafts and prompts: as many as fill the rows, whose pages are read once) and one KV head.
// Few such units with long tables are split: workgroups score a run of pages each, and the last of a unit to arrive
// chooses from the keys of all in the workspace.
//
// Bound by latencies, not by the bounds' bytes: starts and lengths, ids, bounds, then the choice, one behind the other (64
// users of up to 250 pages, 18 MB: 10.6 us, of which the choice is 2.5; one of 8188 pages, 17 MB: 12.4 us, of which the
// choice is 4; vector unit busy 15 % of the cycles).  A unit that is not split is one workgroup's, however long: 16 users
// of 2000 pages 24 us, 67 MB; one of 8000 pages among 64 users 75 us.  Keys take a word of LDS a column of the table,
// whatever the lengths: 64 short users on a table of 260 or 8001 columns 9.9 us, of 32768 14.7.
#include <algorithm>

#include "paged_attend.h"

namespace spectra {

typedef int pi4_t __attribute__((ext_vector_type(4)));

constexpr int kSelMost = 32768;                        // pages of a table
constexpr int kSelBits = 8, kSelBins = 1 << kSelBits;  // parts of a range that keys are counted in
constexpr int kSelWave = 512;                          // keys that one wave chooses from in its registers
constexpr int kSelRegs = 16;                           // keys that a lane holds where a workgroup chooses from more
constexpr int kSelLds = 160 * 1024 - 1024;             // codes, keys and counts of a workgroup
constexpr int kSelSplit = 64;                          // units whose pages are split among workgroups: at most as many
constexpr int kSelApart = 256;                         // bytes from one unit's counter to the next one's (atomics on one line wait for each other)
constexpr size_t kSelCounters = kSelApart * kSelSplit;
constexpr uint32_t kSelForced = ~0u, kSelOdd = ~0u - 1;
constexpr float kSelLeast = 7.8886091e-31f;  // 2^-100

struct PagedSelect {
  const int8_t* codes;  // [pages][kv_heads][2][hd]
  const float* scales;  // [pages][kv_heads]
  int64_t code_step, scale_step;
  int count, sink, local;
  int pitch;  // keys a row in LDS
  // units whose pages are split among `chunks` workgroups (of `chunk` pages): their arrivals, and the keys that meet
  int chunks, chunk;
  uint32_t *counters, *keys;
};

// A score as an unsigned key of the same order.
__device__ __forceinline__ uint32_t sel_key(float s) {
  const uint32_t u = __builtin_bit_cast(uint32_t, s + 0.0f);
  return u ^ (u >> 31 ? ~0u : 0x80000000u);
}

template <int LB>
__device__ __forceinline__ uint32_t lane_xor_u(uint32_t v, int lane) {
  return __builtin_bit_cast(uint32_t, lane_xor<LB>(__builtin_bit_cast(float, v), lane));
}
template <typename F>
__device__ __forceinline__ uint32_t wave_meet(uint32_t v, F f) {
  const int lane = __lane_id();
  v = f(v, lane_xor_u<32>(v, lane));
  v = f(v, lane_xor_u<16>(v, lane));
  v = f(v, lane_xor_u<8>(v, lane));
  v = f(v, lane_xor_u<4>(v, lane));
  v = f(v, lane_xor_u<2>(v, lane));
  return f(v, lane_xor_u<1>(v, lane));
}
__device__ __forceinline__ uint32_t wave_most(uint32_t v) {
  return wave_meet(v, [](uint32_t a, uint32_t b) { return max(a, b); });
}
__device__ __forceinline__ uint32_t wave_least(uint32_t v) {
  return wave_meet(v, [](uint32_t a, uint32_t b) { return min(a, b); });
}
__device__ __forceinline__ int wave_total(int v) { return __builtin_amdgcn_readlane(wave_scan(v), 63); }

__device__ __forceinline__ void store_dev1(uint32_t* p, uint32_t v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ uint32_t load_dev1(const uint32_t* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// K keys a lane, 0 where there is none: the largest t that at least `count` of them reach, or, with `slack`, a t that
// between count and count + slack reach where bisection meets one on its way.
template <int K>
__device__ __forceinline__ uint32_t sel_kth(const uint32_t (&k)[K], int count, int slack) {
  auto reach = [&](uint32_t t) __attribute__((always_inline)) {
    int c = 0;
#pragma unroll
    for (int r = 0; r < K; ++r) c += __builtin_popcountll(__ballot(k[r] >= t));
    return c;
  };
  uint32_t hi = 0, lo = ~0u;  // of the scores
#pragma unroll
  for (int r = 0; r < K; ++r) {
    const bool score = k[r] != 0 && k[r] < kSelOdd;
    hi = max(hi, score ? k[r] : 0u);
    lo = min(lo, score ? k[r] : ~0u);
  }
  hi = sread((int)wave_most(hi));
  lo = sread((int)wave_least(lo));
  if (reach(kSelForced) >= count) return kSelForced;
  if (reach(kSelOdd) >= count) return kSelOdd;
  if (reach(hi) >= count) return hi;
  // `count` reach lo, but not hi; three places between them at a time, whose counts do not wait for each other
  while (hi - lo > 1) {
    const uint32_t q = max((hi - lo) >> 2, 1u), t1 = lo + q, t2 = min(lo + 2 * q, hi), t3 = min(lo + 3 * q, hi);
    const int c1 = reach(t1), c2 = reach(t2), c3 = reach(t3);
    int c = c3;
    if (c3 >= count) {
      lo = t3;
    } else if (c2 >= count) {
      lo = t2;
      hi = t3;
      c = c2;
    } else if (c1 >= count) {
      lo = t1;
      hi = t2;
      c = c1;
    } else {
      hi = t1;
    }
    if (c >= count && c <= count + slack) break;
  }
  return lo;
}
// The `count` largest of K keys a lane, the first on ties (keys 64 r + lane), by one wave: their places, or what `of`
// has there, in order.
template <int K>
__device__ __forceinline__ void sel_wave(const uint32_t* key, int n, int count, const uint32_t* of, int* out) {
  const int lane = __lane_id();
  uint32_t k[K];
#pragma unroll
  for (int r = 0; r < K; ++r) k[r] = 64 * r + lane < n ? key[64 * r + lane] : 0u;
  const uint32_t t = sel_kth<K>(k, count, 0);
  int above = 0, spare = count;  // of those equal to t
#pragma unroll
  for (int r = 0; r < K; ++r) spare -= __builtin_popcountll(__ballot(k[r] > t));
  int equal = 0;
  const uint64_t below = (1ull << lane) - 1;
#pragma unroll
  for (int r = 0; r < K; ++r) {
    const uint64_t ab = __ballot(k[r] > t), eb = __ballot(k[r] == t);
    const int e = equal + __builtin_popcountll(eb & below), j = 64 * r + lane;
    if ((ab >> lane & 1) || ((eb >> lane & 1) && e < spare))
      out[above + __builtin_popcountll(ab & below) + min(e, spare)] = of != nullptr ? (int)of[j] : j;
    above += __builtin_popcountll(ab);
    equal += __builtin_popcountll(eb);
  }
}
__device__ __forceinline__ void sel_wave(const uint32_t* key, int n, int count, const uint32_t* of, int* out) {
  if (n <= 128) sel_wave<2>(key, n, count, of, out);
  else if (n <= 256) sel_wave<4>(key, n, count, of, out);
  else sel_wave<kSelWave / 64>(key, n, count, of, out);
}

// What the waves that work on one row of keys tell each other: one wave by itself, or all of a workgroup, each with a
// part of the keys.
struct SelAlone {
  static constexpr int parts = 1, part = 0, room = kSelBins;
  uint32_t* bins;  // [2][kSelBins], or `room` keys and their places
  __device__ __forceinline__ uint32_t kth(uint32_t v, int count) {
    const uint32_t k[1] = {v};
    return sel_kth<1>(k, count, max(min(count, room / 2 - count), 8));
  }
  __device__ __forceinline__ void sync() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }
  template <int N>
  __device__ __forceinline__ void all(uint32_t (&v)[N], const uint32_t (&none)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = __lane_id() == 0 ? v[i] : none[i];
  }
};
struct SelTogether {
  static constexpr int room = kSelWave;
  int parts, part;
  uint32_t* bins;  // [2][kSelBins], or `room` keys and their places
  uint32_t* box;   // [2][3][16]
  int turn = 0;
  // Of a value a lane; where twice as many groups of 2 or 4 lanes are left as are wanted, of their maxima, which are fewer.
  __device__ __forceinline__ uint32_t kth(uint32_t v, int count) {
    const int lane = __lane_id();
    const int few = 2 * count <= 16 * parts ? 2 : 2 * count <= 32 * parts ? 1 : 0;
    if (few > 0) v = max(v, lane_xor_u<1>(v, lane));
    if (few > 1) v = max(v, lane_xor_u<2>(v, lane));
    if ((lane & ((1 << few) - 1)) == 0) bins[(64 * part + lane) >> few] = v;
    __syncthreads();
    if (part == 0) {
      const int n = 64 * parts >> few, slack = few > 0 ? 8 : max(min(count, room / 2 - count), 8);
      const uint32_t t = n <= 128 ? of<2>(n, count, slack) : n <= 256 ? of<4>(n, count, slack) : of<kSelWave / 64>(n, count, slack);
      if (lane == 0) box[96] = t;
    }
    __syncthreads();
    return (uint32_t)sread((int)box[96]);
  }
  template <int K>
  __device__ __forceinline__ uint32_t of(int n, int count, int slack) {
    const int lane = __lane_id();
    uint32_t k[K];
#pragma unroll
    for (int r = 0; r < K; ++r) k[r] = 64 * r + lane < n ? bins[64 * r + lane] : 0u;
    return sel_kth(k, count, slack);
  }
  __device__ __forceinline__ void sync() { __syncthreads(); }
  // every wave's values, in lanes 0 .. parts - 1
  template <int N>
  __device__ __forceinline__ void all(uint32_t (&v)[N], const uint32_t (&none)[N]) {
    uint32_t* b = box + 48 * turn;
    turn ^= 1;
    const int lane = __lane_id();
    if (lane == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) b[16 * i + part] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = lane < parts ? b[16 * i + (lane & 15)] : none[i];
  }
};

// What is left for one wave to choose from: keys, and the places that they have (or their own); none: all is chosen.
struct SelFew {
  const uint32_t *key, *of;
  int n;
};

// The `count` largest of n > count keys, the first on ties, written in their order, by parts of 64 lanes, or a few keys for
// the first part's wave to choose from.
//
// Few keys are one wave's, in its registers.  Of more, each lane's largest is found first: as many of these as are wanted
// lie at or past the `count`-th largest of them, and so do as many keys, so only keys from there on are candidates: little
// more than `count` (64 of 8190 keys by 512 lanes: some 70, by 128 groups of 4 lanes: some 90), which one wave chooses from.
// Where that leaves too many, or more are wanted than there are lanes, the range that holds the count-th
// largest is narrowed by counting the keys in kSelBins equal parts of it; some two rounds leave as many keys as are
// wanted, or keys that are all the same.
template <typename W>
__device__ __forceinline__ SelFew sel_pick(const uint32_t* key, int n, int count, int* out, W w) {
  const int lane = __lane_id();
  if (n <= kSelWave) return {key, nullptr, n};
  const int each = ((n + w.parts - 1) / w.parts + 63) & ~63;
  const int from = min(each * w.part, n), to = min(from + each, n);
  // f of all keys of this part, a lane's each, the loads of four in flight together
  auto over = [&](auto f) __attribute__((always_inline)) {
    constexpr int U = 4;
    for (int j0 = from; j0 < to; j0 += 64 * U) {
      uint32_t k[U];
#pragma unroll
      for (int e = 0; e < U; ++e) k[e] = key[min(j0 + 64 * e + lane, to - 1)];
#pragma unroll
      for (int e = 0; e < U; ++e) f(k[e], j0 + 64 * e + lane < to, j0 + 64 * e + lane);
    }
  };
  if (count <= 64 * w.parts) {
    uint32_t best = 0;
    over([&](uint32_t k, bool there, int) __attribute__((always_inline)) { best = max(best, there ? k : 0u); });
    const uint32_t from_on = w.kth(best, count);
    int c = 0;
    over([&](uint32_t k, bool there, int) __attribute__((always_inline)) { c += __builtin_popcountll(__ballot(there && k >= from_on)); });
    uint32_t met[1] = {(uint32_t)c};
    w.all(met, {0u});
    const int upto = wave_scan((int)met[0]), all = __builtin_amdgcn_readlane(upto, 63);
    if (all >= count && all <= w.room) {  // (lanes without keys may have been counted on)
      int at = __builtin_amdgcn_readlane(upto, w.part) - c;
      uint32_t *keys = w.bins, *places = w.bins + w.room;
      const uint64_t below = (1ull << lane) - 1;
      over([&](uint32_t k, bool there, int j) __attribute__((always_inline)) {
        const uint64_t take = __ballot(there && k >= from_on);
        if (take >> lane & 1) {
          const int p = at + __builtin_popcountll(take & below);
          keys[p] = k;
          places[p] = (uint32_t)j;
        }
        at += __builtin_popcountll(take);
      });
      w.sync();
      return {keys, places, all};
    }
    w.sync();  // (the counts start anew)
  }
  uint32_t hi = 0, lo = ~0u;
  int first = 0;  // keys before all scores
  over([&](uint32_t k, bool there, int) __attribute__((always_inline)) {
    const bool score = there && k < kSelOdd;
    first += there && k >= kSelOdd;
    hi = max(hi, score ? k : 0u);
    lo = min(lo, score ? k : ~0u);
  });
  for (int i = w.part * 64 + lane; i < 2 * kSelBins; i += w.parts * 64) w.bins[i] = 0;
  uint32_t met[3] = {wave_most(hi), wave_least(lo), (uint32_t)wave_total(first)};
  w.all(met, {0u, ~0u, 0u});
  hi = wave_most(met[0]);
  lo = wave_least(met[1]);
  int above = wave_total((int)met[2]);  // keys past hi
  if (above >= count) {
    above = 0;
    hi = kSelForced;
    lo = kSelOdd;
  }
  for (int turn = 0;; turn ^= 1) {
    const int shift = hi - lo < kSelBins ? 0 : 32 - __builtin_clz(hi - lo) - kSelBits;
    uint32_t* bins = w.bins + turn * kSelBins;
    if (hi != lo) {
      over([&](uint32_t k, bool there, int) __attribute__((always_inline)) {
        if (there && k >= lo && k <= hi) atomicAdd(&bins[(k - lo) >> shift], 1u);
      });
      w.sync();
      // the parts from the last on: lane l has parts 255 - 4 l - 0 .. 3
      const uint4 c = *(const uint4*)(bins + kSelBins - 4 - 4 * lane);
      const int mine = (int)(c.x + c.y + c.z + c.w), upto = above + wave_scan(mine);
      const uint64_t enough = __ballot(upto >= count);
      const int at = __builtin_ctzll(enough);
      int before = __builtin_amdgcn_readlane(upto - mine, at), part = kSelBins - 1 - 4 * at, of = 0;
      const uint32_t v[4] = {(uint32_t)__builtin_amdgcn_readlane((int)c.w, at), (uint32_t)__builtin_amdgcn_readlane((int)c.z, at),
                             (uint32_t)__builtin_amdgcn_readlane((int)c.y, at), (uint32_t)__builtin_amdgcn_readlane((int)c.x, at)};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (of == 0) {
          if (before + (int)v[e] >= count) {
            of = (int)v[e];
          } else {
            before += (int)v[e];
            --part;
          }
        }
      above = before;
      lo += (uint32_t)part << shift;
      hi = lo + min(hi - lo, (1u << shift) - 1);  // (a part of scores near the type's end may pass 32 bits)
      if (shift == 0 || above + of == count) break;
      // (the counts of the round before this one, which nobody reads any more)
      for (int i = w.part * 64 + lane; i < kSelBins; i += w.parts * 64) w.bins[(turn ^ 1) * kSelBins + i] = 0;
      w.sync();
    } else {
      break;
    }
  }
  // keys past hi, and the first of those from lo to hi
  const int spare = count - above;
  int a = 0, e = 0;
  over([&](uint32_t k, bool there, int) __attribute__((always_inline)) {
    a += __builtin_popcountll(__ballot(there && k > hi));
    e += __builtin_popcountll(__ballot(there && k >= lo && k <= hi));
  });
  uint32_t both[2] = {(uint32_t)a, (uint32_t)e};
  w.all(both, {0u, 0u});
  a = __builtin_amdgcn_readlane(wave_scan((int)both[0]), w.part) - a;
  e = __builtin_amdgcn_readlane(wave_scan((int)both[1]), w.part) - e;
  const uint64_t below = (1ull << lane) - 1;
  over([&](uint32_t k, bool there, int j) __attribute__((always_inline)) {
    const uint64_t ab = __ballot(there && k > hi), eb = __ballot(there && k >= lo && k <= hi);
    if ((ab | eb) == 0) return;
    const int ea = e + __builtin_popcountll(eb & below);
    if ((ab >> lane & 1) || ((eb >> lane & 1) && ea < spare)) out[a + __builtin_popcountll(ab & below) + min(ea, spare)] = j;
    a += __builtin_popcountll(ab);
    e += __builtin_popcountll(eb);
  });
  return {nullptr, nullptr, 0};
}

// The same of up to 64 R keys a wave, which stay in registers; key(j): the j-th.  None: more candidates than fit, or more
// wanted than there are lanes, and nothing done.  For keys that have met in the workspace: brought to LDS first and read there
// three times, one of 8188 pages took 15.2 us, not 12.4.  Keys that are in LDS already are read from there (sel_pick): 16
// users of 600 pages 12.6 us (by registers 12.8), of 2000 24.3 (24.6), 64 of 600 21.4 (21.7), of 1000 35.9 (36.2); only
// the longest gain by registers, 16 of 8000 103.7 (102.3).
template <int R, typename F>
__device__ __forceinline__ SelFew sel_pick_in_registers(F key, int n, int count, SelTogether w) {
  if (count > 64 * w.parts) return {nullptr, nullptr, 0};
  const int lane = __lane_id();
  const int each = ((n + w.parts - 1) / w.parts + 63) & ~63;
  const int from = min(each * w.part, n), to = min(from + each, n);
  uint32_t k[R], best = 0;
#pragma unroll
  for (int r = 0; r < R; ++r) k[r] = key(min(from + 64 * r + lane, n - 1));
#pragma unroll
  for (int r = 0; r < R; ++r) {
    k[r] = from + 64 * r + lane < to ? k[r] : 0u;
    best = max(best, k[r]);
  }
  const uint32_t from_on = max(w.kth(best, count), 1u);
  int c = 0;
#pragma unroll
  for (int r = 0; r < R; ++r) c += __builtin_popcountll(__ballot(k[r] >= from_on));
  uint32_t met[1] = {(uint32_t)c};
  w.all(met, {0u});
  const int upto = wave_scan((int)met[0]), all = __builtin_amdgcn_readlane(upto, 63);
  if (all < count || all > w.room) return {nullptr, nullptr, 0};
  int at = __builtin_amdgcn_readlane(upto, w.part) - c;
  uint32_t *keys = w.bins, *places = w.bins + w.room;
  const uint64_t below = (1ull << lane) - 1;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const uint64_t take = __ballot(k[r] >= from_on);
    if (take == 0) continue;
    if (take >> lane & 1) {
      const int p = at + __builtin_popcountll(take & below);
      keys[p] = k[r];
      places[p] = (uint32_t)(from + 64 * r + lane);
    }
    at += __builtin_popcountll(take);
  }
  w.sync();
  return {keys, places, all};
}

// GP: rows a token takes of a tile of 16 (its heads, rounded up to 4, 8, 16); more than 16 heads take several tiles.
template <int HD, bool BF, int GP>
__global__ void __launch_bounds__(512) paged_select_kernel(const PagedKv kv, const PagedSelect sel,
                                                            const uint16_t* __restrict__ q, int64_t ldq, int heads, int g,
                                                            int tokens_a_group, int* __restrict__ blocks) {
  constexpr int KS = 2 * HD / 64;  // matrix instructions of a tile
  constexpr int TOK = 16 / GP;     // tokens of a tile
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ uint32_t box[97];
  __shared__ int flag;
  const int tid = threadIdx.x, lane = tid & 63, wave = sread(tid >> 6), waves = sread((int)(blockDim.x >> 6));
  const int c16 = lane & 15, q4 = lane >> 4;
  const int tiles = (g + 15) / 16;  // of a token's heads (GP 16)
  uint8_t* qc = smem;               // [rows][2 hd] codes of the queries
  uint32_t* bins = (uint32_t*)(smem + 16 * tiles * 2 * HD);  // (a wave's each, or the workgroup's)
  const bool alone = tokens_a_group > 1;                     // (rows of keys are a wave's each)
  uint32_t* keys = bins + 2 * (alone ? waves * SelAlone::room : SelTogether::room);
  uint32_t* mine = sel.keys + (int64_t)blockIdx.x * tokens_a_group * sel.pitch;  // (split units only)
  const int kvh = blockIdx.x % kv.kv_heads, first = (blockIdx.x / kv.kv_heads) * tokens_a_group;
  const int past = min(first + tokens_a_group, kv.tokens);
  // A token's heads as a wave holds them: eight dims of a row a lane, the rows of a tile (what a token of more than 16 heads
  // has beside them is read again).
  constexpr int NCH = GP * HD / 8 > 64 ? GP * HD / 512 : 1;
  uint4 u[NCH];
  auto ask = [&](int token) __attribute__((always_inline)) {
    const uint16_t* qr = q + (int64_t)token * ldq + (int64_t)kvh * g * HD;
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      const int x = lane + 64 * k, r = x / (HD / 8), d = 8 * (x % (HD / 8));
      u[k] = *(const uint4*)(qr + min(r, g - 1) * HD + d);
    }
  };
  // (on their way while the sequence is found)
  const PagedStarts starts = paged_starts_of(kv, lane);
  if (!alone) ask(first);
  for (int t0 = first; t0 < past;) {
    PagedSeq sq;
    const int seq = paged_where(kv, starts, t0, lane, sq);
    if (seq >= kv.batch) return;  // behind the last sequence: left alone
    const int n = max(min(min(sq.q0 + sq.n, past) - t0, TOK), 1);  // tokens of this step (starts that are no batch's: one)
    const int i0 = sq.len - sq.n + (t0 - sq.q0);           // position of the first
    const int most = min(((i0 + n - 1) >> kv.page_shift) + 1, kv.table_width);  // pages that the last sees
    int* to = blocks + ((int64_t)t0 * kv.kv_heads + kvh) * sel.count;
    const int64_t row = (int64_t)kv.kv_heads * sel.count;  // from a token's to the next one's
    if (most <= sel.count && blockIdx.y > 0) return;
    SelFew few = {nullptr, nullptr, 0};
    auto visible = [&](int t) __attribute__((always_inline)) {
      return i0 + t < 0 ? 0 : min(((i0 + t) >> kv.page_shift) + 1, kv.table_width);
    };
    if (most > sel.count) {
      const int* tab = kv.table + seq * kv.table_stride;
      const int begin = blockIdx.y * sel.chunk, end = min(most, begin + sel.chunk), step = 16 * waves;
      // 16 pages a wave and step: ids two steps ahead, bounds one
      auto page_of = [&](int j0) __attribute__((always_inline)) { return tab[min(j0 + c16, end - 1)]; };
      struct Bounds {
        pi4_t b[KS];
        float scale;
        bool bad;
      };
      auto bounds_of = [&](Bounds& x, int page) __attribute__((always_inline)) {
        x.bad = (uint32_t)page >= (uint32_t)kv.num_pages;
        page = x.bad ? 0 : page;
        const int8_t* at = sel.codes + page * sel.code_step + (int64_t)kvh * 2 * HD + 16 * q4;
#pragma unroll
        for (int s = 0; s < KS; ++s) x.b[s] = *(const pi4_t*)(at + 64 * s);
        x.scale = sel.scales[page * sel.scale_step + kvh];
      };
      int j0 = begin + 16 * wave;
      Bounds ba, bb;
      int pa = 0, pb = 0;
      if (j0 < end) {
        pa = page_of(j0);
        pb = page_of(j0 + step);
        bounds_of(ba, pa);
        bounds_of(bb, pb);
        pa = page_of(j0 + 2 * step);
        pb = page_of(j0 + 3 * step);
      }
      // ---- the queries' codes: a wave a token
      auto encode = [&](int t) __attribute__((always_inline)) {
        const uint16_t* qr = q + (int64_t)(t0 + min(t, n - 1)) * ldq + (int64_t)kvh * g * HD;
        uint32_t big = 0;
        auto magnitude = [&](const uint4& x) __attribute__((always_inline)) {
          const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t m = w[e] & 0x7fff7fffu;
            big = max(big, max(m & 0xffffu, m >> 16));
          }
        };
#pragma unroll
        for (int k = 0; k < NCH; ++k) magnitude(u[k]);
        for (int x = 16 * HD + 8 * lane; x < g * HD; x += 512) magnitude(*(const uint4*)(qr + x));
        big = wave_most(big);
        const float a = BF ? bf2f((uint16_t)big) : h2f((uint16_t)big);
        const float inv = big >= (BF ? 0x7f80u : 0x7c00u) || a < kSelLeast ? 0.0f : 127.0f / a;
        auto codes = [&](const uint4& y, int x) __attribute__((always_inline)) {  // of chunk x of the rows
          const int r = x / (HD / 8), d = 8 * (x % (HD / 8));
          const uint32_t w[4] = {y.x, y.y, y.z, y.w};
          uint32_t up[2] = {0, 0}, dn[2] = {0, 0};
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const uint16_t h = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
            const int c = inv == 0.0f ? 0 : (int)rintf((BF ? bf2f(h) : h2f(h)) * inv);
            up[e >> 2] |= (uint32_t)(max(c, 0) & 255) << (8 * (e & 3));
            dn[e >> 2] |= (uint32_t)(min(c, 0) & 255) << (8 * (e & 3));
          }
          uint8_t* dst = qc + (t * GP + r) * 2 * HD + d;
          *(uint2*)dst = make_uint2(up[0], up[1]);
          *(uint2*)(dst + HD) = make_uint2(dn[0], dn[1]);
        };
#pragma unroll
        for (int k = 0; k < NCH; ++k)
          if (lane + 64 * k < GP * HD / 8) codes(u[k], lane + 64 * k);
        for (int x = 16 * HD / 8 + lane; x < 16 * tiles * (HD / 8); x += 64)
          codes(*(const uint4*)(qr + min(x / (HD / 8), g - 1) * HD + 8 * (x % (HD / 8))), x);
      };
      // (apart: loads that only one of both asks for would have the bounds waited for, too)
      if (!alone) {
        if (wave == 0) encode(0);
      } else {
        for (int t = wave; t < TOK; t += waves) {
          ask(t0 + min(t, n - 1));
          encode(t);
        }
      }
      __syncthreads();
      // ---- scores
      pi4_t qa[KS];
      auto rows = [&](int tile) __attribute__((always_inline)) {
#pragma unroll
        for (int s = 0; s < KS; ++s) qa[s] = *(const pi4_t*)(qc + (16 * tile + c16) * 2 * HD + 64 * s + 16 * q4);
      };
      rows(0);
      auto score = [&](const Bounds& x, int j0) __attribute__((always_inline)) {
        const int j = j0 + c16;
        int m = -0x7fffffff;
        for (int tile = 0; tile < tiles; ++tile) {
          if (tiles > 1) rows(tile);
          pi4_t acc = {0, 0, 0, 0};
#pragma unroll
          for (int s = 0; s < KS; ++s) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(qa[s], x.b[s], acc, 0, 0, 0);
#pragma unroll
          for (int r = 0; r < 4; ++r) m = max(m, acc[r]);
        }
        if (GP >= 8) m = max(m, (int)lane_xor_u<16>((uint32_t)m, lane));
        if (GP >= 16) m = max(m, (int)lane_xor_u<32>((uint32_t)m, lane));
        const int t = q4 * 4 / GP;  // the token of the lane's rows
        if (q4 % (GP / 4) == 0 && t < n && j < end) {
          const int cur = (i0 + t) >> kv.page_shift;
          uint32_t k = x.bad || x.scale == INFINITY ? kSelOdd : min(max(sel_key((float)m * x.scale), 1u), kSelOdd - 1);
          if (j < sel.sink || j > min(cur, kv.table_width - 1) - sel.local) k = kSelForced;
          if (sel.chunks > 1) store_dev1(mine + t * sel.pitch + j, k);
          else keys[t * sel.pitch + j] = k;
        }
      };
      // (behind the last pages the loads go on, at the last one: with a branch around them the bounds before them are waited
      // for as if they were the newest)
      while (j0 < end) {
        score(ba, j0);
        bounds_of(ba, pa);
        pa = page_of(j0 + 4 * step);
        if (j0 + step >= end) break;
        score(bb, j0 + step);
        bounds_of(bb, pb);
        pb = page_of(j0 + 5 * step);
        j0 += 2 * step;
      }
      if (sel.chunks > 1) {  // (a unit of one step) the last to arrive chooses
        if (!paged_arrive(sel.counters + blockIdx.x * (kSelApart / 4), sel.chunks, &flag)) return;
        if (!alone && most <= 64 * kSelRegs * waves)
          few = sel_pick_in_registers<kSelRegs>([&](int j) __attribute__((always_inline)) { return load_dev1(mine + j); }, most,
                                                sel.count, SelTogether{waves, wave, bins, box});
        constexpr int U = 8;  // loads in flight
        if (few.n == 0) {
          for (int t = 0; t < n; ++t)
            for (int j = tid; j < most; j += U * blockDim.x) {
              uint32_t k[U];
#pragma unroll
              for (int e = 0; e < U; ++e) k[e] = load_dev1(mine + t * sel.pitch + min(j + e * (int)blockDim.x, most - 1));
#pragma unroll
              for (int e = 0; e < U; ++e)
                if (j + e * (int)blockDim.x < most) keys[t * sel.pitch + j + e * blockDim.x] = k[e];
            }
        }
      }
      __syncthreads();
    }
    // ---- the choice
    if (!alone && most > sel.count) {
      if (few.n == 0) few = sel_pick(keys, most, sel.count, to, SelTogether{waves, wave, bins, box});
      if (few.n > 0 && wave == 0) sel_wave(few.key, few.n, sel.count, few.of, to);
    } else {
      for (int t = wave; t < n; t += waves) {
        const int v = visible(t);
        if (v > sel.count) {
          const SelFew left = sel_pick(keys + t * sel.pitch, v, sel.count, to + t * row, SelAlone{bins + wave * 2 * SelAlone::room});
          if (left.n > 0) sel_wave(left.key, left.n, sel.count, left.of, to + t * row);
        } else {
          for (int x = lane; x < sel.count; x += 64) to[t * row + x] = x < v ? x : -1;
        }
      }
    }
    t0 += n;
    if (t0 < past) __syncthreads();  // (codes and keys are read)
  }
}

template <int HD, bool BF>
static const void* select_of(int gp) {
  return gp == 4   ? (const void*)paged_select_kernel<HD, BF, 4>
         : gp == 8 ? (const void*)paged_select_kernel<HD, BF, 8>
                   : (const void*)paged_select_kernel<HD, BF, 16>;
}

}  // namespace spectra

using namespace spectra;

extern "C" size_t spectra_paged_select_workspace(void) { return kSelCounters + (size_t)kSelSplit * kSelLds; }

extern "C" int spectra_paged_select(const spectra_paged_kv_t* kv, const spectra_paged_bounds_t* bounds, const void* q,
                                    int64_t ldq, int32_t act_dtype, int64_t tokens, int32_t heads, int32_t count, int32_t sink,
                                    int32_t local, void* workspace, size_t workspace_bytes, int32_t* blocks,
                                    spectra_stream_t stream) {
  SPECTRA_REQUIRE(kv != nullptr, "paged KV descriptor is NULL");
  spectra_paged_kv_t d = *kv;  // (neither keys nor values are read, nor need they be given)
  d.kind = SPECTRA_KV_4BIT;
  d.k = d.v = d.k_scales = d.v_scales = d.k_zeros = d.v_zeros = (void*)16;
  d.page_stride = d.scale_stride = d.zero_stride = 1LL << 32;
  kv = &d;
  PagedKv p;
  if (int st = paged_args(kv, tokens, heads, &p); st != SPECTRA_OK) return st;
  const int hd = kv->head_dim, g = heads / kv->kv_heads;
  if (int st = paged_bounds_args(bounds, kv->num_pages, kv->kv_heads, hd); st != SPECTRA_OK) return st;
  SPECTRA_REQUIRE(act_dtype == SPECTRA_F16 || act_dtype == SPECTRA_BF16, "q must be fp16 or bf16");
  SPECTRA_REQUIRE(q && blocks, "NULL pointer");
  SPECTRA_REQUIRE(ldq >= (int64_t)heads * hd && ldq % 8 == 0, "q token stride too small or not a multiple of 8");
  SPECTRA_REQUIRE(reinterpret_cast<uintptr_t>(q) % 16 == 0 && reinterpret_cast<uintptr_t>(blocks) % 4 == 0,
                  "q must be 16-byte aligned, blocks aligned");
  SPECTRA_REQUIRE(sink >= 0 && local >= 1 && count >= 1 && (int64_t)sink + local <= count,
                  "count must hold the first `sink` and the last `local` (at least one) blocks");
  SPECTRA_REQUIRE(count <= kSelMost, "count out of range");
  SPECTRA_REQUIRE(tokens * kv->kv_heads < (1LL << 31), "tokens out of range");
  if (kv->table_width > kSelMost) return fail(SPECTRA_ERR_UNSUPPORTED, "block tables of more than 32768 pages");
  const int pitch = (kv->table_width + 63) & ~63, rows = 16 * ((g + 15) / 16);
  // (64 users of up to 250 pages: 12.6 us with 256 or 512 threads; a chunk of 300 on 30000 keys 21.5 with 256, 24.7 with 512,
  // 34.6 with 1024; one user of 250 pages 9.0 with 256, 8.4 with 512, 9.7 with 1024)
  const int threads = tokens * kv->kv_heads >= 512 ? 256 : 512;
  // codes, counts and keys of a workgroup of `group` tokens
  auto lds_of = [&](int group) { return rows * 2 * hd + 8 * (group > 1 ? threads / 64 * SelAlone::room : SelTogether::room) + 4 * group * pitch; };
  if (g > 256 || lds_of(1) > kSelLds)
    return fail(SPECTRA_ERR_UNSUPPORTED, "too many query heads a KV head, with a block table of this width");
  if (workspace != nullptr) {
    if (workspace_bytes < spectra_paged_select_workspace())
      return fail(SPECTRA_ERR_WORKSPACE, "workspace smaller than spectra_paged_select_workspace bytes");
    SPECTRA_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, "workspace must be 16-byte aligned");
  }
  if (int st = paged_apart({{"blocks", blocks, tokens * kv->kv_heads * count * 4, 0, 1},
                            {"the workspace", workspace, (int64_t)spectra_paged_select_workspace(), 0, 1}},
                           {{"q", q, (int64_t)heads * hd * 2, ldq * 2, tokens},
                            paged_bound_codes(bounds, kv->num_pages, kv->kv_heads, hd),
                            paged_bound_scales(bounds, kv->num_pages, kv->kv_heads),
                            paged_table(kv), paged_lens(kv), paged_starts(kv)});
      st != SPECTRA_OK)
    return st;
  const bool one = kv->num_pages == 1;
  PagedSelect sel = {bounds->codes, bounds->scales, one ? 0 : bounds->code_stride, one ? 0 : bounds->scale_stride,
                     count, sink, local, pitch, 1, kSelMost, nullptr, nullptr};
  int gp = g <= 4 ? 4 : g <= 8 ? 8 : 16, gv = g, hv = heads;
  // tokens a workgroup takes: as many as fill a tile's rows, but one where sequences have less than two tiles (5 drafted
  // tokens of 12 sequences: one 10.6 us, four 15.4; a chunk of 100 on 30000 keys: 21.9 and 13.3)
  const int64_t seqs = std::min<int64_t>(tokens, kv->batch);
  int group = tokens < 32 / gp * seqs ? 1 : 16 / gp;
  while (lds_of(group) > kSelLds) group /= 2;
  const int64_t groups = (tokens + group - 1) / group * kv->kv_heads;
  const int lds = lds_of(group);
  // units of one step each, few of them, and pages enough for several workgroups
  if (workspace != nullptr && groups <= kSelSplit && kv->table_width >= 1024 && (group == 1 || kv->batch == 1)) {
    sel.chunks = (int)std::min<int64_t>(256 / groups, (kv->table_width + 255) / 256);
    sel.chunk = ((kv->table_width + sel.chunks - 1) / sel.chunks + 15) & ~15;
    sel.counters = (uint32_t*)workspace;
    sel.keys = (uint32_t*)((uint8_t*)workspace + kSelCounters);
  }
  const void* kern = hd == 64 ? (act_dtype == SPECTRA_BF16 ? select_of<64, true>(gp) : select_of<64, false>(gp))
                              : (act_dtype == SPECTRA_BF16 ? select_of<128, true>(gp) : select_of<128, false>(gp));
  if (int st = ensure_lds_limit(kern); st != SPECTRA_OK) return st;
  void* args[] = {(void*)&p, (void*)&sel, (void*)&q, (void*)&ldq, (void*)&hv, (void*)&gv, (void*)&group, (void*)&blocks};
  SPECTRA_HIP_CHECK(hipLaunchKernel(kern, dim3((unsigned)groups, (unsigned)sel.chunks), dim3(threads), args, lds, (hipStream_t)stream));
  SPECTRA_HIP_CHECK(hipGetLastError());
  return SPECTRA_OK;
}
