// The paged KV cache: what its kernels share.
//
// A pool of pages, each [kv_heads][page][head_dim] (one KV head's rows of a page are one contiguous
// run), in fp16, bf16, or 4 bits (codes, fp16 scales and zero points of groups of 32 dims, the
// layout of the contiguous 4-bit cache with a page in the place of max_seq).  Sequence b's
// position p is row p % page of page table[b][p / page].  Its last n = q_start[b + 1] -
// q_start[b] positions of kv_lens[b] are the tokens q_start[b] .. of the call.
//
// Tables and lengths live on the device and are read by every kernel, so a captured step follows
// them without the host; the kernels take them as they come: ids outside the pool and positions
// outside the table are never turned into addresses.
#pragma once

#include <initializer_list>

#include "common.h"

namespace spectra {

constexpr int kPagedPieces = 128;  // most pieces of a tile's keys

struct PagedKv {
  uint8_t *k, *v;    // 16-bit rows, or 4-bit codes
  uint8_t *ks, *vs;  // 4-bit: scales (fp16)
  uint8_t *kz, *vz;  // 4-bit: zero points
  uint32_t page_step, scale_step, zero_step;  // from one page to the next, in 16 bytes
  const int *table, *lens, *q_start;
  int64_t table_stride;
  int num_pages, kv_heads, page_shift, batch, table_width, tokens;
};

// Bytes from the pool's start to a page.
__device__ __forceinline__ uint64_t paged_at(int page, uint32_t step) { return ((uint64_t)(uint32_t)page * step) << 4; }

// Validates the descriptor for a call of `tokens` tokens and `heads` query heads, and fills the
// device form (api side of every paged entry).
int paged_args(const spectra_paged_kv_t* kv, int64_t tokens, int32_t heads, PagedKv* out);

// An operand in memory: n runs of `bytes` bytes, `step` bytes from one to the next (pages of a pool, rows of a wider
// matrix: what lies between them is not the operand's).
struct PagedRegion {
  const char* name;
  const void* at;
  int64_t bytes, step, n;
};
// Whether some run of a and some run of b share a byte.
inline bool paged_meet(const PagedRegion& a, const PagedRegion& b) {
  typedef __int128 wide;
  if (a.at == nullptr || b.at == nullptr || a.bytes == 0 || b.bytes == 0) return false;
  const wide x = reinterpret_cast<uintptr_t>(a.at), y = reinterpret_cast<uintptr_t>(b.at);
  const int64_t as = a.n > 1 ? a.step : 0, bs = b.n > 1 ? b.step : 0;
  if (x + (wide)(a.n - 1) * as + a.bytes <= y || y + (wide)(b.n - 1) * bs + b.bytes <= x) return false;
  if (a.n > 1 && b.n > 1 && as != bs) {  // (pools that lie among each other with other strides)
    const PagedRegion &few = a.n < b.n ? a : b, &all = a.n < b.n ? b : a;
    for (int64_t i = 0; i < few.n; ++i)
      if (paged_meet({few.name, (const uint8_t*)few.at + i * few.step, few.bytes, 0, 1}, all)) return true;
    return false;
  }
  // Run j of b lies y - x + k step after run i of a, k = j - i if both have that step: the least k for which it does not
  // end before a's begins.
  const int64_t step = a.n > 1 ? as : bs;
  wide k = 1 - a.n;
  if (step > 0) {
    const wide past = x - y - b.bytes, floor = past / step - (past % step < 0);
    k = floor + 1 > k ? floor + 1 : k;
  }
  return k < b.n && y - x + k * step > -(wide)b.bytes && y - x + k * step < a.bytes;
}
// Refuses a call that writes memory which another of its operands has too: each region written against the others
// written and those read.
int paged_apart(std::initializer_list<PagedRegion> written, std::initializer_list<PagedRegion> read);
// The caches' regions, keys and values of pages, scales and zero points (of no bytes where there are none).
struct PagedPools {
  PagedRegion k, v, ks, vs, kz, vz;
};
PagedPools paged_pools(const spectra_paged_kv_t* kv);
// The bounds of a pool's keys: checks of the descriptor, and its regions.
int paged_bounds_args(const spectra_paged_bounds_t* b, int64_t num_pages, int32_t kv_heads, int32_t hd);
PagedRegion paged_bound_codes(const spectra_paged_bounds_t* b, int64_t num_pages, int32_t kv_heads, int32_t hd);
PagedRegion paged_bound_scales(const spectra_paged_bounds_t* b, int64_t num_pages, int32_t kv_heads);
// The block table, the lengths and the starts.
inline PagedRegion paged_table(const spectra_paged_kv_t* kv) {
  return {"block_table", kv->block_table, 4LL * kv->table_width, 4 * kv->table_stride, kv->batch};
}
inline PagedRegion paged_lens(const spectra_paged_kv_t* kv) { return {"kv_lens", kv->kv_lens, 4LL * kv->batch, 0, 1}; }
inline PagedRegion paged_starts(const spectra_paged_kv_t* kv) { return {"q_start", kv->q_start, 4LL * (kv->batch + 1), 0, 1}; }

// A sequence's part of the call: its first token, how many, and its keys after them.  Starts are clamped to the
// call's tokens, lengths at zero.  (Lengths past what the table holds stay: rows that would see such positions are NaN,
// and no position past it is read.)
struct PagedSeq {
  int q0, n, len;
};
__device__ __forceinline__ PagedSeq paged_seq(int s0, int s1, int len, int tokens) {
  s0 = min(max(s0, 0), tokens);
  s1 = min(max(s1, s0), tokens);
  return {s0, s1 - s0, max(len, 0)};
}

__device__ __forceinline__ int sread(int v) { return __builtin_amdgcn_readfirstlane(v); }

// A scalar load: p the same in every lane, its memory not written while the kernel runs.
__device__ __forceinline__ int sload(const int* p) {
  return *(const __attribute__((address_space(4))) int*)p;
}

// The sequence of token t, found by the whole wave: 64 starts a step, so up to 64 sequences cost
// one load.  batch when t lies behind the last sequence.
__device__ __forceinline__ int paged_find(const int* q_start, int batch, int t, int lane) {
  int lo = 0, span = batch;
  while (span > 0) {
    const int step = (span + 63) >> 6, at = lo + (lane + 1) * step;
    const int v = at <= lo + span ? q_start[at] : 0x7fffffff;
    lo += step * __builtin_popcountll(__ballot(at <= lo + span && v <= t));
    if (step == 1) break;
    span = min(step, batch - lo);
  }
  return sread(lo);
}

// The sequence of token t and its part of the call.  Up to 64 sequences' starts and lengths are a lane's each, asked for at
// once and early, where paged_find and three scalar loads are one behind the other.
struct PagedStarts {
  int s0, s1, len;  // of sequence `lane`, or the last
};
__device__ __forceinline__ PagedStarts paged_starts_of(const PagedKv& kv, int lane) {
  const int b = min(lane, kv.batch - 1);
  return {kv.q_start[b], kv.q_start[b + 1], kv.lens[b]};
}
__device__ __forceinline__ int paged_where(const PagedKv& kv, const PagedStarts& st, int t, int lane, PagedSeq& sq) {
  if (kv.batch <= 64) {
    const int seq = __builtin_popcountll(__ballot(lane < kv.batch && st.s1 <= t));
    const int at = min(seq, kv.batch - 1);
    sq = paged_seq(__builtin_amdgcn_readlane(st.s0, at), __builtin_amdgcn_readlane(st.s1, at), __builtin_amdgcn_readlane(st.len, at), kv.tokens);
    return seq;
  }
  const int seq = paged_find(kv.q_start, kv.batch, t, lane), at = min(seq, kv.batch - 1);
  sq = paged_seq(sload(kv.q_start + at), sload(kv.q_start + at + 1), sload(kv.lens + at), kv.tokens);
  return seq;
}

// ---- attention: scores, and the shares of the work ----------------------------------------------

// What turns products x = q . k into scores in log2 units, up to a constant of the row (softmax
// knows none): mul x, or with a cap
//   cap2 tanh(y) = cap2 (1 - 2 / (1 + 2^(t2 x)))  ->  2 cap2 (-1 / (1 + 2^(t2 x)))
// (y = scale x / cap, t2 = 2 log2(e) scale / cap, cap2 = cap log2(e)); less slope2 |i - j|, which for keys up to the
// row's position is slope2 (j - i).  That form's error is some 2^-22 of the cap whatever the score: up to kPagedCap a
// tenth of a weight's rounding to fp16 (a cap of 256: weights off by 4e-5; of 1e6, by 15 %).  Past it, where |y| < 1/4
// (the subtraction would cancel), tanh(y) is y times the Taylor polynomial of tanh(y) / y in y^2, whose next term is
// below 2^-26: an error of 2^-19 of the score at most.
// It has kernels of its own: as a branch beside the other form its registers made chunks with a cap of 50 2 % slower.
constexpr float kPagedCap = 256.0f * 1.44269504f;  // of cap2
enum { kModNone, kMod, kModLargeCap };             // what becomes of scores
struct PagedScore {
  float mul;           // scale log2(e); with a cap t2
  float cap2;          // 0: no cap
  const float* slopes; // [heads] or NULL
  const int* prefix;   // [batch] or NULL
  int window;          // 0: none
};

// Applies cap and bias to T tiles of N products; far: the row's position less the first key's, at(n):
// the n-th product's key after it (tiles 32 or 16 N / 4 keys apart).  The scores are the result's
// factor times what is left in s.
template <int MOD, int T, int N, typename V, typename F>
__device__ __forceinline__ float paged_scores(V (&s)[T], const PagedScore& sc, float slope2, float far, F at) {
  float mul = sc.mul;
  if constexpr (MOD == kModLargeCap) {
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const float y = s[t][n] * (0.34657359f * mul), z = y * y;  // (ln(2) / 2)
        const float p = __builtin_fmaf(__builtin_fmaf(__builtin_fmaf(__builtin_fmaf(62.0f / 2835.0f, z, -17.0f / 315.0f), z, 2.0f / 15.0f), z, -1.0f / 3.0f), z, 1.0f);
        const float r = __builtin_amdgcn_rcpf(-1.0f - __builtin_amdgcn_exp2f(s[t][n] * mul));
        s[t][n] = __builtin_fabsf(y) < 0.25f ? y * p : __builtin_fmaf(2.0f, r, 1.0f);
      }
    mul = sc.cap2;
  } else if (sc.cap2 > 0.0f) {
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
      for (int n = 0; n < N; ++n)
        s[t][n] = __builtin_amdgcn_rcpf(-1.0f - __builtin_amdgcn_exp2f(s[t][n] * mul));
    mul = 2.0f * sc.cap2;
  }
  if (sc.slopes != nullptr) {
    constexpr int STEP = N == 16 ? 32 : 16;
    if (sc.prefix == nullptr) {
      const float first = -slope2 * far;
#pragma unroll
      for (int t = 0; t < T; ++t)
#pragma unroll
        for (int n = 0; n < N; ++n)
          s[t][n] = __builtin_fmaf(s[t][n], mul, __builtin_fmaf(slope2, (float)(STEP * t + at(n)), first));
    } else {  // (keys after the row's position too)
#pragma unroll
      for (int t = 0; t < T; ++t)
#pragma unroll
        for (int n = 0; n < N; ++n)
          s[t][n] = __builtin_fmaf(s[t][n], mul, -slope2 * __builtin_fabsf(far - (float)(STEP * t + at(n))));
    }
    mul = 1.0f;
  }
  return mul;
}

// Keys [lo, hi) that the query at position i sees, of a sequence of len keys.
struct PagedRange {
  int lo, hi;
};
__device__ __forceinline__ PagedRange paged_range(int i, int len, int prefix, int window) {
  const int hi = min(max(i + 1, prefix), len);
  return {window > 0 ? max(i - window + 1, 0) : 0, hi};
}

// A unit of work: one piece of the keys of one tile of `rows` query rows (token-major, the g heads
// of a KV head beside each other) of one KV head of one sequence.
struct PagedUnit {
  PagedSeq seq;
  int b, kvh, tile, piece, pieces, slot, prefix;
};

// Inclusive sum over the lanes up to this one, on the VALU (row shifts, then row broadcasts).
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
  return v;
}

// What the plans need of a wave, an Int being one value a lane: on the GPU a register, in a test on the host an
// array of 64.
struct Wave {
  typedef int Int;
  static __device__ __forceinline__ int read(const int* p, int at) { return p[at]; }   // a lane's own element
  static __device__ __forceinline__ int load(const int* p) { return sread(sload(p)); }  // the same in every lane
  static __device__ __forceinline__ int uniform(int v) { return sread(v); }             // (known to be so)
  static __device__ __forceinline__ int least(int a, int b) { return min(a, b); }
  static __device__ __forceinline__ int most(int a, int b) { return max(a, b); }
  static __device__ __forceinline__ int select(bool c, int a, int b) { return c ? a : b; }
  static __device__ __forceinline__ int quotient(int a, int b) { return (int)((uint32_t)a / (uint32_t)b); }
  static __device__ __forceinline__ uint64_t above(int a, int b) { return __ballot(a > b); }
  static __device__ __forceinline__ int of(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }
  static __device__ __forceinline__ int scan(int v) { return wave_scan(v); }  // sums up to each lane
  static __device__ __forceinline__ float product(int a, int b) { return wave_sum((float)a * (float)b); }  // their sum
};

// 64 sequences' parts of the call, a lane each: their tiles of `rows` rows, and a tile's key steps.
template <typename W>
struct PagedTake {
  typename W::Int q0, n, len, tiles, steps;
};
template <typename W>
__host__ __device__ __forceinline__ PagedTake<W> paged_take(const PagedKv& kv, const PagedScore& sc, int g, int rows, int tokens,
                                                            int ks, int c0, typename W::Int lane) {
  typedef typename W::Int Int;
  const Int b = W::least(lane + c0, kv.batch - 1);
  PagedTake<W> t;
  t.q0 = W::least(W::most(W::read(kv.q_start, b), 0), kv.tokens);
  t.n = W::least(W::most(W::read(kv.q_start, b + 1), t.q0), kv.tokens) - t.q0;
  t.len = W::most(W::read(kv.lens, b), 0);
  t.tiles = W::select(lane + c0 < kv.batch, (t.n * g + (rows - 1)) / rows, 0);
  Int span = W::least(t.len, kv.table_width << kv.page_shift);
  if (sc.window > 0 && sc.prefix == nullptr) span = W::least(span, sc.window + tokens + 16);
  t.steps = (span + (ks - 1)) / ks;
  return t;
}

// A batch's tiles and their key steps in one line, the steps of a tile beside each other, and one of
// equal shares of it: what a workgroup works through, whole tiles and at most two parts of one (a
// tile's steps by the table's lengths, an upper bound: a part is a fraction of what the rows of the
// tile see).  Worked out by every wave from the lengths themselves, so ragged batches are shared
// out evenly with no plan on the host.
struct PagedLine {
  int total, each, more;  // the line's length; shares hold `each` steps, the first `more` of them one more
  int begin, end;         // this share

  __host__ __device__ __forceinline__ int start(int w) const { return w * each + (w < more ? w : more); }
  __host__ __device__ __forceinline__ int owner(int x) const {  // the share that holds step x
    const int big = more * (each + 1);
    return (int)(x < big ? (uint32_t)x / (uint32_t)(each + 1) : more + (uint32_t)(x - big) / (uint32_t)each);
  }
  // Records of partial sums: two a share, of the part that it begins with and of a later one.
  __host__ __device__ __forceinline__ int record(int w, int x) const { return 2 * w + (x != begin); }
};
// A tile whose steps several shares hold: the parts' records, in the order of their keys.
struct PagedCut {
  int first, share, pieces;
  __host__ __device__ __forceinline__ PagedCut(const PagedLine& ln, int t0, int steps) {
    share = ln.owner(t0);
    pieces = ln.owner(t0 + steps - 1) - share + 1;
    first = 2 * share + (ln.start(share) != t0);
  }
  __host__ __device__ __forceinline__ int record(int p) const { return p == 0 ? first : 2 * (share + p); }
};
struct PagedPart {
  PagedSeq seq;
  int b, kvh, tile, prefix;
  int t0, steps;  // the tile's place in the line, its steps
  int from, to;   // this part of them
};
template <typename W>
class PagedWalk {
 public:
  typedef typename W::Int Int;
  PagedLine line;

  // wide: the line may pass 32 bits; tokens: about what a tile has
  __host__ __device__ __forceinline__ PagedWalk(const PagedKv& kv, int g, int rows, int tokens, int ks, const PagedScore& sc, int w,
                                                int groups, bool wide, Int lane)
      : kv_(kv), sc_(sc), g_(g), rows_(rows), toks_(tokens), ks_(ks), lane_(lane), grain_(0), pad_(0), c0_(0), base_(0) {
    if (wide) {
      float sum = 0.0f;  // (the same in every lane and wave)
      for (int c0 = 0; c0 < kv.batch; c0 += 64) {
        take(c0);
        sum += W::product(t_.tiles, t_.steps);
      }
      sum *= (float)kv.kv_heads;
      while (sum > 536870912.0f) {  // steps of 2, 4, .. steps
        sum *= 0.5f;
        ++grain_;
      }
    }
    if (kv.batch <= 64) take(0);
    int tiles = 0, total = count(tiles);
    total = total > 0 ? total : 0;
    line.each = (int)((uint32_t)total / (uint32_t)groups);
    line.more = total - line.each * groups;
    // Where the tiles can be cut into as many equal pieces of their own, no share has parts of two.  Not with more
    // tiles than shares, each of a piece at least; so what is summed is at most 2 groups pad_, twice the line: more
    // tiles than that, each of pad_ steps, would pass 32 bits and could come round to a sum that seems to fit.
    pad_ = line.each + (line.more > 0);
    const bool tried = pad_ > 1 && tiles <= groups;
    const int padded = tried ? count(tiles) : total;
    if (pad_ == 1 || (tried && padded <= groups * (int64_t)pad_)) {
      total = padded;
      line.each = pad_;
      line.more = 0;
    } else {
      pad_ = 0;
      if (kv.batch <= 64 && tried) take(0);
    }
    if (kv.batch > 64) take(0);
    scan_ = W::scan(t_.tiles * t_.steps * kv.kv_heads);
    line.total = total;
    line.begin = W::uniform(least(line.start(w), total));
    line.end = W::uniform(least(line.start(w + 1), total));
  }

  // The part of the share that begins at x; x never goes back.  false: there is none.
  __host__ __device__ __forceinline__ bool part(int x, PagedPart& p) {
    uint64_t past;
    while ((past = W::above(scan_ + base_, x)) == 0) {
      base_ += W::of(scan_, 63);
      c0_ += 64;
      if (c0_ >= kv_.batch) return false;
      take(c0_);
      scan_ = W::scan(t_.tiles * t_.steps * kv_.kv_heads);
    }
    const int at = __builtin_ctzll(past);
    const int steps = W::of(t_.steps, at), nt = W::of(t_.tiles, at);
    const int r = x - (base_ + W::of(scan_ - t_.tiles * t_.steps * kv_.kv_heads, at));
    if (r < 0 || steps <= 0 || nt <= 0) return false;  // (starts that never were a batch: sums that wrapped)
    const int t = r / steps, from = r - t * steps;
    if ((int64_t)x - from + steps > line.total) return false;
    // (the same in every lane, told to the compiler: addresses made of them stay scalar)
    p.seq = {W::uniform(W::of(t_.q0, at)), W::uniform(W::of(t_.n, at)), W::uniform(W::of(t_.len, at))};
    p.b = W::uniform(c0_ + at);
    p.kvh = W::uniform(t / nt);
    p.tile = W::uniform(t % nt);
    p.steps = W::uniform(steps);
    p.from = W::uniform(from);
    p.t0 = W::uniform(x - from);
    p.to = W::uniform(least(steps, from + line.end - x));
    p.prefix = 0;
    if (sc_.prefix != nullptr) {
      p.prefix = W::load(sc_.prefix + p.b);
      p.prefix = p.prefix > 0 ? p.prefix : 0;
    }
    return p.kvh < kv_.kv_heads;
  }

 private:
  static __host__ __device__ __forceinline__ int least(int a, int b) { return a < b ? a : b; }
  // The line's length, with tiles of whole pad_ steps where there is one; and how many tiles.
  __host__ __device__ __forceinline__ int count(int& tiles) {
    int total = 0;
    tiles = 0;
    for (int c0 = 0; c0 < kv_.batch; c0 += 64) {
      if (kv_.batch > 64 || pad_ > 1) take(c0);
      total += W::of(W::scan(t_.tiles * t_.steps * kv_.kv_heads), 63);
      tiles += W::of(W::scan(t_.tiles * kv_.kv_heads), 63);
    }
    return total;
  }
  __host__ __device__ __forceinline__ void take(int c0) {
    t_ = paged_take<W>(kv_, sc_, g_, rows_, toks_, ks_, c0, lane_);
    t_.steps = W::most((t_.steps + ((1 << grain_) - 1)) >> grain_, 1);
    if (pad_ > 1) t_.steps = W::quotient(t_.steps + (pad_ - 1), pad_) * pad_;
  }
  const PagedKv& kv_;
  const PagedScore& sc_;
  int g_, rows_, toks_, ks_;
  Int lane_;
  int grain_, pad_, c0_, base_;
  Int scan_;
  PagedTake<W> t_;
};

// The u-th unit, worked out by every wave from the lengths themselves, so that ragged batches are
// shared out evenly with no plan on the host: the tiles' key steps (of `ks` keys) are counted, and
// tiles of more steps than target units would get each (and than min_steps) are cut into pieces.  A
// piece costs some 5 steps beside its own (its partial sums, and the join), so tiles of up to half as many again as
// min_steps stay whole (16 steps: 17.6 us, 23.6 on 4-bit pages in two pieces, 17.7 and 30.2 in one; 9 steps: 13.4 whole).
// Pieces are rounded up where that is 2 or 3 (2 of 64 steps 80 us, 1 of 128
// 113) and down past that, where a unit that finds every compute unit taken costs more (6 of 11
// steps 36 us, 5 of 13 31).  At most tiles + target units; pieces' partial results take slots, less than
// 2 target of them (a cut tile has fewer than twice its steps over the steps of a piece).
// Lengths that did not fit in max_slots would leave a tile in one piece.  false: u is past the last unit.
template <typename W>
__host__ __device__ __forceinline__ bool paged_unit(const PagedKv& kv, int g, int rows, int ks, int min_steps, int target,
                                                    int max_slots, const PagedScore& sc, int u, typename W::Int lane,
                                                    PagedUnit& un) {
  typedef typename W::Int Int;
  PagedTake<W> t;
  auto take = [&](int c0) __attribute__((always_inline)) {
    t = paged_take<W>(kv, sc, g, rows, rows / g, ks, c0, lane);
    t.steps = W::most(t.steps, 1);
  };
  float work = 0.0f;  // (the same in every lane and wave)
  for (int c0 = 0; c0 < kv.batch; c0 += 64) {
    take(c0);
    work += W::product(t.tiles, t.steps);
  }
  work *= (float)kv.kv_heads;
  // (2^25: more steps than any tile has, and three times as many fit in 32 bits)
  const int piece_steps = (int)__builtin_fminf(__builtin_fmaxf(__builtin_ceilf(work / (float)target), (float)min_steps), 33554432.0f);
  int base = 0, slot0 = 0;
  for (int c0 = 0; c0 < kv.batch; c0 += 64) {
    if (kv.batch > 64) take(c0);
    const Int up = W::select(t.steps < 3 * piece_steps, piece_steps - 1, 0);
    const Int pieces = W::select(t.steps * 2 <= 3 * min_steps, 1, W::least((t.steps + up) / piece_steps, kPagedPieces));
    const Int units = t.tiles * pieces * kv.kv_heads, slots = W::select(pieces > 1, units, 0);
    const Int end = W::scan(units) + base, send = W::scan(slots) + slot0;
    const uint64_t past = W::above(end, u);
    if (past != 0) {
      const int at = __builtin_ctzll(past);
      auto of = [&](Int v) __attribute__((always_inline)) { return W::uniform(W::of(v, at)); };
      const int nt = of(t.tiles), first = of(send - slots), begin = of(end - units);
      int r = u - begin;
      // (the same in every lane, told to the compiler: addresses made of them stay scalar)
      un.seq = {of(t.q0), of(t.n), of(t.len)};
      un.b = W::uniform(c0 + at);
      un.pieces = of(pieces);
      un.kvh = W::uniform(r % kv.kv_heads);
      r /= kv.kv_heads;
      un.piece = W::uniform(r % un.pieces);
      un.tile = W::uniform(nt - 1 - r / un.pieces);  // (causal tiles: the longest first)
      if (u < begin || un.tile < 0) return false;    // (starts that never were a batch: sums that wrapped)
      const int slot = first + (un.kvh * nt + un.tile) * un.pieces;
      if (un.pieces > 1 && (slot < 0 || slot > max_slots - un.pieces)) {
        if (un.piece > 0) return false;
        un.pieces = 1;
      }
      un.slot = W::uniform(slot + un.piece);
      un.prefix = 0;
      if (sc.prefix != nullptr) {
        un.prefix = W::load(sc.prefix + un.b);
        un.prefix = un.prefix > 0 ? un.prefix : 0;
      }
      return true;
    }
    base = W::of(end, 63);
    slot0 = W::of(send, 63);
  }
  return false;
}

}  // namespace spectra
