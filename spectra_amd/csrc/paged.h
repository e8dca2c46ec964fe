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

// Whether two runs of bytes overlap (an operand that others still read while it is written).
inline bool paged_overlap(const void* a, int64_t na, const void* b, int64_t nb) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return x < y + (uintptr_t)nb && y < x + (uintptr_t)na;
}

// A sequence's part of the call: its first token, how many, and its keys after them.  Starts
// are clamped to the call's tokens, lengths to what the table can hold plus one (a position past
// it is a fault of the caller's that its rows report as NaN).
struct PagedSeq {
  int q0, n, len;
};
__device__ __forceinline__ PagedSeq paged_seq(int s0, int s1, int len, int tokens) {
  s0 = min(max(s0, 0), tokens);
  s1 = min(max(s1, s0), tokens);
  return {s0, s1 - s0, max(len, 0)};
}

__device__ __forceinline__ int sread(int v) { return __builtin_amdgcn_readfirstlane(v); }

// A scalar load: p the same in every lane, its memory written by no kernel of this library.
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

// ---- attention: scores, and the shares of the work ----------------------------------------------

// What turns products x = q . k into scores in log2 units, up to a constant of the row (softmax
// knows none): mul x, or with a cap
//   cap2 tanh(t x / 2) = cap2 (1 - 2 / (1 + 2^(t2 x)))  ->  2 cap2 (-1 / (1 + 2^(t2 x)))
// (t2 = 2 log2(e) scale / cap, cap2 = cap log2(e)); less slope2 |i - j|, which for keys up to the row's
// position is slope2 (j - i).
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
template <int T, int N, typename V, typename F>
__device__ __forceinline__ float paged_scores(V (&s)[T], const PagedScore& sc, float slope2, float far, F at) {
  float mul = sc.mul;
  if (sc.cap2 > 0.0f) {
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

// Key steps that a tile of about `tokens` tokens may have.
__device__ __forceinline__ int paged_steps(const PagedKv& kv, const PagedScore& sc, int len, int tokens, int ks) {
  int span = min(len, kv.table_width << kv.page_shift);
  if (sc.window > 0 && sc.prefix == nullptr) span = (int)min((int64_t)span, (int64_t)sc.window + tokens + 16);
  return (span + ks - 1) / ks;
}

// A batch's tiles and their key steps in one line, the steps of a tile beside each other, and one of
// equal shares of it: what a workgroup works through, whole tiles and at most two parts of one (a
// tile's steps by the table's lengths, an upper bound: a part is a fraction of what the rows of the
// tile see).  Worked out by every wave from the lengths themselves, so ragged batches are shared
// out evenly with no plan on the host.
struct PagedLine {
  int total, each, more;  // the line's length; shares hold `each` steps, the first `more` of them one more
  int begin, end;         // this share

  __device__ __forceinline__ int start(int w) const { return w * each + min(w, more); }
  __device__ __forceinline__ int owner(int x) const {  // the share that holds step x
    const int big = more * (each + 1);
    return (int)(x < big ? (uint32_t)x / (uint32_t)(each + 1) : more + (uint32_t)(x - big) / (uint32_t)each);
  }
};
struct PagedPart {
  PagedSeq seq;
  int b, kvh, tile, prefix;
  int t0, steps;  // the tile's place in the line, its steps
  int from, to;   // this part of them
};
class PagedWalk {
 public:
  PagedLine line;

  // wide: the line may pass 32 bits; tokens: about what a tile has
  __device__ __forceinline__ PagedWalk(const PagedKv& kv, int g, int rows, int tokens, int ks, const PagedScore& sc, int w, int groups,
                                       bool wide, int lane)
      : kv_(kv), sc_(sc), g_(g), rows_(rows), toks_(tokens), ks_(ks), lane_(lane), grain_(0), pad_(0), c0_(0), base_(0) {
    if (wide) {
      float sum = 0.0f;
      for (int c0 = 0; c0 < kv.batch; c0 += 64) {
        take(c0);
        sum += (float)tiles_ * (float)steps_;
      }
      sum = wave_sum(sum) * (float)kv.kv_heads;  // (the same in every lane and wave)
      while (sum > 536870912.0f) {               // steps of 2, 4, .. steps
        sum *= 0.5f;
        ++grain_;
      }
    }
    if (kv.batch <= 64) take(0);
    int total = count();
    line.each = (int)((uint32_t)max(total, 0) / (uint32_t)groups);
    line.more = max(total, 0) - line.each * groups;
    // where the tiles can be cut into as many equal pieces of their own, no share has parts of two
    pad_ = line.each + (line.more > 0);
    const int padded = pad_ > 1 ? count() : total;
    if (pad_ > 0 && padded >= 0 && padded <= groups * (int64_t)pad_) {
      total = padded;
      line.each = pad_;
      line.more = 0;
    } else {
      if (kv.batch <= 64 && pad_ > 1) {
        pad_ = 0;
        take(0);
      }
      pad_ = 0;
    }
    if (kv.batch > 64) take(0);
    scan_ = wave_scan(kv.kv_heads * tiles_ * steps_);
    line.total = max(total, 0);
    line.begin = sread(min(line.start(w), line.total));
    line.end = sread(min(line.start(w + 1), line.total));
  }

  // The part of the share that begins at x; x never goes back.  false: there is none.
  __device__ __forceinline__ bool part(int x, PagedPart& p) {
    uint64_t past;
    while ((past = __ballot(base_ + scan_ > x)) == 0) {
      base_ += __builtin_amdgcn_readlane(scan_, 63);
      c0_ += 64;
      if (c0_ >= kv_.batch) return false;
      take(c0_);
      scan_ = wave_scan(kv_.kv_heads * tiles_ * steps_);
    }
    const int at = __builtin_ctzll(past);
    auto of = [&](int v) __attribute__((always_inline)) { return __builtin_amdgcn_readlane(v, at); };
    const int steps = of(steps_), nt = of(tiles_), r = x - (base_ + of(scan_ - kv_.kv_heads * tiles_ * steps_));
    if (r < 0 || steps <= 0 || nt <= 0) return false;  // (starts that never were a batch: sums that wrapped)
    const int t = r / steps, from = r - t * steps;
    if ((int64_t)x - from + steps > line.total) return false;
    // (the same in every lane, told to the compiler: addresses made of them stay scalar)
    p.seq = {sread(of(seq_.q0)), sread(of(seq_.n)), sread(of(seq_.len))};
    p.b = sread(c0_ + at);
    p.kvh = sread(t / nt);
    p.tile = sread(t % nt);
    p.steps = sread(steps);
    p.from = sread(from);
    p.t0 = sread(x - from);
    p.to = sread(min(steps, from + line.end - x));
    p.prefix = sc_.prefix != nullptr ? max(sread(sload(sc_.prefix + p.b)), 0) : 0;
    return p.kvh < kv_.kv_heads;
  }

 private:
  // The line's length, with tiles of whole pad_ steps where there is one.
  __device__ __forceinline__ int count() {
    int total = 0;
    for (int c0 = 0; c0 < kv_.batch; c0 += 64) {
      if (kv_.batch > 64 || pad_ > 1) take(c0);
      total += __builtin_amdgcn_readlane(wave_scan(kv_.kv_heads * tiles_ * steps_), 63);
    }
    return total;
  }
  __device__ __forceinline__ void take(int c0) {
    const int b = min(c0 + lane_, kv_.batch - 1);
    seq_ = paged_seq(kv_.q_start[b], kv_.q_start[b + 1], kv_.lens[b], kv_.tokens);
    tiles_ = c0 + lane_ < kv_.batch ? (seq_.n * g_ + rows_ - 1) / rows_ : 0;
    steps_ = paged_steps(kv_, sc_, seq_.len, toks_, ks_);
    steps_ = max((steps_ + (1 << grain_) - 1) >> grain_, 1);
    if (pad_ > 1) steps_ = (int)((uint32_t)(steps_ + pad_ - 1) / (uint32_t)pad_) * pad_;
  }
  const PagedKv& kv_;
  const PagedScore& sc_;
  int g_, rows_, toks_, ks_, lane_, grain_, pad_, c0_, base_, scan_, tiles_, steps_;
  PagedSeq seq_;
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
__device__ __forceinline__ bool paged_unit(const PagedKv& kv, int g, int rows, int ks, int min_steps, int target,
                                           int max_slots,
                                           const PagedScore& sc, int u, int lane, PagedUnit& un) {
  PagedSeq sq;
  int tiles, steps;
  auto take = [&](int c0) __attribute__((always_inline)) {
    const int b = min(c0 + lane, kv.batch - 1);
    sq = paged_seq(kv.q_start[b], kv.q_start[b + 1], kv.lens[b], kv.tokens);
    tiles = c0 + lane < kv.batch ? (sq.n * g + rows - 1) / rows : 0;
    steps = max(paged_steps(kv, sc, sq.len, rows / g, ks), 1);
  };
  float work = 0.0f;
  for (int c0 = 0; c0 < kv.batch; c0 += 64) {
    take(c0);
    work += (float)tiles * (float)steps;
  }
  work = wave_sum(work) * (float)kv.kv_heads;  // (the same in every lane and wave)
  const int piece_steps = (int)fminf(fmaxf(ceilf(work / (float)target), (float)min_steps), 1e9f);
  int base = 0, slot0 = 0;
  for (int c0 = 0; c0 < kv.batch; c0 += 64) {
    if (kv.batch > 64) take(c0);
    const int up = steps < 3 * piece_steps ? piece_steps - 1 : 0;
    const int pieces = 2 * steps <= 3 * min_steps ? 1 : min((steps + up) / piece_steps, kPagedPieces);
    const int units = kv.kv_heads * tiles * pieces;
    const int end = base + wave_scan(units), slots = pieces > 1 ? units : 0, send = slot0 + wave_scan(slots);
    const uint64_t past = __ballot(end > u);
    if (past != 0) {
      const int at = __builtin_ctzll(past);
      auto of = [&](int v) __attribute__((always_inline)) { return __builtin_amdgcn_readlane(v, at); };
      un.b = c0 + at;
      un.seq = {of(sq.q0), of(sq.n), of(sq.len)};
      un.pieces = of(pieces);
      const int nt = of(tiles), first = of(send - slots);
      int r = u - of(end - units);
      un.kvh = r % kv.kv_heads;
      r /= kv.kv_heads;
      un.piece = r % un.pieces;
      un.tile = nt - 1 - r / un.pieces;  // (causal tiles: the longest first)
      if (u < of(end - units) || un.tile < 0) return false;  // (starts that never were a batch: sums that wrapped)
      const int slot = first + (un.kvh * nt + un.tile) * un.pieces;
      if (un.pieces > 1 && (slot < 0 || slot > max_slots - un.pieces)) {
        if (un.piece > 0) return false;
        un.pieces = 1;
      }
      un.slot = slot + un.piece;
      un.prefix = sc.prefix != nullptr ? max(sload(sc.prefix + un.b), 0) : 0;
      // (the same in every lane, told to the compiler: addresses made of them stay scalar)
      un = {{sread(un.seq.q0), sread(un.seq.n), sread(un.seq.len)}, sread(un.b), sread(un.kvh), sread(un.tile),
            sread(un.piece), sread(un.pieces), sread(un.slot), sread(un.prefix)};
      return true;
    }
    base = __builtin_amdgcn_readlane(end, 63);
    slot0 = __builtin_amdgcn_readlane(send, 63);
  }
  return false;
}

}  // namespace spectra
