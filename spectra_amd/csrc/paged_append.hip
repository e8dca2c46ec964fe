// Appending to a paged KV cache with the rotation on the way (the paged counterpart of
// rope_append, whose arithmetic it shares bit for bit): for token t of sequence b at position p,
//   q_rot[t]               = R(p) q[t]
//   K page row of p        = R(p) k[t]     V page row of p = v[t]
// R(p) the rotation of the pairs (i, i + d/2) by the table's angles (fp32, one rounding at the
// end); a 4-bit pool takes the rows through the 4-bit quantizer, scale and zero point beside the
// codes.
//
// With axes (AXES) the pairs of a head turn by positions of their own: pair i by row positions[axis[i]][t] of the tables
// (images and video: time, height and width), while the cache's row stays the sequence's position.  A wave gathers its
// token's angles once, a pair a lane, and its heads read them from LDS.
//
// A pass over the rows: 8 rotation pairs (two 16-byte loads and stores) or 8 values of v a lane.
// The waves of a token are its own, so its sequence, position and page are found once a wave, by
// scalar loads behind a search of the starts that the row's loads overlap.  Bound by that chain
// of dependent loads for a few tokens (one: 3.5 to 4.5 us, most of it the launch), by memory for prompts: 8.1
// thousand bf16 tokens (32 heads of 128 on 8) read and write 199 MB in 34 us, 5.8 TB/s.  With axes, a token of each of 48
// users 3.1 us in a graph, 126 MB of bf16 prompts 27.8 us, 4.5 TB/s (40.1 where every lane gathered its pairs' angles); on
// 4-bit pages 3.9 us, and the prompts' 112 MB 28.2 us, 4.0 TB/s (the plain append 25.6).
// Roundings: the rotated values to their 16 bits, once, from fp32 products and sums; 4-bit rows as the
// quantizer rounds.
#include <algorithm>

#include "kv4.h"
#include "paged.h"

namespace spectra {

constexpr int kPaThreads = 256;
constexpr int kPagedAxes = 4;  // most axes

template <bool BF>
__device__ __forceinline__ void unpack8t(const uint4& u, float (&f)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    f[2 * e] = BF ? bf2f((uint16_t)w[e]) : h2f((uint16_t)w[e]);
    f[2 * e + 1] = BF ? bf2f((uint16_t)(w[e] >> 16)) : h2f((uint16_t)(w[e] >> 16));
  }
}

// Positions of the rotation by axis, and the axis of every pair (AXES only).
struct PagedAxes {
  const int* pos;  // [axes][tokens], rows `stride` apart
  int64_t stride;
  const uint8_t* axis;  // [head_dim / 2]; a pair whose axis is past the last stays as it is
  int axes;
};

template <bool BF, bool Q4, bool AXES>
__global__ void __launch_bounds__(kPaThreads) paged_append_kernel(const uint16_t* __restrict__ qkv, int64_t ldqkv,
                                                                  const float* __restrict__ cos_t,
                                                                  const float* __restrict__ sin_t, int64_t rope_rows,
                                                                  int heads, int hd, int waves, const PagedKv kv,
                                                                  uint16_t* __restrict__ q_rot, const PagedAxes ax) {
  __shared__ __align__(16) float angles[AXES ? kPaThreads / 64 : 1][128];  // a wave's token's cosines and sines
  // neighbouring blocks go to different XCDs: an eighth of the tokens each, so that rows beside each
  // other meet in one L2 (4-bit rows are less than a line)
  const uint32_t run = gridDim.x < 64 ? blockIdx.x : (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
  const int lane = threadIdx.x & 63, wv = sread((int)(run * (kPaThreads / 64) + (threadIdx.x >> 6)));
  const int t = wv / waves;  // this wave's token
  if (t >= kv.tokens) return;
  const int it = (wv - t * waves) * 64 + lane;  // item of the token
  const int h2 = hd >> 1, g2 = hd >> 4, nrot = (heads + kv.kv_heads) * g2;
  const bool rot = it < nrot, val = !rot && it - nrot < kv.kv_heads * 2 * g2;
  const uint16_t* row = qkv + (int64_t)t * ldqkv;
  // rotation item: head hh (queries, then keys), dims i .. i + 7 and their partners; value item: dims i ..
  const int j = rot ? it : it - nrot, per = rot ? g2 : 2 * g2;
  const int hh = j / per, i = 8 * (j - hh * per);
  uint4 a = make_uint4(0, 0, 0, 0), b = a;
  if (rot || val) {
    const uint16_t* src = row + (int64_t)(rot ? hh : heads + kv.kv_heads + hh) * hd + i;
    a = *(const uint4*)src;
    if (rot) b = *(const uint4*)(src + h2);
  }
  int axis = 255;  // of the lane's pair
  if constexpr (AXES) {
    if (lane < h2) axis = ax.axis[lane];
  }
  const int seq = paged_find(kv.q_start, kv.batch, t, lane);
  if (seq >= kv.batch) return;  // behind the last sequence: left alone
  const PagedSeq sq = paged_seq(sload(kv.q_start + seq), sload(kv.q_start + seq + 1), sload(kv.lens + seq), kv.tokens);
  const int pos = sq.len - sq.n + (t - sq.q0);
  bool turn = cos_t == nullptr || (pos >= 0 && pos < rope_rows);
  uint64_t turned = 0;  // pairs that turn
  if constexpr (AXES) {
    turn = true;
    int64_t row = 0;  // of the table, the lane's pair's
#pragma unroll
    for (int e = 0; e < kPagedAxes; ++e) {
      const int at = e < ax.axes ? sload(ax.pos + e * ax.stride + t) : 0;
      turn = turn && at >= 0 && at < rope_rows;
      row = axis == e ? at : row;
    }
    turned = __ballot(axis < ax.axes);
    if (turn && lane < h2) {  // (a wave's own: read back behind the wave's own wait)
      angles[threadIdx.x >> 6][lane] = cos_t[row * h2 + lane];
      angles[threadIdx.x >> 6][64 + lane] = sin_t[row * h2 + lane];
    }
    __builtin_amdgcn_wave_barrier();
  }
  int page = -1;
  if (turn && pos >= 0 && (pos >> kv.page_shift) < kv.table_width)
    page = sload(kv.table + seq * kv.table_stride + (pos >> kv.page_shift));
  const bool keep = page >= 0 && page < kv.num_pages;  // there is a row to write
  const int r = pos & ((1 << kv.page_shift) - 1);
  if (rot) {
    uint4 lo = a, hi = b;
    if (cos_t != nullptr && turn) {
      float c[8], s[8], x[8], y[8];
      uint32_t still = 0;  // pairs that do not turn (not by an angle of 0: its product with an infinite partner is NaN)
      if constexpr (AXES) {
        const float* mine = angles[threadIdx.x >> 6];
        *(float4*)c = *(const float4*)(mine + i);
        *(float4*)(c + 4) = *(const float4*)(mine + i + 4);
        *(float4*)s = *(const float4*)(mine + 64 + i);
        *(float4*)(s + 4) = *(const float4*)(mine + 64 + i + 4);
        still = (uint32_t)(turned >> i) & 255u ^ 255u;
      } else {
        *(float4*)c = *(const float4*)(cos_t + (int64_t)pos * h2 + i);
        *(float4*)(c + 4) = *(const float4*)(cos_t + (int64_t)pos * h2 + i + 4);
        *(float4*)s = *(const float4*)(sin_t + (int64_t)pos * h2 + i);
        *(float4*)(s + 4) = *(const float4*)(sin_t + (int64_t)pos * h2 + i + 4);
      }
      unpack8t<BF>(a, x);
      unpack8t<BF>(b, y);
      uint32_t lw[4] = {0, 0, 0, 0}, hw[4] = {0, 0, 0, 0};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float u = x[e] * c[e] - y[e] * s[e], w = y[e] * c[e] + x[e] * s[e];
        if (AXES && (still >> e & 1)) {
          u = x[e];
          w = y[e];
        }
        lw[e >> 1] |= (uint32_t)(BF ? f2bf(u) : f2h(u)) << (16 * (e & 1));
        hw[e >> 1] |= (uint32_t)(BF ? f2bf(w) : f2h(w)) << (16 * (e & 1));
      }
      lo = make_uint4(lw[0], lw[1], lw[2], lw[3]);
      hi = make_uint4(hw[0], hw[1], hw[2], hw[3]);
    } else if (!turn) {  // no angle for this position: NaN queries
      const uint32_t nan2 = BF ? 0x7fc07fc0u : 0x7e007e00u;
      lo = hi = make_uint4(nan2, nan2, nan2, nan2);
    }
    if (hh < heads) {
      uint16_t* dst = q_rot + ((int64_t)t * heads + hh) * hd + i;
      *(uint4*)dst = lo;
      *(uint4*)(dst + h2) = hi;
    }
    if (Q4 && hh >= heads) {  // (the lanes of a group of 32 dims are four of one head)
      uint32_t pk[2];
      uint16_t sb[2];
      uint8_t zb[2];
      kv4_quant_chunk(lo, pk[0], sb[0], zb[0]);
      kv4_quant_chunk(hi, pk[1], sb[1], zb[1]);
      if (keep) {
        const int64_t hr = ((int64_t)(hh - heads) << kv.page_shift) + r;  // row of the page
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          const int d = i + p * h2;
          *(uint32_t*)(kv.k + paged_at(page, kv.page_step) + hr * (hd / 2) + d / 2) = pk[p];
          if ((d & 31) == 0) {
            *(uint16_t*)(kv.ks + paged_at(page, kv.scale_step) + 2 * (hr * (hd / 32) + d / 32)) = sb[p];
            kv.kz[paged_at(page, kv.zero_step) + hr * (hd / 32) + d / 32] = zb[p];
          }
        }
      }
    } else if (hh >= heads && keep) {
      const int64_t hr = ((int64_t)(hh - heads) << kv.page_shift) + r;
      uint16_t* dst = (uint16_t*)(kv.k + paged_at(page, kv.page_step)) + hr * hd + i;
      *(uint4*)dst = lo;
      *(uint4*)(dst + h2) = hi;
    }
  } else if (val) {
    const int64_t hr = ((int64_t)hh << kv.page_shift) + r;
    if (Q4) {
      uint32_t pk;
      uint16_t sb;
      uint8_t zb;
      kv4_quant_chunk(a, pk, sb, zb);
      if (keep) {
        *(uint32_t*)(kv.v + paged_at(page, kv.page_step) + hr * (hd / 2) + i / 2) = pk;
        if ((i & 31) == 0) {
          *(uint16_t*)(kv.vs + paged_at(page, kv.scale_step) + 2 * (hr * (hd / 32) + i / 32)) = sb;
          kv.vz[paged_at(page, kv.zero_step) + hr * (hd / 32) + i / 32] = zb;
        }
      }
    } else if (keep) {
      *(uint4*)((uint16_t*)(kv.v + paged_at(page, kv.page_step)) + hr * hd + i) = a;
    }
  }
}

int paged_args(const spectra_paged_kv_t* kv, int64_t tokens, int32_t heads, PagedKv* out) {
  SPECTRA_REQUIRE(kv != nullptr, "paged KV descriptor is NULL");
  SPECTRA_REQUIRE(kv->kind == SPECTRA_KV_F16 || kv->kind == SPECTRA_KV_BF16 || kv->kind == SPECTRA_KV_4BIT,
                  "unknown paged KV kind");
  const bool q4 = kv->kind == SPECTRA_KV_4BIT;
  const int d = kv->head_dim;
  SPECTRA_REQUIRE(kv->kv_heads > 0 && heads > 0 && heads % kv->kv_heads == 0, "heads must be a multiple of kv_heads");
  SPECTRA_REQUIRE(heads <= (1 << 20), "heads out of range");
  if (d != 64 && d != 128) return fail(SPECTRA_ERR_UNSUPPORTED, "paged KV head_dim must be 64 or 128");
  SPECTRA_REQUIRE(kv->page_size >= 16 && kv->page_size <= 65536 && is_pow2(kv->page_size),
                  "page_size must be a power of two, at least 16");
  SPECTRA_REQUIRE(kv->num_pages > 0 && kv->num_pages < (1LL << 31), "num_pages out of range");
  SPECTRA_REQUIRE(kv->batch > 0 && kv->batch <= (1 << 20) && kv->table_width > 0, "empty batch or block table");
  SPECTRA_REQUIRE(kv->table_stride >= kv->table_width || kv->batch == 1, "block table row stride too small");
  SPECTRA_REQUIRE((int64_t)kv->table_width * kv->page_size < (1LL << 30), "block table covers too many positions");
  SPECTRA_REQUIRE(tokens > 0 && tokens < (1LL << 31) && tokens * (heads / kv->kv_heads) < (1LL << 30),
                  "tokens out of range");
  SPECTRA_REQUIRE(kv->k && kv->v && kv->block_table && kv->kv_lens && kv->q_start, "NULL pointer");
  SPECTRA_REQUIRE((reinterpret_cast<uintptr_t>(kv->block_table) | reinterpret_cast<uintptr_t>(kv->kv_lens) |
                   reinterpret_cast<uintptr_t>(kv->q_start)) % 4 == 0,
                  "block table, lengths and starts must be aligned");
  const int64_t rows = (int64_t)kv->kv_heads * kv->page_size;
  const int64_t row = q4 ? d / 2 : 2 * d;
  SPECTRA_REQUIRE(rows * row < (1LL << 31), "page too large");
  // (a pool of one page may have any page stride)
  SPECTRA_REQUIRE(kv->num_pages == 1 || kv->page_stride >= rows * (q4 ? d / 2 : d), "page stride too small");
  uintptr_t at = reinterpret_cast<uintptr_t>(kv->k) | reinterpret_cast<uintptr_t>(kv->v);
  int64_t step = kv->page_stride * (q4 ? 1 : 2);
  if (q4) {
    SPECTRA_REQUIRE(kv->k_scales && kv->v_scales && kv->k_zeros && kv->v_zeros, "4-bit pages need scales and zero points");
    SPECTRA_REQUIRE(kv->num_pages == 1 || (kv->scale_stride >= rows * (d / 32) && kv->zero_stride >= rows * (d / 32)),
                    "scale or zero-point page stride too small");
    at |= reinterpret_cast<uintptr_t>(kv->k_scales) | reinterpret_cast<uintptr_t>(kv->v_scales) |
          reinterpret_cast<uintptr_t>(kv->k_zeros) | reinterpret_cast<uintptr_t>(kv->v_zeros);
    step |= kv->scale_stride * 2 | kv->zero_stride;
  }
  SPECTRA_REQUIRE(at % 16 == 0 && (kv->num_pages == 1 || step % 16 == 0),
                  "pages must start at 16-byte aligned addresses");
  const int64_t far = kv->page_stride * (q4 ? 1 : 2);
  SPECTRA_REQUIRE(kv->num_pages == 1 || (far >> 4 < (1LL << 32) && kv->scale_stride >> 3 < (1LL << 32) && kv->zero_stride >> 4 < (1LL << 32)),
                  "page stride too large");
  const bool one = kv->num_pages == 1;
  int shift = 0;
  while ((1 << shift) < kv->page_size) ++shift;
  *out = PagedKv{(uint8_t*)kv->k, (uint8_t*)kv->v, (uint8_t*)kv->k_scales, (uint8_t*)kv->v_scales,
                 (uint8_t*)kv->k_zeros, (uint8_t*)kv->v_zeros, one ? 0 : (uint32_t)(far >> 4),
                 one ? 0 : (uint32_t)(kv->scale_stride >> 3), one ? 0 : (uint32_t)(kv->zero_stride >> 4),
                 kv->block_table, kv->kv_lens, kv->q_start, kv->table_stride, (int)kv->num_pages, kv->kv_heads, shift,
                 kv->batch, kv->table_width, (int)tokens};
  return SPECTRA_OK;
}

PagedPools paged_pools(const spectra_paged_kv_t* kv) {
  const bool q4 = kv->kind == SPECTRA_KV_4BIT;
  const int64_t rows = (int64_t)kv->kv_heads * kv->page_size, d = kv->head_dim, n = kv->num_pages;
  const int64_t row = q4 ? d / 2 : 2 * d, step = kv->page_stride * (q4 ? 1 : 2), sb = q4 ? rows * (d / 32) * 2 : 0, zb = sb / 2;
  return {{"the key pages", kv->k, rows * row, step, n},
          {"the value pages", kv->v, rows * row, step, n},
          {"the keys' scales", kv->k_scales, sb, kv->scale_stride * 2, n},
          {"the values' scales", kv->v_scales, sb, kv->scale_stride * 2, n},
          {"the keys' zero points", kv->k_zeros, zb, kv->zero_stride, n},
          {"the values' zero points", kv->v_zeros, zb, kv->zero_stride, n}};
}

int paged_apart(std::initializer_list<PagedRegion> written, std::initializer_list<PagedRegion> read) {
  // first by what the regions span, worked out once (most pairs lie apart: 0.1 us for all of a call's)
  constexpr int kMost = 24;
  const PagedRegion* r[kMost];
  uintptr_t from[kMost], to[kMost];
  int n = 0, nw = 0;
  for (const auto* list : {&written, &read}) {
    for (const PagedRegion& x : *list) {
      if (x.at == nullptr || x.bytes == 0) continue;
      const unsigned __int128 end = (unsigned __int128)reinterpret_cast<uintptr_t>(x.at) + x.bytes +
                                    (x.n > 1 ? (unsigned __int128)(x.n - 1) * (uint64_t)x.step : 0);
      r[n] = &x;
      from[n] = reinterpret_cast<uintptr_t>(x.at);
      to[n++] = end > UINTPTR_MAX ? UINTPTR_MAX : (uintptr_t)end;
    }
    if (list == &written) nw = n;
  }
  for (int i = 0; i < nw; ++i)
    for (int j = i + 1; j < n; ++j)
      if (from[i] < to[j] && from[j] < to[i] && paged_meet(*r[i], *r[j]))
        return fail(SPECTRA_ERR_INVALID, std::string(r[i]->name) + " must not overlap " + r[j]->name);
  return SPECTRA_OK;
}

}  // namespace spectra

using namespace spectra;

namespace {
// Both entries: positions of the sequences, or of axes of their own.
int append(const spectra_paged_kv_t* kv, const void* qkv, int64_t ldqkv, int64_t tokens, const PagedAxes* axes,
           const float* cos_t, const float* sin_t, int64_t rope_rows, int32_t heads, void* q_rot, spectra_stream_t stream) {
  PagedKv p;
  if (int st = paged_args(kv, tokens, heads, &p); st != SPECTRA_OK) return st;
  SPECTRA_REQUIRE(qkv && q_rot, "NULL pointer");
  SPECTRA_REQUIRE((cos_t == nullptr) == (sin_t == nullptr), "cos and sin must both be given or both be NULL");
  SPECTRA_REQUIRE(cos_t == nullptr || rope_rows > 0, "rope_rows must be positive");
  const int hd = kv->head_dim;
  SPECTRA_REQUIRE(ldqkv >= (int64_t)(heads + 2 * kv->kv_heads) * hd, "qkv row stride too small");
  SPECTRA_REQUIRE(((reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(q_rot) |
                    reinterpret_cast<uintptr_t>(cos_t) | reinterpret_cast<uintptr_t>(sin_t)) % 16) == 0 &&
                      ldqkv % 8 == 0,
                  "operands and qkv rows must be 16-byte aligned");
  PagedAxes ax{};
  if (axes != nullptr) {
    ax = *axes;
    SPECTRA_REQUIRE(ax.pos && ax.axis && cos_t, "NULL pointer");
    SPECTRA_REQUIRE(ax.axes >= 1 && ax.axes <= kPagedAxes, "one to four axes");
    SPECTRA_REQUIRE(ax.stride >= tokens || ax.axes == 1, "positions' row stride too small");
    SPECTRA_REQUIRE(reinterpret_cast<uintptr_t>(ax.pos) % 4 == 0, "positions must be aligned");
  }
  const PagedPools pools = paged_pools(kv);
  const int64_t turned = 2 * std::min<int64_t>(rope_rows, 1LL << 31) * hd;  // bytes of each table that positions name
  if (int st = paged_apart({{"q_rot", q_rot, tokens * heads * hd * 2, 0, 1}, pools.k, pools.v, pools.ks, pools.vs, pools.kz, pools.vz},
                           {{"qkv", qkv, (int64_t)(heads + 2 * kv->kv_heads) * hd * 2, ldqkv * 2, tokens},
                            {"cos", cos_t, turned, 0, 1},
                            {"sin", sin_t, turned, 0, 1},
                            {"positions", ax.pos, 4 * tokens, 4 * ax.stride, ax.axes},
                            {"axis", ax.axis, hd / 2, 0, 1},
                            paged_table(kv),
                            paged_lens(kv),
                            paged_starts(kv)});
      st != SPECTRA_OK)
    return st;
  int waves = ((heads + kv->kv_heads) * (hd / 16) + kv->kv_heads * (hd / 8) + 63) / 64;
  int64_t blocks = (tokens * waves + kPaThreads / 64 - 1) / (kPaThreads / 64);
  if (blocks >= 64) blocks = (blocks + 7) / 8 * 8;
  SPECTRA_REQUIRE(tokens * waves < (1LL << 31) - 256, "tokens out of range");
  const bool q4 = kv->kind == SPECTRA_KV_4BIT, bf = kv->kind == SPECTRA_KV_BF16;
  const void* kern = axes == nullptr ? (q4   ? (const void*)paged_append_kernel<false, true, false>
                                        : bf ? (const void*)paged_append_kernel<true, false, false>
                                             : (const void*)paged_append_kernel<false, false, false>)
                     : q4 ? (const void*)paged_append_kernel<false, true, true>
                     : bf ? (const void*)paged_append_kernel<true, false, true>
                          : (const void*)paged_append_kernel<false, false, true>;
  int hdv = hd;
  void* args[] = {(void*)&qkv, (void*)&ldqkv, (void*)&cos_t, (void*)&sin_t, (void*)&rope_rows, (void*)&heads,
                  (void*)&hdv, (void*)&waves, (void*)&p, (void*)&q_rot, (void*)&ax};
  SPECTRA_HIP_CHECK(hipLaunchKernel(kern, dim3((unsigned)blocks), dim3(kPaThreads), args, 0, (hipStream_t)stream));
  SPECTRA_HIP_CHECK(hipGetLastError());
  return SPECTRA_OK;
}
}  // namespace

extern "C" int spectra_paged_rope_append(const spectra_paged_kv_t* kv, const void* qkv, int64_t ldqkv, int64_t tokens,
                                         const float* cos_t, const float* sin_t, int64_t rope_rows, int32_t heads,
                                         void* q_rot, spectra_stream_t stream) {
  return append(kv, qkv, ldqkv, tokens, nullptr, cos_t, sin_t, rope_rows, heads, q_rot, stream);
}

extern "C" int spectra_paged_rope_axes_append(const spectra_paged_kv_t* kv, const void* qkv, int64_t ldqkv, int64_t tokens,
                                              const int32_t* positions, int64_t ldpos, int32_t axes, const uint8_t* axis,
                                              const float* cos_t, const float* sin_t, int64_t rope_rows, int32_t heads,
                                              void* q_rot, spectra_stream_t stream) {
  const PagedAxes ax = {positions, ldpos, axis, axes};
  return append(kv, qkv, ldqkv, tokens, &ax, cos_t, sin_t, rope_rows, heads, q_rot, stream);
}
