// Rotation and the 4-bit KV quantizer, shared by the contiguous and the paged caches.
#pragma once

#include "common.h"

namespace spectra {

__device__ __forceinline__ void unpack8(const uint4& u, float (&f)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    f[2 * e] = h2f((uint16_t)w[e]);
    f[2 * e + 1] = h2f((uint16_t)(w[e] >> 16));
  }
}

// The reference's 4-bit KV quantizer (engine.py:624-656) on fp16 values, for the 8 values
// of one lane; the 32-value group is 4 consecutive lanes.  Each torch op rounds where the
// reference's does: range and scale to fp16 (range / 15), zero point fp16(-min / scale)
// rounded half to even and clamped to [0, 15], codes round((t + z * s) / s) in fp32 clamped
// to [0, 15]; in fp16 the reference's 1e-8 threshold and scale floor are 0, so a constant
// group has scale 0 (its codes and zero point come from inf / NaN: NaN -> 0, +inf -> 15).
__device__ __forceinline__ void kv4_quant_chunk(const uint4& x, uint32_t& packed, uint16_t& sbits, uint8_t& zero) {
  float f[8];
  unpack8(x, f);
  float mn = f[0], mx = f[0];
#pragma unroll
  for (int e = 1; e < 8; ++e) {
    mn = fminf(mn, f[e]);
    mx = fmaxf(mx, f[e]);
  }
  mn = fminf(mn, __shfl_xor(mn, 1, 64));
  mn = fminf(mn, __shfl_xor(mn, 2, 64));
  mx = fmaxf(mx, __shfl_xor(mx, 1, 64));
  mx = fmaxf(mx, __shfl_xor(mx, 2, 64));
  const float diff = h2f(f2h(mx - mn));
  const float sc = h2f(f2h(diff / 15.0f));
  const float zq = h2f(f2h(-mn / sc));
  const float zf = fminf(fmaxf(rintf(zq), 0.0f), 15.0f);  // NaN -> 0 (fmaxf returns the number)
  uint32_t pk = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float qv = fminf(fmaxf(rintf((f[e] + zf * sc) / sc), 0.0f), 15.0f);
    pk |= (uint32_t)qv << (4 * e);
  }
  packed = pk;
  sbits = f2h(sc);
  zero = (uint8_t)zf;
}

// Rotation of the 8-dim chunk `own` of a head whose partner chunk (dims -+ head_dim/2) is
// `partner`, with the cos/sin of the chunk's pair indices: the lower half takes
// a*c - b*s, the upper half b*c + a*s (a = dim i, b = dim i + head_dim/2), each product and
// the sum rounded in fp32 as written, the result to fp16 -- the rope_append arithmetic.
__device__ __forceinline__ uint4 rope_chunk(const uint4& own, const uint4& partner, const float (&c)[8],
                                            const float (&s)[8], bool upper) {
  float x[8], y[8];
  unpack8(own, x);
  unpack8(partner, y);
  uint32_t o[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float r[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int i = 2 * e + h;
      r[h] = upper ? x[i] * c[i] + y[i] * s[i] : x[i] * c[i] - y[i] * s[i];
    }
    o[e] = (uint32_t)f2h(r[0]) | ((uint32_t)f2h(r[1]) << 16);
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

// Partials cross workgroups (and XCDs, whose L2 caches are not coherent with each other)
// as device-scope relaxed atomics: stores write through to the device's coherence point,
// loads read from it.
__device__ __forceinline__ void store_dev(float* p, float v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float load_dev(const float* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

}  // namespace spectra
