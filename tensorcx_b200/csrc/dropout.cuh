// The dropout map shared by the elementwise kernel (dropout.cu) and the norm kernels that
// apply it on the way (norm_train.cu). Element e of a call is kept when the uniform value of
// place start + e in the seed's stream, a whole number w of 24 bits times 2^-24, is at least
// p: w >= threshold = ceil(p * 2^24), so the mask equals rand_uniform(...) >= p exactly. The
// mask is a function of (seed, place): nothing stores it, the backward pass makes it again.
// A kept element is multiplied by scale = 1 / (1 - p) rounded to float32; a dropped one is 0
// whatever it held (infinities and NaN included).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <cmath>

#include "common.cuh"
#include "philox.cuh"

namespace tcx {

struct Dropout {
  uint2 key;
  uint64_t offset;             // place of element 0
  const int64_t* step_offset;  // added to it when not NULL (a device value: see the header)
  uint32_t threshold;          // 0 keeps everything
  float scale;
};

// The call's parameters; false (with the error set) when p is not in [0, 1].
inline bool make_dropout(Dropout& d, double p, uint64_t seed, uint64_t offset, const int64_t* step_offset) {
  if (!(p >= 0.0 && p <= 1.0)) {
    set_error("dropout probability must be in [0, 1]");
    return false;
  }
  d.key = make_uint2(static_cast<uint32_t>(seed), static_cast<uint32_t>(seed >> 32));
  d.offset = offset;
  d.step_offset = step_offset;
  d.threshold = static_cast<uint32_t>(std::ceil(p * 16777216.0));  // exact: p * 2^24 only moves the exponent
  d.scale = p < 1.0 ? static_cast<float>(1.0 / (1.0 - p)) : 0.0f;
  return true;
}

__device__ __forceinline__ uint64_t dropout_start(const Dropout& d) {
  return d.offset + (d.step_offset ? static_cast<uint64_t>(__ldg(d.step_offset)) : 0);
}

__device__ __forceinline__ uint32_t word_of(uint4 w, uint32_t i) {
  const uint32_t lo = i & 1u ? w.y : w.x, hi = i & 1u ? w.w : w.z;
  return i & 2u ? hi : lo;
}

// The words of places e .. e + 3: one block when e starts one, else two.
__device__ __forceinline__ uint4 words_at(uint64_t e, const philox::RoundKeys& rk) {
  const uint4 a = philox::block_words(e >> 2, rk);
  const uint32_t r = static_cast<uint32_t>(e & 3);
  if (r == 0) return a;
  const uint4 b = philox::block_words((e >> 2) + 1, rk);
  return r == 1 ? make_uint4(a.y, a.z, a.w, b.x) : r == 2 ? make_uint4(a.z, a.w, b.x, b.y) : make_uint4(a.w, b.x, b.y, b.z);
}

__device__ __forceinline__ bool kept(uint32_t word, uint32_t threshold) { return (word >> 8) >= threshold; }

__device__ __forceinline__ float dropped(float x, bool keep, float scale) {
  return keep ? __fmul_rn(x, scale) : 0.0f;
}

// Bit j: place e + j is kept.
__device__ __forceinline__ uint32_t kept4(uint64_t e, const philox::RoundKeys& rk, uint32_t threshold) {
  const uint4 w = words_at(e, rk);
  return (kept(w.x, threshold) ? 1u : 0u) | (kept(w.y, threshold) ? 2u : 0u) | (kept(w.z, threshold) ? 4u : 0u) |
         (kept(w.w, threshold) ? 8u : 0u);
}

__device__ __forceinline__ float4 dropped4(float4 x, uint64_t e, const philox::RoundKeys& rk, uint32_t threshold,
                                           float scale) {
  const uint4 w = words_at(e, rk);
  return make_float4(dropped(x.x, kept(w.x, threshold), scale), dropped(x.y, kept(w.y, threshold), scale),
                     dropped(x.z, kept(w.z, threshold), scale), dropped(x.w, kept(w.w, threshold), scale));
}

}  // namespace tcx
