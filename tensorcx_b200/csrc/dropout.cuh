// The dropout map shared by the elementwise kernel (dropout.cu) and the norm kernels that
// apply it on the way (norm_train.cu). Element e of a call is kept when the uniform value of
// place start + e in the seed's stream, a whole number w of 24 bits times 2^-24, is at least
// p: w >= threshold = ceil(p * 2^24), so the mask equals rand_uniform(...) >= p with p as the
// 64-bit number that it is (rounded to 32 bits first, a p above 1/2 may move by one of the 2^24
// values). The mask is a function of (seed, place): nothing stores it, the backward pass makes it again.
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

// output = residual + dropout(input), or dropout(input) without a residual (dropout.cu).
void launch_dropout(cudaStream_t s, const float* input, const float* residual, float* output, int64_t count,
                    const Dropout& d);

__device__ __forceinline__ uint64_t dropout_start(const Dropout& d) {
  return d.offset + (d.step_offset ? static_cast<uint64_t>(__ldg(d.step_offset)) : 0);
}

__device__ __forceinline__ uint32_t word_of(uint4 w, uint32_t i) {
  const uint32_t lo = i & 1u ? w.y : w.x, hi = i & 1u ? w.w : w.z;
  return i & 2u ? hi : lo;
}

__device__ __forceinline__ bool kept(uint32_t word, uint32_t threshold) { return (word >> 8) >= threshold; }

__device__ __forceinline__ float dropped(float x, bool keep, float scale) {
  return keep ? __fmul_rn(x, scale) : 0.0f;
}

// Bit j: word j of the block is kept. Places are taken modulo 2^64, so that blocks are modulo
// 2^62: the next one after the stream's last is its first.
__device__ __forceinline__ uint32_t kept_block(uint64_t block, const philox::RoundKeys& rk, uint32_t threshold) {
  const uint4 w = philox::block_words(block & (~0ull >> 2), rk);
  return (kept(w.x, threshold) ? 1u : 0u) | (kept(w.y, threshold) ? 2u : 0u) | (kept(w.z, threshold) ? 4u : 0u) |
         (kept(w.w, threshold) ? 8u : 0u);
}

// Bit 4 k + j: place e + 4 k stride + j is kept, k < WORDS (at most 8). For whole warps, the
// places of whose LANES lanes (32, or each 16 or 8 of them) lie 4 apart. Where they do not start
// a block, a lane's words end in the next lane's blocks, and the last lane's in WORDS blocks of
// which each lane makes one. e must lie alike within a block for all lanes of the warp.
template <int WORDS, int LANES = 32>
__device__ __forceinline__ uint32_t kept_words(uint64_t e, uint32_t stride, const philox::RoundKeys& rk,
                                               uint32_t threshold) {
  static_assert(WORDS <= 8, "the mask's bits");
  static_assert(WORDS <= LANES, "a lane to each of the last lane's blocks");
  const uint64_t block = e >> 2;
  const int r = static_cast<int>(e & 3);  // the same for all lanes
  uint32_t mask = 0;
#pragma unroll
  for (int k = 0; k < WORDS; ++k) mask |= kept_block(block + k * stride, rk, threshold) << (4 * k);
  if (r == 0) return mask;
  const int lane = threadIdx.x & (LANES - 1);
  uint32_t next = __shfl_down_sync(0xffffffffu, mask, 1, LANES), ends = 0;
  const uint64_t after = __shfl_sync(0xffffffffu, block, LANES - 1, LANES) + 1;
  if (lane < WORDS) ends = kept_block(after + lane * stride, rk, threshold) << (4 * lane);
  if (LANES == 32) {
    ends = __reduce_or_sync(0xffffffffu, ends);
  } else {
#pragma unroll
    for (int off = LANES / 2; off > 0; off >>= 1) ends |= __shfl_xor_sync(0xffffffffu, ends, off);
  }
  if (lane == LANES - 1) next = ends;
  // bits r .. 3 of each word's own block, then bits 0 .. r - 1 of the next one
  const uint32_t low = 0x11111111u * (0xfu >> r);
  return ((mask >> r) & low) | ((next << (4 - r)) & ~low);
}

}  // namespace tcx
