// The counter-based generator behind every random number of the library: Philox4x32-10
// (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC'11).
// Element e of the stream of `seed` is word e % 4 of the block of counter (e / 4, 0, 0)
// under the key `seed`, so a value depends on (seed, e) alone.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace tcx {
namespace philox {

constexpr uint32_t kPhiloxM0 = 0xD2511F53u, kPhiloxM1 = 0xCD9E8D57u;  // round multipliers
constexpr uint32_t kPhiloxW0 = 0x9E3779B9u, kPhiloxW1 = 0xBB67AE85u;  // key schedule (Weyl)
// The ten round keys of `key` (the Weyl sequence), computed once per thread.
struct RoundKeys {
  uint32_t x[10], y[10];
};
__device__ __forceinline__ RoundKeys round_keys(uint2 k) {
  RoundKeys rk;
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    rk.x[r] = k.x + static_cast<uint32_t>(r) * kPhiloxW0;
    rk.y[r] = k.y + static_cast<uint32_t>(r) * kPhiloxW1;
  }
  return rk;
}

__device__ __forceinline__ uint4 philox4x32_10(uint4 c, const RoundKeys& rk) {
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t p0 = static_cast<uint64_t>(kPhiloxM0) * c.x, p1 = static_cast<uint64_t>(kPhiloxM1) * c.z;
    const uint32_t hi0 = static_cast<uint32_t>(p0 >> 32), lo0 = static_cast<uint32_t>(p0);
    const uint32_t hi1 = static_cast<uint32_t>(p1 >> 32), lo1 = static_cast<uint32_t>(p1);
    c = make_uint4(hi1 ^ c.y ^ rk.x[r], lo1, hi0 ^ c.w ^ rk.y[r], lo0);
  }
  return c;
}

__device__ __forceinline__ uint4 block_words(uint64_t blk, const RoundKeys& rk) {
  return philox4x32_10(make_uint4(static_cast<uint32_t>(blk), static_cast<uint32_t>(blk >> 32), 0u, 0u), rk);
}

}  // namespace philox
}  // namespace tcx
