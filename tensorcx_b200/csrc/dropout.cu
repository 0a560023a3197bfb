// Dropout on sm_100a: output = residual + (kept ? input * scale : 0), the mask from the
// counter-based stream (dropout.cuh). The backward pass is the same map on the gradient.
//
// Bound by memory (8 bytes an element, 12 with a residual) as long as the mask costs less than
// the bytes do: a Philox block, some 60 integer instructions, serves four elements. Each thread
// takes kWords words of 16 bytes, a block's threads side by side, and makes their mask while
// its loads are on their way. Where element 0 does not stand at the start of a random block, a
// word takes its bits from two blocks; the second is the next lane's first.
//
// Measured on one B200: [16384, 4096] with a residual 119 us (6.8 TB/s, 1.04 of a copy's rate),
// without 90, the vector units issuing 46 % of the time. Buffers that are not 16-byte aligned take
// an element to a thread and a Philox block to each: 272 and 257 us.
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"
#include "dropout.cuh"

namespace tcx {
namespace {

constexpr int kThreads = 256, kWords = 4;  // words of a thread per turn

template <bool RESIDUAL>
__global__ void __launch_bounds__(kThreads)
dropout_kernel(const float* x, const float* residual, float* out, int64_t count, Dropout d) {
  const philox::RoundKeys rk = philox::round_keys(d.key);
  const uint64_t start = dropout_start(d);
  const int64_t words = count >> 2, span = kThreads * kWords;
  for (int64_t base = blockIdx.x * span; base < words; base += gridDim.x * span) {
    const int64_t first = base + threadIdx.x;
    float4 v[kWords], r[kWords];
#pragma unroll
    for (int k = 0; k < kWords; ++k) {
      const int64_t w = first + k * kThreads;
      if (w < words) {
        v[k] = __ldcs(reinterpret_cast<const float4*>(x) + w);
        if (RESIDUAL) r[k] = __ldcs(reinterpret_cast<const float4*>(residual) + w);
      }
    }
    uint32_t mask = ~0u;
    if (d.threshold) mask = kept_words<kWords>(start + 4 * static_cast<uint64_t>(first), kThreads, rk, d.threshold);
#pragma unroll
    for (int k = 0; k < kWords; ++k) {
      const int64_t w = first + k * kThreads;
      if (w < words) {
        const uint32_t m = mask >> (4 * k);
        float4 y = make_float4(dropped(v[k].x, m & 1, d.scale), dropped(v[k].y, m & 2, d.scale),
                               dropped(v[k].z, m & 4, d.scale), dropped(v[k].w, m & 8, d.scale));
        if (RESIDUAL)
          y = make_float4(__fadd_rn(r[k].x, y.x), __fadd_rn(r[k].y, y.y), __fadd_rn(r[k].z, y.z),
                          __fadd_rn(r[k].w, y.w));
        __stcs(reinterpret_cast<float4*>(out) + w, y);
      }
    }
  }
  // the last elements of a count that is not a multiple of 4
  const int64_t i = 4 * words + threadIdx.x;
  if (blockIdx.x == 0 && i < count) {
    const uint64_t e = start + static_cast<uint64_t>(i);
    const uint4 w = philox::block_words(e >> 2, rk);
    const float y = dropped(x[i], kept(word_of(w, static_cast<uint32_t>(e & 3)), d.threshold), d.scale);
    out[i] = RESIDUAL ? __fadd_rn(residual[i], y) : y;
  }
}

// Buffers that are not 16-byte aligned: an element to a thread.
__global__ void __launch_bounds__(kThreads)
dropout_elements_kernel(const float* x, const float* residual, float* out, int64_t count, Dropout d) {
  const philox::RoundKeys rk = philox::round_keys(d.key);
  const uint64_t start = dropout_start(d);
  const int64_t stride = static_cast<int64_t>(gridDim.x) * kThreads;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < count; i += stride) {
    const uint64_t e = start + static_cast<uint64_t>(i);
    const uint4 w = philox::block_words(e >> 2, rk);
    const float y = dropped(x[i], kept(word_of(w, static_cast<uint32_t>(e & 3)), d.threshold), d.scale);
    out[i] = residual ? __fadd_rn(residual[i], y) : y;
  }
}

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace

void launch_dropout(cudaStream_t s, const float* input, const float* residual, float* output, int64_t count,
                    const Dropout& d) {
  if (aligned(input) && aligned(residual) && aligned(output)) {
    const int64_t want = count < 4 ? 1 : ceil_div(count >> 2, kThreads * kWords);
    const unsigned grid = static_cast<unsigned>(want < (1 << 30) ? want : 1 << 30);
    if (residual) dropout_kernel<true><<<grid, kThreads, 0, s>>>(input, residual, output, count, d);
    else dropout_kernel<false><<<grid, kThreads, 0, s>>>(input, residual, output, count, d);
  } else {
    const int64_t want = ceil_div(count, kThreads);
    const unsigned grid = static_cast<unsigned>(want < 16 * sm_count() ? want : 16 * sm_count());
    dropout_elements_kernel<<<grid, kThreads, 0, s>>>(input, residual, output, count, d);
  }
}

}  // namespace tcx

using namespace tcx;

extern "C" int tcx_sm100_dropout(tcx_stream_t stream, const float* input, const float* residual, float* output,
                                 int64_t count, double p, uint64_t seed, uint64_t offset,
                                 const int64_t* step_offset) {
  clear_error();
  if (count < 0) return invalid("negative element count");
  Dropout d;
  if (!make_dropout(d, p, seed, offset, step_offset)) return TCX_INVALID_ARGUMENT;
  if (count == 0) return TCX_OK;
  if (!input || !output) return invalid("missing buffer");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  TimedLaunch timer("dropout", s);
  launch_dropout(s, input, residual, output, count, d);
  return launch_status("dropout");
}
