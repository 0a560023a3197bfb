// Dropout on sm_100a: output = residual + (kept ? input * scale : 0), the mask from the
// counter-based stream (dropout.cuh). The backward pass is the same map on the gradient.
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"
#include "dropout.cuh"

namespace tcx {
namespace {

__global__ void __launch_bounds__(256)
dropout_kernel(const float* __restrict__ x, const float* __restrict__ residual, float* __restrict__ out,
               int64_t count, Dropout d) {
  const philox::RoundKeys rk = philox::round_keys(d.key);
  const uint64_t start = dropout_start(d);
  const int64_t stride = static_cast<int64_t>(gridDim.x) * blockDim.x;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < count; i += stride) {
    const uint64_t e = start + static_cast<uint64_t>(i);
    const uint4 w = philox::block_words(e >> 2, rk);
    const float y = dropped(x[i], kept(word_of(w, static_cast<uint32_t>(e & 3)), d.threshold), d.scale);
    out[i] = residual ? __fadd_rn(residual[i], y) : y;
  }
}

}  // namespace
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
  const int64_t want = ceil_div(count, 256);
  const int grid = static_cast<int>(want < 8 * sm_count() ? want : 8 * sm_count());
  TimedLaunch timer("dropout", s);
  dropout_kernel<<<grid, 256, 0, s>>>(input, residual, output, count, d);
  return launch_status("dropout");
}
