// Layer norm for training on sm_100a: the forward pass that keeps its row statistics and the
// backward pass with the weight's and the bias's gradients, both with the dropout and the
// residual addition around the norm in the same pass. Rows are the last axis.
//
//   total = residual + dropout(x),  mean = sum(total) / n,
//   rstd = 1 / sqrt(sum((total - mean)^2) / n + eps),  y = (total - mean) rstd w + b
//
//   xhat = (total - mean) rstd,  g = dy w,
//   dtotal' = dtotal + rstd (g - sum(g) / n - xhat sum(g xhat) / n),
//   dx = dropout'(dtotal'),  dw = sum over rows of dy xhat,  db = sum over rows of dy
//
// The mean is taken about the row's first element f and corrected about its own first value:
// m1 = f + sum(x - f) / n, mean = m1 + sum(x - m1) / n, and the variance is
// sum((x - m1)^2) / n - (sum(x - m1) / n)^2. A constant row then has mean f and variance 0
// exactly, and a row whose level is far above its spread loses nothing in the sum.
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "common.cuh"
#include "dropout.cuh"
#include "rowmath.cuh"

namespace tcx {
namespace {

using rowmath::Block;

constexpr int kThreads = 256;

struct ForwardArgs {
  const float *x, *residual, *weight, *bias;
  float *y, *total, *mean, *rstd;
  int64_t rows, cols;
  float eps;
  Dropout drop;
};

__global__ void __launch_bounds__(kThreads) norm_forward_kernel(ForwardArgs a) {
  __shared__ float smem[64];
  using B = Block<kThreads>;
  const philox::RoundKeys rk = philox::round_keys(a.drop.key);
  const uint64_t start = dropout_start(a.drop);
  const float n = static_cast<float>(a.cols);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const int64_t base = row * a.cols;
    auto value = [&](int64_t c) {
      float v = a.x[base + c];
      if (a.drop.threshold) {
        const uint64_t e = start + static_cast<uint64_t>(base + c);
        const uint4 w = philox::block_words(e >> 2, rk);
        v = dropped(v, kept(word_of(w, static_cast<uint32_t>(e & 3)), a.drop.threshold), a.drop.scale);
      }
      return a.residual ? __fadd_rn(a.residual[base + c], v) : v;
    };
    const float first = value(0);
    float s = 0.0f;
    for (int64_t c = threadIdx.x; c < a.cols; c += kThreads) {
      const float v = value(c);
      if (a.total) a.total[base + c] = v;
      s += v - first;
    }
    const float m1 = first + B::sum(s, smem) / n;
    const float* t = a.total ? a.total : a.x;
    float s1 = 0.0f, s2 = 0.0f;
    for (int64_t c = threadIdx.x; c < a.cols; c += kThreads) {
      const float dlt = t[base + c] - m1;
      s1 += dlt;
      s2 += dlt * dlt;
    }
    const float2 r = B::sum2(s1, s2, smem);
    const float shift = r.x / n;
    const float mean = m1 + shift;
    float var = r.y / n - shift * shift;
    if (var < 0.0f) var = 0.0f;  // rounding; a NaN stays one
    const float rstd = 1.0f / sqrtf(var + a.eps);
    for (int64_t c = threadIdx.x; c < a.cols; c += kThreads) {
      float y = (t[base + c] - mean) * rstd;
      if (a.weight) y *= a.weight[c];
      if (a.bias) y += a.bias[c];
      a.y[base + c] = y;
    }
    if (threadIdx.x == 0) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
    __syncthreads();
  }
}

struct BackwardArgs {
  const float *dy, *total, *mean, *rstd, *weight, *dtotal;
  float *dresidual, *dx;
  int64_t rows, cols;
  Dropout drop;
};

__global__ void __launch_bounds__(kThreads) norm_backward_kernel(BackwardArgs a) {
  __shared__ float smem[64];
  using B = Block<kThreads>;
  const philox::RoundKeys rk = philox::round_keys(a.drop.key);
  const uint64_t start = dropout_start(a.drop);
  const float n = static_cast<float>(a.cols);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const int64_t base = row * a.cols;
    const float mean = a.mean[row], rstd = a.rstd[row];
    float s1 = 0.0f, s2 = 0.0f;
    for (int64_t c = threadIdx.x; c < a.cols; c += kThreads) {
      const float g = a.weight ? a.dy[base + c] * a.weight[c] : a.dy[base + c];
      s1 += g;
      s2 += g * ((a.total[base + c] - mean) * rstd);
    }
    const float2 r = B::sum2(s1, s2, smem);
    const float c1 = r.x / n, c2 = r.y / n;
    for (int64_t c = threadIdx.x; c < a.cols; c += kThreads) {
      const float g = a.weight ? a.dy[base + c] * a.weight[c] : a.dy[base + c];
      const float hat = (a.total[base + c] - mean) * rstd;
      float d = rstd * (g - c1 - hat * c2);
      if (a.dtotal) d += a.dtotal[base + c];
      a.dresidual[base + c] = d;
      if (a.dx) {
        const uint64_t e = start + static_cast<uint64_t>(base + c);
        const uint4 w = philox::block_words(e >> 2, rk);
        a.dx[base + c] = dropped(d, kept(word_of(w, static_cast<uint32_t>(e & 3)), a.drop.threshold), a.drop.scale);
      }
    }
    __syncthreads();
  }
}

// Partial column sums of rows [split * per, (split + 1) * per): partial[2 split] holds the
// weight's, partial[2 split + 1] the bias's.
__global__ void __launch_bounds__(kThreads) norm_columns_kernel(BackwardArgs a, float* partial, int64_t per) {
  const int64_t c = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (c >= a.cols) return;
  const int64_t r0 = blockIdx.y * per, r1 = min(r0 + per, a.rows);
  float dw = 0.0f, db = 0.0f;
  for (int64_t r = r0; r < r1; ++r) {
    const float dy = a.dy[r * a.cols + c];
    dw += dy * ((a.total[r * a.cols + c] - a.mean[r]) * a.rstd[r]);
    db += dy;
  }
  partial[(2 * blockIdx.y) * a.cols + c] = dw;
  partial[(2 * blockIdx.y + 1) * a.cols + c] = db;
}

__global__ void __launch_bounds__(kThreads)
norm_columns_join_kernel(const float* partial, int64_t splits, int64_t cols, float* dweight, float* dbias) {
  const int64_t c = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (c >= cols) return;
  float dw = 0.0f, db = 0.0f;
  for (int64_t i = 0; i < splits; ++i) {
    dw += partial[2 * i * cols + c];
    db += partial[(2 * i + 1) * cols + c];
  }
  dweight[c] = dw;
  dbias[c] = db;
}

int64_t splits_of(int64_t rows) { return std::max<int64_t>(1, std::min<int64_t>(64, rows / 16)); }

int check_norm(int64_t rows, int64_t cols) {
  if (rows < 0 || cols < 0) return invalid("negative extent");
  if (cols == 0) return invalid("layer norm requires a non-empty last axis");
  if (rows > INT64_MAX / cols) return invalid("element count overflows");
  return TCX_OK;
}

}  // namespace
}  // namespace tcx

using namespace tcx;

extern "C" int tcx_sm100_layernorm_forward(tcx_stream_t stream, const float* input, const float* residual,
                                           const float* weight, const float* bias, float* output, float* total,
                                           float* mean, float* rstd, int64_t rows, int64_t cols, float epsilon,
                                           double p, uint64_t seed, uint64_t offset, const int64_t* step_offset) {
  clear_error();
  if (int rc = check_norm(rows, cols)) return rc;
  if (!(epsilon >= 0.0f) || epsilon == INFINITY) return invalid("epsilon must be finite and non-negative");
  ForwardArgs a{input, residual, weight, bias, output, total, mean, rstd, rows, cols, epsilon, {}};
  if (!make_dropout(a.drop, p, seed, offset, step_offset)) return TCX_INVALID_ARGUMENT;
  if (rows == 0) return TCX_OK;
  if (!input || !output || !mean || !rstd) return invalid("missing buffer");
  if ((residual || a.drop.threshold) && !total) return invalid("dropout or a residual needs a buffer for the total");
  if (!residual && !a.drop.threshold) a.total = nullptr;  // it is the input
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const int grid = static_cast<int>(std::min<int64_t>(rows, 8 * sm_count()));
  TimedLaunch timer("norm_forward", s);
  norm_forward_kernel<<<grid, kThreads, 0, s>>>(a);
  return launch_status("layer norm forward");
}

extern "C" size_t tcx_sm100_layernorm_backward_workspace_bytes(int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0) return 0;
  return static_cast<size_t>(splits_of(rows)) * 2 * cols * sizeof(float);
}

extern "C" int tcx_sm100_layernorm_backward(tcx_stream_t stream, const float* dy, const float* total,
                                            const float* mean, const float* rstd, const float* weight,
                                            const float* dtotal, float* dresidual, float* dx, float* dweight,
                                            float* dbias, int64_t rows, int64_t cols, double p, uint64_t seed,
                                            uint64_t offset, const int64_t* step_offset, void* workspace,
                                            size_t workspace_bytes) {
  clear_error();
  if (int rc = check_norm(rows, cols)) return rc;
  BackwardArgs a{dy, total, mean, rstd, weight, dtotal, dresidual, dx, rows, cols, {}};
  if (!make_dropout(a.drop, p, seed, offset, step_offset)) return TCX_INVALID_ARGUMENT;
  if ((dweight == nullptr) != (dbias == nullptr))
    return invalid("the weight's and the bias's gradient are given together or not at all");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (rows == 0) {
    if (dweight) {
      cudaMemsetAsync(dweight, 0, cols * sizeof(float), s);
      cudaMemsetAsync(dbias, 0, cols * sizeof(float), s);
    }
    return launch_status("layer norm backward");
  }
  if (!dy || !total || !mean || !rstd || !dresidual) return invalid("missing buffer");
  if (a.drop.threshold && !dx) return invalid("dropout needs a buffer for the input's gradient");
  if (!a.drop.threshold) a.dx = nullptr;  // it is the residual's gradient
  if (dweight && workspace_bytes < tcx_sm100_layernorm_backward_workspace_bytes(rows, cols))
    return invalid("workspace too small for the layer norm gradient");
  TimedLaunch timer("norm_backward", s);
  const int grid = static_cast<int>(std::min<int64_t>(rows, 8 * sm_count()));
  norm_backward_kernel<<<grid, kThreads, 0, s>>>(a);
  if (dweight) {
    const int64_t splits = splits_of(rows);
    const unsigned blocks = static_cast<unsigned>(ceil_div(cols, kThreads));
    float* partial = static_cast<float*>(workspace);
    norm_columns_kernel<<<dim3(blocks, static_cast<unsigned>(splits)), kThreads, 0, s>>>(a, partial,
                                                                                         ceil_div(rows, splits));
    norm_columns_join_kernel<<<blocks, kThreads, 0, s>>>(partial, splits, cols, dweight, dbias);
  }
  return launch_status("layer norm backward");
}
