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
#include "ptx.cuh"
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

__global__ void __launch_bounds__(kThreads) norm_forward_any_kernel(ForwardArgs a) {
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

__global__ void __launch_bounds__(kThreads) norm_backward_any_kernel(BackwardArgs a) {
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

// ------------------------------------------------------------------ rows in registers
// The tensor is read in 16-byte words at places that are multiples of 4 of the whole tensor,
// whatever the row length: a row of an odd length starts `phase` elements into its first word,
// and the words it shares with its neighbours are stored element by element. So every access
// is 128 bits wide, and a word of the tensor is a block of the random stream.
template <bool ODD>
struct Words {
  int64_t at;       // of the row's first word in the tensor
  int phase, cols;  // elements of that word before the row; elements of the row
  int64_t count;    // of the tensor

  __device__ Words(int64_t row, int64_t n, int64_t rows) {
    const int64_t first = row * n;
    phase = ODD ? static_cast<int>(first & 3) : 0;
    at = first - phase;
    cols = static_cast<int>(n);
    count = rows * n;
  }
  __device__ bool holds(int word) const { return 4 * word - phase < cols; }
  __device__ bool whole(int word) const { return !ODD || (4 * word >= phase && 4 * word + 4 - phase <= cols); }
  __device__ bool valid(int word, int j) const {
    const int c = 4 * word + j - phase;
    return !ODD || (c >= 0 && c < cols);
  }
  __device__ __forceinline__ float4 load(const float* p, int word) const {
    const int64_t i = at + 4 * static_cast<int64_t>(word);
    if (!ODD || i + 4 <= count) return __ldcs(reinterpret_cast<const float4*>(p + i));
    float4 v = make_float4(p[i], 0.0f, 0.0f, 0.0f);
    if (i + 1 < count) v.y = p[i + 1];
    if (i + 2 < count) v.z = p[i + 2];
    return v;
  }
  __device__ __forceinline__ void store(float* p, int word, float4 v) const {
    float* const q = p + at + 4 * static_cast<int64_t>(word);
    if (whole(word)) {
      __stcs(reinterpret_cast<float4*>(q), v);
    } else {
      if (valid(word, 0)) q[0] = v.x;
      if (valid(word, 1)) q[1] = v.y;
      if (valid(word, 2)) q[2] = v.z;
      if (valid(word, 3)) q[3] = v.w;
    }
  }
  // A word of a vector over the columns (nothing outside the row).
  __device__ __forceinline__ float4 column(const float* p, int word) const {
    if (!ODD) return __ldg(reinterpret_cast<const float4*>(p) + word);
    const float* const q = p + 4 * word - phase;
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (valid(word, 0)) v.x = __ldg(q);
    if (valid(word, 1)) v.y = __ldg(q + 1);
    if (valid(word, 2)) v.z = __ldg(q + 2);
    if (valid(word, 3)) v.w = __ldg(q + 3);
    return v;
  }
};

// One block to a row, VPT words to a thread. Each element is read once and written once; the
// statistics take two block reductions.
template <int THREADS, int VPT, bool ODD, bool FUSED>
__global__ void __launch_bounds__(THREADS) norm_forward_kernel(ForwardArgs a) {
  __shared__ float smem[64];
  using B = Block<THREADS>;
  const int tid = threadIdx.x;
  const float n = static_cast<float>(a.cols);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const Words<ODD> words(row, a.cols, a.rows);
    float v[VPT][4];
    const int64_t first = row * a.cols;
    float level;  // what the sums are taken about: the row's first element, or near it
    if (FUSED) {
      level = a.residual ? __ldg(a.residual + first) : 0.0f;
      if (!a.drop.threshold) level += __ldg(a.x + first);
    } else {
      level = __ldg(a.x + first);
    }
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      const int word = tid + k * THREADS;
      float4 t = make_float4(level, level, level, level);
      if (words.holds(word)) t = words.load(a.x, word);
      v[k][0] = t.x, v[k][1] = t.y, v[k][2] = t.z, v[k][3] = t.w;
    }
    if (FUSED) {
      const philox::RoundKeys rk = philox::round_keys(a.drop.key);
      const uint64_t start = dropout_start(a.drop) + static_cast<uint64_t>(words.at);
#pragma unroll
      for (int k = 0; k < VPT; ++k) {
        const int word = tid + k * THREADS;
        if (words.holds(word)) {
          float4 t = make_float4(v[k][0], v[k][1], v[k][2], v[k][3]);
          if (a.drop.threshold) t = dropped4(t, start + 4 * static_cast<uint64_t>(word), rk, a.drop.threshold, a.drop.scale);
          if (a.residual) {
            const float4 r = words.load(a.residual, word);
            t = make_float4(__fadd_rn(r.x, t.x), __fadd_rn(r.y, t.y), __fadd_rn(r.z, t.z), __fadd_rn(r.w, t.w));
          }
          words.store(a.total, word, t);
          v[k][0] = t.x, v[k][1] = t.y, v[k][2] = t.z, v[k][3] = t.w;
        }
      }
    }
    float s = 0.0f;
#pragma unroll
    for (int k = 0; k < VPT; ++k)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (words.valid(tid + k * THREADS, j)) s += v[k][j] - level;  // 0 past the row's words
    const float m1 = level + __fdiv_rn(B::sum(s, smem), n);
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      const int word = tid + k * THREADS;
      if (words.holds(word)) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v[k][j] -= m1;
          if (words.valid(word, j)) {
            s1 += v[k][j];
            s2 = fmaf(v[k][j], v[k][j], s2);
          }
        }
      }
    }
    const float2 r = B::sum2(s1, s2, smem);
    const float shift = __fdiv_rn(r.x, n);
    float var = __fdiv_rn(r.y, n) - shift * shift;
    if (var < 0.0f) var = 0.0f;  // rounding; a NaN stays one
    const float rstd = __fdiv_rn(1.0f, __fsqrt_rn(var + a.eps));
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      const int word = tid + k * THREADS;
      if (words.holds(word)) {
        float4 y = make_float4((v[k][0] - shift) * rstd, (v[k][1] - shift) * rstd, (v[k][2] - shift) * rstd,
                               (v[k][3] - shift) * rstd);
        if (a.weight) {
          const float4 w = words.column(a.weight, word);
          y = make_float4(y.x * w.x, y.y * w.y, y.z * w.z, y.w * w.w);
        }
        if (a.bias) {
          const float4 b = words.column(a.bias, word);
          y = make_float4(y.x + b.x, y.y + b.y, y.z + b.z, y.w + b.w);
        }
        words.store(a.y, word, y);
      }
    }
    if (tid == 0) {
      a.mean[row] = m1 + shift;
      a.rstd[row] = rstd;
    }
  }
}

// TPR threads (of CLUSTER blocks) to a row, VPT words to each, GROUPS rows to a block at a
// time. A group's rows are a multiple of 4 apart, so that they all start in the same phase
// and a thread's columns are the same in each: the weight's and the bias's gradients add up in
// its registers over the group's rows, the groups' in shared memory, and the blocks' in a
// second kernel, each in a fixed order. The next row's words are loaded before this row's sums
// are taken.
template <int TPR, int GROUPS, int VPT, int CLUSTER, bool ODD, bool FUSED>
__global__ void __launch_bounds__(TPR* GROUPS, 512 / (TPR * GROUPS)) norm_backward_kernel(BackwardArgs a, float* partial,
                                                                                        int* err) {
  constexpr int kWarps = TPR / 32, kSpan = TPR * VPT;  // words of a block's part of a row
  static_assert(CLUSTER == 1 || GROUPS == 1, "");
  __shared__ float2 sums[2][GROUPS][kWarps];
  __shared__ float2 peers[2][CLUSTER];
  __shared__ __align__(8) uint64_t arrived[2];
  __shared__ float columns[GROUPS > 1 ? 2 * 4 * kSpan : 1];
  const int tid = threadIdx.x % TPR, group = threadIdx.x / TPR, lane = tid & 31, warp = tid >> 5;
  const int rank = CLUSTER > 1 ? static_cast<int>(ptx::cluster_rank()) : 0;
  const int64_t step = static_cast<int64_t>(gridDim.x / CLUSTER) * GROUPS;
  const int64_t opening = static_cast<int64_t>(blockIdx.x / CLUSTER) * GROUPS + group;
  const float n = static_cast<float>(a.cols);
  if (CLUSTER > 1) {
    if (threadIdx.x == 0) {
      ptx::mbar_init(ptx::smem_u32(&arrived[0]), 1);
      ptx::mbar_init(ptx::smem_u32(&arrived[1]), 1);
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    ptx::cluster_sync_all();
  }
  bool live = true;  // false once a wait gave up: later ones are skipped

  float dw[VPT][4], db[VPT][4];
#pragma unroll
  for (int k = 0; k < VPT; ++k)
#pragma unroll
    for (int j = 0; j < 4; ++j) dw[k][j] = db[k][j] = 0.0f;
  float4 dy[VPT], t[VPT];
  float mean = 0.0f, rstd = 0.0f;
  auto fetch = [&](int64_t row) {
    if (row >= a.rows) return;
    const Words<ODD> words(row, a.cols, a.rows);
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      const int word = rank * kSpan + tid + k * TPR;
      if (words.holds(word)) {
        dy[k] = words.load(a.dy, word);
        t[k] = words.load(a.total, word);
      }
    }
    mean = __ldg(a.mean + row);
    rstd = __ldg(a.rstd + row);
  };
  fetch(opening);
  const philox::RoundKeys rk = philox::round_keys(a.drop.key);
  const uint64_t place = FUSED ? dropout_start(a.drop) : 0;
  unsigned turn = 0;
  for (int64_t row = opening; row < a.rows; row += step, ++turn) {
    const Words<ODD> words(row, a.cols, a.rows);
    float g[VPT][4], hat[VPT][4];
    const float r = rstd;
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      const int word = rank * kSpan + tid + k * TPR;
      const bool in = words.holds(word);
      float4 w = make_float4(1.0f, 1.0f, 1.0f, 1.0f);
      if (a.weight && in) w = words.column(a.weight, word);
      const float y4[4] = {dy[k].x, dy[k].y, dy[k].z, dy[k].w}, t4[4] = {t[k].x, t[k].y, t[k].z, t[k].w};
      const float w4[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool ok = in && words.valid(word, j);
        const float d = ok ? y4[j] : 0.0f;
        hat[k][j] = ok ? (t4[j] - mean) * r : 0.0f;
        g[k][j] = d * w4[j];
        s1 += g[k][j];
        s2 = fmaf(g[k][j], hat[k][j], s2);
        dw[k][j] = fmaf(d, hat[k][j], dw[k][j]);
        db[k][j] += d;
      }
    }
    fetch(row + step);
    float4 extra[FUSED ? VPT : 1];
    if (FUSED && a.dtotal) {
#pragma unroll
      for (int k = 0; k < VPT; ++k) {
        const int word = rank * kSpan + tid + k * TPR;
        if (words.holds(word)) extra[FUSED ? k : 0] = words.load(a.dtotal, word);
      }
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
      s1 += __shfl_xor_sync(0xffffffffu, s1, off);
      s2 += __shfl_xor_sync(0xffffffffu, s2, off);
    }
    if (kWarps > 1) {
      if (lane == 0) sums[turn & 1][group][warp] = make_float2(s1, s2);
      asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "r"(TPR) : "memory");
      s1 = s2 = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float2 v = sums[turn & 1][group][w];
        s1 += v.x;
        s2 += v.y;
      }
    }
    if (CLUSTER > 1) {
      // this block's sums go to every block of the cluster, its own too; the slots of a parity
      // are read (before the block's next barrier) ahead of the row after next's sums
      const uint32_t bar = ptx::smem_u32(&arrived[turn & 1]);
      if (threadIdx.x == 0) ptx::mbar_expect_tx(bar, CLUSTER * 8);
      if (threadIdx.x < CLUSTER) {
        const uint32_t peer = threadIdx.x;
        const uint32_t slot = ptx::map_rank(ptx::smem_u32(&peers[turn & 1][rank]), peer);
        const uint32_t its = ptx::map_rank(bar, peer);
        asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v2.b32 [%0], {%1, %2}, [%3];" ::"r"(slot),
                     "r"(__float_as_uint(s1)), "r"(__float_as_uint(s2)), "r"(its)
                     : "memory");
      }
      if (live) live = ptx::wait_or_give_up(bar, (turn >> 1) & 1, err, 0x601);
      s1 = s2 = 0.0f;
#pragma unroll
      for (int c = 0; c < CLUSTER; ++c) {
        const float2 v = peers[turn & 1][c];
        s1 += v.x;
        s2 += v.y;
      }
    }
    const float c1 = __fdiv_rn(s1, n), c2 = __fdiv_rn(s2, n);
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      const int word = rank * kSpan + tid + k * TPR;
      if (!words.holds(word)) continue;
      float4 d = make_float4(r * (g[k][0] - c1 - hat[k][0] * c2), r * (g[k][1] - c1 - hat[k][1] * c2),
                             r * (g[k][2] - c1 - hat[k][2] * c2), r * (g[k][3] - c1 - hat[k][3] * c2));
      if (FUSED && a.dtotal) {
        const float4 e = extra[FUSED ? k : 0];
        d = make_float4(d.x + e.x, d.y + e.y, d.z + e.z, d.w + e.w);
      }
      words.store(a.dresidual, word, d);
      if (FUSED && a.dx)
        words.store(a.dx, word,
                    dropped4(d, place + static_cast<uint64_t>(words.at) + 4 * static_cast<uint64_t>(word), rk,
                             a.drop.threshold, a.drop.scale));
    }
  }
  dependents_may_launch();
  if (CLUSTER > 1) ptx::cluster_sync_all();  // no block leaves while a peer may still send to it
  if (!partial) return;

  const int64_t at = static_cast<int64_t>(blockIdx.x / CLUSTER) * 2 * a.cols;
  if (GROUPS == 1) {
    // a group without rows has the phase that its rows would have
    const Words<ODD> words(opening, a.cols, a.rows);
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      const int word = rank * kSpan + tid + k * TPR;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int c = 4 * word + j - words.phase;
        if (c >= 0 && c < words.cols) {
          partial[at + c] = dw[k][j];
          partial[at + a.cols + c] = db[k][j];
        }
      }
    }
  } else {
    for (int i = threadIdx.x; i < 2 * 4 * kSpan; i += TPR * GROUPS) columns[i] = 0.0f;
    for (int turn_of = 0; turn_of < GROUPS; ++turn_of) {
      __syncthreads();
      if (group != turn_of) continue;
      const Words<ODD> words(opening, a.cols, a.rows);
#pragma unroll
      for (int k = 0; k < VPT; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int c = 4 * (tid + k * TPR) + j - words.phase;
          if (c >= 0 && c < words.cols) {
            columns[c] += dw[k][j];
            columns[4 * kSpan + c] += db[k][j];
          }
        }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < static_cast<int>(a.cols); c += TPR * GROUPS) {
      partial[at + c] = columns[c];
      partial[at + a.cols + c] = columns[4 * kSpan + c];
    }
  }
}

// Adds the blocks' column sums: a block to 32 columns, a warp to every 32nd of the partial
// rows, then the warps in order.
__global__ void __launch_bounds__(1024)
norm_join_kernel(const float* __restrict__ partial, int splits, int64_t cols, float* dweight, float* dbias) {
  __shared__ float2 sums[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + lane;
  wait_for_prior_grid();
  float2 s = make_float2(0.0f, 0.0f);
  if (c < cols) {
#pragma unroll 8
    for (int i = warp; i < splits; i += 32) {
      s.x += __ldcg(partial + 2 * i * cols + c);
      s.y += __ldcg(partial + (2 * i + 1) * cols + c);
    }
  }
  sums[warp][lane] = s;
  __syncthreads();
  s = sums[lane][warp];
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    s.x += __shfl_xor_sync(0xffffffffu, s.x, off);
    s.y += __shfl_xor_sync(0xffffffffu, s.y, off);
  }
  const int64_t column = static_cast<int64_t>(blockIdx.x) * 32 + warp;
  if (lane == 0 && column < cols) {
    dweight[column] = s.x;
    dbias[column] = s.y;
  }
}

// ------------------------------------------------------------------------- launches
bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Words that a row can touch.
int64_t words_of(int64_t cols) { return cols % 4 ? (cols + 6) / 4 : cols / 4; }

template <int THREADS, int VPT>
void launch_forward(cudaStream_t s, const ForwardArgs& a, bool odd, bool fused) {
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(a.rows, 1 << 30));
  if (odd) {
    if (fused) norm_forward_kernel<THREADS, VPT, true, true><<<grid, THREADS, 0, s>>>(a);
    else norm_forward_kernel<THREADS, VPT, true, false><<<grid, THREADS, 0, s>>>(a);
  } else {
    if (fused) norm_forward_kernel<THREADS, VPT, false, true><<<grid, THREADS, 0, s>>>(a);
    else norm_forward_kernel<THREADS, VPT, false, false><<<grid, THREADS, 0, s>>>(a);
  }
}

// Blocks (or clusters) that the backward kernel runs as: what the machine holds at a time, no
// more than there are rows for, and a multiple of 4 groups (rows a group apart keep the phase).
int64_t backward_blocks(int64_t rows, int groups, int resident) {
  const int64_t want = std::min<int64_t>(ceil_div(rows, groups), resident);
  return ceil_div(want, 4) * 4;
}

struct BackwardPlan {
  int threads, groups, cluster;  // threads of a block, rows of a block at a time, blocks of a row; threads 0: none
  int64_t blocks;                // or clusters: partial rows
};

BackwardPlan backward_plan(int64_t rows, int64_t cols) {
  const int64_t words = words_of(cols);
  if (words > 8 * 2048) return {0, 0, 0, 0};
  const int tpr = words <= 128 ? 32 : words <= 256 ? 64 : words <= 512 ? 128 : words <= 1024 ? 256 : 512;
  const int cluster = words <= 2048 ? 1 : words <= 4096 ? 2 : words <= 8192 ? 4 : 8;
  const int groups = tpr < 256 ? 256 / tpr : 1, threads = tpr * groups;
  return {threads, groups, cluster, backward_blocks(rows, groups, 512 / threads * sm_count() / cluster)};
}

template <int TPR, int GROUPS, int VPT, int CLUSTER, bool ODD, bool FUSED>
void launch_backward(cudaStream_t s, const BackwardArgs& a, float* partial, const BackwardPlan& plan) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(plan.blocks * CLUSTER));
  cfg.blockDim = dim3(TPR * GROUPS);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {CLUSTER, 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = CLUSTER > 1 ? 1 : 0;
  cudaLaunchKernelEx(&cfg, norm_backward_kernel<TPR, GROUPS, VPT, CLUSTER, ODD, FUSED>, a, partial, device_error_word());
}

template <int TPR, int GROUPS, int VPT, int CLUSTER>
void launch_backward(cudaStream_t s, const BackwardArgs& a, float* partial, const BackwardPlan& plan, bool odd,
                     bool fused) {
  if (odd) {
    if (fused) launch_backward<TPR, GROUPS, VPT, CLUSTER, true, true>(s, a, partial, plan);
    else launch_backward<TPR, GROUPS, VPT, CLUSTER, true, false>(s, a, partial, plan);
  } else {
    if (fused) launch_backward<TPR, GROUPS, VPT, CLUSTER, false, true>(s, a, partial, plan);
    else launch_backward<TPR, GROUPS, VPT, CLUSTER, false, false>(s, a, partial, plan);
  }
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
  TimedLaunch timer("norm_forward", s);
  const int64_t words = words_of(cols);
  if (words > 8192 || !aligned(input) || !aligned(residual) || !aligned(output) || !aligned(a.total)) {
    const int grid = static_cast<int>(std::min<int64_t>(rows, 8 * sm_count()));
    norm_forward_any_kernel<<<grid, kThreads, 0, s>>>(a);
    return launch_status("layer norm forward");
  }
  const bool odd = cols % 4 != 0 || !aligned(weight) || !aligned(bias), fused = a.total != nullptr;
  if (words <= 32) launch_forward<32, 1>(s, a, odd, fused);
  else if (words <= 64) launch_forward<32, 2>(s, a, odd, fused);
  else if (words <= 128) launch_forward<32, 4>(s, a, odd, fused);
  else if (words <= 256) launch_forward<32, 8>(s, a, odd, fused);
  else if (words <= 512) launch_forward<32, 16>(s, a, odd, fused);
  else if (words <= 1024) launch_forward<64, 16>(s, a, odd, fused);
  else if (words <= 2048) launch_forward<128, 16>(s, a, odd, fused);
  else if (words <= 4096) launch_forward<256, 16>(s, a, odd, fused);
  else launch_forward<512, 16>(s, a, odd, fused);
  return launch_status("layer norm forward");
}

extern "C" size_t tcx_sm100_layernorm_backward_workspace_bytes(int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0) return 0;
  // either path's partial column sums
  const int64_t splits = std::max(splits_of(rows), backward_plan(rows, cols).blocks);
  return static_cast<size_t>(splits) * 2 * cols * sizeof(float);
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
  float* partial = dweight ? static_cast<float*>(workspace) : nullptr;
  const BackwardPlan plan = backward_plan(rows, cols);
  if (plan.threads && aligned(dy) && aligned(total) && aligned(dtotal) && aligned(dresidual) && aligned(a.dx)) {
    const bool odd = cols % 4 != 0 || !aligned(weight), fused = dtotal || a.dx;
    const int64_t words = words_of(cols);
    if (words <= 32) launch_backward<32, 8, 1, 1>(s, a, partial, plan, odd, fused);
    else if (words <= 64) launch_backward<32, 8, 2, 1>(s, a, partial, plan, odd, fused);
    else if (words <= 128) launch_backward<32, 8, 4, 1>(s, a, partial, plan, odd, fused);
    else if (words <= 256) launch_backward<64, 4, 4, 1>(s, a, partial, plan, odd, fused);
    else if (words <= 512) launch_backward<128, 2, 4, 1>(s, a, partial, plan, odd, fused);
    else if (words <= 1024) launch_backward<256, 1, 4, 1>(s, a, partial, plan, odd, fused);
    else if (words <= 2048) launch_backward<512, 1, 4, 1>(s, a, partial, plan, odd, fused);
    else if (words <= 4096) launch_backward<512, 1, 4, 2>(s, a, partial, plan, odd, fused);
    else if (words <= 8192) launch_backward<512, 1, 4, 4>(s, a, partial, plan, odd, fused);
    else launch_backward<512, 1, 4, 8>(s, a, partial, plan, odd, fused);
    if (partial)
      launch_after(norm_join_kernel, dim3(static_cast<unsigned>(ceil_div(cols, 32))), dim3(1024), s, 0, partial,
                   static_cast<int>(plan.blocks), cols, dweight, dbias);
    return launch_status("layer norm backward");
  }
  const int grid = static_cast<int>(std::min<int64_t>(rows, 8 * sm_count()));
  norm_backward_any_kernel<<<grid, kThreads, 0, s>>>(a);
  if (dweight) {
    const int64_t splits = splits_of(rows);
    const unsigned blocks = static_cast<unsigned>(ceil_div(cols, kThreads));
    norm_columns_kernel<<<dim3(blocks, static_cast<unsigned>(splits)), kThreads, 0, s>>>(a, partial,
                                                                                         ceil_div(rows, splits));
    norm_columns_join_kernel<<<blocks, kThreads, 0, s>>>(partial, splits, cols, dweight, dbias);
  }
  return launch_status("layer norm backward");
}
