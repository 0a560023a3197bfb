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
// exactly, and a row whose level is far above its spread loses nothing in the sum. (With a
// dropout in front f is the residual's first element.) All sums are float32.
//
// Bound by memory: 8 bytes an element forward and 12 backward, 16 and 20 with the dropout and
// the residual. Measured on one B200, calls back to back on changing inputs (those bytes over the
// call's time, against a copy's 6.55 TB/s): [16384, 4096] forward 90 us (0.91), with dropout and
// residual 182 us (0.90), backward 131 us (0.94; its first kernel 120 us), with dropout and residual
// 229 us (0.89); [16383, 4095] with both forward 214 us (0.76), backward plain 159 us (0.77);
// [2048, 32768] backward 167 us (0.74), forward 118 us (0.69), with both 243 us (0.67); [65536, 256]
// backward 39 us (0.78). Where a comment below gives two figures for a choice, they were taken side
// by side when it was made.
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>

#include "common.cuh"
#include "dropout.cuh"
#include "ptx.cuh"
#include "rowmath.cuh"

namespace tcx {
namespace {

using rowmath::Block;

// ------------------------------------------------------------------------ any row
// For buffers that are not 16-byte aligned and rows longer than the kernels below hold (32768
// forward, 65536 backward): an element to a thread, a row's block reading it again for each
// of its sums and once more for its outputs, and the columns' sums in a pass of their own. One
// element off the alignment [16384, 4096] takes 155 us forward and 516 with dropout and residual,
// 301 and 636 backward; [500000, 64], a block to each short row, 1634 and 1575 us; [2048, 70001],
// aligned or not, 638 and 1138.
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

// Rows of a column that are added one after the other before their sum joins the others': a
// float32 that takes all rows in turn is off by as many roundings (a constant gradient of 0.1
// over a million rows, 64 splits: by 1.5e-4 of the sum).
constexpr int kSpan = 16;

// Partial column sums of rows [split * per, (split + 1) * per): partial[2 split] holds the
// weight's, partial[2 split + 1] the bias's.
__global__ void __launch_bounds__(kThreads) norm_columns_kernel(BackwardArgs a, float* partial, int64_t per) {
  const int64_t c = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (c >= a.cols) return;
  const int64_t r0 = blockIdx.y * per, r1 = min(r0 + per, a.rows);
  float dw = 0.0f, db = 0.0f;
  for (int64_t from = r0; from < r1; from += kSpan) {
    const int64_t to = min(from + kSpan, r1);
    float span_w = 0.0f, span_b = 0.0f;
    for (int64_t r = from; r < to; ++r) {
      const float dy = a.dy[r * a.cols + c];
      span_w += dy * ((a.total[r * a.cols + c] - a.mean[r]) * a.rstd[r]);
      span_b += dy;
    }
    dw += span_w;
    db += span_b;
  }
  partial[(2 * blockIdx.y) * a.cols + c] = dw;
  partial[(2 * blockIdx.y + 1) * a.cols + c] = db;
}

// ------------------------------------------------------------------ rows in registers
// A row as its whole 16-byte words, at places that are multiples of 4 of the whole tensor
// whatever the row length, and where rows start elsewhere (ODD) up to 3 loose elements before
// and after them: a lane of the row's first warp to each. So all but a few accesses are 128 bits
// wide, and a word of the tensor is a block of the random stream.
template <bool ODD>
struct Words {
  int64_t at;             // of the first whole word in the tensor: a multiple of 4, words or none
  int head, words, tail;  // loose elements before the whole words, those, and loose elements after

  __device__ Words(int64_t row, int64_t n) {
    const int64_t first = row * n;
    const int cols = static_cast<int>(n);
    const int ahead = ODD ? static_cast<int>(-first & 3) : 0;
    at = first + ahead;
    head = min(ahead, cols);
    words = (cols - head) >> 2;
    tail = ODD ? cols - head - 4 * words : 0;
  }
  __device__ bool holds(int word) const { return word < words; }
  __device__ __forceinline__ float4 load(const float* p, int word) const {
    return __ldcs(reinterpret_cast<const float4*>(p + at) + word);
  }
  __device__ __forceinline__ void store(float* p, int word, float4 v) const {
    __stcs(reinterpret_cast<float4*>(p + at) + word, v);
  }
  // A word's columns of a vector over the row.
  __device__ __forceinline__ float4 column(const float* p, int word) const {
    if (!ODD) return __ldg(reinterpret_cast<const float4*>(p) + word);
    const float* const q = p + head + 4 * word;
    return make_float4(__ldg(q), __ldg(q + 1), __ldg(q + 2), __ldg(q + 3));
  }
  __device__ bool loose(int lane) const { return ODD && lane < head + tail; }
  __device__ int loose_column(int lane) const { return lane < head ? lane : 4 * words + lane; }
};

// Place e of the stream is kept.
__device__ __forceinline__ bool kept_place(uint64_t e, const philox::RoundKeys& rk, uint32_t threshold) {
  return kept(word_of(philox::block_words(e >> 2, rk), static_cast<uint32_t>(e & 3)), threshold);
}

// Two sums over LANES lanes in one butterfly: the lower half ends with a's, the upper with b's.
template <int LANES>
__device__ __forceinline__ float lane_sums(float a, float b) {
  const bool upper = threadIdx.x & (LANES / 2);
  float s = (upper ? b : a) + __shfl_xor_sync(0xffffffffu, upper ? a : b, LANES / 2);
#pragma unroll
  for (int off = LANES / 4; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
  return s;
}

// Two sums over `warps` warps that share `smem` and the barrier, or over LANES lanes of one;
// every thread receives them.
template <int LANES = 32>
__device__ __forceinline__ float2 row_sums(float a, float b, float2* smem, int warps, int warp, int barrier) {
  const float s = lane_sums<LANES>(a, b);
  const int lane = threadIdx.x & 31;
  if (warps == 1)
    return make_float2(__shfl_sync(0xffffffffu, s, 0, LANES), __shfl_sync(0xffffffffu, s, LANES / 2, LANES));
  if ((lane & 15) == 0) (lane ? smem[warp].y : smem[warp].x) = s;
  asm volatile("bar.sync %0, %1;" ::"r"(barrier), "r"(32 * warps) : "memory");
  float2 sums = make_float2(0.0f, 0.0f);
#pragma unroll 4
  for (int w = 0; w < warps; ++w) {
    const float2 v = smem[w];
    sums.x += v.x;
    sums.y += v.y;
  }
  return sums;
}

// Kernels for a known number of warps to a row (WARPS), or any up to kMostWarps (0).
constexpr int kMostWarps = 16, kPairWarps = 10;
// Threads of a forward block at most, and of the blocks that an SM holds of them.
constexpr int most_threads(int warps) { return 32 * (warps == 1 ? 2 : warps ? warps : kMostWarps); }
constexpr int resident_threads(int vpt, bool fused) {
  return fused ? (vpt < 4 ? 1024 : vpt < 8 ? 768 : 512) : vpt < 4 ? 1536 : vpt < 8 ? 1024 : 768;
}
// What their registers are bounded by. Blocks of any number of warps as if they were as large as
// that: 64 registers for 8 words of one input, 80 for 16 (an SM holds 3 blocks of 8 warps instead
// of two: [4096, 16384] 110 -> 98 us), 96 for 8 of two ([9500, 6001] 207 -> 177; 80 are too few).
// Some kernels spill 4 to 36 bytes a thread for it. Fused short rows, with the registers not to
// (512 threads to an SM for 4 words, 768 for fewer): [200000, 100] 74 us against 62, [100000, 401]
// 160 against 150, [500000, 64] 105 against 94, [600000, 33] 107 against 103.
constexpr int bound_threads(int vpt, int warps, bool fused, int staged) {
  if (staged == 2) return 32 * kPairWarps;
  if (staged || warps) return most_threads(warps);
  return fused ? 640 : vpt == 8 ? 1024 : 768;
}
constexpr int bound_blocks(int vpt, int warps, bool fused, int staged) {
  if (staged) return staged;
  return warps ? resident_threads(vpt, fused) / most_threads(warps) : 1;
}

// One block to a row, VPT words to a thread, as many warps as the row needs. Each element is
// read once and written once; the statistics take two block reductions. STAGED: the 1 or 2 blocks
// that fit an SM take rows in turn, and the next row's words come into shared memory (cp.async; a
// thread copies and reads its own only) while this one is worked on. Two blocks of up to 10 warps
// and 96 registers ([7800, 8400] with dropout and residual: 217 us against 256 with one of 128,
// [3000, 20000] 102 against 131), one of more ([5500, 12000] 211 against 243 with the registers
// of two).
// Rows of one warp or less (LANES lanes) share a block: with a block and a whole warp to each,
// the starts of the blocks took [500000, 64] to 264 us against 56, [125000, 256] 72 against 47,
// [600000, 33] with dropout and residual 459 against 117.
template <int VPT, int WARPS, int LANES, bool ODD, bool FUSED, int STAGED>
__global__ void __launch_bounds__(bound_threads(VPT, WARPS, FUSED, STAGED), bound_blocks(VPT, WARPS, FUSED, STAGED))
norm_forward_kernel(ForwardArgs a) {
  static_assert(LANES == 32 || (WARPS == 1 && LANES >= 8), "a lane to each loose element");
  constexpr bool SHARED = WARPS == 1;
  extern __shared__ __align__(16) float4 stage[];
  __shared__ float2 smem[2][kMostWarps];
  const int warps = WARPS ? WARPS : blockDim.x >> 5, warp = SHARED ? 0 : threadIdx.x >> 5;
  const int lane = threadIdx.x & (LANES - 1), mine = warp * 32 * VPT + lane;  // its first word, of a warp's 32 VPT
  const int group = SHARED ? threadIdx.x / LANES : 0, groups = SHARED ? blockDim.x / LANES : 1;
  const float n = static_cast<float>(a.cols);
  const philox::RoundKeys rk = philox::round_keys(a.drop.key);
  float4* const place = stage + warp * (FUSED ? 2 : 1) * 32 * VPT + lane;
  auto copy = [&](int64_t row) {
    if (row < a.rows) {
      const Words<ODD> words(row, a.cols);
#pragma unroll
      for (int k = 0; k < VPT; ++k) {
        if (words.holds(mine + 32 * k)) {
          const int64_t i = words.at + 4 * static_cast<int64_t>(mine) + 128 * k;
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(ptx::smem_u32(place + 32 * k)), "l"(a.x + i)
                       : "memory");
          if (FUSED && a.residual)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(ptx::smem_u32(place + 32 * (VPT + k))),
                         "l"(a.residual + i)
                         : "memory");
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  if (STAGED) copy(blockIdx.x);
  for (int64_t first_row = static_cast<int64_t>(blockIdx.x) * groups; first_row < a.rows;
       first_row += static_cast<int64_t>(gridDim.x) * groups) {
    // past the last row, an empty one
    const bool live = !SHARED || first_row + group < a.rows;
    const int64_t row = live ? first_row + group : 0;
    const Words<ODD> words(row, live ? a.cols : 0);
    float v[VPT][4];
    if (STAGED) asm volatile("cp.async.wait_group 0;" ::: "memory");
    const int64_t first = row * a.cols;
    float level;  // what the sums are taken about: the row's first element, or near it
    if (FUSED) {
      level = a.residual ? __ldg(a.residual + first) : 0.0f;
      if (!a.drop.threshold) level += __ldg(a.x + first);
    } else {
      level = __ldg(a.x + first);
    }
    float4 res[FUSED ? VPT : 1];
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      const int word = mine + LANES * k;
      float4 t = make_float4(level, level, level, level);
      if (words.holds(word)) t = STAGED ? place[32 * k] : words.load(a.x, word);
      v[k][0] = t.x, v[k][1] = t.y, v[k][2] = t.z, v[k][3] = t.w;
    }
    if (FUSED && a.residual) {
#pragma unroll
      for (int k = 0; k < VPT; ++k)
        if (words.holds(mine + LANES * k))
          res[FUSED ? k : 0] = STAGED ? place[32 * (VPT + k)] : words.load(a.residual, mine + LANES * k);
    }
    if (STAGED) copy(row + gridDim.x);
    // a loose element, with `level` for none
    const bool loose = ODD && warp == 0 && words.loose(lane);
    const int column = ODD ? words.loose_column(lane) : 0;
    float one = level;
    if (ODD && loose) one = __ldcs(a.x + first + column);
    if (FUSED) {
      const uint64_t start = a.drop.threshold ? dropout_start(a.drop) : 0;
      if (a.drop.threshold) {
        // the mask while the loads are on their way: 4 bits to a word
        const uint64_t place_0 = start + static_cast<uint64_t>(words.at) + 4 * static_cast<uint64_t>(mine);
        uint32_t mask[(VPT + 7) / 8];
#pragma unroll
        for (int k = 0; k < VPT; k += 8)
          mask[k / 8] =
              kept_words<(VPT < 8 ? VPT : 8), LANES>(place_0 + 4 * LANES * static_cast<uint64_t>(k), LANES, rk,
                                                     a.drop.threshold);
#pragma unroll
        for (int k = 0; k < VPT; ++k)
#pragma unroll
          for (int j = 0; j < 4; ++j) v[k][j] = dropped(v[k][j], mask[k / 8] >> (4 * (k % 8) + j) & 1, a.drop.scale);
      }
#pragma unroll
      for (int k = 0; k < VPT; ++k) {
        const int word = mine + LANES * k;
        if (words.holds(word)) {
          if (a.residual) {
            const float4 r = res[FUSED ? k : 0];
            v[k][0] = __fadd_rn(r.x, v[k][0]), v[k][1] = __fadd_rn(r.y, v[k][1]);
            v[k][2] = __fadd_rn(r.z, v[k][2]), v[k][3] = __fadd_rn(r.w, v[k][3]);
          }
          words.store(a.total, word, make_float4(v[k][0], v[k][1], v[k][2], v[k][3]));
        } else {
          v[k][0] = v[k][1] = v[k][2] = v[k][3] = level;
        }
      }
      if (ODD && loose) {
        if (a.drop.threshold)
          one = dropped(one, kept_place(start + static_cast<uint64_t>(first + column), rk, a.drop.threshold),
                        a.drop.scale);
        if (a.residual) one = __fadd_rn(__ldcs(a.residual + first + column), one);
        a.total[first + column] = one;
      }
    }
    float s = ODD ? one - level : 0.0f;
#pragma unroll
    for (int k = 0; k < VPT; ++k)
#pragma unroll
      for (int j = 0; j < 4; ++j) s += v[k][j] - level;
    const float m1 = level + __fdiv_rn(row_sums<LANES>(s, 0.0f, smem[0], warps, warp, 0).x, n);
    one = ODD && loose ? one - m1 : 0.0f;
    float s1 = one, s2 = one * one;
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      if (words.holds(mine + LANES * k)) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v[k][j] -= m1;
          s1 += v[k][j];
          s2 = fmaf(v[k][j], v[k][j], s2);
        }
      }
    }
    const float2 r = row_sums<LANES>(s1, s2, smem[1], warps, warp, 0);
    const float shift = __fdiv_rn(r.x, n);
    float var = __fdiv_rn(r.y, n) - shift * shift;
    if (var < 0.0f) var = 0.0f;  // rounding; a NaN stays one
    const float rstd = __fdiv_rn(1.0f, __fsqrt_rn(var + a.eps));
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      const int word = mine + LANES * k;
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
    if (ODD && loose) {
      float y = (one - shift) * rstd;
      if (a.weight) y *= __ldg(a.weight + column);
      if (a.bias) y += __ldg(a.bias + column);
      a.y[first + column] = y;
    }
    if (SHARED ? live && lane == 0 : threadIdx.x == 0) {
      a.mean[row] = m1 + shift;
      a.rstd[row] = rstd;
    }
  }
}

// The gradient. Its floor is one pass over dy and total, so a row stays with its block between
// its sums and its gradient, and the columns' sums are taken on the way: [16384, 4096] took
// 484 us with passes of their own for those.
//
// Some warps of a block (of each of CLUSTER blocks) to a row, VPT words to a thread, and several
// rows to a block at a time where they are short, a group of warps to each. A group's rows are
// a multiple of 4 apart, so that they all start at the same place of a word and a thread's
// columns are the same in each: the weight's and the bias's gradients add up in its registers
// over the group's rows (at most 128: see kMostRows), the groups' in shared memory, and the blocks'
// in a second kernel, each in a fixed order. A chain of additions that long is what the sums' error
// is: 1.6e-7 (2-norm) with 55 rows at [16384, 4096], where torch's sum over the rows has 1.4e-7, and
// half of torch's at [65536, 256]. Joining spans of 16 rows on the way costs more than it gives:
// through the workspace 146 us against 138 at [16384, 4096], through tensor memory 149.
//
// dy and total come through a ring of places in shared memory (cp.async; a thread copies and
// reads its own words only, so that needs no barrier): a place is copied into again as soon as
// its row is in registers, while that row's sums cross the block. Where a block has several
// rows, dtotal has two places of its own, in use until the row's gradient is stored, and the
// ring one less ([8191, 1001]: 60 -> 50 us); a longer row's is loaded when its turn comes
// ([16384, 4096]: 216 us against 250). The weight lies beside the places where its words are
// not aligned or the block's rows share them; else it is read through the first-level cache
// ([8192, 8192]: 157 us against 169). 16 warps of 128 registers and three rows' places to an SM:
// two places, and 24 warps of 85 registers, took 140 us for [16384, 4096] against 134.
//
// Rows of more than 4096 take up to 16 warps of one block, one to an SM ([8192, 8192]: 132 us
// against 157 as two blocks of 8 warps); longer ones go to a cluster of blocks of 8: its blocks'
// sums cross by st.async, and there are as many clusters as the device holds at a time (33 of 8
// blocks: a few more and their rows came in a second round, 245 us against 154 for [2048,
// 32768]; 4 blocks of 16 warps took 179).

// Warps to an SM: 128 registers a thread, or 85 where it holds one word of each array.
// Odd rows with dropout or dtotal spill 32 to 68 bytes a thread at that, with more registers an SM
// would hold half the warps.
constexpr int warps_per_sm(int vpt) { return vpt == 1 ? 24 : 16; }

template <int VPT, int WARPS, bool ODD, bool FUSED>
struct Places {
  static constexpr bool kExtra = FUSED && WARPS, kWeight = ODD || WARPS;
  static constexpr int kRing = kExtra ? 2 : 3;
  static constexpr int kWarp = 32 * VPT * (kRing * 2 + (kExtra ? 2 : 0) + (kWeight ? 1 : 0));  // words of a warp
  // with several rows to a block their column sums take the rows' place in the end
  static constexpr int bytes(int threads) { return kWarp * (threads / 32) * 16; }
};

// WARPS: warps of a row, with 8 / WARPS rows to a block (groups); 0: any number, one row to a
// block; 1 with fewer LANES than 32: several rows to a warp ([500000, 64]: 71 us
// against 95 with a warp to each, with dropout and residual 118 against 263).
template <int VPT, int WARPS, int LANES, int CLUSTER, bool ODD, bool FUSED>
__global__ void __launch_bounds__(WARPS ? 256 : 512, WARPS ? warps_per_sm(VPT) / 8 : 1)
norm_backward_kernel(BackwardArgs a, float* partial, int* err) {
  static_assert(CLUSTER == 1 || WARPS == 0, "");
  static_assert(LANES == 32 || (WARPS == 1 && LANES >= 8), "a lane to each loose element");
  constexpr bool MULTI = WARPS != 0, SHARED = LANES < 32;
  const int warps = MULTI ? WARPS : blockDim.x >> 5;
  extern __shared__ __align__(16) float4 stage[];
  __shared__ float2 sums[2][kMostWarps];
  __shared__ float2 peers[2][CLUSTER];
  __shared__ __align__(8) uint64_t arrived[2];
  const int part = warps * 32 * VPT;  // words of a block's part of a row
  constexpr int kGroup = LANES * (MULTI ? WARPS : 1), groups = MULTI ? 256 / kGroup : 1;
  const int group = MULTI ? threadIdx.x / kGroup : 0;
  const int lane = threadIdx.x & (LANES - 1), warp = SHARED ? 0 : (threadIdx.x >> 5) - group * warps;
  const int rank = CLUSTER > 1 ? static_cast<int>(ptx::cluster_rank()) : 0;
  const int first_word = rank * part + warp * 32 * VPT + lane;  // a warp's words are side by side
  const int64_t step = static_cast<int64_t>(gridDim.x / CLUSTER) * groups;
  const int64_t opening = static_cast<int64_t>(blockIdx.x / CLUSTER) * groups + group;
  const float share = 1.0f / static_cast<float>(a.cols);
  if (CLUSTER > 1) {
    if (threadIdx.x == 0) {
      ptx::mbar_init(ptx::smem_u32(&arrived[0]), 1);
      ptx::mbar_init(ptx::smem_u32(&arrived[1]), 1);
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    ptx::cluster_sync_all();
  }
  bool live = true;  // false once a wait gave up: later ones are skipped

  using P = Places<VPT, WARPS, ODD, FUSED>;
  constexpr int kRing = P::kRing;
  float4* const mine = stage + (threadIdx.x >> 5) * P::kWarp + (threadIdx.x & 31);  // this thread's first place
  float4* const mine_extra = mine + kRing * 2 * VPT * 32;             // of dtotal
  float4* const weight = mine + (kRing * 2 + (P::kExtra ? 2 : 0)) * VPT * 32;
  const Words<ODD> words(opening, a.cols);  // but for their places, those of all its rows
  const int ahead = static_cast<int>(words.at - opening * a.cols);
  const bool loose = rank == 0 && warp == 0 && words.loose(lane);
  const int column = ODD ? words.loose_column(lane) : 0;
  float loose_dw = 0.0f, loose_db = 0.0f, loose_w = 1.0f;
  if (ODD && loose && a.weight) loose_w = __ldg(a.weight + column);
  float dw[VPT][4], db[VPT][4];
#pragma unroll
  for (int k = 0; k < VPT; ++k) {
#pragma unroll
    for (int j = 0; j < 4; ++j) dw[k][j] = db[k][j] = 0.0f;
    if (P::kWeight)
      weight[32 * k] = a.weight && words.holds(first_word + LANES * k)
                           ? words.column(a.weight, first_word + LANES * k)
                           : make_float4(1.0f, 1.0f, 1.0f, 1.0f);
  }

  // Copies a row into a place: word k of dy and of total.
  auto copy = [&](int place, int64_t row) {
    if (row < a.rows) {
      float4* const to = mine + place * (2 * VPT * 32);
      const int64_t at = row * a.cols + words.head + 4 * static_cast<int64_t>(first_word);
#pragma unroll
      for (int k = 0; k < VPT; ++k) {
        if (words.holds(first_word + LANES * k)) {
          const int64_t i = at + 4 * LANES * k;
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(ptx::smem_u32(to + 32 * k)), "l"(a.dy + i)
                       : "memory");
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(ptx::smem_u32(to + 32 * (VPT + k))),
                       "l"(a.total + i)
                       : "memory");
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  auto copy_extra = [&](int place, int64_t row) {
    if (a.dtotal && row < a.rows) {
      const int64_t at = row * a.cols + words.head + 4 * static_cast<int64_t>(first_word);
#pragma unroll
      for (int k = 0; k < VPT; ++k)
        if (words.holds(first_word + LANES * k))
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                           ptx::smem_u32(mine_extra + (place * VPT + k) * 32)),
                       "l"(a.dtotal + at + 4 * LANES * k)
                       : "memory");
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  auto statistics = [&](int64_t row, float& m, float& r) {
    m = row < a.rows ? __ldg(a.mean + row) : 0.0f;
    r = row < a.rows ? __ldg(a.rstd + row) : 0.0f;
  };
  auto loose_of = [&](int64_t row, float& d, float& t) {
    if (ODD && loose && row < a.rows) {
      d = __ldcs(a.dy + row * a.cols + column);
      t = __ldcs(a.total + row * a.cols + column);
    }
  };

  const philox::RoundKeys rk = philox::round_keys(a.drop.key);
  const uint64_t from = FUSED ? dropout_start(a.drop) : 0;
#pragma unroll
  for (int k = 0; k < kRing; ++k) {
    copy(k, opening + k * step);
    if (P::kExtra) copy_extra(k, opening + k * step);
  }
  float mean, rstd, next_mean, next_rstd, loose_d = 0.0f, loose_t = 0.0f;
  statistics(opening, mean, rstd);
  loose_of(opening, loose_d, loose_t);
  unsigned turn = 0;
  int place = 0;
  for (int64_t row = opening; row - (SHARED ? group : 0) < a.rows; row += step, ++turn) {
    const bool present = !SHARED || row < a.rows;  // a warp's rows run on past the last one together
    const int64_t at = row * a.cols;
    statistics(row + step, next_mean, next_rstd);
    float4 extra[FUSED && !P::kExtra ? VPT : 1];
    if (FUSED && !P::kExtra && a.dtotal) {
#pragma unroll
      for (int k = 0; k < VPT; ++k)
        if (words.holds(first_word + LANES * k))
          extra[P::kExtra ? 0 : k] =
              __ldcs(reinterpret_cast<const float4*>(a.dtotal + at + words.head) + first_word + 32 * k);
    }
    asm volatile("cp.async.wait_group %0;" ::"n"(P::kExtra ? 3 : kRing - 1) : "memory");
    const float4* const here = mine + place * (2 * VPT * 32);
    float g[VPT][4], hat[VPT][4];
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      const int word = first_word + LANES * k;
      const bool in = present && words.holds(word);
      float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f), t = make_float4(mean, mean, mean, mean);
      float4 w = P::kWeight ? weight[32 * k] : make_float4(1.0f, 1.0f, 1.0f, 1.0f);
      if (in) {
        y = here[32 * k];
        t = here[32 * (VPT + k)];
        if (!P::kWeight && a.weight) w = words.column(a.weight, word);
      }
      const float y4[4] = {y.x, y.y, y.z, y.w}, t4[4] = {t.x, t.y, t.z, t.w}, w4[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        hat[k][j] = (t4[j] - mean) * rstd;
        g[k][j] = y4[j] * w4[j];
        s1 += g[k][j];
        s2 = fmaf(g[k][j], hat[k][j], s2);
        dw[k][j] = fmaf(y4[j], hat[k][j], dw[k][j]);
        db[k][j] += y4[j];
      }
    }
    float loose_g = 0.0f, loose_hat = 0.0f;
    if (ODD && loose && present) {
      loose_hat = (loose_t - mean) * rstd;
      loose_g = loose_d * loose_w;
      s1 += loose_g;
      s2 = fmaf(loose_g, loose_hat, s2);
      loose_dw = fmaf(loose_d, loose_hat, loose_dw);
      loose_db += loose_d;
      loose_of(row + step, loose_d, loose_t);
    }
    copy(place, row + kRing * step);
    uint32_t mask = 0;
    if (FUSED && a.dx)
      mask = kept_words<VPT, LANES>(from + static_cast<uint64_t>(at + ahead) + 4 * static_cast<uint64_t>(first_word),
                                    LANES, rk, a.drop.threshold);
    const float2 sums_all = row_sums<LANES>(s1, s2, sums[turn & 1] + group * warps, warps, warp, 1 + group);
    s1 = sums_all.x, s2 = sums_all.y;
    if (CLUSTER > 1) {
      // This block's sums go to every block of the cluster, its own too. A peer that sends
      // those of the row after next has this block's of the next row, which are sent when all
      // of its threads have read this row's slots.
      const uint32_t bar = ptx::smem_u32(&arrived[turn & 1]);
      if (threadIdx.x == 0) ptx::mbar_expect_tx(bar, CLUSTER * 8);
      if (threadIdx.x < CLUSTER) {
        const uint32_t slot = ptx::map_rank(ptx::smem_u32(&peers[turn & 1][rank]), threadIdx.x);
        const uint32_t its = ptx::map_rank(bar, threadIdx.x);
        asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v2.b32 [%0], {%1, %2}, [%3];" ::"r"(slot),
                     "r"(__float_as_uint(s1)), "r"(__float_as_uint(s2)), "r"(its)
                     : "memory");
      }
      if (live) live = ptx::wait_or_give_up(bar, turn >> 1 & 1, err, 0x601);
      s1 = s2 = 0.0f;
#pragma unroll
      for (int c = 0; c < CLUSTER; ++c) {
        const float2 v = peers[turn & 1][c];
        s1 += v.x;
        s2 += v.y;
      }
    }
    const float c1 = -rstd * (s1 * share), c2 = -rstd * (s2 * share);
    if (P::kExtra) asm volatile("cp.async.wait_group 3;" ::: "memory");
    float4* const out = reinterpret_cast<float4*>(a.dresidual + at + words.head) + first_word;
    float4* const out_x = FUSED && a.dx ? reinterpret_cast<float4*>(a.dx + at + words.head) + first_word : nullptr;
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      const int word = first_word + LANES * k;
      if (!present || !words.holds(word)) continue;
      float d[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) d[j] = fmaf(hat[k][j], c2, fmaf(g[k][j], rstd, c1));
      if (FUSED && a.dtotal) {
        const float4 e = P::kExtra ? mine_extra[(place * VPT + k) * 32] : extra[P::kExtra ? 0 : k];
        d[0] += e.x, d[1] += e.y, d[2] += e.z, d[3] += e.w;
      }
      __stcs(out + LANES * k, make_float4(d[0], d[1], d[2], d[3]));
      if (FUSED && a.dx) {
#pragma unroll
        for (int j = 0; j < 4; ++j) d[j] = dropped(d[j], mask >> (4 * k + j) & 1, a.drop.scale);
        __stcs(out_x + LANES * k, make_float4(d[0], d[1], d[2], d[3]));
      }
    }
    if (ODD && loose && present) {
      const int64_t i = at + column;
      float d = fmaf(loose_hat, c2, fmaf(loose_g, rstd, c1));
      if (FUSED && a.dtotal) d += __ldcs(a.dtotal + i);
      a.dresidual[i] = d;
      if (FUSED && a.dx)
        a.dx[i] = dropped(d, kept_place(from + static_cast<uint64_t>(i), rk, a.drop.threshold), a.drop.scale);
    }
    if (P::kExtra) copy_extra(place, row + kRing * step);
    place = place + 1 == kRing ? 0 : place + 1;
    mean = next_mean, rstd = next_rstd;
  }
  dependents_may_launch();
  if (CLUSTER > 1) ptx::cluster_sync_all();  // no block leaves while a peer may still send to it
  if (!partial) return;

  const int64_t at = static_cast<int64_t>(blockIdx.x / CLUSTER) * 2 * a.cols;
  if (!MULTI) {  // a block without rows leaves zeros
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      if (!words.holds(first_word + 32 * k)) continue;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t c = at + words.head + 4 * (first_word + 32 * k) + j;
        partial[c] = dw[k][j];
        partial[c + a.cols] = db[k][j];
      }
    }
    if (ODD && loose) {
      partial[at + column] = loose_dw;
      partial[at + a.cols + column] = loose_db;
    }
  } else {
    float* const columns = reinterpret_cast<float*>(stage);
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
    constexpr int kMostColumns = 4 * kGroup * VPT + 4;  // whole words, and fewer loose ones than a word
    static_assert(groups * 2 * kMostColumns * 4 <= P::kWarp * 8 * 16, "the rows' place");
    // 2 or 4 rows at a time add in turn, more lie side by side and add at one barrier: [8191, 1001]
    // with dropout and residual 48 us in turn and 52 otherwise, [1, 512] 11 and 9.
    if constexpr (groups <= 4) {
      for (int i = threadIdx.x; i < 2 * kMostColumns; i += blockDim.x) columns[i] = 0.0f;
      for (int whose = 0; whose < groups; ++whose) {
        __syncthreads();
        if (group != whose) continue;
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
          if (!words.holds(first_word + LANES * k)) continue;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int c = words.head + 4 * (first_word + LANES * k) + j;
            columns[c] += dw[k][j];
            columns[kMostColumns + c] += db[k][j];
          }
        }
        if (ODD && loose) {
          columns[column] += loose_dw;
          columns[kMostColumns + column] += loose_db;
        }
      }
      __syncthreads();
      for (int c = threadIdx.x; c < static_cast<int>(a.cols); c += blockDim.x) {
        partial[at + c] = columns[c];
        partial[at + a.cols + c] = columns[kMostColumns + c];
      }
    } else {
      float* const its = columns + group * 2 * kMostColumns;
#pragma unroll
      for (int k = 0; k < VPT; ++k) {
        if (!words.holds(first_word + LANES * k)) continue;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int c = words.head + 4 * (first_word + LANES * k) + j;
          its[c] = dw[k][j];
          its[kMostColumns + c] = db[k][j];
        }
      }
      if (ODD && loose) {
        its[column] = loose_dw;
        its[kMostColumns + column] = loose_db;
      }
      __syncthreads();
      const int cols = static_cast<int>(a.cols);
      for (int i = threadIdx.x; i < 2 * cols; i += blockDim.x) {
        const float* const sum = columns + (i < cols ? i : kMostColumns + i - cols);
        float t = 0.0f;
#pragma unroll
        for (int g = 0; g < groups; g += 4)
          t += (sum[g * 2 * kMostColumns] + sum[(g + 1) * 2 * kMostColumns]) +
               (sum[(g + 2) * 2 * kMostColumns] + sum[(g + 3) * 2 * kMostColumns]);
        partial[at + i] = t;
      }
    }
  }
}

// Adds the blocks' column sums: a block to 32 columns, a warp to every WARPS-th of the partial
// rows, then the warps four at a time. 32 warps for many partial rows, 8 for few. LONG: a warp
// adds 20 of its rows before their sum joins its own, for more than 640 (with that loop the
// kernel has 46 registers instead of 32: [4096, 8192], 148 partial rows, 76 us against 74).
constexpr int kTwenty = 20;
template <int WARPS, bool LONG>
__global__ void __launch_bounds__(32 * WARPS)
norm_join_kernel(const float* __restrict__ partial, int splits, int64_t cols, float* dweight, float* dbias) {
  __shared__ float2 sums[WARPS][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + lane;
  wait_for_prior_grid();
  float2 s = make_float2(0.0f, 0.0f);
  auto add = [&](float2& t, int i) {
    t.x += __ldcg(partial + 2 * static_cast<int64_t>(i) * cols + c);
    t.y += __ldcg(partial + (2 * static_cast<int64_t>(i) + 1) * cols + c);
  };
  if (c < cols) {
    if constexpr (LONG) {
      for (int from = warp; from < splits; from += kTwenty * WARPS) {
        const int to = min(splits, from + kTwenty * WARPS);
        float2 t = make_float2(0.0f, 0.0f);
#pragma unroll 5
        for (int i = from; i < to; i += WARPS) add(t, i);
        s.x += t.x;
        s.y += t.y;
      }
    } else {
#pragma unroll 5
      for (int i = warp; i < splits; i += WARPS) add(s, i);
    }
  }
  sums[warp][lane] = s;
  __syncthreads();
  if (warp < 2 && c < cols) {  // a warp to each gradient
    float t = 0.0f;
#pragma unroll
    for (int w = 0; w < WARPS; w += 4) {
      const float2 q0 = sums[w][lane], q1 = sums[w + 1][lane], q2 = sums[w + 2][lane], q3 = sums[w + 3][lane];
      t += warp ? (q0.y + q1.y) + (q2.y + q3.y) : (q0.x + q1.x) + (q2.x + q3.x);
    }
    (warp ? dbias : dweight)[c] = t;
  }
}

void join_columns(cudaStream_t s, const float* partial, int64_t splits, int64_t cols, float* dweight, float* dbias) {
  const dim3 grid(static_cast<unsigned>(ceil_div(cols, 32)));
  auto* kernel = splits > kTwenty * 32 ? norm_join_kernel<32, true>
                 : splits > 64         ? norm_join_kernel<32, false>
                                       : norm_join_kernel<8, false>;
  launch_after(kernel, grid, dim3(splits > 64 ? 1024 : 256), s, 0, partial, splits, cols, dweight, dbias);
}

// ------------------------------------------------------------------------- launches
bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Whole words of a row, at most.
int64_t words_of(int64_t cols) { return std::max<int64_t>(1, cols / 4); }

// Rows of one warp or less: blocks of 2 warps, or 1 where that leaves an SM without one.
template <int VPT, int WARPS, int LANES, bool FUSED>
void launch_forward(cudaStream_t s, const ForwardArgs& a, int warps, bool odd) {
  const int64_t all = ceil_div(a.rows * LANES, 32);
  if (WARPS == 1) warps = static_cast<int>(std::min<int64_t>(ceil_div(all, sm_count()), 2));
  const unsigned grid =
      static_cast<unsigned>(std::min<int64_t>(WARPS == 1 ? ceil_div(all, warps) : a.rows, 1 << 30));
  if (odd) norm_forward_kernel<VPT, WARPS, LANES, true, FUSED, 0><<<grid, 32 * warps, 0, s>>>(a);
  else norm_forward_kernel<VPT, WARPS, LANES, false, FUSED, 0><<<grid, 32 * warps, 0, s>>>(a);
}

template <int VPT, int BLOCKS, bool ODD, bool FUSED>
void launch_staged(cudaStream_t s, const ForwardArgs& a, int warps) {
  auto* kernel = norm_forward_kernel<VPT, 0, 32, ODD, FUSED, BLOCKS>;
  constexpr int kWarpBytes = (FUSED ? 2 : 1) * 32 * VPT * 16;
  static std::atomic<bool> attr_done[64];  // host threads may meet here
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !attr_done[dev].load(std::memory_order_relaxed)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (BLOCKS == 2 ? kPairWarps : kMostWarps) * kWarpBytes) != cudaSuccess)
      return;  // the call's error
    if (dev >= 0 && dev < 64) attr_done[dev].store(true, std::memory_order_relaxed);
  }
  const int64_t grid = std::min<int64_t>(a.rows, BLOCKS * sm_count());
  kernel<<<static_cast<unsigned>(grid), 32 * warps, warps * kWarpBytes, s>>>(a);
}

constexpr int kStagedWarps = 9;  // rows whose blocks an SM holds one or two of

template <int VPT, bool ODD, bool FUSED>
void launch_staged(cudaStream_t s, const ForwardArgs& a, int warps) {
  if (warps <= kPairWarps) launch_staged<VPT, 2, ODD, FUSED>(s, a, warps);
  else launch_staged<VPT, 1, ODD, FUSED>(s, a, warps);
}

template <int VPT, bool FUSED>
void launch_forward(cudaStream_t s, const ForwardArgs& a, int64_t words, bool odd) {
  const int warps = static_cast<int>(ceil_div(words, 32 * VPT));
  if (warps >= kStagedWarps && odd) return launch_staged<VPT, true, FUSED>(s, a, warps);
  if (warps >= kStagedWarps) return launch_staged<VPT, false, FUSED>(s, a, warps);
  if (warps == 1) return launch_forward<VPT, 1, 32, FUSED>(s, a, warps, odd);
  if constexpr (VPT < 16) {  // 513 to 1024 words are never 16 to a thread
    if (warps == 2) return launch_forward<VPT, 2, 32, FUSED>(s, a, warps, odd);
  }
  if (warps == 4) return launch_forward<VPT, 4, 32, FUSED>(s, a, warps, odd);
  launch_forward<VPT, 0, 32, FUSED>(s, a, warps, odd);
}

// 32 values to a thread, of each of two inputs where there are two. Where there are rows to
// fill the machine a dozen times, 64 of one input in half as many warps: rows of 257 to 384
// words, which leave one warp no block to wait for ([40000, 1100]: 66 us against 76; [50000,
// 800] 67 against 56), and rows of 7 warps and more, of which an SM then holds twice as many
// ([8192, 8191]: 121 us against 150; [8192, 8400] 111 against 184; [16384, 4096] 92 against 88).
// Fewer rows finish sooner with more warps to each ([148, 8192]: 12 us against 16).
template <bool FUSED>
void launch_forward(cudaStream_t s, const ForwardArgs& a, int64_t words, bool odd) {
  const bool many = !FUSED && (words > 1536 || (words > 256 && words <= 384)) &&
                    a.rows >= 12 * static_cast<int64_t>(sm_count());
  if (words <= 8) launch_forward<1, 1, 8, FUSED>(s, a, 1, odd);
  else if (words <= 16) launch_forward<2, 1, 8, FUSED>(s, a, 1, odd);
  else if (words <= 32) launch_forward<4, 1, 8, FUSED>(s, a, 1, odd);
  else if (words <= 64) launch_forward<4, 1, 16, FUSED>(s, a, 1, odd);
  else if (words <= 128) launch_forward<4, 1, 32, FUSED>(s, a, 1, odd);
  else if (words <= 4096 && !many) launch_forward<8, FUSED>(s, a, words, odd);
  else if constexpr (!FUSED) launch_forward<16, FUSED>(s, a, words, odd);
}

// Blocks (or clusters) that the backward kernel runs as: what the machine holds at a time, or as
// many times that as leave a group no more than 128 rows (but for the rounding below): a thread
// adds its columns over them one after the other, and each row is a rounding of the sum so far
// ([190000, 8192], a constant gradient: off by 1.9e-5 of the sum with 1284 rows to a block). It
// costs nothing where an SM holds several blocks ([800000, 1024] 1477 us against 1525 with one
// round, 1468 with at most 64 rows), the blocks' starts where it holds one ([100000, 8192] 1558
// against 1505, 1587 with 64; a block of [16384, 4096] has 55 rows). No more blocks than there
// are rows for; where rows start anywhere in a word, a multiple of 4 (the rows of a group are
// that far apart).
constexpr int64_t kMostRows = 128;
int64_t backward_blocks(int64_t rows, int64_t cols, int groups, int64_t resident) {
  const int64_t blocks = ceil_div(rows, groups);
  const int64_t want = std::min(blocks, resident * ceil_div(blocks, resident * kMostRows));
  return cols % 4 == 0 ? want : std::max<int64_t>(4, want / 4 * 4);
}

struct BackwardPlan {
  int vpt, warps, lanes, cluster, groups;  // words of a thread; warps of a block to a row; vpt 0: no such kernel
  int per_sm;                       // blocks that an SM's registers and shared memory hold
};

BackwardPlan backward_plan(int64_t cols) {
  const int64_t words = words_of(cols);
  if (words > 8 * 128 * kMostWarps) return {0, 0, 0, 0, 0, 0};
  BackwardPlan plan;
  plan.vpt = words <= 8 ? 1 : words <= 64 ? 2 : 4;
  plan.lanes = words <= 16 ? 8 : words <= 32 ? 16 : 32;
  const int warps = static_cast<int>(ceil_div(words, plan.lanes * plan.vpt));
  plan.cluster = warps <= kMostWarps ? 1 : warps <= 32 ? 4 : 8;
  plan.warps = static_cast<int>(ceil_div(warps, plan.cluster));
  plan.groups = plan.warps == 1 || plan.warps == 2 || plan.warps == 4 ? 256 / (plan.warps * plan.lanes) : 1;
  plan.per_sm = std::max(1, warps_per_sm(plan.vpt) * 32 / (plan.warps * plan.lanes * plan.groups));
  return plan;
}

// As many at most, whatever the device holds at a time up to what its registers and memory say:
// whole rounds of that are fewer than the blocks that kMostRows asks for and one round more.
int64_t most_blocks(int64_t rows, int64_t cols, const BackwardPlan& plan) {
  const int64_t places = plan.per_sm * sm_count() / plan.cluster, blocks = ceil_div(rows, plan.groups);
  const int64_t most = std::min(blocks, ceil_div(blocks, kMostRows) + places);
  return cols % 4 == 0 ? most : std::max<int64_t>(4, most);
}

template <int VPT, int WARPS, int LANES, int CLUSTER, bool ODD, bool FUSED>
int64_t launch_backward(cudaStream_t s, const BackwardArgs& a, float* partial, const BackwardPlan& plan) {
  auto* kernel = norm_backward_kernel<VPT, WARPS, LANES, CLUSTER, ODD, FUSED>;
  const int threads = plan.warps * plan.groups * plan.lanes;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = Places<VPT, WARPS, ODD, FUSED>::bytes(threads);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {CLUSTER, 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = CLUSTER > 1 ? 1 : 0;
  // how many blocks or clusters the device holds at a time, looked up once for each size (or by
  // each of two host threads that meet here)
  static std::atomic<int> resident[64][kMostWarps + 1];
  int dev = 0, held = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64) held = resident[dev][plan.warps].load(std::memory_order_relaxed);
  if (held == 0) {
    // a lookup that fails is not kept, and its error is the call's: nothing is launched
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             Places<VPT, WARPS, ODD, FUSED>::bytes(kMostWarps * 32)) != cudaSuccess)
      return 0;
    held = plan.per_sm * sm_count() / CLUSTER;
    if (CLUSTER > 1) {
      cfg.gridDim = dim3(static_cast<unsigned>(held * CLUSTER));
      int clusters = 0;
      if (cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg) != cudaSuccess) return 0;
      held = std::max(1, std::min(held, clusters));
    }
    if (dev >= 0 && dev < 64) resident[dev][plan.warps].store(held, std::memory_order_relaxed);
  }
  const int64_t blocks = backward_blocks(a.rows, a.cols, plan.groups, held);
  cfg.gridDim = dim3(static_cast<unsigned>(blocks * CLUSTER));
  cudaLaunchKernelEx(&cfg, kernel, a, partial, device_error_word());
  return blocks;
}

template <int VPT, int WARPS, int LANES, int CLUSTER>
int64_t launch_backward(cudaStream_t s, const BackwardArgs& a, float* partial, const BackwardPlan& plan, bool odd) {
  const bool fused = a.dtotal || a.dx;
  if (odd)
    return fused ? launch_backward<VPT, WARPS, LANES, CLUSTER, true, true>(s, a, partial, plan)
                 : launch_backward<VPT, WARPS, LANES, CLUSTER, true, false>(s, a, partial, plan);
  return fused ? launch_backward<VPT, WARPS, LANES, CLUSTER, false, true>(s, a, partial, plan)
               : launch_backward<VPT, WARPS, LANES, CLUSTER, false, false>(s, a, partial, plan);
}

// Returns the partial rows that it leaves, or 0 with the runtime's error set.
int64_t launch_backward(cudaStream_t s, const BackwardArgs& a, float* partial, const BackwardPlan& plan, bool odd) {
  switch (plan.cluster) {
    case 4: return launch_backward<4, 0, 32, 4>(s, a, partial, plan, odd);
    case 8: return launch_backward<4, 0, 32, 8>(s, a, partial, plan, odd);
    default: break;
  }
  if (plan.vpt == 1) return launch_backward<1, 1, 8, 1>(s, a, partial, plan, odd);
  if (plan.lanes == 8) return launch_backward<2, 1, 8, 1>(s, a, partial, plan, odd);
  if (plan.lanes == 16) return launch_backward<2, 1, 16, 1>(s, a, partial, plan, odd);
  if (plan.vpt == 2) return launch_backward<2, 1, 32, 1>(s, a, partial, plan, odd);
  switch (plan.warps) {
    case 1: return launch_backward<4, 1, 32, 1>(s, a, partial, plan, odd);
    case 2: return launch_backward<4, 2, 32, 1>(s, a, partial, plan, odd);
    case 4: return launch_backward<4, 4, 32, 1>(s, a, partial, plan, odd);
    default: return launch_backward<4, 0, 32, 1>(s, a, partial, plan, odd);
  }
}

// Splits of the rows for the columns' sums in a pass of their own, of 16 rows or more: blocks to
// fill the machine where the columns are few, 64 where they are many.
int64_t splits_of(int64_t rows, int64_t cols) {
  const int64_t most = std::max<int64_t>(64, 4 * sm_count() / ceil_div(cols, kThreads));
  return std::max<int64_t>(1, std::min(most, rows / kSpan));
}

// An output that equals another tensor, where the caller has a buffer of its own for it.
void copy_output(cudaStream_t s, const float* from, float* to, int64_t count) {
  if (to && to != from) cudaMemcpyAsync(to, from, count * sizeof(float), cudaMemcpyDeviceToDevice, s);
}

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
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  TimedLaunch timer("norm_forward", s);
  if (!residual && !a.drop.threshold) {
    copy_output(s, input, total, rows * cols);
    a.total = nullptr;  // the kernels have no other than the input
  }
  const int64_t words = words_of(cols);
  if (words > 8192 || !aligned(input) || !aligned(residual) || !aligned(output) || !aligned(a.total)) {
    const int grid = static_cast<int>(std::min<int64_t>(rows, 8 * sm_count()));
    norm_forward_any_kernel<<<grid, kThreads, 0, s>>>(a);
    return launch_status("layer norm forward");
  }
  const bool odd = cols % 4 != 0 || !aligned(weight) || !aligned(bias);
  if (a.total && words > 4096) {
    // a row of two inputs would fill an SM's shared memory: the total by itself, then its norm
    launch_dropout(s, input, residual, total, rows * cols, a.drop);
    a.x = total, a.residual = nullptr, a.total = nullptr;
    a.drop.threshold = 0;
  }
  if (a.total) launch_forward<true>(s, a, words, odd);
  else launch_forward<false>(s, a, words, odd);
  return launch_status("layer norm forward");
}

extern "C" size_t tcx_sm100_layernorm_backward_workspace_bytes(int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0) return 0;
  // either path's partial column sums
  const BackwardPlan plan = backward_plan(cols);
  int64_t splits = splits_of(rows, cols);
  if (plan.vpt)
    splits = std::max(splits, most_blocks(rows, cols, plan));
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
  if (!a.drop.threshold) a.dx = nullptr;  // the kernels have no other than the residual's
  if (dweight && (!workspace || workspace_bytes < tcx_sm100_layernorm_backward_workspace_bytes(rows, cols)))
    return invalid("workspace too small for the layer norm gradient");
  TimedLaunch timer("norm_backward", s);
  float* partial = dweight ? static_cast<float*>(workspace) : nullptr;
  const BackwardPlan plan = backward_plan(cols);
  if (plan.vpt && aligned(dy) && aligned(total) && aligned(dtotal) && aligned(dresidual) && aligned(a.dx)) {
    const int64_t splits = launch_backward(s, a, partial, plan, cols % 4 != 0 || !aligned(weight));
    if (splits == 0) return launch_status("layer norm backward");
    if (partial) join_columns(s, partial, splits, cols, dweight, dbias);
  } else {
    const int grid = static_cast<int>(std::min<int64_t>(rows, 8 * sm_count()));
    norm_backward_any_kernel<<<grid, kThreads, 0, s>>>(a);
    if (dweight) {
      const int64_t splits = splits_of(rows, cols);
      const unsigned blocks = static_cast<unsigned>(ceil_div(cols, kThreads));
      norm_columns_kernel<<<dim3(blocks, static_cast<unsigned>(splits)), kThreads, 0, s>>>(a, partial,
                                                                                           ceil_div(rows, splits));
      join_columns(s, partial, splits, cols, dweight, dbias);
    }
  }
  if (!a.dx) copy_output(s, dresidual, dx, rows * cols);
  return launch_status("layer norm backward");
}
