// Gated linear recurrence over [batch, time, channels] on sm_100a and its backward pass.
//
//   decay form:    h_t = a_t h_(t-1) + x_t,            a = gate
//   sigmoid form:  h_t = s_t h_(t-1) + (1 - s_t) x_t,  s = 1 / (1 + e^-gate)
//
// each channel by itself, from `initial` (0 without one). Steps at and beyond a sequence's
// length hold the state: h_t = h_(t-1), whatever gate and x hold there. Backward, with c the
// gradient that reaches the state before step t (c after the last step is dstate, or 0):
//
//   G_t = dh_t + c_(t+1),  c_t = a_t G_t,  dinitial = c_first
//   decay form:    dx_t = G_t,            dgate_t = G_t h_(t-1)
//   sigmoid form:  dx_t = (1 - s_t) G_t,  dgate_t = G_t (h_(t-1) - x_t) s_t (1 - s_t)
//
// and c_t = G_t, dx_t = dgate_t = 0 at steps that a sequence does not have.
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "common.cuh"
#include "ptx.cuh"
#include "rowmath.cuh"

namespace tcx {
namespace {

struct Args {
  const float *gate, *x, *initial;
  const int32_t* lengths;
  float *h, *state;
  const float *dh, *hs, *dstate;  // backward: the gradients that come in and the forward's h
  float *dgate, *dx, *dinitial;
  int64_t batch, time, channels;
};

// s and 1 - s without cancellation: both from e^-|z|.
__device__ __forceinline__ void sigmoid_pair(float z, float& s, float& rest) {
  const float e = rowmath::exp_ex2(-fabsf(z)), big = __fdividef(1.0f, 1.0f + e), small = e * big;
  s = z >= 0.0f ? big : small;
  rest = z >= 0.0f ? small : big;
}

__device__ __forceinline__ int64_t length_of(const Args& a, int64_t b) {
  if (!a.lengths) return a.time;
  const int64_t n = a.lengths[b];
  return n < 0 ? 0 : n > a.time ? a.time : n;
}

template <int VEC>
__device__ __forceinline__ void load(float (&v)[VEC], const float* p) {
  if constexpr (VEC == 4) {
    const float4 t = __ldcs(reinterpret_cast<const float4*>(p));
    v[0] = t.x, v[1] = t.y, v[2] = t.z, v[3] = t.w;
  } else if constexpr (VEC == 2) {
    const float2 t = __ldcs(reinterpret_cast<const float2*>(p));
    v[0] = t.x, v[1] = t.y;
  } else {
    v[0] = __ldcs(p);
  }
}

template <int VEC>
__device__ __forceinline__ void store(float* p, const float (&v)[VEC]) {
  if constexpr (VEC == 4) __stcs(reinterpret_cast<float4*>(p), make_float4(v[0], v[1], v[2], v[3]));
  else if constexpr (VEC == 2) __stcs(reinterpret_cast<float2*>(p), make_float2(v[0], v[1]));
  else __stcs(p, v[0]);
}

// Loads and stores of values that other blocks of the grid write or read (L2, never L1).
template <int VEC>
__device__ __forceinline__ void load_shared(float (&v)[VEC], const float* p) {
  if constexpr (VEC == 4) {
    const float4 t = __ldcg(reinterpret_cast<const float4*>(p));
    v[0] = t.x, v[1] = t.y, v[2] = t.z, v[3] = t.w;
  } else if constexpr (VEC == 2) {
    const float2 t = __ldcg(reinterpret_cast<const float2*>(p));
    v[0] = t.x, v[1] = t.y;
  } else {
    v[0] = __ldcg(p);
  }
}

template <int VEC>
__device__ __forceinline__ void store_shared(float* p, const float (&v)[VEC]) {
  if constexpr (VEC == 4) __stcg(reinterpret_cast<float4*>(p), make_float4(v[0], v[1], v[2], v[3]));
  else if constexpr (VEC == 2) __stcg(reinterpret_cast<float2*>(p), make_float2(v[0], v[1]));
  else __stcg(p, v[0]);
}

template <int VEC>
__device__ __forceinline__ void start_of(float (&v)[VEC], const float* p, int64_t at) {
#pragma unroll
  for (int i = 0; i < VEC; ++i) v[i] = p ? __ldg(p + at + i) : 0.0f;
}

// The state after a part of a sequence with product A and state-from-zero B, entered with h.
// From a zero state it is B alone: a product that overflowed says nothing about it.
__device__ __forceinline__ float advance(float h, float A, float B) { return h == 0.0f ? B : fmaf(A, h, B); }

// What the second half of a backward step needs from memory.
template <int VEC, bool SIGMOID>
struct Reads {
  float before[VEC], x[SIGMOID ? VEC : 1];
};

template <int VEC, bool SIGMOID>
__device__ __forceinline__ void backward_step(const float (&gate)[VEC], const float (&dh)[VEC],
                                              const Reads<VEC, SIGMOID>& r, bool live, float (&c)[VEC],
                                              float (&dgate)[VEC], float (&dx)[VEC]) {
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    const float g = dh[i] + c[i];
    float s = gate[i], rest = 1.0f;
    if (SIGMOID) sigmoid_pair(s, s, rest);
    const float d = SIGMOID ? g * rest : g;
    dx[i] = live ? d : 0.0f;
    dgate[i] = live ? (SIGMOID ? d * s * (r.before[i] - r.x[SIGMOID ? i : 0]) : d * r.before[i]) : 0.0f;
    c[i] = live ? s * g : g;
  }
}

// ------------------------------------------------------- one thread per VEC channels
// Walks through time by itself. For short sequences: a token of each running sequence is
// one step of this kernel.
template <int VEC, bool SIGMOID>
__global__ void __launch_bounds__(256) walk_forward_kernel(Args a) {
  const int64_t i = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * VEC;
  if (i >= a.batch * a.channels) return;
  const int64_t b = i / a.channels, n = length_of(a, b);
  float h[VEC];
  start_of<VEC>(h, a.initial, i);
  int64_t at = b * (a.time - 1) * a.channels + i;
  for (int64_t t = 0; t < a.time; ++t, at += a.channels) {
    if (t < n) {
      float g[VEC], x[VEC];
      load<VEC>(g, a.gate + at);
      load<VEC>(x, a.x + at);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        if (SIGMOID) {
          float rest;
          sigmoid_pair(g[j], g[j], rest);
          x[j] *= rest;
        }
        h[j] = fmaf(g[j], h[j], x[j]);
      }
    }
    store<VEC>(a.h + at, h);
  }
  if (a.state) store<VEC>(a.state + i, h);
}

template <int VEC, bool SIGMOID>
__global__ void __launch_bounds__(256) walk_backward_kernel(Args a) {
  const int64_t i = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * VEC;
  if (i >= a.batch * a.channels) return;
  const int64_t b = i / a.channels, n = length_of(a, b);
  float c[VEC];
  start_of<VEC>(c, a.dstate, i);
  int64_t at = b * (a.time - 1) * a.channels + i + (a.time - 1) * a.channels;
  for (int64_t t = a.time - 1; t >= 0; --t, at -= a.channels) {
    float gate[VEC] = {}, dh[VEC], dgate[VEC], dx[VEC];
    Reads<VEC, SIGMOID> r = {};
    load<VEC>(dh, a.dh + at);
    if (t < n) {
      load<VEC>(gate, a.gate + at);
      if (t) load<VEC>(r.before, a.hs + at - a.channels);
      else start_of<VEC>(r.before, a.initial, i);
      if constexpr (SIGMOID) load<VEC>(r.x, a.x + at);
    }
    backward_step<VEC, SIGMOID>(gate, dh, r, t < n, c, dgate, dx);
    store<VEC>(a.dgate + at, dgate);
    store<VEC>(a.dx + at, dx);
  }
  if (a.dinitial) store<VEC>(a.dinitial + i, c);
}

// --------------------------------------------------------- scan over parts of the time
// A sequence of one batch entry and 32 VEC channels (a chain) is cut into chunks of
// kWarps * kSteps steps, a block to a chunk: each warp holds kSteps steps of its 32 VEC
// channels in registers, so memory is read once and written once. A part's effect on a
// state is (A, B): the product of its gates and its last state from zero. The warps' parts
// meet in shared memory; the chunks' in the workspace: a block publishes its (A, B), walks
// back over its chain's published parts to the nearest chunk whose last state is known,
// advances that state through the parts between, and publishes its own. Chunks are handed
// out in order of a ticket, so what a block waits for has always begun; the waits are
// bounded all the same.
//
// The state that enters a chunk is always the previous chunk's entering state advanced by
// that chunk's (A, B), whether a published state or the parts themselves bring it: the
// result does not depend on the order in which blocks run.
//
// Backward the same scan runs from the last step to the first, on c_t = a_t (c_(t+1) + dh_t).
constexpr int kWarps = 8, kSteps = 8, kChunk = kWarps * kSteps;
constexpr int64_t kWalkSteps = 16;  // up to so many steps a thread walks through time alone

struct Scan {
  unsigned* ticket;
  unsigned* flags;  // per chunk: 0 nothing, 1 parts, 2 the last state
  float* parts;     // per chunk: A, then B
  float* states;    // per chunk
  int32_t blocks;   // channel blocks
  int64_t chains, chunks;
};

__device__ __forceinline__ unsigned load_flag(const unsigned* p) {
  unsigned v;
  asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}

// By one warp, after its lanes' store_shared.
__device__ __forceinline__ void publish(unsigned* flag, unsigned value, int lane) {
  __threadfence();
  __syncwarp();
  if (lane == 0) asm volatile("st.release.gpu.global.u32 [%0], %1;" ::"l"(flag), "r"(value) : "memory");
}

// How many chunks before `chunk` have to be advanced through to reach it from a known state
// (that of chunk - 1 - result, or the sequence's start when that is -1). One warp.
__device__ int64_t walk_back(const unsigned* flags, int64_t chunk, int lane, int* err) {
  int64_t depth = 0;
  uint64_t began = 0;
  for (;;) {
    const int64_t at = chunk - 1 - depth - lane;
    const unsigned f = at < 0 ? 2u : load_flag(flags + at);
    const unsigned known = __ballot_sync(0xffffffffu, f == 2u), there = __ballot_sync(0xffffffffu, f != 0u);
    if (known) {
      const int j = __ffs(known) - 1;
      const unsigned need = (1u << j) - 1u;
      if ((there & need) == need) return depth + j;
    } else if (there == 0xffffffffu) {
      depth += 32;
      continue;
    }
    const uint64_t now = ptx::globaltimer();
    if (!began) began = now;
    if (__any_sync(0xffffffffu, now - began > ptx::kWaitLimitNs)) {
      if (lane == 0) record_device_error(err, 0x501);
      return 0;
    }
  }
}

template <int VEC, bool SIGMOID, bool BACK>
__global__ void __launch_bounds__(kWarps * 32, 2) scan_kernel(Args a, Scan sc, int* err) {
  constexpr int kWide = 32 * VEC;
  __shared__ __align__(16) float part[kWarps][2][kWide];
  __shared__ __align__(16) float entry[kWide], ended[kWide];
  __shared__ unsigned mine;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) mine = atomicAdd(sc.ticket, 1u);
  __syncthreads();
  const int64_t chain = mine % sc.chains, chunk = mine / sc.chains;
  const int64_t b = chain / sc.blocks, c0 = (chain % sc.blocks) * kWide + lane * VEC;
  const bool inside = c0 < a.channels;
  const int64_t n = length_of(a, b);
  const int64_t first = chunk * kChunk + warp * kSteps;  // in the scan's own order
  const int64_t base = b * a.time * a.channels + c0;
  auto step_of = [&](int s) { return BACK ? a.time - 1 - (first + s) : first + s; };

  float g[kSteps][VEC], v[kSteps][VEC];  // gate and x, or gate and dh
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    const int64_t t = step_of(s);
    const bool in = inside && first + s < a.time;
#pragma unroll
    for (int i = 0; i < VEC; ++i) g[s][i] = BACK && SIGMOID ? 0.0f : 1.0f, v[s][i] = 0.0f;
    if (in && t < n) load<VEC>(g[s], a.gate + base + t * a.channels);
    if (in && (BACK || t < n)) load<VEC>(v[s], (BACK ? a.dh : a.x) + base + t * a.channels);
  }
  float A[VEC], B[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) A[i] = 1.0f, B[i] = 0.0f;
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    const bool live = first + s < a.time && step_of(s) < n;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      if (BACK) {
        float s1 = g[s][i], rest;
        if (SIGMOID) sigmoid_pair(s1, s1, rest);
        if (!live) s1 = 1.0f;
        A[i] *= s1;
        B[i] = s1 * (B[i] + v[s][i]);
      } else {
        if (SIGMOID && live) {
          float rest;
          sigmoid_pair(g[s][i], g[s][i], rest);
          v[s][i] *= rest;
        }
        A[i] *= g[s][i];
        B[i] = fmaf(g[s][i], B[i], v[s][i]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < VEC; ++i) part[warp][0][lane * VEC + i] = A[i], part[warp][1][lane * VEC + i] = B[i];
  __syncthreads();

  // A forward chunk in which the sequence ends: what is held after it is the state itself,
  // not one advanced by (A, B), so this chunk publishes that state alone.
  const bool ends = !BACK && n < a.time && n > chunk * kChunk && n <= chunk * kChunk + kChunk;
  const int64_t row = chain * sc.chunks + chunk;
  unsigned* flag = sc.flags + row;
  if (warp == 0) {
    float h[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) A[i] = 1.0f, B[i] = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float wa = part[w][0][lane * VEC + i];
        A[i] *= wa;
        B[i] = fmaf(wa, B[i], part[w][1][lane * VEC + i]);
      }
    int64_t depth = 0;
    if (chunk > 0) {
      if (!ends && load_flag(flag - 1) != 2u) {
        store_shared<VEC>(sc.parts + row * 2 * kWide + lane * VEC, A);
        store_shared<VEC>(sc.parts + row * 2 * kWide + kWide + lane * VEC, B);
        publish(flag, 1u, lane);
      }
      depth = walk_back(flag - chunk, chunk, lane, err);
    }
    if (chunk - depth > 0) {
      load_shared<VEC>(h, sc.states + (row - 1 - depth) * kWide + lane * VEC);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) h[i] = 0.0f;
      if (inside) start_of<VEC>(h, BACK ? a.dstate : a.initial, b * a.channels + c0);
    }
#pragma unroll 4
    for (int64_t q = row - depth; q < row; ++q) {
      float qa[VEC], qb[VEC];
      load_shared<VEC>(qa, sc.parts + q * 2 * kWide + lane * VEC);
      load_shared<VEC>(qb, sc.parts + q * 2 * kWide + kWide + lane * VEC);
#pragma unroll
      for (int i = 0; i < VEC; ++i) h[i] = advance(h[i], qa[i], qb[i]);
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) entry[lane * VEC + i] = h[i];
    if (chunk + 1 < sc.chunks && !ends) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) h[i] = advance(h[i], A[i], B[i]);
      store_shared<VEC>(sc.states + row * kWide + lane * VEC, h);
      publish(flag, 2u, lane);
    }
  }
  __syncthreads();
  float h[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) h[i] = entry[lane * VEC + i];
  for (int w = 0; w < warp; ++w)
#pragma unroll
    for (int i = 0; i < VEC; ++i) h[i] = advance(h[i], part[w][0][lane * VEC + i], part[w][1][lane * VEC + i]);

  if constexpr (BACK) {
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int64_t t = step_of(s);
      if (!inside || first + s >= a.time) continue;
      const int64_t at = base + t * a.channels;
      Reads<VEC, SIGMOID> r = {};
      if (t < n) {
        if (t) load<VEC>(r.before, a.hs + at - a.channels);
        else start_of<VEC>(r.before, a.initial, b * a.channels + c0);
        if constexpr (SIGMOID) load<VEC>(r.x, a.x + at);
      }
      float dgate[VEC], dx[VEC];
      backward_step<VEC, SIGMOID>(g[s], v[s], r, t < n, h, dgate, dx);
      store<VEC>(a.dgate + at, dgate);
      store<VEC>(a.dx + at, dx);
    }
  } else {
    auto write = [&](int s) {
      const int64_t t = first + s;
#pragma unroll
      for (int i = 0; i < VEC; ++i) h[i] = fmaf(g[s][i], h[i], v[s][i]);
      if (inside && t < a.time) store<VEC>(a.h + base + t * a.channels, h);
    };
    const bool held = ends && first >= n;  // this warp's steps come after the end
    if (!held) {
#pragma unroll
      for (int s = 0; s < kSteps; ++s) write(s);
    }
    if (ends) {
      if (n > first && n <= first + kSteps) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) ended[lane * VEC + i] = h[i];
        if (chunk + 1 < sc.chunks) {
          store_shared<VEC>(sc.states + row * kWide + lane * VEC, h);
          publish(flag, 2u, lane);
        }
      }
      __syncthreads();
      if (held) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) h[i] = ended[lane * VEC + i];
#pragma unroll
        for (int s = 0; s < kSteps; ++s) write(s);
      }
    }
  }
  float* last = BACK ? a.dinitial : a.state;
  if (last && inside && first < a.time && first + kSteps >= a.time) store<VEC>(last + b * a.channels + c0, h);
}

// ------------------------------------------------------------------------- launches
bool aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// Channels per thread: as wide as the channel count and every buffer's alignment allow.
int width_of(const Args& a) {
  const void* all[] = {a.gate, a.x, a.h, a.state, a.dh, a.hs, a.dgate, a.dx, a.dinitial};
  for (int vec = 4; vec > 1; vec /= 2) {
    bool fits = a.channels % vec == 0;
    for (const void* p : all) fits = fits && aligned(p, 4 * vec);
    // half a warp's lanes would stand idle: take narrower ones
    if (fits && (a.channels > 16 * vec || vec == 1)) return vec;
  }
  return 1;
}

int64_t chains_of(int64_t batch, int64_t channels, int vec) { return batch * ceil_div(channels, 32 * vec); }

template <int VEC, bool SIGMOID, bool BACK>
int launch(cudaStream_t s, const Args& a, void* workspace) {
  if (a.time <= kWalkSteps) {
    const unsigned grid = static_cast<unsigned>(ceil_div(a.batch * a.channels, 256 * VEC));
    TimedLaunch timer(BACK ? "recurrence_walk_backward" : "recurrence_walk", s);
    if (BACK) walk_backward_kernel<VEC, SIGMOID><<<grid, 256, 0, s>>>(a);
    else walk_forward_kernel<VEC, SIGMOID><<<grid, 256, 0, s>>>(a);
    return launch_status("recurrence");
  }
  Scan sc;
  sc.blocks = static_cast<int32_t>(ceil_div(a.channels, 32 * VEC));
  sc.chains = a.batch * sc.blocks;
  sc.chunks = ceil_div(a.time, kChunk);
  const int64_t tiles = sc.chains * sc.chunks;
  if (tiles > INT32_MAX) return invalid("recurrence is too large for one call");
  float* f = static_cast<float*>(workspace);
  sc.parts = f;
  sc.states = f + tiles * 64 * VEC;
  sc.flags = reinterpret_cast<unsigned*>(sc.states + tiles * 32 * VEC);
  sc.ticket = sc.flags + tiles;
  cudaMemsetAsync(sc.flags, 0, (tiles + 1) * sizeof(unsigned), s);
  TimedLaunch timer(BACK ? "recurrence_scan_backward" : "recurrence_scan", s);
  scan_kernel<VEC, SIGMOID, BACK><<<static_cast<unsigned>(tiles), kWarps * 32, 0, s>>>(a, sc, device_error_word());
  return launch_status("recurrence");
}

template <bool SIGMOID, bool BACK>
int launch_width(cudaStream_t s, const Args& a, void* workspace) {
  switch (width_of(a)) {
    case 4: return launch<4, SIGMOID, BACK>(s, a, workspace);
    case 2: return launch<2, SIGMOID, BACK>(s, a, workspace);
    default: return launch<1, SIGMOID, BACK>(s, a, workspace);
  }
}

// A call of no steps: the state goes through.
int pass_through(cudaStream_t s, const float* from, float* to, int64_t count) {
  if (!to) return TCX_OK;
  const cudaError_t e = from ? cudaMemcpyAsync(to, from, count * sizeof(float), cudaMemcpyDeviceToDevice, s)
                             : cudaMemsetAsync(to, 0, count * sizeof(float), s);
  return e == cudaSuccess ? TCX_OK : launch_status("recurrence");
}

int check_recurrence(int form, int64_t batch, int64_t time, int64_t channels) {
  if (form != TCX_RECURRENCE_DECAY && form != TCX_RECURRENCE_SIGMOID) return invalid("unknown recurrence form");
  if (batch < 0 || time < 0 || channels < 0) return invalid("negative extent");
  if (batch && channels > INT64_MAX / 8 / batch) return invalid("element count overflows");
  if (batch * channels && time > INT64_MAX / 8 / (batch * channels)) return invalid("element count overflows");
  return TCX_OK;
}

}  // namespace
}  // namespace tcx

using namespace tcx;

extern "C" size_t tcx_sm100_recurrence_workspace_bytes(int64_t batch, int64_t time, int64_t channels) {
  if (check_recurrence(TCX_RECURRENCE_DECAY, batch, time, channels) || time <= kWalkSteps) return 0;
  // three values per channel and chunk, and a flag per chunk: the narrowest blocks have the
  // most flags, the widest the most channels past the end
  const int64_t chunks = ceil_div(time, kChunk);
  return static_cast<size_t>(chains_of(batch, channels, 4) * 128 * 3 * chunks + chains_of(batch, channels, 1) * chunks +
                             1) * sizeof(float);
}

extern "C" int tcx_sm100_recurrence_forward(tcx_stream_t stream, int form, const float* gate, const float* x,
                                            const float* initial, const int32_t* lengths, float* h, float* state,
                                            int64_t batch, int64_t time, int64_t channels, void* workspace,
                                            size_t workspace_bytes) {
  clear_error();
  if (int rc = check_recurrence(form, batch, time, channels)) return rc;
  if (batch == 0 || channels == 0) return TCX_OK;
  if (time && (!gate || !x || !h)) return invalid("missing buffer");
  if (workspace_bytes < tcx_sm100_recurrence_workspace_bytes(batch, time, channels))
    return invalid("workspace too small for the recurrence");
  Args a{gate, x, initial, lengths, h, state, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, batch, time,
         channels};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (time == 0) return pass_through(s, initial, state, batch * channels);
  return form == TCX_RECURRENCE_SIGMOID ? launch_width<true, false>(s, a, workspace)
                                        : launch_width<false, false>(s, a, workspace);
}

extern "C" int tcx_sm100_recurrence_backward(tcx_stream_t stream, int form, const float* dh, const float* gate,
                                             const float* x, const float* h, const float* initial,
                                             const int32_t* lengths, const float* dstate, float* dgate, float* dx,
                                             float* dinitial, int64_t batch, int64_t time, int64_t channels,
                                             void* workspace, size_t workspace_bytes) {
  clear_error();
  if (int rc = check_recurrence(form, batch, time, channels)) return rc;
  if (batch == 0 || channels == 0) return TCX_OK;
  if (time && (!dh || !gate || !h || !dgate || !dx)) return invalid("missing buffer");
  if (time && form == TCX_RECURRENCE_SIGMOID && !x) return invalid("the sigmoid form's gradient needs x");
  if (workspace_bytes < tcx_sm100_recurrence_workspace_bytes(batch, time, channels))
    return invalid("workspace too small for the recurrence");
  Args a{gate, x, initial, lengths, nullptr, nullptr, dh, h, dstate, dgate, dx, dinitial, batch, time, channels};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (time == 0) return pass_through(s, dstate, dinitial, batch * channels);
  return form == TCX_RECURRENCE_SIGMOID ? launch_width<true, true>(s, a, workspace)
                                        : launch_width<false, true>(s, a, workspace);
}
