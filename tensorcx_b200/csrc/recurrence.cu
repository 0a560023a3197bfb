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
#include <type_traits>

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
// A sequence of one batch entry and 32 channels (a chain) is cut into chunks of time, a block
// to a chunk at a time. A row of a chunk is 128 bytes: 32 / VEC lanes of a warp read it, so a
// warp's lanes form VEC groups, and each group of each warp takes kSteps steps of its own.
// Memory is read once and written once. A part's effect on a state is (A, B): the product of
// its gates and its last state from zero. The groups' parts meet by shuffles, the warps' in
// shared memory and the chunks' in the workspace: a block publishes its (A, B), walks back
// over its chain's published parts to the nearest chunk whose last state is known, advances
// that state through the parts between, and publishes its own. Blocks stay on their SM and
// take chunks in order of a ticket, each in the order it got them, so what a block waits for
// has always begun; the waits are bounded all the same. The next chunk's data come into
// shared memory (cp.async; a thread copies and reads its own places only, so that needs no
// barrier) as soon as the values there have been taken into registers or used.
//
// The state that enters a chunk is always the previous chunk's entering state advanced by
// that chunk's (A, B), whether a published state or the parts themselves bring it: the
// result does not depend on the order in which blocks run.
//
// Backward the same scan runs from the last step to the first, on c_t = a_t (c_(t+1) + dh_t).
constexpr int kWide = 32;            // channels of a chain
constexpr int64_t kWalkSteps = 16;   // up to so many steps a thread walks through time alone
constexpr int kLeastChunk = 64;      // no shape has shorter chunks (the workspace is sized by it)

template <int VEC, bool SIGMOID, bool BACK>
struct Shape {
  static constexpr int kWarps = 4, kPerSm = 3, kThreads = kWarps * 32;
  static constexpr int kSteps = 32 / VEC;      // of one group
  static constexpr int kRing = BACK ? 1 : 2;   // chunks whose data are on their way
  static constexpr int kChunk = kWarps * VEC * kSteps;
  static constexpr int kArrays = BACK ? (SIGMOID ? 4 : 3) : 2;  // gate, x | gate, dh, the state before, x
  static constexpr int kArray = kChunk * kWide, kPlace = kArrays * kArray, kBytes = kRing * kPlace * 4;
  static_assert(kChunk >= kLeastChunk, "the workspace is sized for chunks of kLeastChunk steps or more");
  static_assert(kBytes * kPerSm <= 216 * 1024, "the blocks of an SM share its memory");
};

// What a chunk tells the later ones about one channel, written and read in one 128-bit access.
struct __align__(16) Record {
  float A, B;      // its part's effect
  float state;     // its last state
  unsigned known;  // 0: nothing yet, 1: A and B, 2: the state
};

struct Scan {
  unsigned* ticket;
  Record* records;                         // [chain, chunk, kWide], zero at the start
  unsigned blocks, chains, chunks, tiles;  // channel blocks; batch * blocks; per chain; in all
};

__device__ __forceinline__ void put(Record* p, float A, float B, float state, unsigned known) {
  asm volatile("{\n .reg .b64 lo, hi;\n .reg .b128 v;\n mov.b64 lo, {%1, %2};\n mov.b64 hi, {%3, %4};\n"
               " mov.b128 v, {lo, hi};\n st.relaxed.gpu.global.b128 [%0], v;\n}\n" ::"l"(p), "f"(A), "f"(B), "f"(state),
               "r"(known)
               : "memory");
}
__device__ __forceinline__ Record get(const Record* p) {
  Record r;
  asm volatile("{\n .reg .b64 lo, hi;\n .reg .b128 v;\n ld.relaxed.gpu.global.b128 v, [%4];\n mov.b128 {lo, hi}, v;\n"
               " mov.b64 {%0, %1}, lo;\n mov.b64 {%2, %3}, hi;\n}\n"
               : "=f"(r.A), "=f"(r.B), "=f"(r.state), "=r"(r.known)
               : "l"(p)
               : "memory");
  return r;
}

// The state that enters chunk `chunk` > 0 of a chain, a lane to a channel; `start` is the
// sequence's, `mine` the lane's record of the chunk. Looks at kLook chunks at a time.
constexpr int kLook = 8;
__device__ float enter(const Record* mine, int chunk, float start, int lane, int* err) {
  uint64_t began = 0;
  for (int depth = 0;;) {  // chunks that are known to have parts, nearest first
    Record r[kLook];
#pragma unroll
    for (int j = 0; j < kLook; ++j) {
      const int back = depth + j + 1;
      r[j].known = 2u, r[j].state = start, r[j].A = 1.0f, r[j].B = 0.0f;
      if (back <= chunk) r[j] = get(mine - static_cast<int64_t>(back) * kWide);
    }
    unsigned known = 0, there = 0;  // bit j: every lane sees it
#pragma unroll
    for (int j = 0; j < kLook; ++j) {
      known |= (__all_sync(0xffffffffu, r[j].known == 2u) ? 1u : 0u) << j;
      there |= (__all_sync(0xffffffffu, r[j].known != 0u) ? 1u : 0u) << j;
    }
    const int at = __ffs(known) - 1;
    const unsigned need = known ? (1u << at) - 1u : (1u << kLook) - 1u;
    if ((there & need) == need) {
      if (!known) {
        depth += kLook;
        continue;
      }
      float h = 0.0f;
#pragma unroll
      for (int j = kLook - 1; j >= 0; --j) {
        if (j == at) h = r[j].state;
        if (j < at) h = advance(h, r[j].A, r[j].B);
      }
#pragma unroll 4
      for (int back = depth; back > 0; --back) {
        const Record q = get(mine - static_cast<int64_t>(back) * kWide);
        h = advance(h, q.A, q.B);
      }
      return h;
    }
    const uint64_t now = ptx::globaltimer();
    if (!began) began = now;
    if (__any_sync(0xffffffffu, now - began > ptx::kWaitLimitNs)) {
      if (lane == 0) record_device_error(err, 0x501);
      return start;
    }
  }
}

// Copies VEC floats to shared memory, or zeros.
template <int VEC>
__device__ __forceinline__ void copy_async(uint32_t to, const float* from, bool there) {
  const int bytes = there ? 4 * VEC : 0;
  if constexpr (VEC == 4)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
  else if constexpr (VEC == 2)
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}

template <int VEC>
__device__ __forceinline__ void load_place(float (&v)[VEC], const float* p) {
  if constexpr (VEC == 4) {
    const float4 t = *reinterpret_cast<const float4*>(p);
    v[0] = t.x, v[1] = t.y, v[2] = t.z, v[3] = t.w;
  } else if constexpr (VEC == 2) {
    const float2 t = *reinterpret_cast<const float2*>(p);
    v[0] = t.x, v[1] = t.y;
  } else {
    v[0] = *p;
  }
}

template <int VEC>
__device__ __forceinline__ void store_place(float* p, const float (&v)[VEC]) {
  if constexpr (VEC == 4) *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  else if constexpr (VEC == 2) *reinterpret_cast<float2*>(p) = make_float2(v[0], v[1]);
  else *p = v[0];
}

// A thread's share of a chunk: kSteps steps of VEC channels.
struct Share {
  unsigned tile, chain, chunk;
  int64_t b, c;      // batch entry, first channel
  int64_t n, first;  // the sequence's length, the first step in the scan's own order
  int64_t at;        // of the first step in the arrays
  bool inside, full;  // the channels exist; so do all the steps
};

template <int VEC, bool SIGMOID, bool BACK>
__device__ __forceinline__ Share share_of(const Args& a, const Scan& sc, unsigned tile, int column, int before_me) {
  using Sh = Shape<VEC, SIGMOID, BACK>;
  Share m;
  m.tile = tile;
  m.chunk = tile / sc.chains;
  m.chain = tile - m.chunk * sc.chains;
  const unsigned b = m.chain / sc.blocks;
  m.b = b;
  m.c = static_cast<int64_t>(m.chain - b * sc.blocks) * kWide + column;
  m.n = length_of(a, m.b);
  m.first = static_cast<int64_t>(m.chunk) * Sh::kChunk + before_me;
  const int64_t t = BACK ? a.time - 1 - m.first : m.first;
  m.at = (m.b * a.time + t) * a.channels + m.c;
  m.inside = m.c < a.channels;
  m.full = m.inside && m.first + Sh::kSteps <= a.time && (BACK ? t < m.n : t + Sh::kSteps <= m.n);
  return m;
}

template <int VEC, bool SIGMOID, bool BACK>
__global__ void __launch_bounds__(Shape<VEC, SIGMOID, BACK>::kWarps * 32, Shape<VEC, SIGMOID, BACK>::kPerSm)
scan_kernel(Args a, Scan sc, int* err) {
  using Sh = Shape<VEC, SIGMOID, BACK>;
  constexpr int kWarps = Sh::kWarps, kSteps = Sh::kSteps, kChunk = Sh::kChunk, kArray = Sh::kArray, kRing = Sh::kRing;
  constexpr int kRow = 32 / VEC;       // lanes of a row
  constexpr int kNext = 32 * VEC;      // from one step's place in shared memory to the next one's
  extern __shared__ __align__(16) float stage[];
  __shared__ float parts[kWarps][2][kWide];
  __shared__ __align__(16) float entries[kWarps][kWide], ended[kWide];
  __shared__ unsigned queue[2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, group = lane / kRow;
  const int column = (lane % kRow) * VEC;              // within the chain
  const int before_me = (warp * VEC + group) * kSteps;  // steps of the chunk
  float* const place = stage + (warp * kSteps * 32 + lane) * VEC;
  const uint32_t place_at = ptx::smem_u32(place);
  const int64_t stride = BACK ? -a.channels : a.channels;

  // Step s of the share exists; the sequence has it.
  auto exists = [&](const Share& m, int s) { return m.full || (m.inside && m.first + s < a.time); };
  auto lives = [&](const Share& m, int s) {
    return m.full || (m.first + s < a.time && (BACK ? a.time - 1 - (m.first + s) : m.first + s) < m.n);
  };
  // What the parts are made from: gate and x, or gate and dh.
  auto fetch = [&](const Share& m, unsigned turn) {
    if (m.tile < sc.tiles) {
      const uint32_t to = place_at + (turn % kRing) * (Sh::kPlace * 4);
      const float *p = a.gate + m.at, *q = (BACK ? a.dh : a.x) + m.at;
#pragma unroll
      for (int s = 0; s < kSteps; ++s, p += stride, q += stride) {
        const bool live = m.inside && lives(m, s);
        copy_async<VEC>(to + 4 * s * kNext, live ? p : a.gate, live);
        const bool has = BACK ? exists(m, s) : live;
        copy_async<VEC>(to + 4 * (kArray + s * kNext), has ? q : a.gate, has);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  // What a backward chunk needs besides once its entering state is known.
  auto fetch_rest = [&](const Share& m) {
    if (m.tile < sc.tiles) {
      const float *p = a.hs + m.at - a.channels, *q = SIGMOID ? a.x + m.at : nullptr;
#pragma unroll
      for (int s = 0; s < kSteps; ++s, p += stride, q += stride) {
        const bool live = m.inside && lives(m, s), opening = m.first + s == a.time - 1;  // t = 0
        const bool has = live && (!opening || a.initial);
        copy_async<VEC>(place_at + 4 * (2 * kArray + s * kNext),
                        !has ? a.gate : opening ? a.initial + m.b * a.channels + m.c : p, has);
        if constexpr (SIGMOID) copy_async<VEC>(place_at + 4 * (3 * kArray + s * kNext), live ? q : a.gate, live);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };

  Share line[kRing];  // this chunk and those whose data are on their way
#pragma unroll
  for (int k = 0; k < kRing; ++k) {
    if (threadIdx.x == 0) queue[k & 1] = atomicAdd(sc.ticket, 1u);
    __syncthreads();
    line[k] = share_of<VEC, SIGMOID, BACK>(a, sc, queue[k & 1], column, before_me);
    fetch(line[k], k);
  }
  if (BACK) fetch_rest(line[0]);
  unsigned later = threadIdx.x == 0 ? atomicAdd(sc.ticket, 1u) : 0;
  __syncthreads();
  for (unsigned turn = 0; line[0].tile < sc.tiles; ++turn) {  // tickets past the end stay past it
    const Share m = line[0];
    const float* const here = place + (turn % kRing) * Sh::kPlace;
    asm volatile("cp.async.wait_group %0;" ::"n"(BACK ? 1 : kRing - 1) : "memory");
    float g[kSteps][VEC], v[kSteps][VEC];  // gate and x, or gate and dh
    float A[VEC], B[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) A[i] = 1.0f, B[i] = 0.0f;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      load_place<VEC>(g[s], here + s * kNext);
      load_place<VEC>(v[s], here + kArray + s * kNext);
      const bool live = lives(m, s);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        if (BACK) {
          float s1 = g[s][i], rest;
          if (SIGMOID) sigmoid_pair(s1, s1, rest);
          if (!live) s1 = 1.0f;
          A[i] *= s1;
          B[i] = s1 * (B[i] + v[s][i]);
        } else {
          if (SIGMOID) {
            float rest;
            sigmoid_pair(g[s][i], g[s][i], rest);
            v[s][i] *= rest;
          }
          if (!live) g[s][i] = 1.0f;  // and v is 0
          A[i] *= g[s][i];
          B[i] = fmaf(g[s][i], B[i], v[s][i]);
        }
      }
    }
    // the groups before this one, then with it; the last group has the warp's part
    float eA[VEC], eB[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
#pragma unroll
      for (int off = 1; off < VEC; off *= 2) {
        const float pa = __shfl_up_sync(0xffffffffu, A[i], off * kRow), pb = __shfl_up_sync(0xffffffffu, B[i], off * kRow);
        if (group >= off) {
          B[i] = fmaf(A[i], pb, B[i]);
          A[i] *= pa;
        }
      }
      eA[i] = eB[i] = 0.0f;
      if (VEC > 1) {
        eA[i] = __shfl_up_sync(0xffffffffu, A[i], kRow);
        eB[i] = __shfl_up_sync(0xffffffffu, B[i], kRow);
      }
      if (group == VEC - 1) parts[warp][0][column + i] = A[i], parts[warp][1][column + i] = B[i];
    }
    if (threadIdx.x == 0) queue[0] = later;
    __syncthreads();
#pragma unroll
    for (int k = 0; k + 1 < kRing; ++k) line[k] = line[k + 1];
    line[kRing - 1] = share_of<VEC, SIGMOID, BACK>(a, sc, queue[0], column, before_me);

    // A forward chunk in which the sequence ends: what is held after it is the state itself,
    // not one advanced by (A, B), so this chunk publishes that state alone.
    const int64_t opens = m.first - before_me;
    const bool ends = !BACK && m.n < a.time && m.n > opens && m.n <= opens + kChunk;
    Record* const record = sc.records + (static_cast<int64_t>(m.chain) * sc.chunks + m.chunk) * kWide;
    if (warp == 0) {  // a lane to a channel
      float wA = 1.0f, wB = 0.0f, state = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        wB = fmaf(parts[w][0][lane], wB, parts[w][1][lane]);
        wA *= parts[w][0][lane];
      }
      const int64_t channel = m.c - column + lane;
      const float* start = BACK ? a.dstate : a.initial;
      if (start && channel < a.channels) state = __ldg(start + m.b * a.channels + channel);
      const bool goes_on = m.chunk + 1 < sc.chunks && !ends;
      if (m.chunk > 0) {
        if (goes_on) put(record + lane, wA, wB, 0.0f, 1u);
        state = enter(record + lane, static_cast<int>(m.chunk), state, lane, err);
      }
      if (goes_on) put(record + lane, wA, wB, advance(state, wA, wB), 2u);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        entries[w][lane] = state;
        state = advance(state, parts[w][0][lane], parts[w][1][lane]);
      }
    }
    fetch(line[kRing - 1], turn);
    if (threadIdx.x == 0) later = atomicAdd(sc.ticket, 1u);
    __syncthreads();
    float h[VEC];
    load_place<VEC>(h, &entries[warp][column]);
    if (group > 0) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) h[i] = advance(h[i], eA[i], eB[i]);
    }

    if constexpr (BACK) {
      asm volatile("cp.async.wait_group 1;" ::: "memory");
      float *p = a.dgate + m.at, *q = a.dx + m.at;
#pragma unroll
      for (int s = 0; s < kSteps; ++s, p += stride, q += stride) {
        Reads<VEC, SIGMOID> r;
        load_place<VEC>(r.before, place + 2 * kArray + s * kNext);
        if constexpr (SIGMOID) load_place<VEC>(r.x, place + 3 * kArray + s * kNext);
        if (!exists(m, s)) continue;
        float dgate[VEC], dx[VEC];
        backward_step<VEC, SIGMOID>(g[s], v[s], r, lives(m, s), h, dgate, dx);
        store<VEC>(p, dgate);
        store<VEC>(q, dx);
      }
      fetch_rest(line[0]);
    } else {
      auto write = [&]() {
        float* p = a.h + m.at;
#pragma unroll
        for (int s = 0; s < kSteps; ++s, p += stride) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) h[i] = fmaf(g[s][i], h[i], v[s][i]);
          if (exists(m, s)) store<VEC>(p, h);
        }
      };
      const bool held = ends && m.first >= m.n;  // this group's steps come after the end
      if (!held) write();
      if (ends) {
        if (m.n > m.first && m.n <= m.first + kSteps) {  // the group that has the last step
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            ended[column + i] = h[i];
            if (m.chunk + 1 < sc.chunks) put(record + column + i, 1.0f, 0.0f, h[i], 2u);
          }
        }
        __syncthreads();
        if (held) {
          load_place<VEC>(h, ended + column);
          write();
        }
      }
    }
    float* last = BACK ? a.dinitial : a.state;
    if (last && m.inside && m.first < a.time && m.first + kSteps >= a.time)
      store<VEC>(last + m.b * a.channels + m.c, h);
  }
}

// ---------------------------------------------------------------- the forward scan
// The same scan with the walk back taken out of the blocks' way: kWarps warps make the parts
// of chunk i + 1 and then write the states of chunk i, while two more warps publish the parts
// (the teller) and bring the state that enters chunk i + 1 (the carrier). The values wait in
// shared memory between the two uses, in the places that the next chunks' data come into.
template <int VEC>
struct Forward {
  static constexpr int kWarps = 4, kRing = 3, kPerSm = 2;
  static constexpr int kSteps = 32 / VEC;  // of one group
  static constexpr int kChunk = kWarps * VEC * kSteps;
  static constexpr int kArray = kChunk * kWide, kPlace = 2 * kArray, kBytes = kRing * kPlace * 4;  // gate, x
  static constexpr int kThreads = (kWarps + 2) * 32;
  static_assert(kChunk >= kLeastChunk, "the workspace is sized for chunks of kLeastChunk steps or more");
  static_assert(kBytes * kPerSm <= 216 * 1024, "the blocks of an SM share its memory");
};

// A chunk as its block sees it.
struct Tile {
  int64_t at;            // of its first step and channel in the arrays
  int64_t edge;          // of its first channel in the states
  int channels, steps;   // that exist, of kWide and kChunk; no channels: there is no such chunk
  int live;              // steps that the sequence has
  unsigned row, chunk;   // its records; its place in the chain
  int ends, last;        // the sequence ends in it, before time does; no chunk comes after it
};

// The block's chunk number i. With records: the one that a ticket names. Without: whole chains,
// chunk after chunk.
template <int VEC, bool WHOLE>
__device__ Tile next_tile(const Args& a, const Scan& sc, unsigned i) {
  using F = Forward<VEC>;
  Tile m = {};
  unsigned chain;
  if (!WHOLE) {
    const unsigned tile = atomicAdd(sc.ticket, 1u);
    if (tile >= sc.tiles) return m;
    m.chunk = tile / sc.chains;
    chain = tile - m.chunk * sc.chains;
  } else {
    const unsigned turn = i / sc.chunks;
    m.chunk = i - turn * sc.chunks;
    chain = blockIdx.x + turn * gridDim.x;
    if (chain >= sc.chains) return m;
  }
  const unsigned b = chain / sc.blocks, block = chain - b * sc.blocks;
  const int64_t n = length_of(a, b), opens = static_cast<int64_t>(m.chunk) * F::kChunk;
  const int64_t c = static_cast<int64_t>(block) * kWide;
  m.at = (b * a.time + opens) * a.channels + c;
  m.edge = b * a.channels + c;
  m.channels = static_cast<int>(min(a.channels - c, static_cast<int64_t>(kWide)));
  m.steps = static_cast<int>(min(a.time - opens, static_cast<int64_t>(F::kChunk)));
  m.live = static_cast<int>(max(min(n - opens, static_cast<int64_t>(F::kChunk)), static_cast<int64_t>(0)));
  m.row = chain * sc.chunks + m.chunk;
  m.ends = n < a.time && n > opens && n <= opens + F::kChunk;
  m.last = m.chunk + 1 == sc.chunks;
  return m;
}

// Barriers between the warps that work and the carrier, two of each by the chunk's parity.
enum { kPartsMade = 1, kEntryKnown = 3, kEndKnown = 5, kEndTold = 6, kPartsTold = 7 };
__device__ __forceinline__ void meet(int barrier, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(barrier), "r"(threads) : "memory");
}
__device__ __forceinline__ void signal(int barrier, int threads) {
  asm volatile("bar.arrive %0, %1;" ::"r"(barrier), "r"(threads) : "memory");
}

template <int VEC, bool SIGMOID, bool WHOLE>
__global__ void __launch_bounds__(Forward<VEC>::kThreads, Forward<VEC>::kPerSm)
scan_forward_kernel(Args a, Scan sc, int* err) {
  using F = Forward<VEC>;
  constexpr int kWarps = F::kWarps, kSteps = F::kSteps, kRing = F::kRing, kArray = F::kArray;
  constexpr int kAll = (kWarps + 1) * 32;  // the warps that work, and one of the two others
  constexpr int kRow = 32 / VEC, kNext = 32 * VEC;
  extern __shared__ __align__(16) float stage[];
  __shared__ float parts[2][kWarps][2][kWide], joined[2][2][kWide];  // the warps' and the chunk's
  __shared__ __align__(16) float entries[2][kWarps][kWide], ended[kWide];
  // Chunk i's at i % 8. The carrier sets i's in its turn i - kRing, before it signals that
  // turn's entry. The warps that work see that signal before they make chunk i - 1's parts
  // (kRing >= 3), and the teller reads i's after those were made; the slots in use at a time
  // are those from one chunk behind the carrier's to kRing beyond it.
  __shared__ Tile line[8];
  static_assert(kRing >= 3 && kRing + 3 <= 8, "a chunk's line is set before it is read, and kept until it is done");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;

  if (warp == kWarps + 1) {  // the teller
    for (int k = 0; k < kRing; ++k) __syncthreads();
    for (unsigned i = 0;; ++i) {
      const Tile& m = line[i & 7];
      if (m.channels == 0) return;
      meet(kPartsMade + (i & 1), kAll);
      const float (*part)[2][kWide] = parts[i & 1];
      float A = 1.0f, B = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        B = fmaf(part[w][0][lane], B, part[w][1][lane]);
        A *= part[w][0][lane];
      }
      joined[i & 1][0][lane] = A;
      joined[i & 1][1][lane] = B;
      if (!WHOLE && m.chunk > 0 && !m.last && !m.ends)
        put(sc.records + static_cast<int64_t>(m.row) * kWide + lane, A, B, 0.0f, 1u);
      signal(kPartsTold + (i & 1), 64);
    }
  }
  if (warp == kWarps) {  // the carrier
    for (int k = 0; k < kRing; ++k) {
      if (lane == 0) line[k] = next_tile<VEC, WHOLE>(a, sc, k);
      __syncthreads();
    }
    float state = 0.0f;
    bool ended_before = false;
    for (unsigned i = 0;; ++i) {
      const Tile m = line[i & 7];
      if (m.channels == 0) return;
      if (lane == 0) line[(i + kRing) & 7] = next_tile<VEC, WHOLE>(a, sc, i + kRing);
      const float start = a.initial && lane < m.channels ? __ldg(a.initial + m.edge + lane) : 0.0f;
      meet(kPartsTold + (i & 1), 64);
      const float (*part)[2][kWide] = parts[i & 1];
      const float A = joined[i & 1][0][lane], B = joined[i & 1][1][lane];
      if (!WHOLE) {
        Record* const record = sc.records + static_cast<int64_t>(m.row) * kWide + lane;
        state = m.chunk > 0 ? enter(record, static_cast<int>(m.chunk), start, lane, err) : start;
        if (!m.last && !m.ends) put(record, A, B, advance(state, A, B), 2u);
      } else {
        if (ended_before) {
          meet(kEndTold, kAll);
          state = ended[lane];
        }
        if (m.chunk == 0) state = start;
        ended_before = m.ends && !m.last;
      }
      float h = state;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        entries[i & 1][w][lane] = h;
        h = advance(h, part[w][0][lane], part[w][1][lane]);
      }
      state = advance(state, A, B);
      __syncwarp();
      signal(kEntryKnown + (i & 1), kAll);
    }
  }

  const int group = lane / kRow, column = (lane % kRow) * VEC;
  const int before_me = (warp * VEC + group) * kSteps;  // steps of the chunk
  float* const places = stage + (warp * kSteps * 32 + lane) * VEC;
  const uint32_t places_at = ptx::smem_u32(places);
  const int64_t mine = before_me * a.channels + column;

  auto fetch = [&](unsigned i) {
    const Tile& m = line[i & 7];
    if (m.channels) {
      const float *p = a.gate + m.at + mine, *q = a.x + m.at + mine;
      const uint32_t to = places_at + (i % kRing) * (F::kPlace * 4);
      if (column < m.channels && before_me + kSteps <= m.live) {
#pragma unroll 8
        for (int s = 0; s < kSteps; ++s, p += a.channels, q += a.channels) {
          copy_async<VEC>(to + 4 * s * kNext, p, true);
          copy_async<VEC>(to + 4 * (kArray + s * kNext), q, true);
        }
      } else {
#pragma unroll 4
        for (int s = 0; s < kSteps; ++s, p += a.channels, q += a.channels) {
          const bool live = column < m.channels && before_me + s < m.live;
          copy_async<VEC>(to + 4 * s * kNext, live ? p : a.gate, live);
          copy_async<VEC>(to + 4 * (kArray + s * kNext), live ? q : a.x, live);
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  // The parts of chunk i; the effect of the groups before this one into (eA, eB).
  auto make = [&](unsigned i, float (&eA)[VEC], float (&eB)[VEC]) {
    float* const place = places + (i % kRing) * F::kPlace;
    const int live = line[i & 7].live - before_me;
    float A[VEC], B[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) A[j] = 1.0f, B[j] = 0.0f;
#pragma unroll 8
    for (int s = 0; s < kSteps; ++s) {
      float g[VEC], v[VEC];
      load_place<VEC>(g, place + s * kNext);
      load_place<VEC>(v, place + kArray + s * kNext);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        if (SIGMOID) {
          float rest;
          sigmoid_pair(g[j], g[j], rest);
          v[j] *= rest;
        }
        if (s >= live) g[j] = 1.0f;  // and v is 0
        A[j] *= g[j];
        B[j] = fmaf(g[j], B[j], v[j]);
      }
      if (SIGMOID) {
        store_place<VEC>(place + s * kNext, g);
        store_place<VEC>(place + kArray + s * kNext, v);
      }
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
#pragma unroll
      for (int off = 1; off < VEC; off *= 2) {
        const float pa = __shfl_up_sync(0xffffffffu, A[j], off * kRow), pb = __shfl_up_sync(0xffffffffu, B[j], off * kRow);
        if (group >= off) {
          B[j] = fmaf(A[j], pb, B[j]);
          A[j] *= pa;
        }
      }
      eA[j] = eB[j] = 0.0f;
      if (VEC > 1) {
        eA[j] = __shfl_up_sync(0xffffffffu, A[j], kRow);
        eB[j] = __shfl_up_sync(0xffffffffu, B[j], kRow);
      }
      if (group == VEC - 1) parts[i & 1][warp][0][column + j] = A[j], parts[i & 1][warp][1][column + j] = B[j];
    }
    signal(kPartsMade + (i & 1), kAll);
  };

#pragma unroll
  for (int k = 0; k < kRing; ++k) {
    __syncthreads();
    fetch(k);
  }
  float eA[VEC], eB[VEC], nA[VEC], nB[VEC];
  if (line[0].channels) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kRing - 1) : "memory");
    make(0, eA, eB);
  }
  for (unsigned i = 0; line[i & 7].channels; ++i) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kRing - 2) : "memory");
    if (line[(i + 1) & 7].channels) make(i + 1, nA, nB);
    const Tile& m = line[i & 7];
    meet(kEntryKnown + (i & 1), kAll);
    float h[VEC];
    load_place<VEC>(h, &entries[i & 1][warp][column]);
    if (group > 0) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) h[j] = advance(h[j], eA[j], eB[j]);
    }
    const float* const place = places + (i % kRing) * F::kPlace;
    const bool inside = column < m.channels;
    auto write = [&](bool whole) {
      float* p = a.h + m.at + mine;
#pragma unroll 8
      for (int s = 0; s < kSteps; ++s, p += a.channels) {
        float g[VEC], v[VEC];
        load_place<VEC>(g, place + s * kNext);
        load_place<VEC>(v, place + kArray + s * kNext);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          if (!SIGMOID && !whole && before_me + s >= m.live) g[j] = 1.0f;
          h[j] = fmaf(g[j], h[j], v[j]);
        }
        if (whole || (inside && before_me + s < m.steps)) store<VEC>(p, h);
      }
    };
    if (inside && before_me + kSteps <= m.live) {
      write(true);
    } else if (!(m.ends && before_me >= m.live)) {
      write(false);
    }
    if (m.ends) {
      // what is held after the end is the state itself, not one advanced by (A, B): this
      // chunk publishes that state alone
      if (m.live > before_me && m.live <= before_me + kSteps) {  // the group that has the last step
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          ended[column + j] = h[j];
          if (!WHOLE && !m.last) put(sc.records + static_cast<int64_t>(m.row) * kWide + column + j, 1.0f, 0.0f, h[j], 2u);
        }
      }
      meet(kEndKnown, kWarps * 32);
      if (WHOLE && !m.last) signal(kEndTold, kAll);
      if (before_me >= m.live) {
        load_place<VEC>(h, ended + column);
        write(false);
      }
    }
    if (a.state && inside && before_me < m.steps && m.last && before_me + kSteps >= m.steps)
      store<VEC>(a.state + m.edge + column, h);
    fetch(i + kRing);
#pragma unroll
    for (int j = 0; j < VEC; ++j) eA[j] = nA[j], eB[j] = nB[j];
  }
}

// ------------------------------------------------------------------------- launches
bool aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// Channels per thread: as wide as the channel count and every buffer's alignment allow.
int width_of(const Args& a) {
  const void* all[] = {a.gate, a.x, a.initial, a.h, a.state, a.dh, a.hs, a.dstate, a.dgate, a.dx, a.dinitial};
  for (int vec = 4; vec > 1; vec /= 2) {
    bool fits = a.channels % vec == 0;
    for (const void* p : all) fits = fits && aligned(p, 4 * vec);
    if (fits) return vec;
  }
  return 1;
}

// Whole chains to a block, where the last of their rounds leaves few blocks idle.
bool walks(int64_t chains, int64_t blocks) { return chains * 10 >= ceil_div(chains, blocks) * blocks * 8; }

// `whole`: a block takes whole chains, and there are no records.
template <typename Sh>
int launch_scan(cudaStream_t s, const Args& a, void (*kernel)(Args, Scan, int*), bool whole, void* workspace) {
  const int64_t blocks = ceil_div(a.channels, kWide), chunks = ceil_div(a.time, Sh::kChunk);
  const int64_t tiles = a.batch * blocks * chunks;
  if (tiles > INT32_MAX) return invalid("recurrence is too large for one call");
  Scan sc;
  sc.blocks = static_cast<unsigned>(blocks);
  sc.chains = static_cast<unsigned>(a.batch * blocks);
  sc.chunks = static_cast<unsigned>(chunks);
  sc.tiles = static_cast<unsigned>(tiles);
  sc.records = whole ? nullptr : static_cast<Record*>(workspace);
  sc.ticket = whole ? nullptr : reinterpret_cast<unsigned*>(sc.records + tiles * kWide);
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::kBytes) != cudaSuccess)
    return launch_status("recurrence shared memory attribute");
  if (!whole) cudaMemsetAsync(workspace, 0, tiles * kWide * sizeof(Record) + sizeof(unsigned), s);
  const int64_t grid = std::min<int64_t>(whole ? sc.chains : tiles, Sh::kPerSm * sm_count());
  TimedLaunch timer("recurrence_scan", s);
  kernel<<<static_cast<unsigned>(grid), Sh::kThreads, Sh::kBytes, s>>>(a, sc, device_error_word());
  return launch_status("recurrence");
}

template <int VEC, bool SIGMOID, bool BACK>
int launch(cudaStream_t s, const Args& a, void* workspace) {
  if (a.time <= kWalkSteps) {
    const unsigned grid = static_cast<unsigned>(ceil_div(a.batch * a.channels, 256 * VEC));
    TimedLaunch timer(BACK ? "recurrence_walk_backward" : "recurrence_walk", s);
    if (BACK) walk_backward_kernel<VEC, SIGMOID><<<grid, 256, 0, s>>>(a);
    else walk_forward_kernel<VEC, SIGMOID><<<grid, 256, 0, s>>>(a);
    return launch_status("recurrence");
  }
  const int64_t chains = a.batch * ceil_div(a.channels, kWide);
  if constexpr (BACK) {
    return launch_scan<Shape<VEC, SIGMOID, true>>(s, a, scan_kernel<VEC, SIGMOID, true>, false, workspace);
  } else {
    if (walks(chains, Forward<VEC>::kPerSm * sm_count()))
      return launch_scan<Forward<VEC>>(s, a, scan_forward_kernel<VEC, SIGMOID, true>, true, workspace);
    return launch_scan<Forward<VEC>>(s, a, scan_forward_kernel<VEC, SIGMOID, false>, false, workspace);
  }
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
  // a record per channel for each chunk, and the ticket
  const int64_t tiles = batch * ceil_div(channels, kWide) * ceil_div(time, kLeastChunk);
  return static_cast<size_t>(tiles) * kWide * sizeof(Record) + sizeof(unsigned);
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
