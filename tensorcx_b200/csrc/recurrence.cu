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
//
// Bound by memory: 12 bytes an element forward (gate, x, h), 20 or 24 backward (dh, gate, the
// state before and, in the sigmoid form, x; dgate and dx), with 2 to 10 operations for them.
// What stands between that and the dependence of each step on the one before is the scan below.
// States, gradients and the parts' products are float32; the sigmoid's exponential is the
// hardware's base-2 one (2 ulp, plus the rounding of its argument).
//
// Measured on one B200, calls back to back on changing inputs (bytes that the form cannot do without
// over the call's time, against a copy's 6.55 TB/s): [1, 65536, 1024] decay forward 140 us (5.8
// TB/s, 0.88), [4, 8192, 2048] sigmoid forward 143 us (0.86), [2, 16384, 2048] sigmoid backward
// 261 us (6.2 TB/s, 0.94), decay 215 us (0.95), [2, 16384, 2049] 374 us (0.66) and forward 207 us
// (0.59), [64, 32, 4096] sigmoid forward 18.5 us and backward 31 to 36 (some of it from the second-
// level cache). Where a comment below gives two figures for a choice, they were taken side by side
// when it was made.
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>

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

// VEC = 4 channels or 1 of global memory that is read or written once, and of shared memory.
template <int VEC>
__device__ __forceinline__ void load(float (&v)[VEC], const float* p) {
  if constexpr (VEC == 4) {
    const float4 t = __ldcs(reinterpret_cast<const float4*>(p));
    v[0] = t.x, v[1] = t.y, v[2] = t.z, v[3] = t.w;
  } else {
    v[0] = __ldcs(p);
  }
}

template <int VEC>
__device__ __forceinline__ void store(float* p, const float (&v)[VEC]) {
  if constexpr (VEC == 4) __stcs(reinterpret_cast<float4*>(p), make_float4(v[0], v[1], v[2], v[3]));
  else __stcs(p, v[0]);
}

template <int VEC>
__device__ __forceinline__ void load_shared(float (&v)[VEC], const float* p) {
  if constexpr (VEC == 4) {
    const float4 t = *reinterpret_cast<const float4*>(p);
    v[0] = t.x, v[1] = t.y, v[2] = t.z, v[3] = t.w;
  } else {
    v[0] = *p;
  }
}

template <int VEC>
__device__ __forceinline__ void store_shared(float* p, const float (&v)[VEC]) {
  if constexpr (VEC == 4) *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  else *p = v[0];
}

// The state that a sequence starts from (or the gradient that reaches its last one).
template <int VEC>
__device__ __forceinline__ void start_of(float (&v)[VEC], const float* p, int64_t at) {
#pragma unroll
  for (int i = 0; i < VEC; ++i) v[i] = p ? __ldg(p + at + i) : 0.0f;
}

// The state after a part of a sequence with product A and state-from-zero B, entered with h.
// From a zero state it is B alone: a product that overflowed says nothing about it.
__device__ __forceinline__ float advance(float h, float A, float B) { return h == 0.0f ? B : fmaf(A, h, B); }

template <int VEC, bool SIGMOID>
__device__ __forceinline__ void backward_step(const float (&gate)[VEC], const float (&dh)[VEC],
                                              const float (&before)[VEC], const float (&x)[VEC], bool live,
                                              float (&c)[VEC], float (&dgate)[VEC], float (&dx)[VEC]) {
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    const float g = dh[i] + c[i];
    float s = gate[i], rest = 1.0f;
    if (SIGMOID) sigmoid_pair(s, s, rest);
    const float d = SIGMOID ? g * rest : g;
    dx[i] = live ? d : 0.0f;
    dgate[i] = live ? (SIGMOID ? d * s * (before[i] - x[i]) : d * before[i]) : 0.0f;
    c[i] = live ? s * g : g;
  }
}

// ------------------------------------------------------- one thread per VEC channels
// Walks through time by itself, the loads of AHEAD steps at a time. For short sequences (a
// token of each running sequence is one step of this kernel) and for batches wide enough.
// Four steps' loads of 4 channels in flight: [64, 32, 4096] forward 24 us, 28 with two, 26 with
// eight; eight of one channel: [100, 100, 1001] forward 35 us against 39. A call of one step
// has its own kernel, of which an SM holds more threads ([4096, 1, 4096]: forward 59 us before
// and 43 so, sigmoid backward 150 and 92). Its forward one is held to 32 registers and spills 24 to
// 76 bytes a thread: with 40 (4 to 40 bytes, 6 blocks to an SM) 41.2 us against 41.0.
template <int VEC>
constexpr int kAhead = VEC == 4 ? 4 : 8;

template <int VEC, int AHEAD, bool SIGMOID>
__global__ void __launch_bounds__(256, AHEAD == 1 ? 8 : 4) walk_forward_kernel(Args a) {
  const int64_t i = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * VEC;
  if (i >= a.batch * a.channels) return;
  const int64_t b = a.batch == 1 ? 0 : i / a.channels, n = length_of(a, b);
  float h[VEC];
  start_of<VEC>(h, a.initial, i);
  int64_t at = b * (a.time - 1) * a.channels + i;
  for (int64_t t0 = 0; t0 < a.time; t0 += AHEAD) {
    float g[AHEAD][VEC], x[AHEAD][VEC];
#pragma unroll
    for (int s = 0; s < AHEAD; ++s) {
      if (t0 + s < n) {
        load<VEC>(g[s], a.gate + at + s * a.channels);
        load<VEC>(x[s], a.x + at + s * a.channels);
      }
    }
#pragma unroll
    for (int s = 0; s < AHEAD; ++s, at += a.channels) {
      if (t0 + s >= a.time) break;
      if (t0 + s < n) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          if (SIGMOID) {
            float rest;
            sigmoid_pair(g[s][j], g[s][j], rest);
            x[s][j] *= rest;
          }
          h[j] = fmaf(g[s][j], h[j], x[s][j]);
        }
      }
      store<VEC>(a.h + at, h);
    }
  }
  if (a.state) store<VEC>(a.state + i, h);
}

template <int VEC, int AHEAD, bool SIGMOID>
__global__ void __launch_bounds__(256) walk_backward_kernel(Args a) {
  const int64_t i = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * VEC;
  if (i >= a.batch * a.channels) return;
  const int64_t b = a.batch == 1 ? 0 : i / a.channels, n = length_of(a, b);
  float c[VEC];
  start_of<VEC>(c, a.dstate, i);
  int64_t at = b * (a.time - 1) * a.channels + i + (a.time - 1) * a.channels;
  for (int64_t t0 = a.time - 1; t0 >= 0; t0 -= AHEAD) {
    float gate[AHEAD][VEC], dh[AHEAD][VEC], before[AHEAD][VEC], x[AHEAD][VEC];
#pragma unroll
    for (int s = 0; s < AHEAD; ++s) {
      const int64_t t = t0 - s, here = at - s * a.channels;
      if (t < 0) break;
      load<VEC>(dh[s], a.dh + here);
      if (t < n) {
        load<VEC>(gate[s], a.gate + here);
        if (t) load<VEC>(before[s], a.hs + here - a.channels);
        else start_of<VEC>(before[s], a.initial, i);
        if (SIGMOID) load<VEC>(x[s], a.x + here);
      }
    }
#pragma unroll
    for (int s = 0; s < AHEAD; ++s, at -= a.channels) {
      if (t0 - s < 0) break;
      float dgate[VEC], dx[VEC];
      backward_step<VEC, SIGMOID>(gate[s], dh[s], before[s], x[s], t0 - s < n, c, dgate, dx);
      store<VEC>(a.dgate + at, dgate);
      store<VEC>(a.dx + at, dx);
    }
  }
  if (a.dinitial) store<VEC>(a.dinitial + i, c);
}

// --------------------------------------------------------- scan over parts of the time
// A sequence of one batch entry and 32 channels (a chain) is cut into chunks of kChunk steps,
// which blocks take one at a time. Memory is read once and written once: a chunk's rows of
// 128 bytes come into shared memory (cp.async) while the block works on earlier chunks. With
// VEC = 4, 8 lanes hold a row, so that a warp's lanes form 4 groups; with VEC = 1 all 32 do.
// Each group of each warp takes kSteps steps of its own. A part's effect on a state is (A, B):
// the product of its gates and its last state from zero. The groups' parts meet by shuffles,
// the warps' in shared memory and the chunks' in the workspace, as records: a block publishes
// its chunk's (A, B), walks back over its chain's published parts to the nearest chunk whose
// last state is known, advances that state through the parts between, and publishes its own
// (the method of Merrill and Garland, "Single-pass parallel prefix scan with decoupled
// look-back", 2016).
// Blocks stay on their SM and take chunks in order of a ticket, each in the order it got
// them, so what a block waits for has always begun; the waits are bounded all the same.
//
// The state that enters a chunk is always the previous chunk's entering state advanced by
// that chunk's (A, B), whether a published state or the parts themselves bring it: the
// result does not depend on the order in which blocks run.
//
// Backward the same scan runs from the last step to the first, on c_t = a_t (c_(t+1) + dh_t).
constexpr int kWide = 32;   // channels of a chain
constexpr int kChunk = 128;

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

// Nothing is known at the start, and the ticket after the last record is 0.
__global__ void __launch_bounds__(256) clear_records_kernel(uint4* records, int64_t count) {
  dependents_may_launch();
  const int64_t stride = static_cast<int64_t>(gridDim.x) * 256;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < count; i += stride)
    records[i] = make_uint4(0, 0, 0, 0);
}

// The state that enters chunk `chunk` > 0 of a chain, a lane to a channel; `start` is the
// sequence's, `mine` the lane's record of the chunk. Looks at kLook chunks at a time: some 296
// blocks are on their way at once, so that a chain of [1, 65536, 1024], one of 32, has nine
// open chunks (4: 144 us, 8: 140 us, 16: 171 us, whose registers spill).
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

// A chunk as its block sees it; steps are numbered in the scan's own order.
struct Tile {
  int64_t at;           // of its first step and channel in the arrays
  int64_t edge;         // of its first channel in the states
  int channels, steps;  // that exist, of kWide and kChunk; no channels: there is no such chunk
  int from, to;         // steps that the sequence has
  unsigned row, chunk;  // its records; its place in the chain
  int ends, last;       // the sequence ends in it, before time does; no chunk comes after it
};

// The chunk that a ticket names; WHOLE: the block's chunk number i, where it takes whole
// chains, chunk after chunk.
template <bool BACK, bool WHOLE>
__device__ Tile tile_of(const Args& a, const Scan& sc, unsigned i) {
  Tile m = {};
  unsigned chain;
  if (WHOLE) {
    const unsigned turn = i / sc.chunks;
    m.chunk = i - turn * sc.chunks;
    chain = blockIdx.x + turn * gridDim.x;
    if (chain >= sc.chains) return m;
  } else {
    if (i >= sc.tiles) return m;
    m.chunk = i / sc.chains;
    chain = i - m.chunk * sc.chains;
  }
  const unsigned b = chain / sc.blocks, block = chain - b * sc.blocks;
  const int64_t n = length_of(a, b), opens = static_cast<int64_t>(m.chunk) * kChunk;
  const int64_t c = static_cast<int64_t>(block) * kWide;
  auto local = [&](int64_t v) {
    return static_cast<int>(max(min(v - opens, static_cast<int64_t>(kChunk)), static_cast<int64_t>(0)));
  };
  m.at = (b * a.time + (BACK ? a.time - 1 - opens : opens)) * a.channels + c;
  m.edge = b * a.channels + c;
  m.channels = static_cast<int>(min(a.channels - c, static_cast<int64_t>(kWide)));
  m.steps = local(a.time);
  m.from = BACK ? local(a.time - n) : 0;
  m.to = BACK ? m.steps : local(n);
  m.row = chain * sc.chunks + m.chunk;
  m.ends = !BACK && n < a.time && n > opens && n <= opens + kChunk;
  m.last = m.chunk + 1 == sc.chunks;
  return m;
}

// A thread's rows of an array of a chunk in shared memory. VEC = 4: each thread copies and
// reads places of its own (16 bytes of a row). VEC = 1 and SHIFTED: rows start at any element
// of an aligned array, so a warp copies the 16-byte words that hold its rows, 9 to a row, and a
// lane reads its channel at the row's own distance (shift) from the first word's start, which is
// the same in every array. VEC = 1 alone: arrays at any address, copied element by element (an
// instruction that copies 4 bytes a lane takes the load unit some 30 cycles: only where needed;
// one element off the alignment [2, 16384, 2048] takes 226 to 243 us forward and 285 to 357 backward).
template <int VEC, bool SHIFTED>
struct Rows {
  static constexpr int kWarps = VEC == 4 ? 4 : 8;           // that work on a chunk
  static constexpr int kSteps = kChunk / (kWarps * VEC);    // of one group
  static constexpr int kGroup = 32 / VEC;                   // lanes of a group
  static constexpr int kNext = SHIFTED ? 36 : 32 * VEC;     // floats from one step's place to the next one's
  static constexpr int kArray = kWarps * kSteps * kNext;    // floats of an array
  static_assert(kWarps * VEC * kSteps == kChunk, "");
  int lane, warp, column, mine;  // its first channel within the chain, its first step of the chunk
  float* place;                  // its first place in the first array

  __device__ explicit Rows(float* stage) {
    lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    column = (lane % kGroup) * VEC;
    mine = (warp * VEC + lane / kGroup) * kSteps;
    place = stage + warp * kSteps * kNext + (SHIFTED ? 0 : lane * VEC);
  }
  __device__ int group() const { return lane / kGroup; }

  // Copies steps [from, to) of `channels` channels; `row` points at the chunk's first channel
  // and step, `all` at the array of `count` elements, and a step is `stride` elements. Places
  // of steps outside become 0.
  __device__ __forceinline__ void copy(int array, const float* all, int64_t count, const float* row, int64_t stride,
                                       int channels, int from, int to) const {
    uint32_t dst = ptx::smem_u32(place + array * kArray);
    if constexpr (!SHIFTED) {
      const float* p = row + mine * stride + column;
      if (column < channels && mine >= from && mine + kSteps <= to) {
#pragma unroll
        for (int s = 0; s < kSteps; ++s, p += stride) {
          if constexpr (VEC == 4)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + 4 * s * kNext), "l"(p) : "memory");
          else
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst + 4 * s * kNext), "l"(p) : "memory");
        }
      } else {
#pragma unroll
        for (int s = 0; s < kSteps; ++s, p += stride) {
          const bool in = column < channels && mine + s >= from && mine + s < to;
          if constexpr (VEC == 4)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + 4 * s * kNext), "l"(in ? p : all),
                         "r"(in ? 16 : 0)
                         : "memory");
          else
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst + 4 * s * kNext), "l"(in ? p : all),
                         "r"(in ? 4 : 0)
                         : "memory");
        }
      }
    } else {
      if (lane >= 27) return;  // 9 lanes to a row, 3 rows at a time
      const int third = lane / 9, q4 = 4 * (lane - 9 * third);
      const float* start = row + (mine + third) * stride;
      dst += 4 * (third * kNext + q4);
      const int64_t on = all + count - row;  // the array goes on for so many elements
      if (channels == kWide && mine >= from && mine + kSteps <= to &&
          on > (kChunk + 1) * max(stride, static_cast<int64_t>(0)) + 64) {  // every row is there, with all its words
#pragma unroll
        for (int k = 0; k < kSteps; k += 3, start += 3 * stride) {
          const int reach = q4 - (static_cast<int>(reinterpret_cast<uintptr_t>(start) >> 2) & 3);
          if (reach < kWide && k + third < kSteps)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + 4 * k * kNext), "l"(start + reach)
                         : "memory");
        }
      } else {
#pragma unroll 1
        for (int k = 0; k + third < kSteps; k += 3, start += 3 * stride) {
          const int step = mine + k + third;
          const int reach = q4 - (static_cast<int>(reinterpret_cast<uintptr_t>(start) >> 2) & 3);
          const bool in = step >= from && step < to && reach < channels;
          const float* const word = in ? start + reach : all;
          const int bytes = in ? 4 * static_cast<int>(min(all + count - word, static_cast<int64_t>(4))) : 0;
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + 4 * k * kNext), "l"(word), "r"(bytes)
                       : "memory");
        }
      }
    }
  }
  // The shift of this thread's first step, and of the next one; rows of all arrays have it.
  __device__ __forceinline__ int shift(int64_t at, int64_t stride) const {
    return SHIFTED ? static_cast<int>(at + mine * stride) & 3 : 0;
  }
  __device__ __forceinline__ float* at(int array, int s, int shift) const {
    return place + array * kArray + s * kNext + (SHIFTED ? shift + lane : 0);
  }
  // The copies of this thread's warp, all but the last N groups, are there.
  template <int N>
  __device__ __forceinline__ void arrived() const {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
    if (SHIFTED) __syncwarp();
  }
  // Its places may be copied into again.
  __device__ __forceinline__ void done() const {
    if (SHIFTED) __syncwarp();
  }
};

// Joins the groups' parts of a warp: (A, B) becomes the effect of the groups up to this one,
// (eA, eB) that of the groups before it; the last group writes the warp's to `part`.
template <int VEC>
__device__ __forceinline__ void join_groups(float (&A)[VEC], float (&B)[VEC], float (&eA)[VEC], float (&eB)[VEC],
                                            int group, int column, float (*part)[kWide]) {
  constexpr int kGroup = 32 / VEC;
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
#pragma unroll
    for (int off = 1; off < VEC; off *= 2) {
      const float pa = __shfl_up_sync(0xffffffffu, A[i], off * kGroup);
      const float pb = __shfl_up_sync(0xffffffffu, B[i], off * kGroup);
      if (group >= off) {
        B[i] = fmaf(A[i], pb, B[i]);
        A[i] *= pa;
      }
    }
    eA[i] = eB[i] = 0.0f;
    if (VEC > 1) {
      eA[i] = __shfl_up_sync(0xffffffffu, A[i], kGroup);
      eB[i] = __shfl_up_sync(0xffffffffu, B[i], kGroup);
    }
    if (group == VEC - 1) part[0][column + i] = A[i], part[1][column + i] = B[i];
  }
}

// The state that enters this thread's steps, from the one that enters its warp's.
template <int VEC>
__device__ __forceinline__ void enter_group(float (&h)[VEC], const float* entry, const float (&eA)[VEC],
                                            const float (&eB)[VEC], int group, int column) {
  load_shared<VEC>(h, entry + column);
  if (group > 0) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) h[i] = advance(h[i], eA[i], eB[i]);
  }
}

// ---------------------------------------------------------------- the forward scan
// kWarps warps make the parts of chunk i + 1 and then write the states of chunk i, while two
// more warps publish the parts (the teller) and bring the state that enters a chunk (the
// carrier): the walk back does not stand between a chunk's loads and its stores. The values
// wait in shared memory between their two uses. A block that takes whole chains (WHOLE) has
// the entering state from its own last chunk, and there are no records.
//
// What a chunk waits for bounds this kernel, not its bandwidth alone: with the walk back in
// the working warps [1, 65536, 1024] took 188 us, with a carrier 171, and with parts that the
// teller publishes a chunk ahead 140. Three chunks' places (96 KiB) and two blocks to an SM;
// eight warps on chunks of 256 steps and one block took 134 us there but 144 against 136 at
// [1, 32768, 2048] and 152 against 133 at [4, 8192, 2048].
template <int VEC, bool SHIFTED>
struct Forward {
  static constexpr int kRing = 3, kPerSm = 2, kThreads = (Rows<VEC, SHIFTED>::kWarps + 2) * 32;
  static constexpr int kBytes = kRing * 2 * Rows<VEC, SHIFTED>::kArray * 4;  // gate, x
};

// Barriers of the working warps with the teller and with the carrier, and of those two; two
// of a kind go by the chunk's parity.
enum { kPartsMade = 1, kEntryKnown = 3, kEndKnown = 5, kEndTold = 6, kPartsTold = 7 };
__device__ __forceinline__ void meet(int barrier, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(barrier), "r"(threads) : "memory");
}
__device__ __forceinline__ void signal(int barrier, int threads) {
  asm volatile("bar.arrive %0, %1;" ::"r"(barrier), "r"(threads) : "memory");
}

template <int VEC, bool SHIFTED, bool SIGMOID, bool WHOLE>
__global__ void __launch_bounds__(Forward<VEC, SHIFTED>::kThreads, Forward<VEC, SHIFTED>::kPerSm)
scan_forward_kernel(Args a, Scan sc, int* err) {
  using R = Rows<VEC, SHIFTED>;
  constexpr int kRing = Forward<VEC, SHIFTED>::kRing, kSteps = R::kSteps, kWarps = R::kWarps;
  constexpr int kAll = (kWarps + 1) * 32;  // the warps that work, and one of the two others
  extern __shared__ __align__(16) float stage[];
  // The warps' parts. The teller puts the whole chunk's in the place of the last warp's, which
  // nothing else needs; the carrier puts the state that enters a warp's steps in that of A.
  __shared__ __align__(16) float parts[2][kWarps][2][kWide], ended[kWide];
  // Chunk i's at i % 8. The carrier sets i's in its turn i - kRing, before it signals that
  // turn's entry. The warps that work see that signal before they make chunk i - 1's parts
  // (kRing >= 3), and the teller reads i's after those were made; the slots in use at a time
  // are those from one chunk behind the carrier's to kRing beyond it.
  __shared__ Tile line[8];
  static_assert(kRing >= 3 && kRing + 3 <= 8, "a chunk's line is set before it is read, and kept until it is done");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;

  if (!WHOLE) wait_for_prior_grid();  // the records are clear

  if (warp == kWarps + 1) {  // the teller
    for (int k = 0; k < kRing; ++k) __syncthreads();
    for (unsigned i = 0;; ++i) {
      const Tile& m = line[i & 7];
      if (m.channels == 0) return;
      meet(kPartsMade + (i & 1), kAll);
      float (*const part)[2][kWide] = parts[i & 1];
      float A = 1.0f, B = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        B = fmaf(part[w][0][lane], B, part[w][1][lane]);
        A *= part[w][0][lane];
      }
      part[kWarps - 1][0][lane] = A;
      part[kWarps - 1][1][lane] = B;
      if (!WHOLE && m.chunk > 0 && !m.last && !m.ends)
        put(sc.records + static_cast<int64_t>(m.row) * kWide + lane, A, B, 0.0f, 1u);
      signal(kPartsTold + (i & 1), 64);
    }
  }
  if (warp == kWarps) {  // the carrier
    for (int k = 0; k < kRing; ++k) {
      if (lane == 0) line[k] = tile_of<false, WHOLE>(a, sc, WHOLE ? k : atomicAdd(sc.ticket, 1u));
      __syncthreads();
    }
    float state = 0.0f;
    bool ended_before = false;
    for (unsigned i = 0;; ++i) {
      const Tile m = line[i & 7];
      if (m.channels == 0) return;
      if (lane == 0)
        line[(i + kRing) & 7] = tile_of<false, WHOLE>(a, sc, WHOLE ? i + kRing : atomicAdd(sc.ticket, 1u));
      const float start = a.initial && lane < m.channels ? __ldg(a.initial + m.edge + lane) : 0.0f;
      meet(kPartsTold + (i & 1), 64);
      float (*const part)[2][kWide] = parts[i & 1];
      const float A = part[kWarps - 1][0][lane], B = part[kWarps - 1][1][lane];
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
        const float before = h;
        h = advance(h, part[w][0][lane], part[w][1][lane]);
        part[w][0][lane] = before;
      }
      state = advance(state, A, B);
      __syncwarp();
      signal(kEntryKnown + (i & 1), kAll);
    }
  }

  const R rows(stage);
  const int group = rows.group(), column = rows.column, mine = rows.mine;
  const int64_t count = a.batch * a.time * a.channels;
  const int turn_by = static_cast<int>(a.channels & 3);

  auto fetch = [&](unsigned i) {
    const Tile& m = line[i & 7];
    if (m.channels) {
      const int first = 2 * (i % kRing);  // array
      rows.copy(first, a.gate, count, a.gate + m.at, a.channels, m.channels, m.from, m.to);
      rows.copy(first + 1, a.x, count, a.x + m.at, a.channels, m.channels, m.from, m.to);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  // The parts of chunk i; the effect of the groups before this one into (eA, eB).
  auto make = [&](unsigned i, float (&eA)[VEC], float (&eB)[VEC]) {
    const Tile& m = line[i & 7];
    const int first = 2 * (i % kRing), live = m.to - mine;
    int shift = rows.shift(m.at, a.channels);
    float A[VEC], B[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) A[j] = 1.0f, B[j] = 0.0f;
#pragma unroll 8
    for (int s = 0; s < kSteps; ++s, shift = (shift + turn_by) & 3) {
      float* const gp = rows.at(first, s, shift);
      float* const xp = rows.at(first + 1, s, shift);
      float g[VEC], v[VEC];
      load_shared<VEC>(g, gp);
      load_shared<VEC>(v, xp);
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
        store_shared<VEC>(gp, g);
        store_shared<VEC>(xp, v);
      }
    }
    join_groups<VEC>(A, B, eA, eB, group, column, parts[i & 1][warp]);
    signal(kPartsMade + (i & 1), kAll);
  };

#pragma unroll
  for (int k = 0; k < kRing; ++k) {
    __syncthreads();
    fetch(k);
  }
  float eA[VEC], eB[VEC], nA[VEC], nB[VEC];
  if (line[0].channels) {
    rows.template arrived<kRing - 1>();
    make(0, eA, eB);
  }
  for (unsigned i = 0; line[i & 7].channels; ++i) {
    rows.template arrived<kRing - 2>();
    if (line[(i + 1) & 7].channels) make(i + 1, nA, nB);
    const Tile& m = line[i & 7];
    meet(kEntryKnown + (i & 1), kAll);
    float h[VEC];
    enter_group<VEC>(h, parts[i & 1][warp][0], eA, eB, group, column);
    const int first = 2 * (i % kRing);
    const bool inside = column < m.channels;
    auto write = [&](bool whole) {
      float* p = a.h + m.at + mine * a.channels + column;
      int shift = rows.shift(m.at, a.channels);
#pragma unroll 8
      for (int s = 0; s < kSteps; ++s, p += a.channels, shift = (shift + turn_by) & 3) {
        float g[VEC], v[VEC];
        load_shared<VEC>(g, rows.at(first, s, shift));
        load_shared<VEC>(v, rows.at(first + 1, s, shift));
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          if (!SIGMOID && !whole && mine + s >= m.to) g[j] = 1.0f;
          h[j] = fmaf(g[j], h[j], v[j]);
        }
        if (whole || (inside && mine + s < m.steps)) store<VEC>(p, h);
      }
    };
    if (inside && mine + kSteps <= m.to) {
      write(true);
    } else if (!(m.ends && mine >= m.to)) {
      write(false);
    }
    if (m.ends) {
      // what is held after the end is the state itself, not one advanced by (A, B): this
      // chunk publishes that state alone
      if (m.to > mine && m.to <= mine + kSteps) {  // the group that has the last step
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          ended[column + j] = h[j];
          if (!WHOLE && !m.last)
            put(sc.records + static_cast<int64_t>(m.row) * kWide + column + j, 1.0f, 0.0f, h[j], 2u);
        }
      }
      meet(kEndKnown, kWarps * 32);
      if (WHOLE && !m.last) signal(kEndTold, kAll);
      if (mine >= m.to) {
        load_shared<VEC>(h, ended + column);
        write(false);
      }
    }
    if (a.state && inside && m.last && mine < m.steps && mine + kSteps >= m.steps)
      store<VEC>(a.state + m.edge + column, h);
    rows.done();
    fetch(i + kRing);
#pragma unroll
    for (int j = 0; j < VEC; ++j) eA[j] = nA[j], eB[j] = nB[j];
  }
}

// --------------------------------------------------------------- the backward scan
// A chunk is twice the forward one's bytes, so three blocks to an SM hide each other's walk
// back: gate and dh go into registers for the parts, their places take the next chunk's, and
// the state before each step and x are read when the entering gradient is known. Four warps of
// 32 values a thread; eight warps of 16 spilled at three blocks ([2, 16384, 2048] 366 us).
template <int VEC, bool SHIFTED, bool SIGMOID>
struct Backward {
  static constexpr int kPerSm = VEC == 4 ? 3 : 2, kThreads = Rows<VEC, SHIFTED>::kWarps * 32;
  static constexpr int kBytes = (SIGMOID ? 4 : 3) * Rows<VEC, SHIFTED>::kArray * 4;  // gate, dh, the state before, x
};

template <int VEC, bool SHIFTED, bool SIGMOID>
__global__ void __launch_bounds__(Backward<VEC, SHIFTED, SIGMOID>::kThreads, Backward<VEC, SHIFTED, SIGMOID>::kPerSm)
scan_backward_kernel(Args a, Scan sc, int* err) {
  using R = Rows<VEC, SHIFTED>;
  constexpr int kSteps = R::kSteps, kWarps = R::kWarps;
  extern __shared__ __align__(16) float stage[];
  __shared__ float parts[kWarps][2][kWide];
  __shared__ __align__(16) float entries[kWarps][kWide];
  __shared__ Tile line[2];  // this chunk and the next one, by the turn's parity
  const R rows(stage);
  const int lane = rows.lane, warp = rows.warp, group = rows.group(), column = rows.column, mine = rows.mine;
  const int64_t count = a.batch * a.time * a.channels, stride = -a.channels;
  const int turn_by = static_cast<int>(stride & 3);

  auto fetch = [&](const Tile& m) {
    if (m.channels) {
      rows.copy(0, a.gate, count, a.gate + m.at, stride, m.channels, m.from, m.to);
      rows.copy(1, a.dh, count, a.dh + m.at, stride, m.channels, 0, m.steps);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  auto fetch_rest = [&](const Tile& m) {
    if (m.channels) {
      // the first step of all has no state before it in h
      rows.copy(2, a.hs, count, a.hs + m.at - a.channels, stride, m.channels, m.from, m.last ? m.to - 1 : m.to);
      if (SIGMOID) rows.copy(3, a.x, count, a.x + m.at, stride, m.channels, m.from, m.to);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };

  wait_for_prior_grid();  // the records are clear
  if (threadIdx.x == 0) line[0] = tile_of<true, false>(a, sc, atomicAdd(sc.ticket, 1u));
  __syncthreads();
  fetch(line[0]);
  fetch_rest(line[0]);
  unsigned later = threadIdx.x == 0 ? atomicAdd(sc.ticket, 1u) : 0;
  for (unsigned turn = 0; line[turn & 1].channels; ++turn) {
    const Tile m = line[turn & 1];
    const Tile& next = line[(turn + 1) & 1];
    if (threadIdx.x == 0) line[(turn + 1) & 1] = tile_of<true, false>(a, sc, later);
    const int opening = rows.shift(m.at, stride);
    rows.template arrived<1>();
    float g[kSteps][VEC], v[kSteps][VEC], A[VEC], B[VEC];  // gate and dh
#pragma unroll
    for (int i = 0; i < VEC; ++i) A[i] = 1.0f, B[i] = 0.0f;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int shift = (opening + s * turn_by) & 3;
      load_shared<VEC>(g[s], rows.at(0, s, shift));
      load_shared<VEC>(v[s], rows.at(1, s, shift));
      const bool live = mine + s >= m.from && mine + s < m.to;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        float s1 = g[s][i], rest;
        if (SIGMOID) sigmoid_pair(s1, s1, rest);
        if (!live) s1 = 1.0f;
        A[i] *= s1;
        B[i] = s1 * (B[i] + v[s][i]);
      }
    }
    float eA[VEC], eB[VEC];
    join_groups<VEC>(A, B, eA, eB, group, column, parts[warp]);
    __syncthreads();
    if (warp != 0) fetch(next);
    if (warp == 0) {  // a lane to a channel
      Record* const record = sc.records + static_cast<int64_t>(m.row) * kWide + lane;
      const float start = a.dstate && lane < m.channels ? __ldg(a.dstate + m.edge + lane) : 0.0f;
      float wA = 1.0f, wB = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        wB = fmaf(parts[w][0][lane], wB, parts[w][1][lane]);
        wA *= parts[w][0][lane];
      }
      float state = start;
      if (m.chunk > 0) {
        if (!m.last) put(record, wA, wB, 0.0f, 1u);
        fetch(next);
        state = enter(record, static_cast<int>(m.chunk), start, lane, err);
      } else {
        fetch(next);
      }
      if (!m.last) put(record, wA, wB, advance(state, wA, wB), 2u);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        entries[w][lane] = state;
        state = advance(state, parts[w][0][lane], parts[w][1][lane]);
      }
    }
    if (threadIdx.x == 0) later = atomicAdd(sc.ticket, 1u);
    __syncthreads();
    float c[VEC];
    enter_group<VEC>(c, entries[warp], eA, eB, group, column);
    rows.template arrived<1>();
    float *p = a.dgate + m.at + mine * stride + column, *q = a.dx + m.at + mine * stride + column;
#pragma unroll
    for (int s = 0; s < kSteps; ++s, p += stride, q += stride) {
      if (column >= m.channels || mine + s >= m.steps) continue;
      float before[VEC], x[VEC] = {}, dgate[VEC], dx[VEC];
      load_shared<VEC>(before, rows.at(2, s, (opening + (s + 1) * turn_by) & 3));  // the row before
      if (m.last && mine + s + 1 == m.steps) start_of<VEC>(before, a.initial, m.edge + column);
      if (SIGMOID) load_shared<VEC>(x, rows.at(3, s, (opening + s * turn_by) & 3));
      backward_step<VEC, SIGMOID>(g[s], v[s], before, x, mine + s >= m.from, c, dgate, dx);
      store<VEC>(p, dgate);
      store<VEC>(q, dx);
    }
    if (a.dinitial && column < m.channels && m.last && mine < m.steps && mine + kSteps >= m.steps)
      store<VEC>(a.dinitial + m.edge + column, c);
    rows.done();
    fetch_rest(next);
  }
}

// ------------------------------------------------------------------------- launches
bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Every buffer starts on a 16-byte word.
bool all_aligned(const Args& a) {
  const void* all[] = {a.gate, a.x, a.initial, a.h, a.state, a.dh, a.hs, a.dstate, a.dgate, a.dx, a.dinitial};
  bool fits = true;
  for (const void* p : all) fits = fits && aligned(p);
  return fits;
}

// Threads walk through time alone where there are few steps, and up to a chunk of them where
// the channels fill the machine, or as much less of it as the chunk is emptier: one that is
// mostly empty costs its block as much as a full one. [64, 32, 4096]: walk 24 us, scan 62;
// [64, 32, 1024] 16 and 20; [32, 64, 4096] 31 and 35; [256, 100, 1024] 56 both; [32, 100, 4096]
// 43 and 37; [16, 64, 1024], whose 4096 threads fill nothing, 21 and 11.
constexpr int64_t kWalkSteps = 16;
template <int VEC>
bool walks(const Args& a) {
  return a.time <= kWalkSteps || (a.time <= kChunk && a.batch * a.channels * (kChunk / a.time) >= 256 * VEC * sm_count());
}

// Whole chains to a block, where the last of their rounds leaves few blocks idle: [16, 512,
// 4096], 2048 chains, takes 70 us so and 83 with records. At four fifths of the places in use
// the rounds lose as much as the records cost.
bool takes_whole(int64_t chains, int64_t blocks) { return chains * 10 >= ceil_div(chains, blocks) * blocks * 8; }

template <auto kKernel>
int launch_scan(cudaStream_t s, const Args& a, int threads, int bytes, int per_sm, bool whole, void* workspace) {
  const int64_t blocks = ceil_div(a.channels, kWide), chunks = ceil_div(a.time, kChunk);
  const int64_t tiles = a.batch * blocks * chunks;
  if (tiles > INT32_MAX) return invalid("recurrence is too large for one call");
  Scan sc;
  sc.blocks = static_cast<unsigned>(blocks);
  sc.chains = static_cast<unsigned>(a.batch * blocks);
  sc.chunks = static_cast<unsigned>(chunks);
  sc.tiles = static_cast<unsigned>(tiles);
  sc.records = whole ? nullptr : static_cast<Record*>(workspace);
  sc.ticket = whole ? nullptr : reinterpret_cast<unsigned*>(sc.records + tiles * kWide);
  static std::atomic<bool> attr_done[64];  // host threads may meet here
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !attr_done[dev].load(std::memory_order_relaxed)) {
    if (cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess)
      return launch_status("recurrence shared memory attribute");
    if (dev >= 0 && dev < 64) attr_done[dev].store(true, std::memory_order_relaxed);
  }
  const dim3 grid(static_cast<unsigned>(std::min<int64_t>(whole ? sc.chains : tiles, per_sm * sm_count())));
  if (whole) {
    kKernel<<<grid, threads, bytes, s>>>(a, sc, device_error_word());
  } else {
    const int64_t records = tiles * kWide + 1;
    const unsigned clears = static_cast<unsigned>(std::min<int64_t>(ceil_div(records, 256), 8 * sm_count()));
    clear_records_kernel<<<clears, 256, 0, s>>>(reinterpret_cast<uint4*>(workspace), records);
    launch_after(kKernel, grid, dim3(threads), s, bytes, a, sc, device_error_word());
  }
  return launch_status("recurrence");
}

template <int VEC, bool SHIFTED, bool SIGMOID>
int launch_forward(cudaStream_t s, const Args& a, void* workspace) {
  if (walks<VEC>(a)) {
    TimedLaunch timer("recurrence_walk", s);
    auto* kernel = a.time == 1 ? walk_forward_kernel<VEC, 1, SIGMOID> : walk_forward_kernel<VEC, kAhead<VEC>, SIGMOID>;
    kernel<<<static_cast<unsigned>(ceil_div(a.batch * a.channels, 256 * VEC)), 256, 0, s>>>(a);
    return launch_status("recurrence");
  }
  using F = Forward<VEC, SHIFTED>;
  TimedLaunch timer("recurrence_scan", s);
  const bool whole = takes_whole(a.batch * ceil_div(a.channels, kWide), F::kPerSm * sm_count());
  if (whole)
    return launch_scan<scan_forward_kernel<VEC, SHIFTED, SIGMOID, true>>(s, a, F::kThreads, F::kBytes, F::kPerSm, true,
                                                                         nullptr);
  return launch_scan<scan_forward_kernel<VEC, SHIFTED, SIGMOID, false>>(s, a, F::kThreads, F::kBytes, F::kPerSm, false,
                                                                        workspace);
}

template <int VEC, bool SHIFTED, bool SIGMOID>
int launch_backward(cudaStream_t s, const Args& a, void* workspace) {
  if (walks<VEC>(a)) {
    TimedLaunch timer("recurrence_walk_backward", s);
    auto* kernel = a.time == 1 ? walk_backward_kernel<VEC, 1, SIGMOID> : walk_backward_kernel<VEC, kAhead<VEC>, SIGMOID>;
    kernel<<<static_cast<unsigned>(ceil_div(a.batch * a.channels, 256 * VEC)), 256, 0, s>>>(a);
    return launch_status("recurrence");
  }
  using K = Backward<VEC, SHIFTED, SIGMOID>;
  TimedLaunch timer("recurrence_scan_backward", s);
  return launch_scan<scan_backward_kernel<VEC, SHIFTED, SIGMOID>>(s, a, K::kThreads, K::kBytes, K::kPerSm, false,
                                                                  workspace);
}

// One step of whole sequences: the batch's channels lie in a row, as one sequence's do. Then no
// thread divides by the channels, and rows of any length are words ([1024, 1, 4097]: 31 us and
// 18 forward, 41 and 27 backward).
Args one_row(Args a) {
  if (a.time == 1 && !a.lengths) a.channels *= a.batch, a.batch = 1;
  return a;
}

template <bool SIGMOID>
int launch_forward(cudaStream_t s, const Args& a, void* workspace) {
  if (!all_aligned(a)) return launch_forward<1, false, SIGMOID>(s, a, workspace);
  if (a.channels % 4) return launch_forward<1, true, SIGMOID>(s, a, workspace);
  return launch_forward<4, false, SIGMOID>(s, a, workspace);
}

template <bool SIGMOID>
int launch_backward(cudaStream_t s, const Args& a, void* workspace) {
  if (!all_aligned(a)) return launch_backward<1, false, SIGMOID>(s, a, workspace);
  if (a.channels % 4) return launch_backward<1, true, SIGMOID>(s, a, workspace);
  return launch_backward<4, false, SIGMOID>(s, a, workspace);
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
  // a record per channel for each chunk, and the ticket in one more's place
  const int64_t tiles = batch * ceil_div(channels, kWide) * ceil_div(time, kChunk);
  return (static_cast<size_t>(tiles) * kWide + 1) * sizeof(Record);
}

static int check_workspace(int64_t batch, int64_t time, int64_t channels, const void* workspace, size_t bytes) {
  const size_t need = tcx_sm100_recurrence_workspace_bytes(batch, time, channels);
  if (bytes < need) return invalid("workspace too small for the recurrence");
  if (need && (!workspace || !aligned(workspace))) return invalid("the recurrence's workspace must be 16-byte aligned");
  return TCX_OK;
}

extern "C" int tcx_sm100_recurrence_forward(tcx_stream_t stream, int form, const float* gate, const float* x,
                                            const float* initial, const int32_t* lengths, float* h, float* state,
                                            int64_t batch, int64_t time, int64_t channels, void* workspace,
                                            size_t workspace_bytes) {
  clear_error();
  if (int rc = check_recurrence(form, batch, time, channels)) return rc;
  if (batch == 0 || channels == 0) return TCX_OK;
  if (time && (!gate || !x || !h)) return invalid("missing buffer");
  if (int rc = check_workspace(batch, time, channels, workspace, workspace_bytes)) return rc;
  Args a{gate, x, initial, lengths, h, state, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, batch, time,
         channels};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (time == 0) return pass_through(s, initial, state, batch * channels);
  return form == TCX_RECURRENCE_SIGMOID ? launch_forward<true>(s, one_row(a), workspace)
                                        : launch_forward<false>(s, one_row(a), workspace);
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
  if (int rc = check_workspace(batch, time, channels, workspace, workspace_bytes)) return rc;
  Args a{gate, x, initial, lengths, nullptr, nullptr, dh, h, dstate, dgate, dx, dinitial, batch, time, channels};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (time == 0) return pass_through(s, dstate, dinitial, batch * channels);
  return form == TCX_RECURRENCE_SIGMOID ? launch_backward<true>(s, one_row(a), workspace)
                                        : launch_backward<false>(s, one_row(a), workspace);
}
