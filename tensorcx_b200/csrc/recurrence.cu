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
  const float e = expf(-fabsf(z)), big = 1.0f / (1.0f + e), small = e * big;
  s = z >= 0.0f ? big : small;
  rest = z >= 0.0f ? small : big;
}

__device__ __forceinline__ int64_t length_of(const Args& a, int64_t b) {
  if (!a.lengths) return a.time;
  const int64_t n = a.lengths[b];
  return n < 0 ? 0 : n > a.time ? a.time : n;
}

template <bool SIGMOID>
__global__ void __launch_bounds__(256) recurrence_forward_kernel(Args a) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= a.batch * a.channels) return;
  const int64_t b = i / a.channels, c = i % a.channels, n = length_of(a, b);
  float h = a.initial ? a.initial[i] : 0.0f;
  int64_t at = b * a.time * a.channels + c;
  for (int64_t t = 0; t < a.time; ++t, at += a.channels) {
    if (t < n) {
      float g = a.gate[at], x = a.x[at];
      if (SIGMOID) {
        float rest;
        sigmoid_pair(g, g, rest);
        x *= rest;
      }
      h = fmaf(g, h, x);
    }
    a.h[at] = h;
  }
  if (a.state) a.state[i] = h;
}

template <bool SIGMOID>
__global__ void __launch_bounds__(256) recurrence_backward_kernel(Args a) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= a.batch * a.channels) return;
  const int64_t b = i / a.channels, c = i % a.channels, n = length_of(a, b);
  float carry = a.dstate ? a.dstate[i] : 0.0f;
  int64_t at = (b * a.time + a.time - 1) * a.channels + c;
  for (int64_t t = a.time - 1; t >= 0; --t, at -= a.channels) {
    const float g = a.dh[at] + carry;
    float dgate = 0.0f, dx = 0.0f;
    carry = g;
    if (t < n) {
      const float before = t > 0 ? a.hs[at - a.channels] : a.initial ? a.initial[i] : 0.0f;
      float s = a.gate[at], rest = 1.0f;
      if (SIGMOID) {
        sigmoid_pair(s, s, rest);
        dx = g * rest;
        dgate = dx * s * (before - a.x[at]);
      } else {
        dx = g;
        dgate = g * before;
      }
      carry = s * g;
    }
    a.dgate[at] = dgate;
    a.dx[at] = dx;
  }
  if (a.dinitial) a.dinitial[i] = carry;
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
  (void)batch, (void)time, (void)channels;
  return 0;
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
  TimedLaunch timer("recurrence_forward", s);
  const unsigned grid = static_cast<unsigned>(ceil_div(batch * channels, 256));
  if (form == TCX_RECURRENCE_SIGMOID) recurrence_forward_kernel<true><<<grid, 256, 0, s>>>(a);
  else recurrence_forward_kernel<false><<<grid, 256, 0, s>>>(a);
  return launch_status("recurrence forward");
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
  TimedLaunch timer("recurrence_backward", s);
  const unsigned grid = static_cast<unsigned>(ceil_div(batch * channels, 256));
  if (form == TCX_RECURRENCE_SIGMOID) recurrence_backward_kernel<true><<<grid, 256, 0, s>>>(a);
  else recurrence_backward_kernel<false><<<grid, 256, 0, s>>>(a);
  return launch_status("recurrence backward");
}
