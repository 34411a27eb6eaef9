// Gated linear recurrence over time, forward, backward and one step, for
// float, bfloat16 and half sequences with float32 states.
//
//   f_t = sigmoid(g_t), h_t = f_t h_{t-1} + (1 - f_t) x_t
//   lam_t = dy_t + f_{t+1} lam_{t+1} (lam beyond the end is dstate),
//   dx_t = (1 - f_t) lam_t, dg_t = lam_t (h_{t-1} - x_t) f_t (1 - f_t),
//   dh0 = f_1 lam_1
//
// A sequence of length L < T keeps its state from frame L on: its outputs
// there are 0, its gradients 0, and x and g are not read.
//
// The forward saves the state before every SCAN_CHUNK-th frame in float32;
// the backward recomputes the states inside a chunk from it, so no rounded
// output enters a gradient and the outputs are not read again.
#include "../../include/torchwarp_b200.h"
#include "element.cuh"

namespace tw {
namespace {

constexpr int SCAN_CHUNK = 32;
constexpr int SCAN_THREADS = 128;

__device__ __forceinline__ int live_len(const int64_t* lengths, int b, int T) {
  if (!lengths) return T;
  const long long n = lengths[b];
  return n < 0 ? 0 : n > T ? T : (int)n;
}

// One frame: f h + (1 - f) x as a step from the nearer of the two, so that the
// rounding of a gate near 1 does not decay a state that should last.
__device__ __forceinline__ float advance(float f, float omf, float h, float x) {
  return f >= 0.5f ? fmaf(omf, x - h, h) : fmaf(f, h - x, x);
}
// f l, likewise.
__device__ __forceinline__ float decay(float f, float omf, float l) {
  return f >= 0.5f ? fmaf(-omf, l, l) : f * l;
}

template <typename T>
__global__ void __launch_bounds__(SCAN_THREADS)
    scan_fwd_kernel(const T* __restrict__ x, size_t xb, size_t xt, const T* __restrict__ g,
                    size_t gb, size_t gt, const float* __restrict__ h0,
                    const int64_t* __restrict__ lengths, int B, int TT, int D, T* __restrict__ y,
                    float* __restrict__ state, float* __restrict__ carry) {
  const size_t id = (size_t)blockIdx.x * SCAN_THREADS + threadIdx.x;
  if (id >= (size_t)B * D) return;
  const int b = (int)(id / D), d = (int)(id - (size_t)b * D);
  const int L = live_len(lengths, b, TT), nC = (TT + SCAN_CHUNK - 1) / SCAN_CHUNK;
  float h = h0 ? h0[id] : 0.f;
  for (int t = 0; t < L; ++t) {
    if (carry && t % SCAN_CHUNK == 0) carry[((size_t)b * nC + t / SCAN_CHUNK) * D + d] = h;
    float f, omf;
    sigmoid_pair(to_f(g[b * gb + t * gt + d]), f, omf);
    h = advance(f, omf, h, to_f(x[b * xb + t * xt + d]));
    y[((size_t)b * TT + t) * D + d] = from_f<T>(h);
  }
  for (int t = L; t < TT; ++t) y[((size_t)b * TT + t) * D + d] = from_f<T>(0.f);
  state[id] = h;
}

template <typename T>
__global__ void __launch_bounds__(SCAN_THREADS)
    scan_bwd_kernel(const T* __restrict__ dy, size_t yb, size_t yt,
                    const float* __restrict__ dstate, const T* __restrict__ x, size_t xb,
                    size_t xt, const T* __restrict__ g, size_t gb, size_t gt,
                    const int64_t* __restrict__ lengths, const float* __restrict__ carry, int B,
                    int TT, int D, T* __restrict__ dx, T* __restrict__ dg,
                    float* __restrict__ dh0) {
  const size_t id = (size_t)blockIdx.x * SCAN_THREADS + threadIdx.x;
  if (id >= (size_t)B * D) return;
  const int b = (int)(id / D), d = (int)(id - (size_t)b * D);
  const int L = live_len(lengths, b, TT), nC = (TT + SCAN_CHUNK - 1) / SCAN_CHUNK;
  for (int t = L; t < TT; ++t) {
    dx[((size_t)b * TT + t) * D + d] = from_f<T>(0.f);
    dg[((size_t)b * TT + t) * D + d] = from_f<T>(0.f);
  }
  float lam = dstate ? dstate[id] : 0.f;  // f_{t+1} lam_{t+1}
  for (int c = (L + SCAN_CHUNK - 1) / SCAN_CHUNK - 1; c >= 0; --c) {
    const int t0 = c * SCAN_CHUNK, n = min(SCAN_CHUNK, L - t0);
    float hp[SCAN_CHUNK];
    float h = carry[((size_t)b * nC + c) * D + d];
    for (int k = 0; k < n; ++k) {
      hp[k] = h;
      float f, omf;
      sigmoid_pair(to_f(g[b * gb + (t0 + k) * gt + d]), f, omf);
      h = advance(f, omf, h, to_f(x[b * xb + (t0 + k) * xt + d]));
    }
    for (int k = n - 1; k >= 0; --k) {
      const int t = t0 + k;
      float f, omf;
      sigmoid_pair(to_f(g[b * gb + t * gt + d]), f, omf);
      const float l = to_f(dy[b * yb + t * yt + d]) + lam;
      dx[((size_t)b * TT + t) * D + d] = from_f<T>(omf * l);
      dg[((size_t)b * TT + t) * D + d] =
          from_f<T>(l * (hp[k] - to_f(x[b * xb + t * xt + d])) * (f * omf));
      lam = decay(f, omf, l);
    }
  }
  if (dh0) dh0[id] = lam;
}

template <typename T>
__global__ void __launch_bounds__(SCAN_THREADS)
    scan_step_kernel(const T* __restrict__ x, size_t xs, const T* __restrict__ g, size_t gs,
                     float* __restrict__ state, int B, int D, T* __restrict__ y) {
  const size_t id = (size_t)blockIdx.x * SCAN_THREADS + threadIdx.x;
  if (id >= (size_t)B * D) return;
  const size_t b = id / D, d = id - b * D;
  float f, omf;
  sigmoid_pair(to_f(g[b * gs + d]), f, omf);
  const float h = advance(f, omf, state[id], to_f(x[b * xs + d]));
  state[id] = h;
  y[id] = from_f<T>(h);
}

int check(const char* who, int B, int TT, int D) {
  if (B < 0 || TT < 0 || D <= 0)
    return set_error(kInvalid, "%s: invalid sizes B=%d T=%d D=%d (need B, T >= 0, D > 0)", who, B,
                     TT, D);
  if ((size_t)B * D / SCAN_THREADS >= 0x7fffffffu)
    return set_error(kUnsupported, "%s: B * D too large", who);
  return kOk;
}

int launched(const char* who) {
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_error(kLaunch, "%s: %s", who, cudaGetErrorString(e));
  return kOk;
}

unsigned grid_of(int B, int D) {
  return (unsigned)(((size_t)B * D + SCAN_THREADS - 1) / SCAN_THREADS);
}

template <typename T>
int fwd(const void* x, size_t xb, size_t xt, const void* g, size_t gb, size_t gt, const float* h0,
        const int64_t* lengths, int B, int TT, int D, void* y, float* state, void* carry,
        size_t carry_bytes, void* stream) {
  set_error(kOk, "%s", "");
  if (int e = check("tw_gated_scan_forward", B, TT, D)) return e;
  if (B == 0) return kOk;
  if (!state || (TT && (!x || !g || !y)))
    return set_error(kInvalid, "tw_gated_scan_forward: null pointer argument");
  if (carry && carry_bytes < tw_gated_scan_carry_bytes(B, TT, D))
    return set_error(kWorkspace, "tw_gated_scan_forward: carry needs %zu bytes",
                     tw_gated_scan_carry_bytes(B, TT, D));
  scan_fwd_kernel<T><<<grid_of(B, D), SCAN_THREADS, 0, (cudaStream_t)stream>>>(
      (const T*)x, xb, xt, (const T*)g, gb, gt, h0, lengths, B, TT, D, (T*)y, state,
      (float*)carry);
  return launched("tw_gated_scan_forward");
}

template <typename T>
int bwd(const void* dy, size_t yb, size_t yt, const float* dstate, const void* x, size_t xb,
        size_t xt, const void* g, size_t gb, size_t gt, const int64_t* lengths, const void* carry,
        size_t carry_bytes, int B, int TT, int D, void* dx, void* dg, float* dh0, void* stream) {
  set_error(kOk, "%s", "");
  if (int e = check("tw_gated_scan_backward", B, TT, D)) return e;
  if (B == 0) return kOk;
  if (TT && (!dy || !x || !g || !carry || !dx || !dg))
    return set_error(kInvalid, "tw_gated_scan_backward: null pointer argument");
  if (carry_bytes < tw_gated_scan_carry_bytes(B, TT, D))
    return set_error(kWorkspace, "tw_gated_scan_backward: carry needs %zu bytes",
                     tw_gated_scan_carry_bytes(B, TT, D));
  scan_bwd_kernel<T><<<grid_of(B, D), SCAN_THREADS, 0, (cudaStream_t)stream>>>(
      (const T*)dy, yb, yt, dstate, (const T*)x, xb, xt, (const T*)g, gb, gt, lengths,
      (const float*)carry, B, TT, D, (T*)dx, (T*)dg, dh0);
  return launched("tw_gated_scan_backward");
}

template <typename T>
int step(const void* x, size_t xs, const void* g, size_t gs, float* state, int B, int D, void* y,
         void* stream) {
  set_error(kOk, "%s", "");
  if (int e = check("tw_gated_scan_step", B, 1, D)) return e;
  if (B == 0) return kOk;
  if (!x || !g || !state || !y)
    return set_error(kInvalid, "tw_gated_scan_step: null pointer argument");
  scan_step_kernel<T><<<grid_of(B, D), SCAN_THREADS, 0, (cudaStream_t)stream>>>(
      (const T*)x, xs, (const T*)g, gs, state, B, D, (T*)y);
  return launched("tw_gated_scan_step");
}

}  // namespace
}  // namespace tw

extern "C" {

size_t tw_gated_scan_carry_bytes(int B, int T, int D) {
  if (B <= 0 || T <= 0 || D <= 0) return 0;
  return (size_t)B * ((T + tw::SCAN_CHUNK - 1) / tw::SCAN_CHUNK) * D * sizeof(float);
}

#define TW_GATED_SCAN(SUFFIX, E)                                                                 \
  int tw_gated_scan_forward_##SUFFIX(                                                            \
      const void* x, size_t x_batch, size_t x_time, const void* gate, size_t g_batch,            \
      size_t g_time, const float* h0, const int64_t* lengths, int B, int T, int D, void* y,      \
      float* state, void* carry, size_t carry_bytes, void* stream) {                             \
    return tw::fwd<E>(x, x_batch, x_time, gate, g_batch, g_time, h0, lengths, B, T, D, y, state, \
                      carry, carry_bytes, stream);                                               \
  }                                                                                              \
  int tw_gated_scan_backward_##SUFFIX(                                                           \
      const void* dy, size_t dy_batch, size_t dy_time, const float* dstate, const void* x,       \
      size_t x_batch, size_t x_time, const void* gate, size_t g_batch, size_t g_time,            \
      const int64_t* lengths, const void* carry, size_t carry_bytes, int B, int T, int D,        \
      void* dx, void* dgate, float* dh0, void* stream) {                                         \
    return tw::bwd<E>(dy, dy_batch, dy_time, dstate, x, x_batch, x_time, gate, g_batch, g_time,  \
                      lengths, carry, carry_bytes, B, T, D, dx, dgate, dh0, stream);             \
  }                                                                                              \
  int tw_gated_scan_step_##SUFFIX(const void* x, size_t x_batch, const void* gate,               \
                                  size_t g_batch, float* state, int B, int D, void* y,           \
                                  void* stream) {                                                \
    return tw::step<E>(x, x_batch, gate, g_batch, state, B, D, y, stream);                       \
  }

TW_GATED_SCAN(f32, float)
TW_GATED_SCAN(bf16, __nv_bfloat16)
TW_GATED_SCAN(f16, __half)

}  // extern "C"
