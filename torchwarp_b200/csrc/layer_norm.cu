// Layer norm over the last dimension, forward and backward, for float,
// bfloat16 and half rows.
//
//   mean = sum x / D, rstd = 1 / sqrt(sum (x - mean)^2 / D + eps)
//   xhat = (x - mean) rstd, y = xhat w + b
//   q = dy w, dx = rstd (q - mean(q) - xhat mean(q xhat))
//   dw = sum_rows dy xhat, db = sum_rows dy
//
// Statistics and sums are float32.  The variance is the sum of squared
// differences from the mean (not E x^2 - mean^2, which cancels for rows with
// a large offset).
#include "../../include/torchwarp_b200.h"
#include "element.cuh"

namespace tw {
namespace {

constexpr int LN_THREADS = 256;

// Sum over the block; every thread gets it.
__device__ __forceinline__ float block_sum(float v, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < LN_THREADS / 32; ++i) s += red[i];
  return s;
}

template <typename T, typename P>
__global__ void __launch_bounds__(LN_THREADS)
    ln_fwd_kernel(const T* __restrict__ x, size_t xs, const P* __restrict__ w,
                  const P* __restrict__ b, size_t rows, int D, float eps, T* __restrict__ y,
                  float* __restrict__ mean, float* __restrict__ rstd) {
  __shared__ float red[LN_THREADS / 32];
  for (size_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* xr = x + r * xs;
    float s = 0.f;
    for (int d = threadIdx.x; d < D; d += LN_THREADS) s += to_f(xr[d]);
    const float mu = block_sum(s, red) / D;
    s = 0.f;
    for (int d = threadIdx.x; d < D; d += LN_THREADS) {
      const float c = to_f(xr[d]) - mu;
      s = fmaf(c, c, s);
    }
    const float rs = 1.f / sqrtf(block_sum(s, red) / D + eps);
    for (int d = threadIdx.x; d < D; d += LN_THREADS) {
      const float xh = (to_f(xr[d]) - mu) * rs;
      y[r * D + d] = from_f<T>(fmaf(xh, w ? to_f(w[d]) : 1.f, b ? to_f(b[d]) : 0.f));
    }
    if (mean && threadIdx.x == 0) {
      mean[r] = mu;
      rstd[r] = rs;
    }
  }
}

template <typename T, typename P>
__global__ void __launch_bounds__(LN_THREADS)
    ln_dx_kernel(const T* __restrict__ dy, size_t dys, const T* __restrict__ x, size_t xs,
                 const P* __restrict__ w, const float* __restrict__ mean,
                 const float* __restrict__ rstd, size_t rows, int D, T* __restrict__ dx) {
  __shared__ float red[LN_THREADS / 32];
  for (size_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const float mu = mean[r], rs = rstd[r];
    float s1 = 0.f, s2 = 0.f;
    for (int d = threadIdx.x; d < D; d += LN_THREADS) {
      const float q = to_f(dy[r * dys + d]) * (w ? to_f(w[d]) : 1.f);
      s1 += q;
      s2 = fmaf(q, (to_f(x[r * xs + d]) - mu) * rs, s2);
    }
    const float c1 = block_sum(s1, red) / D, c2 = block_sum(s2, red) / D;
    for (int d = threadIdx.x; d < D; d += LN_THREADS) {
      const float q = to_f(dy[r * dys + d]) * (w ? to_f(w[d]) : 1.f);
      const float xh = (to_f(x[r * xs + d]) - mu) * rs;
      dx[r * D + d] = from_f<T>(rs * (q - c1 - xh * c2));
    }
  }
}

// One block: 32 columns, all rows, in a fixed order.
template <typename T, typename P>
__global__ void __launch_bounds__(LN_THREADS)
    ln_dw_kernel(const T* __restrict__ dy, size_t dys, const T* __restrict__ x, size_t xs,
                 const float* __restrict__ mean, const float* __restrict__ rstd, size_t rows,
                 int D, P* __restrict__ dw, P* __restrict__ db) {
  __shared__ float sw[8][33], sb[8][33];
  const int c = threadIdx.x & 31, g = threadIdx.x >> 5, d = blockIdx.x * 32 + c;
  float aw = 0.f, ab = 0.f;
  if (d < D)
    for (size_t r = g; r < rows; r += 8) {
      const float v = to_f(dy[r * dys + d]);
      ab += v;
      aw = fmaf(v, (to_f(x[r * xs + d]) - mean[r]) * rstd[r], aw);
    }
  sw[g][c] = aw;
  sb[g][c] = ab;
  __syncthreads();
  if (g == 0 && d < D) {
    for (int i = 1; i < 8; ++i) {
      aw += sw[i][c];
      ab += sb[i][c];
    }
    if (dw) dw[d] = from_f<P>(aw);
    if (db) db[d] = from_f<P>(ab);
  }
}

int check(const char* who, size_t rows, int D, size_t xs) {
  if (D <= 0) return set_error(kInvalid, "%s: invalid D=%d (need D > 0)", who, D);
  if (rows > (size_t)1 << 40) return set_error(kInvalid, "%s: too many rows", who);
  if (rows > 1 && xs < (size_t)D && xs != 0)
    return set_error(kInvalid, "%s: row stride %zu is below D=%d", who, xs, D);
  return kOk;
}

int launched(const char* who) {
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_error(kLaunch, "%s: %s", who, cudaGetErrorString(e));
  return kOk;
}

int grid_of(size_t rows) { return (int)(rows < 148 * 8 ? rows : 148 * 8); }

template <typename T, typename P>
int fwd_p(const void* x, size_t xs, const void* w, const void* b, size_t rows, int D, float eps,
          void* y, float* mean, float* rstd, cudaStream_t st) {
  ln_fwd_kernel<T, P><<<grid_of(rows), LN_THREADS, 0, st>>>(
      (const T*)x, xs, (const P*)w, (const P*)b, rows, D, eps, (T*)y, mean, rstd);
  return launched("tw_layer_norm_forward");
}

template <typename T>
int fwd(const void* x, size_t xs, const void* w, const void* b, int pf32, size_t rows, int D,
        double eps, void* y, float* mean, float* rstd, void* stream) {
  set_error(kOk, "%s", "");
  if (int e = check("tw_layer_norm_forward", rows, D, xs)) return e;
  if (!(eps >= 0)) return set_error(kInvalid, "tw_layer_norm_forward: eps must be >= 0");
  if (rows == 0) return kOk;
  if (!x || !y || (mean == nullptr) != (rstd == nullptr))
    return set_error(kInvalid, "tw_layer_norm_forward: null pointer argument");
  cudaStream_t st = (cudaStream_t)stream;
  return pf32 ? fwd_p<T, float>(x, xs, w, b, rows, D, (float)eps, y, mean, rstd, st)
              : fwd_p<T, T>(x, xs, w, b, rows, D, (float)eps, y, mean, rstd, st);
}

template <typename T, typename P>
int bwd_p(const void* dy, size_t dys, const void* x, size_t xs, const void* w, const float* mean,
          const float* rstd, size_t rows, int D, void* dx, void* dw, void* db, cudaStream_t st) {
  if (dx && rows)
    ln_dx_kernel<T, P><<<grid_of(rows), LN_THREADS, 0, st>>>((const T*)dy, dys, (const T*)x, xs,
                                                             (const P*)w, mean, rstd, rows, D,
                                                             (T*)dx);
  if (dw || db)
    ln_dw_kernel<T, P><<<(D + 31) / 32, LN_THREADS, 0, st>>>(
        (const T*)dy, dys, (const T*)x, xs, mean, rstd, rows, D, (P*)dw, (P*)db);
  return launched("tw_layer_norm_backward");
}

template <typename T>
int bwd(const void* dy, size_t dys, const void* x, size_t xs, const void* w, int pf32,
        const float* mean, const float* rstd, size_t rows, int D, void* dx, void* dw, void* db,
        void* ws, size_t ws_bytes, void* stream) {
  set_error(kOk, "%s", "");
  if (int e = check("tw_layer_norm_backward", rows, D, xs)) return e;
  if (int e = check("tw_layer_norm_backward", rows, D, dys)) return e;
  if (rows && (!dy || !x || !mean || !rstd))
    return set_error(kInvalid, "tw_layer_norm_backward: null pointer argument");
  if (ws_bytes < tw_layer_norm_workspace_bytes(rows, D) || (ws_bytes && !ws))
    return set_error(kWorkspace, "tw_layer_norm_backward: workspace needs %zu bytes",
                     tw_layer_norm_workspace_bytes(rows, D));
  cudaStream_t st = (cudaStream_t)stream;
  return pf32 ? bwd_p<T, float>(dy, dys, x, xs, w, mean, rstd, rows, D, dx, dw, db, st)
              : bwd_p<T, T>(dy, dys, x, xs, w, mean, rstd, rows, D, dx, dw, db, st);
}

}  // namespace
}  // namespace tw

extern "C" {

size_t tw_layer_norm_workspace_bytes(size_t rows, int D) {
  (void)rows;
  (void)D;
  return 0;
}

#define TW_LAYER_NORM(SUFFIX, T)                                                                \
  int tw_layer_norm_forward_##SUFFIX(const void* x, size_t x_stride, const void* weight,        \
                                     const void* bias, int params_f32, size_t rows, int D,      \
                                     double eps, void* y, float* mean, float* rstd,             \
                                     void* stream) {                                            \
    return tw::fwd<T>(x, x_stride, weight, bias, params_f32, rows, D, eps, y, mean, rstd,       \
                      stream);                                                                  \
  }                                                                                             \
  int tw_layer_norm_backward_##SUFFIX(const void* dy, size_t dy_stride, const void* x,          \
                                      size_t x_stride, const void* weight, int params_f32,      \
                                      const float* mean, const float* rstd, size_t rows, int D, \
                                      void* dx, void* dweight, void* dbias, void* workspace,    \
                                      size_t ws_bytes, void* stream) {                          \
    return tw::bwd<T>(dy, dy_stride, x, x_stride, weight, params_f32, mean, rstd, rows, D, dx,  \
                      dweight, dbias, workspace, ws_bytes, stream);                             \
  }

TW_LAYER_NORM(f32, float)
TW_LAYER_NORM(bf16, __nv_bfloat16)
TW_LAYER_NORM(f16, __half)

}  // extern "C"
