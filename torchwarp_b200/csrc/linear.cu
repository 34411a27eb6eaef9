// Linear layer with its epilogue, forward and backward, for float, bfloat16
// and half.
//
//   z = x w^T + b, y = act(z) + residual
//   dz = dy act'(z), dx = dz w, dw = dz^T x, db = sum_rows dz
//
// Products accumulate in float32; z is saved in the element type (only when
// there is an activation), the activation itself is taken of the unrounded z.
#include "../../include/torchwarp_b200.h"
#include "element.cuh"

namespace tw {
namespace {

constexpr int LT = 64;   // tile of the output
constexpr int LK = 16;   // depth of a step
constexpr int L_THREADS = 256;

// out[m, n] = epilogue(sum_k A(m, k) B(n, k)), A(m, k) = A[m * am + k * ak].
template <typename T, int ACT>
__global__ void __launch_bounds__(L_THREADS)
    linear_kernel(const T* __restrict__ A, size_t am, size_t ak, const T* __restrict__ Bm,
                  size_t bn, size_t bk, int M, int N, int K, const T* __restrict__ bias,
                  const T* __restrict__ res, size_t ldr, T* __restrict__ out,
                  T* __restrict__ z) {
  __shared__ float sa[LK][LT + 1], sb[LK][LT + 1];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int tiles_n = (N + LT - 1) / LT;
  const int m0 = (int)(blockIdx.x / tiles_n) * LT, n0 = (int)(blockIdx.x % tiles_n) * LT;
  float acc[4][4] = {};
  for (int k0 = 0; k0 < K; k0 += LK) {
    for (int i = threadIdx.x; i < LT * LK; i += L_THREADS) {
      const int r = i / LK, k = i % LK;
      const bool in = k0 + k < K;
      sa[k][r] = in && m0 + r < M ? to_f(A[(size_t)(m0 + r) * am + (size_t)(k0 + k) * ak]) : 0.f;
      sb[k][r] = in && n0 + r < N ? to_f(Bm[(size_t)(n0 + r) * bn + (size_t)(k0 + k) * bk]) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < LK; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          acc[i][j] = fmaf(sa[k][ty + 16 * i], sb[k][tx + 16 * j], acc[i][j]);
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int m = m0 + ty + 16 * i, n = n0 + tx + 16 * j;
      if (m < M && n < N) {
        const float zv = add_rn(acc[i][j], bias ? to_f(bias[n]) : 0.f);
        if (z) z[(size_t)m * N + n] = from_f<T>(zv);
        const float v = add_rn(act_value<ACT>(zv), res ? to_f(res[(size_t)m * ldr + n]) : 0.f);
        out[(size_t)m * N + n] = from_f<T>(v);
      }
    }
}

template <typename T, int ACT>
__global__ void __launch_bounds__(L_THREADS)
    linear_dz_kernel(const T* __restrict__ dy, size_t ldy, const T* __restrict__ z, int M, int N,
                     T* __restrict__ dz) {
  const size_t n = (size_t)M * N;
  for (size_t i = (size_t)blockIdx.x * L_THREADS + threadIdx.x; i < n;
       i += (size_t)gridDim.x * L_THREADS) {
    const size_t m = i / N, c = i - m * N;
    const float s = ACT == kActNone ? 1.f : act_slope<ACT>(to_f(z[i]));
    dz[i] = from_f<T>(to_f(dy[m * ldy + c]) * s);
  }
}

template <typename T, int ACT>
__global__ void __launch_bounds__(L_THREADS)
    linear_db_kernel(const T* __restrict__ dy, size_t ldy, const T* __restrict__ z, int M, int N,
                     T* __restrict__ db) {
  __shared__ float sh[8][33];
  const int c = threadIdx.x & 31, g = threadIdx.x >> 5, n = blockIdx.x * 32 + c;
  float s = 0.f;
  if (n < N)
    for (int m = g; m < M; m += 8)
      s += to_f(dy[(size_t)m * ldy + n]) *
           (ACT == kActNone ? 1.f : act_slope<ACT>(to_f(z[(size_t)m * N + n])));
  sh[g][c] = s;
  __syncthreads();
  if (g == 0 && n < N) {
    for (int i = 1; i < 8; ++i) s += sh[i][c];
    db[n] = from_f<T>(s);
  }
}

int launched(const char* who) {
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_error(kLaunch, "%s: %s", who, cudaGetErrorString(e));
  return kOk;
}

template <typename T, int ACT>
int product(const T* A, size_t am, size_t ak, const T* B, size_t bn, size_t bk, int M, int N,
            int K, const T* bias, const T* res, size_t ldr, T* out, T* z, cudaStream_t st) {
  const unsigned grid = (unsigned)(((M + LT - 1) / LT) * (size_t)((N + LT - 1) / LT));
  linear_kernel<T, ACT><<<grid, L_THREADS, 0, st>>>(A, am, ak, B, bn, bk, M, N, K, bias, res, ldr,
                                                    out, z);
  return launched("tw_linear");
}

int check(const char* who, int M, int N, int K, int act) {
  if (M < 0 || N <= 0 || K <= 0)
    return set_error(kInvalid, "%s: invalid sizes M=%d N=%d K=%d (need M >= 0, N, K > 0)", who, M,
                     N, K);
  if (act < kActNone || act > kActSigmoid)
    return set_error(kInvalid, "%s: unknown activation %d", who, act);
  const size_t big = 0x7fffffff;
  if ((size_t)((M + LT - 1) / LT) * ((N + LT - 1) / LT) > big ||
      (size_t)((M + LT - 1) / LT) * ((K + LT - 1) / LT) > big ||
      (size_t)((N + LT - 1) / LT) * ((K + LT - 1) / LT) > big)
    return set_error(kUnsupported, "%s: too many tiles", who);
  return kOk;
}

template <typename T>
int fwd(const void* x, size_t ldx, const void* w, size_t ldw, const void* bias, const void* res,
        size_t ldr, int M, int N, int K, int act, void* y, void* z, void* stream) {
  set_error(kOk, "%s", "");
  if (int e = check("tw_linear_forward", M, N, K, act)) return e;
  if (M == 0) return kOk;
  if (!x || !w || !y) return set_error(kInvalid, "tw_linear_forward: null pointer argument");
  cudaStream_t st = (cudaStream_t)stream;
#define TW_CASE(A)                                                                               \
  case A:                                                                                        \
    return product<T, A>((const T*)x, ldx, 1, (const T*)w, ldw, 1, M, N, K, (const T*)bias,      \
                         (const T*)res, ldr, (T*)y, (T*)z, st)
  switch (act) {
    TW_CASE(kActNone);
    TW_CASE(kActRelu);
    TW_CASE(kActGelu);
    TW_CASE(kActSilu);
    default:
      TW_CASE(kActSigmoid);
  }
#undef TW_CASE
}

template <typename T, int ACT>
int bwd_act(const T* dy, size_t ldy, const T* x, size_t ldx, const T* w, size_t ldw, const T* z,
            int M, int N, int K, T* dx, T* dw, T* db, T* dz, cudaStream_t st) {
  if (db) linear_db_kernel<T, ACT><<<(N + 31) / 32, L_THREADS, 0, st>>>(dy, ldy, z, M, N, db);
  size_t ldz = ldy;
  if (ACT != kActNone && M) {
    linear_dz_kernel<T, ACT><<<148 * 8, L_THREADS, 0, st>>>(dy, ldy, z, M, N, dz);
    dy = dz;
    ldz = N;
  }
  int e = launched("tw_linear_backward");
  if (!e && dx && M)
    e = product<T, kActNone>(dy, ldz, 1, w, 1, ldw, M, K, N, nullptr, nullptr, 0, dx, nullptr, st);
  if (!e && dw)
    e = product<T, kActNone>(dy, 1, ldz, x, 1, ldx, N, K, M, nullptr, nullptr, 0, dw, nullptr, st);
  return e;
}

template <typename T>
int bwd(const void* dy, size_t ldy, const void* x, size_t ldx, const void* w, size_t ldw,
        const void* z, int M, int N, int K, int act, void* dx, void* dw, void* db, void* ws,
        size_t ws_bytes, void* stream) {
  set_error(kOk, "%s", "");
  if (int e = check("tw_linear_backward", M, N, K, act)) return e;
  if (M && (!dy || (dx && !w) || (dw && !x) || (act != kActNone && !z)))
    return set_error(kInvalid, "tw_linear_backward: null pointer argument");
  const size_t need = tw_linear_workspace_bytes(M, N, K, (int)sizeof(T), act, 1);
  if (ws_bytes < need || (need && !ws))
    return set_error(kWorkspace, "tw_linear_backward: workspace needs %zu bytes", need);
  cudaStream_t st = (cudaStream_t)stream;
#define TW_CASE(A)                                                                              \
  case A:                                                                                       \
    return bwd_act<T, A>((const T*)dy, ldy, (const T*)x, ldx, (const T*)w, ldw, (const T*)z, M, \
                         N, K, (T*)dx, (T*)dw, (T*)db, (T*)ws, st)
  switch (act) {
    TW_CASE(kActNone);
    TW_CASE(kActRelu);
    TW_CASE(kActGelu);
    TW_CASE(kActSilu);
    default:
      TW_CASE(kActSigmoid);
  }
#undef TW_CASE
}

}  // namespace
}  // namespace tw

extern "C" {

size_t tw_linear_workspace_bytes(int M, int N, int K, int dtype_bytes, int act, int backward) {
  (void)K;
  if (!backward || act == tw::kActNone || M <= 0) return 0;
  return (size_t)M * N * dtype_bytes;
}

#define TW_LINEAR(SUFFIX, T)                                                                     \
  int tw_linear_forward_##SUFFIX(const void* x, size_t ldx, const void* w, size_t ldw,           \
                                 const void* bias, const void* residual, size_t ldr, int M,      \
                                 int N, int K, int act, void* y, void* z, void* workspace,       \
                                 size_t ws_bytes, void* stream) {                                \
    (void)workspace;                                                                             \
    (void)ws_bytes;                                                                              \
    return tw::fwd<T>(x, ldx, w, ldw, bias, residual, ldr, M, N, K, act, y, z, stream);          \
  }                                                                                              \
  int tw_linear_backward_##SUFFIX(const void* dy, size_t lddy, const void* x, size_t ldx,        \
                                  const void* w, size_t ldw, const void* z, int M, int N, int K, \
                                  int act, void* dx, void* dw, void* dbias, void* workspace,     \
                                  size_t ws_bytes, void* stream) {                               \
    return tw::bwd<T>(dy, lddy, x, ldx, w, ldw, z, M, N, K, act, dx, dw, dbias, workspace,       \
                      ws_bytes, stream);                                                         \
  }

TW_LINEAR(f32, float)
TW_LINEAR(bf16, __nv_bfloat16)
TW_LINEAR(f16, __half)

}  // extern "C"
