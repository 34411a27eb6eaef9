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
constexpr int BWD_THREADS = 128;  // of a backward block whose warps hold whole rows

// Sum over the block; every thread gets it.
__device__ __forceinline__ float block_sum(float v, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.f;
  for (int i = 0; i < (int)(blockDim.x >> 5); ++i) s += red[i];
  return s;
}

// Sum over the threads of a row: `tpr` lanes of a warp, or the block.
template <bool BLOCK>
__device__ __forceinline__ float row_sum(float v, int tpr, float* red) {
  if constexpr (BLOCK) {
    return block_sum(v, red);
  } else {
    for (int o = tpr >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  }
}

// N values of a thread, two an instruction where N is even.
template <int N> struct Width { static constexpr int W = N % 2 == 0 ? 2 : 1; };
template <int N>
__device__ __forceinline__ Vec<Width<N>::W> at(const float* v, int i) {
  Vec<Width<N>::W> r;
#pragma unroll
  for (int k = 0; k < Width<N>::W; ++k) r.v[k] = v[i + k];
  return r;
}
template <int N>
__device__ __forceinline__ void put(float* v, int i, Vec<Width<N>::W> r) {
#pragma unroll
  for (int k = 0; k < Width<N>::W; ++k) v[i + k] = r.v[k];
}
#define TW_EACH for (int i = 0, W = Width<N>::W; i < N; i += W)
template <int N> __device__ __forceinline__ void shift_n(float* v, float c) {
#pragma unroll
  TW_EACH put<N>(v, i, add_v(at<N>(v, i), splat<Width<N>::W>(c)));
}
template <int N> __device__ __forceinline__ void scale_n(float* v, float c) {
#pragma unroll
  TW_EACH put<N>(v, i, mul_v(at<N>(v, i), splat<Width<N>::W>(c)));
}
template <int N> __device__ __forceinline__ void times_n(float* v, const float* p) {
#pragma unroll
  TW_EACH put<N>(v, i, mul_v(at<N>(v, i), at<N>(p, i)));
}
template <int N> __device__ __forceinline__ void plus_n(float* v, const float* p) {
#pragma unroll
  TW_EACH put<N>(v, i, add_v(at<N>(v, i), at<N>(p, i)));
}
template <int N>  // v += p q
__device__ __forceinline__ void fma_n(float* v, const float* p, const float* q) {
#pragma unroll
  TW_EACH put<N>(v, i, fma_v(at<N>(p, i), at<N>(q, i), at<N>(v, i)));
}
template <int N> __device__ __forceinline__ float total(Vec<Width<N>::W> s) {
  float t = s.v[0];
  if (Width<N>::W == 2) t += s.v[Width<N>::W - 1];
  return t;
}
template <int N> __device__ __forceinline__ float sum_of(const float* v) {
  Vec<Width<N>::W> s = splat<Width<N>::W>(0.f);
#pragma unroll
  TW_EACH s = add_v(s, at<N>(v, i));
  return total<N>(s);
}
template <int N> __device__ __forceinline__ float dot_of(const float* p, const float* q) {
  Vec<Width<N>::W> s = splat<Width<N>::W>(0.f);
#pragma unroll
  TW_EACH s = fma_v(at<N>(p, i), at<N>(q, i), s);
  return total<N>(s);
}
template <int N> __device__ __forceinline__ float square_sum_of(const float* v) {
  return dot_of<N>(v, v);
}

// Rows that fit the registers of `tpr` threads, E values each (VEC: in
// 16-byte pieces, so that a row is read with whole-sector loads; else value
// by value, neighbours in neighbouring lanes).  BLOCK: one row a block, else
// 32 / tpr rows a warp.  x is read once; the two passes of the statistics run
// on registers.  32768 x 1024 bfloat16: 25.6 us, 5.2 TB/s, 81% of a copy's rate
// (102 us with one block a row, reading it three times).
template <typename T, typename P, bool VEC, int E, bool BLOCK>
__global__ void __launch_bounds__(LN_THREADS)
    ln_fwd_kernel(const T* __restrict__ x, size_t xs, const P* __restrict__ w,
                  const P* __restrict__ b, size_t rows, int D, int tpr_log, float inv_d, float eps,
                  T* __restrict__ y, float* __restrict__ mean, float* __restrict__ rstd) {
  constexpr int V = VEC ? 16 / (int)sizeof(T) : 1, NV = E / V;
  __shared__ float red[LN_THREADS / 32];
  const int tpr = BLOCK ? blockDim.x : 1 << tpr_log;
  const int t = BLOCK ? threadIdx.x : threadIdx.x & (tpr - 1);
  const size_t r = BLOCK ? blockIdx.x
                         : ((size_t)blockIdx.x * LN_THREADS + threadIdx.x) >> tpr_log;
  const bool in = r < rows;
  const T* xr = x + (in ? r : rows - 1) * xs;
  float v[E];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int d = (j * tpr + t) * V;
    if (d < D) {
      load_n<VEC, V>(xr + d, v + j * V);
    } else {
#pragma unroll
      for (int q = 0; q < V; ++q) v[j * V + q] = 0.f;
    }
  }
  const float mu = row_sum<BLOCK>(sum_of<E>(v), tpr, red) * inv_d;
#pragma unroll
  for (int j = 0; j < NV; ++j)
    if ((j * tpr + t) * V < D) shift_n<V>(v + j * V, -mu);
  const float rs = rsqrtf(row_sum<BLOCK>(square_sum_of<E>(v), tpr, red) * inv_d + eps);
  if (!in) return;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int d = (j * tpr + t) * V;
    if (d < D) {
      float* o = v + j * V;
      float p[V];
      scale_n<V>(o, rs);
      if (w) {
        load_n<VEC, V>(w + d, p);
        times_n<V>(o, p);
      }
      if (b) {
        load_n<VEC, V>(b + d, p);
        plus_n<V>(o, p);
      }
      store_n<VEC, V>(y + r * D + d, o);
    }
  }
  if (mean && t == 0) {
    mean[r] = mu;
    rstd[r] = rs;
  }
}

// dx, and this block's sums for dw and db: a thread keeps the same columns
// for all its rows, so both sums stay in registers until the block's last
// row.  x and dy are read once.  AHEAD: each thread brings its own pieces of
// the next row to shared memory with cp.async while it works on this one, and
// reads them from there for both passes; no barrier, as nobody else reads
// them.  Blocks of 4 warps, as many as the registers of 32 values a thread
// allow.  32768 x 1024 bfloat16: 146 us with blocks of 8 warps and the row in
// registers, 62 with 4, 50 with the next row ahead.  part:
// [gridDim.x][2][D] (NULL: only dx).
template <typename T, typename P, bool VEC, int E, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? LN_THREADS : BWD_THREADS,
                                  BLOCK ? 1 : VEC && sizeof(T) == 2 ? 4 : 3)
    ln_bwd_kernel(const T* __restrict__ dy, size_t dys, const T* __restrict__ x, size_t xs,
                  const P* __restrict__ w, const float* __restrict__ mean,
                  const float* __restrict__ rstd, size_t rows, int D, int tpr,
                  T* __restrict__ dx, float* __restrict__ part) {
  constexpr int V = VEC ? 16 / (int)sizeof(T) : 1, NV = E / V;
  constexpr bool AHEAD = VEC && !BLOCK;
  // first the rows ahead: [2][x, dy][NV] pieces of every thread; at the end
  // [2][D] sums of the block's warps, one after the other
  extern __shared__ __align__(16) uint8_t room[];
  float* acc_s = reinterpret_cast<float*>(room);
  __shared__ float red[LN_THREADS / 32];
  const int t = BLOCK ? threadIdx.x : threadIdx.x & (tpr - 1);
  const int per = BLOCK ? 1 : BWD_THREADS / tpr;  // rows of a block's step
  const float inv_d = 1.f / D;
  float aw[E], ab[E];
#pragma unroll
  for (int i = 0; i < E; ++i) aw[i] = ab[i] = 0.f;
  const size_t stride = (size_t)gridDim.x * per;
  const size_t mine = BLOCK ? 0 : threadIdx.x / tpr;
  auto piece = [&](int stage, int array, int j) {
    return room + ((((stage * 2 + array) * NV + j) * BWD_THREADS + threadIdx.x) << 4);
  };
  float mu_next = 0.f, rs_next = 0.f;
  auto fetch = [&](size_t r, int stage) {
    if (r < rows) {
      mu_next = mean[r];
      rs_next = rstd[r];
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int d = (j * tpr + t) * V;
      const bool in = r < rows && d < D;
      cp_async16(piece(stage, 0, j), in ? x + r * xs + d : x, in ? 16 : 0);
      cp_async16(piece(stage, 1, j), in ? dy + r * dys + d : dy, in ? 16 : 0);
    }
    cp_async_commit();
  };
  int stage = 0;
  if (AHEAD) fetch((size_t)blockIdx.x * per + mine, 0);
  for (size_t r0 = (size_t)blockIdx.x * per; r0 < rows; r0 += stride) {
    const size_t r = r0 + mine;
    const bool in = r < rows;
    const size_t rc = in ? r : rows - 1;
    float mu, rs;
    Raw<VEC, V, T> gr[NV], hr[NV];  // in shared memory when AHEAD
    float s1 = 0.f, s2 = 0.f;
    if constexpr (AHEAD) {
      mu = mu_next;
      rs = rs_next;
      fetch(r + stride, stage ^ 1);
      asm volatile("cp.async.wait_group 1;\n" ::: "memory");
    } else {
      mu = mean[rc];
      rs = rstd[rc];
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int d = (j * tpr + t) * V;
        if (in && d < D) {
          gr[j].load(dy + rc * dys + d);
          hr[j].load(x + rc * xs + d);
        } else {
          gr[j].zero();
          hr[j].zero();
        }
      }
    }
    auto row = [&](int j, float* g, float* h) {
      if constexpr (AHEAD) {
        unpack16<T>(*reinterpret_cast<const uint4*>(piece(stage, 1, j)), g);
        unpack16<T>(*reinterpret_cast<const uint4*>(piece(stage, 0, j)), h);
      } else {
        gr[j].get(g);
        hr[j].get(h);
      }
    };
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int d = (j * tpr + t) * V;
      float g[V], h[V];
      row(j, g, h);
      shift_n<V>(h, -mu);
      scale_n<V>(h, rs);
      plus_n<V>(ab + j * V, g);
      fma_n<V>(aw + j * V, g, h);
      if (w && d < D) {
        float wv[V];
        load_n<VEC, V>(w + d, wv);
        times_n<V>(g, wv);
      }
      s1 += sum_of<V>(g);
      s2 += dot_of<V>(g, h);
    }
    if (dx) {
      const float c1 = row_sum<BLOCK>(s1, tpr, red) * inv_d;
      const float c2 = row_sum<BLOCK>(s2, tpr, red) * inv_d;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int d = (j * tpr + t) * V;
        if (in && d < D) {
          float g[V], h[V];
          row(j, g, h);
          if (w) {
            float wv[V];
            load_n<VEC, V>(w + d, wv);
            times_n<V>(g, wv);
          }
          shift_n<V>(h, -mu);
          scale_n<V>(h, rs);
          scale_n<V>(h, -c2);
          shift_n<V>(g, -c1);
          plus_n<V>(g, h);
          scale_n<V>(g, rs);
          store_n<VEC, V>(dx + r * D + d, g);
        }
      }
    }
    stage ^= 1;
    // this row's pieces were read before the copies that replace them start
    asm volatile("" ::: "memory");
  }
  if (AHEAD) {
    asm volatile("cp.async.wait_group 0;\n" ::: "memory");
    __syncthreads();  // the rows' room becomes the sums'
  }
  if (!part) return;
  if (!BLOCK) {  // the rows of a warp's other lanes, then the warps in their order
    for (int o = tpr; o < 32; o <<= 1)
#pragma unroll
      for (int i = 0; i < E; ++i) {
        aw[i] += __shfl_xor_sync(0xffffffffu, aw[i], o);
        ab[i] += __shfl_xor_sync(0xffffffffu, ab[i], o);
      }
    const int warp = threadIdx.x >> 5;
    for (int k = 0; k < BWD_THREADS / 32; ++k) {
      __syncthreads();
      if (warp == k && (threadIdx.x & 31) < tpr) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          const int d = (j * tpr + t) * V;
          if (d < D)
#pragma unroll
            for (int q = 0; q < V; ++q) {
              const int i = j * V + q;
              if (k == 0) {
                acc_s[d + q] = aw[i];
                acc_s[D + d + q] = ab[i];
              } else {
                acc_s[d + q] += aw[i];
                acc_s[D + d + q] += ab[i];
              }
            }
        }
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * D; i += BWD_THREADS)
      part[(size_t)blockIdx.x * 2 * D + i] = acc_s[i];
  } else {
    float* o = part + (size_t)blockIdx.x * 2 * D;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int d = (j * tpr + t) * V;
      if (d < D) {
        store_n<false, V>(o + d, aw + j * V);
        store_n<false, V>(o + D + d, ab + j * V);
      }
    }
  }
}

// dw and db from the blocks' sums, in a fixed order: 32 columns a block, whose
// 32 warps share the rows (8 warps took 9.4 us for 444 x 2048, a chain of 55
// loads).
template <typename P>
__global__ void __launch_bounds__(1024)
    ln_join_kernel(const float* __restrict__ part, int blocks, int D, P* __restrict__ dw,
                   P* __restrict__ db) {
  __shared__ float red[32][33];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5, c = blockIdx.x * 32 + tx;
  float s = 0.f;
  if (c < 2 * D)
#pragma unroll 8
    for (int k = ty; k < blocks; k += 32) s += part[(size_t)k * 2 * D + c];
  red[ty][tx] = s;
  __syncthreads();
  s = red[tx][ty];  // warp ty sums column ty
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  const int col = blockIdx.x * 32 + ty;
  if (tx == 0 && col < 2 * D) {
    if (col < D && dw) dw[col] = from_f<P>(s);
    if (col >= D && db) db[col - D] = from_f<P>(s);
  }
}

// ---- rows longer than a block's registers: read again from the caches

template <typename T, typename P>
__global__ void __launch_bounds__(LN_THREADS)
    ln_fwd_long_kernel(const T* __restrict__ x, size_t xs, const P* __restrict__ w,
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
    const float rs = rsqrtf(block_sum(s, red) / D + eps);
    for (int d = threadIdx.x; d < D; d += LN_THREADS) {
      const float xh = mul_rn(to_f(xr[d]) - mu, rs);
      y[r * D + d] = from_f<T>(add_rn(mul_rn(xh, w ? to_f(w[d]) : 1.f), b ? to_f(b[d]) : 0.f));
    }
    if (mean && threadIdx.x == 0) {
      mean[r] = mu;
      rstd[r] = rs;
    }
  }
}

template <typename T, typename P>
__global__ void __launch_bounds__(LN_THREADS)
    ln_dx_long_kernel(const T* __restrict__ dy, size_t dys, const T* __restrict__ x, size_t xs,
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
    ln_dw_long_kernel(const T* __restrict__ dy, size_t dys, const T* __restrict__ x, size_t xs,
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

// How a row of D values is spread: E values a thread (the fewest of 8, 16, 32
// that let a warp hold the row), `tpr` threads; a longer row over a block.
// Read value by value (not vec) a thread takes at most 16, as its bounds
// checks are one a value and 32 of them spill.  tpr 0: too long for a block.
struct RowPlan {
  int e, tpr, per;  // per: rows of a block
  int per_sm;       // backward blocks a SM holds at 32 values a thread (16: one more)
};

RowPlan row_plan(int D, bool vec, int per_sm = 3) {
  const int most = vec ? 32 : 16;
  RowPlan p = {most, 0, 1, per_sm};
  if (D > most * LN_THREADS) return p;
  if (D <= 32 * most) {
    p.e = D <= 256 ? 8 : D <= 512 ? 16 : 32;
    p.tpr = 1;
    while (p.tpr * p.e < D) p.tpr *= 2;
    p.per = LN_THREADS / p.tpr;
  } else {
    p.tpr = (D + 32 * most - 1) / (32 * most) * 32;
  }
  return p;
}

// Blocks of the backward: what a SM holds, fewer when there are fewer rows.
int bwd_per(const RowPlan& p) { return p.tpr > 32 ? 1 : BWD_THREADS / p.tpr; }
int bwd_blocks(size_t rows, const RowPlan& p) {
  const int per_sm = p.tpr > 32 ? 1024 / p.tpr / 2 : p.e == 8 ? 8 : p.e == 16 ? p.per_sm + 1 : p.per_sm;
  const size_t steps = (rows + bwd_per(p) - 1) / bwd_per(p), most = 148 * (per_sm < 1 ? 1 : per_sm);
  return (int)(steps < most ? steps : most);
}

int check(const char* who, size_t rows, int D) {
  if (D <= 0) return set_error(kInvalid, "%s: invalid D=%d (need D > 0)", who, D);
  if (rows > (size_t)1 << 40) return set_error(kInvalid, "%s: too many rows", who);
  return kOk;
}

int launched(const char* who) {
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_error(kLaunch, "%s: %s", who, cudaGetErrorString(e));
  return kOk;
}

int grid_of(size_t rows) { return (int)(rows < 148 * 8 ? rows : 148 * 8); }

bool aligned16(const void* p, size_t stride_bytes) {
  return (uintptr_t)p % 16 == 0 && stride_bytes % 16 == 0;
}

int log2_of(int n) {
  int l = 0;
  while ((1 << l) < n) ++l;
  return l;
}

// The instance of a row kernel for a plan.
#define TW_ROW_KERNEL(KERNEL)                                                          \
  (!vec ? (plan.tpr > 32 ? KERNEL<T, P, false, 16, true>                               \
           : plan.e == 8 ? KERNEL<T, P, false, 8, false> : KERNEL<T, P, false, 16, false>) \
   : plan.tpr > 32 ? KERNEL<T, P, true, 32, true>                                      \
   : plan.e == 8 ? KERNEL<T, P, true, 8, false>                                        \
   : plan.e == 16 ? KERNEL<T, P, true, 16, false> : KERNEL<T, P, true, 32, false>)

template <typename T, typename P>
int fwd_p(const void* x, size_t xs, const void* w, const void* b, size_t rows, int D, float eps,
          void* y, float* mean, float* rstd, cudaStream_t st) {
  const bool vec = D * sizeof(T) % 16 == 0 && aligned16(x, xs * sizeof(T)) && aligned16(y, 0) &&
                   aligned16(w, 0) && aligned16(b, 0);
  const RowPlan plan = row_plan(D, vec);
  if (plan.tpr == 0) {
    ln_fwd_long_kernel<T, P><<<grid_of(rows), LN_THREADS, 0, st>>>(
        (const T*)x, xs, (const P*)w, (const P*)b, rows, D, eps, (T*)y, mean, rstd);
    return launched("tw_layer_norm_forward");
  }
  const size_t blocks = (rows + plan.per - 1) / plan.per;
  if (blocks > 0x7fffffff) return set_error(kUnsupported, "tw_layer_norm_forward: too many rows");
  auto kernel = TW_ROW_KERNEL(ln_fwd_kernel);
  kernel<<<(unsigned)blocks, plan.tpr > 32 ? plan.tpr : LN_THREADS, 0, st>>>(
      (const T*)x, xs, (const P*)w, (const P*)b, rows, D, log2_of(plan.tpr), 1.f / D, eps,
      (T*)y, mean, rstd);
  return launched("tw_layer_norm_forward");
}

template <typename T>
int fwd(const void* x, size_t xs, const void* w, const void* b, int pf32, size_t rows, int D,
        double eps, void* y, float* mean, float* rstd, void* stream) {
  set_error(kOk, "%s", "");
  if (int e = check("tw_layer_norm_forward", rows, D)) return e;
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
          const float* rstd, size_t rows, int D, void* dx, void* dw, void* db, void* ws,
          cudaStream_t st) {
  const bool vec = D * sizeof(T) % 16 == 0 && aligned16(x, xs * sizeof(T)) &&
                   aligned16(dy, dys * sizeof(T)) && aligned16(w, 0) && aligned16(dx, 0);
  const RowPlan plan = row_plan(D, vec, !vec ? 2 : sizeof(T) == 2 ? 4 : 3);
  if (plan.tpr == 0) {
    if (dx && rows)
      ln_dx_long_kernel<T, P><<<grid_of(rows), LN_THREADS, 0, st>>>(
          (const T*)dy, dys, (const T*)x, xs, (const P*)w, mean, rstd, rows, D, (T*)dx);
    if (dw || db)
      ln_dw_long_kernel<T, P><<<(D + 31) / 32, LN_THREADS, 0, st>>>(
          (const T*)dy, dys, (const T*)x, xs, mean, rstd, rows, D, (P*)dw, (P*)db);
    return launched("tw_layer_norm_backward");
  }
  const int blocks = bwd_blocks(rows, plan);
  float* part = dw || db ? (float*)ws : nullptr;
  if (blocks) {
    auto kernel = TW_ROW_KERNEL(ln_bwd_kernel);
    size_t smem = part && plan.tpr <= 32 ? 2 * (size_t)D * sizeof(float) : 0;
    const size_t ahead = (size_t)plan.e * sizeof(T) * 2 * 2 * BWD_THREADS;
    if (vec && plan.tpr <= 32 && smem < ahead) smem = ahead;
    if (smem > 48 * 1024) {
      const cudaError_t e = cudaFuncSetAttribute(
          (const void*)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
      if (e != cudaSuccess)
        return set_error(kLaunch, "tw_layer_norm_backward: %s", cudaGetErrorString(e));
    }
    kernel<<<blocks, plan.tpr > 32 ? plan.tpr : BWD_THREADS, smem, st>>>(
        (const T*)dy, dys, (const T*)x, xs, (const P*)w, mean, rstd, rows, D, plan.tpr, (T*)dx,
        part);
  }
  if (dw || db)
    ln_join_kernel<P><<<(2 * D + 31) / 32, 1024, 0, st>>>(part, blocks, D, (P*)dw, (P*)db);
  return launched("tw_layer_norm_backward");
}

template <typename T>
int bwd(const void* dy, size_t dys, const void* x, size_t xs, const void* w, int pf32,
        const float* mean, const float* rstd, size_t rows, int D, void* dx, void* dw, void* db,
        void* ws, size_t ws_bytes, void* stream) {
  set_error(kOk, "%s", "");
  if (int e = check("tw_layer_norm_backward", rows, D)) return e;
  if (rows && (!dy || !x || !mean || !rstd))
    return set_error(kInvalid, "tw_layer_norm_backward: null pointer argument");
  if (ws_bytes < tw_layer_norm_workspace_bytes(rows, D) || (ws_bytes && !ws))
    return set_error(kWorkspace, "tw_layer_norm_backward: workspace needs %zu bytes",
                     tw_layer_norm_workspace_bytes(rows, D));
  cudaStream_t st = (cudaStream_t)stream;
  return pf32 ? bwd_p<T, float>(dy, dys, x, xs, w, mean, rstd, rows, D, dx, dw, db, ws, st)
              : bwd_p<T, T>(dy, dys, x, xs, w, mean, rstd, rows, D, dx, dw, db, ws, st);
}

}  // namespace
}  // namespace tw

extern "C" {

size_t tw_layer_norm_workspace_bytes(size_t rows, int D) {
  if (D <= 0) return 0;
  int blocks = 0;  // of either way to read a row
  for (int vec = 0; vec < 2; ++vec) {
    const tw::RowPlan p = tw::row_plan(D, vec != 0, 4);
    const int b = p.tpr ? tw::bwd_blocks(rows, p) : 0;
    if (b > blocks) blocks = b;
  }
  return (size_t)blocks * 2 * D * sizeof(float);
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
