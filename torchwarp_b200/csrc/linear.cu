// Linear layer with its epilogue, forward and backward, for float, bfloat16
// and half.
//
//   z = x w^T + b, y = act(z) + residual
//   dz = dy act'(z), dx = dz w, dw = dz^T x, db = sum_rows dz
//
// Products run on the tensor cores (linear_gemm.cuh) and accumulate in
// float32.  Up to SMALL_ROWS rows (single tokens) the forward reads the
// weight once with plain loads instead.  z is saved in the element type and
// only when there is an activation; the activation itself is taken of the
// unrounded z.  dz is rounded to the element type once, as the operand of its
// two products; db sums it before that rounding.
//
// An operand goes to the tensor cores as it lies in memory when TMA can read
// it (16-byte aligned rows).  Otherwise, and for float32, which is taken as
// three bfloat16 planes, a pass writes it to the workspace first.
#include "../../include/torchwarp_b200.h"
#include "element.cuh"
#include "linear_gemm.h"

namespace tw {

// One CTA pair computes a 256 x 256 tile at the tensor cores' full rate; it
// takes 48 such tiles (of the 74 pairs) to beat single CTAs with narrower
// tiles, which spread a small product over more SMs.  Where even those leave
// a third of the SMs idle, the contraction is split, down to 4 chunks (256
// values) a part (2 chunks for float32, whose chunks take six products).
GemmPlan gemm_plan(int M, int N, int K, int planes) {
  const long long nK = (K + 63) / 64;
  if (planes == 1) {
    const long long pairs = (long long)((M + 255) / 256) * ((N + 255) / 256);
    if (pairs >= 48) return {2, 256, 1};
  }
  const long long rows = (M + 127) / 128;
  const int tn = N > 64 && rows * ((N + 127) / 128) >= 74 ? 128 : 64;
  const long long tiles = rows * ((N + tn - 1) / tn);
  long long splits = 1;
  if (tiles < 100) {
    splits = 148 / tiles;
    const long long most = nK / (planes == 1 ? 4 : 2);
    if (splits > most) splits = most;
    if (splits < 1) splits = 1;
  }
  return {1, tn, (int)splits};
}

namespace {

constexpr int SMALL_ROWS = 8;
constexpr int SMALL_COLS = 4;  // output columns of a warp

// --------------------------------------------------------- few rows

// Sums C values over the warp so that lane l ends with value l / (32 / C):
// each step sends the half of the values that the other lanes keep.
template <int C>
__device__ __forceinline__ float scatter_sum(float (&v)[C], int lane) {
  int o = 16;
#pragma unroll
  for (int n = C; n > 1; n /= 2, o /= 2) {
    const bool up = lane & o;
#pragma unroll
    for (int i = 0; i < n / 2; ++i) {
      const float send = up ? v[i] : v[i + n / 2], keep = up ? v[i + n / 2] : v[i];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
    }
  }
  float s = v[0];
#pragma unroll
  for (; o > 0; o /= 2) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}

// M <= MT rows: a warp owns 4 output columns, its lanes the contraction.
// Bound by the one read of the weight; x stays in the caches.  8 x 1024 x 4096
// bfloat16: 6.8 us a call with the launch (127 us on 64 x 64 tiles of plain
// FMAs).
template <typename T, int MT, bool VEC>
__global__ void __launch_bounds__(128)
    linear_small_kernel(const T* __restrict__ x, size_t ldx, const T* __restrict__ w, size_t ldw,
                        int M, int N, int K, const T* __restrict__ bias,
                        const T* __restrict__ res, size_t ldr, int act, T* __restrict__ y,
                        T* __restrict__ z) {
  constexpr int V = VEC ? 16 / (int)sizeof(T) : 1;
  const int lane = threadIdx.x & 31;
  const int n0 = (blockIdx.x * 4 + (threadIdx.x >> 5)) * SMALL_COLS;
  if (n0 >= N) return;
  const T* wr[SMALL_COLS];
  const T* xr[MT];
#pragma unroll
  for (int j = 0; j < SMALL_COLS; ++j) wr[j] = w + (size_t)min(n0 + j, N - 1) * ldw;
#pragma unroll
  for (int i = 0; i < MT; ++i) xr[i] = x + (size_t)min(i, M - 1) * ldx;
  float acc[MT * SMALL_COLS];
#pragma unroll
  for (int i = 0; i < MT * SMALL_COLS; ++i) acc[i] = 0.f;
  const int whole = K / V * V;
#pragma unroll 2
  for (int k = lane * V; k < whole; k += 32 * V) {
    float wv[SMALL_COLS][V];
#pragma unroll
    for (int j = 0; j < SMALL_COLS; ++j) load_n<VEC, V>(wr[j] + k, wv[j]);
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      float xv[V];
      load_n<VEC, V>(xr[i] + k, xv);
#pragma unroll
      for (int j = 0; j < SMALL_COLS; ++j)
#pragma unroll
        for (int q = 0; q < V; ++q)
          acc[i * SMALL_COLS + j] = fmaf(xv[q], wv[j][q], acc[i * SMALL_COLS + j]);
    }
  }
  if (whole + lane < K) {  // fewer than V values are left
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < SMALL_COLS; ++j)
        acc[i * SMALL_COLS + j] = fmaf(to_f(xr[i][whole + lane]), to_f(wr[j][whole + lane]),
                                       acc[i * SMALL_COLS + j]);
  }
  constexpr int C = MT * SMALL_COLS, REP = 32 / C;
  float v = scatter_sum<C>(acc, lane);
  const int id = lane / REP, m = id / SMALL_COLS, n = n0 + id % SMALL_COLS;
  if (lane % REP || m >= M || n >= N) return;
  v = add_rn(v, bias ? to_f(bias[n]) : 0.f);
  if (z) z[(size_t)m * N + n] = from_f<T>(v);
  v = activate1<sizeof(T) == 2>(v, act);
  y[(size_t)m * N + n] = from_f<T>(add_rn(v, res ? to_f(res[(size_t)m * ldr + n]) : 0.f));
}

template <typename T>
int launch_small(const T* x, size_t ldx, const T* w, size_t ldw, int M, int N, int K,
                 const T* bias, const T* res, size_t ldr, int act, T* y, T* z, cudaStream_t st) {
  const bool vec = (uintptr_t)x % 16 == 0 && (uintptr_t)w % 16 == 0 &&
                   (M == 1 || ldx * sizeof(T) % 16 == 0) && (N == 1 || ldw * sizeof(T) % 16 == 0);
  const unsigned grid = (unsigned)((N + 4 * SMALL_COLS - 1) / (4 * SMALL_COLS));
#define TW_SMALL(MT)                                                                             \
  (vec ? linear_small_kernel<T, MT, true><<<grid, 128, 0, st>>>(x, ldx, w, ldw, M, N, K, bias,   \
                                                                res, ldr, act, y, z)             \
       : linear_small_kernel<T, MT, false><<<grid, 128, 0, st>>>(x, ldx, w, ldw, M, N, K, bias,  \
                                                                 res, ldr, act, y, z))
  if (M == 1) TW_SMALL(1);
  else if (M == 2) TW_SMALL(2);
  else if (M <= 4) TW_SMALL(4);
  else TW_SMALL(8);
#undef TW_SMALL
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_error(kLaunch, "tw_linear_forward: %s", cudaGetErrorString(e));
  return kOk;
}

// ------------------------------------------- operands for the tensor cores

template <typename T> struct Packed {
  using E = T;
  static constexpr int PL = 1;
};
template <> struct Packed<float> {
  using E = __nv_bfloat16;
  static constexpr int PL = 3;
};

// x = p0 + p1 + p2 exactly (8 + 8 + 8 bits; from 2^-110 on), each the bfloat16 nearest to what
// is left: x becomes p0.  An infinity or NaN stays in p0.
__device__ __forceinline__ void split3(float& x, float& p1, float& p2) {
  float h = __bfloat162float(__float2bfloat16_rn(x));
  if (fabsf(h) == INFINITY)  // x rounded past the largest value, or is infinite
    h = __uint_as_float(__float_as_uint(x) & 0xFFFF0000u);
  const float r = fabsf(x) < INFINITY ? x - h : 0.f;
  p1 = __bfloat162float(__float2bfloat16_rn(r));
  p2 = r - p1;
  x = h;
}

constexpr int PACK_ROWS = 8, PACK_COLS = 256;  // rows and columns of a block's step

// One matrix to write as the tensor cores read it: src [R, C], or src *
// act'(z), in rows of Cp (a multiple of 8) values, in planes.  dst NULL: no
// copy; sums: column sums of each block's `rb` rows, in float32 before
// rounding, or NULL.
template <typename T> struct PackJob {
  const T* src;
  const T* z;
  typename Packed<T>::E* dst;
  float* sums;
  size_t ld, pitch, plane;
  int R, C, Cp, rb, vec, cols, first;  // blocks along the columns; number of the first block
};
// The matrices of a call go in one launch, side by side.
constexpr int MOST_JOBS = 3;
template <typename T> struct PackJobs {
  PackJob<T> j[MOST_JOBS];
  int count;
};

// Bound by HBM: each value is read once and written once, 8 neighbouring
// columns a thread; with 16-byte loads where the rows are aligned (`vec`).
// Single loads of neighbours still end in 16-byte stores: giving a thread
// every 32nd column instead made the stores single too and took 44 in place of
// 19 us for 7000 x 385 float32.
template <typename T, int ACT>
__device__ __forceinline__ void pack_block(const PackJob<T>& j, int bx, int by, float* s) {
  constexpr int PL = Packed<T>::PL;
  using E = typename Packed<T>::E;
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int c0 = bx * PACK_COLS + tx * 8, C = j.C;
  const int r0 = by * j.rb, r1 = r0 + min(j.R - r0, j.rb);  // (by + 1) rb may pass 2^31
  if (c0 >= j.Cp) return;
  const size_t ld = j.ld, pitch = j.pitch, plane = j.plane;
  const T* __restrict__ src = j.src + c0;
  const T* __restrict__ z = ACT == kActNone ? nullptr : j.z + c0;
  E* __restrict__ dst = j.dst;
  const bool vec = j.vec;
#pragma unroll 2
  for (int r = r0 + ty; r < r1; r += PACK_ROWS) {
    const T* p = src + (size_t)r * ld;
    const T* zp = ACT == kActNone ? nullptr : z + (size_t)r * C;
    float v[8], zv[8];
    if (vec) {  // then C is a multiple of 8
      load_n<true, 8>(p, v);
      if (ACT != kActNone) load_n<true, 8>(zp, zv);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[i] = c0 + i < C ? to_f(p[i]) : 0.f;
        if (ACT != kActNone) zv[i] = c0 + i < C ? to_f(zp[i]) : 0.f;
      }
    }
    if (ACT != kActNone)
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        const Vec<2> d = act_slope<ACT, sizeof(T) == 2>(Vec<2>{{zv[i], zv[i + 1]}});
        v[i] *= d.v[0];
        v[i + 1] *= d.v[1];
      }
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] += v[i];
    if (dst) {
      E* o = dst + (size_t)r * pitch + c0;
      if constexpr (PL == 3) {
        float p1[8], p2[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) split3(v[i], p1[i], p2[i]);
        *reinterpret_cast<uint4*>(o + plane) = pack16<E>(p1);
        *reinterpret_cast<uint4*>(o + 2 * plane) = pack16<E>(p2);
      }
      *reinterpret_cast<uint4*>(o) = pack16<E>(v);
    }
  }
}

// ACT is the first matrix's, the others have none: chosen at compile time it
// takes 128 us for 32768 x 4096 bfloat16 gelu, chosen inside 142.
template <typename T, int ACT>
__global__ void __launch_bounds__(256, 4)
    linear_pack_kernel(const __grid_constant__ PackJobs<T> jobs) {
  __shared__ float red[PACK_ROWS][PACK_COLS + 8];
  let_next_start();  // the first of a call: behind an ordinary launch
  int k = jobs.count - 1;
  while (k > 0 && (int)blockIdx.x < jobs.j[k].first) --k;
  const PackJob<T>& j = jobs.j[k];
  const int block = blockIdx.x - j.first, by = block / j.cols, bx = block - by * j.cols;
  float s[8] = {};
  if (k == 0) pack_block<T, ACT>(j, bx, by, s);
  else pack_block<T, kActNone>(j, bx, by, s);
  if (!j.sums) return;
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
#pragma unroll
  for (int i = 0; i < 8; ++i) red[ty][tx * 8 + i] = s[i];
  __syncthreads();
  const int c = bx * PACK_COLS + threadIdx.x;
  if (c < j.C) {
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < PACK_ROWS; ++i) t += red[i][threadIdx.x];
    j.sums[(size_t)by * j.C + c] = t;
  }
}

// db[c] = the blocks' column sums, in a fixed order: 32 columns a block, whose
// 32 warps share the rows.
template <typename T>
__global__ void __launch_bounds__(1024)
    linear_db_kernel(const float* __restrict__ sums, int blocks, int C, T* __restrict__ db) {
  __shared__ float red[32][33];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5, c = blockIdx.x * 32 + tx;
  float s = 0.f;
  after_previous();
  let_next_start();
  if (c < C)
#pragma unroll 8
    for (int b = ty; b < blocks; b += 32) s += sums[(size_t)b * C + c];
  red[ty][tx] = s;
  __syncthreads();
  s = red[tx][ty];  // warp ty sums column ty
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  const int col = blockIdx.x * 32 + ty;
  if (tx == 0 && col < C) db[col] = from_f<T>(s);
}

size_t up8(size_t n) { return (n + 7) / 8 * 8; }
// Elements from one packed row to the next: whole 128-byte lines, so that a
// line of a chunk is one of memory (7000 x 257 x 385 forward, rows of 264 or 320
// elements: float32 36 or 34 us, bfloat16 31 or 27).
size_t pitch_of(size_t n) { return (n + 63) / 64 * 64; }
size_t up256(size_t n) { return (n + 255) / 256 * 256; }

// Rows of a block of the pack kernel: 16, or more where that makes over 256
// blocks along the rows (their sums are read back).
int rows_per_block(int R) {
  const int rb = (R + 255) / 256;
  return rb < 16 ? 16 : (rb + 7) / 8 * 8;
}
int row_blocks(int R) {
  const int rb = rows_per_block(R);
  return (int)(((long long)R + rb - 1) / rb);
}

template <typename T>
bool tma_reads(const void* p, size_t ld, int rows, int cols) {
  return sizeof(T) == 2 && (uintptr_t)p % 16 == 0 &&
         (rows == 1 || (ld % 8 == 0 && ld >= (size_t)cols));
}

template <typename T>
size_t packed_bytes(int R, int C) {
  return up256((size_t)Packed<T>::PL * R * pitch_of(C) * 2);
}

int launched(const char* who) {
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_error(kLaunch, "%s: %s", who, cudaGetErrorString(e));
  return kOk;
}

// The matrices of a call to be packed, and how many blocks they take.
template <typename T> struct Packing {
  PackJobs<T> jobs = {};
  unsigned blocks = 0;
  int act = kActNone;  // of the first

  void add(const T* src, size_t ld, const T* z, int R, int C, void* dst, float* sums) {
    PackJob<T>& j = jobs.j[jobs.count++];
    j.src = src;
    j.z = z;
    j.dst = (typename Packed<T>::E*)dst;
    j.sums = sums;
    j.ld = ld;
    j.R = R;
    j.C = C;
    j.Cp = (int)up8(C);
    j.pitch = pitch_of(C);
    j.plane = (size_t)R * j.pitch;
    j.rb = rows_per_block(R);
    j.vec = C % 8 == 0 && (uintptr_t)src % 16 == 0 && ld * sizeof(T) % 16 == 0 &&
            (uintptr_t)z % 16 == 0;
    j.cols = (j.Cp + PACK_COLS - 1) / PACK_COLS;
    j.first = (int)blocks;
    blocks += (unsigned)(j.cols * row_blocks(R));
  }
  // src as an operand: as it lies, or packed into `ws` (taken when `packs`).
  GemmOperand operand(const T* src, size_t ld, int R, int C, bool k_major, bool packs, void* ws) {
    if (!packs) return {src, R == 1 ? up8(C) : ld, 0, R, C, k_major};
    add(src, ld, nullptr, R, C, ws, nullptr);
    return {ws, pitch_of(C), (size_t)R * pitch_of(C), R, C, k_major};
  }
  int run(const char* who, cudaStream_t st) {
    if (blocks) {
      auto kernel = act == kActRelu      ? linear_pack_kernel<T, kActRelu>
                    : act == kActGelu    ? linear_pack_kernel<T, kActGelu>
                    : act == kActSilu    ? linear_pack_kernel<T, kActSilu>
                    : act == kActSigmoid ? linear_pack_kernel<T, kActSigmoid>
                                         : linear_pack_kernel<T, kActNone>;
      kernel<<<blocks, 256, 0, st>>>(jobs);
    }
    return launched(who);
  }
};

size_t partial_bytes(int M, int N, int K, int planes) {
  const GemmPlan p = gemm_plan(M, N, K, planes);
  return p.splits > 1 ? up256((size_t)p.splits * M * N * sizeof(float)) : 0;
}

// Workspace of a call, in this order.
struct Layout {
  size_t dz, x, w, sums, partial, total;
};

template <typename T>
Layout layout(int M, int N, int K, int act, bool backward, bool pack_dy, bool pack_x, bool pack_w) {
  constexpr int PL = Packed<T>::PL;
  Layout l = {};
  if (M <= 0 || (!backward && M <= SMALL_ROWS)) return l;
  size_t at = 0;
  l.dz = at;
  if (backward && (act != kActNone || pack_dy)) at += packed_bytes<T>(M, N);
  l.x = at;
  if (pack_x) at += packed_bytes<T>(M, K);
  l.w = at;
  if (pack_w) at += packed_bytes<T>(N, K);
  l.sums = at;
  if (backward) at += up256((size_t)row_blocks(M) * N * sizeof(float));
  l.partial = at;
  if (backward) {
    const size_t a = partial_bytes(M, K, N, PL), b = partial_bytes(N, K, M, PL);
    at += a > b ? a : b;
  } else {
    at += partial_bytes(M, N, K, PL);
  }
  l.total = at;
  return l;
}

int check(const char* who, int M, int N, int K, int act) {
  if (M < 0 || N <= 0 || K <= 0)
    return set_error(kInvalid, "%s: invalid sizes M=%d N=%d K=%d (need M >= 0, N, K > 0)", who, M,
                     N, K);
  if (act < kActNone || act > kActSigmoid)
    return set_error(kInvalid, "%s: unknown activation %d", who, act);
  if (M > 0x7fffffff - 512 || N > 0x7fffffff - 512 || K > 0x7fffffff - 512)
    return set_error(kUnsupported, "%s: a size is too large", who);
  return kOk;
}

int check_ws(const char* who, size_t have, size_t need, const void* ws) {
  if (have < need || (need && (!ws || (uintptr_t)ws % 256)))
    return set_error(kWorkspace, "%s: workspace needs %zu bytes, 256-byte aligned", who, need);
  return kOk;
}

template <typename T>
int fwd(const void* xv, size_t ldx, const void* wv, size_t ldw, const void* bias, const void* res,
        size_t ldr, int M, int N, int K, int act, void* y, void* z, void* ws, size_t ws_bytes,
        void* stream) {
  set_error(kOk, "%s", "");
  if (int e = check("tw_linear_forward", M, N, K, act)) return e;
  if (M == 0) return kOk;
  if (!xv || !wv || !y) return set_error(kInvalid, "tw_linear_forward: null pointer argument");
  cudaStream_t st = (cudaStream_t)stream;
  const T* x = (const T*)xv;
  const T* w = (const T*)wv;
  if (M <= SMALL_ROWS)
    return launch_small<T>(x, ldx, w, ldw, M, N, K, (const T*)bias, (const T*)res, ldr, act,
                           (T*)y, (T*)z, st);
  const bool px = !tma_reads<T>(x, ldx, M, K), pw = !tma_reads<T>(w, ldw, N, K);
  const Layout l = layout<T>(M, N, K, act, false, false, px, pw);
  if (int e = check_ws("tw_linear_forward", ws_bytes, l.total, ws)) return e;
  char* base = (char*)ws;
  GemmProblem p = {};
  Packing<T> packing;
  p.a = packing.operand(x, ldx, M, K, true, px, base + l.x);
  p.b = packing.operand(w, ldw, N, K, true, pw, base + l.w);
  p.M = M;
  p.N = N;
  p.K = K;
  p.bias = bias;
  p.residual = res;
  p.ldr = ldr;
  p.act = act;
  p.out = y;
  p.z = act == kActNone ? nullptr : z;
  p.partial = (float*)(base + l.partial);
  if (int e = packing.run("tw_linear_forward", st)) return e;
  p.after = packing.blocks != 0;
  return gemm_run<T>(p, st);
}

template <typename T>
int bwd(const void* dyv, size_t ldy, const void* xv, size_t ldx, const void* wv, size_t ldw,
        const void* z, int M, int N, int K, int act, void* dx, void* dw, void* db, void* ws,
        size_t ws_bytes, void* stream) {
  set_error(kOk, "%s", "");
  if (int e = check("tw_linear_backward", M, N, K, act)) return e;
  const T* dy = (const T*)dyv;
  const T* x = (const T*)xv;
  const T* w = (const T*)wv;
  if (M && (!dy || (dx && !w) || (dw && !x) || (act != kActNone && !z)))
    return set_error(kInvalid, "tw_linear_backward: null pointer argument");
  cudaStream_t st = (cudaStream_t)stream;
  if (M == 0) {  // sums over no rows
    if (dw) cudaMemsetAsync(dw, 0, (size_t)N * K * sizeof(T), st);
    if (db) cudaMemsetAsync(db, 0, (size_t)N * sizeof(T), st);
    return launched("tw_linear_backward");
  }
  const bool px = dw && !tma_reads<T>(x, ldx, M, K), pw = dx && !tma_reads<T>(w, ldw, N, K);
  const bool pdy = !tma_reads<T>(dy, ldy, M, N);
  const Layout l = layout<T>(M, N, K, act, true, pdy, px, pw);
  if (int e = check_ws("tw_linear_backward", ws_bytes, l.total, ws)) return e;
  char* base = (char*)ws;
  const bool packs = (dx || dw) && (act != kActNone || pdy);
  float* sums = db ? (float*)(base + l.sums) : nullptr;
  Packing<T> packing;
  if (packs || db) {
    packing.add(dy, ldy, (const T*)z, M, N, packs ? base + l.dz : nullptr, sums);
    packing.act = act;
  }
  GemmOperand dz = {dy, M == 1 ? up8(N) : ldy, 0, M, N, true};
  if (packs) dz = {base + l.dz, pitch_of(N), (size_t)M * pitch_of(N), M, N, true};
  GemmOperand bw = {}, bx = {};
  if (dx) bw = packing.operand(w, ldw, N, K, false, pw, base + l.w);
  if (dw) bx = packing.operand(x, ldx, M, K, false, px, base + l.x);
  if (int e = packing.run("tw_linear_backward", st)) return e;
  if (db) {
    const cudaError_t e = launch_after(true, linear_db_kernel<T>, dim3((N + 31) / 32), dim3(1024),
                                       0, 1, st, (const float*)sums, row_blocks(M), N, (T*)db);
    if (e != cudaSuccess)
      return set_error(kLaunch, "tw_linear_backward: %s", cudaGetErrorString(e));
  }
  GemmProblem p = {};
  p.after = packing.blocks != 0;
  p.partial = (float*)(base + l.partial);
  if (dx) {
    p.a = dz;
    p.b = bw;
    p.M = M;
    p.N = K;
    p.K = N;
    p.out = dx;
    if (int e = gemm_run<T>(p, st)) return e;
    p.after = true;
  }
  if (dw) {
    p.a = dz;
    p.a.k_major = false;
    p.b = bx;
    p.M = N;
    p.N = K;
    p.K = M;
    p.out = dw;
    if (int e = gemm_run<T>(p, st)) return e;
  }
  return launched("tw_linear_backward");
}

}  // namespace

// Errors of the product's kernels, of all types.
int linear_take_device_error() {
  const int a = gemm_take_device_error<float>(), b = gemm_take_device_error<__nv_bfloat16>(),
            c = gemm_take_device_error<__half>();
  return a != 0 ? a : b != 0 ? b : c;
}

}  // namespace tw

extern "C" {

size_t tw_linear_workspace_bytes(int M, int N, int K, int dtype_bytes, int act, int backward,
                                 int unaligned) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  const bool u = unaligned != 0;
  if (dtype_bytes == 4) return tw::layout<float>(M, N, K, act, backward != 0, true, true, true).total;
  return tw::layout<__nv_bfloat16>(M, N, K, act, backward != 0, u || N % 8, u || K % 8,
                                   u || K % 8).total;
}

#define TW_LINEAR(SUFFIX, T)                                                                     \
  int tw_linear_forward_##SUFFIX(const void* x, size_t ldx, const void* w, size_t ldw,           \
                                 const void* bias, const void* residual, size_t ldr, int M,      \
                                 int N, int K, int act, void* y, void* z, void* workspace,       \
                                 size_t ws_bytes, void* stream) {                                \
    return tw::fwd<T>(x, ldx, w, ldw, bias, residual, ldr, M, N, K, act, y, z, workspace,        \
                      ws_bytes, stream);                                                         \
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
