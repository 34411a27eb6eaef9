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
// One pass over the data.  The channels of all sequences, c = b D + d, are
// numbered through; a block of 128 threads owns 32 lanes of channel pairs (or
// 16, or 8) and walks time in tiles of 4 (8, 16) runs of 8 frames.  A thread
// reads its 8 frames into registers, composes them to (A, B) with h_out = A
// h_in + B, learns its h_in from the runs before it, and goes over its frames
// again in registers to write the outputs.  Few channels: up to 8 blocks of a
// cluster take neighbouring tiles and compose their (A, B) through each
// other's shared memory, so that a long sequence still fills the GPU.
// Everything is summed in a fixed order.
//
// The forward saves h before every 8th frame in float32 (0.5 bytes a value);
// the backward recomputes the states of a thread's frames from it, so no
// rounded output enters a gradient and the outputs are not read again.  8
// frames of two channels, the next tile's loads under way among them, fit 128
// registers; 16 did not (32 x 1024 x 1024 bfloat16: 200 us with the spills).
#include "../../include/torchwarp_b200.h"
#include "element.cuh"

namespace tw {
namespace {

constexpr int SCAN_FRAMES = 8;  // of a thread
constexpr int SCAN_THREADS = 128;
// LPR lanes a frame: 128 / LPR runs a tile.
constexpr int tile_of(int lpr) { return SCAN_THREADS / lpr * SCAN_FRAMES; }

__device__ __forceinline__ int live_len(const int64_t* lengths, int b, int T) {
  if (!lengths) return T;
  const long long n = lengths[b];
  return n < 0 ? 0 : n > T ? T : (int)n;
}

// A gate as one number n: the smaller of 1 - f and f, which keeps its relative
// precision, negative when it is 1 - f.  -0 keeps the state.
template <int V>
__device__ __forceinline__ Vec<V> gate_of(Vec<V> z) {
  const Vec<V> t = mul_v(z, splat<V>(1.4426950408889634f));
  Vec<V> e, r;
#pragma unroll
  for (int i = 0; i < V; ++i) e.v[i] = ex2(-fabsf(t.v[i]));
  r = add_v(e, splat<V>(1.f));
#pragma unroll
  for (int i = 0; i < V; ++i) r.v[i] = rcp(r.v[i]);
  r = mul_v(e, r);
#pragma unroll
  for (int i = 0; i < V; ++i)
    r.v[i] = __uint_as_float((__float_as_uint(r.v[i]) & 0x7FFFFFFFu) |
                             (~__float_as_uint(z.v[i]) & 0x80000000u));
  return r;
}
// a where n is 1 - f, b where it is f.
template <int V>
__device__ __forceinline__ Vec<V> pick(Vec<V> n, Vec<V> a, Vec<V> b) {
  Vec<V> r;
#pragma unroll
  for (int i = 0; i < V; ++i) r.v[i] = __float_as_int(n.v[i]) < 0 ? a.v[i] : b.v[i];
  return r;
}
// f h + (1 - f) x as a step from the nearer of the two, so that the rounding
// of a gate near 1 does not decay a state that should last: h - (1 - f)(h - x)
// or x + f (h - x).  diff is h - x.
template <int V>
__device__ __forceinline__ Vec<V> advance(Vec<V> n, Vec<V> h, Vec<V> x, Vec<V> diff) {
  return fma_v(n, diff, pick(n, h, x));
}
// f l, likewise.
template <int V>
__device__ __forceinline__ Vec<V> decay(Vec<V> n, Vec<V> l) {
  return fma_v(n, l, pick(n, l, splat<V>(0.f)));
}
// (1 - f) l, from -l.
template <int V>
__device__ __forceinline__ Vec<V> passed(Vec<V> n, Vec<V> l, Vec<V> neg_l) {
  return fma_v(n, neg_l, pick(n, splat<V>(0.f), l));
}

// VC neighbouring channels of a frame, as they lie in memory.
template <typename T, int VC> struct Frame {
  T t;
  __device__ __forceinline__ Vec<1> get() const { return {{to_f(t)}}; }
  static __device__ __forceinline__ Frame zero() { return {from_f<T>(0.f)}; }
  static __device__ __forceinline__ Frame of(Vec<1> v) { return {from_f<T>(v.v[0])}; }
};
template <> struct Frame<float, 2> {
  float2 t;
  __device__ __forceinline__ Vec<2> get() const { return {{t.x, t.y}}; }
  static __device__ __forceinline__ Frame zero() { return {make_float2(0.f, 0.f)}; }
  static __device__ __forceinline__ Frame of(Vec<2> v) { return {make_float2(v.v[0], v.v[1])}; }
};
template <typename T> struct Frame<T, 2> {
  uint32_t u;
  __device__ __forceinline__ Vec<2> get() const {
    Vec<2> r;
    Pair<T>::unpack(u, r.v[0], r.v[1]);
    return r;
  }
  static __device__ __forceinline__ Frame zero() { return {0u}; }
  static __device__ __forceinline__ Frame of(Vec<2> v) { return {Pair<T>::pack(v.v[0], v.v[1])}; }
};

// p + step, hidden from the compiler: it would otherwise keep the addresses of
// all frames of all arrays in registers at once, 70 of them.
template <typename P, typename S>
__device__ __forceinline__ void walk(P*& p, S step) {
  p += step;
  asm("" : "+l"(p));
}

// A thread's frames from p on, `step` bytes apart; frames from `n` on are zero
// and not read.
template <typename T, int VC>
__device__ __forceinline__ void load_frames(Frame<T, VC> (&f)[SCAN_FRAMES], const char* p,
                                            size_t step, int n) {
  if (n >= SCAN_FRAMES) {
#pragma unroll
    for (int k = 0; k < SCAN_FRAMES; ++k) {
      f[k] = *reinterpret_cast<const Frame<T, VC>*>(p);
      walk(p, step);
    }
  } else {
#pragma unroll
    for (int k = 0; k < SCAN_FRAMES; ++k) {
      f[k] = k < n ? *reinterpret_cast<const Frame<T, VC>*>(p) : Frame<T, VC>::zero();
      walk(p, step);
    }
  }
}

__device__ __forceinline__ float peer_read(const float* p, uint32_t rank) {
  uint32_t a;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <int VC, int LPR> struct ScanShared {
  static constexpr int RUNS = SCAN_THREADS / LPR, CH = LPR * VC;
  float a[2][RUNS][CH], b[2][RUNS][CH];  // of the runs
  float tile_a[2][CH], tile_b[2][CH];    // of the block's tile
  float start[2][CH];                    // before the tile
};

// Composes the runs' (A, B) of step `it` and returns what enters this
// thread's frames; REV: time goes from the last run and the last block of the
// cluster.  `run` is what enters the cluster's tiles, kept by run 0's threads.
// One block barrier a step when S is 1 (the buffers alternate), else one of
// the cluster and one more of the block.
template <int VC, int LPR, bool REV>
__device__ __forceinline__ void compose(ScanShared<VC, LPR>& sh, int it, int S, int rank, int part,
                                        int lane, Vec<VC> A, Vec<VC> B, Vec<VC>& run,
                                        Vec<VC>& enter) {
  constexpr int RUNS = ScanShared<VC, LPR>::RUNS;
  const int p = it & 1;
#pragma unroll
  for (int v = 0; v < VC; ++v) {
    sh.a[p][part][lane * VC + v] = A.v[v];
    sh.b[p][part][lane * VC + v] = B.v[v];
  }
  __syncthreads();
  if (S > 1) {
    if (part == 0) {
#pragma unroll
      for (int v = 0; v < VC; ++v) {
        float ta = 1.f, tb = 0.f;
#pragma unroll
        for (int i = 0; i < RUNS; ++i) {
          const int w = REV ? RUNS - 1 - i : i;
          const float wa = sh.a[p][w][lane * VC + v];
          tb = fmaf(wa, tb, sh.b[p][w][lane * VC + v]);
          ta *= wa;
        }
        sh.tile_a[p][lane * VC + v] = ta;
        sh.tile_b[p][lane * VC + v] = tb;
      }
    }
    cluster_sync_all();
    if (part == 0) {
#pragma unroll
      for (int v = 0; v < VC; ++v) {
        float ta[8], tb[8];
#pragma unroll
        for (int r = 0; r < 8; ++r)
          if (r < S) {
            ta[r] = peer_read(&sh.tile_a[p][lane * VC + v], r);
            tb[r] = peer_read(&sh.tile_b[p][lane * VC + v], r);
          }
        float h = run.v[v];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int r = REV ? 7 - i : i;
          if (r < S) {
            if (r == rank) sh.start[p][lane * VC + v] = h;
            h = fmaf(ta[r], h, tb[r]);
          }
        }
        run.v[v] = h;
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int v = 0; v < VC; ++v) {
    float h = sh.start[p][lane * VC + v];
#pragma unroll
    for (int i = 0; i < RUNS; ++i) {
      const int w = REV ? RUNS - 1 - i : i;
      if (REV ? w > part : w < part)
        h = fmaf(sh.a[p][w][lane * VC + v], h, sh.b[p][w][lane * VC + v]);
    }
    enter.v[v] = h;
  }
}

// What a block works on: its channels' sequence, feature and length.
struct Channel {
  size_t c, b, d;
  bool live;
  int L;
  __device__ __forceinline__ Channel(size_t first, int lane, int vc, size_t BD, int D, int TT,
                                     const int64_t* lengths) {
    c = first + lane * vc;
    live = c < BD;
    b = live ? c / D : 0;
    d = live ? c - b * D : 0;
    L = live ? live_len(lengths, (int)b, TT) : 0;
  }
};

template <typename T, int VC, int LPR>
__global__ void __launch_bounds__(SCAN_THREADS, 4)
    scan_fwd_kernel(const T* __restrict__ x, size_t xb, size_t xt, const T* __restrict__ g,
                    size_t gb, size_t gt, const float* __restrict__ h0,
                    const int64_t* __restrict__ lengths, size_t BD, int TT, int D, int S,
                    T* __restrict__ y, float* __restrict__ state, float* __restrict__ carry) {
  constexpr int TILE = tile_of(LPR);
  __shared__ ScanShared<VC, LPR> sh;
  const int part = threadIdx.x / LPR, lane = threadIdx.x & (LPR - 1);
  const int rank = blockIdx.x % S;
  const Channel ch((size_t)(blockIdx.x / S) * (LPR * VC), lane, VC, BD, D, TT, lengths);
  const char* xp = reinterpret_cast<const char*>(x + ch.b * xb + ch.d);
  const char* gp = reinterpret_cast<const char*>(g + ch.b * gb + ch.d);
  char* yp = reinterpret_cast<char*>(y + ch.b * (size_t)TT * D + ch.d);
  const size_t xs = xt * sizeof(T), gs = gt * sizeof(T), ys = D * sizeof(T);
  Vec<VC> run;
#pragma unroll
  for (int v = 0; v < VC; ++v) {
    run.v[v] = ch.live && h0 ? h0[ch.c + v] : 0.f;
    if (part == 0) sh.start[0][lane * VC + v] = run.v[v];
  }
  const int steps = (TT + TILE * S - 1) / (TILE * S);
  int t0 = rank * TILE + part * SCAN_FRAMES;
  Frame<T, VC> xr[SCAN_FRAMES], gr[SCAN_FRAMES];
  load_frames<T, VC>(gr, gp + (size_t)t0 * gs, gs, ch.L - t0);
  load_frames<T, VC>(xr, xp + (size_t)t0 * xs, xs, ch.L - t0);
  for (int it = 0; it < steps; ++it, t0 += TILE * S) {
    const int n = ch.L - t0;
    Vec<VC> s[SCAN_FRAMES];
    Frame<T, VC> xk[SCAN_FRAMES];  // as it lies: pairs in one register
#pragma unroll
    for (int k = 0; k < SCAN_FRAMES; ++k) {
      s[k] = gate_of(gr[k].get());
      xk[k] = xr[k];
    }
    if (n < SCAN_FRAMES)
#pragma unroll
      for (int k = 0; k < SCAN_FRAMES; ++k)
        if (k >= n) s[k] = splat<VC>(-0.f);
    // the next tile's loads are under way while the blocks wait for each other
    const int t1 = t0 + TILE * S;
    load_frames<T, VC>(gr, gp + (size_t)t1 * gs, gs, ch.L - t1);
    load_frames<T, VC>(xr, xp + (size_t)t1 * xs, xs, ch.L - t1);
    Vec<VC> A = splat<VC>(1.f), B = splat<VC>(0.f), h;
#pragma unroll
    for (int k = 0; k < SCAN_FRAMES; ++k) {
      const Vec<VC> x = xk[k].get();
      B = advance(s[k], B, x, sub_v(B, x));
      A = decay(s[k], A);
    }
    compose<VC, LPR, false>(sh, it, S, rank, part, lane, A, B, run, h);
    if (carry && ch.live && t0 < TT)
#pragma unroll
      for (int v = 0; v < VC; ++v)
        carry[(size_t)(t0 / SCAN_FRAMES) * BD + ch.c + v] = h.v[v];
    char* o = yp + (size_t)t0 * ys;
    if (n >= SCAN_FRAMES) {
#pragma unroll
      for (int k = 0; k < SCAN_FRAMES; ++k) {
        const Vec<VC> x = xk[k].get();
        h = advance(s[k], h, x, sub_v(h, x));
        *reinterpret_cast<Frame<T, VC>*>(o) = Frame<T, VC>::of(h);
        walk(o, ys);
      }
    } else {
#pragma unroll
      for (int k = 0; k < SCAN_FRAMES; ++k) {
        const Vec<VC> x = xk[k].get();
        h = advance(s[k], h, x, sub_v(h, x));
        if (ch.live && t0 + k < TT)
          *reinterpret_cast<Frame<T, VC>*>(o) = k < n ? Frame<T, VC>::of(h) : Frame<T, VC>::zero();
        walk(o, ys);
      }
    }
    if (S == 1 && part == SCAN_THREADS / LPR - 1)
#pragma unroll
      for (int v = 0; v < VC; ++v) sh.start[(it + 1) & 1][lane * VC + v] = h.v[v];
  }
  __syncthreads();
  if (ch.live && part == 0 && rank == 0)
#pragma unroll
    for (int v = 0; v < VC; ++v)
      state[ch.c + v] = S > 1 ? run.v[v] : sh.start[steps & 1][lane * VC + v];
  if (S > 1) cluster_sync_all();  // the others may still read this block's tile
}

// The same walk from the end.
template <typename T, int VC, int LPR>
__global__ void __launch_bounds__(SCAN_THREADS, 4)
    scan_bwd_kernel(const T* __restrict__ dy, size_t yb, size_t yt,
                    const float* __restrict__ dstate, const T* __restrict__ x, size_t xb,
                    size_t xt, const T* __restrict__ g, size_t gb, size_t gt,
                    const int64_t* __restrict__ lengths, const float* __restrict__ carry,
                    size_t BD, int TT, int D, int S, T* __restrict__ dx, T* __restrict__ dg,
                    float* __restrict__ dh0) {
  constexpr int TILE = tile_of(LPR);
  __shared__ ScanShared<VC, LPR> sh;
  const int part = threadIdx.x / LPR, lane = threadIdx.x & (LPR - 1);
  const int rank = blockIdx.x % S;
  const Channel ch((size_t)(blockIdx.x / S) * (LPR * VC), lane, VC, BD, D, TT, lengths);
  const char* xp = reinterpret_cast<const char*>(x + ch.b * xb + ch.d);
  const char* gp = reinterpret_cast<const char*>(g + ch.b * gb + ch.d);
  const char* yp = reinterpret_cast<const char*>(dy + ch.b * yb + ch.d);
  const size_t at = ch.b * (size_t)TT * D + ch.d;
  const size_t xs = xt * sizeof(T), gs = gt * sizeof(T), ys = yt * sizeof(T);
  const ptrdiff_t os = (ptrdiff_t)(D * sizeof(T));
  Vec<VC> run;  // f_{t+1} lam_{t+1} beyond the frames done
#pragma unroll
  for (int v = 0; v < VC; ++v) {
    run.v[v] = ch.live && dstate ? dstate[ch.c + v] : 0.f;
    if (part == 0) sh.start[0][lane * VC + v] = run.v[v];
  }
  const int steps = (TT + TILE * S - 1) / (TILE * S);
  int t0 = ((steps - 1) * S + rank) * TILE + part * SCAN_FRAMES;
  Frame<T, VC> xr[SCAN_FRAMES], gr[SCAN_FRAMES], yr[SCAN_FRAMES];
  Vec<VC> hr;
  auto load = [&](int t) {
    const int n = t >= 0 ? ch.L - t : 0;
    const size_t tt = t >= 0 ? t : 0;
    load_frames<T, VC>(gr, gp + tt * gs, gs, n);
    load_frames<T, VC>(yr, yp + tt * ys, ys, n);
    load_frames<T, VC>(xr, xp + tt * xs, xs, n);
#pragma unroll
    for (int v = 0; v < VC; ++v)
      hr.v[v] = n > 0 ? carry[(tt / SCAN_FRAMES) * BD + ch.c + v] : 0.f;
  };
  load(t0);
  for (int it = 0; it < steps; ++it, t0 -= TILE * S) {
    const int n = ch.L - t0;
    Vec<VC> s[SCAN_FRAMES], diff[SCAN_FRAMES];  // the gates; h_{t-1} - x_t
    Vec<VC> h = hr, lam;
    Frame<T, VC> yk[SCAN_FRAMES];
#pragma unroll
    for (int k = 0; k < SCAN_FRAMES; ++k) {
      s[k] = gate_of(gr[k].get());
      yk[k] = yr[k];
    }
    if (n < SCAN_FRAMES)
#pragma unroll
      for (int k = 0; k < SCAN_FRAMES; ++k)
        if (k >= n) s[k] = splat<VC>(-0.f);
#pragma unroll
    for (int k = 0; k < SCAN_FRAMES; ++k) {
      const Vec<VC> x = xr[k].get();
      diff[k] = sub_v(h, x);
      h = advance(s[k], h, x, diff[k]);
    }
    load(t0 - TILE * S);  // under way while the blocks wait for each other
    Vec<VC> A = splat<VC>(1.f), B = splat<VC>(0.f);
#pragma unroll
    for (int k = SCAN_FRAMES - 1; k >= 0; --k) {
      B = decay(s[k], add_v(yk[k].get(), B));
      A = decay(s[k], A);
    }
    compose<VC, LPR, true>(sh, it, S, rank, part, lane, A, B, run, lam);
    const size_t last = (at + (size_t)(t0 + SCAN_FRAMES - 1) * D) * sizeof(T);
    char* ox = reinterpret_cast<char*>(dx) + last;
    char* og = reinterpret_cast<char*>(dg) + last;
#pragma unroll
    for (int k = SCAN_FRAMES - 1; k >= 0; --k) {
      const Vec<VC> l = add_v(yk[k].get(), lam);
      lam = decay(s[k], l);
      const Vec<VC> pass = passed(s[k], l, negated(l));
      const Frame<T, VC> vx = Frame<T, VC>::of(pass);
      // f (1 - f) l (h - x)
      const Frame<T, VC> vg = Frame<T, VC>::of(mul_v(decay(s[k], pass), diff[k]));
      if (n >= SCAN_FRAMES) {
        *reinterpret_cast<Frame<T, VC>*>(ox) = vx;
        *reinterpret_cast<Frame<T, VC>*>(og) = vg;
      } else if (ch.live && t0 + k < TT) {
        *reinterpret_cast<Frame<T, VC>*>(ox) = k < n ? vx : Frame<T, VC>::zero();
        *reinterpret_cast<Frame<T, VC>*>(og) = k < n ? vg : Frame<T, VC>::zero();
      }
      walk(ox, -os);
      walk(og, -os);
    }
    if (S == 1 && part == 0)
#pragma unroll
      for (int v = 0; v < VC; ++v) sh.start[(it + 1) & 1][lane * VC + v] = lam.v[v];
  }
  __syncthreads();
  if (ch.live && dh0 && part == 0 && rank == 0)
#pragma unroll
    for (int v = 0; v < VC; ++v)
      dh0[ch.c + v] = S > 1 ? run.v[v] : sh.start[steps & 1][lane * VC + v];
  if (S > 1) cluster_sync_all();
}

template <typename T>
__global__ void __launch_bounds__(SCAN_THREADS)
    scan_step_kernel(const T* __restrict__ x, size_t xs, const T* __restrict__ g, size_t gs,
                     float* __restrict__ state, int B, int D, T* __restrict__ y) {
  const size_t id = (size_t)blockIdx.x * SCAN_THREADS + threadIdx.x;
  if (id >= (size_t)B * D) return;
  const size_t b = id / D, d = id - b * D;
  const Vec<1> n = gate_of(Vec<1>{{to_f(g[b * gs + d])}});
  const Vec<1> was = {{state[id]}}, in = {{to_f(x[b * xs + d])}};
  const float h = advance(n, was, in, sub_v(was, in)).v[0];
  state[id] = h;
  y[id] = from_f<T>(h);
}

int check(const char* who, int B, int TT, int D) {
  if (B < 0 || TT < 0 || D <= 0)
    return set_error(kInvalid, "%s: invalid sizes B=%d T=%d D=%d (need B, T >= 0, D > 0)", who, B,
                     TT, D);
  if ((size_t)B * D / 8 >= 0x7fffffffu / 8 || TT > 0x7fffffff - 8 * 128)
    return set_error(kUnsupported, "%s: sizes too large", who);
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

// How the channels and the time of a call are spread over blocks: 32 lanes of
// channels a frame while that gives the SMs three blocks each; else more
// blocks take part of the time, as many as there are tiles; else fewer lanes.
struct ScanPlan {
  int lpr, S;
  size_t groups;
};
ScanPlan scan_plan(size_t BD, int vc, int TT) {
  ScanPlan p = {32, 1, 0};
  for (;; p.lpr /= 2) {
    p.groups = (BD + p.lpr * vc - 1) / (p.lpr * vc);
    p.S = 1;
    while (p.S < 8 && p.groups * p.S < 148 * 3 && (long long)p.S * tile_of(p.lpr) < TT) p.S *= 2;
    if (p.lpr == 8 || p.groups * p.S >= 148 * 3) return p;
  }
}

template <typename... Params, typename... Args>
int launch(const char* who, void (*kernel)(Params...), size_t groups, int S, void* stream,
           Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(groups * S));
  cfg.blockDim = dim3(SCAN_THREADS);
  cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = S;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = S > 1 ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  if (e != cudaSuccess) return set_error(kLaunch, "%s: %s", who, cudaGetErrorString(e));
  return kOk;
}

template <typename T>
bool pairs_ok(const void* p, size_t s1, size_t s2) {
  return (uintptr_t)p % (2 * sizeof(T)) == 0 && s1 % 2 == 0 && s2 % 2 == 0;
}

// The instance of a kernel for plan p and `pairs`.
#define TW_SCAN_KERNEL(KERNEL)                                                   \
  (pairs ? (p.lpr == 32 ? KERNEL<T, 2, 32> : p.lpr == 16 ? KERNEL<T, 2, 16>      \
                                                         : KERNEL<T, 2, 8>)      \
         : (p.lpr == 32 ? KERNEL<T, 1, 32> : p.lpr == 16 ? KERNEL<T, 1, 16>      \
                                                         : KERNEL<T, 1, 8>))

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
  const char* who = "tw_gated_scan_forward";
  const size_t BD = (size_t)B * D;
  const bool pairs = D % 2 == 0 && pairs_ok<T>(x, xb, xt) && pairs_ok<T>(g, gb, gt) &&
                     pairs_ok<T>(y, 0, 0);
  const ScanPlan p = scan_plan(BD, pairs ? 2 : 1, TT);
  return launch(who, TW_SCAN_KERNEL(scan_fwd_kernel), p.groups, p.S, stream, (const T*)x, xb, xt,
                (const T*)g, gb, gt, h0, lengths, BD, TT, D, p.S, (T*)y, state, (float*)carry);
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
  const char* who = "tw_gated_scan_backward";
  const size_t BD = (size_t)B * D;
  const bool pairs = D % 2 == 0 && pairs_ok<T>(x, xb, xt) && pairs_ok<T>(g, gb, gt) &&
                     pairs_ok<T>(dy, yb, yt) && pairs_ok<T>(dx, 0, 0) && pairs_ok<T>(dg, 0, 0);
  const ScanPlan p = scan_plan(BD, pairs ? 2 : 1, TT);
  return launch(who, TW_SCAN_KERNEL(scan_bwd_kernel), p.groups, p.S, stream, (const T*)dy, yb, yt,
                dstate, (const T*)x, xb, xt, (const T*)g, gb, gt, lengths, (const float*)carry, BD,
                TT, D, p.S, (T*)dx, (T*)dg, dh0);
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
  return (size_t)B * D * ((T + tw::SCAN_FRAMES - 1) / tw::SCAN_FRAMES) * sizeof(float);
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
