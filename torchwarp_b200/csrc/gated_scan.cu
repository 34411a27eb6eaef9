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
// numbered through; a block owns a line of them (128 or 64 bytes a frame, two
// channels a lane) and walks time in tiles, which cp.async brings to shared
// memory while the ones before are worked on.  A thread takes runs of 16 frames
// (8 of float32) and writes the outputs in the place of the inputs, from where
// whole 16-byte pieces go out.  Two ways to walk:
//   alone (16 bits, forward, many lines): a block is one warp, a tile one run;
//   the state passes from run to run in registers.
//   composed: a block is 128 threads, a tile 4 to 16 runs.  A thread composes the
//   frames of its run to (A, B) with h_out = A h_in + B, learns its h_in from the
//   runs before it, and goes over its frames again.
// Few channels: time is cut into segments, a first kernel composes each to one
// (A, B), and a segment's blocks start from what the segments before them give.
// That reads two arrays twice, and still takes 34 us forward and 50 us backward
// for 1 x 32768 x 256 float32, where 8 blocks of a cluster, exchanging (A, B) at
// every tile, took 105 and 127: a step of those waits for the slowest of the 8.
// Everything is summed in a fixed order.
//
// 32 x 1024 x 1024: float32 75 us forward and 121 backward, 82% and 85% of what
// a copy of the same bytes takes; bfloat16 53 (alone) and 73 (composed), where
// the bytes are half and the instructions, some 30 a value composed (gate,
// composition, second walk), are not: with the few warps that 512 lines give an
// SM the schedulers issue in 55 to 60% of their cycles.
//
// The forward saves h before every run in float32 (0.25 bytes a 16-bit value,
// 0.5 a float32 one); the backward recomputes the states of a run from it, so
// no rounded output enters a gradient and the outputs are not read again.
//
// Rows that are not 16-byte aligned take a second form, one channel a lane,
// whose frames go through registers: there each frame's address costs the
// instructions that a 16-byte copy shares among 4 to 8 values.  Its long
// sequences of few channels are shared by up to 8 blocks of a cluster, which
// take neighbouring tiles and compose their (A, B) through each other's shared
// memory (1 x 32768 x 257 float32: 121 us forward, 155 backward).
#include "../../include/torchwarp_b200.h"
#include "element.cuh"

namespace tw {
namespace {

constexpr int SCAN_THREADS = 128;
// Frames of a run: what a thread holds of the gates (and in the backward of
// the differences) of two channels without spilling.
constexpr int frames_of(size_t type_bytes) { return type_bytes == 4 ? 8 : 16; }
// LPR lanes a frame: 128 / LPR runs a tile.
constexpr int tile_of(int lpr, size_t type_bytes) {
  return SCAN_THREADS / lpr * frames_of(type_bytes);
}

__device__ __forceinline__ int live_len(const int64_t* lengths, int b, int T) {
  if (!lengths) return T;
  const long long n = lengths[b];
  return n < 0 ? 0 : n > T ? T : (int)n;
}

// A gate as one number n: the smaller of 1 - f and f, which keeps its relative
// precision, negative when it is 1 - f.  -0 keeps the state.  The product z
// log2(e) is rounded and the exponential flushes: that number's relative error
// grows as |z| 2^-24 (5e-7 at 9) and below 2^-126 it is 0.  The exact product
// would cost each value of an issue-bound kernel two instructions more.
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

// The steps above hold for finite values; an infinity meets itself in h - x or
// in l - (1 - f) l.  Once there, what is not finite stays so to the end of a run,
// so a run looks once and then goes again by the definition (`define`,
// `define_back`), reading global memory, frame by frame.  A neighbour that shares
// its thread, and frames before the first infinity, keep their bits.
template <int V>
__device__ __forceinline__ bool finite(Vec<V> v) {
  bool r = true;
#pragma unroll
  for (int i = 0; i < V; ++i) r = r && fabsf(v.v[i]) < INFINITY;
  return r;
}
template <int V>
__device__ __forceinline__ void both_gates(Vec<V> n, Vec<V>& f, Vec<V>& omf) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const float a = fabsf(n.v[i]);
    f.v[i] = __float_as_int(n.v[i]) < 0 ? 1.f - a : a;
    omf.v[i] = __float_as_int(n.v[i]) < 0 ? a : 1.f - a;
  }
}
// a where it is finite, else b.
template <int V>
__device__ __forceinline__ Vec<V> unless_odd(Vec<V> a, Vec<V> b) {
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (!(fabsf(a.v[i]) < INFINITY)) a.v[i] = b.v[i];
  return a;
}
// f h + (1 - f) x
template <int V>
__device__ __forceinline__ Vec<V> advance_any(Vec<V> n, Vec<V> h, Vec<V> x) {
  Vec<V> f, omf;
  both_gates(n, f, omf);
  return unless_odd(advance(n, h, x, sub_v(h, x)), fma_v(f, h, mul_v(omf, x)));
}
// A product of gates that are not zero is not zero: it carries an infinite
// state.  1.4e-45 times a finite one is below its rounding.
__device__ __forceinline__ float times_gate(float a, float by) {
  const float r = a * by;
  return r == 0.f && a != 0.f && by != 0.f ? 1.4e-45f : r;
}

// f l, (1 - f) l and f (1 - f) l diff.  With a = |n| and b = a l: the smaller of
// the first two is b, the other l - b; f (1 - f) l = b - a b.
template <int V>
__device__ __forceinline__ void gradients(Vec<V> n, Vec<V> l, Vec<V> diff, Vec<V>& fl, Vec<V>& dx,
                                          Vec<V>& dg) {
  Vec<V> a;
#pragma unroll
  for (int v = 0; v < V; ++v) a.v[v] = fabsf(n.v[v]);
  const Vec<V> b = mul_v(a, l), c = sub_v(l, b);
  fl = pick(n, c, b);
  dx = pick(n, b, c);
  dg = mul_v(fma_v(negated(a), b, b), diff);
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
template <typename T, int VC, int FR>
__device__ __forceinline__ void load_frames(Frame<T, VC> (&f)[FR], const char* p,
                                            size_t step, int n) {
  if (n >= FR) {
#pragma unroll
    for (int k = 0; k < FR; ++k) {
      f[k] = *reinterpret_cast<const Frame<T, VC>*>(p);
      walk(p, step);
    }
  } else {
#pragma unroll
    for (int k = 0; k < FR; ++k) {
      f[k] = k < n ? *reinterpret_cast<const Frame<T, VC>*>(p) : Frame<T, VC>::zero();
      walk(p, step);
    }
  }
}

// A channel's run in global memory, for what is not finite: frames `step` bytes
// apart from p on.
template <typename T, int VC> struct Far {
  const char* p;
  size_t step;
  __device__ __forceinline__ Vec<VC> operator[](int k) const {
    return reinterpret_cast<const Frame<T, VC>*>(p + (size_t)k * step)->get();
  }
};
// The states of n frames by the definition; put(k, h) takes each.
template <typename T, int VC, typename Put>
__device__ __forceinline__ Vec<VC> define(Far<T, VC> x, Far<T, VC> g, int n, Vec<VC> h, Put put) {
#pragma unroll 1
  for (int k = 0; k < n; ++k) {
    h = advance_any(gate_of(g[k]), h, x[k]);
    put(k, h);
  }
  return h;
}
// The adjoints of n frames, from the last: l beyond them to l before them;
// put(k, dx, dg).  The state before each frame is walked to anew from h.
template <typename T, int VC, typename Put>
__device__ __forceinline__ Vec<VC> define_back(Far<T, VC> y, Far<T, VC> x, Far<T, VC> g, int n,
                                               Vec<VC> h, Vec<VC> l, Put put) {
#pragma unroll 1
  for (int k = n - 1; k >= 0; --k) {
    const Vec<VC> before = define(x, g, k, h, [](int, Vec<VC>) {});
    const Vec<VC> n = gate_of(g[k]), diff = sub_v(before, x[k]);
    const Vec<VC> all = add_v(y[k], l);
    Vec<VC> f, omf, dx, dg;
    both_gates(n, f, omf);
    gradients(n, all, diff, l, dx, dg);
    l = unless_odd(l, mul_v(f, all));
    put(k, unless_odd(dx, mul_v(omf, all)),
        unless_odd(dg, mul_v(mul_v(mul_v(all, diff), f), omf)));
  }
  return l;
}
// B of a run, anew, for one that is not finite: from state 0 forward, REV: of
// f (l + v) from 0 backward.
template <bool REV, typename T, int VC>
__device__ __forceinline__ Vec<VC> define_sum(Far<T, VC> v, Far<T, VC> g, int n) {
  Vec<VC> B = splat<VC>(0.f);
#pragma unroll 1
  for (int i = 0; i < n; ++i) {
    const int k = REV ? n - 1 - i : i;
    const Vec<VC> s = gate_of(g[k]);
    Vec<VC> f, omf;
    both_gates(s, f, omf);
    if (REV) {
      const Vec<VC> l = add_v(v[k], B);
      B = unless_odd(decay(s, l), mul_v(f, l));
    } else {
      B = advance_any(s, B, v[k]);
    }
  }
  return B;
}
// A run's A as times_gate would have it; gate(k): a frame's gate as it lies.
template <int FR, int V, typename Gate>
__device__ __forceinline__ void keep_product(Vec<V>& A, Gate gate) {
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (A.v[i] == 0.f) {
      float least = 0.f;
#pragma unroll
      for (int k = 0; k < FR; ++k) least = fminf(least, gate(k).v[i]);
      if (least > -87.f) A.v[i] = 1.4e-45f;  // below, sigmoid itself is 0
    }
}
// The same from gate_of's numbers, where 0 that is not -0 is a closed gate.
template <int FR, int V>
__device__ __forceinline__ void keep_product(Vec<V>& A, const Vec<V> (&s)[FR]) {
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (A.v[i] == 0.f) {
      bool closed = false;
#pragma unroll
      for (int k = 0; k < FR; ++k) closed = closed || __float_as_uint(s[k].v[i]) == 0u;
      if (!closed) A.v[i] = 1.4e-45f;
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
  __syncwarp();  // the barrier wants whole warps
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
          ta = times_gate(ta, wa);
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
  constexpr int FR = frames_of(sizeof(T)), TILE = tile_of(LPR, sizeof(T));
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
  int t0 = rank * TILE + part * FR;
  Frame<T, VC> xr[FR], gr[FR];
  load_frames(gr, gp + (size_t)t0 * gs, gs, ch.L - t0);
  load_frames(xr, xp + (size_t)t0 * xs, xs, ch.L - t0);
  for (int it = 0; it < steps; ++it, t0 += TILE * S) {
    const int n = ch.L - t0;
    Vec<VC> s[FR];
    Frame<T, VC> xk[FR];  // as it lies: pairs in one register
#pragma unroll
    for (int k = 0; k < FR; ++k) {
      s[k] = gate_of(gr[k].get());
      xk[k] = xr[k];
    }
    if (n < FR)
#pragma unroll
      for (int k = 0; k < FR; ++k)
        if (k >= n) s[k] = splat<VC>(-0.f);
    // the next tile's loads are under way while the blocks wait for each other
    const int t1 = t0 + TILE * S;
    load_frames(gr, gp + (size_t)t1 * gs, gs, ch.L - t1);
    load_frames(xr, xp + (size_t)t1 * xs, xs, ch.L - t1);
    Vec<VC> A = splat<VC>(1.f), B = splat<VC>(0.f), h;
#pragma unroll
    for (int k = 0; k < FR; ++k) {
      const Vec<VC> x = xk[k].get();
      B = advance(s[k], B, x, sub_v(B, x));
      A = decay(s[k], A);
    }
    const Far<T, VC> fx = {xp + (size_t)t0 * xs, xs}, fg = {gp + (size_t)t0 * gs, gs};
    const int in = min(n, FR);
    bool plain = finite(B);
    if (!plain) B = define_sum<false>(fx, fg, in);
    keep_product<FR>(A, s);
    compose<VC, LPR, false>(sh, it, S, rank, part, lane, A, B, run, h);
    plain = plain && finite(h);
    if (carry && ch.live && t0 < TT)
#pragma unroll
      for (int v = 0; v < VC; ++v)
        carry[(size_t)(t0 / FR) * BD + ch.c + v] = h.v[v];
    char* o = yp + (size_t)t0 * ys;
    if (!plain) {
      h = define(fx, fg, in, h, [&](int k, Vec<VC> v) {
        *reinterpret_cast<Frame<T, VC>*>(o + (size_t)k * ys) = Frame<T, VC>::of(v);
      });
#pragma unroll 1
      for (int k = max(in, 0); ch.live && k < FR && t0 + k < TT; ++k)
        *reinterpret_cast<Frame<T, VC>*>(o + (size_t)k * ys) = Frame<T, VC>::zero();
    } else if (n >= FR) {
#pragma unroll
      for (int k = 0; k < FR; ++k) {
        const Vec<VC> x = xk[k].get();
        h = advance(s[k], h, x, sub_v(h, x));
        *reinterpret_cast<Frame<T, VC>*>(o) = Frame<T, VC>::of(h);
        walk(o, ys);
      }
    } else {
#pragma unroll
      for (int k = 0; k < FR; ++k) {
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
  constexpr int FR = frames_of(sizeof(T)), TILE = tile_of(LPR, sizeof(T));
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
  int t0 = ((steps - 1) * S + rank) * TILE + part * FR;
  Frame<T, VC> xr[FR], gr[FR], yr[FR];
  Vec<VC> hr;
  auto load = [&](int t) {
    const int n = t >= 0 ? ch.L - t : 0;
    const size_t tt = t >= 0 ? t : 0;
    load_frames(gr, gp + tt * gs, gs, n);
    load_frames(yr, yp + tt * ys, ys, n);
    load_frames(xr, xp + tt * xs, xs, n);
#pragma unroll
    for (int v = 0; v < VC; ++v)
      hr.v[v] = n > 0 ? carry[(tt / FR) * BD + ch.c + v] : 0.f;
  };
  load(t0);
  for (int it = 0; it < steps; ++it, t0 -= TILE * S) {
    const int n = ch.L - t0;
    Vec<VC> s[FR], diff[FR];  // the gates; h_{t-1} - x_t
    Vec<VC> h = hr, lam;
    Frame<T, VC> yk[FR];
#pragma unroll
    for (int k = 0; k < FR; ++k) {
      s[k] = gate_of(gr[k].get());
      yk[k] = yr[k];
    }
    if (n < FR)
#pragma unroll
      for (int k = 0; k < FR; ++k)
        if (k >= n) s[k] = splat<VC>(-0.f);
#pragma unroll
    for (int k = 0; k < FR; ++k) {
      const Vec<VC> x = xr[k].get();
      diff[k] = sub_v(h, x);
      h = advance(s[k], h, x, diff[k]);
    }
    const Vec<VC> first = hr;
    load(t0 - TILE * S);  // under way while the blocks wait for each other
    Vec<VC> A = splat<VC>(1.f), B = splat<VC>(0.f);
#pragma unroll
    for (int k = FR - 1; k >= 0; --k) {
      B = decay(s[k], add_v(yk[k].get(), B));
      A = decay(s[k], A);
    }
    const Far<T, VC> fy = {yp + (size_t)t0 * ys, ys}, fx = {xp + (size_t)t0 * xs, xs},
                     fg = {gp + (size_t)t0 * gs, gs};
    const int in = min(n, FR);
    bool plain = finite(B) && finite(h);
    if (!finite(B)) B = define_sum<true>(fy, fg, in);
    keep_product<FR>(A, s);
    compose<VC, LPR, true>(sh, it, S, rank, part, lane, A, B, run, lam);
    plain = plain && finite(lam);
    const size_t last = (at + (size_t)(t0 + FR - 1) * D) * sizeof(T);
    char* ox = reinterpret_cast<char*>(dx) + last;
    char* og = reinterpret_cast<char*>(dg) + last;
    if (!plain) {
      auto at_frame = [&](char* p, int k) {
        return reinterpret_cast<Frame<T, VC>*>(p - (FR - 1 - k) * os);
      };
      lam = define_back(fy, fx, fg, in, first, lam, [&](int k, Vec<VC> vx, Vec<VC> vg) {
        *at_frame(ox, k) = Frame<T, VC>::of(vx);
        *at_frame(og, k) = Frame<T, VC>::of(vg);
      });
#pragma unroll 1
      for (int k = max(in, 0); ch.live && k < FR && t0 + k < TT; ++k)
        *at_frame(ox, k) = *at_frame(og, k) = Frame<T, VC>::zero();
    } else
#pragma unroll
    for (int k = FR - 1; k >= 0; --k) {
      const Vec<VC> l = add_v(yk[k].get(), lam);
      lam = decay(s[k], l);
      const Vec<VC> pass = passed(s[k], l, negated(l));
      const Frame<T, VC> vx = Frame<T, VC>::of(pass);
      // f (1 - f) l (h - x)
      const Frame<T, VC> vg = Frame<T, VC>::of(mul_v(decay(s[k], pass), diff[k]));
      if (n >= FR) {
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

// ------------------------------------------- tiles in shared memory

// Like common.cuh's, and a barrier to the compiler: a slot is refilled after
// it was read.
__device__ __forceinline__ void fetch16(uint32_t dst, const void* src, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src),
               "r"(in ? 16 : 0)
               : "memory");
}

// NT threads a block, LPR lanes a frame.  NT 32 and LPR 32: one warp walks its
// channels through all of time, a run at a time; nothing is composed and
// nobody waits for anybody, so a frame costs half the instructions.
template <typename T, int LPR, int NT> struct Staged {
  static constexpr int FR = frames_of(sizeof(T)), RUNS = NT / LPR;
  static constexpr int TILE = RUNS * FR;
  static constexpr int LINE = LPR * 2 * (int)sizeof(T);              // bytes a frame
  static constexpr int PITCH = FR * LINE;                            // of a run
  static constexpr int SLOT = RUNS * PITCH;                          // of an array's tile
  // Half lines: odd runs swap neighbouring frames, so that the two runs that a
  // half-warp reads at once lie in different banks.
  static constexpr bool SWAP = LINE < 128;
  static constexpr int CPL = LINE / 16, ROWS = NT / CPL;             // 16-byte pieces of a frame
  static constexpr int PASSES = TILE / ROWS;
  static constexpr int STEP = ROWS >= FR ? ROWS / FR * PITCH : ROWS * LINE;
  static constexpr int STAGES = NT == 32 ? 6 : 2;
};

template <int NT>
__device__ __forceinline__ void block_sync() {
  if (NT == 32) __syncwarp();
  else __syncthreads();
}

// A run's frames of a lane in a slot.
template <typename T, int LPR, int NT> struct RunFrames {
  using G = Staged<T, LPR, NT>;
  using F = Frame<T, 2>;
  F* even;
  F* odd;
  __device__ __forceinline__ RunFrames(uint8_t* slot, int part, int lane) {
    F* p = reinterpret_cast<F*>(slot + part * G::PITCH) + lane;
    const int by = G::SWAP && (part & 1) ? LPR : 0;
    even = p + by;
    odd = p - by;
  }
  __device__ __forceinline__ F& operator[](int k) const { return (k & 1 ? odd : even)[k * LPR]; }
};

// A thread's share of moving tiles: piece `threadIdx % CPL` of every ROWS-th
// frame.
template <typename T, int LPR, int NT> struct Mover {
  using G = Staged<T, LPR, NT>;
  size_t b, d;
  bool live;
  int L, row;
  uint32_t at;  // in a slot
  __device__ __forceinline__ Mover(size_t first, size_t BD, int D, int TT,
                                   const int64_t* lengths) {
    const int piece = threadIdx.x % G::CPL;
    row = threadIdx.x / G::CPL;
    const size_t c = first + piece * (16 / sizeof(T));
    live = c < BD;
    b = live ? c / D : 0;
    d = live ? c - b * D : 0;
    L = live ? live_len(lengths, (int)b, TT) : 0;
    const int r = row / G::FR, k = row % G::FR;
    at = r * G::PITCH + (G::SWAP ? k ^ (r & 1) : k) * G::LINE + piece * 16;
  }
  // frames t.. of an array (its frames `step` bytes apart, p at this thread's
  // piece of frame 0) into the slot at shared address `slot`; past L: zeros
  __device__ __forceinline__ void fetch(uint32_t slot, const char* p, size_t step, int t) const {
    const char* q = p + (size_t)(t + row) * step;
#pragma unroll
    for (int i = 0; i < G::PASSES; ++i) {
      const bool in = t + row + i * G::ROWS < L;
      fetch16(slot + at + i * G::STEP, in ? q : p, in);
      q += G::ROWS * step;
    }
  }
  __device__ __forceinline__ void put(const uint8_t* slot, char* p, size_t step, int t,
                                      int TT) const {
    char* q = p + (size_t)(t + row) * step;
#pragma unroll
    for (int i = 0; i < G::PASSES; ++i) {
      if (live && t + row + i * G::ROWS < TT)
        *reinterpret_cast<uint4*>(q) = *reinterpret_cast<const uint4*>(slot + at + i * G::STEP);
      q += G::ROWS * step;
    }
  }
};

template <typename T>
__device__ __forceinline__ Far<T, 2> far_run(const T* p, size_t b, size_t t, const Channel& ch,
                                             int t0) {
  return {reinterpret_cast<const char*>(p + ch.b * b + (size_t)t0 * t + ch.d), t * sizeof(T)};
}

// What segments of time do to the state: (A, B) of every segment and channel.
struct Segments {
  int tiles;         // of a segment
  int count;
  float2* sums;      // [count][BD], or NULL when there is one segment
};

// The state that enters segment z: from `h`, through the segments before it
// (REV: after it).
template <bool REV>
__device__ __forceinline__ float entering(const Segments& seg, int z, size_t BD, size_t c,
                                          float h) {
  const int n = REV ? seg.count - 1 - z : z;
#pragma unroll 8
  for (int i = 0; i < n; ++i) {
    const float2 ab = seg.sums[(size_t)(REV ? seg.count - 1 - i : i) * BD + c];
    h = fmaf(ab.x, h, ab.y);
  }
  return h;
}

// (A, B) of each segment: of f h + (1 - f) v forward in time, or REV of
// f (l + v) backward.
template <typename T, int LPR, bool REV>
__global__ void __launch_bounds__(SCAN_THREADS, 4)
    scan_sum_tiles_kernel(const T* __restrict__ v, size_t vb, size_t vt, const T* __restrict__ g,
                          size_t gb, size_t gt, const int64_t* __restrict__ lengths, size_t BD,
                          int TT, int D, Segments seg) {
  using G = Staged<T, LPR, SCAN_THREADS>;
  constexpr int FR = G::FR;
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ ScanShared<2, LPR> sh;
  const int part = threadIdx.x / LPR, lane = threadIdx.x & (LPR - 1);
  // the last segment in time's order is not needed
  const int z = blockIdx.x % (seg.count - 1) + (REV ? 1 : 0);
  const size_t first = (size_t)(blockIdx.x / (seg.count - 1)) * (2 * LPR);
  const Channel ch(first, lane, 2, BD, D, TT, lengths);
  const Mover<T, LPR, SCAN_THREADS> mv(first, BD, D, TT, lengths);
  const char* vp = reinterpret_cast<const char*>(v + mv.b * vb + mv.d);
  const char* gp = reinterpret_cast<const char*>(g + mv.b * gb + mv.d);
  const size_t vs = vt * sizeof(T), gs = gt * sizeof(T);
  const int steps = min(seg.tiles, (TT + G::TILE - 1) / G::TILE - z * seg.tiles);
  auto tile_of_step = [&](int it) {
    return (z * seg.tiles + (REV ? steps - 1 - it : it)) * G::TILE;
  };
  auto fetch = [&](int it) {
    if (it < steps) {
      const uint32_t slot = smem_u32(ring) + (it % G::STAGES) * 2 * G::SLOT;
      mv.fetch(slot, gp, gs, tile_of_step(it));
      mv.fetch(slot + G::SLOT, vp, vs, tile_of_step(it));
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < G::STAGES; ++i) fetch(i);
  float2 total[2] = {make_float2(1.f, 0.f), make_float2(1.f, 0.f)};  // of run 0's threads
  bool closed[2] = {false, false};
  for (int it = 0; it < steps; ++it) {
    uint8_t* gsl = ring + (it % G::STAGES) * 2 * G::SLOT;
    const int n = ch.L - (tile_of_step(it) + part * FR), p = it & 1;
    const RunFrames<T, LPR, SCAN_THREADS> gf(gsl, part, lane), vf(gsl + G::SLOT, part, lane);
    cp_async_wait<G::STAGES - 1>();
    __syncthreads();
    Vec<2> A = splat<2>(1.f), B = splat<2>(0.f);
#pragma unroll
    for (int i = 0; i < FR; ++i) {
      const int k = REV ? FR - 1 - i : i;
      const Vec<2> s = k < n ? gate_of(gf[k].get()) : splat<2>(-0.f), x = vf[k].get();
      B = REV ? decay(s, add_v(x, B)) : advance(s, B, x, sub_v(B, x));
      A = decay(s, A);
    }
    if (!finite(B)) {
      const int t0 = tile_of_step(it) + part * FR;
      B = define_sum<REV>(far_run<T>(v, vb, vt, ch, t0), far_run<T>(g, gb, gt, ch, t0), min(n, FR));
    }
    keep_product<FR>(A, [&](int k) { return k < n ? gf[k].get() : splat<2>(0.f); });
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      sh.a[p][part][lane * 2 + q] = A.v[q];
      sh.b[p][part][lane * 2 + q] = B.v[q];
    }
    __syncthreads();
    if (part == 0)
#pragma unroll
      for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int i = 0; i < G::RUNS; ++i) {
          const int w = REV ? G::RUNS - 1 - i : i;
          const float wa = sh.a[p][w][lane * 2 + q];
          total[q].y = fmaf(wa, total[q].y, sh.b[p][w][lane * 2 + q]);
          total[q].x *= wa;
          closed[q] = closed[q] || wa == 0.f;
        }
    fetch(it + G::STAGES);  // all have read this tile
  }
  if (ch.live && part == 0)
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      if (total[q].x == 0.f && !closed[q]) total[q].x = 1.4e-45f;  // as times_gate
      seg.sums[(size_t)z * BD + ch.c + q] = total[q];
    }
}

template <typename T, int LPR, int NT>
__global__ void __launch_bounds__(NT, NT == 32 ? 8 : 4)
    scan_fwd_tiles_kernel(const T* __restrict__ x, size_t xb, size_t xt, const T* __restrict__ g,
                          size_t gb, size_t gt, const float* __restrict__ h0,
                          const int64_t* __restrict__ lengths, size_t BD, int TT, int D, Segments seg,
                          T* __restrict__ y, float* __restrict__ state,
                          float* __restrict__ carry) {
  using G = Staged<T, LPR, NT>;
  constexpr int FR = G::FR;
  extern __shared__ __align__(128) uint8_t ring[];
  constexpr bool ALONE = G::RUNS == 1;
  __shared__ ScanShared<2, LPR> sh;
  const int part = threadIdx.x / LPR, lane = threadIdx.x & (LPR - 1);
  const int z = blockIdx.x % seg.count;
  const size_t first = (size_t)(blockIdx.x / seg.count) * (2 * LPR);
  const Channel ch(first, lane, 2, BD, D, TT, lengths);
  const Mover<T, LPR, NT> mv(first, BD, D, TT, lengths);
  const char* xp = reinterpret_cast<const char*>(x + mv.b * xb + mv.d);
  const char* gp = reinterpret_cast<const char*>(g + mv.b * gb + mv.d);
  char* yp = reinterpret_cast<char*>(y + mv.b * (size_t)TT * D + mv.d);
  const size_t xs = xt * sizeof(T), gs = gt * sizeof(T), ys = D * sizeof(T);
  Vec<2> run = splat<2>(0.f);
  if (part == 0)
#pragma unroll
    for (int v = 0; v < 2; ++v)
      run.v[v] = sh.start[0][lane * 2 + v] =
          ch.live ? entering<false>(seg, z, BD, ch.c + v, h0 ? h0[ch.c + v] : 0.f) : 0.f;
  const int tiles = (TT + G::TILE - 1) / G::TILE, tile0 = z * seg.tiles;
  const int steps = min(seg.tiles, tiles - tile0);
  auto fetch = [&](int it) {
    if (it < steps) {
      const uint32_t slot = smem_u32(ring) + (it % G::STAGES) * 2 * G::SLOT;
      const int t = (tile0 + it) * G::TILE;
      mv.fetch(slot, gp, gs, t);
      mv.fetch(slot + G::SLOT, xp, xs, t);
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < G::STAGES; ++i) fetch(i);
  for (int it = 0; it < steps; ++it) {
    uint8_t* gsl = ring + (it % G::STAGES) * 2 * G::SLOT;
    uint8_t* xsl = gsl + G::SLOT;
    const int tile = (tile0 + it) * G::TILE, t0 = tile + part * FR, n = ch.L - t0;
    using F = Frame<T, 2>;
    const RunFrames<T, LPR, NT> gf(gsl, part, lane), xf(xsl, part, lane);
    cp_async_wait<G::STAGES - 1>();
    block_sync<NT>();
    Vec<2> s[FR], A = splat<2>(1.f), B = splat<2>(0.f), h;
#pragma unroll
    for (int k = 0; k < FR; ++k) s[k] = gate_of(gf[k].get());
    if (n < FR)
#pragma unroll
      for (int k = 0; k < FR; ++k)
        if (k >= n) s[k] = splat<2>(-0.f);
    const int in = min(n, FR);
    bool plain = true;
    auto far_x = [&] { return far_run<T>(x, xb, xt, ch, t0); };
    auto far_g = [&] { return far_run<T>(g, gb, gt, ch, t0); };
    if constexpr (ALONE) {
      h = run;
    } else {
#pragma unroll
      for (int k = 0; k < FR; ++k) {
        const Vec<2> xv = xf[k].get();
        B = advance(s[k], B, xv, sub_v(B, xv));
        A = decay(s[k], A);
      }
      plain = finite(B);
      if (!plain) B = define_sum<false>(far_x(), far_g(), in);
      keep_product<FR>(A, s);
      compose<2, LPR, false>(sh, it, 1, 0, part, lane, A, B, run, h);
      plain = plain && finite(h);
    }
    if (carry && ch.live && t0 < TT)
      *reinterpret_cast<float2*>(carry + (size_t)(t0 / FR) * BD + ch.c) =
          make_float2(h.v[0], h.v[1]);
    auto finish = [&](bool all) {
#pragma unroll
      for (int k = 0; k < FR; ++k) {
        const Vec<2> xv = xf[k].get();
        h = advance(s[k], h, xv, sub_v(h, xv));
        xf[k] = all || k < n ? F::of(h) : F::zero();
      }
    };
    auto finish_any = [&](Vec<2> from) {
      h = define(far_x(), far_g(), in, from, [&](int k, Vec<2> v) { xf[k] = F::of(v); });
#pragma unroll 1
      for (int k = max(in, 0); k < FR; ++k) xf[k] = F::zero();
    };
    if (!plain) finish_any(h);
    else if (n >= FR) finish(true);
    else finish(false);
    if (ALONE) {
      if (!finite(h)) finish_any(run);
      run = h;
    }
    if (part == G::RUNS - 1)
#pragma unroll
      for (int v = 0; v < 2; ++v) sh.start[(it + 1) & 1][lane * 2 + v] = h.v[v];
    block_sync<NT>();
    mv.put(xsl, yp, ys, tile, TT);
    fetch(it + G::STAGES);  // into the places this thread has just read
  }
  block_sync<NT>();
  if (ch.live && part == 0 && z == seg.count - 1)
#pragma unroll
    for (int v = 0; v < 2; ++v) state[ch.c + v] = sh.start[steps & 1][lane * 2 + v];
}

// The same walk from the end, always in the 128-thread form: alone, a warp
// took 101 us where the four runs take 85 (32 x 1024 x 1024 bfloat16).
template <typename T, int LPR>
__global__ void __launch_bounds__(SCAN_THREADS, 4)
    scan_bwd_tiles_kernel(const T* __restrict__ dy, size_t yb, size_t yt,
                          const float* __restrict__ dstate, const T* __restrict__ x, size_t xb,
                          size_t xt, const T* __restrict__ g, size_t gb, size_t gt,
                          const int64_t* __restrict__ lengths, const float* __restrict__ carry,
                          size_t BD, int TT, int D, Segments seg, T* __restrict__ dx, T* __restrict__ dg,
                          float* __restrict__ dh0) {
  using G = Staged<T, LPR, SCAN_THREADS>;
  constexpr int FR = G::FR;
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ ScanShared<2, LPR> sh;
  const int part = threadIdx.x / LPR, lane = threadIdx.x & (LPR - 1);
  const int z = blockIdx.x % seg.count;
  const size_t first = (size_t)(blockIdx.x / seg.count) * (2 * LPR);
  const Channel ch(first, lane, 2, BD, D, TT, lengths);
  const Mover<T, LPR, SCAN_THREADS> mv(first, BD, D, TT, lengths);
  const char* xp = reinterpret_cast<const char*>(x + mv.b * xb + mv.d);
  const char* gp = reinterpret_cast<const char*>(g + mv.b * gb + mv.d);
  const char* yp = reinterpret_cast<const char*>(dy + mv.b * yb + mv.d);
  const size_t out = mv.b * (size_t)TT * D + mv.d;
  char* ox = reinterpret_cast<char*>(dx + out);
  char* og = reinterpret_cast<char*>(dg + out);
  const size_t xs = xt * sizeof(T), gs = gt * sizeof(T), ys = yt * sizeof(T), os = D * sizeof(T);
  // f_{t+1} lam_{t+1} beyond the frames done
  Vec<2> run = splat<2>(0.f);
  if (part == 0)
#pragma unroll
    for (int v = 0; v < 2; ++v)
      sh.start[0][lane * 2 + v] =
          ch.live ? entering<true>(seg, z, BD, ch.c + v, dstate ? dstate[ch.c + v] : 0.f) : 0.f;
  const int tiles = (TT + G::TILE - 1) / G::TILE, tile0 = z * seg.tiles;
  const int steps = min(seg.tiles, tiles - tile0);
  auto fetch = [&](int it) {
    if (it < steps) {
      const uint32_t slot = smem_u32(ring) + (it % G::STAGES) * 3 * G::SLOT;
      const int t = (tile0 + steps - 1 - it) * G::TILE;
      mv.fetch(slot, gp, gs, t);
      mv.fetch(slot + G::SLOT, xp, xs, t);
      mv.fetch(slot + 2 * G::SLOT, yp, ys, t);
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < G::STAGES; ++i) fetch(i);
  for (int it = 0; it < steps; ++it) {
    uint8_t* gsl = ring + (it % G::STAGES) * 3 * G::SLOT;
    uint8_t* xsl = gsl + G::SLOT;
    uint8_t* ysl = xsl + G::SLOT;
    const int tile = (tile0 + steps - 1 - it) * G::TILE, t0 = tile + part * FR,
              n = ch.L - t0;
    using F = Frame<T, 2>;
    const RunFrames<T, LPR, SCAN_THREADS> gf(gsl, part, lane), xf(xsl, part, lane), yf(ysl, part, lane);
    float2 h2 = make_float2(0.f, 0.f);
    if (n > 0)
      h2 = *reinterpret_cast<const float2*>(carry + (size_t)(t0 / FR) * BD + ch.c);
    cp_async_wait<G::STAGES - 1>();
    __syncthreads();
    Vec<2> s[FR], diff[FR];  // the gates; h_{t-1} - x_t
    Vec<2> A = splat<2>(1.f), B = splat<2>(0.f), h = {{h2.x, h2.y}}, lam;
#pragma unroll
    for (int k = 0; k < FR; ++k) s[k] = gate_of(gf[k].get());
    if (n < FR)
#pragma unroll
      for (int k = 0; k < FR; ++k)
        if (k >= n) s[k] = splat<2>(-0.f);
#pragma unroll
    for (int k = FR - 1; k >= 0; --k) {
      B = decay(s[k], add_v(yf[k].get(), B));
      A = decay(s[k], A);
    }
#pragma unroll
    for (int k = 0; k < FR; ++k) {
      const Vec<2> xv = xf[k].get();
      diff[k] = sub_v(h, xv);
      h = advance(s[k], h, xv, diff[k]);
    }
    bool plain = finite(B) && finite(h);
    const int in = min(n, FR);
    auto far_y = [&] { return far_run<T>(dy, yb, yt, ch, t0); };
    auto far_g = [&] { return far_run<T>(g, gb, gt, ch, t0); };
    if (!finite(B)) B = define_sum<true>(far_y(), far_g(), in);
    keep_product<FR>(A, s);
    compose<2, LPR, true>(sh, it, 1, 0, part, lane, A, B, run, lam);
    plain = plain && finite(lam);
    auto finish = [&](bool all) {
#pragma unroll
      for (int k = FR - 1; k >= 0; --k) {
        const Vec<2> l = add_v(yf[k].get(), lam);
        Vec<2> dxv, dgv;
        gradients(s[k], l, diff[k], lam, dxv, dgv);
        const F vx = F::of(dxv), vg = F::of(dgv);
        xf[k] = all || k < n ? vx : F::zero();
        gf[k] = all || k < n ? vg : F::zero();
      }
    };
    if (!plain) {
      lam = define_back(far_y(), far_run<T>(x, xb, xt, ch, t0), far_g(), in, Vec<2>{{h2.x, h2.y}}, lam,
                        [&](int k, Vec<2> vx, Vec<2> vg) {
                          xf[k] = F::of(vx);
                          gf[k] = F::of(vg);
                        });
#pragma unroll 1
      for (int k = max(in, 0); k < FR; ++k) xf[k] = gf[k] = F::zero();
    } else if (n >= FR) {
      finish(true);
    } else {
      finish(false);
    }
    if (part == 0)
#pragma unroll
      for (int v = 0; v < 2; ++v) sh.start[(it + 1) & 1][lane * 2 + v] = lam.v[v];
    __syncthreads();
    mv.put(xsl, ox, os, tile, TT);
    mv.put(gsl, og, os, tile, TT);
    fetch(it + G::STAGES);  // into places that this thread, or all before the barrier, have read
  }
  __syncthreads();
  if (ch.live && dh0 && part == 0 && z == 0)
#pragma unroll
    for (int v = 0; v < 2; ++v) dh0[ch.c + v] = sh.start[steps & 1][lane * 2 + v];
}

// One frame against the running states, a channel a thread.  For a few streams
// the launch is its time (64 x 1024: 6 us a call, 0.14 us of bytes).
template <typename T>
__global__ void __launch_bounds__(SCAN_THREADS)
    scan_step_kernel(const T* __restrict__ x, size_t xs, const T* __restrict__ g, size_t gs,
                     float* __restrict__ state, int B, int D, T* __restrict__ y) {
  const size_t id = (size_t)blockIdx.x * SCAN_THREADS + threadIdx.x;
  if (id >= (size_t)B * D) return;
  const size_t b = id / D, d = id - b * D;
  const Vec<1> n = gate_of(Vec<1>{{to_f(g[b * gs + d])}});
  const Vec<1> was = {{state[id]}}, in = {{to_f(x[b * xs + d])}};
  float h = advance(n, was, in, sub_v(was, in)).v[0];
  if (!(fabsf(h) < INFINITY)) h = advance_any(n, was, in).v[0];
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

// How the channels of a call are spread over blocks of the second form, 32 or
// 16 lanes a frame, and its time over S blocks of a cluster: whole lanes while
// the SMs get three blocks each, then as many time blocks as there are tiles.
struct ScanPlan {
  int lpr, S;
  size_t groups;
};
ScanPlan scan_plan(size_t BD, int TT, size_t type_bytes) {
  ScanPlan p = {32, 1, 0};
  for (;; p.lpr = 16) {
    p.groups = (BD + p.lpr - 1) / p.lpr;
    p.S = 1;
    while (p.S < 8 && p.groups * p.S < 148 * 3 &&
           (long long)p.S * tile_of(p.lpr, type_bytes) < TT)
      p.S *= 2;
    if (p.lpr == 16 || p.groups * p.S >= 148 * 3) return p;
  }
}

// Of the first form.  Whole 128-byte lines while they give the SMs two blocks
// each; half lines while those give them three for two; below that segments of
// time, of at least 2 tiles, as many as the SMs hold blocks of (4 each; more
// would start when the first end: 640 blocks took 240 us where 576 take 175, 4 x
// 32768 x 256 float32 backward).
struct TilePlan {
  bool whole, alone;
  int segments, tiles;  // tiles of a segment
  size_t groups;
};

// Forward, 16 bits, and lines for three warps a SM at least: a warp alone walks
// a line (measured when it was added: 32 x 1024 x 1024 bfloat16 51 us against 56
// of blocks whose four runs are composed; 64 x 64 x 2048 13.4 against 16.9; other
// shapes were not compared).  float32 is within a fifth
// of a copy's time without it.
constexpr size_t ALONE_FROM = 148 * 3;
template <typename T>
TilePlan tile_plan(size_t BD, int TT, bool forward) {
  constexpr int MOST = 64 / sizeof(T);  // lanes of a whole line, two channels each
  const size_t lines = (BD + 2 * MOST - 1) / (2 * MOST), halves = (BD + MOST - 1) / MOST;
  TilePlan p = {lines >= 148 * 2 || halves < 222, forward && sizeof(T) == 2 && lines >= ALONE_FROM, 1,
                0, 0};
  p.groups = p.whole ? lines : halves;
  const int tile = p.alone ? frames_of(sizeof(T)) : tile_of(p.whole ? MOST : MOST / 2, sizeof(T));
  const int tiles = (TT + tile - 1) / tile;
  if (halves < 222 && lines) {
    const size_t want = 148 * 4 / lines;
    p.segments = want < (size_t)(tiles / 2) ? (int)want : tiles / 2;
    if (p.segments < 1) p.segments = 1;
  }
  p.tiles = (tiles + p.segments - 1) / p.segments;
  p.segments = p.tiles ? (tiles + p.tiles - 1) / p.tiles : 1;
  return p;
}

template <typename T>
size_t sums_bytes(int B, int TT, int D) {
  if (D * sizeof(T) % 16) return 0;
  const TilePlan p = tile_plan<T>((size_t)B * D, TT, false);  // same segments
  return p.segments > 1 ? (size_t)p.segments * B * D * sizeof(float2) : 0;
}

template <typename... Params, typename... Args>
int launch(const char* who, void (*kernel)(Params...), size_t groups, int S, int threads,
           size_t smem, void* stream, Args... args) {
  if (smem) {
    const cudaError_t e = cudaFuncSetAttribute(
        (const void*)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return set_error(kLaunch, "%s: %s", who, cudaGetErrorString(e));
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(groups * S));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
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

// The first form's launches: the segments' sums when there are several, then
// the scan.
template <typename T, int LPR, int NT>
int fwd_tiles(const TilePlan& p, const T* x, size_t xb, size_t xt, const T* g, size_t gb,
              size_t gt, const float* h0, const int64_t* lengths, size_t BD, int TT, int D, T* y,
              float* state, float* carry, float2* sums, void* stream) {
  using G = Staged<T, LPR, NT>;
  using GS = Staged<T, LPR, SCAN_THREADS>;
  const char* who = "tw_gated_scan_forward";
  const Segments seg = {p.tiles, p.segments, sums};
  if (p.segments > 1)
    if (int e = launch(who, scan_sum_tiles_kernel<T, LPR, false>, p.groups * (p.segments - 1), 1,
                       SCAN_THREADS, (size_t)GS::STAGES * 2 * GS::SLOT, stream, x, xb, xt, g, gb, gt, lengths, BD, TT, D, seg))
      return e;
  return launch(who, scan_fwd_tiles_kernel<T, LPR, NT>, p.groups * p.segments, 1, NT,
                (size_t)G::STAGES * 2 * G::SLOT, stream, x, xb, xt, g, gb, gt, h0, lengths, BD, TT, D, seg, y, state, carry);
}

template <typename T, int LPR>
int bwd_tiles(const TilePlan& p, const T* dy, size_t yb, size_t yt, const float* dstate,
              const T* x, size_t xb, size_t xt, const T* g, size_t gb, size_t gt,
              const int64_t* lengths, const float* carry, size_t BD, int TT, int D, T* dx, T* dg,
              float* dh0, float2* sums, void* stream) {
  using G = Staged<T, LPR, SCAN_THREADS>;
  const char* who = "tw_gated_scan_backward";
  const Segments seg = {p.tiles, p.segments, sums};
  if (p.segments > 1)
    if (int e = launch(who, scan_sum_tiles_kernel<T, LPR, true>, p.groups * (p.segments - 1), 1,
                       SCAN_THREADS, (size_t)G::STAGES * 2 * G::SLOT, stream, dy, yb, yt, g, gb, gt, lengths, BD,
                       TT, D, seg))
      return e;
  return launch(who, scan_bwd_tiles_kernel<T, LPR>, p.groups * p.segments, 1, SCAN_THREADS,
                (size_t)G::STAGES * 3 * G::SLOT, stream, dy, yb, yt, dstate, x, xb, xt, g, gb, gt,
                lengths, carry, BD, TT, D, seg, dx, dg, dh0);
}

// Whether frames can move in 16-byte pieces.
template <typename T>
bool pieces(const void* p, size_t s1, size_t s2) {
  return (uintptr_t)p % 16 == 0 && s1 * sizeof(T) % 16 == 0 && s2 * sizeof(T) % 16 == 0;
}

// The saved states of a call; its segments' sums lie behind them.
template <typename T>
size_t states_bytes(int B, int TT, int D) {
  const int fr = frames_of(sizeof(T));
  const size_t n = (size_t)B * D * ((TT + fr - 1) / fr) * sizeof(float);
  return (n + 15) / 16 * 16;
}

template <typename T>
int fwd(const void* xv, size_t xb, size_t xt, const void* gv, size_t gb, size_t gt,
        const float* h0, const int64_t* lengths, int B, int TT, int D, void* y, float* state,
        void* carry, size_t carry_bytes, void* stream) {
  set_error(kOk, "%s", "");
  const char* who = "tw_gated_scan_forward";
  if (int e = check(who, B, TT, D)) return e;
  if (B == 0) return kOk;
  if (!state || (TT && (!xv || !gv || !y)))
    return set_error(kInvalid, "tw_gated_scan_forward: null pointer argument");
  const size_t states = states_bytes<T>(B, TT, D), sums = sums_bytes<T>(B, TT, D);
  const bool saves = carry && carry_bytes >= states + sums;
  if (carry && !saves && (sums == 0 || carry_bytes < sums))
    return set_error(kWorkspace, "tw_gated_scan_forward: carry needs %zu bytes (%zu without a "
                     "backward)", states + sums, sums);
  const T* x = (const T*)xv;
  const T* g = (const T*)gv;
  const size_t BD = (size_t)B * D;
  float* saved = saves ? (float*)carry : nullptr;
  if (D * sizeof(T) % 16 == 0 && pieces<T>(x, xb, xt) && pieces<T>(g, gb, gt) &&
      pieces<T>(y, 0, 0) && (uintptr_t)carry % 16 == 0) {
    TilePlan p = tile_plan<T>(BD, TT, true);
    if (p.segments > 1 && !carry) {  // no room for their sums
      p.tiles *= p.segments;
      p.segments = 1;
    }
    float2* room = (float2*)((char*)carry + (saves ? states : 0));
    constexpr int MOST = 64 / sizeof(T);
    if constexpr (MOST == 32)
      if (p.alone)
        return fwd_tiles<T, 32, 32>(p, x, xb, xt, g, gb, gt, h0, lengths, BD, TT, D, (T*)y, state,
                                    saved, room, stream);
    return p.whole ? fwd_tiles<T, MOST, SCAN_THREADS>(p, x, xb, xt, g, gb, gt, h0, lengths, BD, TT, D, (T*)y,
                                        state, saved, room, stream)
                   : fwd_tiles<T, MOST / 2, SCAN_THREADS>(p, x, xb, xt, g, gb, gt, h0, lengths, BD, TT, D,
                                            (T*)y, state, saved, room, stream);
  }
  const ScanPlan p = scan_plan(BD, TT, sizeof(T));
  return launch(who, p.lpr == 32 ? scan_fwd_kernel<T, 1, 32> : scan_fwd_kernel<T, 1, 16>,
                p.groups, p.S, SCAN_THREADS, 0, stream, x, xb, xt, g, gb, gt, h0, lengths, BD, TT, D, p.S,
                (T*)y, state, saved);
}

template <typename T>
int bwd(const void* dyv, size_t yb, size_t yt, const float* dstate, const void* xv, size_t xb,
        size_t xt, const void* gv, size_t gb, size_t gt, const int64_t* lengths,
        const void* carry, size_t carry_bytes, int B, int TT, int D, void* dx, void* dg,
        float* dh0, void* ws, size_t ws_bytes, void* stream) {
  set_error(kOk, "%s", "");
  const char* who = "tw_gated_scan_backward";
  if (int e = check(who, B, TT, D)) return e;
  if (B == 0) return kOk;
  if (TT && (!dyv || !xv || !gv || !carry || !dx || !dg))
    return set_error(kInvalid, "tw_gated_scan_backward: null pointer argument");
  if (carry_bytes < states_bytes<T>(B, TT, D))
    return set_error(kWorkspace, "tw_gated_scan_backward: carry needs %zu bytes",
                     states_bytes<T>(B, TT, D));
  const size_t sums = sums_bytes<T>(B, TT, D);
  if (sums && (!ws || (uintptr_t)ws % 16 || ws_bytes < sums))
    return set_error(kWorkspace, "tw_gated_scan_backward: workspace needs %zu bytes, 16-byte "
                     "aligned", sums);
  const T* dy = (const T*)dyv;
  const T* x = (const T*)xv;
  const T* g = (const T*)gv;
  const size_t BD = (size_t)B * D;
  if (D * sizeof(T) % 16 == 0 && pieces<T>(x, xb, xt) && pieces<T>(g, gb, gt) &&
      pieces<T>(dy, yb, yt) && pieces<T>(dx, 0, 0) && pieces<T>(dg, 0, 0) &&
      (uintptr_t)carry % 8 == 0) {
    const TilePlan p = tile_plan<T>(BD, TT, false);
    constexpr int MOST = 64 / sizeof(T);
    return p.whole
               ? bwd_tiles<T, MOST>(p, dy, yb, yt, dstate, x, xb, xt, g, gb, gt, lengths,
                                    (const float*)carry, BD, TT, D, (T*)dx, (T*)dg, dh0,
                                    (float2*)ws, stream)
               : bwd_tiles<T, MOST / 2>(p, dy, yb, yt, dstate, x, xb, xt, g, gb, gt, lengths,
                                        (const float*)carry, BD, TT, D, (T*)dx, (T*)dg, dh0,
                                        (float2*)ws, stream);
  }
  const ScanPlan p = scan_plan(BD, TT, sizeof(T));
  return launch(who, p.lpr == 32 ? scan_bwd_kernel<T, 1, 32> : scan_bwd_kernel<T, 1, 16>,
                p.groups, p.S, SCAN_THREADS, 0, stream, dy, yb, yt, dstate, x, xb, xt, g, gb, gt, lengths,
                (const float*)carry, BD, TT, D, p.S, (T*)dx, (T*)dg, dh0);
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

size_t tw_gated_scan_carry_bytes(int B, int T, int D, int dtype_bytes) {
  if (B <= 0 || T <= 0 || D <= 0) return 0;
  return tw_gated_scan_workspace_bytes(B, T, D, dtype_bytes) +
         (dtype_bytes == 4 ? tw::states_bytes<float>(B, T, D)
                           : tw::states_bytes<__nv_bfloat16>(B, T, D));
}
size_t tw_gated_scan_workspace_bytes(int B, int T, int D, int dtype_bytes) {
  if (B <= 0 || T <= 0 || D <= 0) return 0;
  return dtype_bytes == 4 ? tw::sums_bytes<float>(B, T, D)
                          : tw::sums_bytes<__nv_bfloat16>(B, T, D);
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
      void* dx, void* dgate, float* dh0, void* workspace, size_t ws_bytes, void* stream) {                                         \
    return tw::bwd<E>(dy, dy_batch, dy_time, dstate, x, x_batch, x_time, gate, g_batch, g_time,  \
                      lengths, carry, carry_bytes, B, T, D, dx, dgate, dh0, workspace, ws_bytes, stream);             \
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
