// Element types of the encoder operators (layer norm, linear, gated scan,
// AdamW): float, bfloat16 and half in memory, float in registers.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"

namespace tw {

// A kernel launched with launch_after may start while the one before it runs:
// after_previous() waits until that one is complete and its writes are seen
// (it returns at once after an ordinary launch), let_next_start() lets the one
// behind it start.  Every kernel of such a chain calls both, the wait before
// it touches global memory, so a kernel's inputs may come from any before it.
__device__ __forceinline__ void after_previous() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}
__device__ __forceinline__ void let_next_start() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// Launches a kernel behind the last one of `stream`, as above when `after`.
template <typename... Params, typename... Args>
cudaError_t launch_after(bool after, void (*kernel)(Params...), dim3 grid, dim3 block, size_t smem,
                         int cluster, cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  if (cluster > 1) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = cluster;
    attr[cfg.numAttrs].val.clusterDim.y = attr[cfg.numAttrs].val.clusterDim.z = 1;
    ++cfg.numAttrs;
  }
  if (after) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
    ++cfg.numAttrs;
  }
  cfg.attrs = attr;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }

// One rounding, to nearest even, when a result leaves the registers.
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <> __device__ __forceinline__ __half from_f<__half>(float v) {
  return __float2half_rn(v);
}

// Two 16-bit elements of a word as floats, and back: one conversion a pair.
template <typename T> struct Pair;
template <> struct Pair<__nv_bfloat16> {
  static __device__ __forceinline__ void unpack(uint32_t u, float& a, float& b) {
    a = __uint_as_float(u << 16);
    b = __uint_as_float(u & 0xFFFF0000u);
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
};
template <> struct Pair<__half> {
  static __device__ __forceinline__ void unpack(uint32_t u, float& a, float& b) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u));
    a = f.x;
    b = f.y;
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
};

// The 16 / sizeof(T) elements of 16 bytes as floats, and back.
template <typename T>
__device__ __forceinline__ void unpack16(const uint4& u, float* v) {
  if constexpr (sizeof(T) == 4) {
    v[0] = __uint_as_float(u.x);
    v[1] = __uint_as_float(u.y);
    v[2] = __uint_as_float(u.z);
    v[3] = __uint_as_float(u.w);
  } else {
    Pair<T>::unpack(u.x, v[0], v[1]);
    Pair<T>::unpack(u.y, v[2], v[3]);
    Pair<T>::unpack(u.z, v[4], v[5]);
    Pair<T>::unpack(u.w, v[6], v[7]);
  }
}
template <typename T>
__device__ __forceinline__ uint4 pack16(const float* v) {
  if constexpr (sizeof(T) == 4)
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]),
                      __float_as_uint(v[3]));
  else
    return make_uint4(Pair<T>::pack(v[0], v[1]), Pair<T>::pack(v[2], v[3]),
                      Pair<T>::pack(v[4], v[5]), Pair<T>::pack(v[6], v[7]));
}

// N consecutive elements as floats, and back; with VEC in pieces of 16 bytes
// (the address is 16-byte aligned), else one by one.
template <bool VEC, int N, typename T>
__device__ __forceinline__ void load_n(const T* p, float* v) {
  constexpr int PER = 16 / sizeof(T);
  if constexpr (VEC && N % PER == 0) {
#pragma unroll
    for (int i = 0; i < N / PER; ++i)
      unpack16<T>(__ldg(reinterpret_cast<const uint4*>(p) + i), v + i * PER);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = to_f(p[i]);
  }
}
template <bool VEC, int N, typename T>
__device__ __forceinline__ void store_n(T* p, const float* v) {
  constexpr int PER = 16 / sizeof(T);
  if constexpr (VEC && N % PER == 0) {
#pragma unroll
    for (int i = 0; i < N / PER; ++i)
      reinterpret_cast<uint4*>(p)[i] = pack16<T>(v + i * PER);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = from_f<T>(v[i]);
  }
}

// What load_n reads, kept as it is until it is used: half the registers of
// 16-bit elements as floats.
template <bool VEC, int N, typename T> struct Raw {
  static constexpr int PER = 16 / sizeof(T);
  static constexpr int WORDS = VEC ? N / PER : N;
  typename std::conditional<VEC, uint4, T>::type w[WORDS];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < WORDS; ++i) w[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
    } else {
#pragma unroll
      for (int i = 0; i < WORDS; ++i) w[i] = p[i];
    }
  }
  __device__ __forceinline__ void zero() {
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < WORDS; ++i) w[i] = make_uint4(0, 0, 0, 0);
    } else {
#pragma unroll
      for (int i = 0; i < WORDS; ++i) w[i] = from_f<T>(0.f);
    }
  }
  __device__ __forceinline__ void get(float* v) const {
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < WORDS; ++i) unpack16<T>(w[i], v + i * PER);
    } else {
#pragma unroll
      for (int i = 0; i < WORDS; ++i) v[i] = to_f(w[i]);
    }
  }
};

// V floats that go through the arithmetic together: pairs use the packed
// instructions (two results each), which halve its issue slots.
template <int V> struct Vec { float v[V]; };

template <int V>
__device__ __forceinline__ Vec<V> splat(float x) {
  Vec<V> r;
#pragma unroll
  for (int i = 0; i < V; ++i) r.v[i] = x;
  return r;
}
__device__ __forceinline__ uint64_t two(const Vec<2>& a) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a.v[0]), "f"(a.v[1]));
  return r;
}
__device__ __forceinline__ Vec<2> of_two(uint64_t a) {
  Vec<2> r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.v[0]), "=f"(r.v[1]) : "l"(a));
  return r;
}
__device__ __forceinline__ Vec<1> fma_v(Vec<1> a, Vec<1> b, Vec<1> c) {
  return {{fmaf(a.v[0], b.v[0], c.v[0])}};
}
__device__ __forceinline__ Vec<2> fma_v(Vec<2> a, Vec<2> b, Vec<2> c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(two(a)), "l"(two(b)), "l"(two(c)));
  return of_two(r);
}
__device__ __forceinline__ Vec<1> add_v(Vec<1> a, Vec<1> b) { return {{a.v[0] + b.v[0]}}; }
__device__ __forceinline__ Vec<2> add_v(Vec<2> a, Vec<2> b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(two(a)), "l"(two(b)));
  return of_two(r);
}
__device__ __forceinline__ Vec<1> mul_v(Vec<1> a, Vec<1> b) { return {{a.v[0] * b.v[0]}}; }
__device__ __forceinline__ Vec<2> mul_v(Vec<2> a, Vec<2> b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(two(a)), "l"(two(b)));
  return of_two(r);
}
template <int V>
__device__ __forceinline__ Vec<V> sub_v(Vec<V> a, Vec<V> b) {  // a - b
  return fma_v(b, splat<V>(-1.f), a);
}

template <int V>
__device__ __forceinline__ Vec<V> negated(Vec<V> s) {
#pragma unroll
  for (int i = 0; i < V; ++i) s.v[i] = -s.v[i];
  return s;
}

// e^-|z| for float32 results: 2^(-|z| log2(e) / 2) squared, so that it reaches
// the subnormals (ex2 flushes them), times 1 + what the product's rounding left
// over; within 2^-21.  It is 0 from 110 on.
template <int V>
__device__ __forceinline__ Vec<V> exp_minus_abs(Vec<V> z) {
  constexpr double C = 0.72134752044448170368;  // log2(e) / 2
  constexpr float HI = (float)C, LO = (float)(C - (double)HI);
  Vec<V> a, e;
#pragma unroll
  for (int i = 0; i < V; ++i)  // -|z|, not below -110; a NaN stays one
    asm("max.NaN.f32 %0, %1, 0fC2DC0000;" : "=f"(a.v[i]) : "f"(fminf(z.v[i], -z.v[i])));
  const Vec<V> t = mul_v(a, splat<V>(HI));
  // minus (a log2(e) / 2 - t)
  const Vec<V> rest = fma_v(a, splat<V>(-LO), fma_v(a, splat<V>(-HI), t));
#pragma unroll
  for (int i = 0; i < V; ++i) e.v[i] = ex2(t.v[i]);
  e = mul_v(e, e);
  return fma_v(e, mul_v(rest, splat<V>(-1.3862943611198906f)), e);
}

// f = sigmoid(z) and 1 - f: the smaller of the two from exp(-|z|), which
// neither overflows nor cancels, to a few ulp of itself, down to the smallest
// float; the larger is one minus it, correctly rounded.  FAST: for results of
// 16 bits; the product z log2(e) is rounded, so the smaller one's relative
// error grows as |z| 2^-24, and below 2^-126 it is 0.
template <bool FAST, int V>
__device__ __forceinline__ void sigmoid_pair(Vec<V> z, Vec<V>& f, Vec<V>& omf) {
  Vec<V> e, r;
  if constexpr (FAST) {
    e = mul_v(z, splat<V>(1.4426950408889634f));
#pragma unroll
    for (int i = 0; i < V; ++i) e.v[i] = ex2(-fabsf(e.v[i]));
  } else {
    e = exp_minus_abs(z);
  }
  r = add_v(e, splat<V>(1.f));
#pragma unroll
  for (int i = 0; i < V; ++i) r.v[i] = rcp(r.v[i]);
  const Vec<V> lo = mul_v(e, r), hi = sub_v(splat<V>(1.f), lo);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    f.v[i] = z.v[i] >= 0.f ? hi.v[i] : lo.v[i];
    omf.v[i] = z.v[i] >= 0.f ? lo.v[i] : hi.v[i];
  }
}

// Activations of the linear operator (values of the `act` argument).
enum Act : int { kActNone = 0, kActRelu = 1, kActGelu = 2, kActSilu = 3, kActSigmoid = 4 };

// Upper tail of the normal distribution at |z| (results rounded to 16 bits),
// through Abramowitz & Stegun 7.1.26: erfc(x) = (a1 t + .. + a5 t^5) e^(-x^2)
// with t = 1 / (1 + p x), |error| <= 1.5e-7, x = |z| / sqrt 2; one exponential
// and one reciprocal in place of erff's two polynomial branches.  The factor
// 1/2 is in the coefficients.  az is |z| (cut at 30, where the tail is 0, so
// that an infinity times it is not a NaN), e is e^(-z^2 / 2).
template <int V>
__device__ __forceinline__ Vec<V> normal_tail(Vec<V> z, Vec<V>& az, Vec<V>& e) {
#pragma unroll
  for (int i = 0; i < V; ++i) az.v[i] = fminf(fabsf(z.v[i]), 30.f);
  Vec<V> t = fma_v(az, splat<V>(0.3275911f * 0.70710678118654752f), splat<V>(1.f));
  e = mul_v(mul_v(z, z), splat<V>(-0.72134752044448170f));
#pragma unroll
  for (int i = 0; i < V; ++i) {
    t.v[i] = rcp(t.v[i]);
    e.v[i] = ex2(e.v[i]);
  }
  Vec<V> q = fma_v(splat<V>(0.5f * 1.061405429f), t, splat<V>(-0.5f * 1.453152027f));
  q = fma_v(q, t, splat<V>(0.5f * 1.421413741f));
  q = fma_v(q, t, splat<V>(-0.5f * 0.284496736f));
  q = fma_v(q, t, splat<V>(0.5f * 0.254829592f));
  return mul_v(mul_v(q, t), e);
}

// act(z).  FAST: for results of 16 bits.  The roundings are explicit: a call
// that saves z gives the bits of one that does not, whatever the compiler
// contracts around it.
template <int ACT, bool FAST, int V>
__device__ __forceinline__ Vec<V> act_value(Vec<V> z) {
  if constexpr (ACT == kActGelu && FAST) {  // z Phi(z) = max(z, 0) - |z| tail(|z|)
    Vec<V> az, e, r;
    const Vec<V> q = normal_tail(z, az, e);
#pragma unroll
    for (int i = 0; i < V; ++i) r.v[i] = fmaxf(z.v[i], 0.f);
    return fma_v(negated(az), q, r);
  } else if constexpr ((ACT == kActSilu || ACT == kActSigmoid) && FAST) {
    Vec<V> f = mul_v(z, splat<V>(-1.4426950408889634f));
#pragma unroll
    for (int i = 0; i < V; ++i) f.v[i] = ex2(f.v[i]);
    f = add_v(f, splat<V>(1.f));
#pragma unroll
    for (int i = 0; i < V; ++i) f.v[i] = rcp(f.v[i]);
    return ACT == kActSilu ? mul_v(z, f) : f;
  } else if constexpr (ACT == kActSilu || ACT == kActSigmoid) {
    Vec<V> f, omf;
    sigmoid_pair<false>(z, f, omf);
    return ACT == kActSilu ? mul_v(z, f) : f;
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float& v = z.v[i];
      if (ACT == kActRelu) v = v < 0.f ? 0.f : v;  // a NaN stays a NaN
      if (ACT == kActGelu) {
        const float h = mul_rn(0.5f, v);
        v = __fmaf_rn(h, erff(mul_rn(v, 0.70710678118654752f)), h);
      }
    }
    return z;
  }
}

// d act / dz at z.  z may be infinite where the forward was not: a saved z is
// rounded to 16 bits.  Where a factor vanishes or is 1, the z it meets is cut
// to a finite value; a NaN stays in the other factor.
template <int ACT, bool FAST, int V>
__device__ __forceinline__ Vec<V> act_slope(Vec<V> z) {
  if constexpr (ACT == kActGelu && FAST) {  // Phi(z) + z phi(z)
    Vec<V> az, e;
    Vec<V> c = fma_v(normal_tail(z, az, e), splat<V>(-1.f), splat<V>(0.5f));
#pragma unroll
    for (int i = 0; i < V; ++i) {
      c.v[i] = copysignf(c.v[i], z.v[i]);
      az.v[i] = copysignf(az.v[i], z.v[i]);  // at the cut e is 0
    }
    return fma_v(mul_v(az, splat<V>(0.39894228040143268f)), e, add_v(c, splat<V>(0.5f)));
  } else if constexpr (ACT == kActSilu || ACT == kActSigmoid) {
    Vec<V> f, omf;
    sigmoid_pair<FAST>(z, f, omf);
    if constexpr (ACT == kActSigmoid) {
      return mul_v(f, omf);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) z.v[i] = fmaxf(fminf(z.v[i], 128.f), -128.f);
      return mul_v(f, fma_v(z, omf, splat<V>(1.f)));
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float& v = z.v[i];
      if (ACT == kActRelu) v = v > 0.f ? 1.f : (v != v ? v : 0.f);
      if (ACT == kActGelu) {
        const float cdf = 0.5f * (1.f + erff(v * 0.70710678118654752f));
        const float e = 0.39894228040143268f * ex2(-0.72134752044448170f * v * v);
        v = fmaf(fmaxf(fminf(v, 30.f), -30.f), e, cdf);
      }
      if (ACT == kActNone) v = 1.f;
    }
    return z;
  }
}

// One value, the activation chosen at run time.
template <bool FAST>
__device__ __forceinline__ float activate1(float v, int act) {
  const Vec<1> z = {{v}};
  switch (act) {
    case kActRelu: return act_value<kActRelu, FAST>(z).v[0];
    case kActGelu: return act_value<kActGelu, FAST>(z).v[0];
    case kActSilu: return act_value<kActSilu, FAST>(z).v[0];
    case kActSigmoid: return act_value<kActSigmoid, FAST>(z).v[0];
    default: return v;
  }
}

}  // namespace tw
