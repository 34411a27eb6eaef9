// Element types of the encoder operators (layer norm, linear, gated scan,
// AdamW): float, bfloat16 and half in memory, float in registers.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"

namespace tw {

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

// f = sigmoid(z) and 1 - f: the smaller of the two from exp(-|z|), which
// neither overflows nor cancels, to a few ulp of itself; the larger is one
// minus it, correctly rounded.
__device__ __forceinline__ void sigmoid_pair(float z, float& f, float& omf) {
  const float e = ex2(-1.4426950408889634f * fabsf(z));
  const float lo = e * rcp(1.f + e), hi = 1.f - lo;
  f = z >= 0.f ? hi : lo;
  omf = z >= 0.f ? lo : hi;
}

// Activations of the linear operator (values of the `act` argument).
enum Act : int { kActNone = 0, kActRelu = 1, kActGelu = 2, kActSilu = 3, kActSigmoid = 4 };

// FAST (results rounded to 16 bits): the normal distribution function
// through Abramowitz & Stegun 7.1.26, erfc(x) = (a1 t + .. + a5 t^5) e^(-x^2)
// with t = 1 / (1 + p x), |error| <= 1.5e-7: one exponential and one
// reciprocal in place of erff's two polynomial branches.  e is e^(-z^2/2).
__device__ __forceinline__ float normal_cdf_fast(float z, float& e) {
  const float t = rcp(__fmaf_rn(0.3275911f * 0.70710678118654752f, fabsf(z), 1.f));
  e = ex2(mul_rn(mul_rn(-0.72134752044448170f, z), z));
  float q = __fmaf_rn(1.061405429f, t, -1.453152027f);
  q = __fmaf_rn(q, t, 1.421413741f);
  q = __fmaf_rn(q, t, -0.284496736f);
  q = __fmaf_rn(q, t, 0.254829592f);
  q = mul_rn(mul_rn(mul_rn(q, t), 0.5f), e);
  return z < 0.f ? q : add_rn(1.f, -q);
}

// The roundings are explicit: a call that saves z gives the bits of one that
// does not, whatever the compiler contracts around it.
template <int ACT, bool FAST>
__device__ __forceinline__ float act_value(float z) {
  if (ACT == kActRelu) return z < 0.f ? 0.f : z;  // a NaN stays a NaN
  if (ACT == kActGelu && FAST) {
    float e;
    return mul_rn(z, normal_cdf_fast(z, e));
  }
  if (ACT == kActGelu) {
    const float h = mul_rn(0.5f, z);
    return __fmaf_rn(h, erff(mul_rn(z, 0.70710678118654752f)), h);
  }
  if (ACT == kActSilu || ACT == kActSigmoid) {
    float f, omf;
    sigmoid_pair(z, f, omf);
    return ACT == kActSilu ? mul_rn(z, f) : f;
  }
  return z;
}

// d act / dz at z.
template <int ACT, bool FAST>
__device__ __forceinline__ float act_slope(float z) {
  if (ACT == kActRelu) return z > 0.f ? 1.f : (z != z ? z : 0.f);
  if (ACT == kActGelu) {
    float cdf, e;
    if (FAST) {
      cdf = normal_cdf_fast(z, e);
    } else {
      cdf = 0.5f * (1.f + erff(z * 0.70710678118654752f));
      e = ex2(-0.72134752044448170f * z * z);
    }
    return fmaf(z, 0.39894228040143268f * e, cdf);
  }
  if (ACT == kActSilu || ACT == kActSigmoid) {
    float f, omf;
    sigmoid_pair(z, f, omf);
    return ACT == kActSilu ? f * fmaf(z, omf, 1.f) : f * omf;
  }
  return 1.f;
}

}  // namespace tw
