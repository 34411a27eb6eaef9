// One AdamW step over many tensors in one launch, states in 32 or 8 bits.
//
//   m = b1 m + (1 - b1) g, v = b2 v + (1 - b2) g^2
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// The states of all tensors lie in flat buffers, each tensor's on a boundary
// of 256 values.  In 8 bits m and sqrt(v) are e4m3 codes with one float32
// scale per 256 values (scale = largest magnitude / 448); sqrt(v), not v,
// because its square then spans 2^36 within a block.  Codes are rounded
// stochastically: a moving average moves by (1 - b2) of its distance a step,
// far less than half an e4m3 spacing, so rounding to nearest would never
// move it.  The random bits are a hash of the value's place, the step and
// the seed, so a step is reproducible.  The weight's update uses m and v in
// float32, before they are rounded.  An infinity or NaN becomes the code of
// NaN and has no part in its block's scale.
//
// The step count lives on the device, so a step can be captured in a CUDA
// graph: every block reads it, the last block to have read it stores the new
// one.
#include <cuda_fp8.h>

#include "../../include/torchwarp_b200.h"
#include "element.cuh"

namespace tw {
namespace {

constexpr int AD_UNIT = 256;     // values per scale, and per warp and turn
constexpr int AD_THREADS = 256;
constexpr int AD_TENSORS = 480;  // per launch

struct AdamEntry {
  void* p;
  const void* g;
  unsigned long long n;       // values
  unsigned long long offset;  // of its states, a multiple of AD_UNIT
};
struct AdamTable {
  AdamEntry e[AD_TENSORS];
  unsigned first[AD_TENSORS + 1];  // units before tensor i
  int count;
};
struct AdamState {
  float* m32;
  float* v32;
  uint8_t* m8;
  float* ms;
  uint8_t* r8;
  float* rs;
};
struct AdamScalars {
  double lr, b1, b2, eps, wd;
  const float* lr_dev;
  uint32_t seed;
  int* step;  // [0] steps done, [1] blocks that have read it
  int last;   // this launch ends the step
};

__device__ __forceinline__ uint32_t lowbias32(uint32_t h) {  // C. Wellons, hash prospector
  h ^= h >> 16;
  h *= 0x7FEB352Du;
  h ^= h >> 15;
  h *= 0x846CA68Bu;
  return h ^ (h >> 16);
}

// The maximum that keeps a NaN.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// The e4m3 value next to y >= 0 (in units of the scale): below, or above with
// the probability of the part of a spacing that is cut off, r in [0, 2^20)
// being the random number.  A float has 20 bits below e4m3's three, so adding
// r and clearing them does it; below 2^-6, where e4m3's spacing stays 2^-9,
// after adding 2^-6, which has that spacing.
__device__ __forceinline__ float round_e4m3(float y, uint32_t r) {
  const float low = y < 0.015625f ? 0.015625f : 0.f;
  const uint32_t bits = (__float_as_uint(y + low) + r) & 0xFFF00000u;
  return fminf(__uint_as_float(bits) - low, 448.f);
}

// b^t by squaring, to a few ulp.
__device__ __forceinline__ double power(double b, int t) {
  double r = 1.0;
  for (; t > 0; t >>= 1, b *= b)
    if (t & 1) r *= b;
  return r;
}

__device__ __forceinline__ float sqrt_fast(float x) {
  float y;
  asm("sqrt.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// Eight neighbours.  Plain loads: the kernel writes these arrays too.
template <typename T>
__device__ __forceinline__ void read8(const T* p, float* v) {
  constexpr int PER = 16 / sizeof(T);
#pragma unroll
  for (int i = 0; i < 8 / PER; ++i)
    unpack16<T>(reinterpret_cast<const uint4*>(p)[i], v + i * PER);
}

// Eight neighbouring e4m3 codes as floats, and back.
__device__ __forceinline__ void decode8(uint2 c, float scale, float* v) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_fp8x2_storage_t two = (__nv_fp8x2_storage_t)((i < 2 ? c.x : c.y) >> (16 * (i & 1)));
    const float2 f = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(two, __NV_E4M3)));
    v[2 * i] = f.x * scale;
    v[2 * i + 1] = f.y * scale;
  }
}
__device__ __forceinline__ unsigned long long encode8(const float* v) {
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    w[i] = (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(v[4 * i], v[4 * i + 1]), __NV_SATFINITE,
                                              __NV_E4M3) |
           (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(v[4 * i + 2], v[4 * i + 3]),
                                              __NV_SATFINITE, __NV_E4M3)
               << 16;
  return (unsigned long long)w[1] << 32 | w[0];
}

// A warp takes a unit of 256 values a turn, 8 neighbours a lane.  Bound by HBM
// (28 bytes a float32 weight with 32-bit states, 16 with 8-bit ones): every
// array is read with 16-byte loads, all issued before the first is used.  A
// unit whose parameter or gradient is not 16-byte aligned, and a tensor's
// last, partial unit, go value by value.  67 million float32 weights with
// 32-bit states: 285 us, 6.6 TB/s, a copy's rate (622 us value by value).
// 2.1 million bfloat16 weights with 8-bit states: 15 us, of which the bytes are
// 3; half of the issue slots are empty, as each short-lived block reads the step,
// raises the betas to it and meets at a barrier before its first load.
template <typename T, bool BITS8>
__global__ void __launch_bounds__(AD_THREADS)
    adamw_kernel(const __grid_constant__ AdamTable tab, AdamState s, AdamScalars a) {
  __shared__ float sc[4];
  __shared__ uint32_t skey;
  if (threadIdx.x < 2) {  // one thread for each beta
    const int t = *(volatile int*)a.step + 1;
    const double lr = a.lr_dev ? (double)*a.lr_dev : a.lr;
    const double rest = 1.0 - power(threadIdx.x ? a.b2 : a.b1, t);
    if (threadIdx.x == 0) {
      sc[0] = (float)(1.0 - lr * a.wd);
      sc[1] = (float)(lr / rest);
      skey = a.seed * 0x9E3779B1u + (uint32_t)t * 0x85EBCA77u;
    } else {
      sc[2] = (float)(1.0 / sqrt(rest));
    }
    __syncwarp(3);
    if (threadIdx.x == 0) {
      __threadfence();
      if (a.last && atomicAdd(&a.step[1], 1) == (int)gridDim.x - 1) {
        a.step[1] = 0;
        a.step[0] = t;
      }
    }
  }
  __syncthreads();
  const float keep = sc[0], alpha = sc[1], root2 = sc[2];
  const float b1 = (float)a.b1, c1 = (float)(1.0 - a.b1), b2 = (float)a.b2,
              c2 = (float)(1.0 - a.b2), eps = (float)a.eps;
  const uint32_t key = skey;
  const int lane = threadIdx.x & 31;
  const unsigned units = tab.first[tab.count];
  int lo = 0;
  for (unsigned u = blockIdx.x * (AD_THREADS / 32) + (threadIdx.x >> 5); u < units;
       u += gridDim.x * (AD_THREADS / 32)) {
    int hi = tab.count - 1;  // the tensor of this unit: not before the last one's
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (tab.first[mid] <= u) lo = mid; else hi = mid - 1;
    }
    const unsigned long long at = (unsigned long long)(u - tab.first[lo]) * AD_UNIT;
    const unsigned long long so = tab.e[lo].offset + at;
    const int n = (int)min((unsigned long long)AD_UNIT, tab.e[lo].n - at) - 8 * lane;  // lane's
    T* p = (T*)tab.e[lo].p + at + 8 * lane;
    const T* g = (const T*)tab.e[lo].g + at + 8 * lane;
    const unsigned long long sl = so + 8 * lane;
    const bool vec = n >= 8 && (((uintptr_t)p | (uintptr_t)g) & 15) == 0;
    float m[8], r[8], pv[8], gv[8];
    // the states' buffers are padded to whole units
    if (BITS8) {
      const uint2 mc = *reinterpret_cast<const uint2*>(s.m8 + sl);
      const uint2 rc = *reinterpret_cast<const uint2*>(s.r8 + sl);
      const float ms = s.ms[so / AD_UNIT], rs = s.rs[so / AD_UNIT];
      decode8(mc, ms, m);
      decode8(rc, rs, r);
    } else {
      read8(s.m32 + sl, m);
      read8(s.v32 + sl, r);
    }
    if (vec) {
      load_n<true, 8>(g, gv);
      read8(p, pv);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        gv[i] = i < n ? to_f(g[i]) : 0.f;
        pv[i] = i < n ? to_f(p[i]) : 0.f;
      }
    }
    float mmax = 0.f, rmax = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float v = fmaf(b2, BITS8 ? r[i] * r[i] : r[i], c2 * (gv[i] * gv[i]));
      m[i] = fmaf(b1, m[i], c1 * gv[i]);
      r[i] = sqrt_fast(v);
      pv[i] = pv[i] * keep - alpha * __fdividef(m[i], fmaf(r[i], root2, eps));
      if (!BITS8) r[i] = v;
      mmax = max_nan(mmax, fabsf(m[i]));
      rmax = max_nan(rmax, r[i]);
    }
    if (vec) {
      store_n<true, 8>(p, pv);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < n) p[i] = from_f<T>(pv[i]);
    }
    if (!BITS8) {
      store_n<true, 8>(s.m32 + sl, m);
      store_n<true, 8>(s.v32 + sl, r);
    } else {
      unsigned long long spoiled_m = 0, spoiled_r = 0;  // codes of NaN
      mmax = warp_max(mmax);
      rmax = warp_max(rmax);
      if (!(mmax < INFINITY && rmax < INFINITY)) {
        // an infinity or NaN stays in its place, as the code of NaN: the scale
        // is that of the finite values
        mmax = rmax = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (!(fabsf(m[i]) < INFINITY)) {
            m[i] = 0.f;
            spoiled_m |= 0x7Full << (8 * i);
          }
          if (!(r[i] < INFINITY)) {
            r[i] = 0.f;
            spoiled_r |= 0x7Full << (8 * i);
          }
          mmax = fmaxf(mmax, fabsf(m[i]));
          rmax = fmaxf(rmax, r[i]);
        }
        mmax = warp_max(mmax);
        rmax = warp_max(rmax);
      }
      // a block below 1e-37, whose scale has no reciprocal, is zero
      float nms = mmax / 448.f, nrs = rmax / 448.f;
      if (nms < 1e-37f) nms = 0.f;
      if (nrs < 1e-37f) nrs = 0.f;
      const float ims = nms > 0.f ? 1.f / nms : 0.f, irs = nrs > 0.f ? 1.f / nrs : 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t h = lowbias32((uint32_t)(sl + i) ^ key);
        const float yr = r[i] * irs;
        m[i] = copysignf(round_e4m3(fabsf(m[i]) * ims, (h & 0xFFFFu) << 4),
                         m[i]);
        r[i] = round_e4m3(yr, (h >> 16) << 4);
        // a second moment that is not zero stays above zero: it divides m
        if (yr > 0.f) r[i] = fmaxf(r[i], 0.001953125f);
      }
      // a spoiled value was made zero: 0x7F over its code, whatever its sign
      *reinterpret_cast<unsigned long long*>(s.m8 + sl) = encode8(m) | spoiled_m;
      *reinterpret_cast<unsigned long long*>(s.r8 + sl) = encode8(r) | spoiled_r;
      if (lane == 0) {
        s.ms[so / AD_UNIT] = nms;
        s.rs[so / AD_UNIT] = nrs;
      }
    }
  }
}

template <typename T>
int step(const uint64_t* table, int count, int bits, void* m, float* ms, void* v, float* vs,
         int* step_state, double lr, const float* lr_dev, double b1, double b2, double eps,
         double wd, size_t seed, void* stream) {
  set_error(kOk, "%s", "");
  if (count < 0 || (bits != 8 && bits != 32))
    return set_error(kInvalid, "tw_adamw_step: invalid count=%d or state_bits=%d (8 or 32)", count,
                     bits);
  if (!(b1 >= 0 && b1 < 1 && b2 >= 0 && b2 < 1 && eps >= 0))
    return set_error(kInvalid, "tw_adamw_step: need 0 <= beta < 1 and eps >= 0");
  if (!step_state || (count && (!table || !m || !v || (bits == 8 && (!ms || !vs)))))
    return set_error(kInvalid, "tw_adamw_step: null pointer argument");
  AdamState s = {};
  if (bits == 32) {
    s.m32 = (float*)m;
    s.v32 = (float*)v;
  } else {
    s.m8 = (uint8_t*)m;
    s.ms = ms;
    s.r8 = (uint8_t*)v;
    s.rs = vs;
  }
  AdamScalars a = {lr, b1, b2, eps, wd, lr_dev, (uint32_t)seed, step_state, 0};
  int at = 0;
  do {
    AdamTable tab;
    tab.count = 0;
    unsigned long long units = 0;
    tab.first[0] = 0;
    for (; at < count && tab.count < AD_TENSORS; ++at) {
      const uint64_t* e = table + 4 * (size_t)at;
      if (e[2] == 0) continue;
      if (!e[0] || !e[1] || e[3] % AD_UNIT)
        return set_error(kInvalid, "tw_adamw_step: tensor %d has a null pointer or a state offset "
                         "that is no multiple of %d", at, AD_UNIT);
      const unsigned long long mine = (e[2] + AD_UNIT - 1) / AD_UNIT;
      if (mine >= 0x7fffffffull)
        return set_error(kUnsupported, "tw_adamw_step: tensor %d is too large", at);
      if (units + mine >= 0x7fffffffull) break;
      units += mine;
      tab.e[tab.count] = {(void*)e[0], (const void*)e[1], e[2], e[3]};
      tab.first[++tab.count] = (unsigned)units;
    }
    a.last = at >= count;
    const unsigned long long blocks = (units + AD_THREADS / 32 - 1) / (AD_THREADS / 32);
    // short-lived blocks: what is in flight then lies close together in memory
    // (67 million float32 weights: 345 us with 8 blocks a SM that stride through
    // all, 302 with 16, 290 with 32, 285 with 64, 315 with one turn a block)
    const unsigned most = 148 * 64;
    const unsigned grid = (unsigned)(blocks < 1 ? 1 : blocks < most ? blocks : most);
    cudaStream_t st = (cudaStream_t)stream;
    if (bits == 8)
      adamw_kernel<T, true><<<grid, AD_THREADS, 0, st>>>(tab, s, a);
    else
      adamw_kernel<T, false><<<grid, AD_THREADS, 0, st>>>(tab, s, a);
    const cudaError_t err = cudaGetLastError();
    if (err != cudaSuccess)
      return set_error(kLaunch, "tw_adamw_step: %s", cudaGetErrorString(err));
  } while (at < count);
  return kOk;
}

}  // namespace
}  // namespace tw

extern "C" {

#define TW_ADAMW(SUFFIX, T)                                                                       \
  int tw_adamw_step_##SUFFIX(const uint64_t* table, int count, int state_bits, void* exp_avg,     \
                             float* exp_avg_scale, void* exp_avg_sq, float* exp_avg_sq_scale,     \
                             int* step, double lr, const float* lr_device, double beta1,          \
                             double beta2, double eps, double weight_decay, size_t seed,          \
                             void* stream) {                                                      \
    return tw::step<T>(table, count, state_bits, exp_avg, exp_avg_scale, exp_avg_sq,              \
                       exp_avg_sq_scale, step, lr, lr_device, beta1, beta2, eps, weight_decay,    \
                       seed, stream);                                                             \
  }

TW_ADAMW(f32, float)
TW_ADAMW(bf16, __nv_bfloat16)
TW_ADAMW(f16, __half)

}  // extern "C"
