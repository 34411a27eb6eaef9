// The tensor-core product of the linear operator: tcgen05.mma with TMA-fed
// shared memory and accumulators in TMEM, for one output type T per
// translation unit.
//
//   out = act(A B^T + bias) + residual, either operand K-major or MN-major
//
// Tiles are 128 rows a CTA by TN columns; in the pair form (CG = 2) two CTAs
// share a 256 x TN tile, each with its own half of A and of B in shared
// memory, so that a chunk costs 32 KB of L2 traffic per 128 x 256 x 64
// products where one CTA alone would load 48 KB.
//
// float32 operands come as three bfloat16 planes whose sum is exact (8 + 8 +
// 8 mantissa bits) down to 2^-110, below which the last bits fall under
// bfloat16's smallest value, 2^-133.  The six products of weight 2^-16 and above are taken:
// p0 q0 in one accumulator, the five small ones in another, so that the
// rounding of the large sum does not reach them.  An infinity or NaN is in p0
// or q0 alone; in the small products it meets planes that are 0 or of the other
// sign, so where the large sum is not finite it counts alone.  The tensor core
// truncates its accumulator; every SEG_CHUNKS chunks the two are added to float32
// registers, rounding to nearest, which keeps that bias to a few steps.
//
// Warps 0 .. EW - 1: epilogue (TMEM lane quadrant warp % 4, a share of the
// columns each); then one warp for TMA and one for TMEM allocation and MMA
// issue (of the pair's first CTA).  A warp's way through a piece is a chain of
// latencies (TMEM, exponential and reciprocal, staging, fence), so wide tiles
// take 16 of them: with 8 the gelu epilogue paced the 32768 x 1024 x 4096
// product (262 us).  Two accumulator sets let the epilogue of a tile overlap the next
// tile's products.  No atomics: results are reproducible.
//
// 32768 x 4096 x 1024 bfloat16 (dz w): 176 us, 1560 TFLOP/s, the tensor pipe
// active in 90% of the cycles.  32768 x 1024 x 4096 with gelu and z: 230 us, 67%:
// the two 16-bit outputs pass through shared memory beside the operands.
// 4096^3 float32: 640 us, 215 TFLOP/s of float32 products.
#pragma once

#include "element.cuh"
#include "linear_gemm.h"
#include "tc_common.cuh"

namespace tw {
namespace {

using namespace tc;

__device__ int g_gemm_error;

constexpr int BK = 64;                // contraction values per chunk: one 128-byte line
constexpr int A_PLANE = 128 * BK * 2;
constexpr int SMEM_MAX = 232448;
constexpr int SHARED_MAX = 2048;

template <typename T> struct Elem {
  static constexpr int PL = 1;
  static constexpr uint32_t FMT = 1;  // bfloat16
  static constexpr int STG = 4096;    // y and z: 32 rows x 64 bytes each, or 32 x 32 floats
};
template <> struct Elem<__half> {
  static constexpr int PL = 1;
  static constexpr uint32_t FMT = 0;
  static constexpr int STG = 4096;
};
template <> struct Elem<float> {
  static constexpr int PL = 3;
  static constexpr uint32_t FMT = 1;
  static constexpr int STG = 4096;
};

template <typename T, int CG, int TN> struct Geom {
  static constexpr int PL = Elem<T>::PL;
  static constexpr int B_ROWS = TN / CG;
  static constexpr int B_PLANE = B_ROWS * BK * 2;
  static constexpr int STAGE = PL * (A_PLANE + B_PLANE);
  // float32 keeps 8: its stages leave no room for more staging
  static constexpr int EW = TN >= 128 && PL == 1 ? 16 : 8;  // epilogue warps
  static constexpr int THREADS = 32 * (EW + 2);
  static constexpr int FIT = (SMEM_MAX - SHARED_MAX - EW * Elem<T>::STG) / STAGE;
  static constexpr int STAGES = FIT < 8 ? FIT : 8;
  static constexpr int SEG_CHUNKS = 2;
  static constexpr int ACC = TN * (PL == 3 ? 2 : 1);  // TMEM columns of one accumulator set
  static constexpr int SMEM = STAGES * STAGE + EW * Elem<T>::STG + SHARED_MAX;
  static constexpr int COLS = TN / (EW / 4);          // of a warp
  static constexpr int CHUNKS32 = COLS / 32;          // in pieces of 32
};

struct GemmShared {
  __align__(16) uint8_t bias[1024];  // of each epilogue warp: 32 elements
  uint64_t full[8], empty[8], accf[2], acce[2], mma_done;
  uint32_t tmem_base;
  int abort;
};
static_assert(sizeof(GemmShared) <= SHARED_MAX, "shared block");

template <typename T> struct GemmArgs {
  int M, N, K, nK, tiles_m, tiles_n, items, splits, per_split;
  const T* bias;
  const T* res;
  size_t ldr;
  T* out;
  T* z;
  float* partial;
  int act, res_vec, tma_store;
};

// The tile of an item: bands of TILE_BAND rows of tiles, down a band's columns,
// so that the tiles in flight at once are near a square and share their A and
// B panels in L2.
constexpr int TILE_BAND = 8;
struct TileAt {
  int m, n, split;
};
template <typename T>
__device__ __forceinline__ TileAt tile_at(int w, const GemmArgs<T>& g) {
  const int tile = w / g.splits;
  const int per_band = TILE_BAND * g.tiles_n, band = tile / per_band;
  const int rows = min(TILE_BAND, g.tiles_m - band * TILE_BAND), r = tile - band * per_band;
  return {band * TILE_BAND + r % rows, r / rows, w - tile * g.splits};
}

__device__ __forceinline__ uint32_t cta_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The address, in the cluster's window, of a shared object of CTA `rank`.
__device__ __forceinline__ uint32_t peer_addr(const void* p, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  return a;
}
__device__ __forceinline__ void arrive_at(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr)
               : "memory");
}

// Waits give up after this many cycles (some seconds): a correct pipeline
// never comes close.
constexpr long long WAIT_CYCLES = 1LL << 33;

__device__ __forceinline__ bool wait_plain(uint64_t* bar, unsigned parity) {
  const long long t0 = clock64();
  while (!mbar_try_wait(bar, parity))
    if (clock64() - t0 > WAIT_CYCLES) return false;
  return true;
}
// The same, also ended by another role that gave up; then records it.
__device__ __forceinline__ bool wait_for(uint64_t* bar, unsigned parity, volatile int* abort) {
  if (mbar_try_wait(bar, parity)) return true;
  const long long t0 = clock64();
  while (!mbar_try_wait(bar, parity)) {
    if (*abort || clock64() - t0 > WAIT_CYCLES) {
      *abort = 1;
      atomicExch(&g_gemm_error, kTimeout);
      return false;
    }
  }
  return true;
}

// One lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r));
  return r != 0;
}

template <int CG>
__device__ __forceinline__ void load_box(void* dst, const CUtensorMap* map, uint32_t bar, int x,
                                         int y, int z) {
  if (CG == 2)
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2"
        " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
}

template <int CG>
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                        uint32_t accumulate) {
  if (CG == 2)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}

// Arrives at `bar` (of both CTAs of a pair) when the MMAs issued so far are done.
template <int CG>
__device__ __forceinline__ void commit_to(uint64_t* bar) {
  if (CG == 2)
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64"
        " [%0], %1;" ::"r"(smem_u32(bar)),
        "h"((uint16_t)3)
        : "memory");
  else
    mma_commit(bar);
}

template <int CG>
__device__ __forceinline__ void alloc_tmem(uint32_t* dst, unsigned cols) {
  if (CG == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(dst)),
                 "r"(cols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  } else {
    tmem_alloc(dst, cols);
  }
}
template <int CG>
__device__ __forceinline__ void free_tmem(uint32_t addr, unsigned cols) {
  if (CG == 2)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols)
                 : "memory");
  else
    tmem_dealloc(addr, cols);
}

template <int ACT, bool FAST>
__device__ __forceinline__ void activate_all(float (&v)[32]) {
#pragma unroll
  for (int i = 0; i < 32; i += 2) {
    const Vec<2> r = act_value<ACT, FAST>(Vec<2>{{v[i], v[i + 1]}});
    v[i] = r.v[0];
    v[i + 1] = r.v[1];
  }
}
// silu (or sigmoid) of n float32 values of any size, one after the other, in the
// long form where a value needs it: not inlined, as a kernel of one or two tiles
// pays for every line of code once.
__device__ __noinline__ void sigmoid_far(float* v, int n, bool silu) {
#pragma unroll 1
  for (int i = 0; i < n; ++i) {
    const Vec<1> z = {{v[i]}};
    const float f = fabsf(v[i]) <= 6.f ? act_value<kActSigmoid, true>(z).v[0]
                                       : act_value<kActSigmoid, false>(z).v[0];
    v[i] = silu ? mul_rn(v[i], f) : f;
  }
}
// float32: up to |z| = 6 the relative error of the 16-bit results' form of silu
// and sigmoid is below 2^-20, a few ulp.  Pieces that go further are rare (7000 x
// 257 x 385 training: 101.9 us with that form everywhere, 107.2 with the long one
// inline, which is as much if no value needs it, 103.5 so).
template <int ACT>
__device__ __forceinline__ void activate_sigmoid(float (&v)[32]) {
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 32; ++i) m = fmaxf(m, fabsf(v[i]));
  if (m <= 6.f) {
    activate_all<ACT, true>(v);
  } else {
    float far[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) far[i] = v[i];
    sigmoid_far(far, 32, ACT == kActSilu);
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = far[i];
  }
}
template <bool FAST>
__device__ __forceinline__ void activate(float (&v)[32], int act) {
  switch (act) {
    case kActRelu: activate_all<kActRelu, FAST>(v); break;
    case kActGelu: activate_all<kActGelu, FAST>(v); break;
    case kActSilu:
      if (FAST) activate_all<kActSilu, true>(v);
      else activate_sigmoid<kActSilu>(v);
      break;
    case kActSigmoid:
      if (FAST) activate_all<kActSigmoid, true>(v);
      else activate_sigmoid<kActSigmoid>(v);
      break;
    default: break;
  }
}

// A warp's 32 x 32 piece (a row a thread) to row-major memory of any
// alignment: through shared memory, so that a store instruction writes 32
// neighbours.
template <typename U>
__device__ __forceinline__ void store_piece(float* stg, const float (&v)[32], U* out, int m0,
                                            int n0, int M, int N, int lane) {
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 32; ++i) stg[lane * 32 + (i ^ lane)] = v[i];
  __syncwarp();
  const int rows = min(32, M - m0);
  if (n0 + lane < N) {
    U* o = out + (size_t)m0 * N + n0 + lane;
#pragma unroll 8
    for (int r = 0; r < rows; ++r) o[(size_t)r * N] = from_f<U>(stg[r * 32 + (lane ^ r)]);
  }
}

// A thread's 32 values as 16-bit elements in the warp's 64-byte-swizzled box.
template <typename T>
__device__ __forceinline__ void stage_piece(uint8_t* box, const float (&v)[32], int lane) {
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    *reinterpret_cast<uint4*>(box + lane * 64 + ((c ^ ((lane >> 1) & 3)) << 4)) =
        pack16<T>(v + 8 * c);
  }
}
template <> __device__ __forceinline__ void stage_piece<float>(uint8_t*, const float (&)[32], int) {}

// Bias, activation, residual and the stores of a warp's 32 x 32 piece at
// (m0, n0); `bias` is that of column n0 + lane, bias_s the warp's room for 32,
// `ahead` the row's residual when it was fetched before (16-bit, aligned, a
// whole piece).
template <typename T>
__device__ __forceinline__ void finish_piece(float (&v)[32], int m0, int n0, const GemmArgs<T>& g,
                                             T bias, T* bias_s, const Raw<true, 32, T>& ahead,
                                             uint8_t* stg, const CUtensorMap* mapY,
                                             const CUtensorMap* mapZ, int lane, int split) {
  if (m0 >= g.M || n0 >= g.N) return;
  if (g.partial) {
    store_piece<float>(reinterpret_cast<float*>(stg), v, g.partial + (size_t)split * g.M * g.N, m0,
                       n0, g.M, g.N, lane);
    return;
  }
  constexpr bool FAST = sizeof(T) == 2;
  if (g.bias) {
    constexpr int PER = 16 / sizeof(T);
    __syncwarp();
    bias_s[lane] = bias;
    __syncwarp();
#pragma unroll
    for (int c = 0; c < 32 / PER; ++c) {
      float q[PER];
      unpack16<T>(reinterpret_cast<const uint4*>(bias_s)[c], q);
#pragma unroll
      for (int i = 0; i < PER; ++i) v[c * PER + i] = add_rn(v[c * PER + i], q[i]);
    }
  }
  if (g.tma_store) {
    if (lane == 0) bulk_wait_read<0>();  // the boxes of the last piece are free
    __syncwarp();
    if (g.z) stage_piece<T>(stg + 2048, v, lane);
  } else if (g.z) {
    store_piece<T>(reinterpret_cast<float*>(stg), v, g.z, m0, n0, g.M, g.N, lane);
  }
  activate<FAST>(v, g.act);
  if (g.res) {
    if (g.res_vec && n0 + 32 <= g.N) {
      if (m0 + lane < g.M) {
        constexpr int PER = 16 / sizeof(T);
        Raw<true, 32, T> here;
        if (sizeof(T) == 4) here.load(g.res + (size_t)(m0 + lane) * g.ldr + n0);
#pragma unroll
        for (int c = 0; c < 32 / PER; ++c) {
          float q[PER];
          unpack16<T>(sizeof(T) == 4 ? here.w[c] : ahead.w[c], q);
#pragma unroll
          for (int i = 0; i < PER; ++i) v[c * PER + i] = add_rn(v[c * PER + i], q[i]);
        }
      }
    } else if (m0 + lane < g.M) {
      const T* r = g.res + (size_t)(m0 + lane) * g.ldr + n0;
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (n0 + i < g.N) v[i] = add_rn(v[i], to_f(r[i]));
    }
  }
  if (g.tma_store) {
    stage_piece<T>(stg, v, lane);
    fence_async_smem();
    __syncwarp();
    if (lane == 0) {
      tma_store_3d(mapY, stg, n0, m0, 0);
      if (g.z) tma_store_3d(mapZ, stg + 2048, n0, m0, 0);
      bulk_commit();
    }
  } else {
    store_piece<T>(reinterpret_cast<float*>(stg), v, g.out, m0, n0, g.M, g.N, lane);
  }
}

template <typename T, int CG, int TN, bool A_MN, bool B_MN>
__global__ void __launch_bounds__(Geom<T, CG, TN>::THREADS, 1)
    gemm_kernel(const __grid_constant__ CUtensorMap mapA, const __grid_constant__ CUtensorMap mapB,
                const __grid_constant__ CUtensorMap mapY, const __grid_constant__ CUtensorMap mapZ,
                const GemmArgs<T> g) {
  using G = Geom<T, CG, TN>;
  constexpr int PL = G::PL, STAGES = G::STAGES, NP = G::CHUNKS32, EW = G::EW;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* stg_base = smem + STAGES * G::STAGE;
  GemmShared& sh = *reinterpret_cast<GemmShared*>(stg_base + EW * Elem<T>::STG);
  volatile int* abort = &sh.abort;
  const int tid = threadIdx.x, lane = tid & 31;
  // the same in all lanes, and known to be: a role's loop runs on uniform registers
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const int rank = CG == 2 ? (int)cta_rank() : 0;
  const int unit = blockIdx.x / CG, units = gridDim.x / CG;

  if (tid == 0) {
    sh.abort = 0;
    if ((smem_u32(smem) & 1023u) != 0) {
      atomicExch(&g_gemm_error, kLaunch);
      sh.abort = 1;
    }
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&sh.full[s], 1);
      mbar_init(&sh.empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&sh.accf[a], 1);
      mbar_init(&sh.acce[a], EW * CG);
    }
    mbar_init(&sh.mma_done, 1);
    fence_barrier_init();
  }
  if (warp == EW + 1) alloc_tmem<CG>(&sh.tmem_base, 2 * G::ACC);
  tc_fence_before();
  __syncthreads();
  if (CG == 2) cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem = sh.tmem_base;
  after_previous();  // all above overlaps its end
  let_next_start();
  // the alignment of shared memory is the same in every CTA, so a pair
  // leaves together
  const bool dead = *abort != 0;

  if (!dead && warp == EW) {
    // ---------------------------------------------------- TMA producer
    if (lane == 0) {
      int it = 0, s = 0;
      uint32_t ph = 1;
      bool ok = true;
      for (int w = unit; ok && w < g.items; w += units) {
        const TileAt t = tile_at(w, g);
        const int m0 = t.m * 128 * CG + rank * 128;
        const int n0 = t.n * TN + rank * G::B_ROWS;
        const int k1 = min(g.nK, (t.split + 1) * g.per_split);
        for (int kc = t.split * g.per_split; kc < k1; ++kc, ++it) {
          if (!wait_for(&sh.empty[s], ph, abort)) {
            ok = false;
            break;
          }
          uint8_t* pa = smem + s * G::STAGE;
          uint8_t* pb = pa + PL * A_PLANE;
          // in a pair the first CTA's barrier counts the bytes of both
          if (rank == 0) mbar_arrive_expect_tx(&sh.full[s], CG * G::STAGE);
          const uint32_t bar = CG == 2 ? peer_addr(&sh.full[s], 0) : smem_u32(&sh.full[s]);
          if (!A_MN) {
            load_box<CG>(pa, &mapA, bar, kc * BK, m0, 0);
          } else {
#pragma unroll
            for (int p = 0; p < PL; ++p)
#pragma unroll
              for (int j = 0; j < 2; ++j)
                load_box<CG>(pa + p * A_PLANE + j * 8192, &mapA, bar, m0 + 64 * j, kc * BK, p);
          }
          if (!B_MN) {
            load_box<CG>(pb, &mapB, bar, kc * BK, n0, 0);
          } else {
#pragma unroll
            for (int p = 0; p < PL; ++p)
#pragma unroll
              for (int j = 0; j < G::B_ROWS / 64; ++j)
                load_box<CG>(pb + p * G::B_PLANE + j * 8192, &mapB, bar, n0 + 64 * j, kc * BK, p);
          }
          if (++s == STAGES) {
            s = 0;
            ph ^= 1;
          }
        }
      }
      if (*abort && rank == 0) {  // copies in flight land before shared memory is given up
        for (int i = it > STAGES ? it - STAGES : 0; i < it; ++i)
          wait_plain(&sh.full[i % STAGES], (unsigned)(i / STAGES) & 1u);
      }
    }
    __syncwarp();
  } else if (!dead && warp == EW + 1) {
    // ------------------------------------------------------ MMA issuer
    // The whole warp walks the loop, so that descriptors stay in uniform
    // registers, where tcgen05.mma takes them, and one lane issues: moving
    // them there for every product from one lane's registers cost 10% of the
    // rate (8192^3: 823 against 720 us).
    if (rank == 0) {
      constexpr uint32_t IDESC = (1u << 4) | (Elem<T>::FMT << 7) | (Elem<T>::FMT << 10) |
                                 ((uint32_t)A_MN << 15) | ((uint32_t)B_MN << 16) |
                                 ((uint32_t)(TN >> 3) << 17) |
                                 ((uint32_t)((128 * CG) >> 4) << 24);
      // a step of 16 contraction values: 32 bytes along a K-major line, 16
      // lines of an MN-major box
      constexpr uint32_t STEP_A = (A_MN ? 2048 : 32) >> 4, STEP_B = (B_MN ? 2048 : 32) >> 4;
      constexpr uint32_t LBO = 8192;  // between 64-wide boxes of an MN-major operand
      const uint64_t a0 = smem_desc_sw128(smem_u32(smem), LBO, 1024);
      const uint64_t b0 = smem_desc_sw128(smem_u32(smem) + PL * A_PLANE, LBO, 1024);
      const bool leader = elect_one();
      int s = 0, si = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int w = unit; ok && w < g.items; w += units) {
        const int split = w % g.splits;
        const int k0 = split * g.per_split, k1 = min(g.nK, k0 + g.per_split);
        for (int kc = k0; ok && kc < k1;) {
          const int seg_end = PL == 3 ? min(k1, kc + G::SEG_CHUNKS) : k1;
          const int a = si & 1;
          ok = __all_sync(0xffffffffu,
                          wait_for(&sh.acce[a], ((unsigned)(si >> 1) & 1u) ^ 1u, abort));
          if (!ok) break;
          tc_fence_after();
          const uint32_t d = tmem + (uint32_t)(a * G::ACC);
          uint32_t more = 0;
          for (; kc < seg_end; ++kc) {
            ok = __all_sync(0xffffffffu, wait_for(&sh.full[s], ph, abort));
            if (!ok) break;
            tc_fence_after();
            const uint64_t da = a0 + (uint64_t)(s * (G::STAGE >> 4));
            const uint64_t db = b0 + (uint64_t)(s * (G::STAGE >> 4));
            if (leader) {
#pragma unroll
              for (int kk = 0; kk < BK / 16; ++kk) {
                const uint64_t ka = da + kk * STEP_A, kb = db + kk * STEP_B;
                const uint32_t acc = kk > 0 ? 1u : more;
                mma_f16<CG>(d, ka, kb, IDESC, acc);
                if (PL == 3) {
                  constexpr uint32_t PA = A_PLANE >> 4, PB = G::B_PLANE >> 4;
                  mma_f16<CG>(d + TN, ka, kb + 2 * PB, IDESC, acc);
                  mma_f16<CG>(d + TN, ka + 2 * PA, kb, IDESC, 1);
                  mma_f16<CG>(d + TN, ka + PA, kb + PB, IDESC, 1);
                  mma_f16<CG>(d + TN, ka, kb + PB, IDESC, 1);
                  mma_f16<CG>(d + TN, ka + PA, kb, IDESC, 1);
                }
              }
              commit_to<CG>(&sh.empty[s]);
            }
            __syncwarp();
            more = 1;
            if (++s == STAGES) {
              s = 0;
              ph ^= 1;
            }
          }
          if (!ok) break;
          if (leader) commit_to<CG>(&sh.accf[a]);
          __syncwarp();
          ++si;
        }
      }
      // every MMA issued has finished before TMEM is released
      if (leader) {
        if (CG == 2)
          asm volatile(
              "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                  smem_u32(&sh.mma_done))
              : "memory");
        else
          mma_commit(&sh.mma_done);
      }
      wait_plain(&sh.mma_done, 0);
    }
    __syncwarp();
  } else if (!dead) {
    // -------------------------------------------------------- epilogue
    const int quad = warp & 3, share = warp >> 2;
    uint8_t* stg = stg_base + warp * Elem<T>::STG;
    T* bias_s = reinterpret_cast<T*>(sh.bias) + 32 * warp;
    const uint32_t lanes = tmem + ((uint32_t)(32 * quad) << 16);
    int si = 0;
    bool ok = true;
    for (int w = unit; ok && w < g.items; w += units) {
      const TileAt t = tile_at(w, g);
      const int split = t.split;
      const int m0 = t.m * 128 * CG + rank * 128 + 32 * quad;
      const int n0 = t.n * TN + share * G::COLS;
      // what the epilogue adds is fetched while the products run
      T bias[NP];
#pragma unroll
      for (int c = 0; c < NP; ++c) {
        const int n = n0 + 32 * c + lane;
        bias[c] = g.bias && n < g.N ? g.bias[n] : from_f<T>(0.f);
        if (g.res && m0 + lane < g.M && n0 + 32 * c < g.N)
          asm volatile("prefetch.global.L2 [%0];" ::"l"(g.res + (size_t)(m0 + lane) * g.ldr + n0 +
                                                        32 * c));
      }
      Raw<true, 32, T> ahead;
      auto fetch_residual = [&](int c) {
        if (sizeof(T) == 2 && g.res_vec && m0 + lane < g.M && n0 + 32 * c + 32 <= g.N)
          ahead.load(g.res + (size_t)(m0 + lane) * g.ldr + n0 + 32 * c);
      };
      fetch_residual(0);
      if (PL == 1) {
        const int a = si & 1;
        if (!wait_for(&sh.accf[a], (unsigned)(si >> 1) & 1u, abort)) {
          break;
        }
        ++si;
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < NP; ++c) {
          float v[32];
          tmem_ld32(lanes + (uint32_t)(a * G::ACC + share * G::COLS + 32 * c), v);
          if (c == NP - 1) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
              if (CG == 2) arrive_at(peer_addr(&sh.acce[a], 0));
              else mbar_arrive(&sh.acce[a]);
            }
          }
          finish_piece<T>(v, m0, n0 + 32 * c, g, bias[c], bias_s, ahead, stg, &mapY, &mapZ, lane,
                          split);
          if (c + 1 < NP) fetch_residual(c + 1);
        }
      } else {
        const int k0 = split * g.per_split, k1 = min(g.nK, k0 + g.per_split);
        float acc[NP][32];
#pragma unroll
        for (int c = 0; c < NP; ++c)
#pragma unroll
          for (int i = 0; i < 32; ++i) acc[c][i] = 0.f;
        for (int kc = k0; kc < k1; kc += G::SEG_CHUNKS, ++si) {
          const int a = si & 1;
          if (!wait_for(&sh.accf[a], (unsigned)(si >> 1) & 1u, abort)) {
            ok = false;
            break;
          }
          tc_fence_after();
#pragma unroll
          for (int c = 0; c < NP; ++c) {
            float big[32], small[32];
            const uint32_t col = lanes + (uint32_t)(a * G::ACC + share * G::COLS + 32 * c);
            tmem_ld32(col, big);
            tmem_ld32(col + TN, small);
            // in pairs; the values' sum tells, for one addition a pair, whether
            // any of them is not finite
            Vec<2> all[2] = {splat<2>(0.f), splat<2>(0.f)};
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              const Vec<2> t = add_v(Vec<2>{{big[i], big[i + 1]}}, Vec<2>{{small[i], small[i + 1]}});
              small[i] = t.v[0];
              small[i + 1] = t.v[1];
              all[i / 2 & 1] = add_v(all[i / 2 & 1], t);
            }
            all[0] = add_v(all[0], all[1]);
            if (!(fabsf(all[0].v[0] + all[0].v[1]) < INFINITY))
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (!(fabsf(big[i]) < INFINITY)) small[i] = big[i];
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              const Vec<2> s = add_v(Vec<2>{{acc[c][i], acc[c][i + 1]}},
                                     Vec<2>{{small[i], small[i + 1]}});
              acc[c][i] = s.v[0];
              acc[c][i + 1] = s.v[1];
            }
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if (CG == 2) arrive_at(peer_addr(&sh.acce[a], 0));
            else mbar_arrive(&sh.acce[a]);
          }
        }
        if (!ok) break;
#pragma unroll
        for (int c = 0; c < NP; ++c)
          finish_piece<T>(acc[c], m0, n0 + 32 * c, g, bias[c], bias_s, ahead, stg, &mapY, &mapZ,
                          lane, split);
      }
    }
    if (lane == 0) bulk_wait_all();
    __syncwarp();
  }

  tc_fence_before();
  __syncthreads();
  if (CG == 2) cluster_sync_all();
  tc_fence_after();
  if (warp == EW + 1) free_tmem<CG>(tmem, 2 * G::ACC);
  if (CG == 2) cluster_sync_all();
}

// Sums the splits' partial products in their order and finishes the result.
template <typename T>
__global__ void __launch_bounds__(256)
    gemm_join_kernel(const float* __restrict__ partial, int splits, const GemmArgs<T> g) {
  const size_t n = (size_t)g.M * g.N;
  constexpr bool FAST = sizeof(T) == 2;
  after_previous();
  let_next_start();
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) {
    float v = 0.f;
    for (int s = 0; s < splits; ++s) v += __ldcs(partial + s * n + i);
    const size_t m = i / g.N, c = i - m * g.N;
    if (g.bias) v = add_rn(v, to_f(g.bias[c]));
    if (g.z) g.z[i] = from_f<T>(v);
    v = activate1<FAST>(v, g.act);
    if (g.res) v = add_rn(v, to_f(g.res[m * g.ldr + c]));
    g.out[i] = from_f<T>(v);
  }
}

// ------------------------------------------------------------------ host

template <typename T> struct MapType {
  static constexpr CUtensorMapDataType value = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
};
template <> struct MapType<__half> {
  static constexpr CUtensorMapDataType value = CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
};

template <typename T>
int operand_map(CUtensorMap* map, const GemmOperand& o, int tile_rows) {
  const int planes = Elem<T>::PL;
  const uint32_t box[3] = {BK, o.k_major ? (uint32_t)tile_rows : BK,
                           o.k_major ? (uint32_t)planes : 1};
  const uint64_t dims[3] = {(uint64_t)o.cols, (uint64_t)o.rows, (uint64_t)planes};
  const uint64_t row = o.ld * 2;
  const uint64_t strides[2] = {row, planes > 1 ? o.plane * 2 : row};
  return make_map_3d(map, MapType<T>::value, o.base, dims, strides, box,
                     CU_TENSOR_MAP_SWIZZLE_128B);
}

template <typename T>
int output_map(CUtensorMap* map, void* base, int M, int N) {
  const uint32_t box[3] = {32, 32, 1};
  const uint64_t dims[3] = {(uint64_t)N, (uint64_t)M, 1};
  const uint64_t strides[2] = {(uint64_t)N * 2, (uint64_t)N * 2};
  return make_map_3d(map, MapType<T>::value, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_64B);
}

template <typename T, int CG, int TN, bool A_MN, bool B_MN>
int gemm_launch(const GemmProblem& p, const GemmPlan& plan, cudaStream_t st) {
  using G = Geom<T, CG, TN>;
  auto kernel = gemm_kernel<T, CG, TN, A_MN, B_MN>;
  static_assert(G::STAGES >= 2 && G::SMEM <= SMEM_MAX, "shared memory");
  CUtensorMap mapA, mapB, mapY = {}, mapZ = {};
  if (int e = operand_map<T>(&mapA, p.a, 128)) return e;
  if (int e = operand_map<T>(&mapB, p.b, G::B_ROWS)) return e;
  GemmArgs<T> g;
  g.M = p.M;
  g.N = p.N;
  g.K = p.K;
  g.nK = (p.K + BK - 1) / BK;
  g.tiles_m = (p.M + 128 * CG - 1) / (128 * CG);
  g.tiles_n = (p.N + TN - 1) / TN;
  g.per_split = (g.nK + plan.splits - 1) / plan.splits;
  g.splits = (g.nK + g.per_split - 1) / g.per_split;
  const long long items = (long long)g.tiles_m * g.tiles_n * g.splits;
  if (items > 0x7fffffff / 2) return set_error(kUnsupported, "tw_linear: too many tiles");
  g.items = (int)items;
  g.bias = (const T*)p.bias;
  g.res = (const T*)p.residual;
  g.ldr = p.ldr;
  g.out = (T*)p.out;
  g.z = (T*)p.z;
  g.act = p.act;
  g.partial = plan.splits > 1 ? p.partial : nullptr;
  g.res_vec = p.residual && (uintptr_t)p.residual % 16 == 0 && p.ldr * sizeof(T) % 16 == 0;
  g.tma_store = sizeof(T) == 2 && !g.partial && p.N % 8 == 0 && (uintptr_t)p.out % 16 == 0 &&
                (uintptr_t)p.z % 16 == 0;
  if (g.tma_store) {
    if (int e = output_map<T>(&mapY, p.out, p.M, p.N)) return e;
    if (p.z)
      if (int e = output_map<T>(&mapZ, p.z, p.M, p.N)) return e;
  }
  cudaError_t err =
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, G::SMEM);
  if (err != cudaSuccess) return set_error(kLaunch, "tw_linear: %s", cudaGetErrorString(err));
  const int most = 148 / CG;
  const unsigned grid = (unsigned)(CG * (g.items < most ? g.items : most));
  err = launch_after(p.after, kernel, dim3(grid), dim3(G::THREADS), G::SMEM, CG, st, mapA, mapB,
                     mapY, mapZ, g);
  if (err == cudaSuccess && g.partial) {
    const size_t n = (size_t)p.M * p.N, blocks = (n + 255) / 256;
    err = launch_after(true, gemm_join_kernel<T>,
                       dim3((unsigned)(blocks < 148 * 8 ? blocks : 148 * 8)), dim3(256), 0, 1, st,
                       (const float*)p.partial, g.splits, g);
  }
  if (err != cudaSuccess) return set_error(kLaunch, "tw_linear: %s", cudaGetErrorString(err));
  return kOk;
}

template <typename T, bool A_MN, bool B_MN>
int gemm_majors(const GemmProblem& p, cudaStream_t st) {
  const GemmPlan plan = gemm_plan(p.M, p.N, p.K, Elem<T>::PL);
  if constexpr (Elem<T>::PL == 1) {
    if (plan.cg == 2) return gemm_launch<T, 2, 256, A_MN, B_MN>(p, plan, st);
  }
  return plan.tn == 128 ? gemm_launch<T, 1, 128, A_MN, B_MN>(p, plan, st)
                        : gemm_launch<T, 1, 64, A_MN, B_MN>(p, plan, st);
}

}  // namespace

template <typename T>
int gemm_run(const GemmProblem& p, cudaStream_t st) {
  // the three products of a linear layer: x w^T, dz w, dz^T x
  if (p.a.k_major) return p.b.k_major ? gemm_majors<T, false, false>(p, st)
                                      : gemm_majors<T, false, true>(p, st);
  return gemm_majors<T, true, true>(p, st);
}

template <typename T>
int gemm_take_device_error() {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_gemm_error, sizeof(int)) != cudaSuccess) return kLaunch;
  if (v != 0) {
    const int zero = 0;
    cudaMemcpyToSymbol(g_gemm_error, &zero, sizeof(int));
  }
  return v;
}

}  // namespace tw
