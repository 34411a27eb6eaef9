// Host interface of the tensor-core product behind the linear operator.
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace tw {

// A matrix [rows][cols] in memory (cols contiguous, `ld` elements a row), of
// 16-bit elements, or of `planes` = 3 bfloat16 planes `plane` elements apart
// whose sum is a float32 matrix.  k_major: its columns are the contraction;
// else its rows are.
struct GemmOperand {
  const void* base;
  size_t ld, plane;
  int rows, cols;
  bool k_major;
};

// out[m, n] = act(sum_k A(m, k) B(n, k) + bias[n]) + residual[m, n], z[m, n]
// the argument of act.  out and z are dense.  partial: float32 scratch of
// splits * M * N when the plan has more than one split.
struct GemmProblem {
  GemmOperand a, b;
  int M, N, K;
  const void* bias;
  const void* residual;
  size_t ldr;
  int act;
  void* out;
  void* z;
  float* partial;
  bool after;  // the kernel before this one on the stream is the operator's own
};

// How a product is cut: CTAs per tile (1, or a pair), tile width, and parts
// of the contraction that are summed by a second kernel.
struct GemmPlan {
  int cg, tn, splits;
};

GemmPlan gemm_plan(int M, int N, int K, int planes);

template <typename T>
int gemm_run(const GemmProblem& p, cudaStream_t st);

// The error word of this type's kernels (a bounded wait ran out), cleared.
template <typename T>
int gemm_take_device_error();

}  // namespace tw
