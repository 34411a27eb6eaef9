// The linear operator's tensor-core product for __nv_bfloat16 results.
#include "linear_gemm.cuh"

namespace tw {
template int gemm_run<__nv_bfloat16>(const GemmProblem&, cudaStream_t);
template int gemm_take_device_error<__nv_bfloat16>();
}  // namespace tw
