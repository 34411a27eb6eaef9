// The linear operator's tensor-core product for __half results.
#include "linear_gemm.cuh"

namespace tw {
template int gemm_run<__half>(const GemmProblem&, cudaStream_t);
template int gemm_take_device_error<__half>();
}  // namespace tw
