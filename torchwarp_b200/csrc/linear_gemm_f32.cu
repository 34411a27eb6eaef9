// The linear operator's tensor-core product for float results.
#include "linear_gemm.cuh"

namespace tw {
template int gemm_run<float>(const GemmProblem&, cudaStream_t);
template int gemm_take_device_error<float>();
}  // namespace tw
