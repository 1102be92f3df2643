// The row kernels for rows of half.
#include "w8a8_rows.cuh"

namespace glowq {

cudaError_t launch_rows_f16(const RowsParams& params, int norm, int sms, cudaStream_t stream) {
  return launch_rows_typed<__half>(params, norm, sms, stream);
}
cudaError_t launch_norm_grad_f16(const GradParams& params, cudaStream_t stream) {
  return launch_grad_typed<__half>(params, stream);
}

}  // namespace glowq
