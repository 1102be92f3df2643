// The row kernels for rows of nv_bfloat16.
#include "w8a8_rows.cuh"

namespace glowq {

cudaError_t launch_rows_bf16(const RowsParams& params, int norm, int sms, cudaStream_t stream) {
  return launch_rows_typed<__nv_bfloat16>(params, norm, sms, stream);
}
cudaError_t launch_norm_grad_bf16(const GradParams& params, cudaStream_t stream) {
  return launch_grad_typed<__nv_bfloat16>(params, stream);
}

}  // namespace glowq
