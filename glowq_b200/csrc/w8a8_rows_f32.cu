// The row kernels for rows of float.
#include "w8a8_rows.cuh"

namespace glowq {

cudaError_t launch_rows_f32(const RowsParams& params, int norm, int sms, cudaStream_t stream) {
  return launch_rows_typed<float>(params, norm, sms, stream);
}
cudaError_t launch_norm_grad_f32(const GradParams& params, cudaStream_t stream) {
  return launch_grad_typed<float>(params, stream);
}

}  // namespace glowq
