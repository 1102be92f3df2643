// Launch functions of the 8-bit path, shared by its translation units.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/glowq_w8a8.h"

namespace glowq {

// abi.cu
int tensor_map_2d_ex(CUtensorMap* out, CUtensorMapDataType dtype, const void* ptr, uint64_t dim0, uint64_t dim1,
                     uint64_t stride_bytes, uint32_t box0, uint32_t box1, int swizzle);
int current_device_sms(int* sms);          // GLOWQ_* status: the current device is one that the library runs on
int note_cuda_error(cudaError_t e);        // GLOWQ_OK, or GLOWQ_ERR_CUDA with the error kept for glowq_w4a16_last_cuda_error
bool use_pdl();

// w8a8_rows.cu
cudaError_t launch_rows(const glowq_w8a8_rows_t& p, int sms, cudaStream_t stream);
// An empty kernel in stream order: what is launched behind it begins when all in front of it is complete and visible, even a kernel that
// reads before its dependency wait.
cudaError_t launch_settle(cudaStream_t stream);
// Below, ahead: the launch may begin, and read its constant operands, while the one in front of it still runs.
// codes, scales and r of a few tokens in one launch
bool few_tokens(const glowq_w8a8_linear_t& g);
cudaError_t launch_few_tokens(const glowq_w8a8_linear_t& g, bool ahead, cudaStream_t stream);
cudaError_t launch_layer_norm_grad(const glowq_layer_norm_grad_t& g, cudaStream_t stream);
size_t layer_norm_grad_bytes(int M, int K);

// w8a8_stream.cu
int w8a8_stream_split(long long tiles, int steps, int sms);   // CTAs of a cluster
int w8a8_stream_forward(const glowq_w8a8_linear_t& g, bool ahead, int sms, cudaStream_t stream);
// beside: the launch in front makes the codes of the same x, and began after all that came before it was complete
int w8a8_right_factor(const glowq_w8a8_linear_t& g, bool beside, bool ahead, int sms, cudaStream_t stream);
cudaError_t w8a8_stream_status(uint32_t* out, cudaStream_t stream);

// w8a8_pair.cu: tiles of 256 tokens x n channels (64, 128, 192 or 256)
int w8a8_pair_forward(const glowq_w8a8_linear_t& g, int n, bool ahead, int sms, cudaStream_t stream);
cudaError_t w8a8_pair_status(uint32_t* out, cudaStream_t stream);

// Reads a file's status word and clears it.
template <typename Symbol> cudaError_t take_status(Symbol& word, uint32_t* out, cudaStream_t stream) {
  cudaError_t e = cudaMemcpyFromSymbolAsync(out, word, sizeof(uint32_t), 0, cudaMemcpyDeviceToHost, stream);
  if (e == cudaSuccess) e = cudaStreamSynchronize(stream);
  if (e != cudaSuccess || *out == 0) return e;
  static const uint32_t zero = 0;
  return cudaMemcpyToSymbolAsync(word, &zero, sizeof(zero), 0, cudaMemcpyHostToDevice, stream);
}

inline size_t dtype_bytes(int dtype) { return dtype == GLOWQ_F32 ? 4 : 2; }

}  // namespace glowq
