// The norms with their residual, rows of bf16.
#include "residual_norm_kernels.cuh"

namespace resnorm {

cudaError_t forward_bf16(const Args& a, cudaStream_t stream) { return forward_of<lin::bf16>(a, stream); }

cudaError_t backward_bf16(const Args& a, const Grid& grid, cudaStream_t stream) {
  return backward_of<lin::bf16>(a, grid, stream);
}

}  // namespace resnorm
