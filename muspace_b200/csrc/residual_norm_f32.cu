// The norms with their residual, rows of f32.
#include "residual_norm_kernels.cuh"

namespace resnorm {

cudaError_t forward_f32(const Args& a, cudaStream_t stream) { return forward_of<float>(a, stream); }

cudaError_t backward_f32(const Args& a, const Grid& grid, cudaStream_t stream) {
  return backward_of<float>(a, grid, stream);
}

}  // namespace resnorm
