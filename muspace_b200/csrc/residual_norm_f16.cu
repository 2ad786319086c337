// The norms with their residual, rows of f16.
#include "residual_norm_kernels.cuh"

namespace resnorm {

cudaError_t forward_f16(const Args& a, cudaStream_t stream) { return forward_of<__half>(a, stream); }

cudaError_t backward_f16(const Args& a, const Grid& grid, cudaStream_t stream) {
  return backward_of<__half>(a, grid, stream);
}

}  // namespace resnorm
