// Host-side interface of dropout (dropout.cu), and the rule that the kernels with
// dropout inside them (residual_norm, gated_linear) share with it.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace drop {

enum class DType : int { kF32 = 0, kBF16 = 1, kF16 = 2 };

// Drops an element with probability threshold / 65536; what is kept is multiplied by
// scale. A threshold of 0 is no dropout.
struct Rule {
  uint32_t threshold = 0;
  float scale = 1.f;
  uint64_t seed = 0, sequence = 0;
  const int64_t* seed_at = nullptr;  // on the device: takes the place of seed
};

inline float scale_of(uint32_t threshold) {
  return threshold >= 65536 ? 0.f : static_cast<float>(65536.0 / (65536.0 - threshold));
}

// y = D(x); y is contiguous, rows of x are x_stride elements apart.
cudaError_t dropout(DType dtype, const void* x, int64_t x_stride, int64_t rows, int64_t cols, const Rule& rule, void* y,
                    cudaStream_t stream);

}  // namespace drop
