// Host-side interface of layer norm (layer_norm.cu) and of 8-bit activation
// checkpoints (checkpoint8.cu).
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace lnorm {

enum class DType : int { kF32 = 0, kBF16 = 1 };

struct Args {
  DType dtype, weight_dtype;  // of x, y, g, dx; of w, b, dw, db (dtype or kF32)
  int64_t rows, cols;
  int64_t x_stride, g_stride;  // y and dx are contiguous
  float eps;
  const void* x;   // forward; backward without codes
  const void* w;   // may be null: ones
  const void* b;   // may be null: zeros
  void* y;         // forward
  float* mean;     // [rows]; forward: written where not null; backward without codes: read
  float* rstd;     // [rows]
  int8_t* codes;   // forward: the 8-bit checkpoint of x, written where not null
  uint8_t* exps;
  const void* g;   // backward
  const int8_t* codes_in;  // backward from the checkpoint: statistics are taken from it again
  const uint8_t* exps_in;
  void* dx;        // may be null
  void* dw;        // may be null
  void* db;        // may be null
  float* parts;    // backward with dw or db: backward_parts(rows, cols) * 2 * cols floats
};

int backward_parts(int64_t rows, int64_t cols);
cudaError_t forward(const Args& a, cudaStream_t stream);
cudaError_t backward(const Args& a, cudaStream_t stream);
cudaError_t wait_timeouts(unsigned int* count);
// A kernel with one wait that runs out after `clocks`, and no copies: what wait_timeouts counts, on purpose.
cudaError_t wait_probe(int64_t clocks, cudaStream_t stream);

}  // namespace lnorm

namespace ckpt {

cudaError_t pack(bool bf16, const void* x, int64_t x_stride, int64_t rows, int64_t cols, int8_t* codes, uint8_t* exps,
                 cudaStream_t stream);
cudaError_t unpack(bool bf16, const int8_t* codes, const uint8_t* exps, int64_t rows, int64_t cols, void* x,
                   cudaStream_t stream);

}  // namespace ckpt
