// Host-side interface of the norms with the residual they belong to
// (residual_norm.cu, residual_norm_kernels.cuh).
//
//   add_norm   s = alpha r + gate * D(h),  y = norm(s)
//   norm_add   s = alpha r + gate * D(norm(h))
//   norm(x) = (x - mean) rstd w + b; kind rms: mean is 0
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "dropout.h"

namespace resnorm {

using drop::DType;

struct Args {
  DType dtype;               // of h, r, y, s and the gradients of rows
  bool weight_f32, gate_f32;  // w, b, dw, db; gate, dgate: float32, or dtype
  bool branch;               // norm_add
  bool rms;
  bool keep;                 // add_norm forward: s is for the backward alone (kept_normal)
  int64_t rows, cols;
  int64_t h_stride, r_stride, gate_stride, gy_stride, gs_stride, sum_stride;
  int64_t gate_groups;       // rows of the gate
  int64_t gate_rows;         // neighbouring rows that share one: rows / gate_groups
  float alpha, eps;
  float share;               // 1 / cols
  drop::Rule rule;
  const void* h;             // forward; backward: norm_add, and with dgate
  const void* r;             // forward
  const void* gate;          // may be null: ones
  const void* w;             // may be null: ones
  const void* b;             // may be null: zeros
  void* y;                   // add_norm forward, contiguous
  void* s;                   // forward, contiguous; add_norm: may be null
  float* mean;               // [rows]; forward: written where not null; backward: read (null with rms);
                             // add_norm: of s as it is stored; rstd below 0: s is normalised (kept_normal)
  float* rstd;
  const void* gy;            // backward, add_norm: may be null
  const void* gs;            // backward; add_norm: may be null
  const void* sum;           // backward, add_norm: s of the forward
  void* dh;                  // contiguous, may be null
  void* dr;                  // contiguous, may be null
  void* dw;                  // may be null
  void* db;                  // may be null
  void* dgate;               // [gate_groups, cols] contiguous, may be null
  float* parts;              // backward: backward_parts(a) floats
};

// Floats of `parts` that the backward needs.
int64_t backward_parts(const Args& a);
cudaError_t forward(const Args& a, cudaStream_t stream);
cudaError_t backward(const Args& a, cudaStream_t stream);

// Of one storage type (residual_norm_<type>.cu).
struct Grid {
  int blocks = 0;
  int64_t units = 0, unit_rows = 0, group_units = 0, group_rows = 0;
  bool sums_gate = false;  // the gate's gradient is a sum over rows
};
Grid backward_grid(const Args& a);
cudaError_t forward_f32(const Args& a, cudaStream_t stream);
cudaError_t forward_bf16(const Args& a, cudaStream_t stream);
cudaError_t forward_f16(const Args& a, cudaStream_t stream);
cudaError_t backward_f32(const Args& a, const Grid& grid, cudaStream_t stream);
cudaError_t backward_bf16(const Args& a, const Grid& grid, cudaStream_t stream);
cudaError_t backward_f16(const Args& a, const Grid& grid, cudaStream_t stream);

}  // namespace resnorm
