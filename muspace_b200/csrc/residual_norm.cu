// The norms with their residual: which blocks take which rows, and the second kernel
// of the backward pass, which adds the blocks' sums in order.
#include "residual_norm.h"

#include <algorithm>

#include "linear_device.cuh"

namespace resnorm {
namespace {

using lin::from_float;

// dw, db and dgate from the blocks' parts: a block takes 32 columns of one of them,
// warps take parts in turn. blockIdx.y: dw, db, then the gate's rows.
template <typename W, typename D>
__global__ void __launch_bounds__(1024) join_kernel(const Args a, const Grid grid) {
  __shared__ float buf[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c = blockIdx.x * 32ll + lane;
  const int64_t groups = grid.sums_gate ? a.gate_groups : 0;
  for (int64_t which = blockIdx.y; which < 2 + groups; which += gridDim.y) {
    if ((which == 0 && !a.dw) || (which == 1 && !a.db)) continue;
    const float* parts = a.parts + which * a.cols;  // dw's and db's lie in turn
    int64_t count = grid.blocks, ld = 2 * a.cols;
    if (which >= 2) {
      count = grid.group_units, ld = a.cols;
      parts = a.parts + (2ll * grid.blocks + (which - 2) * grid.group_units) * a.cols;
    }
    float s = 0.f;
    if (c < a.cols) {
#pragma unroll 4
      for (int64_t i = warp; i < count; i += 32) s += parts[i * ld + c];
    }
    __syncthreads();
    buf[warp][lane] = s;
    __syncthreads();
    if (warp != 0 || c >= a.cols) continue;
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) s += buf[i][lane];
    if (which == 0)
      static_cast<W*>(a.dw)[c] = from_float<W>(s);
    else if (which == 1)
      static_cast<W*>(a.db)[c] = from_float<W>(s);
    else
      static_cast<D*>(a.dgate)[(which - 2) * a.cols + c] = from_float<D>(s);
  }
}

template <typename T>
cudaError_t join(const Args& a, const Grid& grid, cudaStream_t stream) {
  const int64_t groups = grid.sums_gate ? a.gate_groups : 0;
  const dim3 blocks(static_cast<unsigned>((a.cols + 31) / 32),
                    static_cast<unsigned>(std::min<int64_t>(2 + groups, 32768)));
  const auto kernel = a.weight_f32 ? (a.gate_f32 ? join_kernel<float, float> : join_kernel<float, T>)
                                   : (a.gate_f32 ? join_kernel<T, float> : join_kernel<T, T>);
  kernel<<<blocks, 1024, 0, stream>>>(a, grid);
  return cudaGetLastError();
}

}  // namespace

Grid backward_grid(const Args& a) {
  Grid grid;
  grid.sums_gate = a.dgate && a.gate_rows != 1;
  grid.group_rows = grid.sums_gate ? a.gate_rows : a.rows;
  const int64_t groups = a.rows / grid.group_rows;
  // rows that a block has under way, and blocks that are under way together
  // (two to a warp, where vectors fit; backward and joining of 2000 x 128 bfloat16 6.7 us, in units
  // of eight 7.5, 5000 x 128 8.7 and 8.7)
  const int rows = a.cols <= 128 && a.cols % 8 == 0 ? 16 : a.cols <= 256 ? 8 : 1;
  const int threads = a.cols <= 256 ? 256 : a.cols <= 512 ? 64 : a.cols <= 1024 ? 128 : a.cols <= 2048 ? 256 : 512;
  const int64_t most = 148ll * (512 / threads);
  const int64_t wanted = std::max<int64_t>(1, most / groups);
  grid.unit_rows = (grid.group_rows + wanted - 1) / wanted;
  grid.unit_rows = (grid.unit_rows + rows - 1) / rows * rows;
  grid.group_units = (grid.group_rows + grid.unit_rows - 1) / grid.unit_rows;
  grid.units = groups * grid.group_units;
  grid.blocks = static_cast<int>(std::min<int64_t>(grid.units, most));
  return grid;
}

int64_t backward_parts(const Args& a) {
  if (a.rows == 0 || a.cols == 0 || (!a.dw && !a.db && !a.dgate)) return 0;
  const Grid grid = backward_grid(a);
  return (2 * grid.blocks + (grid.sums_gate ? grid.units : 0)) * a.cols;
}

cudaError_t forward(const Args& a, cudaStream_t stream) {
  if (a.rows == 0 || a.cols == 0) return cudaSuccess;
  if (a.dtype == DType::kF32) return forward_f32(a, stream);
  return a.dtype == DType::kBF16 ? forward_bf16(a, stream) : forward_f16(a, stream);
}

cudaError_t backward(const Args& a, cudaStream_t stream) {
  if (a.cols == 0) return cudaSuccess;
  if (a.rows == 0) {  // empty sums
    const auto zero = [&](void* p, int64_t rows, bool f32) {
      return p && rows ? cudaMemsetAsync(p, 0, rows * a.cols * (f32 || a.dtype == DType::kF32 ? 4 : 2), stream) : cudaSuccess;
    };
    cudaError_t err = zero(a.dw, 1, a.weight_f32);
    if (err == cudaSuccess) err = zero(a.db, 1, a.weight_f32);
    return err == cudaSuccess ? zero(a.dgate, a.gate_groups, a.gate_f32) : err;
  }
  const Grid grid = backward_grid(a);
  const cudaError_t err = a.dtype == DType::kF32    ? backward_f32(a, grid, stream)
                          : a.dtype == DType::kBF16 ? backward_bf16(a, grid, stream)
                                                    : backward_f16(a, grid, stream);
  if (err != cudaSuccess || (!a.dw && !a.db && !grid.sums_gate)) return err;
  if (a.dtype == DType::kF32) return join<float>(a, grid, stream);
  return a.dtype == DType::kBF16 ? join<lin::bf16>(a, grid, stream) : join<__half>(a, grid, stream);
}

}  // namespace resnorm
