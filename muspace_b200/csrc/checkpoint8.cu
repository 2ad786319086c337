// 8-bit activation checkpoints as tensors: pack and unpack. Both read and
// write every element once and are bound by memory.
//
// A thread holds eight neighbouring columns, four threads a block of 32, whose
// largest magnitude they find with two shuffles. A row's threads are padded to
// whole blocks, so the four are always neighbours in one warp.
#include <algorithm>

#include "checkpoint8.cuh"
#include "layer_norm.h"
#include "linear_device.cuh"

namespace ckpt {
namespace {

using lin::bf16;

constexpr int kThreads = 256;

template <typename T>
__global__ void __launch_bounds__(kThreads)
    pack_kernel(const T* __restrict__ x, int64_t stride, bool vec, int64_t rows, int64_t cols,
                int8_t* __restrict__ codes, bool code_vec, uint8_t* __restrict__ exps) {
  const int64_t blocks = blocks_of(cols), per_row = blocks * 4, total = rows * per_row;
  // every lane of a warp runs the same rounds: the shuffles need whole warps
  const int64_t first = blockIdx.x * static_cast<int64_t>(kThreads) + threadIdx.x;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kThreads;
  for (int64_t i = first; i - (threadIdx.x & 31) < total; i += step) {
    const int64_t r = i / per_row, g = i - r * per_row, c = g * 8;
    const int count = i < total && c < cols ? static_cast<int>(cols - c < 8 ? cols - c : 8) : 0;
    float v[8];
    if (count > 0)
      lin::load_some(x + r * stride + c, count, vec && count == 8, v);
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (count == 0) v[j] = 0.f;
      top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
    }
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const uint32_t e = exponent_of(top);
    if (count > 0) store_codes8(codes + r * cols + c, count, code_vec && count == 8, e, v);
    if (count > 0 && (g & 3) == 0) exps[r * blocks + (g >> 2)] = static_cast<uint8_t>(e);
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
    unpack_kernel(const int8_t* __restrict__ codes, bool code_vec, const uint8_t* __restrict__ exps, int64_t rows,
                  int64_t cols, T* __restrict__ x, bool vec) {
  const int64_t per_row = (cols + 7) / 8, total = rows * per_row, blocks = blocks_of(cols);
  for (int64_t i = blockIdx.x * static_cast<int64_t>(kThreads) + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * kThreads) {
    const int64_t r = i / per_row, c = (i - r * per_row) * 8;
    const int count = static_cast<int>(cols - c < 8 ? cols - c : 8);
    float v[8];
    load_codes8(codes + r * cols + c, count, code_vec && count == 8, exps[r * blocks + c / kBlock], v);
    lin::store_some(x + r * cols + c, count, vec && count == 8, v);
  }
}

inline int grid_for(int64_t threads) {
  return static_cast<int>(std::min<int64_t>((threads + kThreads - 1) / kThreads, 148 * 16));
}

inline bool aligned(const void* p, unsigned to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

}  // namespace

cudaError_t pack(bool is_bf16, const void* x, int64_t stride, int64_t rows, int64_t cols, int8_t* codes, uint8_t* exps,
                 cudaStream_t stream) {
  const int64_t threads = rows * blocks_of(cols) * 4;
  if (threads == 0) return cudaSuccess;
  const bool vec = aligned(x, 16) && stride % (is_bf16 ? 8 : 4) == 0;
  const bool code_vec = aligned(codes, 8) && cols % 8 == 0;
  if (is_bf16)
    pack_kernel<<<grid_for(threads), kThreads, 0, stream>>>(static_cast<const bf16*>(x), stride, vec, rows, cols, codes,
                                                           code_vec, exps);
  else
    pack_kernel<<<grid_for(threads), kThreads, 0, stream>>>(static_cast<const float*>(x), stride, vec, rows, cols,
                                                           codes, code_vec, exps);
  return cudaGetLastError();
}

cudaError_t unpack(bool is_bf16, const int8_t* codes, const uint8_t* exps, int64_t rows, int64_t cols, void* x,
                   cudaStream_t stream) {
  const int64_t threads = rows * ((cols + 7) / 8);
  if (threads == 0) return cudaSuccess;
  const bool code_vec = aligned(codes, 8) && cols % 8 == 0;
  const bool vec = aligned(x, 16) && cols % (is_bf16 ? 8 : 4) == 0;
  if (is_bf16)
    unpack_kernel<<<grid_for(threads), kThreads, 0, stream>>>(codes, code_vec, exps, rows, cols, static_cast<bf16*>(x),
                                                             vec);
  else
    unpack_kernel<<<grid_for(threads), kThreads, 0, stream>>>(codes, code_vec, exps, rows, cols,
                                                             static_cast<float*>(x), vec);
  return cudaGetLastError();
}

}  // namespace ckpt
