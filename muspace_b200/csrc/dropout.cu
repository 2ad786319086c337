// Dropout: y = D(x), forward and (of a gradient) backward alike. Reads and writes
// each element once; a thread takes eight neighbouring columns of a row, which are
// one call of the generator.
#include <algorithm>

#include "dropout_device.cuh"
#include "linear_device.cuh"

namespace drop {
namespace {

constexpr int kThreads = 256;

// A thread's groups of eight are `step` apart; their rows and places follow by
// addition, as a division of 64 bits would cost as much as the generator.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    dropout_kernel(const T* __restrict__ x, int64_t x_stride, bool x_vec, int64_t rows, int64_t cols, bool y_vec,
                   const Rule rule, T* __restrict__ y) {
  const int64_t per_row = (cols + 7) / 8, step = static_cast<int64_t>(gridDim.x) * kThreads;
  const int64_t step_rows = step / per_row, step_groups = step - step_rows * per_row;
  const int64_t first = blockIdx.x * static_cast<int64_t>(kThreads) + threadIdx.x;
  int64_t r = first / per_row, g = first - r * per_row;
  const Key key = key_of(rule);
  for (; r < rows;) {
    const int64_t c = g * 8;
    const int count = static_cast<int>(cols - c < 8 ? cols - c : 8);
    float v[8];
    lin::load_some(x + r * x_stride + c, count, x_vec && count == 8, v);
    if (rule.threshold) apply8(key, numbers(key, static_cast<uint32_t>(r), static_cast<uint32_t>(g)), v);
    lin::store_some(y + r * cols + c, count, y_vec && count == 8, v);
    r += step_rows, g += step_groups;
    if (g >= per_row) g -= per_row, ++r;
  }
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <typename T>
cudaError_t launch(const void* x, int64_t x_stride, int64_t rows, int64_t cols, const Rule& rule, void* y,
                   cudaStream_t stream) {
  const int64_t groups = rows * ((cols + 7) / 8);
  if (groups == 0) return cudaSuccess;
  const bool x_vec = aligned16(x) && (x_stride * sizeof(T)) % 16 == 0;
  const bool y_vec = aligned16(y) && (cols * sizeof(T)) % 16 == 0;
  const int blocks = static_cast<int>(std::min<int64_t>((groups + kThreads - 1) / kThreads, 148 * 16));
  dropout_kernel<T><<<blocks, kThreads, 0, stream>>>(static_cast<const T*>(x), x_stride, x_vec, rows, cols, y_vec, rule,
                                                    static_cast<T*>(y));
  return cudaGetLastError();
}

}  // namespace

cudaError_t dropout(DType dtype, const void* x, int64_t x_stride, int64_t rows, int64_t cols, const Rule& rule, void* y,
                    cudaStream_t stream) {
  if (dtype == DType::kF32) return launch<float>(x, x_stride, rows, cols, rule, y, stream);
  if (dtype == DType::kBF16) return launch<lin::bf16>(x, x_stride, rows, cols, rule, y, stream);
  return launch<__half>(x, x_stride, rows, cols, rule, y, stream);
}

}  // namespace drop
