// Dropout: y = D(x), forward and (of a gradient) backward alike. Reads and writes each
// element once; a thread takes eight neighbouring columns, which are one call of the
// generator, and walks down the rows with them: with the column's and the sequence's
// words of the counter constant, so are four of the generator's twenty wide
// multiplications, which beside memory are the bound. 40000 x 512 bfloat16: 15.8
// us, 5.2 TB/s (17.7 with a thread's columns changing, 21 with 64-bit arithmetic for
// each group as well), 8192 x 8192 47 us, 5.7 TB/s; float32 40000 x 512 31 us.
#include <algorithm>

#include "dropout_device.cuh"
#include "linear_device.cuh"

namespace drop {
namespace {

constexpr int kThreads = 256;
constexpr int kBlocks = 8;  // to an SM, in 32 registers; five of them with two rows on their way 16.5 us, eight 17.1 (spills)

// Whole eights at 16-byte boundaries. blockIdx.y: ranges of `span` groups of eight
// columns, more than one only for rows of more columns than threads have. kSome:
// something may be dropped.
template <typename T, bool kSome>
__global__ void __launch_bounds__(kThreads, kBlocks)
    vector_kernel(const T* __restrict__ x, int64_t x_stride, uint32_t rows, int64_t cols, uint32_t span, const Rule rule,
                  T* __restrict__ y) {
  const uint32_t g0 = blockIdx.y * span, here = min(span, static_cast<uint32_t>(cols / 8) - g0);
  const uint32_t step = gridDim.x * kThreads / here;  // rows that a pass takes
  const uint32_t first = blockIdx.x * kThreads + threadIdx.x;
  uint32_t r = first / here;
  const uint32_t g = g0 + first - r * here;
  if (r >= step) return;  // the threads that are left over beyond whole rows
  const Key key = key_of(rule);
  const int64_t x_step = step * x_stride, y_step = step * cols;
  x += r * x_stride + g * 8ll;
  y += r * cols + g * 8ll;
  for (; r < rows; r += step) {
    float v[8];
    lin::load8(x, v);
    if (kSome) apply8(key, numbers(key, r, g), v);
    lin::store8(y, v);
    x += x_step, y += y_step;
  }
}

// Any rows: a warp takes 256 columns of a row at a time, a lane every 32nd of them, so
// that narrow accesses are neighbours; their 32 calls of the generator are one to a
// lane, and a lane fetches its bits from the lanes that have them. 40001 x 250
// bfloat16: 16.6 us (26 with eight neighbouring columns a thread).
template <typename T>
__global__ void __launch_bounds__(kThreads)
    ragged_kernel(const T* __restrict__ x, int64_t x_stride, int64_t rows, int64_t cols, const Rule rule,
                  T* __restrict__ y) {
  const int lane = threadIdx.x & 31;
  const int64_t chunks = (cols + 255) / 256, step = gridDim.x * (kThreads / 32ll);
  const int64_t step_rows = step / chunks, step_chunks = step - step_rows * chunks;
  const int64_t first = (blockIdx.x * static_cast<int64_t>(kThreads) + threadIdx.x) / 32;
  int64_t r = first / chunks, chunk = first - r * chunks;
  const Key key = key_of(rule);
  while (r < rows) {
    const T* from = x + r * x_stride + chunk * 256 + lane;
    T* to = y + r * cols + chunk * 256 + lane;
    const int count = static_cast<int>(cols - chunk * 256 < 256 ? cols - chunk * 256 : 256) - lane;  // of the columns from this lane's first on
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = 32 * j < count ? lin::to_float(from[32 * j]) : 0.f;
    if (rule.threshold) {
      const uint32_t group = static_cast<uint32_t>(chunk) * 32 + lane;
      const uint32_t mine = bits8(key, numbers(key, static_cast<uint32_t>(r), group));
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t bits = __shfl_sync(0xffffffffu, mine, j * 4 + lane / 8);
        v[j] = bits >> (lane % 8) & 1u ? v[j] * key.scale : 0.f;
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (32 * j < count) to[32 * j] = lin::from_float<T>(v[j]);
    r += step_rows, chunk += step_chunks;
    if (chunk >= chunks) chunk -= chunks, ++r;
  }
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <typename T>
cudaError_t launch(const void* x, int64_t x_stride, int64_t rows, int64_t cols, const Rule& rule, void* y,
                   cudaStream_t stream) {
  if (rows == 0 || cols == 0) return cudaSuccess;
  const int64_t most = 148 * kBlocks;
  if (aligned16(x) && (x_stride * sizeof(T)) % 16 == 0 && aligned16(y) && cols % 8 == 0) {
    const int64_t per_row = cols / 8, span = std::min<int64_t>(per_row, most * kThreads);
    const int64_t blocks = std::min<int64_t>((rows * span + kThreads - 1) / kThreads, most);
    const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>((per_row + span - 1) / span));
    const auto kernel = rule.threshold ? vector_kernel<T, true> : vector_kernel<T, false>;
    kernel<<<grid, kThreads, 0, stream>>>(static_cast<const T*>(x), x_stride, static_cast<uint32_t>(rows), cols,
                                          static_cast<uint32_t>(span), rule, static_cast<T*>(y));
  } else {
    const int64_t warps = rows * ((cols + 255) / 256);
    const int blocks = static_cast<int>(std::min<int64_t>((warps + kThreads / 32 - 1) / (kThreads / 32), most));
    ragged_kernel<T><<<blocks, kThreads, 0, stream>>>(static_cast<const T*>(x), x_stride, rows, cols, rule,
                                                     static_cast<T*>(y));
  }
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
