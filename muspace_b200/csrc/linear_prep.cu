// Operand layouts of the fused linear kernels: what the tensor maps cannot
// read as it stands (rows off 16-byte boundaries, float32, 8-bit checkpoints,
// gradients still to be multiplied by the activation's slope) is laid out once
// here. All of these kernels read and write each element once and are bound by
// memory; a thread takes eight neighbouring columns of a row.
#include <algorithm>

#include "checkpoint8.cuh"
#include "linear_device.cuh"

namespace lin {
namespace {

constexpr int kThreads = 256;

inline int blocks_for(int64_t groups) {
  return static_cast<int>(std::min<int64_t>((groups + kThreads - 1) / kThreads, 148 * 16));
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <typename T>
__device__ __forceinline__ void put(bf16* dst, int64_t plane, const float v[8]) {
  if (sizeof(T) == 4)
    store_planes(dst, plane, 8, true, v);
  else
    store8(dst, v);
}

// dst = src, or src * slope. A row of dst is padded to a multiple of eight
// elements, so its vectors always fit; what they hold beyond `cols` is zero.
template <typename T, bool kScale>
__global__ void __launch_bounds__(kThreads)
    operand_kernel(const T* __restrict__ src, int64_t src_ld, bool src_vec,
                   const typename SlopeOf<T>::type* __restrict__ slope, bool slope_vec, bf16* __restrict__ dst,
                   int64_t dst_ld, int64_t plane, int64_t rows, int64_t cols) {
  const int64_t per_row = (cols + 7) / 8, total = rows * per_row;
  for (int64_t i = blockIdx.x * static_cast<int64_t>(kThreads) + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * kThreads) {
    const int64_t r = i / per_row, c = (i - r * per_row) * 8;
    const int count = static_cast<int>(cols - c < 8 ? cols - c : 8);
    float v[8];
    load_some(src + r * src_ld + c, count, src_vec && count == 8, v);
    if (kScale) {
      float s[8];
      load_some(slope + r * cols + c, count, slope_vec && count == 8, s);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] *= s[j];
    }
    put<T>(dst + r * dst_ld + c, plane, v);
  }
}

template <typename T, bool kScale>
cudaError_t launch_operand(const void* src, int64_t src_ld, const void* slope, const Operand& dst, cudaStream_t stream) {
  using S = typename SlopeOf<T>::type;
  const int64_t groups = dst.rows * ((dst.cols + 7) / 8);
  if (groups == 0) return cudaSuccess;
  const bool src_vec = aligned16(src) && (src_ld * sizeof(T)) % 16 == 0;
  const bool slope_vec = aligned16(slope) && (dst.cols * sizeof(S)) % 16 == 0;
  operand_kernel<T, kScale><<<blocks_for(groups), kThreads, 0, stream>>>(
      static_cast<const T*>(src), src_ld, src_vec, static_cast<const S*>(slope), slope_vec, const_cast<bf16*>(dst.p),
      dst.ld, dst.plane, dst.rows, dst.cols);
  return cudaGetLastError();
}

__global__ void __launch_bounds__(kThreads)
    unpack_kernel(const int8_t* __restrict__ codes, bool vec, const uint8_t* __restrict__ exps, bf16* __restrict__ dst,
                  int64_t dst_ld, int64_t rows, int64_t cols) {
  const int64_t per_row = (cols + 7) / 8, total = rows * per_row;
  const int64_t blocks = ckpt::blocks_of(cols);
  for (int64_t i = blockIdx.x * static_cast<int64_t>(kThreads) + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * kThreads) {
    const int64_t r = i / per_row, c = (i - r * per_row) * 8;
    const int count = static_cast<int>(cols - c < 8 ? cols - c : 8);
    float v[8];
    ckpt::load_codes8(codes + r * cols + c, count, vec, exps[r * blocks + c / ckpt::kBlock], v);
    store8(dst + r * dst_ld + c, v);  // exact: 7 bits and a power of two
  }
}

// ---- column sums -------------------------------------------------------------------

// A block takes 256 columns (a lane eight of them, a warp a row at a time) and a
// range of rows; the ranges' sums go to `parts` and are added in order by the
// second kernel, so the result does not depend on scheduling. 40000 x 512:
// two columns a lane and at most 64 ranges left too few loads on their way
// (25 us, 1.6 TB/s).
constexpr int kSumCols = 256, kSumWarps = 8;

// The block's warps' sums, in order, as part blockIdx.y.
__device__ __forceinline__ void put_sums(float (*buf)[kSumCols], const float s[8], int64_t cols, float* parts) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int j = 0; j < 8; ++j) buf[warp][lane + 32 * j] = s[j];
  __syncthreads();
  const int64_t c = blockIdx.x * static_cast<int64_t>(kSumCols) + lane * 8 + warp;  // column `warp` of the lane's eight
  float sum = 0.f;
#pragma unroll
  for (int w = 0; w < kSumWarps; ++w) sum += buf[w][lane + 32 * warp];
  if (c < cols) parts[blockIdx.y * cols + c] = sum;
}

// kRagged: cols is no multiple of eight. Rows are multiples of eight apart, so a
// vector that reaches beyond a row ends before the next one, and what it holds
// there is not kept; but the last row may be the end of a caller's memory, and is
// read element by element. (In one kernel for both, 8192 x 8192 took 32 us instead
// of 23: the loop's end then costs it loads on their way.)
template <bool kRagged>
__global__ void __launch_bounds__(32 * kSumWarps)
    column_parts_kernel(const bf16* __restrict__ src, int64_t ld, int64_t rows, int64_t cols, int64_t rows_per_part,
                        float* __restrict__ parts) {
  __shared__ float buf[kSumWarps][kSumCols];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c = blockIdx.x * static_cast<int64_t>(kSumCols) + lane * 8;
  const int64_t begin = blockIdx.y * rows_per_part, end = min(rows, begin + rows_per_part);
  const int64_t whole = kRagged ? min(end, rows - 1) : end;
  float s[8] = {};
  if (c < cols) {
#pragma unroll 4
    for (int64_t r = begin + warp; r < whole; r += kSumWarps) {
      float v[8];
      load8(src + r * ld + c, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) s[j] += v[j];
    }
    if (kRagged && whole < end && (end - 1 - begin) % kSumWarps == warp) {
      float v[8];
      load_some(src + (rows - 1) * ld + c, static_cast<int>(cols - c < 8 ? cols - c : 8), false, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) s[j] += v[j];
    }
  }
  put_sums(buf, s, cols, parts);
}

// operand_kernel with the sums of what it writes, before it is rounded. Bound by
// memory: 8192 x 8192 bfloat16 with a float16 slope (403 MB) takes 67 us, 6.0 TB/s.
// Two rows unrolled in 64 registers, four blocks to an SM; four rows unrolled
// without a bound on the registers took 94 us, in 64 registers 83 (they spill).
template <typename T, bool kScale>
__global__ void __launch_bounds__(32 * kSumWarps, 4)
    operand_sums_kernel(const T* __restrict__ src, int64_t src_ld, bool src_vec,
                        const typename SlopeOf<T>::type* __restrict__ slope, bool slope_vec, bf16* __restrict__ dst,
                        int64_t dst_ld, int64_t plane, int64_t rows, int64_t cols, int64_t rows_per_part,
                        float* __restrict__ parts) {
  __shared__ float buf[kSumWarps][kSumCols];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c = blockIdx.x * static_cast<int64_t>(kSumCols) + lane * 8;
  const int64_t begin = blockIdx.y * rows_per_part, end = min(rows, begin + rows_per_part);
  const int count = static_cast<int>(cols - c < 8 ? cols - c : 8);
  float s[8] = {};
  if (c < cols) {
#pragma unroll 2
    for (int64_t r = begin + warp; r < end; r += kSumWarps) {
      float v[8];
      load_some(src + r * src_ld + c, count, src_vec && count == 8, v);
      if (kScale) {
        float f[8];
        load_some(slope + r * cols + c, count, slope_vec && count == 8, f);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] *= f[j];
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) s[j] += v[j];
      put<T>(dst + r * dst_ld + c, plane, v);
    }
  }
  put_sums(buf, s, cols, parts);
}

template <typename T, bool kScale>
cudaError_t launch_operand_sums(const void* src, int64_t src_ld, const void* slope, const Operand& dst, float* parts,
                                cudaStream_t stream) {
  using S = typename SlopeOf<T>::type;
  const int64_t count = column_parts(dst.rows, dst.cols);
  if (dst.rows == 0 || dst.cols == 0) return cudaSuccess;
  const bool src_vec = aligned16(src) && (src_ld * sizeof(T)) % 16 == 0;
  const bool slope_vec = aligned16(slope) && (dst.cols * sizeof(S)) % 16 == 0;
  const dim3 grid(static_cast<unsigned>((dst.cols + kSumCols - 1) / kSumCols), static_cast<unsigned>(count));
  operand_sums_kernel<T, kScale><<<grid, 32 * kSumWarps, 0, stream>>>(
      static_cast<const T*>(src), src_ld, src_vec, static_cast<const S*>(slope), slope_vec, const_cast<bf16*>(dst.p),
      dst.ld, dst.plane, dst.rows, dst.cols, (dst.rows + count - 1) / count, parts);
  return cudaGetLastError();
}

template <typename T>
__global__ void __launch_bounds__(1024)
    add_parts_kernel(const float* __restrict__ parts, int64_t count, int64_t cols, T* __restrict__ sums) {
  __shared__ float buf[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c = blockIdx.x * 32ll + lane;
  float s = 0.f;
  if (c < cols) {
#pragma unroll 8
    for (int64_t i = warp; i < count; i += 32) s += parts[i * cols + c];
  }
  buf[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && c < cols) {
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) s += buf[i][lane];
    sums[c] = from_float<T>(s);
  }
}

}  // namespace

cudaError_t copy_operand(DType dtype, const void* src, int64_t src_ld, const Operand& dst, cudaStream_t stream) {
  return dtype == DType::kF32 ? launch_operand<float, false>(src, src_ld, nullptr, dst, stream)
                              : launch_operand<bf16, false>(src, src_ld, nullptr, dst, stream);
}

cudaError_t scale_operand(DType dtype, const void* g, int64_t g_ld, const void* slope, const Operand& dst,
                          cudaStream_t stream) {
  return dtype == DType::kF32 ? launch_operand<float, true>(g, g_ld, slope, dst, stream)
                              : launch_operand<bf16, true>(g, g_ld, slope, dst, stream);
}

cudaError_t unpack_operand(const int8_t* codes, const uint8_t* exps, const Operand& dst, cudaStream_t stream) {
  const int64_t groups = dst.rows * ((dst.cols + 7) / 8);
  if (groups == 0) return cudaSuccess;
  const bool vec = (reinterpret_cast<uintptr_t>(codes) & 7) == 0 && dst.cols % 8 == 0;
  unpack_kernel<<<blocks_for(groups), kThreads, 0, stream>>>(codes, vec, exps, const_cast<bf16*>(dst.p), dst.ld,
                                                            dst.rows, dst.cols);
  return cudaGetLastError();
}

int column_parts(int64_t rows, int64_t cols) {
  const int64_t across = (cols + kSumCols - 1) / kSumCols;
  return static_cast<int>(std::min<int64_t>((rows + 31) / 32, std::max<int64_t>(1, 148 * 4 / std::max<int64_t>(across, 1))));
}

cudaError_t operand_and_sums(DType dtype, const void* g, int64_t g_ld, const void* slope, const Operand& dst,
                             float* parts, cudaStream_t stream) {
  if (dtype == DType::kF32)
    return slope ? launch_operand_sums<float, true>(g, g_ld, slope, dst, parts, stream)
                 : launch_operand_sums<float, false>(g, g_ld, nullptr, dst, parts, stream);
  return slope ? launch_operand_sums<bf16, true>(g, g_ld, slope, dst, parts, stream)
               : launch_operand_sums<bf16, false>(g, g_ld, nullptr, dst, parts, stream);
}

cudaError_t column_sums(const Operand& src, float* parts, cudaStream_t stream) {
  if (src.cols == 0 || src.rows == 0) return cudaSuccess;
  const int count = column_parts(src.rows, src.cols);
  const dim3 grid(static_cast<unsigned>((src.cols + kSumCols - 1) / kSumCols), static_cast<unsigned>(count));
  const auto kernel = src.cols % 8 == 0 ? column_parts_kernel<false> : column_parts_kernel<true>;
  kernel<<<grid, 32 * kSumWarps, 0, stream>>>(src.p, src.ld, src.rows, src.cols, (src.rows + count - 1) / count, parts);
  return cudaGetLastError();
}

cudaError_t add_parts(DType out_dtype, const float* parts, int64_t count, int64_t cols, void* sums,
                      cudaStream_t stream) {
  const unsigned blocks = static_cast<unsigned>((cols + 31) / 32);
  if (blocks == 0) return cudaSuccess;
  if (out_dtype == DType::kF32)
    add_parts_kernel<<<blocks, 1024, 0, stream>>>(parts, count, cols, static_cast<float*>(sums));
  else
    add_parts_kernel<<<blocks, 1024, 0, stream>>>(parts, count, cols, static_cast<bf16*>(sums));
  return cudaGetLastError();
}

}  // namespace lin
