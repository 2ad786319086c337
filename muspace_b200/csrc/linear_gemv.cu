// The forward product for a few rows (one token, a few queries): bound by
// reading the weight once, so a warp takes a few rows of it, 16 bytes a lane at a
// time, against all rows of x (which stay in L1), in float32 arithmetic. The
// tensor-core kernel needs several times the set-up (tensor maps, tensor memory,
// barriers, a second kernel for its ranges of k), multiplies 128 rows, and in
// float32 first lays the weight out in planes. 1 x 4096 x 4096 in bfloat16: 8.2
// us, 4.1 TB/s; see few_rows for where the one or the other is the faster.

#include "linear_device.cuh"

namespace lin {
namespace {

constexpr int kWarps = 8;

template <typename T>
__device__ __forceinline__ void load_vec(const T* p, float v[16 / sizeof(T)]);
template <>
__device__ __forceinline__ void load_vec<bf16>(const bf16* p, float v[8]) {
  load8(p, v);
}
template <>
__device__ __forceinline__ void load_vec<float>(const float* p, float v[4]) {
  const float4 a = *reinterpret_cast<const float4*>(p);
  v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
}

// kRows rows of x (from blockIdx.y * kRows on) against kCols rows of the weight,
// whose columns `split` neighbouring warps share: few rows of a long weight are
// work for many warps, and their sums are added in order.
template <typename T, int kRows, int kCols, int kUnroll, int split, bool kVec>
__global__ void __launch_bounds__(32 * kWarps) gemv_kernel(const Args a) {
  constexpr int kPer = kVec ? 16 / sizeof(T) : 1, kOut = kCols * kRows, step = 32 * kPer * split;
  __shared__ float parts[split > 1 ? kWarps : 1][kOut];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t n0 = (blockIdx.x * static_cast<int64_t>(kWarps / split) + warp / split) * kCols;
  const int64_t m0 = blockIdx.y * static_cast<int64_t>(kRows);
  const int cols = static_cast<int>(a.out - n0 < kCols ? a.out - n0 : kCols);
  const int rows = static_cast<int>(a.rows - m0 < kRows ? a.rows - m0 : kRows);
  float acc[kCols][kRows] = {};
  if (cols > 0) {
    const T* w = static_cast<const T*>(a.w) + n0 * a.w_stride;
    const T* x = static_cast<const T*>(a.x) + m0 * a.x_stride;
    const auto load_w = [&](int64_t k, float u[kCols][kPer]) {
#pragma unroll
      for (int c = 0; c < kCols; ++c) {
        const T* p = w + (c < cols ? c : 0) * a.w_stride + k;  // a row that is not there repeats the first
        if constexpr (kVec)
          load_vec<T>(p, u[c]);
        else
          u[c][0] = to_float(*p);
      }
    };
    const auto multiply = [&](int64_t k, const float u[kCols][kPer]) {
#pragma unroll
      for (int m = 0; m < kRows; ++m) {
        if (m < rows) {
          float v[kPer];
          if constexpr (kVec)
            load_vec<T>(x + m * a.x_stride + k, v);
          else
            v[0] = to_float(x[m * a.x_stride + k]);
#pragma unroll
          for (int c = 0; c < kCols; ++c)
#pragma unroll
            for (int j = 0; j < kPer; ++j) acc[c][m] = fmaf(u[c][j], v[j], acc[c][m]);
        }
      }
    };
    int64_t k = (warp % split * 32 + lane) * kPer;
    for (; k + (kUnroll - 1) * step < a.in; k += kUnroll * step) {  // this many loads on their way together
      float u[kUnroll][kCols][kPer];
#pragma unroll
      for (int q = 0; q < kUnroll; ++q) load_w(k + q * step, u[q]);
#pragma unroll
      for (int q = 0; q < kUnroll; ++q) multiply(k + q * step, u[q]);
    }
    for (; k < a.in; k += step) {
      float u[kCols][kPer];
      load_w(k, u);
      multiply(k, u);
    }
  }
  const auto finish = [&](int o, float z0) {
    const int c = o / kRows;
    if (c >= cols || o % kRows >= rows) return;
    float z[2] = {z0, 0.f}, s[2];
    const int64_t m = m0 + o % kRows, n = n0 + c;
    if (a.bias) z[0] += to_float(static_cast<const T*>(a.bias)[n]);
    activate<sizeof(T) == 2, true, true, 2>(a.act, z, s);
    if (a.slope)
      static_cast<typename SlopeOf<T>::type*>(a.slope)[m * a.out + n] = from_float<typename SlopeOf<T>::type>(s[0]);
    if (a.r) z[0] += to_float(static_cast<const T*>(a.r)[m * a.r_stride + n]);
    static_cast<T*>(a.y)[m * a.y_stride + n] = from_float<T>(z[0]);
  };
  float mine = 0.f;  // lane o % 32 keeps output o
#pragma unroll
  for (int o = 0; o < kOut; ++o) {
    float t = acc[o / kRows][o % kRows];
#pragma unroll
    for (int d = 16; d; d >>= 1) t += __shfl_xor_sync(0xffffffffu, t, d);
    if (lane == o % 32) mine = t;
  }
  static_assert(kOut <= 32, "an output to a lane");
  if (split == 1) {
    if (lane < kOut) finish(lane, mine);
    return;
  }
  if (lane < kOut) parts[warp][lane] = mine;
  __syncthreads();
  if (warp % split != 0 || lane >= kOut) return;  // the first of the warps finishes
  float sum = 0.f;
#pragma unroll
  for (int q = 0; q < split; ++q) sum += parts[warp + q][lane];
  finish(lane, sum);
}

template <typename T, int kRows, int kCols, int kUnroll>
cudaError_t launch(const Args& a, bool vec, cudaStream_t stream) {
  const int64_t steps = a.in / (32 * (vec ? 16 / sizeof(T) : 1)), groups = (a.out + kCols - 1) / kCols;
  // Four warps to a weight row where one each would leave half of the GPU's
  // warps idle over rows of eight steps or more (bfloat16, one row of 8192:
  // 1024 weight rows 16 us with one warp, 7 with four; 4096 x 4096 8.4 and 10).
  const bool shared = steps >= 8 && groups < 148 * 16;
  const int64_t per_block = (shared ? kWarps / 4 : kWarps) * kCols;
  const dim3 grid(static_cast<unsigned>((a.out + per_block - 1) / per_block),
                  static_cast<unsigned>((a.rows + kRows - 1) / kRows));
  const auto kernel = shared ? (vec ? gemv_kernel<T, kRows, kCols, kUnroll, 4, true>
                                    : gemv_kernel<T, kRows, kCols, kUnroll, 4, false>)
                             : (vec ? gemv_kernel<T, kRows, kCols, kUnroll, 1, true>
                                    : gemv_kernel<T, kRows, kCols, kUnroll, 1, false>);
  kernel<<<grid, 32 * kWarps, 0, stream>>>(a);
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch_rows(const Args& a, cudaStream_t stream) {
  const auto aligned = [](const void* p, int64_t stride) {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (stride * sizeof(T)) % 16 == 0;
  };
  const bool vec = aligned(a.x, a.rows == 1 ? 0 : a.x_stride) && aligned(a.w, a.out == 1 ? 0 : a.w_stride) &&
                   (a.in * sizeof(T)) % 16 == 0;
  if (a.rows == 1) return launch<T, 1, 1, 4>(a, vec, stream);
  if (a.rows <= 4) return launch<T, 4, 1, 2>(a, vec, stream);
  return launch<T, 8, 2, 2>(a, vec, stream);
}

}  // namespace

// Where this kernel is the faster one (B200, us here / on the tensor cores).
// bfloat16: up to 4 rows (1 x 4096 x 4096 8.2 / 13.9; 4 rows 14.1 / 13.9, as good
// as even, and here without sums in a workspace or a second launch), and up
// to 8 of short ones (8 x 256 x 512 4.0 / 6.0; 8 x 1024 x 256 9.1 / 7.0).
// float32, which the tensor cores get in planes: up to 16 rows of any weight (16
// x 4096 x 4096 48 / 86), and more while the products are few (64 x 256 x 512
// 4.5 / 25, 256 x 256 x 1024 18 / 23, 512 x 512 x 512 25 / 18).
bool few_rows(const Args& a) {
  if (a.dtype == DType::kBF16) return a.rows <= (a.in <= 512 ? 8 : 4);
  return a.rows <= 16 || (a.rows <= 1024 && a.rows * a.in * a.out <= 1ll << 26);
}

cudaError_t forward_few_rows(const Args& a, cudaStream_t stream) {
  return a.dtype == DType::kF32 ? launch_rows<float>(a, stream) : launch_rows<bf16>(a, stream);
}

}  // namespace lin
