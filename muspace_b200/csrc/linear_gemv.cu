// The forward product for a few rows (one token, a few queries): bound by
// reading the weight once, so a warp takes one row of it, 16 bytes a lane at a
// time, against all rows of x (which stay in L1), in float32 arithmetic. The
// tensor-core kernel needs several times the set-up (tensor maps, tensor memory,
// barriers, a second kernel for its ranges of k) and would multiply 128 rows.
#include <algorithm>

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

template <typename T, int kRows, bool kVec>
__global__ void __launch_bounds__(32 * kWarps) gemv_kernel(const Args a) {
  constexpr int kPer = kVec ? 16 / sizeof(T) : 1, kStep = 32 * kPer;
  const int lane = threadIdx.x & 31;
  const int64_t n = blockIdx.x * static_cast<int64_t>(kWarps) + (threadIdx.x >> 5);
  if (n >= a.out) return;
  const T* w = static_cast<const T*>(a.w) + n * a.w_stride;
  const T* x = static_cast<const T*>(a.x);
  float acc[kRows] = {};
#pragma unroll 4
  for (int64_t k = lane * kPer; k < a.in; k += kStep) {
    float u[kPer];
    if constexpr (kVec)
      load_vec<T>(w + k, u);
    else
      u[0] = to_float(w[k]);
#pragma unroll
    for (int m = 0; m < kRows; ++m) {
      if (m < a.rows) {
        float v[kPer];
        if constexpr (kVec)
          load_vec<T>(x + m * a.x_stride + k, v);
        else
          v[0] = to_float(x[m * a.x_stride + k]);
#pragma unroll
        for (int j = 0; j < kPer; ++j) acc[m] = fmaf(u[j], v[j], acc[m]);
      }
    }
  }
#pragma unroll
  for (int m = 0; m < kRows; ++m)
#pragma unroll
    for (int d = 16; d; d >>= 1) acc[m] += __shfl_xor_sync(0xffffffffu, acc[m], d);
  if (lane >= a.rows) return;  // lane m finishes row m
  float z[2] = {0.f, 0.f}, s[2];
#pragma unroll
  for (int m = 0; m < kRows; ++m)
    if (lane == m) z[0] = acc[m];
  if (a.bias) z[0] += to_float(static_cast<const T*>(a.bias)[n]);
  activate<sizeof(T) == 2, true, true, 2>(a.act, z, s);
  if (a.slope)
    static_cast<typename SlopeOf<T>::type*>(a.slope)[lane * a.out + n] = from_float<typename SlopeOf<T>::type>(s[0]);
  if (a.r) z[0] += to_float(static_cast<const T*>(a.r)[lane * a.r_stride + n]);
  static_cast<T*>(a.y)[lane * a.y_stride + n] = from_float<T>(z[0]);
}

constexpr int64_t kMostRows = 4;

template <typename T>
cudaError_t launch(const Args& a, cudaStream_t stream) {
  const auto aligned = [](const void* p, int64_t stride) {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (stride * sizeof(T)) % 16 == 0;
  };
  const bool vec = aligned(a.x, a.rows == 1 ? 0 : a.x_stride) && aligned(a.w, a.w_stride) && (a.in * sizeof(T)) % 16 == 0;
  const unsigned blocks = static_cast<unsigned>((a.out + kWarps - 1) / kWarps);
  if (a.rows == 1)
    (vec ? gemv_kernel<T, 1, true> : gemv_kernel<T, 1, false>)<<<blocks, 32 * kWarps, 0, stream>>>(a);
  else
    (vec ? gemv_kernel<T, kMostRows, true> : gemv_kernel<T, kMostRows, false>)<<<blocks, 32 * kWarps, 0, stream>>>(a);
  return cudaGetLastError();
}

}  // namespace

bool few_rows(const Args& a) { return a.rows <= kMostRows; }

cudaError_t forward_few_rows(const Args& a, cudaStream_t stream) {
  return a.dtype == DType::kF32 ? launch<float>(a, stream) : launch<bf16>(a, stream);
}

}  // namespace lin
