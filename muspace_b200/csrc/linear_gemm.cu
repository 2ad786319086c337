// The product D[m, n] = sum_k A(m, k) B(n, k) with the epilogues of the fused
// linear operator. A plain tiled kernel: a block of 256 threads takes 64 x 64
// outputs, 16 of k at a time through shared memory, float32 sums.
#include <algorithm>

#include "linear_device.cuh"

namespace lin {
namespace {

constexpr int kTile = 64, kDepth = 16;

__device__ __forceinline__ float element_of(const Operand& o, bool mn, int64_t i, int64_t k) {
  const int64_t at = mn ? k * o.ld + i : i * o.ld + k;
  float v = 0.f;
  for (int q = o.planes - 1; q >= 0; --q) v += __bfloat162float(o.p[q * o.plane + at]);
  return v;
}

template <typename T>
__global__ void __launch_bounds__(256) product_kernel(const Product pr) {
  __shared__ float as[kDepth][kTile + 1], bs[kDepth][kTile + 1];
  const int64_t m0 = static_cast<int64_t>(blockIdx.y) * kTile, n0 = static_cast<int64_t>(blockIdx.x) * kTile;
  const int tx = threadIdx.x % 8, ty = threadIdx.x / 8;  // 8 columns, 2 rows each
  float acc[2][8] = {};
  for (int64_t k0 = 0; k0 < pr.k; k0 += kDepth) {
    for (int i = threadIdx.x; i < kTile * kDepth; i += 256) {
      const int r = i / kDepth, d = i % kDepth;
      const int64_t k = k0 + d;
      as[d][r] = m0 + r < pr.m && k < pr.k ? element_of(pr.a, pr.a_mn, m0 + r, k) : 0.f;
      bs[d][r] = n0 + r < pr.n && k < pr.k ? element_of(pr.b, pr.b_mn, n0 + r, k) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int d = 0; d < kDepth; ++d)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[i][j] = fmaf(as[d][ty * 2 + i], bs[d][tx * 8 + j], acc[i][j]);
    __syncthreads();
  }
  const int64_t n = n0 + tx * 8;
  if (n >= pr.n) return;
  float b[8];
  load_bias8<T>(pr.epi, n, pr.n, b);
  for (int i = 0; i < 2; ++i)
    if (m0 + ty * 2 + i < pr.m) epilogue8<T>(pr.epi, acc[i], b, m0 + ty * 2 + i, n, pr.n, false);
}

}  // namespace

Plan plan_product(int64_t, int64_t, int64_t, int, bool, int) { return Plan{kTile, 1, 1, 0}; }

cudaError_t launch_product(const Product& pr, const Plan&, cudaStream_t stream) {
  if (pr.m == 0 || pr.n == 0) return cudaSuccess;
  const dim3 grid(static_cast<unsigned>((pr.n + kTile - 1) / kTile), static_cast<unsigned>((pr.m + kTile - 1) / kTile));
  if (pr.dtype == DType::kF32)
    product_kernel<float><<<grid, 256, 0, stream>>>(pr);
  else
    product_kernel<bf16><<<grid, 256, 0, stream>>>(pr);
  return cudaGetLastError();
}

}  // namespace lin
