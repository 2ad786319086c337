// The forward product for a few rows (one token, a few queries): bound by
// reading the weight once, so a warp takes a few rows of it, 16 bytes a lane at a
// time, against all rows of x (which stay in L1), in float32 arithmetic. The
// tensor-core kernel needs several times the set-up (tensor maps, tensor memory,
// barriers, a second kernel for its ranges of k), multiplies 128 rows, and in
// float32 first lays the weight out in planes. 1 x 4096 x 4096 in bfloat16: 8.2
// us, 4.1 TB/s; see few_rows for where the one or the other is the faster.

#include "dropout_device.cuh"
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

// What becomes of a sum of the plain operator, and of the two of the gated one.
template <typename T>
__device__ __forceinline__ void finish(const Args& a, int64_t m, int64_t n, const float sums[1]) {
  float z[2] = {sums[0], 0.f}, s[2];
  if (a.bias) z[0] += to_float(static_cast<const T*>(a.bias)[n]);
  activate<sizeof(T) == 2, true, true, 2>(a.act, z, s);
  if (a.slope)
    static_cast<typename SlopeOf<T>::type*>(a.slope)[m * a.out + n] = from_float<typename SlopeOf<T>::type>(s[0]);
  if (a.r) z[0] += to_float(static_cast<const T*>(a.r)[m * a.r_stride + n]);
  static_cast<T*>(a.y)[m * a.y_stride + n] = from_float<T>(z[0]);
}
template <typename T>
__device__ __forceinline__ void finish(const GatedArgs& a, int64_t m, int64_t n, const float sums[2]) {
  float g[2] = {sums[0], 0.f}, s[2], u = sums[1];
  if (a.bias) {
    g[0] += to_float(static_cast<const T*>(a.bias)[n]);
    u += to_float(static_cast<const T*>(a.bias)[a.out + n]);
  }
  activate<sizeof(T) == 2, true, true, 2>(a.act, g, s);
  bool kept = true;
  if (a.rule.threshold) {
    const drop::Key key = drop::key_of(a.rule);
    const drop::Words words = drop::numbers(key, static_cast<uint32_t>(m), static_cast<uint32_t>(n / 8));
    uint32_t word = words.w[0];  // of column n % 8, without an index into registers
    if (n % 8 >= 2) word = words.w[1];
    if (n % 8 >= 4) word = words.w[2];
    if (n % 8 >= 6) word = words.w[3];
    kept = n % 2 ? word > key.high : (word << 16) > key.low;
    g[0] = kept ? g[0] : 0.f, s[0] = kept ? s[0] : 0.f, u = kept ? u * a.rule.scale : 0.f;
  }
  if (sizeof(T) == 4 && a.factors) {  // float32; the others' need eight neighbours
    float* factors = static_cast<float*>(a.factors) + m * 2 * a.out + n;
    factors[0] = s[0] * u;
    factors[a.out] = kept ? g[0] * a.rule.scale : __uint_as_float(kDroppedFloat);
  }
  static_cast<T*>(a.y)[m * a.y_stride + n] = from_float<T>(g[0] * u);
}

// Rows of the weight to a column of the output.
template <typename A>
constexpr int kHalves = 1;
template <>
constexpr int kHalves<GatedArgs> = 2;

// kRows rows of x (from blockIdx.y * kRows on) against kCols rows of the weight (of
// each half, in the gated operator), whose columns `split` neighbouring warps share:
// few rows of a long weight are work for many warps, and their sums are added in order.
template <typename T, int kRows, int kCols, int kUnroll, int split, bool kVec, typename A>
__global__ void __launch_bounds__(32 * kWarps) gemv_kernel(const A a) {
  constexpr int kPer = kVec ? 16 / sizeof(T) : 1, kOut = kCols * kRows, step = 32 * kPer * split;
  constexpr int kH = kHalves<A>, kW = kH * kCols;  // rows of the weight
  __shared__ float parts[split > 1 ? kWarps : 1][kH * kOut];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t n0 = (blockIdx.x * static_cast<int64_t>(kWarps / split) + warp / split) * kCols;
  const int64_t m0 = blockIdx.y * static_cast<int64_t>(kRows);
  const int cols = static_cast<int>(a.out - n0 < kCols ? a.out - n0 : kCols);
  const int rows = static_cast<int>(a.rows - m0 < kRows ? a.rows - m0 : kRows);
  float acc[kW][kRows] = {};
  if (cols > 0) {
    const T* w = static_cast<const T*>(a.w) + n0 * a.w_stride;
    const T* x = static_cast<const T*>(a.x) + m0 * a.x_stride;
    const auto load_w = [&](int64_t k, float u[kW][kPer]) {
#pragma unroll
      for (int c = 0; c < kW; ++c) {
        // a row that is not there repeats the first
        const T* p = w + ((c % kCols < cols ? c % kCols : 0) + (c < kCols ? 0 : a.out)) * a.w_stride + k;
        if constexpr (kVec)
          load_vec<T>(p, u[c]);
        else
          u[c][0] = to_float(*p);
      }
    };
    const auto multiply = [&](int64_t k, const float u[kW][kPer]) {
#pragma unroll
      for (int m = 0; m < kRows; ++m) {
        if (m < rows) {
          float v[kPer];
          if constexpr (kVec)
            load_vec<T>(x + m * a.x_stride + k, v);
          else
            v[0] = to_float(x[m * a.x_stride + k]);
#pragma unroll
          for (int c = 0; c < kW; ++c)
#pragma unroll
            for (int j = 0; j < kPer; ++j) acc[c][m] = fmaf(u[c][j], v[j], acc[c][m]);
        }
      }
    };
    int64_t k = (warp % split * 32 + lane) * kPer;
    for (; k + (kUnroll - 1) * step < a.in; k += kUnroll * step) {  // this many loads on their way together
      float u[kUnroll][kW][kPer];
#pragma unroll
      for (int q = 0; q < kUnroll; ++q) load_w(k + q * step, u[q]);
#pragma unroll
      for (int q = 0; q < kUnroll; ++q) multiply(k + q * step, u[q]);
    }
    for (; k < a.in; k += step) {
      float u[kW][kPer];
      load_w(k, u);
      multiply(k, u);
    }
  }
  const auto put = [&](int o, const float sums[kH]) {
    const int c = o / kRows;
    if (c < cols && o % kRows < rows) finish<T>(a, m0 + o % kRows, n0 + c, sums);
  };
  float mine[kH] = {};  // lane o % 32 keeps output o
#pragma unroll
  for (int o = 0; o < kOut; ++o)
#pragma unroll
    for (int h = 0; h < kH; ++h) {
      float t = acc[h * kCols + o / kRows][o % kRows];
#pragma unroll
      for (int d = 16; d; d >>= 1) t += __shfl_xor_sync(0xffffffffu, t, d);
      if (lane == o % 32) mine[h] = t;
    }
  static_assert(kOut <= 32, "an output to a lane");
  if (split == 1) {
    if (lane < kOut) put(lane, mine);
    return;
  }
  if (lane < kOut) {
#pragma unroll
    for (int h = 0; h < kH; ++h) parts[warp][h * kOut + lane] = mine[h];
  }
  __syncthreads();
  if (warp % split != 0 || lane >= kOut) return;  // the first of the warps finishes
  float sums[kH] = {};
#pragma unroll
  for (int q = 0; q < split; ++q)
#pragma unroll
    for (int h = 0; h < kH; ++h) sums[h] += parts[warp + q][h * kOut + lane];
  put(lane, sums);
}

template <typename T, int kRows, int kCols, int kUnroll, typename A>
cudaError_t launch(const A& a, bool vec, cudaStream_t stream) {
  const int64_t steps = a.in / (32 * (vec ? 16 / sizeof(T) : 1)), groups = (a.out + kCols - 1) / kCols;
  // Four warps to a weight row where one each would leave half of the GPU's
  // warps idle over rows of eight steps or more (bfloat16, one row of 8192:
  // 1024 weight rows 16 us with one warp, 7 with four; 4096 x 4096 8.4 and 10).
  // The gated operator's warp has two rows to read at a time, and four warps to them
  // are the faster ones up to where each has several (1 x 4096, 2 x 4096 weight rows:
  // 13.2 us, in turn of one step; with one warp to both rows 14.6, in turns of eight 18).
  const bool shared = steps >= 8 && groups < 148 * (kHalves<A> == 2 ? 64 : 16);
  const int64_t per_block = (shared ? kWarps / 4 : kWarps) * kCols;
  const dim3 grid(static_cast<unsigned>((a.out + per_block - 1) / per_block),
                  static_cast<unsigned>((a.rows + kRows - 1) / kRows));
  const auto kernel = shared ? (vec ? gemv_kernel<T, kRows, kCols, kUnroll, 4, true, A>
                                    : gemv_kernel<T, kRows, kCols, kUnroll, 4, false, A>)
                             : (vec ? gemv_kernel<T, kRows, kCols, kUnroll, 1, true, A>
                                    : gemv_kernel<T, kRows, kCols, kUnroll, 1, false, A>);
  kernel<<<grid, 32 * kWarps, 0, stream>>>(a);
  return cudaGetLastError();
}

template <typename T, typename A>
cudaError_t launch_rows(const A& a, cudaStream_t stream) {
  const auto aligned = [](const void* p, int64_t stride) {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (stride * sizeof(T)) % 16 == 0;
  };
  const bool vec = aligned(a.x, a.rows == 1 ? 0 : a.x_stride) && aligned(a.w, kHalves<A> * a.out == 1 ? 0 : a.w_stride) &&
                   (a.in * sizeof(T)) % 16 == 0;
  if (a.rows == 1) return launch<T, 1, 1, kHalves<A> == 2 ? 1 : 4>(a, vec, stream);
  if (a.rows <= 4) return launch<T, 4, 1, 2>(a, vec, stream);
  return launch<T, 8, 2 / kHalves<A>, 2>(a, vec, stream);
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

// The same of the gated operator, whose weight has W = 2 x out x in numbers. bfloat16: one row
// always (4096 x 2 x 4096 13.0 / 20.8, 8192 x 2 x 8192 42.9 / 55.3); two to four while rows x W is
// below 2^27, as the row kernel multiplies on the scalar pipe: 2, 3 and 4 rows of 4096 x 2 x 4096
// 18.0, 19.7 and 21.8 / 20.9, 4 of 4096 x 2 x 2048 13.5 / 14.4, 2 and 4 of 4096 x 2 x 11008 52 and
// 66 / 40; eight of up to 2^21 weights 6.4 / 7.4, of 2^23 16.5 / 11.7. float32 as the plain operator
// of twice the columns: 16 x 4096 x 2 x 4096 103 / 149, 64 x 256 x 2 x 512 7.5 / 15.4, 64 x 1024 x 2 x
// 1024 35 / 21.
// In training, bfloat16's factors share exponents with their neighbours, which other warps hold here.
bool gated_few_rows(const GatedArgs& a) {
  if (a.dtype == DType::kBF16) {
    const int64_t weights = 2 * a.out * a.in;
    return !a.factors && (a.rows == 1 || (a.rows <= 4 && a.rows * weights < 1ll << 27) ||
                          (a.rows <= 8 && weights <= 1ll << 21));
  }
  Args as{};
  as.dtype = a.dtype, as.rows = a.rows, as.in = a.in, as.out = 2 * a.out;
  return few_rows(as);
}

cudaError_t gated_forward_few_rows(const GatedArgs& a, cudaStream_t stream) {
  return a.dtype == DType::kF32 ? launch_rows<float>(a, stream) : launch_rows<bf16>(a, stream);
}

}  // namespace lin
