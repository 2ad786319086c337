// Layer norm over the last dimension, forward and backward.
//
//   mean = sum(x) / n,  rstd = 1 / sqrt(sum((x - mean)^2) / n + eps),  h = (x - mean) rstd
//   y  = h w + b
//   dx = rstd (g w - mean(g w) - h mean(g w h)),  dw = sum over rows of g h,  db = sum over rows of g
//
// Bound by memory: a row is read once into registers (G threads of up to 16
// values each), its statistics are taken there in float32 in two passes (the
// mean first, then the squares of what differs from it, so a large mean costs
// no digits), and it is written once. In the backward pass a thread keeps the
// same columns through all its rows and so sums their dw and db in registers;
// the blocks' sums go to `parts` and a second kernel adds them in order, so the
// gradients do not depend on scheduling. Rows longer than the registers hold
// are read again for each pass, from L2 where they fit.
#include <algorithm>

#include "checkpoint8.cuh"
#include "layer_norm.h"
#include "linear_device.cuh"

namespace lnorm {
namespace {

using lin::bf16;
using lin::from_float;
using lin::to_float;

struct Sums {
  float a, b;
};

__device__ __forceinline__ Sums warp_sums(Sums s) {
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    s.a += __shfl_xor_sync(0xffffffffu, s.a, d);
    s.b += __shfl_xor_sync(0xffffffffu, s.b, d);
  }
  return s;
}

// Sums over the G threads of a row. With more than a warp, `buf` alternates
// between two halves, so one barrier per sum is enough.
template <int G>
__device__ __forceinline__ Sums row_sums(Sums s, Sums* buf, int& turn) {
  s = warp_sums(s);
  if (G == 32) return s;
  constexpr int kWarps = G / 32;
  Sums* half = buf + turn * kWarps;
  turn ^= 1;
  if ((threadIdx.x & 31) == 0) half[threadIdx.x >> 5] = s;
  __syncthreads();
  Sums t = {0.f, 0.f};
#pragma unroll
  for (int w = 0; w < kWarps; ++w) t.a += half[w].a, t.b += half[w].b;
  return t;
}

// The columns of a thread: eight neighbours at a time where vectors fit, else
// one at a time, neighbours in neighbouring threads.
template <int G>
__device__ __forceinline__ int64_t column(bool vec, int lane, int i, int j) {
  return vec ? (static_cast<int64_t>(i) * G + lane) * 8 + j : (static_cast<int64_t>(i) * 8 + j) * G + lane;
}

template <int G, int NV, typename T>
__device__ __forceinline__ void load_row(const T* row, int64_t cols, bool vec, int lane, float v[NV * 8]) {
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (vec) {
      const int64_t c = column<G>(true, lane, i, 0);
      if (c < cols) {
        lin::load8(row + c, v + i * 8);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i * 8 + j] = 0.f;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int64_t c = column<G>(false, lane, i, j);
        v[i * 8 + j] = c < cols ? to_float(row[c]) : 0.f;
      }
    }
  }
}

template <int G, int NV, typename T>
__device__ __forceinline__ void store_row(T* row, int64_t cols, bool vec, int lane, const float v[NV * 8]) {
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (vec) {
      const int64_t c = column<G>(true, lane, i, 0);
      if (c < cols) lin::store8(row + c, v + i * 8);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int64_t c = column<G>(false, lane, i, j);
        if (c < cols) row[c] = from_float<T>(v[i * 8 + j]);
      }
    }
  }
}

// A row of an 8-bit checkpoint. A block of 32 columns is four threads' vectors,
// or one column of a warp's threads.
template <int G, int NV>
__device__ __forceinline__ void load_codes(const int8_t* row, const uint8_t* exps, int64_t cols, bool vec, int lane,
                                           float v[NV * 8]) {
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (vec) {
      const int64_t c = column<G>(true, lane, i, 0);
      if (c < cols) {
        ckpt::load_codes8(row + c, 8, true, exps[c / ckpt::kBlock], v + i * 8);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i * 8 + j] = 0.f;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int64_t c = column<G>(false, lane, i, j);
        v[i * 8 + j] = c < cols ? row[c] * ckpt::scale_of(exps[c / ckpt::kBlock]) : 0.f;
      }
    }
  }
}

template <int G, int NV>
__device__ __forceinline__ void store_codes(int8_t* row, uint8_t* exps, int64_t cols, bool vec, int lane,
                                            const float v[NV * 8]) {
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (vec) {
      const int64_t c = column<G>(true, lane, i, 0);
      uint32_t top = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(v[i * 8 + j]) & 0x7fffffffu);
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const uint32_t e = ckpt::exponent_of(top);
      if (c < cols) {
        ckpt::store_codes8(row + c, 8, true, e, v + i * 8);
        if ((lane & 3) == 0) exps[c / ckpt::kBlock] = static_cast<uint8_t>(e);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int64_t c = column<G>(false, lane, i, j);
        const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(v[i * 8 + j]) & 0x7fffffffu);
        const uint32_t e = ckpt::exponent_of(top);
        if (c < cols) {
          row[c] = static_cast<int8_t>(ckpt::code_of(v[i * 8 + j], e, ckpt::inverse_scale(e)));
          if ((lane & 31) == 0) exps[c / ckpt::kBlock] = static_cast<uint8_t>(e);
        }
      }
    }
  }
}

template <int G, int NV>
__device__ __forceinline__ void statistics(const float v[NV * 8], int64_t cols, bool vec, int lane, float eps,
                                           Sums* buf, int& turn, float& mean, float& rstd) {
  Sums s = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < NV * 8; ++i) s.a += v[i];
  const float n = static_cast<float>(cols);
  mean = row_sums<G>(s, buf, turn).a / n;
  s.a = 0.f;
#pragma unroll
  for (int i = 0; i < NV * 8; ++i) {
    const float d = column<G>(vec, lane, i / 8, i % 8) < cols ? v[i] - mean : 0.f;
    s.a = fmaf(d, d, s.a);
  }
  rstd = rsqrtf(row_sums<G>(s, buf, turn).a / n + eps);
}

// Rows per block and block size for G threads a row.
template <int G>
struct Shape {
  static constexpr int kRows = G == 32 ? 8 : 1;
  static constexpr int kThreads = G * kRows;
  static constexpr int kBuf = G == 32 ? 1 : 2 * (G / 32);
};

template <int G, int NV, typename T, typename W>
__global__ void __launch_bounds__(Shape<G>::kThreads) forward_kernel(const Args a, bool vec) {
  __shared__ Sums buf[Shape<G>::kBuf];
  int turn = 0;
  const int lane = threadIdx.x % G, slot = threadIdx.x / G;
  const T* x = static_cast<const T*>(a.x);
  const W *w = static_cast<const W*>(a.w), *b = static_cast<const W*>(a.b);
  const int64_t blocks = ckpt::blocks_of(a.cols);
  for (int64_t r = blockIdx.x * static_cast<int64_t>(Shape<G>::kRows) + slot; r < a.rows;
       r += static_cast<int64_t>(gridDim.x) * Shape<G>::kRows) {
    float v[NV * 8], p[NV * 8];
    load_row<G, NV>(x + r * a.x_stride, a.cols, vec, lane, v);
    if (a.codes) store_codes<G, NV>(a.codes + r * a.cols, a.exps + r * blocks, a.cols, vec, lane, v);
    float mean, rstd;
    statistics<G, NV>(v, a.cols, vec, lane, a.eps, buf, turn, mean, rstd);
    if (a.mean && lane == 0) {
      a.mean[r] = mean;
      a.rstd[r] = rstd;
    }
#pragma unroll
    for (int i = 0; i < NV * 8; ++i) v[i] = (v[i] - mean) * rstd;
    if (w) {
      load_row<G, NV>(w, a.cols, vec, lane, p);
#pragma unroll
      for (int i = 0; i < NV * 8; ++i) v[i] *= p[i];
    }
    if (b) {
      load_row<G, NV>(b, a.cols, vec, lane, p);
#pragma unroll
      for (int i = 0; i < NV * 8; ++i) v[i] += p[i];
    }
    store_row<G, NV>(static_cast<T*>(a.y) + r * a.cols, a.cols, vec, lane, v);
  }
}

template <int G, int NV, typename T, typename W>
__global__ void __launch_bounds__(Shape<G>::kThreads) backward_kernel(const Args a, bool vec) {
  constexpr int kRows = Shape<G>::kRows;
  __shared__ Sums buf[Shape<G>::kBuf];
  __shared__ float fold[kRows > 1 ? kRows * 32 * 8 : 1];
  int turn = 0;
  const int lane = threadIdx.x % G, slot = threadIdx.x / G;
  const W* w = static_cast<const W*>(a.w);
  const float n = static_cast<float>(a.cols);
  const int64_t blocks = ckpt::blocks_of(a.cols);
  float dw[NV * 8] = {}, db[NV * 8] = {};
  for (int64_t r = blockIdx.x * static_cast<int64_t>(kRows) + slot; r < a.rows;
       r += static_cast<int64_t>(gridDim.x) * kRows) {
    float h[NV * 8], g[NV * 8];
    float mean, rstd;
    load_row<G, NV>(static_cast<const T*>(a.g) + r * a.g_stride, a.cols, vec, lane, g);
    if (a.codes_in) {
      load_codes<G, NV>(a.codes_in + r * a.cols, a.exps_in + r * blocks, a.cols, vec, lane, h);
      statistics<G, NV>(h, a.cols, vec, lane, a.eps, buf, turn, mean, rstd);
    } else {
      load_row<G, NV>(static_cast<const T*>(a.x) + r * a.x_stride, a.cols, vec, lane, h);
      mean = a.mean[r];
      rstd = a.rstd[r];
    }
#pragma unroll
    for (int i = 0; i < NV * 8; ++i) {
      h[i] = (h[i] - mean) * rstd;  // beyond the row g is 0, so h counts for nothing
      dw[i] = fmaf(g[i], h[i], dw[i]);
      db[i] += g[i];
    }
    if (!a.dx) continue;
    if (w) {
      float p[NV * 8];
      load_row<G, NV>(w, a.cols, vec, lane, p);
#pragma unroll
      for (int i = 0; i < NV * 8; ++i) g[i] *= p[i];
    }
    Sums s = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV * 8; ++i) {
      s.a += g[i];
      s.b = fmaf(g[i], h[i], s.b);
    }
    s = row_sums<G>(s, buf, turn);
    const float c1 = s.a / n, c2 = s.b / n;
#pragma unroll
    for (int i = 0; i < NV * 8; ++i) g[i] = rstd * (g[i] - c1 - h[i] * c2);
    store_row<G, NV>(static_cast<T*>(a.dx) + r * a.cols, a.cols, vec, lane, g);
  }
  if (!a.dw && !a.db) return;
  float* part = a.parts + blockIdx.x * 2 * a.cols;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = which ? db[i * 8 + j] : dw[i * 8 + j];
      if (kRows > 1) {  // the block's rows, in order
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 8; ++j) fold[(slot * 8 + j) * 32 + lane] = v[j];
        __syncthreads();
        // thread (slot, lane) adds up column j = slot of lane's eight
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < kRows; ++k) s += fold[(k * 8 + slot) * 32 + lane];
        const int64_t c = column<G>(vec, lane, i, slot);
        if (c < a.cols) part[which * a.cols + c] = s;
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int64_t c = column<G>(vec, lane, i, j);
          if (c < a.cols) part[which * a.cols + c] = v[j];
        }
      }
    }
  }
}

// Rows beyond the registers: a block of 1024 threads a row, the row read again
// for each pass; dw and db are summed in `parts`, whose columns a thread owns.
constexpr int kLong = 1024;

__device__ __forceinline__ float kept(const Args& a, int64_t r, int64_t c) {
  const int64_t blocks = ckpt::blocks_of(a.cols);
  return a.codes_in[r * a.cols + c] * ckpt::scale_of(a.exps_in[r * blocks + c / ckpt::kBlock]);
}

template <typename T>
__device__ __forceinline__ float value_at(const Args& a, int64_t r, int64_t c) {
  return a.codes_in ? kept(a, r, c) : to_float(static_cast<const T*>(a.x)[r * a.x_stride + c]);
}

template <typename T>
__device__ __forceinline__ void long_statistics(const Args& a, int64_t r, Sums* buf, int& turn, float& mean,
                                                float& rstd) {
  const float n = static_cast<float>(a.cols);
  Sums s = {0.f, 0.f};
  for (int64_t c = threadIdx.x; c < a.cols; c += kLong) s.a += value_at<T>(a, r, c);
  mean = row_sums<kLong>(s, buf, turn).a / n;
  s.a = 0.f;
  for (int64_t c = threadIdx.x; c < a.cols; c += kLong) {
    const float d = value_at<T>(a, r, c) - mean;
    s.a = fmaf(d, d, s.a);
  }
  rstd = rsqrtf(row_sums<kLong>(s, buf, turn).a / n + a.eps);
}

template <typename T, typename W>
__global__ void __launch_bounds__(kLong) forward_long_kernel(const Args a) {
  __shared__ Sums buf[2 * kLong / 32];
  int turn = 0;
  const W *w = static_cast<const W*>(a.w), *b = static_cast<const W*>(a.b);
  const int64_t blocks = ckpt::blocks_of(a.cols);
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const T* row = static_cast<const T*>(a.x) + r * a.x_stride;
    float mean, rstd;
    long_statistics<T>(a, r, buf, turn, mean, rstd);
    if (a.mean && threadIdx.x == 0) {
      a.mean[r] = mean;
      a.rstd[r] = rstd;
    }
    for (int64_t c0 = 0; c0 < a.cols; c0 += kLong) {  // whole warps: a warp's columns are a block of 32
      const int64_t c = c0 + threadIdx.x;
      const float v = c < a.cols ? to_float(row[c]) : 0.f;
      if (a.codes) {
        const uint32_t e = ckpt::exponent_of(__reduce_max_sync(0xffffffffu, __float_as_uint(v) & 0x7fffffffu));
        if (c < a.cols) {
          a.codes[r * a.cols + c] = static_cast<int8_t>(ckpt::code_of(v, e, ckpt::inverse_scale(e)));
          if ((threadIdx.x & 31) == 0) a.exps[r * blocks + c / ckpt::kBlock] = static_cast<uint8_t>(e);
        }
      }
      if (c < a.cols) {
        float y = (v - mean) * rstd;
        if (w) y *= to_float(w[c]);
        if (b) y += to_float(b[c]);
        static_cast<T*>(a.y)[r * a.cols + c] = from_float<T>(y);
      }
    }
  }
}

template <typename T, typename W>
__global__ void __launch_bounds__(kLong) backward_long_kernel(const Args a) {
  __shared__ Sums buf[2 * kLong / 32];
  int turn = 0;
  const W* w = static_cast<const W*>(a.w);
  const float n = static_cast<float>(a.cols);
  const bool sums = a.dw || a.db;
  float* part = a.parts + blockIdx.x * 2 * a.cols;
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const T* g = static_cast<const T*>(a.g) + r * a.g_stride;
    float mean, rstd;
    if (a.codes_in) {
      long_statistics<T>(a, r, buf, turn, mean, rstd);
    } else {
      mean = a.mean[r];
      rstd = a.rstd[r];
    }
    Sums s = {0.f, 0.f};
    for (int64_t c = threadIdx.x; c < a.cols; c += kLong) {
      const float h = (value_at<T>(a, r, c) - mean) * rstd, d = to_float(g[c]);
      if (sums) {
        const bool first = r == blockIdx.x;
        part[c] = fmaf(d, h, first ? 0.f : part[c]);
        part[a.cols + c] = d + (first ? 0.f : part[a.cols + c]);
      }
      const float gw = w ? d * to_float(w[c]) : d;
      s.a += gw;
      s.b = fmaf(gw, h, s.b);
    }
    if (!a.dx) continue;
    s = row_sums<kLong>(s, buf, turn);
    const float c1 = s.a / n, c2 = s.b / n;
    for (int64_t c = threadIdx.x; c < a.cols; c += kLong) {
      const float h = (value_at<T>(a, r, c) - mean) * rstd, d = to_float(g[c]);
      const float gw = w ? d * to_float(w[c]) : d;
      static_cast<T*>(a.dx)[r * a.cols + c] = from_float<T>(rstd * (gw - c1 - h * c2));
    }
  }
}

// dw and db from the blocks' parts: a block takes 32 columns of one of them,
// warps take parts in turn.
template <typename W>
__global__ void __launch_bounds__(1024)
    add_parts_kernel(const float* __restrict__ parts, int count, int64_t cols, W* dw, W* db) {
  __shared__ float buf[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c = blockIdx.x * 32ll + lane;
  W* out = blockIdx.y ? db : dw;
  if (!out) return;
  float s = 0.f;
  if (c < cols)
    for (int i = warp; i < count; i += 32) s += parts[(2ll * i + blockIdx.y) * cols + c];
  buf[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && c < cols) {
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) s += buf[i][lane];
    out[c] = from_float<W>(s);
  }
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <typename T, typename W>
bool vectors_fit(const Args& a, bool backward) {
  bool ok = a.cols % 8 == 0 && aligned16(a.w) && aligned16(a.b);
  if (backward) {
    ok = ok && aligned16(a.g) && (a.g_stride * sizeof(T)) % 16 == 0 && aligned16(a.dx);
    ok = ok && (a.codes_in ? (reinterpret_cast<uintptr_t>(a.codes_in) & 7) == 0
                           : aligned16(a.x) && (a.x_stride * sizeof(T)) % 16 == 0);
  } else {
    ok = ok && aligned16(a.x) && (a.x_stride * sizeof(T)) % 16 == 0 && aligned16(a.y) &&
         (reinterpret_cast<uintptr_t>(a.codes) & 7) == 0;
  }
  return ok;
}

constexpr int64_t kMaxRegisters = 16384;

// Threads a row: as few as hold it in 16 values each.
int threads_for(int64_t cols) { return cols <= 512 ? 32 : cols <= 2048 ? 128 : cols <= 8192 ? 512 : 1024; }

template <typename T, typename W, int G, int NV>
cudaError_t launch(const Args& a, bool backward, int grid, bool vec, cudaStream_t stream) {
  if (backward)
    backward_kernel<G, NV, T, W><<<grid, Shape<G>::kThreads, 0, stream>>>(a, vec);
  else
    forward_kernel<G, NV, T, W><<<grid, Shape<G>::kThreads, 0, stream>>>(a, vec);
  return cudaGetLastError();
}

template <typename T, typename W>
cudaError_t dispatch(const Args& a, bool backward, cudaStream_t stream) {
  const int grid =
      backward ? backward_parts(a.rows, a.cols)
               : static_cast<int>(std::min<int64_t>(a.cols <= 512 ? (a.rows + 7) / 8 : a.rows, 148 * 64));
  const bool vec = vectors_fit<T, W>(a, backward);
  if (a.cols > kMaxRegisters) {
    if (backward)
      backward_long_kernel<T, W><<<grid, kLong, 0, stream>>>(a);
    else
      forward_long_kernel<T, W><<<grid, kLong, 0, stream>>>(a);
    return cudaGetLastError();
  }
  const int g = threads_for(a.cols);
  const bool one = a.cols <= 8ll * g;
  if (g == 32) return one ? launch<T, W, 32, 1>(a, backward, grid, vec, stream) : launch<T, W, 32, 2>(a, backward, grid, vec, stream);
  if (g == 128) return one ? launch<T, W, 128, 1>(a, backward, grid, vec, stream) : launch<T, W, 128, 2>(a, backward, grid, vec, stream);
  if (g == 512) return one ? launch<T, W, 512, 1>(a, backward, grid, vec, stream) : launch<T, W, 512, 2>(a, backward, grid, vec, stream);
  return launch<T, W, 1024, 2>(a, backward, grid, vec, stream);
}

cudaError_t dispatch_types(const Args& a, bool backward, cudaStream_t stream) {
  if (a.dtype == DType::kF32) return dispatch<float, float>(a, backward, stream);
  if (a.weight_dtype == DType::kF32) return dispatch<bf16, float>(a, backward, stream);
  return dispatch<bf16, bf16>(a, backward, stream);
}

}  // namespace

int backward_parts(int64_t rows, int64_t cols) {
  const int64_t groups = cols <= 512 ? (rows + 7) / 8 : rows;
  const int per_sm = cols <= 512 ? 4 : cols <= 2048 ? 4 : 1;
  return static_cast<int>(std::min<int64_t>(groups, 148 * per_sm));
}

cudaError_t forward(const Args& a, cudaStream_t stream) {
  return a.rows == 0 || a.cols == 0 ? cudaSuccess : dispatch_types(a, false, stream);
}

cudaError_t backward(const Args& a, cudaStream_t stream) {
  if (a.cols == 0) return cudaSuccess;
  if (a.rows > 0) {
    const cudaError_t err = dispatch_types(a, true, stream);
    if (err != cudaSuccess) return err;
  }
  if (!a.dw && !a.db) return cudaSuccess;
  const dim3 grid(static_cast<unsigned>((a.cols + 31) / 32), 2);
  const int count = backward_parts(a.rows, a.cols);
  if (a.weight_dtype == DType::kF32)
    add_parts_kernel<<<grid, 1024, 0, stream>>>(a.parts, count, a.cols, static_cast<float*>(a.dw),
                                               static_cast<float*>(a.db));
  else
    add_parts_kernel<<<grid, 1024, 0, stream>>>(a.parts, count, a.cols, static_cast<bf16*>(a.dw),
                                               static_cast<bf16*>(a.db));
  return cudaGetLastError();
}

}  // namespace lnorm
