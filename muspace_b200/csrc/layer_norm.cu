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

// The columns of a thread, eight to a chunk: neighbours where vectors fit
// (kVec), else one at a time, neighbours in neighbouring threads.
template <int G, bool kVec>
__device__ __forceinline__ int column(int lane, int i, int j) {
  return kVec ? (i * G + lane) * 8 + j : (i * 8 + j) * G + lane;
}

// Eight values as they lie in memory: they stay so in registers until they are
// used, so that more rows are on their way.
template <typename T, bool kVec>
struct Chunk {
  uint4 u[sizeof(T) / 2];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int k = 0; k < static_cast<int>(sizeof(T) / 2); ++k) u[k] = make_uint4(0, 0, 0, 0);
  }
  template <int G>
  __device__ __forceinline__ void load(const T* row, int cols, int lane, int i) {
    const int c = column<G, true>(lane, i, 0);
    if (c < cols) {
#pragma unroll
      for (int k = 0; k < static_cast<int>(sizeof(T) / 2); ++k) u[k] = __ldg(reinterpret_cast<const uint4*>(row + c) + k);
    } else {
      zero();
    }
  }
  __device__ __forceinline__ void get(float v[8]) const { lin::load8(reinterpret_cast<const T*>(u), v); }
};
template <typename T>
struct Chunk<T, false> {
  float v[8];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = 0.f;
  }
  template <int G>
  __device__ __forceinline__ void load(const T* row, int cols, int lane, int i) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = column<G, false>(lane, i, j);
      v[j] = c < cols ? to_float(row[c]) : 0.f;
    }
  }
  __device__ __forceinline__ void get(float w[8]) const {
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = v[j];
  }
};

// The same of an 8-bit checkpoint.
template <bool kVec>
struct Codes {
  uint2 u;
  uint32_t e;
  template <int G>
  __device__ __forceinline__ void load(const int8_t* row, const uint8_t* exps, int cols, int lane, int i) {
    const int c = column<G, true>(lane, i, 0);
    u = make_uint2(0, 0);
    e = 1;
    if (c < cols) {
      u = __ldg(reinterpret_cast<const uint2*>(row + c));
      e = __ldg(exps + c / ckpt::kBlock);
    }
  }
  __device__ __forceinline__ void get(float v[8]) const { ckpt::values_of(u, e, v); }
};
template <>
struct Codes<false> {
  float v[8];
  template <int G>
  __device__ __forceinline__ void load(const int8_t* row, const uint8_t* exps, int cols, int lane, int i) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = column<G, false>(lane, i, j);
      v[j] = c < cols ? row[c] * ckpt::scale_of(exps[c / ckpt::kBlock]) : 0.f;
    }
  }
  __device__ __forceinline__ void get(float w[8]) const {
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = v[j];
  }
};

template <int G, bool kVec, typename T>
__device__ __forceinline__ void store_chunk(T* row, int cols, int lane, int i, const float v[8]) {
  if (kVec) {
    const int c = column<G, true>(lane, i, 0);
    if (c < cols) lin::store8(row + c, v);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = column<G, false>(lane, i, j);
      if (c < cols) row[c] = from_float<T>(v[j]);
    }
  }
}

// A chunk into the checkpoint. A block of 32 columns is four threads' chunks,
// or one column of a warp's threads.
template <int G, bool kVec>
__device__ __forceinline__ void store_codes(int8_t* row, uint8_t* exps, int cols, int lane, int i, const float v[8]) {
  if (kVec) {
    const int c = column<G, true>(lane, i, 0);
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const uint32_t e = ckpt::exponent_of(top);
    if (c < cols) {
      ckpt::store_codes8(row + c, 8, true, e, v);
      if ((lane & 3) == 0) exps[c / ckpt::kBlock] = static_cast<uint8_t>(e);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = column<G, false>(lane, i, j);
      const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(v[j]) & 0x7fffffffu);
      const uint32_t e = ckpt::exponent_of(top);
      if (c < cols) {
        row[c] = static_cast<int8_t>(ckpt::code_of(v[j], e, ckpt::inverse_scale(e)));
        if ((lane & 31) == 0) exps[c / ckpt::kBlock] = static_cast<uint8_t>(e);
      }
    }
  }
}

template <int G, int NV, bool kVec, typename C>
__device__ __forceinline__ void statistics(const C x[NV], int cols, int lane, float eps, Sums* buf, int& turn,
                                           float& mean, float& rstd) {
  Sums s = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    float v[8];
    x[i].get(v);
#pragma unroll
    for (int j = 0; j < 8; ++j) s.a += v[j];
  }
  const float n = static_cast<float>(cols);
  mean = row_sums<G>(s, buf, turn).a / n;
  s.a = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    float v[8];
    x[i].get(v);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float d = column<G, kVec>(lane, i, kVec ? 0 : j) < cols ? v[j] - mean : 0.f;
      s.a = fmaf(d, d, s.a);
    }
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

template <int G, int NV, bool kVec, bool kCodes, typename T, typename W>
__global__ void __launch_bounds__(Shape<G>::kThreads) forward_kernel(const Args a) {
  __shared__ Sums buf[Shape<G>::kBuf];
  int turn = 0;
  const int lane = threadIdx.x % G, cols = static_cast<int>(a.cols);
  const int64_t step = static_cast<int64_t>(gridDim.x) * Shape<G>::kRows, blocks = ckpt::blocks_of(a.cols);
  const T* x = static_cast<const T*>(a.x);
  int64_t r = blockIdx.x * static_cast<int64_t>(Shape<G>::kRows) + threadIdx.x / G;
  Chunk<T, kVec> next[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (r < a.rows) next[i].template load<G>(x + r * a.x_stride, cols, lane, i);
  for (; r < a.rows; r += step) {
    Chunk<T, kVec> here[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) here[i] = next[i];
    if (r + step < a.rows) {
#pragma unroll
      for (int i = 0; i < NV; ++i) next[i].template load<G>(x + (r + step) * a.x_stride, cols, lane, i);
    }
    float mean, rstd;
    statistics<G, NV, kVec>(here, cols, lane, a.eps, buf, turn, mean, rstd);
    if (a.mean && lane == 0) {
      a.mean[r] = mean;
      a.rstd[r] = rstd;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float v[8], p[8];
      here[i].get(v);
      if (kCodes) store_codes<G, kVec>(a.codes + r * a.cols, a.exps + r * blocks, cols, lane, i, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = (v[j] - mean) * rstd;
      if (a.w) {
        Chunk<W, kVec> w;
        w.template load<G>(static_cast<const W*>(a.w), cols, lane, i);
        w.get(p);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] *= p[j];
      }
      if (a.b) {
        Chunk<W, kVec> b;
        b.template load<G>(static_cast<const W*>(a.b), cols, lane, i);
        b.get(p);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] += p[j];
      }
      store_chunk<G, kVec>(static_cast<T*>(a.y) + r * a.cols, cols, lane, i, v);
    }
  }
}

// The input of the backward pass: x, or what a checkpoint holds of it.
template <int G, int NV, bool kVec, bool kCodes, typename T>
struct Input {
  Chunk<T, kVec> x[NV];
  float mean, rstd;
  __device__ __forceinline__ void load(const Args& a, int64_t r, int cols, int lane) {
    mean = a.mean[r];
    rstd = a.rstd[r];
#pragma unroll
    for (int i = 0; i < NV; ++i)
      x[i].template load<G>(static_cast<const T*>(a.x) + r * a.x_stride, cols, lane, i);
  }
  __device__ __forceinline__ void prepare(const Args&, int, int, Sums*, int&) {}
};
template <int G, int NV, bool kVec, typename T>
struct Input<G, NV, kVec, true, T> {
  Codes<kVec> x[NV];
  float mean, rstd;
  __device__ __forceinline__ void load(const Args& a, int64_t r, int cols, int lane) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      x[i].template load<G>(a.codes_in + r * a.cols, a.exps_in + r * ckpt::blocks_of(a.cols), cols, lane, i);
  }
  __device__ __forceinline__ void prepare(const Args& a, int cols, int lane, Sums* buf, int& turn) {
    statistics<G, NV, kVec>(x, cols, lane, a.eps, buf, turn, mean, rstd);
  }
};

template <int G, int NV, bool kVec, bool kCodes, typename T, typename W>
__global__ void __launch_bounds__(Shape<G>::kThreads) backward_kernel(const Args a) {
  constexpr int kRows = Shape<G>::kRows;
  __shared__ Sums buf[Shape<G>::kBuf];
  __shared__ float fold[kRows > 1 ? kRows * 32 * 8 : 1];
  int turn = 0;
  const int lane = threadIdx.x % G, slot = threadIdx.x / G, cols = static_cast<int>(a.cols);
  const int64_t step = static_cast<int64_t>(gridDim.x) * kRows;
  const T* gradient = static_cast<const T*>(a.g);
  const float n = static_cast<float>(a.cols);
  float dw[NV * 8] = {}, db[NV * 8] = {};
  Input<G, NV, kVec, kCodes, T> next, here;
  Chunk<T, kVec> next_g[NV], g[NV];
  int64_t r = blockIdx.x * static_cast<int64_t>(kRows) + slot;
  const auto load = [&](int64_t row) {
    next.load(a, row, cols, lane);
#pragma unroll
    for (int i = 0; i < NV; ++i) next_g[i].template load<G>(gradient + row * a.g_stride, cols, lane, i);
  };
  if (r < a.rows) load(r);
  for (; r < a.rows; r += step) {
    here = next;
#pragma unroll
    for (int i = 0; i < NV; ++i) g[i] = next_g[i];
    if (r + step < a.rows) load(r + step);
    here.prepare(a, cols, lane, buf, turn);
    Sums s = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float h[8], d[8], p[8];
      here.x[i].get(h);
      g[i].get(d);
      if (a.w) {
        Chunk<W, kVec> w;
        w.template load<G>(static_cast<const W*>(a.w), cols, lane, i);
        w.get(p);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float x = (h[j] - here.mean) * here.rstd;  // beyond the row the gradient is 0, and counts for nothing
        dw[i * 8 + j] = fmaf(d[j], x, dw[i * 8 + j]);
        db[i * 8 + j] += d[j];
        const float gw = a.w ? d[j] * p[j] : d[j];
        s.a += gw;
        s.b = fmaf(gw, x, s.b);
      }
    }
    if (!a.dx) continue;
    s = row_sums<G>(s, buf, turn);
    const float c1 = s.a / n, c2 = s.b / n;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float h[8], d[8], p[8];
      here.x[i].get(h);
      g[i].get(d);
      if (a.w) {
        Chunk<W, kVec> w;
        w.template load<G>(static_cast<const W*>(a.w), cols, lane, i);
        w.get(p);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float x = (h[j] - here.mean) * here.rstd;
        d[j] = here.rstd * ((a.w ? d[j] * p[j] : d[j]) - c1 - x * c2);
      }
      store_chunk<G, kVec>(static_cast<T*>(a.dx) + r * a.cols, cols, lane, i, d);
    }
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
        float sum = 0.f;
#pragma unroll
        for (int k = 0; k < kRows; ++k) sum += fold[(k * 8 + slot) * 32 + lane];
        const int c = column<G, kVec>(lane, i, slot);
        if (c < cols) part[which * a.cols + c] = sum;
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int c = column<G, kVec>(lane, i, j);
          if (c < cols) part[which * a.cols + c] = v[j];
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

// Threads a row and chunks a thread. A backward pass also sums 16 floats a chunk, so it takes fewer.
struct Form {
  int threads, chunks;
};
Form forward_form(int64_t rows, int64_t cols) {
  if (cols <= 1024) return {32, cols <= 256 ? 1 : cols <= 512 ? 2 : 4};
  if (rows < 296 && cols <= 4096) return {512, 1};  // few rows: short ones in time, not many in flight
  return cols <= 4096 ? Form{128, 4} : cols <= 8192 ? Form{256, 4} : cols <= 16384 ? Form{512, 4} : Form{kLong, 0};
}
Form backward_form(int64_t cols) {
  if (cols <= 512) return {32, cols <= 256 ? 1 : 2};
  return cols <= 2048 ? Form{128, 2} : cols <= 4096 ? Form{256, 2} : cols <= 8192 ? Form{512, 2} : Form{kLong, 0};
}

int blocks_of_rows(int64_t rows, const Form& f, int per_sm) {
  const int64_t groups = f.threads == 32 ? (rows + 7) / 8 : rows;
  return static_cast<int>(std::min<int64_t>(groups, 148ll * per_sm));
}

template <typename T, typename W, int G, int NV, bool kVec, bool kCodes>
cudaError_t launch_forward(const Args& a, cudaStream_t stream) {
  const int per_sm = std::max(1, 2048 / Shape<G>::kThreads / 2);
  const int grid = blocks_of_rows(a.rows, Form{G, NV}, per_sm);
  forward_kernel<G, NV, kVec, kCodes, T, W><<<grid, Shape<G>::kThreads, 0, stream>>>(a);
  return cudaGetLastError();
}

template <typename T, typename W, bool kVec, bool kCodes>
cudaError_t dispatch_forward(const Args& a, cudaStream_t stream) {
  const Form f = forward_form(a.rows, a.cols);
  if (f.threads == 32)
    return !kVec || f.chunks == 4 ? launch_forward<T, W, 32, 4, kVec, kCodes>(a, stream)
           : f.chunks == 2        ? launch_forward<T, W, 32, kVec ? 2 : 4, kVec, kCodes>(a, stream)
                                  : launch_forward<T, W, 32, kVec ? 1 : 4, kVec, kCodes>(a, stream);
  if (f.threads == 512)
    return f.chunks == 1 ? launch_forward<T, W, 512, 1, kVec, kCodes>(a, stream)
                         : launch_forward<T, W, 512, 4, kVec, kCodes>(a, stream);
  return f.threads == 128 && kVec ? launch_forward<T, W, kVec ? 128 : 256, 4, kVec, kCodes>(a, stream)
                                  : launch_forward<T, W, 256, 4, kVec, kCodes>(a, stream);
}

template <typename T, typename W, int G, int NV, bool kVec, bool kCodes>
cudaError_t launch_backward(const Args& a, cudaStream_t stream) {
  backward_kernel<G, NV, kVec, kCodes, T, W>
      <<<backward_parts(a.rows, a.cols), Shape<G>::kThreads, 0, stream>>>(a);
  return cudaGetLastError();
}

template <typename T, typename W, bool kVec, bool kCodes>
cudaError_t dispatch_backward(const Args& a, cudaStream_t stream) {
  const Form f = backward_form(a.cols);
  if (f.threads == 32)
    return f.chunks == 1 && kVec ? launch_backward<T, W, 32, kVec ? 1 : 2, kVec, kCodes>(a, stream)
                                 : launch_backward<T, W, 32, 2, kVec, kCodes>(a, stream);
  if (f.threads == 512) return launch_backward<T, W, 512, 2, kVec, kCodes>(a, stream);
  return f.threads == 128 ? launch_backward<T, W, 128, 2, kVec, kCodes>(a, stream)
                          : launch_backward<T, W, 256, 2, kVec, kCodes>(a, stream);
}

template <typename T, typename W>
cudaError_t dispatch(const Args& a, bool backward, cudaStream_t stream) {
  const bool vec = vectors_fit<T, W>(a, backward);
  if (backward) {
    if (backward_form(a.cols).threads == kLong) {
      backward_long_kernel<T, W><<<backward_parts(a.rows, a.cols), kLong, 0, stream>>>(a);
      return cudaGetLastError();
    }
    if (a.codes_in)
      return vec ? dispatch_backward<T, W, true, true>(a, stream) : dispatch_backward<T, W, false, true>(a, stream);
    return vec ? dispatch_backward<T, W, true, false>(a, stream) : dispatch_backward<T, W, false, false>(a, stream);
  }
  if (forward_form(a.rows, a.cols).threads == kLong) {
    forward_long_kernel<T, W><<<blocks_of_rows(a.rows, Form{kLong, 0}, 2), kLong, 0, stream>>>(a);
    return cudaGetLastError();
  }
  if (a.codes)
    return vec ? dispatch_forward<T, W, true, true>(a, stream) : dispatch_forward<T, W, false, true>(a, stream);
  return vec ? dispatch_forward<T, W, true, false>(a, stream) : dispatch_forward<T, W, false, false>(a, stream);
}

cudaError_t dispatch_types(const Args& a, bool backward, cudaStream_t stream) {
  if (a.dtype == DType::kF32) return dispatch<float, float>(a, backward, stream);
  if (a.weight_dtype == DType::kF32) return dispatch<bf16, float>(a, backward, stream);
  return dispatch<bf16, bf16>(a, backward, stream);
}

}  // namespace

int backward_parts(int64_t rows, int64_t cols) {
  const Form f = backward_form(cols);
  return blocks_of_rows(rows, f, f.threads == 32 ? 3 : f.threads == 128 ? 4 : f.threads == 256 ? 2 : 1);
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
