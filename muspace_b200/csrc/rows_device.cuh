// Device code of kernels that hold a row in the registers of G threads: sums over
// a row, the columns of a thread, and loads and stores of them. Shared by the norms.
#pragma once

#include <stdint.h>

#include "linear_device.cuh"

namespace rows {

using lin::from_float;
using lin::to_float;

struct Sums {
  float a, b;
};

// Over N neighbouring lanes.
template <int N = 32>
__device__ __forceinline__ Sums warp_sums(Sums s) {
#pragma unroll
  for (int d = N / 2; d; d >>= 1) {
    s.a += __shfl_xor_sync(0xffffffffu, s.a, d);
    s.b += __shfl_xor_sync(0xffffffffu, s.b, d);
  }
  return s;
}
template <int N = 32>
__device__ __forceinline__ float warp_sums(float s) {
#pragma unroll
  for (int d = N / 2; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
  return s;
}
__device__ __forceinline__ Sums operator+(Sums s, Sums t) { return Sums{s.a + t.a, s.b + t.b}; }

// Sums over the G threads of a row. With more than a warp, `buf` alternates
// between two halves, so one barrier per sum is enough.
template <int G, bool kNamed = false, typename S>
__device__ __forceinline__ S row_sums(S s, Sums* buf, int& turn) {
  s = warp_sums<(G < 32 ? G : 32)>(s);
  if (G <= 32) return s;
  constexpr int kWarps = G <= 32 ? 1 : G / 32;
  S* half = reinterpret_cast<S*>(buf + turn * kWarps);
  turn ^= 1;
  if ((threadIdx.x & 31) == 0) half[(threadIdx.x % G) >> 5] = s;
  if (kNamed)  // one of several groups of G threads in the block
    asm volatile("bar.sync %0, %1;" ::"r"(static_cast<int>(threadIdx.x / G) + 1), "n"(G) : "memory");
  else
    __syncthreads();
  S t = half[0];
#pragma unroll
  for (int w = 1; w < kWarps; ++w) t = t + half[w];
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
  __device__ __forceinline__ void get(float2 v[4]) const { lin::load8(reinterpret_cast<const T*>(u), &v[0].x); }
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
  __device__ __forceinline__ void get(float2 w[4]) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = make_float2(v[2 * j], v[2 * j + 1]);
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

// Rows per block and block size for G threads a row.
template <int G>
struct Shape {
  static constexpr int kRows = G <= 32 ? 256 / G : 1;
  static constexpr int kThreads = G * kRows;
  static constexpr int kBuf = G <= 32 ? 1 : 2 * (G / 32);
};

}  // namespace rows
