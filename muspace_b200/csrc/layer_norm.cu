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

#include "async_device.cuh"
#include "checkpoint8.cuh"
#include "layer_norm.h"
#include "rows_device.cuh"

namespace lnorm {
namespace {

using lin::add2;
using lin::bf16;
using lin::both;
using lin::fma2;
using lin::from_float;
using lin::mul2;
using lin::to_float;
using rows::Chunk;
using rows::column;
using rows::row_sums;
using rows::Shape;
using rows::store_chunk;
using rows::Sums;

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
  __device__ __forceinline__ void get(float2 v[4]) const { ckpt::values_of(u, e, &v[0].x); }
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
  __device__ __forceinline__ void get(float2 w[4]) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = make_float2(v[2 * j], v[2 * j + 1]);
  }
};

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
  float2 t = both(0.f);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    float2 v[4];
    x[i].get(v);
#pragma unroll
    for (int j = 0; j < 4; ++j) t = add2(t, v[j]);
  }
  const float n = static_cast<float>(cols);
  mean = row_sums<G>(t.x + t.y, buf, turn) / n;
  const float2 minus = both(-mean);
  t = both(0.f);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (kVec && column<G, true>(lane, i, 0) >= cols) continue;
    float2 v[4];
    x[i].get(v);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float2 d = add2(v[j], minus);
      if (!kVec) {
        if (column<G, false>(lane, i, 2 * j) >= cols) d.x = 0.f;
        if (column<G, false>(lane, i, 2 * j + 1) >= cols) d.y = 0.f;
      }
      t = fma2(d, d, t);
    }
  }
  rstd = rsqrtf(row_sums<G>(t.x + t.y, buf, turn) / n + eps);
}

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
    const float2 scale = both(rstd), minus = both(-mean);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float2 v[4], p[4];
      here[i].get(v);
      if (kCodes) store_codes<G, kVec>(a.codes + r * a.cols, a.exps + r * blocks, cols, lane, i, &v[0].x);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = mul2(add2(v[j], minus), scale);
      if (a.w) {
        Chunk<W, kVec> w;
        w.template load<G>(static_cast<const W*>(a.w), cols, lane, i);
        w.get(p);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = mul2(v[j], p[j]);
      }
      if (a.b) {
        Chunk<W, kVec> b;
        b.template load<G>(static_cast<const W*>(a.b), cols, lane, i);
        b.get(p);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = add2(v[j], p[j]);
      }
      store_chunk<G, kVec>(static_cast<T*>(a.y) + r * a.cols, cols, lane, i, &v[0].x);
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

// Blocks of the register kernels that an SM holds; as many are launched, so that all
// rows are under way at once. The ring kernel gets the same number, and an SM holds
// one block of it: for 2049 to 4096 columns that makes two waves.
constexpr int backward_blocks(int threads) {
  return threads == 32 ? 3 : threads == 128 ? 4 : threads == 256 ? 2 : 1;
}

template <int G, int NV, bool kVec, bool kCodes, typename T, typename W>
__global__ void __launch_bounds__(Shape<G>::kThreads, G == 32 && (NV > 1 || !kVec) ? 2 : backward_blocks(G))
    backward_kernel(const Args a) {
  constexpr int kRows = Shape<G>::kRows;
  __shared__ Sums buf[Shape<G>::kBuf];
  __shared__ float fold[kRows > 1 ? kRows * 32 * 8 : 1];
  int turn = 0;
  const int lane = threadIdx.x % G, slot = threadIdx.x / G, cols = static_cast<int>(a.cols);
  const int64_t step = static_cast<int64_t>(gridDim.x) * kRows;
  const T* gradient = static_cast<const T*>(a.g);
  const float n = static_cast<float>(a.cols);
  float2 dw[NV][4] = {}, db[NV][4] = {};
  Input<G, NV, kVec, kCodes, T> next, here;
  Chunk<T, kVec> next_g[NV], g[NV];
  int64_t r = blockIdx.x * static_cast<int64_t>(kRows) + slot;
  const auto load = [&](int64_t row) {
    next.load(a, row, cols, lane);
#pragma unroll
    for (int i = 0; i < NV; ++i) next_g[i].template load<G>(gradient + row * a.g_stride, cols, lane, i);
  };
  const auto weight = [&](int i, float2 p[4]) {
    Chunk<W, kVec> w;
    w.template load<G>(static_cast<const W*>(a.w), cols, lane, i);
    w.get(p);
  };
  if (r < a.rows) load(r);
  for (; r < a.rows; r += step) {
    here = next;
#pragma unroll
    for (int i = 0; i < NV; ++i) g[i] = next_g[i];
    if (r + step < a.rows) load(r + step);
    here.prepare(a, cols, lane, buf, turn);
    const float2 scale = both(here.rstd), minus = both(-here.mean);
    float2 sum = both(0.f), dot = both(0.f);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float2 h[4], d[4], p[4];
      here.x[i].get(h);
      g[i].get(d);
      if (a.w) weight(i, p);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        h[j] = mul2(add2(h[j], minus), scale);  // beyond the row the gradient is 0, and counts for nothing
        dw[i][j] = fma2(d[j], h[j], dw[i][j]);
        db[i][j] = add2(db[i][j], d[j]);
        if (a.w) d[j] = mul2(d[j], p[j]);
        sum = add2(sum, d[j]);
        dot = fma2(d[j], h[j], dot);
      }
    }
    if (!a.dx) continue;
    const Sums s = row_sums<G>(Sums{sum.x + sum.y, dot.x + dot.y}, buf, turn);
    // rstd (g w - mean(g w) - h mean(g w h)), with h = (x - mean) rstd
    const float2 c1 = both(-here.rstd * (s.a / n)), c2 = both(-here.rstd * here.rstd * (s.b / n));  // of x - mean
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float2 h[4], d[4], p[4];
      here.x[i].get(h);
      g[i].get(d);
      if (a.w) weight(i, p);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (a.w) d[j] = mul2(d[j], p[j]);
        d[j] = fma2(add2(h[j], minus), c2, fma2(d[j], scale, c1));
      }
      store_chunk<G, kVec>(static_cast<T*>(a.dx) + r * a.cols, cols, lane, i, &d[0].x);
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
      for (int j = 0; j < 4; ++j) {
        v[2 * j] = which ? db[i][j].x : dw[i][j].x;
        v[2 * j + 1] = which ? db[i][j].y : dw[i][j].y;
      }
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

// The backward pass of long rows. A row's sums need a barrier in its middle, and
// registers hold no more than the next row meanwhile (8192 columns of bfloat16:
// 129 us for 8192 rows); so here the rows' data comes to shared memory by bulk
// copies, several rows ahead, and is read from there twice. Two groups of 256
// threads take rows in turn, so that one computes while the other waits at its
// barrier (one group of 512: 113 us; two: 89, 403 MB in and out at 4.5 TB/s). A
// group's stage is free again when its next row's barrier has been passed.
constexpr int kRingThreads = 512, kGroup = 256;
constexpr int kRingBytes = 192 * 1024;
constexpr int kMaxStages = 8;

template <int NV, bool kCodes, typename T, typename W>
__global__ void __launch_bounds__(kRingThreads, 1) backward_ring_kernel(const Args a, int stages) {
  constexpr int G = kGroup, kGroups = kRingThreads / kGroup;
  extern __shared__ __align__(16) uint8_t ring[];  // stages of x (or codes) and g, `stages` for each group
  __shared__ Sums bufs[kGroups][2 * (G / 32)];
  __shared__ __align__(8) uint64_t bars[kGroups][kMaxStages];
  int turn = 0;
  const int lane = threadIdx.x % G, group = threadIdx.x / G, cols = static_cast<int>(a.cols);
  const T* gradient = static_cast<const T*>(a.g);
  const float n = static_cast<float>(a.cols);
  const uint32_t x_bytes = cols * (kCodes ? 1 : sizeof(T)), g_bytes = cols * sizeof(T);
  const uint32_t stage_bytes = x_bytes + g_bytes;
  const int64_t blocks = ckpt::blocks_of(a.cols);
  Sums* buf = bufs[group];
  const uint8_t* mine = ring + group * stages * stage_bytes;
  const uint32_t bar0 = async::smem_addr(bars[group]), ring0 = async::smem_addr(mine);
  if (lane == 0) {
    for (int s = 0; s < stages; ++s) async::barrier_init(bar0 + 8 * s, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  uint32_t fetched = 0;  // by this thread, into the stages in turn
  const auto fetch = [&](int64_t r, int s) {
    ++fetched;
    const uint32_t bar = bar0 + 8 * s, dst = ring0 + s * stage_bytes;
    async::expect_bytes(bar, stage_bytes);
    async::copy_bytes(dst, kCodes ? static_cast<const void*>(a.codes_in + r * a.cols)
                                  : static_cast<const void*>(static_cast<const T*>(a.x) + r * a.x_stride),
                      x_bytes, bar);
    async::copy_bytes(dst + x_bytes, gradient + r * a.g_stride, g_bytes, bar);
  };
  const int64_t step = static_cast<int64_t>(gridDim.x) * kGroups, first = blockIdx.x + static_cast<int64_t>(group) * gridDim.x;
  if (lane == 0)
    for (int s = 0; s < stages; ++s)
      if (first + s * step < a.rows) fetch(first + s * step, s);
  const auto weight = [&](int i, float2 p[4]) {
    Chunk<W, true> w;
    w.template load<G>(static_cast<const W*>(a.w), cols, lane, i);
    w.get(p);
  };
  float2 dw[NV][4] = {}, db[NV][4] = {};
  int stage = 0, last = -1;
  uint32_t phase = 0;
  bool dead = false;
  for (int64_t r = first; r < a.rows; r += step) {
    const uint8_t* at = mine + stage * stage_bytes;
    const T* g_row = reinterpret_cast<const T*>(at + x_bytes);
    uint32_t exps[NV];
    if (kCodes) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = column<G, true>(lane, i, 0);
        exps[i] = c < cols ? __ldg(a.exps_in + r * blocks + c / ckpt::kBlock) : 1u;
      }
    }
    async::wait(bar0 + 8 * stage, phase, dead);
    const auto x_at = [&](int i, float2 v[4]) {
      const int c = column<G, true>(lane, i, 0);
      if (kCodes) {
        ckpt::values_of(*reinterpret_cast<const uint2*>(at + c), exps[i], &v[0].x);
      } else {
        lin::load8(reinterpret_cast<const T*>(at) + c, &v[0].x);
      }
    };
    const auto g_at = [&](int i, float2 v[4]) { lin::load8(g_row + column<G, true>(lane, i, 0), &v[0].x); };
    const auto beyond = [&](int i) { return column<G, true>(lane, i, 0) >= cols; };
    float mean, rstd;
    if (kCodes) {
      float2 t = both(0.f);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (beyond(i)) continue;
        float2 v[4];
        x_at(i, v);
#pragma unroll
        for (int j = 0; j < 4; ++j) t = add2(t, v[j]);
      }
      mean = row_sums<G, true>(t.x + t.y, buf, turn) / n;
      t = both(0.f);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (beyond(i)) continue;
        float2 v[4];
        x_at(i, v);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v[j] = add2(v[j], both(-mean));
          t = fma2(v[j], v[j], t);
        }
      }
      rstd = rsqrtf(row_sums<G, true>(t.x + t.y, buf, turn) / n + a.eps);
    } else {
      mean = __ldg(a.mean + r);
      rstd = __ldg(a.rstd + r);
    }
    const float2 scale = both(rstd), minus = both(-mean);
    float2 sum = both(0.f), dot = both(0.f);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (beyond(i)) continue;
      float2 h[4], d[4], p[4];
      x_at(i, h);
      g_at(i, d);
      if (a.w) weight(i, p);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        h[j] = mul2(add2(h[j], minus), scale);
        dw[i][j] = fma2(d[j], h[j], dw[i][j]);
        db[i][j] = add2(db[i][j], d[j]);
        if (a.w) d[j] = mul2(d[j], p[j]);
        sum = add2(sum, d[j]);
        dot = fma2(d[j], h[j], dot);
      }
    }
    const Sums s = row_sums<G, true>(Sums{sum.x + sum.y, dot.x + dot.y}, buf, turn);
    // every thread is past the row before: its stage takes the row that comes `stages` after it
    if (lane == 0 && last >= 0 && !dead) {
      const int64_t ahead = r + (stages - 1) * step;
      if (ahead < a.rows) fetch(ahead, last);
    }
    if (a.dx) {
      const float2 c1 = both(-rstd * (s.a / n)), c2 = both(-rstd * rstd * (s.b / n));  // of x - mean
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (beyond(i)) continue;
        float2 h[4], d[4], p[4];
        x_at(i, h);
        g_at(i, d);
        if (a.w) weight(i, p);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (a.w) d[j] = mul2(d[j], p[j]);
          d[j] = fma2(add2(h[j], minus), c2, fma2(d[j], scale, c1));
        }
        store_chunk<G, true>(static_cast<T*>(a.dx) + r * a.cols, cols, lane, i, &d[0].x);
      }
    }
    last = stage;
    if (++stage == stages) stage = 0, phase ^= 1;
  }
  if (__syncthreads_or(dead)) {  // a wait ran out: NaNs, once no copy is in flight
    if (lane == 0)
      for (uint32_t i = fetched > stages ? fetched - stages : 0; i < fetched; ++i)
        async::settle(bar0 + 8 * (i % stages), i / stages & 1);
    const float nan = __uint_as_float(~0u);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float all[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) all[j] = nan;
#pragma unroll
      for (int j = 0; j < 4; ++j) dw[i][j] = db[i][j] = both(nan);
      if (a.dx)
        for (int64_t r = first; r < a.rows; r += step)
          store_chunk<G, true>(static_cast<T*>(a.dx) + r * a.cols, cols, lane, i, all);
    }
  }
  if (!a.dw && !a.db) return;
  // the groups' sums, in order, over the ring
  static_assert(kGroups == 2, "the first group adds the second's sums");
  float4* left = reinterpret_cast<float4*>(ring);
  __syncthreads();
  if (group == 1) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < 4; j += 2) {
        left[((i * 4 + j) / 2 * 2) * G + lane] = make_float4(dw[i][j].x, dw[i][j].y, dw[i][j + 1].x, dw[i][j + 1].y);
        left[((i * 4 + j) / 2 * 2 + 1) * G + lane] = make_float4(db[i][j].x, db[i][j].y, db[i][j + 1].x, db[i][j + 1].y);
      }
  }
  __syncthreads();
  if (group == 1) return;
  float* part = a.parts + blockIdx.x * 2 * a.cols;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
#pragma unroll
    for (int j = 0; j < 4; j += 2) {
      const float4 p = left[((i * 4 + j) / 2 * 2) * G + lane], q = left[((i * 4 + j) / 2 * 2 + 1) * G + lane];
      dw[i][j] = add2(dw[i][j], make_float2(p.x, p.y));
      dw[i][j + 1] = add2(dw[i][j + 1], make_float2(p.z, p.w));
      db[i][j] = add2(db[i][j], make_float2(q.x, q.y));
      db[i][j + 1] = add2(db[i][j + 1], make_float2(q.z, q.w));
    }
    const int c = column<G, true>(lane, i, 0);
    if (c < cols) {
      lin::store8(part + c, &dw[i][0].x);
      lin::store8(part + a.cols + c, &db[i][0].x);
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
  float s = 0.f;
  for (int64_t c = threadIdx.x; c < a.cols; c += kLong) s += value_at<T>(a, r, c);
  mean = row_sums<kLong>(s, buf, turn) / n;
  s = 0.f;
  for (int64_t c = threadIdx.x; c < a.cols; c += kLong) {
    const float d = value_at<T>(a, r, c) - mean;
    s = fmaf(d, d, s);
  }
  rstd = rsqrtf(row_sums<kLong>(s, buf, turn) / n + a.eps);
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

// A wait that runs out: nothing ever arrives at its barrier.
__global__ void wait_probe_kernel(long long clocks) {
  __shared__ __align__(8) uint64_t bar;
  if (threadIdx.x != 0) return;
  async::barrier_init(async::smem_addr(&bar), 1);
  bool dead = false;
  async::wait(async::smem_addr(&bar), 0, dead, clocks);
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
  // as many blocks as are under way together: one more a multiprocessor would run alone at the end
  static const int per_sm = [] {
    int n = 0;
    return cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, forward_kernel<G, NV, kVec, kCodes, T, W>,
                                                         Shape<G>::kThreads, 0) == cudaSuccess && n > 0 ? n : 1;
  }();
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

// Rows of the ring: whole 16-byte units, and at least two stages.
template <typename T>
int ring_stages(const Args& a) {
  const int64_t bytes = a.cols * ((a.codes_in ? 1 : sizeof(T)) + sizeof(T));
  if (a.cols % 16 != 0 || (a.codes_in && reinterpret_cast<uintptr_t>(a.codes_in) % 16 != 0)) return 0;
  return static_cast<int>(std::min<int64_t>(kRingBytes / bytes / (kRingThreads / kGroup), kMaxStages));  // of a group
}

template <typename T, typename W, int NV, bool kCodes>
cudaError_t launch_ring(const Args& a, int stages, cudaStream_t stream) {
  const auto kernel = backward_ring_kernel<NV, kCodes, T, W>;
  const cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingBytes);
  if (err != cudaSuccess) return err;
  const size_t rows = static_cast<size_t>(stages) * (kRingThreads / kGroup) * a.cols * ((kCodes ? 1 : sizeof(T)) + sizeof(T));
  const size_t bytes = std::max<size_t>(rows, static_cast<size_t>(NV) * 8 * 2 * kGroup * sizeof(float));  // and one group's sums
  kernel<<<backward_parts(a.rows, a.cols), kRingThreads, bytes, stream>>>(a, stages);
  return cudaGetLastError();
}

template <typename T, typename W>
cudaError_t dispatch(const Args& a, bool backward, cudaStream_t stream) {
  const bool vec = vectors_fit<T, W>(a, backward);
  if (backward) {
    const int stages = ring_stages<T>(a);
    if (vec && a.cols > 2048 && a.cols <= 8192 && stages >= 2) {
      if (a.codes_in)
        return a.cols <= 4096 ? launch_ring<T, W, 2, true>(a, stages, stream) : launch_ring<T, W, 4, true>(a, stages, stream);
      return a.cols <= 4096 ? launch_ring<T, W, 2, false>(a, stages, stream) : launch_ring<T, W, 4, false>(a, stages, stream);
    }
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
  return blocks_of_rows(rows, f, f.threads == 32 && f.chunks > 1 ? 2 : backward_blocks(f.threads));
}

cudaError_t wait_timeouts(unsigned int* count) { return async::read_timeouts(count); }

cudaError_t wait_probe(int64_t clocks, cudaStream_t stream) {
  wait_probe_kernel<<<1, 32, 0, stream>>>(clocks);
  return cudaGetLastError();
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
