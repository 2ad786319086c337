// Norms with the residual they belong to, forward and backward (formulas in
// residual_norm.h), for one storage type.
//
// A row is read once into the registers of G threads, 8 NV values each; dropout, gate,
// residual and norm happen there in float32, and each result is rounded once. A dropout
// mask is made again from its counter wherever it is needed. Short rows in 16 bits are
// bound by issue forward and by latencies backward, long rows by memory and its latency.
//
//   add_norm backward, from what reaches y (gy) and s (gs):
//     ds = gs + rstd (gy w - mean(gy w) - k mean(gy w k)), k = (s - mean) rstd
//     dr = alpha ds,  dh = D'(gate ds),  dgate = sum of ds D(h),  dw = sum of gy k,  db = sum of gy
//   norm_add backward, from what reaches s:
//     dr = alpha gs,  d = gate D'(gs),  dgate = sum of gs D(norm(h)),  dw = sum of d k,  db = sum of d
//     dh = rstd (d w - mean(d w) - k mean(d w k)), k = (h - mean) rstd
//   (kind rms: mean and the mean of d w are 0; D' multiplies as D does)
//
// y is the norm of the sum before s is rounded to its type. The backward pass takes s
// as it was stored, and with it the statistics of what was stored, which the forward
// takes in the same reductions: the gradients are those at the stored sum. (With the
// statistics of the unrounded one, k's sum over a row is not 0, nor that of its squares
// n; where a row's mean is large beside its spread nothing of the gradient is left.) Where
// the sum is not an output, rows that their type cannot hold so are kept normalised (kept_normal).
//
// Times, forward and backward: 40000 x 256 bfloat16 with dropout 22.2 and 20.8 us (82 MB
// each, 3.8 TB/s; 64 and 59 % of the issue slots), 184950 x 256 float16 norm_add with
// dropout and a gate 80 and 108 (67 and 54 %), 8192 x 8192 bfloat16 with a gate and both
// outputs 97 and 166 (537 and 805 MB, 5.5 and 4.8 TB/s).
//
// A backward block takes whole units of neighbouring rows, a unit's rows all under
// one row of the gate: so a thread sums dw, db and dgate of its columns in
// registers, writes them once, and a second kernel adds the blocks' sums in order.
#pragma once

#include <algorithm>

#include "dropout_device.cuh"
#include "residual_norm.h"
#include "rows_device.cuh"

namespace resnorm {
namespace {

using lin::add2;
using lin::both;
using lin::fma2;
using lin::mul2;
using rows::Chunk;
using rows::column;
using rows::row_sums;
using rows::Shape;
using rows::store_chunk;
using rows::Sums;

// Eight values of a parameter, of the rows' type or float32.
template <int G, bool kVec, typename T>
__device__ __forceinline__ void load_param(const void* p, bool f32, int cols, int lane, int i, float2 v[4]) {
  if (sizeof(T) == 4 || f32) {
    Chunk<float, kVec> c;
    c.template load<G>(static_cast<const float*>(p), cols, lane, i);
    c.get(v);
  } else {
    Chunk<T, kVec> c;
    c.template load<G>(static_cast<const T*>(p), cols, lane, i);
    c.get(v);
  }
}

// Which of a thread's eight values are kept. Where they are neighbours, they are one
// call of the generator. Where they are G columns apart, a warp's 256 columns are 32
// calls, one to a lane, and a lane fetches its bits from the lanes that have them.
template <int G, bool kVec>
struct Mask {
  drop::Words n;
  __device__ __forceinline__ void make(const drop::Key& key, uint32_t row, int lane, int i) {
    n = drop::numbers(key, row, i * G + lane);
  }
  __device__ __forceinline__ bool kept(const drop::Key& key, int j) const { return drop::kept(key, n, j); }
};
template <int G>
struct Mask<G, false> {
  uint32_t bits;
  __device__ __forceinline__ void make(const drop::Key& key, uint32_t row, int lane, int i) {
    const int l = lane & 31, group = ((i * 8 + l / 4) * G + lane - l) / 8 + l % 4;
    const uint32_t mine = drop::bits8(key, drop::numbers(key, row, group));
    bits = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) bits |= (__shfl_sync(0xffffffffu, mine, j * 4 + l / 8) >> (l % 8) & 1u) << j;
  }
  __device__ __forceinline__ bool kept(const drop::Key&, int j) const { return bits >> j & 1u; }
};

// A parameter's values of a thread's columns, held in registers through all rows where
// a thread has but one chunk; where there is no parameter, `none`.
template <int G, bool kVec, typename T>
struct Held {
  float2 v[4];
  __device__ __forceinline__ void set(const void* p, bool f32, int there, int lane, float none) {
    if (p) {
      load_param<G, kVec, T>(p, f32, there, lane, 0, v);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = both(none);
    }
  }
};
// Rows of one chunk a thread are bound by issue, and loads and conversions of
// parameters were a fifth of it.
template <int G, int NV>
constexpr bool kHolds = NV == 1;

template <typename M>
__device__ __forceinline__ void apply(const M& mask, const drop::Key& key, float* v) {
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = mask.kept(key, j) ? v[j] * key.scale : 0.f;
}

// The gate's row for a row.
__device__ __forceinline__ const void* gate_at(const Args& a, uint32_t r, int size) {
  if (!a.gate) return nullptr;
  const int64_t g = a.gate_rows == a.rows ? 0 : a.gate_rows == 1 ? r : r / static_cast<uint32_t>(a.gate_rows);
  return static_cast<const char*>(a.gate) + g * a.gate_stride * size;
}

__device__ __forceinline__ float2 stored(float2 v, float) { return v; }
__device__ __forceinline__ float2 stored(float2 v, lin::bf16) { return lin::unpack2(lin::pack2(v.x, v.y)); }
__device__ __forceinline__ float2 stored(float2 v, __half) { return __half22float2(__floats2half2_rn(v.x, v.y)); }

// Rows of several warps are asked for in L2 two rows ahead, by one thread and without
// registers: 8192 x 8192 with a gate 299 -> 279 us, 20000 x 1024 97 -> 85, 8192 x 4096 171
// -> 162. Not rows of one warp, where the requests cost more (184950 x 256 forward 79 ->
// 90 us), nor float32 (4096 x 4096 134 -> 136).
template <int G, bool kVec, typename T>
constexpr bool kPrefetches = kVec && G >= 64 && sizeof(T) == 2;
constexpr uint32_t kDistance = 2;  // three rows 294 us, five 326

// A row of `bytes` (whole 16-byte units) on its way into L2.
__device__ __forceinline__ void prefetch_row(const void* row, uint32_t bytes) {
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(row), "r"(bytes) : "memory");
}

struct Moments {
  float mean, rstd;
};

// Rows of 16 bits whose sum is not an output (Args::keep): the backward pass takes the sum as it
// was stored, so a normalised value k = (s - mean) rstd is off by half a step of |mean| rstd + |k|.
// Where the mean is more than four times the spread, or the type's range does not hold the sum,
// the row is kept normalised instead: k in the place of s, mean 0, and rstd with its sign turned.
template <typename T>
__device__ __forceinline__ bool kept_normal(const Args& a, Moments sum, Moments stored) {
  return sizeof(T) == 2 && a.keep && sum.rstd > 0.f && sum.rstd < 3.402823466e38f &&
         !(fabsf(sum.mean) * sum.rstd <= 4.f && stored.rstd > 0.f);
}

// Whether the warp has columns in its i-th chunk: what has none is skipped.
template <int G, bool kVec>
__device__ __forceinline__ bool any(int cols, int i) {
  return i == 0 || i * G * 8 < cols;
}

// Mean and rstd of the row whose values lie in v; beyond the row v is 0. kBoth: and
// those of the values as T stores them, in the same reductions.
template <int G, int NV, bool kVec, bool kBoth, typename T>
__device__ __forceinline__ Moments moments(const float2 v[NV][4], const Args& a, int cols, int lane, Sums* buf,
                                           int& turn, Moments& of_stored) {
  const float share = a.share;
  const auto over_row = [&](float2 x, float2 y) {
    if constexpr (kBoth)
      return row_sums<G>(Sums{x.x + x.y, y.x + y.y}, buf, turn);
    else
      return Sums{row_sums<G>(x.x + x.y, buf, turn), 0.f};
  };
  Sums mean{0.f, 0.f};
  if (!a.rms) {
    float2 t = both(0.f), u = both(0.f);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        t = add2(t, v[i][j]);
        if (kBoth) u = add2(u, stored(v[i][j], T()));
      }
    mean = over_row(t, u);
    mean.a *= share, mean.b *= share;
  }
  float2 t = both(0.f), u = both(0.f);
  const auto square = [&](int i, int j, float2 d, float2 sum) {
    if (!kVec) {
      if (column<G, false>(lane, i, 2 * j) >= cols) d.x = 0.f;
      if (column<G, false>(lane, i, 2 * j + 1) >= cols) d.y = 0.f;
    }
    return fma2(d, d, sum);
  };
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (kVec && column<G, true>(lane, i, 0) >= cols) continue;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      t = square(i, j, add2(v[i][j], both(-mean.a)), t);
      if (kBoth) u = square(i, j, add2(stored(v[i][j], T()), both(-mean.b)), u);
    }
  }
  const Sums var = over_row(t, u);
  of_stored = Moments{mean.b, rsqrtf(fmaf(var.b, share, a.eps))};
  return Moments{mean.a, rsqrtf(fmaf(var.a, share, a.eps))};
}

// v times, or plus, a parameter's values, chunk by chunk of the row; `there`: cols, or
// 0 where the row is not there, and nothing may be loaded for it.
template <int G, int NV, bool kVec, bool kAdd, typename T>
__device__ __forceinline__ void with_param(const void* p, bool f32, int cols, int there, int lane, float2 v[NV][4]) {
  const auto each = [&](auto type) {
    using P = decltype(type);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (!any<G, kVec>(cols, i)) continue;
      float2 w[4];
      Chunk<P, kVec> c;
      c.template load<G>(static_cast<const P*>(p), there, lane, i);
      c.get(w);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[i][j] = kAdd ? add2(v[i][j], w[j]) : mul2(v[i][j], w[j]);
    }
  };
  if (!p) return;
  if (sizeof(T) == 4 || f32)
    each(float());
  else
    each(T());
}

// Blocks to an SM that 64 registers a thread allow, where they do (8192 x 8192 bfloat16
// 100 us, in 124 registers 138): not for short rows of float32 (44446 x 256: 36 us in 64
// registers, 30 in 78), nor where columns are apart (30000 x 260 bfloat16: 64 and 47
// us). 0: as the compiler likes. Fewer registers spill (40000 x 256 in 51: 25 us, 22).
template <typename T>
constexpr int forward_blocks(int row_threads, int threads, bool vec) {
  return vec && (sizeof(T) == 2 || row_threads == 512) ? 1024 / threads : 0;
}

// With fewer than 32 threads to a row, a warp has several rows under way, of which the
// last may not be there: its loads give 0, and it stores nothing.
template <int G, int NV, bool kVec, bool kBranch, typename T>
__global__ void __launch_bounds__(Shape<G>::kThreads, forward_blocks<T>(G, Shape<G>::kThreads, kVec))
    forward_kernel(const Args a) {
  constexpr int kTogether = G < 32 ? 32 / G : 1;
  __shared__ Sums buf[Shape<G>::kBuf];
  int turn = 0;
  const int lane = threadIdx.x % G, cols = static_cast<int>(a.cols);
  const int gate_size = a.gate_f32 ? 4 : sizeof(T);
  const uint32_t rows = static_cast<uint32_t>(a.rows), step = gridDim.x * Shape<G>::kRows;
  const T *h = static_cast<const T*>(a.h), *res = static_cast<const T*>(a.r);
  const drop::Key key = drop::key_of(a.rule);
  const float2 alpha = both(a.alpha);
  constexpr bool kHold = kHolds<G, NV>;
  Held<G, kVec, T> held_w, held_b, held_gate;
  const bool one_gate = !a.gate || a.gate_rows == a.rows;
  if (kHold) {
    held_w.set(a.w, a.weight_f32, cols, lane, 1.f);
    held_b.set(a.b, a.weight_f32, cols, lane, 0.f);
    held_gate.set(one_gate ? a.gate : nullptr, a.gate_f32, cols, lane, 1.f);
  }
  const uint32_t offset = threadIdx.x / G % kTogether;
  uint32_t r = blockIdx.x * Shape<G>::kRows + threadIdx.x / G;
  Chunk<T, kVec> next_h[NV], next_r[NV];
  const auto load = [&](uint32_t row) {
    const int there = row < rows ? cols : 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      next_h[i].template load<G>(h + row * a.h_stride, there, lane, i);
      next_r[i].template load<G>(res + row * a.r_stride, there, lane, i);
    }
  };
  load(r);
  for (; r - offset < rows; r += step) {
    const int there = r < rows ? cols : 0;
    float2 v[NV][4];
    Chunk<T, kVec> here_r[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      next_h[i].get(v[i]);
      here_r[i] = next_r[i];
    }
    if (r - offset + step < rows) load(r + step);
    if (kPrefetches<G, kVec, T> && lane == 0 && r + kDistance * step < rows) {
      prefetch_row(h + (r + kDistance * step) * a.h_stride, cols * sizeof(T));
      prefetch_row(res + (r + kDistance * step) * a.r_stride, cols * sizeof(T));
    }
    const int64_t at = r * a.cols;
    // D, the gate and the residual
    const auto join = [&] {
      if (a.rule.threshold) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          if (!any<G, kVec>(cols, i)) continue;
          Mask<G, kVec> mask;
          mask.make(key, r, lane, i);
          apply(mask, key, &v[i][0].x);
        }
      }
      if (kHold) {
        if (!one_gate) held_gate.set(gate_at(a, r, gate_size), a.gate_f32, there, lane, 1.f);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[0][j] = mul2(v[0][j], held_gate.v[j]);
      } else {
        with_param<G, NV, kVec, false, T>(gate_at(a, r, gate_size), a.gate_f32, cols, there, lane, v);
      }
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        float2 p[4];
        here_r[i].get(p);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[i][j] = fma2(alpha, p[j], v[i][j]);
      }
      if (a.s) {
#pragma unroll
        for (int i = 0; i < NV; ++i) store_chunk<G, kVec>(static_cast<T*>(a.s) + at, there, lane, i, &v[i][0].x);
      }
    };
    if (!kBranch) join();
    Moments m, kept;
    if (!kBranch && sizeof(T) == 2 && a.rstd) {
      m = moments<G, NV, kVec, true, T>(v, a, cols, lane, buf, turn, kept);
    } else {
      Moments none;
      kept = m = moments<G, NV, kVec, false, T>(v, a, cols, lane, buf, turn, none);
    }
    const bool normal = !kBranch && kept_normal<T>(a, m, kept);
    if (a.rstd && lane == 0 && r < rows) {
      if (a.mean) a.mean[r] = normal ? 0.f : kept.mean;
      a.rstd[r] = normal ? -m.rstd : kept.rstd;
    }
    const float2 scale = both(m.rstd), minus = both(-m.mean);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) v[i][j] = mul2(add2(v[i][j], minus), scale);
    if (normal) {
#pragma unroll
      for (int i = 0; i < NV; ++i) store_chunk<G, kVec>(static_cast<T*>(a.s) + at, there, lane, i, &v[i][0].x);
    }
    if (kHold) {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[0][j] = fma2(v[0][j], held_w.v[j], held_b.v[j]);
    } else {
      with_param<G, NV, kVec, false, T>(a.w, a.weight_f32, cols, cols, lane, v);
      with_param<G, NV, kVec, true, T>(a.b, a.weight_f32, cols, cols, lane, v);
    }
    if (kBranch) {
      join();
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i) store_chunk<G, kVec>(static_cast<T*>(a.y) + at, there, lane, i, &v[i][0].x);
    }
  }
}

// A unit of a backward block: rows [begin, end), all under the gate's row `group`.
struct Unit {
  int64_t begin, end, group;
};
__device__ __forceinline__ Unit unit_of(const Grid& grid, int64_t u) {
  const int64_t group = u / grid.group_units, first = group * grid.group_rows;
  const int64_t begin = first + (u - group * grid.group_units) * grid.unit_rows;
  return Unit{begin, min(begin + grid.unit_rows, first + grid.group_rows), group};
}

// Blocks to an SM: 128 registers a thread, for the sums, the parameters and a row ahead.
// In 80, 20000 x 1024 with a gate takes 54 us instead of 52, 40000 x 512 with one 52
// instead of 46, 44446 x 256 float32 39 instead of 33; 10000 x 2048 the same 47.
constexpr int backward_blocks(int threads) { return 512 / threads; }

template <int G, int NV, bool kVec, bool kBranch, bool kGate, typename T>
__global__ void __launch_bounds__(Shape<G>::kThreads, backward_blocks(Shape<G>::kThreads))
    backward_kernel(const Args a, const Grid grid) {
  constexpr int kRows = Shape<G>::kRows, kTogether = G < 32 ? 32 / G : 1;
  __shared__ Sums buf[Shape<G>::kBuf];
  __shared__ float fold[kRows > 1 ? kRows * G * 8 : 1];
  int turn = 0;
  const int lane = threadIdx.x % G, slot = threadIdx.x / G, cols = static_cast<int>(a.cols);
  const int gate_size = a.gate_f32 ? 4 : sizeof(T);
  const drop::Key key = drop::key_of(a.rule);
  const float2 alpha = both(a.alpha);
  const bool normed = kBranch || a.gy;
  constexpr bool kHold = kHolds<G, NV>;
  Held<G, kVec, T> held_w, held_b, held_gate;
  // a unit's rows share a row of the gate, or else each looks its own up
  const bool one_gate = !a.gate || a.gate_rows == a.rows || grid.sums_gate;
  if (kHold) {
    held_w.set(a.w, a.weight_f32, cols, lane, 1.f);
    if (kBranch && kGate) held_b.set(a.b, a.weight_f32, cols, lane, 0.f);
    if (!one_gate) held_gate.set(nullptr, false, cols, lane, 1.f);
  }
  float2 dw[NV][4] = {}, db[NV][4] = {}, dg[kGate ? NV : 1][4] = {};

  // Sums over the block's rows, of this thread's columns, into `out`.
  const auto put_sums = [&](const float2 (*v)[4], float* out) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const float* mine = &v[i][0].x;
      if (kRows > 1) {  // the block's rows, in order
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 8; ++j) fold[(slot * 8 + j) * G + lane] = mine[j];
        __syncthreads();
        // thread (slot, lane) adds up column j = slot of lane's eight
        if (slot < 8) {
          float sum = 0.f;
#pragma unroll
          for (int k = 0; k < kRows; ++k) sum += fold[(k * 8 + slot) * G + lane];
          const int c = column<G, kVec>(lane, i, slot);
          if (c < cols) out[c] = sum;
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int c = column<G, kVec>(lane, i, j);
          if (c < cols) out[c] = mine[j];
        }
      }
    }
  };

  for (int64_t u = blockIdx.x; u < grid.units; u += gridDim.x) {
    const Unit unit = unit_of(grid, u);
    const uint32_t end = static_cast<uint32_t>(unit.end), offset = slot % kTogether;
    uint32_t r = static_cast<uint32_t>(unit.begin) + slot;
    if (kHold && one_gate)
      held_gate.set(gate_at(a, static_cast<uint32_t>(unit.begin), gate_size), a.gate_f32, cols, lane, 1.f);
    // the norm's rows and what reaches its output, one row ahead
    Chunk<T, kVec> next_x[NV], next_g[NV];
    float next_mean = 0.f, next_rstd = 0.f;
    const auto load = [&](uint32_t row) {
      if (!normed) return;
      const int there = row < end ? cols : 0;
      const T* x = kBranch ? static_cast<const T*>(a.h) + row * a.h_stride : static_cast<const T*>(a.sum) + row * a.sum_stride;
      const T* g = kBranch ? static_cast<const T*>(a.gs) + row * a.gs_stride : static_cast<const T*>(a.gy) + row * a.gy_stride;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        next_x[i].template load<G>(x, there, lane, i);
        next_g[i].template load<G>(g, there, lane, i);
      }
      next_mean = there && a.mean ? a.mean[row] : 0.f;
      next_rstd = there ? a.rstd[row] : 0.f;
    };
    // The longest rows, one to an SM, come from L2 when their turn comes, without registers
    // for the next one: 8192 x 8192 176 -> 166 us, 8192 x 4096 100 -> 95; 2048 columns 47 -> 52.
    constexpr bool kEarly = !(kPrefetches<G, kVec, T> && G == 512);
    if (kEarly) load(r);
    for (; r - offset < end; r += kRows) {
      if (!kEarly) load(r);
      const int there = r < end ? cols : 0;
      const int64_t at = r * a.cols;
      Chunk<T, kVec> x[NV], g[NV];
#pragma unroll
      for (int i = 0; i < NV; ++i) x[i] = next_x[i], g[i] = next_g[i];
      // a row that is kept normalised: rstd below 0, and x is k
      const bool normal = !kBranch && sizeof(T) == 2 && next_rstd < 0.f;
      const float rstd = normal ? -next_rstd : next_rstd, to_k = normal ? 1.f : rstd;
      const float2 scale = both(to_k), minus = both(-next_mean);
      // what else the row needs, on its way while the sums are taken
      Chunk<T, kVec> more[kBranch ? 1 : NV], branch[kGate && !kBranch ? NV : 1];
      if (!kBranch) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          if (a.gs) more[kBranch ? 0 : i].template load<G>(static_cast<const T*>(a.gs) + r * a.gs_stride, there, lane, i);
          if (kGate) branch[kGate && !kBranch ? i : 0].template load<G>(static_cast<const T*>(a.h) + r * a.h_stride, there, lane, i);
        }
      }
      if (kEarly && r - offset + kRows < end) load(r + kRows);
      // Short rows with the gate's gradient, whose kernels wait for loads more than the others:
      // the block's next rows, neighbours, by one request to a tensor (184950 x 256 float16
      // norm_add, with dr written too, 124 -> 112 us, 180000 x 256 add_norm with both outputs
      // 111 -> 95; without a gate, 40000 x 256, 20.7 -> 23).
      if (kVec && kGate && G <= 32 && threadIdx.x == 0 && r + kDistance * kRows < end) {
        const uint32_t row = r + kDistance * kRows, count = min(static_cast<uint32_t>(kRows), end - row);
        const auto ask = [&](const void* p, int64_t stride) {
          if (stride <= 2 * cols)  // not where other columns lie between
            prefetch_row(static_cast<const T*>(p) + row * stride,
                         static_cast<uint32_t>(((count - 1) * stride + cols) * sizeof(T)));
        };
        ask(a.h, a.h_stride);
        if (!kBranch && normed) ask(a.sum, a.sum_stride), ask(a.gy, a.gy_stride);
        if (a.gs) ask(a.gs, a.gs_stride);
      }
      if (kPrefetches<G, kVec, T> && lane == 0 && r + kDistance * kRows < end) {
        const uint32_t row = r + kDistance * kRows, bytes = cols * sizeof(T);
        if (kBranch || kGate) prefetch_row(static_cast<const T*>(a.h) + row * a.h_stride, bytes);
        if (!kBranch && normed) {
          prefetch_row(static_cast<const T*>(a.sum) + row * a.sum_stride, bytes);
          prefetch_row(static_cast<const T*>(a.gy) + row * a.gy_stride, bytes);
        }
        if (a.gs) prefetch_row(static_cast<const T*>(a.gs) + row * a.gs_stride, bytes);
      }
      float2 sum = both(0.f), dot = both(0.f), d[NV][4];
      // x - mean of eight values
      const auto centred = [&](int i, float2 k[4]) {
        x[i].get(k);
#pragma unroll
        for (int j = 0; j < 4; ++j) k[j] = add2(k[j], minus);
      };
      // from d, what reaches the norm's output: dw, db, and d times the weight with its sums
      const auto take_sums = [&] {
        const auto add = [&](bool weighted) {
#pragma unroll
          for (int i = 0; i < NV; ++i) {
            if (!any<G, kVec>(cols, i)) continue;
            float2 k[4], w[4];
            centred(i, k);
            if (kHold) {
#pragma unroll
              for (int j = 0; j < 4; ++j) w[j] = held_w.v[j];
            } else if (weighted) {
              load_param<G, kVec, T>(a.w, a.weight_f32, cols, lane, i, w);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              k[j] = mul2(k[j], scale);  // beyond the row d is 0, and counts for nothing
              dw[i][j] = fma2(d[i][j], k[j], dw[i][j]);
              db[i][j] = add2(db[i][j], d[i][j]);
              if (weighted) d[i][j] = mul2(d[i][j], w[j]);
              sum = add2(sum, d[i][j]);
              dot = fma2(d[i][j], k[j], dot);
            }
          }
        };
        kHold || a.w ? add(true) : add(false);
      };
      // the gradient of the norm's input in the place of d
      const auto through_norm = [&] {
        const Sums t = row_sums<G>(Sums{sum.x + sum.y, dot.x + dot.y}, buf, turn);
        const float2 c1 = both(a.rms ? 0.f : -rstd * (t.a * a.share)), c2 = both(-rstd * to_k * (t.b * a.share));
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          float2 k[4];
          centred(i, k);
#pragma unroll
          for (int j = 0; j < 4; ++j) d[i][j] = fma2(k[j], c2, fma2(d[i][j], both(rstd), c1));
        }
      };
      const auto put_rows = [&](void* p, float2 v[NV][4]) {
#pragma unroll
        for (int i = 0; i < NV; ++i) store_chunk<G, kVec>(static_cast<T*>(p) + at, there, lane, i, &v[i][0].x);
      };
      const auto put_residual = [&] {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          float2 p[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) p[j] = mul2(alpha, d[i][j]);
          store_chunk<G, kVec>(static_cast<T*>(a.dr) + at, there, lane, i, &p[0].x);
        }
      };
      // dgate of eight values, what reaches the sum times the branch's t: added up, or a row of its own
      const auto put_gate = [&](int i, float2 t[4]) {
#pragma unroll
        for (int j = 0; j < 4; ++j) t[j] = mul2(t[j], d[i][j]);
        if (grid.sums_gate) {
#pragma unroll
          for (int j = 0; j < 4; ++j) dg[kGate ? i : 0][j] = add2(dg[kGate ? i : 0][j], t[j]);
        } else if (a.gate_f32) {
          store_chunk<G, kVec>(static_cast<float*>(a.dgate) + at, there, lane, i, &t[0].x);
        } else {
          store_chunk<G, kVec>(static_cast<T*>(a.dgate) + at, there, lane, i, &t[0].x);
        }
      };
      const auto through_gate = [&] {
        if (kHold) {
          if (!one_gate) held_gate.set(gate_at(a, r, gate_size), a.gate_f32, there, lane, 1.f);
#pragma unroll
          for (int j = 0; j < 4; ++j) d[0][j] = mul2(d[0][j], held_gate.v[j]);
        } else {
          with_param<G, NV, kVec, false, T>(gate_at(a, r, gate_size), a.gate_f32, cols, there, lane, d);
        }
      };
      // d through dropout; the gate's gradient on the way, from D of the branch
      const auto through_dropout = [&](auto&& branch_of) {
        const auto each = [&](bool some) {
#pragma unroll
          for (int i = 0; i < NV; ++i) {
            if (!any<G, kVec>(cols, i)) continue;
            Mask<G, kVec> mask;
            if (some) mask.make(key, r, lane, i);
            if (kGate) {
              float2 t[4];
              branch_of(i, t);
              if (some) apply(mask, key, &t[0].x);
              put_gate(i, t);
            }
            if (some) apply(mask, key, &d[i][0].x);
          }
        };
        if (a.rule.threshold)
          each(true);
        else if (kGate)
          each(false);
      };
      if (!kBranch) {
        if (normed) {
#pragma unroll
          for (int i = 0; i < NV; ++i) g[i].get(d[i]);
          take_sums();
          if (!a.dh && !a.dr && !kGate) continue;
          through_norm();
        } else {
#pragma unroll
          for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) d[i][j] = both(0.f);
        }
        if (a.gs) {
#pragma unroll
          for (int i = 0; i < NV; ++i) {
            float2 p[4];
            more[kBranch ? 0 : i].get(p);
#pragma unroll
            for (int j = 0; j < 4; ++j) d[i][j] = add2(d[i][j], p[j]);
          }
        }
        if (a.dr) put_residual();
        through_dropout([&](int i, float2 t[4]) { branch[kGate && !kBranch ? i : 0].get(t); });
        if (!a.dh) continue;
        through_gate();
        put_rows(a.dh, d);
      } else {
#pragma unroll
        for (int i = 0; i < NV; ++i) g[i].get(d[i]);
        if (a.dr) put_residual();
        through_dropout([&](int i, float2 t[4]) {  // norm(h)
          centred(i, t);
#pragma unroll
          for (int j = 0; j < 4; ++j) t[j] = mul2(t[j], scale);
          if (kHold) {
#pragma unroll
            for (int j = 0; j < 4; ++j) t[j] = fma2(t[j], held_w.v[j], held_b.v[j]);
            return;
          }
          float2 p[4];
          if (a.w) {
            load_param<G, kVec, T>(a.w, a.weight_f32, cols, lane, i, p);
#pragma unroll
            for (int j = 0; j < 4; ++j) t[j] = mul2(t[j], p[j]);
          }
          if (a.b) {
            load_param<G, kVec, T>(a.b, a.weight_f32, cols, lane, i, p);
#pragma unroll
            for (int j = 0; j < 4; ++j) t[j] = add2(t[j], p[j]);
          }
        });
        through_gate();
        take_sums();
        if (!a.dh) continue;
        through_norm();
        put_rows(a.dh, d);
      }
    }
    if (kGate && grid.sums_gate) {
      put_sums(dg, a.parts + static_cast<int64_t>(gridDim.x) * 2 * a.cols + u * a.cols);
#pragma unroll
      for (int i = 0; i < (kGate ? NV : 1); ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) dg[i][j] = both(0.f);
    }
  }
  if (!a.dw && !a.db) return;
  float* part = a.parts + blockIdx.x * 2 * a.cols;
  put_sums(dw, part);
  put_sums(db, part + a.cols);
}

// Rows beyond the registers: a block of 1024 threads a row, eight neighbouring columns
// a thread at a time, the row read again for each pass; sums over rows go to `parts`,
// whose columns a thread owns.
constexpr int kLong = 1024;

template <typename T>
struct LongRow {
  const Args& a;
  int64_t r, c;  // c: the first of eight columns
  int count;
  __device__ __forceinline__ LongRow(const Args& args, int64_t row, int64_t column)
      : a(args), r(row), c(column), count(static_cast<int>(args.cols - column < 8 ? args.cols - column : 8)) {}
  __device__ __forceinline__ void rows_of(const void* p, int64_t stride, float v[8]) const {
    lin::load_some(static_cast<const T*>(p) + r * stride + c, count, false, v);
  }
  __device__ __forceinline__ void param(const void* p, bool f32, float none, float v[8]) const {
    if (!p) {
      for (int j = 0; j < 8; ++j) v[j] = none;
    } else if (f32) {
      lin::load_some(static_cast<const float*>(p) + c, count, false, v);
    } else {
      lin::load_some(static_cast<const T*>(p) + c, count, false, v);
    }
  }
  __device__ __forceinline__ void put(void* p, const float v[8]) const {
    lin::store_some(static_cast<T*>(p) + r * a.cols + c, count, false, v);
  }
  __device__ __forceinline__ drop::Words mask(const drop::Key& key) const {
    return drop::numbers(key, static_cast<uint32_t>(r), static_cast<uint32_t>(c / 8));
  }
  // s of add_norm, from its parts
  __device__ __forceinline__ void sum(const drop::Key& key, float v[8]) const {
    float p[8];
    rows_of(a.h, a.h_stride, v);
    if (a.rule.threshold) drop::apply8(key, mask(key), v);
    param(gate_at(a, r, a.gate_f32 ? 4 : sizeof(T)), a.gate_f32, 1.f, p);
    for (int j = 0; j < 8; ++j) v[j] *= p[j];
    rows_of(a.r, a.r_stride, p);
    for (int j = 0; j < 8; ++j) v[j] = fmaf(a.alpha, p[j], v[j]);
  }
};

template <bool kBranch, typename T>
__global__ void __launch_bounds__(kLong) forward_long_kernel(const Args a) {
  __shared__ Sums buf[2 * kLong / 32];
  int turn = 0;
  const drop::Key key = drop::key_of(a.rule);
  const float n = static_cast<float>(a.cols);
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const auto over = [&](auto&& f) {
      for (int64_t c = threadIdx.x * 8ll; c < a.cols; c += kLong * 8) {
        const LongRow<T> at(a, r, c);
        float v[8];
        if (kBranch)
          at.rows_of(a.h, a.h_stride, v);
        else
          at.sum(key, v);
        f(at, v);
      }
    };
    // of the row, and of the row as it is stored
    Sums mean{0.f, 0.f}, t{0.f, 0.f};
    const auto as_stored = [](float v) { return kBranch ? v : lin::to_float(lin::from_float<T>(v)); };
    if (!a.rms) {
      over([&](const LongRow<T>& at, float* v) {
        for (int j = 0; j < at.count; ++j) t = t + Sums{v[j], as_stored(v[j])};
      });
      mean = row_sums<kLong>(t, buf, turn);
      mean.a /= n, mean.b /= n;
    }
    t = Sums{0.f, 0.f};
    over([&](const LongRow<T>& at, float* v) {
      for (int j = 0; j < at.count; ++j) {
        const float d = v[j] - mean.a, e = as_stored(v[j]) - mean.b;
        t = Sums{fmaf(d, d, t.a), fmaf(e, e, t.b)};
      }
    });
    t = row_sums<kLong>(t, buf, turn);
    const float rstd = rsqrtf(t.a / n + a.eps), stored = rsqrtf(t.b / n + a.eps);
    const bool normal = !kBranch && kept_normal<T>(a, Moments{mean.a, rstd}, Moments{mean.b, stored});
    if (a.rstd && threadIdx.x == 0) {
      if (a.mean) a.mean[r] = normal ? 0.f : mean.b;
      a.rstd[r] = normal ? -rstd : stored;
    }
    over([&](const LongRow<T>& at, float* v) {
      float w[8], b[8];
      if (!kBranch && a.s && !normal) at.put(a.s, v);
      at.param(a.w, a.weight_f32, 1.f, w);
      at.param(a.b, a.weight_f32, 0.f, b);
      for (int j = 0; j < 8; ++j) v[j] = (v[j] - mean.a) * rstd;
      if (normal) at.put(a.s, v);
      for (int j = 0; j < 8; ++j) v[j] = fmaf(v[j], w[j], b[j]);
      if (kBranch) {
        if (a.rule.threshold) drop::apply8(key, at.mask(key), v);
        at.param(gate_at(a, r, a.gate_f32 ? 4 : sizeof(T)), a.gate_f32, 1.f, w);
        at.rows_of(a.r, a.r_stride, b);
        for (int j = 0; j < 8; ++j) v[j] = fmaf(a.alpha, b[j], v[j] * w[j]);
        at.put(a.s, v);
      } else {
        at.put(a.y, v);
      }
    });
  }
}

template <bool kBranch, typename T>
__global__ void __launch_bounds__(kLong) backward_long_kernel(const Args a, const Grid grid) {
  __shared__ Sums buf[2 * kLong / 32];
  int turn = 0;
  const drop::Key key = drop::key_of(a.rule);
  const float n = static_cast<float>(a.cols);
  const bool normed = kBranch || a.gy;
  float* part = a.parts + blockIdx.x * 2 * a.cols;
  bool first = true;  // of the block's rows
  for (int64_t u = blockIdx.x; u < grid.units; u += gridDim.x) {
    const Unit unit = unit_of(grid, u);
    float* gate_part = a.parts + static_cast<int64_t>(gridDim.x) * 2 * a.cols + u * a.cols;
    for (int64_t r = unit.begin; r < unit.end; ++r, first = false) {
      const float mean = normed && a.mean ? a.mean[r] : 0.f, kept = normed ? a.rstd[r] : 0.f;
      const bool normal = !kBranch && sizeof(T) == 2 && kept < 0.f;  // the row is kept normalised
      const float rstd = normal ? -kept : kept, to_k = normal ? 1.f : rstd;
      const void* gate = gate_at(a, r, a.gate_f32 ? 4 : sizeof(T));
      // eight normalised values k and what reaches the norm's output, d
      const auto inputs = [&](const LongRow<T>& at, float k[8], float d[8]) {
        at.rows_of(kBranch ? a.h : a.sum, kBranch ? a.h_stride : a.sum_stride, k);
        for (int j = 0; j < 8; ++j) k[j] = (k[j] - mean) * to_k;
        at.rows_of(kBranch ? a.gs : a.gy, kBranch ? a.gs_stride : a.gy_stride, d);
        if (kBranch) {
          float p[8];
          if (a.rule.threshold) drop::apply8(key, at.mask(key), d);
          at.param(gate, a.gate_f32, 1.f, p);
          for (int j = 0; j < 8; ++j) d[j] *= p[j];
        }
      };
      const auto put_gate = [&](const LongRow<T>& at, const float t[8]) {
        if (grid.sums_gate) {
          for (int j = 0; j < at.count; ++j) gate_part[at.c + j] = t[j] + (r == unit.begin ? 0.f : gate_part[at.c + j]);
        } else if (a.gate_f32) {
          lin::store_some(static_cast<float*>(a.dgate) + r * a.cols + at.c, at.count, false, t);
        } else {
          at.put(a.dgate, t);
        }
      };
      Sums s = {0.f, 0.f};
      if (normed) {
        for (int64_t c = threadIdx.x * 8ll; c < a.cols; c += kLong * 8) {
          const LongRow<T> at(a, r, c);
          float k[8], d[8], w[8];
          inputs(at, k, d);
          at.param(a.w, a.weight_f32, 1.f, w);
          for (int j = 0; j < at.count; ++j) {
            if (a.dw || a.db) {
              part[c + j] = fmaf(d[j], k[j], first ? 0.f : part[c + j]);
              part[a.cols + c + j] = d[j] + (first ? 0.f : part[a.cols + c + j]);
            }
            s.a = fmaf(d[j], w[j], s.a);
            s.b = fmaf(d[j] * w[j], k[j], s.b);
          }
        }
        s = row_sums<kLong>(s, buf, turn);
      }
      const float c1 = a.rms ? 0.f : s.a / n, c2 = s.b / n;
      for (int64_t c = threadIdx.x * 8ll; c < a.cols; c += kLong * 8) {
        const LongRow<T> at(a, r, c);
        float k[8] = {}, d[8] = {}, p[8], t[8];
        if (normed) {
          inputs(at, k, d);
          at.param(a.w, a.weight_f32, 1.f, p);
          if (kBranch && a.dgate) {
            at.param(a.b, a.weight_f32, 0.f, t);
            for (int j = 0; j < 8; ++j) t[j] = fmaf(k[j], p[j], t[j]);
            if (a.rule.threshold) drop::apply8(key, at.mask(key), t);
            float g[8];
            at.rows_of(a.gs, a.gs_stride, g);
            for (int j = 0; j < 8; ++j) t[j] *= g[j];
            put_gate(at, t);
          }
          for (int j = 0; j < 8; ++j) d[j] = rstd * (d[j] * p[j] - c1 - k[j] * c2);
        }
        if (kBranch) {
          if (a.dh) at.put(a.dh, d);
          if (a.dr) {
            at.rows_of(a.gs, a.gs_stride, t);
            for (int j = 0; j < 8; ++j) t[j] *= a.alpha;
            at.put(a.dr, t);
          }
          continue;
        }
        if (a.gs) {
          at.rows_of(a.gs, a.gs_stride, t);
          for (int j = 0; j < 8; ++j) d[j] += t[j];
        }
        if (a.dr) {
          for (int j = 0; j < 8; ++j) t[j] = a.alpha * d[j];
          at.put(a.dr, t);
        }
        if (a.dgate) {
          at.rows_of(a.h, a.h_stride, t);
          if (a.rule.threshold) drop::apply8(key, at.mask(key), t);
          for (int j = 0; j < 8; ++j) t[j] *= d[j];
          put_gate(at, t);
        }
        if (a.dh) {
          if (a.rule.threshold) drop::apply8(key, at.mask(key), d);
          at.param(gate, a.gate_f32, 1.f, p);
          for (int j = 0; j < 8; ++j) d[j] *= p[j];
          at.put(a.dh, d);
        }
      }
    }
  }
}

// ---- host --------------------------------------------------------------------------

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <typename T>
bool vectors_fit(const Args& a) {
  const auto rows_fit = [](const void* p, int64_t stride, size_t size) {
    return !p || (aligned16(p) && (stride * size) % 16 == 0);
  };
  bool ok = a.cols % 8 == 0;
  ok = ok && rows_fit(a.h, a.h_stride, sizeof(T)) && rows_fit(a.r, a.r_stride, sizeof(T));
  ok = ok && rows_fit(a.gate, a.gate_stride, a.gate_f32 ? 4 : sizeof(T));
  ok = ok && rows_fit(a.gy, a.gy_stride, sizeof(T)) && rows_fit(a.gs, a.gs_stride, sizeof(T));
  ok = ok && rows_fit(a.sum, a.sum_stride, sizeof(T));
  for (const void* p : {a.w, a.b, static_cast<const void*>(a.y), static_cast<const void*>(a.s),
                        static_cast<const void*>(a.dh), static_cast<const void*>(a.dr),
                        static_cast<const void*>(a.dgate)})
    ok = ok && aligned16(p);
  return ok;
}

template <int G, int NV, bool kVec, bool kBranch, typename T>
cudaError_t launch_forward(const Args& a, cudaStream_t stream) {
  // as many blocks as are under way together
  static const int per_sm = [] {
    int n = 0;
    return cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, forward_kernel<G, NV, kVec, kBranch, T>,
                                                         Shape<G>::kThreads, 0) == cudaSuccess && n > 0 ? n : 1;
  }();
  const int64_t groups = (a.rows + Shape<G>::kRows - 1) / Shape<G>::kRows;
  const int blocks = static_cast<int>(std::min<int64_t>(groups, 148ll * per_sm));
  forward_kernel<G, NV, kVec, kBranch, T><<<blocks, Shape<G>::kThreads, 0, stream>>>(a);
  return cudaGetLastError();
}

template <bool kVec, bool kBranch, typename T>
cudaError_t forward_form(const Args& a, cudaStream_t stream) {
  if (a.cols <= 128) return launch_forward<kVec ? 16 : 32, 1, kVec, kBranch, T>(a, stream);
  if (a.cols <= 256) return launch_forward<32, 1, kVec, kBranch, T>(a, stream);
  if (a.cols <= 512) return launch_forward<64, 1, kVec, kBranch, T>(a, stream);
  if (a.cols <= 1024) return launch_forward<128, 1, kVec, kBranch, T>(a, stream);
  if (a.cols <= 2048) return launch_forward<256, 1, kVec, kBranch, T>(a, stream);
  if (a.cols <= 4096) return launch_forward<512, 1, kVec, kBranch, T>(a, stream);
  if (a.cols <= 8192) return launch_forward<512, 2, kVec, kBranch, T>(a, stream);
  const int blocks = static_cast<int>(std::min<int64_t>(a.rows, 148 * 2));
  forward_long_kernel<kBranch, T><<<blocks, kLong, 0, stream>>>(a);
  return cudaGetLastError();
}

template <typename T>
cudaError_t forward_of(const Args& a, cudaStream_t stream) {
  if (vectors_fit<T>(a))
    return a.branch ? forward_form<true, true, T>(a, stream) : forward_form<true, false, T>(a, stream);
  return a.branch ? forward_form<false, true, T>(a, stream) : forward_form<false, false, T>(a, stream);
}

template <int G, int NV, bool kVec, bool kBranch, bool kGate, typename T>
cudaError_t launch_backward(const Args& a, const Grid& grid, cudaStream_t stream) {
  backward_kernel<G, NV, kVec, kBranch, kGate, T><<<grid.blocks, Shape<G>::kThreads, 0, stream>>>(a, grid);
  return cudaGetLastError();
}

template <bool kVec, bool kBranch, bool kGate, typename T>
cudaError_t backward_form(const Args& a, const Grid& grid, cudaStream_t stream) {
  if (a.cols <= 128) return launch_backward<kVec ? 16 : 32, 1, kVec, kBranch, kGate, T>(a, grid, stream);
  if (a.cols <= 256) return launch_backward<32, 1, kVec, kBranch, kGate, T>(a, grid, stream);
  if (a.cols <= 512) return launch_backward<64, 1, kVec, kBranch, kGate, T>(a, grid, stream);
  if (a.cols <= 1024) return launch_backward<128, 1, kVec, kBranch, kGate, T>(a, grid, stream);
  if (a.cols <= 2048) return launch_backward<256, 1, kVec, kBranch, kGate, T>(a, grid, stream);
  if (a.cols <= 4096) return launch_backward<512, 1, kVec, kBranch, kGate, T>(a, grid, stream);
  if (a.cols <= 8192) return launch_backward<512, 2, kVec, kBranch, kGate, T>(a, grid, stream);
  backward_long_kernel<kBranch, T><<<grid.blocks, kLong, 0, stream>>>(a, grid);
  return cudaGetLastError();
}

template <bool kVec, typename T>
cudaError_t backward_kind(const Args& a, const Grid& grid, cudaStream_t stream) {
  if (a.branch)
    return a.dgate ? backward_form<kVec, true, true, T>(a, grid, stream)
                   : backward_form<kVec, true, false, T>(a, grid, stream);
  return a.dgate ? backward_form<kVec, false, true, T>(a, grid, stream)
                 : backward_form<kVec, false, false, T>(a, grid, stream);
}

template <typename T>
cudaError_t backward_of(const Args& a, const Grid& grid, cudaStream_t stream) {
  return vectors_fit<T>(a) ? backward_kind<true, T>(a, grid, stream) : backward_kind<false, T>(a, grid, stream);
}

}  // namespace
}  // namespace resnorm
