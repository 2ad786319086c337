// The product D[m, n] = sum_k A(m, k) B(n, k) of the fused linear operator on
// the fifth-generation tensor cores, with the operator's epilogues.
//
// One persistent block per SM (or a pair of them on two SMs) of 18 warps:
// a producer thread copies tiles of A and B into a ring of shared-memory stages
// (TMA, 128-byte swizzle), one thread issues tcgen05.mma on them into one of
// two accumulators in tensor memory, and sixteen warps carry the other
// accumulator through the epilogue meanwhile. A lane holds a row there, 16
// columns at a time: tensor memory -> registers, bias, activation, residual ->
// shared memory -> global memory by TMA, which also brings the residual. So
// global memory sees whole rows of 128 bytes, and the code has no addresses or
// bounds. (First form: turned through shared memory in float32 and stored by
// the lanes, 8 columns each; eight times the instructions, and with its loops
// unrolled two thirds of the time went into fetching them. Value projection,
// 184950 x 256 x 256: 360 us unrolled, 74 rolled.)
//
// Either operand may be stored along k or across it: the forward reads both
// along k, dx = dz W reads W across it, dW = dz^T x both. Nothing is transposed
// in memory; the instruction and the tile's layout differ.
//
// float32 (three bfloat16 planes an operand): a stage is the three planes of its
// k, and the six products of planes that reach 2^-24 of the result are issued on
// them. The tensor core's float32 accumulator cuts where an FMA would round:
// 2^-25 of what it holds per step on average, always towards zero. So the five
// small products, 2^-8 of the result and below, have an accumulator of their
// own, taken over 1024 of k, and the sums over 128 of k of the first product are
// added up in registers: the relative error is 1.3e-7, where one accumulator
// over 256 of k had 2.9e-6. A finished tile waits in the small products' columns
// for its epilogue, so the next tile's products go on (22223 x 256 x 1024 with
// slope: 98 us; with the two accumulators side by side and held by the epilogue
// 107). What bounds it: a product of 128 columns takes the time of one of 256
// (2048 x 2048 x 2048: 107 us). Tiles of 256 leave room for one accumulator only;
// with both sums read after every 128 of k they took 105 us there, read after
// every 1024 70, and 20 us more than now where k is 256.
#include <algorithm>

#include "linear_tile.cuh"

namespace lin {
namespace {

constexpr int kFwdSlope = 3;  // beside Epilogue::Mode: kFwd that also writes the slope

// The epilogue's warps, from the first tile to the last. kKind: the mode, the
// activation and whether there is a residual, as constants: with branches in
// here, 16 columns took 170 instructions and more where 50 do, and issuing them
// was the bound of short products; as one function with all kinds it spilled.
// Returns whether a wait ran out.
template <int BN, int CG, typename T, bool kF32, int kKind>
__device__ __noinline__ bool epilogue(const Maps& maps, const Job& job, const Place place) {
  using S = Shape<BN, CG, kF32>;
  constexpr int kMode = kKind / 8;
  constexpr Act kAct = static_cast<Act>(kKind / 2 % 4);
  constexpr bool kExtra = kKind % 2;
  constexpr bool kSlope = kMode == kFwdSlope;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t tmem = place.tmem, rank = place.rank;
  const auto acc_full = [&](int b) { return place.bars + 8 * (2 * S::kStages + b); };
  const auto acc_empty = [&](int b) { return place.bars + 8 * (2 * S::kStages + 2 + b); };
  const auto small_empty = [&](int b) { return place.bars + 8 * (2 * S::kStages + 4 + kEpiWarps + b); };
  const uint32_t items = job.tiles_m * job.tiles_n * job.splits;
  const uint32_t first = blockIdx.x / CG, step = gridDim.x / CG;
  const int chunk = kF32 ? kPromote : job.kblocks;
  bool dead = false;
  constexpr int kBoxCols = 128 / sizeof(T) < S::kCols ? 128 / sizeof(T) : S::kCols;
  constexpr int kRowBytes = kBoxCols * sizeof(T);
  constexpr bool kFast = sizeof(T) == 2;
  constexpr int kParts = S::kCols / kBoxCols;  // more than one only for partial sums
  constexpr int kHalfCols = 64 / sizeof(T), kHalves = S::kCols / kHalfCols;  // with the slope: rows of 64 bytes
  static_assert(!kSlope || kHalves <= 2, "a part to each half of the box");
  const int quad = warp & 3, group = warp >> 2;
  const uint32_t box = place.boxes + warp * kBoxBytes;
  const uint32_t arrived = place.bars + 8 * (2 * S::kStages + 4 + warp);  // the residual's box
  const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
  const int rows_m = static_cast<int>(job.pr.m), rows_n = static_cast<int>(job.pr.n);
  const Epilogue& e = job.pr.epi;
  constexpr bool kPlanes = sizeof(T) == 4 && kMode == Epilogue::kDz;
  const bool extra = kSlope ? e.extra != nullptr : kExtra;
  const bool with_bias = kMode != Epilogue::kStore && e.bias != nullptr;
  const bool bias_vec = reinterpret_cast<uintptr_t>(e.bias) % 16 == 0;
  const auto row_of = [&](const Item& t) { return t.m + static_cast<int>(rank) * kTileM + quad * 32; };
  const auto col_of = [&](const Item& t) { return t.n + group * S::kCols; };
  // a box on its way out; the next may be written when `read`
  const auto send = [&](const CUtensorMap* map, int n, int m, int z, uint32_t src) {
    if (m < rows_m && n < rows_n) store_box(map, n, m, z, src);
  };
  const auto box_written = [&] {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
  };
  const auto box_read = [&] {
    if (lane == 0) stores_read<0>();
    __syncwarp();
  };
  const auto half_read = [&] {
    if (lane == 0) stores_read<1>();
    __syncwarp();
  };
  uint32_t loads = 0;
  const auto load_extra = [&](const Item& t) {
    if (dead) return;
    ++loads;
    if constexpr (kSlope) {
      expect_bytes(arrived, kHalves * kBoxBytes / 2);
#pragma unroll
      for (int p = 0; p < kHalves; ++p)
        copy_box<1>(box + p * kBoxBytes / 2, &maps.extra, col_of(t) + p * kHalfCols, row_of(t), 0, arrived);
    } else {
      expect_bytes(arrived, 32 * kRowBytes);
      copy_box<1>(box, &maps.extra, col_of(t), row_of(t), 0, arrived);
    }
  };
  int buf = 0, small = 0;
  uint32_t acc_phase = 0, extra_phase = 0;
  Item t = first < items ? item_of<BN, CG>(job, first) : Item{};
  if (extra && first < items && lane == 0) load_extra(t);
  for (uint32_t i = first; i < items; i += step) {
    const int m = row_of(t), n0 = col_of(t);
    uint32_t acc_at = tmem + lanes + buf * BN + group * S::kCols;
    if (kF32) {
      float acc[S::kCols / 16][16] = {};
      for (int c = t.kb0, n = 1; c < t.kb1; c += chunk, ++n) {
        wait(acc_full(buf), acc_phase, dead);
        fence_after();
        const bool last = c + chunk >= t.kb1, fold = last || n % kFold == 0;
        const uint32_t main_at = tmem + lanes + buf * BN + group * S::kCols;
        acc_at = tmem + lanes + S::kSmall + small * BN + group * S::kCols;
#pragma unroll
        for (int q = 0; q < S::kCols / 16; ++q) {
          uint32_t r[16];
          tmem_load16(main_at + q * 16, r);
          tmem_wait(r);
#pragma unroll
          for (int x = 0; x < 16; ++x) acc[q][x] += __uint_as_float(r[x]);
        }
        if (fold) {
#pragma unroll
          for (int q = 0; q < S::kCols / 16; ++q) {
            uint32_t r[16];
            tmem_load16(acc_at + q * 16, r);
            tmem_wait(r);
#pragma unroll
            for (int x = 0; x < 16; ++x) acc[q][x] += finite_or_zero(__uint_as_float(r[x]));
            if (last) tmem_store16(acc_at + q * 16, acc[q]);  // the tile waits there for its epilogue
          }
        }
        fence_before();
        __syncwarp();
        if (lane == 0) {
          arrive_in(in_block(acc_empty(buf), 0));
          if (fold && !last) arrive_in(in_block(small_empty(small), 0));
        }
        if (fold && !last) small ^= 1;
        buf ^= 1;
        if (buf == 0) acc_phase ^= 1;
      }
      tmem_stored();
    } else {
      wait(acc_full(buf), acc_phase, dead);
      fence_after();
    }
    if (extra) {
      wait(arrived, extra_phase, dead);
      extra_phase ^= 1;
    }
    if constexpr (kSlope) {
      // Half a box for a part of y, half for a part of the slope, which waits in
      // tensor memory meanwhile: a half is written when all stores but the last
      // one have been read, so no part waits for the store just before it. (Whole
      // boxes in turn: float32, 22223 x 256 x 1024, 130 us; halves 122. In bfloat16
      // the bytes of y and the slope are the bound, 40000 x 256 x 512 37 us either way.)
#pragma unroll 1
      for (int p = 0; p < kHalves; ++p) {
        const int n = n0 + p * kHalfCols;
        const uint32_t half = box + p * kBoxBytes / 2;
        if (!extra) half_read();
#pragma unroll 1
        for (int c = 0; c < kHalfCols; c += 16) {
          const uint32_t at = acc_at + p * kHalfCols + c;
          float v[16], s[16];
          Bias16<T> bias;
          if (with_bias) bias.load(static_cast<const T*>(e.bias) + n + c, bias_vec, rows_n - n - c);
          tmem_take16(at, v);
          if (with_bias) bias.add(v);
          activate<kFast, true, true, 16>(kAct, v, s);
          put_aside(at, s, typename SlopeOf<T>::type());
          if (extra) {
            get16<64>(half, lane, c, s, T());
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j] += s[j];
          }
          put16<64>(half, lane, c, v, T());
        }
        box_written();
        if (lane == 0) {
          send(&maps.out, n, m, 0, half);
          stores_commit();
        }
      }
      tmem_stored();
#pragma unroll 1
      for (int p = 0; p < kHalves; ++p) {
        const uint32_t half = box + (kHalves == 1 ? 1 : p) * kBoxBytes / 2;
        half_read();
#pragma unroll 1
        for (int c = 0; c < kHalfCols; c += 16)
          take_back<64>(half, lane, c, acc_at + p * kHalfCols + c, typename SlopeOf<T>::type());
        box_written();
        if (lane == 0) {
          send(&maps.slope, n0 + p * kHalfCols, m, 0, half);
          stores_commit();
        }
      }
    }
#pragma unroll 1
    for (int p = 0; p < (kSlope ? 0 : kParts); ++p) {
      const int n = n0 + p * kBoxCols;
      if (!extra) box_read();
#pragma unroll 1
      for (int c = 0; c < kBoxCols; c += 16) {
        const uint32_t at = acc_at + p * kBoxCols + c;
        float x[16], v[16], s[16];
        Bias16<T> bias;
        if (kMode != Epilogue::kStore && with_bias)
          bias.load(static_cast<const T*>(e.bias) + n + c, bias_vec, rows_n - n - c);
        if (kExtra) get16<kRowBytes>(box, lane, c, x, T());
        tmem_take16(at, v);
        if (kMode != Epilogue::kStore && with_bias) bias.add(v);
        if (kMode == Epilogue::kDz) {
          activate<kFast, false, true, 16>(kAct, v, s);
#pragma unroll
          for (int j = 0; j < 16; ++j) v[j] = x[j] * s[j];
          if (e.sums) {
            if (m + lane >= rows_m) {  // rows of nothing: their gradient is zero, their slope may be anything
#pragma unroll
              for (int j = 0; j < 16; ++j) v[j] = 0.f;
            }
            const float sum = lane_sums16(v);
            const int col = n + c + lane / 2;
            if ((lane & 1) == 0 && m < rows_m && col < rows_n)
              e.sums[static_cast<int64_t>(m / 32) * rows_n + col] = sum;
          }
          if (sizeof(T) == 4) {
            tmem_store16(at, v);
            continue;
          }
        } else if (kMode == Epilogue::kFwd) {
          activate<kFast, true, false, 16>(kAct, v, s);
          if (kExtra) {
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j] += x[j];
          }
        }
        put16<kRowBytes>(box, lane, c, v, T());
      }
      if constexpr (kPlanes) {
        // dz waits in tensor memory: hi and mid take the gradient's place, then lo theirs
        tmem_stored();
        __syncwarp();
#pragma unroll 1
        for (int c = 0; c < kBoxCols; c += 16) {
          float v[16];
          uint32_t part[3][8];
          tmem_take16(acc_at + c, v);
          split_pairs<16>(v, top_bits<16>(v), part);
#pragma unroll
          for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int u = 0; u < 2; ++u)
              put_unit(unit_at<64>(box + 2048 * k, lane, c / 8 + u), part[k][4 * u], part[k][4 * u + 1],
                       part[k][4 * u + 2], part[k][4 * u + 3]);
          tmem_store8(acc_at + c, part[2]);
        }
        box_written();
        if (lane == 0) {
          send(&maps.out, n, m, 0, box);
          send(&maps.out, n, m, 1, box + 2048);
          stores_commit();
        }
        tmem_stored();
        box_read();
#pragma unroll 1
        for (int c = 0; c < kBoxCols; c += 16) take_back<64>(box, lane, c, acc_at + c, __half());
        box_written();
        if (lane == 0) {
          send(&maps.out, n, m, 2, box);
          stores_commit();
        }
      } else {
        box_written();
        if (lane == 0) {
          send(&maps.out, n, m, job.apart ? t.split : 0, box);
          stores_commit();
        }
      }
    }
    fence_before();
    __syncwarp();
    if (kF32) {
      if (lane == 0) arrive_in(in_block(small_empty(small), 0));
      small ^= 1;
    } else {
      if (lane == 0) arrive_in(in_block(acc_empty(buf), 0));
      buf ^= 1;
      if (buf == 0) acc_phase ^= 1;
    }
    if (i + step < items) {
      t = item_of<BN, CG>(job, i + step);
      if (extra && lane == 0) {
        stores_read<0>();
        load_extra(t);
      }
    }
  }
  if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  if (lane == 0 && dead && loads > 0) settle(arrived, (loads - 1) & 1);
  return dead;
}

// The epilogues of the linear operator, and of products that are stored as they are or as partial sums.
struct PlainEpilogue {
  static constexpr bool kGated = false;

  template <int BN, int CG, typename T, bool kF32>
  static __device__ __forceinline__ bool run(const Maps& maps, const Job& job, const Place place) {
    const Epilogue& e = job.pr.epi;
    const int mode = job.apart ? Epilogue::kStore : e.mode;
    const bool extra = mode != Epilogue::kStore && e.extra != nullptr;
    const int kind = mode == Epilogue::kFwd && e.slope ? kFwdSlope * 8 + static_cast<int>(e.act) * 2
                     : mode == Epilogue::kStore        ? Epilogue::kStore * 8
                                                       : mode * 8 + static_cast<int>(e.act) * 2 + (extra ? 1 : 0);
    if constexpr (sizeof(T) == 4 && !kF32) {  // partial sums
      return epilogue<BN, CG, T, kF32, Epilogue::kStore * 8>(maps, job, place);
    } else {
      switch (kind) {
        case Epilogue::kStore * 8: return epilogue<BN, CG, T, kF32, Epilogue::kStore * 8>(maps, job, place);
        case Epilogue::kFwd * 8: return epilogue<BN, CG, T, kF32, Epilogue::kFwd * 8>(maps, job, place);
        case Epilogue::kFwd * 8 + 1: return epilogue<BN, CG, T, kF32, Epilogue::kFwd * 8 + 1>(maps, job, place);
        case Epilogue::kFwd * 8 + 2: return epilogue<BN, CG, T, kF32, Epilogue::kFwd * 8 + 2>(maps, job, place);
        case Epilogue::kFwd * 8 + 3: return epilogue<BN, CG, T, kF32, Epilogue::kFwd * 8 + 3>(maps, job, place);
        case Epilogue::kFwd * 8 + 4: return epilogue<BN, CG, T, kF32, Epilogue::kFwd * 8 + 4>(maps, job, place);
        case Epilogue::kFwd * 8 + 5: return epilogue<BN, CG, T, kF32, Epilogue::kFwd * 8 + 5>(maps, job, place);
        case Epilogue::kFwd * 8 + 6: return epilogue<BN, CG, T, kF32, Epilogue::kFwd * 8 + 6>(maps, job, place);
        case Epilogue::kFwd * 8 + 7: return epilogue<BN, CG, T, kF32, Epilogue::kFwd * 8 + 7>(maps, job, place);
        case Epilogue::kDz * 8 + 3: return epilogue<BN, CG, T, kF32, Epilogue::kDz * 8 + 3>(maps, job, place);
        case Epilogue::kDz * 8 + 5: return epilogue<BN, CG, T, kF32, Epilogue::kDz * 8 + 5>(maps, job, place);
        case Epilogue::kDz * 8 + 7: return epilogue<BN, CG, T, kF32, Epilogue::kDz * 8 + 7>(maps, job, place);
        case kFwdSlope * 8 + 2: return epilogue<BN, CG, T, kF32, kFwdSlope * 8 + 2>(maps, job, place);
        case kFwdSlope * 8 + 4: return epilogue<BN, CG, T, kF32, kFwdSlope * 8 + 4>(maps, job, place);
        case kFwdSlope * 8 + 6: return epilogue<BN, CG, T, kF32, kFwdSlope * 8 + 6>(maps, job, place);
        default: return epilogue<BN, CG, T, kF32, kFwdSlope * 8>(maps, job, place);
      }
    }
  }

  template <int BN, int CG, typename T, bool kF32>
  static __device__ __noinline__ void spoil(const Maps& maps, const Job& job, const Place place) {
    using S = Shape<BN, CG, kF32>;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Epilogue& e = job.pr.epi;
    const int mode = job.apart ? Epilogue::kStore : e.mode;
    const bool slope = mode == Epilogue::kFwd && e.slope, planes = mode == Epilogue::kDz && sizeof(T) == 4;
    const int wide = 128 / sizeof(T) < S::kCols ? 128 / sizeof(T) : S::kCols;
    const int cols = slope ? 64 / sizeof(T) : planes ? 32 : wide;
    const uint32_t box = place.boxes + warp * kBoxBytes;
    for (int unit = lane; unit < kBoxBytes / 16; unit += 32) put_unit(box + unit * 16, ~0u, ~0u, ~0u, ~0u);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    const uint32_t items = job.tiles_m * job.tiles_n * job.splits;
    for (uint32_t i = blockIdx.x / CG; i < items; i += gridDim.x / CG) {
      const Item t = item_of<BN, CG>(job, i);
      const int m = t.m + static_cast<int>(place.rank) * kTileM + (warp & 3) * 32, n0 = t.n + (warp >> 2) * S::kCols;
      for (int n = n0; n < n0 + S::kCols; n += cols) {
        if (m >= job.pr.m || n >= job.pr.n) continue;
        if (lane == 0) {
          for (int z = 0; z < (planes ? 3 : 1); ++z) store_box(&maps.out, n, m, job.apart ? t.split : z, box);
          if (slope) store_box(&maps.slope, n, m, 0, box);
        }
        if (mode == Epilogue::kDz && e.sums)
          for (int c = lane; c < cols && n + c < job.pr.n; c += 32)
            e.sums[static_cast<int64_t>(m / 32) * job.pr.n + n + c] = __uint_as_float(~0u);
      }
    }
    if (lane == 0) {
      stores_commit();
      asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
  }
};

// Adds up the ranges of k and runs the epilogue: eight columns to kLanes lanes,
// which take the ranges in turn. The order of the additions is fixed.
template <typename T, int kLanes>
__global__ void __launch_bounds__(256) finish_kernel(const __grid_constant__ Job job) {
  const Product& pr = job.pr;
  const int64_t per_row = (pr.n + 7) / 8, total = pr.m * per_row, ld = partial_ld(pr.n);
  const int sub = threadIdx.x % kLanes;
  for (int64_t i = (blockIdx.x * 256ll + threadIdx.x) / kLanes; i - threadIdx.x % 32 / kLanes < total;
       i += gridDim.x * 256ll / kLanes) {
    const bool some = i < total;
    const int64_t m = some ? i / per_row : 0, n = some ? (i - m * per_row) * 8 : 0;
    float v[8] = {};
    if (some) {
      const float* p = pr.partial + m * ld + n;  // rows are padded to eight
#pragma unroll 4
      for (int s = sub; s < job.splits; s += kLanes) {
        float w[8];
        load8(p + s * pr.m * ld, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] += w[j];
      }
    }
#pragma unroll
    for (int d = 1; d < kLanes; d <<= 1)
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] += __shfl_xor_sync(0xffffffffu, v[j], d);
    if (!some || sub != 0) continue;
    if (job.vec && n + 8 <= pr.n) {
      float x[8] = {}, b[8] = {};
      if (pr.epi.bias) load_some(static_cast<const T*>(pr.epi.bias) + n, 8, false, b);
      if (pr.epi.extra) load8(static_cast<const T*>(pr.epi.extra) + m * pr.epi.extra_ld + n, x);
      finish8<T>(pr.epi, v, x, b, m, n, pr.n, 8, true);
    } else {
      finish_some<T>(pr.epi, make_float4(v[0], v[1], v[2], v[3]), make_float4(v[4], v[5], v[6], v[7]), m, n, pr.n);
    }
  }
}

// The columns' sums over 32 rows of what a finished epilogue left before its rounding.
__global__ void __launch_bounds__(256) sums_kernel(const __grid_constant__ Job job) {
  const Product& pr = job.pr;
  const int64_t total = (pr.m + 31) / 32 * pr.n, ld = partial_ld(pr.n);
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
    const int64_t part = i / pr.n, n = i - part * pr.n;
    float s = 0.f;
    for (int64_t m = part * 32; m < min(pr.m, part * 32 + 32); ++m) s += pr.epi.unrounded[m * ld + n];
    pr.epi.sums[i] = s;
  }
}

// ---- host --------------------------------------------------------------------------------

// The maps of the epilogue's outputs and of the residual or gradient.
bool epilogue_maps(Maps& maps, const Product& pr, const Plan& plan, bool apart) {
  const Epilogue& e = pr.epi;
  const auto f32 = CU_TENSOR_MAP_DATA_TYPE_FLOAT32, b16 = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  if (apart)
    return make_map(&maps.out, f32, pr.partial, pr.n, pr.m, plan.splits, partial_ld(pr.n) * 4,
                    pr.m * partial_ld(pr.n) * 4, 32, 32, 128);
  const bool wide = pr.dtype == DType::kF32;
  const int64_t size = wide ? 4 : 2;
  const bool slope = e.mode == Epilogue::kFwd && e.slope;
  const int row_bytes = slope ? 64 : std::min<int>(128, std::max(32, plan.bn / 4) * static_cast<int>(size));
  const int cols = row_bytes / static_cast<int>(size);
  bool ok = true;
  if (e.mode == Epilogue::kDz && wide)
    ok = make_map(&maps.out, b16, e.out, pr.n, pr.m, 3, e.out_ld * 2, e.out_plane * 2, 32, 32, 64);
  else
    ok = make_map(&maps.out, wide ? f32 : b16, e.out, pr.n, pr.m, 1, e.out_ld * size, 0, cols, 32, row_bytes);
  if (ok && e.mode != Epilogue::kStore && e.extra)
    ok = make_map(&maps.extra, wide ? f32 : b16, e.extra, pr.n, pr.m, 1, e.extra_ld * size, 0, cols, 32, row_bytes);
  if (ok && slope)
    ok = make_map(&maps.slope, wide ? f32 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, e.slope, pr.n, pr.m, 1, pr.n * size, 0,
                  cols, 32, row_bytes);
  return ok;
}

// Whether rows of extra, out and slope are what TMA and vectors of eight columns can address.
bool vectors_fit(const Product& pr) {
  const Epilogue& e = pr.epi;
  const int64_t size = pr.dtype == DType::kF32 ? 4 : 2;
  bool ok = aligned16(e.out) && (e.out_ld * (e.out_plane ? 2 : size)) % 16 == 0 && (e.out_plane * 2) % 16 == 0;
  if (e.extra) ok = ok && aligned16(e.extra) && (e.extra_ld * size) % 16 == 0 && e.extra_ld >= pr.n;
  if (e.slope) ok = ok && aligned16(e.slope) && (pr.n * size) % 16 == 0;
  return ok;
}

template <typename T, bool kF32>
cudaError_t launch_tile(const Plan& plan, const Maps& maps, const Job& job, int sms, cudaStream_t stream) {
  if constexpr (kF32) {
    if (plan.bn == 128) return launch<128, 2, T, kF32, PlainEpilogue>(maps, job, sms, stream);
  } else {
    if (plan.bn == 256)
      return plan.pair == 2 ? launch<256, 2, T, kF32, PlainEpilogue>(maps, job, sms, stream)
                            : launch<256, 1, T, kF32, PlainEpilogue>(maps, job, sms, stream);
    if (plan.bn == 128) return launch<128, 1, T, kF32, PlainEpilogue>(maps, job, sms, stream);
  }
  return launch<64, 1, T, kF32, PlainEpilogue>(maps, job, sms, stream);
}

}  // namespace

// The tile and the ranges of k with the shortest estimated time, in clocks of
// one SM: a stage costs the longer of its products (2 clocks per column) and
// its copies (64 bytes a clock), tiles overlap with the epilogue of the one
// before, and partial sums cost their trip through L2 and a second launch.
// Both sides of its choice, us: float32 900 x 256 x 1024 with 64 columns 12.4,
// with 128 14.3; 2221 x 771 x 517 53.5 and 36.4; bfloat16 40000 x 256 x 512 with
// 128 columns 33.6, with 256 30.3.
Plan plan_product(DType dtype, int64_t m, int64_t n, int64_t k, int pairs, int sms) {
  const bool f32 = dtype == DType::kF32;
  const int kblocks = static_cast<int>(ceil_div(k, kBlockK));
  Plan best{64, 1, 1, kblocks};
  if (m == 0 || n == 0 || k == 0) return best;
  double best_time = 1e300;
  const struct {
    int bn, pair;
    bool bf16, f32;
  } shapes[] = {{64, 1, true, true}, {128, 1, true, false}, {128, 2, false, true}, {256, 1, true, false}, {256, 2, true, false}};
  for (const auto& s : shapes) {
    if (!(f32 ? s.f32 : s.bf16)) continue;
    const int64_t tiles = ceil_div(m, kTileM * s.pair) * ceil_div(n, s.bn);
    const int64_t slots = sms / s.pair;
    const double stage = std::max(2.0 * s.bn * pairs, (f32 ? 3 : 1) * (kStageA + s.bn * 128.0 / s.pair) / 64.0);
    const double epilogue = 8.0 * s.bn + 600.0;
    for (int splits = 1; splits <= std::min(kblocks, 64); splits = splits < 4 ? splits + 1 : splits * 5 / 4) {
      const int per = static_cast<int>(ceil_div(kblocks, splits));
      if (ceil_div(kblocks, per) != splits) continue;  // empty ranges
      const double waves = static_cast<double>(ceil_div(tiles * splits, slots));
      double time = waves * std::max(per * stage, epilogue) + std::min(per * stage, epilogue) + 2500.0;
      if (splits > 1) time += 4000.0 + (splits * 8.0 + 4.0) * m * n / 4000.0;
      if (time < best_time) {
        best_time = time;
        best = Plan{s.bn, s.pair, splits, per};
      }
    }
  }
  return best;
}

bool finished_apart(const Product& pr, const Plan& plan) { return plan.splits > 1 || pr.k == 0 || !vectors_fit(pr); }

namespace {

cudaError_t launch_tiles(Job& job, const Plan& plan, cudaStream_t stream) {
  const Product& pr = job.pr;
  int sms = 148;
  const cudaError_t err = prepare(job, plan, plan.bn, &sms);
  if (err != cudaSuccess) return err;
  const int64_t rows_b = plan.bn / plan.pair;
  job.box_a = pr.a_mn ? 64 : static_cast<int>(std::min<int64_t>(kTileM, ceil_div(pr.m, 8) * 8));
  job.box_b = pr.b_mn ? 64 : static_cast<int>(std::min<int64_t>(rows_b, ceil_div(pr.n, 8) * 8));
  Maps maps{};
  if (!operand_map(&maps.a, pr.a, job.box_a) || !operand_map(&maps.b, pr.b, job.box_b) ||
      !epilogue_maps(maps, pr, plan, job.apart))
    return cudaErrorInvalidValue;
  if (pr.dtype == DType::kF32) return launch_tile<float, true>(plan, maps, job, sms, stream);
  return job.apart ? launch_tile<float, false>(plan, maps, job, sms, stream)
                   : launch_tile<bf16, false>(plan, maps, job, sms, stream);
}

}  // namespace

cudaError_t launch_sums(const Product& pr, const Plan& plan, cudaStream_t stream) {
  Job job{};
  job.pr = pr;
  job.splits = plan.splits;
  job.apart = true;
  return launch_tiles(job, plan, stream);
}

cudaError_t launch_product(const Product& pr, const Plan& plan, cudaStream_t stream) {
  if (pr.m == 0 || pr.n == 0) return cudaSuccess;
  Job job{};
  job.pr = pr;
  job.vec = vectors_fit(pr);
  job.splits = plan.splits;
  const bool f32 = pr.dtype == DType::kF32;
  if (pr.k > 0) {
    job.apart = finished_apart(pr, plan);
    const cudaError_t err = launch_tiles(job, plan, stream);
    if (err != cudaSuccess || !job.apart) return err;
  } else {
    job.splits = 0;  // an empty sum
  }
  // in the place of the first range's sums, which a thread has read before it writes there
  const bool sums = pr.epi.mode == Epilogue::kDz && pr.epi.sums;
  if (sums) job.pr.epi.unrounded = pr.partial;
  const int64_t groups = pr.m * ((pr.n + 7) / 8);
  const bool spread = job.splits >= 8;
  const int blocks = static_cast<int>(std::min<int64_t>((groups * (spread ? 8 : 1) + 255) / 256, 148 * 8));
  if (f32)
    (spread ? finish_kernel<float, 8> : finish_kernel<float, 1>)<<<blocks, 256, 0, stream>>>(job);
  else
    (spread ? finish_kernel<bf16, 8> : finish_kernel<bf16, 1>)<<<blocks, 256, 0, stream>>>(job);
  if (sums) {
    const int count = static_cast<int>(std::min<int64_t>(((pr.m + 31) / 32 * pr.n + 255) / 256, 148 * 8));
    sums_kernel<<<count, 256, 0, stream>>>(job);
  }
  return cudaGetLastError();
}

cudaError_t wait_timeouts(unsigned int* count) { return async::read_timeouts(count); }

}  // namespace lin
