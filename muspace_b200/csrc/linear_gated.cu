// The gated product: z = x W^T + b with W's rows [0, n) the gate's and [n, 2 n) up's,
// and of every pair of neighbours in it, y = D(act(z_gate) * z_up), in one kernel.
//
// A tile's columns are a range of the gate's and, behind them, the same range of up's:
// one tcgen05.mma multiplies both, and the lane that holds a row's gate sums in tensor
// memory holds its up sums too, BN / 2 columns on. In a pair of SMs each copies the
// half of the weight's rows that it would anyway: the first the gate's, the second
// up's. So the product is that of linear_gemm.cu, and nothing of size rows x 2 n is
// written in inference. For training the epilogue also writes the factors P = D'(act'(z_gate)
// z_up) and Q = D'(act(z_gate)) (D' multiplies as D does), by which a gradient of y becomes
// those of the gate's and of up's columns: the backward pass needs no generator, no
// exponential and no product for them. Beside bfloat16 they are kept in float16, each
// eight neighbours under an exponent of their own. A dropped element's Q is a NaN of its own, so
// that a gradient that is not finite is left out there and nowhere else.
//
// 8192 x 4096 x 4096 bfloat16 380 us (1.45 PFLOP/s), with factors 410. Where k is short the
// epilogue is the bound, by issue and latencies: 40000 x 256 x 512
// bfloat16 gelu 43 us, with factors and dropout 68; 22223 x 256 x 512 float32 silu with
// factors 92, where products of 128 columns take the time of 256.
#include <algorithm>

#include "dropout_device.cuh"
#include "linear_tile.cuh"

namespace lin {
namespace {

// Eight columns of this warp's 32 lanes of tensor memory, without waiting for them.
__device__ __forceinline__ void ask8(uint32_t addr, uint32_t r[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(addr)
               : "memory");
}

// The loads so far have arrived; the registers pass through, so none is read before.
__device__ __forceinline__ void arrived8(uint32_t r[8]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7])
               :
               : "memory");
}

// Bias of eight columns, the same for all lanes: asked for before the sums it is added to have come.
template <typename T>
struct Bias8 {
  uint4 u[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p, bool vec, int count) {
    if (vec && count >= 8) {
#pragma unroll
      for (int k = 0; k < static_cast<int>(sizeof(T) / 2); ++k) u[k] = __ldg(reinterpret_cast<const uint4*>(p) + k);
    } else {
      float b[8];
      load_some(p, count, false, b);
      store8(reinterpret_cast<T*>(u), b);
    }
  }
  __device__ __forceinline__ void add(float v[8]) const {
    float b[8];
    load8(reinterpret_cast<const T*>(u), b);
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      const float2 s = add2(make_float2(v[j], v[j + 1]), make_float2(b[j], b[j + 1]));
      v[j] = s.x, v[j + 1] = s.y;
    }
  }
};

// Eight values of a row into the box from column `col` on.
template <int kRowBytes>
__device__ __forceinline__ void put8(uint32_t box, int row, int col, const uint32_t w[4]) {
  put_unit(unit_at<kRowBytes>(box, row, col / 8), w[0], w[1], w[2], w[3]);
}
template <int kRowBytes>
__device__ __forceinline__ void put8(uint32_t box, int row, int col, const float v[8]) {
#pragma unroll
  for (int u = 0; u < 2; ++u)
    put_unit(unit_at<kRowBytes>(box, row, col / 4 + u), __float_as_uint(v[4 * u]), __float_as_uint(v[4 * u + 1]),
             __float_as_uint(v[4 * u + 2]), __float_as_uint(v[4 * u + 3]));
}

// Of eight gate sums g and up sums u, both with their bias: the output in g, and with
// kTrain P in s and Q in u, where what is dropped is marked. `words`: the eight's random
// numbers, with dropout. float32.
template <bool kTrain>
__device__ __forceinline__ void gate_values(Act act, const drop::Rule& rule, const drop::Key& key,
                                            const drop::Words& words, float g[8], float u[8], float s[8]) {
  activate<false, true, kTrain, 8>(act, g, s);
  if (rule.threshold) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const bool kept = drop::kept(key, words, j);
      g[j] = kept ? g[j] : 0.f;
      u[j] = kept ? u[j] * rule.scale : 0.f;
      if (kTrain) s[j] = kept ? s[j] : 0.f;
    }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float y = g[j] * u[j];
    if (kTrain) s[j] *= u[j], u[j] = g[j] * rule.scale;
    g[j] = y;
  }
  if (kTrain && rule.threshold) {
#pragma unroll
    for (int j = 0; j < 8; ++j) u[j] = drop::kept(key, words, j) ? u[j] : __uint_as_float(kDroppedFloat);
  }
}

// The same in bfloat16, packed: two columns to a word, and what is dropped is masked there
// (40000 x 256 x 512 gelu 68 us; with three selects a column and the mark by itself 79). Returns P's exponent and, from bit
// 16 on, Q's; the largest of eight, to which they are scaled, may be one that is dropped.
template <bool kTrain>
__device__ __forceinline__ uint32_t gate_words(Act act, const drop::Rule& rule, const drop::Key& key,
                                               const drop::Words& words, float g[8], float u[8], uint32_t y[4],
                                               uint32_t p[4], uint32_t q[4]) {
  float s[8];
  uint32_t exps = 0;
  activate<true, true, kTrain, 8>(act, g, s);
  const float2 scale = both(rule.scale);
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    const float2 a = make_float2(g[j], g[j + 1]), b = mul2(make_float2(u[j], u[j + 1]), scale), v = mul2(a, b);
    y[j / 2] = pack2(v.x, v.y);
    if (kTrain) {
      const float2 to_gate = mul2(make_float2(s[j], s[j + 1]), b), to_up = mul2(a, scale);
      s[j] = to_gate.x, s[j + 1] = to_gate.y;
      g[j] = to_up.x, g[j + 1] = to_up.y;
    }
  }
  if (kTrain) exps = pack_factors8(s, p) | pack_factors8(g, q) << 16;
  if (rule.threshold) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t low = drop::kept(key, words, 2 * j) ? 0xffffu : 0u;
      const uint32_t keep = drop::kept(key, words, 2 * j + 1) ? low | 0xffff0000u : low;
      y[j] &= keep;
      if (kTrain) p[j] &= keep, q[j] = (q[j] & keep) | (~keep & (kDroppedHalf | kDroppedHalf << 16));
    }
  }
  return exps;
}

// kKind: the activation, twice, and one more in training.
template <int BN, int CG, typename T, bool kF32, int kKind>
__device__ __noinline__ bool gated_epilogue(const Maps& maps, const Job& job, const Place place) {
  using S = Shape<BN, CG, kF32, true>;
  constexpr Act kAct = static_cast<Act>(kKind / 2);
  constexpr bool kTrain = kKind % 2;
  constexpr int kOut = S::kCols / 2;  // columns of the output that a warp takes
  constexpr int kRowBytes = kOut * sizeof(T), kPart = 32 * kRowBytes;
  static_assert(kRowBytes == 32 || kRowBytes == 64, "three boxes to a warp");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t tmem = place.tmem, rank = place.rank;
  const auto acc_full = [&](int b) { return place.bars + 8 * (2 * S::kStages + b); };
  const auto acc_empty = [&](int b) { return place.bars + 8 * (2 * S::kStages + 2 + b); };
  const auto small_empty = [&](int b) { return place.bars + 8 * (2 * S::kStages + 4 + kEpiWarps + b); };
  const uint32_t items = job.tiles_m * job.tiles_n * job.splits;
  const uint32_t first = blockIdx.x / CG, step = gridDim.x / CG;
  const int chunk = kF32 ? kPromote : job.kblocks;
  const int quad = warp & 3, group = warp >> 2;
  const uint32_t box = place.boxes + warp * S::kBox;
  const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
  const int rows_m = static_cast<int>(job.pr.m), rows_n = static_cast<int>(job.pr.n);
  const Epilogue& e = job.pr.epi;
  const T* bias_gate = static_cast<const T*>(e.bias);
  const T* bias_up = bias_gate + rows_n;
  const bool with_bias = bias_gate != nullptr;
  const bool bias_vec = reinterpret_cast<uintptr_t>(bias_gate) % 16 == 0 && rows_n * sizeof(T) % 16 == 0;
  const drop::Key key = drop::key_of(e.rule);
  // the warp's q-th sixteen columns of an accumulator: first the gate's, then up's
  const auto sixteen = [&](int q) {
    return q < kOut / 16 ? group * kOut + q * 16 : BN / 2 + group * kOut + (q - kOut / 16) * 16;
  };
  bool dead = false;
  int buf = 0, small = 0, part = 0;
  uint32_t acc_phase = 0;
  for (uint32_t i = first; i < items; i += step) {
    const Item t = item_of<S::kTileN, CG>(job, i);
    const int m = t.m + static_cast<int>(rank) * kTileM + quad * 32, n0 = t.n + group * kOut;
    uint32_t acc_at = tmem + lanes + buf * BN;
    if (kF32) {  // as in linear_gemm.cu's epilogue
      float acc[S::kCols / 16][16] = {};
      for (int c = t.kb0, n = 1; c < t.kb1; c += chunk, ++n) {
        wait(acc_full(buf), acc_phase, dead);
        fence_after();
        const bool last = c + chunk >= t.kb1, fold = last || n % kFold == 0;
        const uint32_t main_at = tmem + lanes + buf * BN;
        acc_at = tmem + lanes + S::kSmall + small * BN;
#pragma unroll
        for (int q = 0; q < S::kCols / 16; ++q) {
          uint32_t r[16];
          tmem_load16(main_at + sixteen(q), r);
          tmem_wait(r);
#pragma unroll
          for (int x = 0; x < 16; ++x) acc[q][x] += __uint_as_float(r[x]);
        }
        if (fold) {
#pragma unroll
          for (int q = 0; q < S::kCols / 16; ++q) {
            uint32_t r[16];
            tmem_load16(acc_at + sixteen(q), r);
            tmem_wait(r);
#pragma unroll
            for (int x = 0; x < 16; ++x) acc[q][x] += finite_or_zero(__uint_as_float(r[x]));
            if (last) tmem_store16(acc_at + sixteen(q), acc[q]);  // the tile waits there for its epilogue
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
    // training: the three boxes at once; inference: one after the other, two on their way out meanwhile
    if (lane == 0) stores_read<kTrain ? 0 : 2>();
    __syncwarp();
    const uint32_t out = kTrain ? box : box + part * kPart;
    const uint32_t gate_at = acc_at + group * kOut, up_at = gate_at + BN / 2;
    uint32_t next_g[8], next_u[8];
    ask8(gate_at, next_g);
    ask8(up_at, next_u);
    uint32_t exps_p = 0, exps_q = 0;  // a byte to eight columns, the first one lowest
#pragma unroll 1
    for (int c = 0; c < kOut; c += 8) {  // sixteen at a time spill: 83 us and 75 without exponents, float32 22223 x 256 x 512 122 and 92
      float g[8], u[8];
      Bias8<T> here_g, here_u;
      if (with_bias) {
        here_g.load(bias_gate + n0 + c, bias_vec, rows_n - n0 - c);
        here_u.load(bias_up + n0 + c, bias_vec, rows_n - n0 - c);
      }
      drop::Words words;
      if (e.rule.threshold) words = drop::numbers(key, m + lane, (n0 + c) / 8);
      arrived8(next_g);
      arrived8(next_u);
#pragma unroll
      for (int j = 0; j < 8; ++j) g[j] = __uint_as_float(next_g[j]), u[j] = __uint_as_float(next_u[j]);
      const int ahead = c + 8 < kOut ? c + 8 : c;  // the last eight are asked for again
      ask8(gate_at + ahead, next_g);
      ask8(up_at + ahead, next_u);
      if (with_bias) here_g.add(g), here_u.add(u);
      if constexpr (sizeof(T) == 2) {
        uint32_t y[4], p[4], q[4];
        const uint32_t exps = gate_words<kTrain>(kAct, e.rule, key, words, g, u, y, p, q);
        put8<kRowBytes>(out, lane, c, y);
        if (kTrain) {
          exps_p |= (exps & 0xffffu) << c, exps_q |= (exps >> 16) << c;
          put8<kRowBytes>(box + kPart, lane, c, p);
          put8<kRowBytes>(box + 2 * kPart, lane, c, q);
        }
      } else {
        float s[8];
        gate_values<kTrain>(kAct, e.rule, key, words, g, u, s);
        put8<kRowBytes>(out, lane, c, g);
        if (kTrain) {
          put8<kRowBytes>(box + kPart, lane, c, s);
          put8<kRowBytes>(box + 2 * kPart, lane, c, u);
        }
      }
    }
    if (kTrain && sizeof(T) == 2 && m + lane < rows_m && n0 < rows_n) {
      uint8_t *at_p = e.exponents + exponent_at(rows_m, rows_n, 0, m + lane, n0),
              *at_q = e.exponents + exponent_at(rows_m, rows_n, 1, m + lane, n0);
      if (kOut == 32)
        *reinterpret_cast<uint32_t*>(at_p) = exps_p, *reinterpret_cast<uint32_t*>(at_q) = exps_q;
      else
        *reinterpret_cast<uint16_t*>(at_p) = exps_p, *reinterpret_cast<uint16_t*>(at_q) = exps_q;
    }
    arrived8(next_g);
    arrived8(next_u);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    fence_before();
    __syncwarp();
    if (lane == 0) {
      if (m < rows_m && n0 < rows_n) {
        store_box(&maps.out, n0, m, 0, out);
        if (kTrain) {
          store_box(&maps.extra, n0, m, 0, box + kPart);
          store_box(&maps.slope, n0, m, 0, box + 2 * kPart);
        }
      }
      stores_commit();
      arrive_in(in_block(kF32 ? small_empty(small) : acc_empty(buf), 0));
    }
    if (kF32) {
      small ^= 1;
    } else {
      buf ^= 1;
      if (buf == 0) acc_phase ^= 1;
    }
    if (++part == 3) part = 0;
  }
  if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  return dead;
}

struct GatedEpilogue {
  static constexpr bool kGated = true;

  template <int BN, int CG, typename T, bool kF32>
  static __device__ __forceinline__ bool run(const Maps& maps, const Job& job, const Place place) {
    const Epilogue& e = job.pr.epi;
    switch (static_cast<int>(e.act) * 2 + (e.slope ? 1 : 0)) {
      case 0: return gated_epilogue<BN, CG, T, kF32, 0>(maps, job, place);
      case 1: return gated_epilogue<BN, CG, T, kF32, 1>(maps, job, place);
      case 2: return gated_epilogue<BN, CG, T, kF32, 2>(maps, job, place);
      case 3: return gated_epilogue<BN, CG, T, kF32, 3>(maps, job, place);
      case 4: return gated_epilogue<BN, CG, T, kF32, 4>(maps, job, place);
      case 5: return gated_epilogue<BN, CG, T, kF32, 5>(maps, job, place);
      case 6: return gated_epilogue<BN, CG, T, kF32, 6>(maps, job, place);
      default: return gated_epilogue<BN, CG, T, kF32, 7>(maps, job, place);
    }
  }

  template <int BN, int CG, typename T, bool kF32>
  static __device__ __noinline__ void spoil(const Maps& maps, const Job& job, const Place place) {
    using S = Shape<BN, CG, kF32, true>;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t box = place.boxes + warp * S::kBox;
    for (int unit = lane; unit < S::kBox / 16; unit += 32) put_unit(box + unit * 16, ~0u, ~0u, ~0u, ~0u);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if (lane != 0) return;
    const uint32_t items = job.tiles_m * job.tiles_n * job.splits;
    for (uint32_t i = blockIdx.x / CG; i < items; i += gridDim.x / CG) {
      const Item t = item_of<S::kTileN, CG>(job, i);
      const int m = t.m + static_cast<int>(place.rank) * kTileM + (warp & 3) * 32, n = t.n + (warp >> 2) * (S::kCols / 2);
      if (m >= job.pr.m || n >= job.pr.n) continue;
      store_box(&maps.out, n, m, 0, box);
      if (job.pr.epi.slope) {
        store_box(&maps.extra, n, m, 0, box);
        store_box(&maps.slope, n, m, 0, box);
      }
    }
    stores_commit();
    asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }
};

// Up to eight packed values of 16 bits.
__device__ __forceinline__ void put_words(void* at, int count, bool vec, const uint32_t w[4]) {
  if (vec) {
    *static_cast<uint4*>(at) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < count) static_cast<unsigned short*>(at)[j] = static_cast<unsigned short>(w[j / 2] >> (16 * (j % 2)));
  }
}

// The same from sums that were finished apart, [splits, m, partial_ld(2 n)]: eight
// columns to kLanes lanes, which take the ranges of k in turn, in a fixed order.
template <typename T, int kLanes>
__global__ void __launch_bounds__(256) gated_finish_kernel(const __grid_constant__ Job job) {
  const Product& pr = job.pr;
  const Epilogue& e = pr.epi;
  const int64_t per_row = (pr.n + 7) / 8, total = pr.m * per_row, ld = partial_ld(2 * pr.n);
  const int sub = threadIdx.x % kLanes;
  const bool up_vec = pr.n % 4 == 0;
  const drop::Key key = drop::key_of(e.rule);
  for (int64_t i = (blockIdx.x * 256ll + threadIdx.x) / kLanes; i - threadIdx.x % 32 / kLanes < total;
       i += gridDim.x * 256ll / kLanes) {
    const bool some = i < total;
    const int64_t m = some ? i / per_row : 0, n = some ? (i - m * per_row) * 8 : 0;
    const int count = static_cast<int>(pr.n - n < 8 ? pr.n - n : 8);
    float g[8] = {}, u[8] = {}, s[8];
    if (some) {
      const float* p = pr.partial + m * ld + n;  // rows are padded to eight
#pragma unroll 2
      for (int split = sub; split < job.splits; split += kLanes) {
        float w[8], x[8];
        load8(p + split * pr.m * ld, w);
        load_some(p + split * pr.m * ld + pr.n, count, up_vec && count == 8, x);
#pragma unroll
        for (int j = 0; j < 8; ++j) g[j] += w[j], u[j] += x[j];
      }
    }
#pragma unroll
    for (int d = 1; d < kLanes; d <<= 1)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        g[j] += __shfl_xor_sync(0xffffffffu, g[j], d);
        u[j] += __shfl_xor_sync(0xffffffffu, u[j], d);
      }
    if (!some || sub != 0) continue;
    const bool vec = job.vec && count == 8;
    if (e.bias) {
      float b[8];
      load_some(static_cast<const T*>(e.bias) + n, count, false, b);
#pragma unroll
      for (int j = 0; j < 8; ++j) g[j] += b[j];
      load_some(static_cast<const T*>(e.bias) + pr.n + n, count, false, b);
#pragma unroll
      for (int j = 0; j < 8; ++j) u[j] += b[j];
    }
    drop::Words words;
    if (e.rule.threshold) words = drop::numbers(key, static_cast<uint32_t>(m), static_cast<uint32_t>(n / 8));
    T* out = static_cast<T*>(e.out) + m * e.out_ld + n;
    if constexpr (sizeof(T) == 4) {
      gate_values<true>(e.act, e.rule, key, words, g, u, s);
      store_some(out, count, vec, g);
      if (e.slope) {
        float* factors = static_cast<float*>(e.slope) + m * 2 * pr.n + n;
        store_some(factors, count, vec, s);
        store_some(factors + pr.n, count, vec, u);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j >= count) g[j] = u[j] = 0.f;  // beyond the row
      uint32_t y[4], p[4], q[4];
      const uint32_t exps = gate_words<true>(e.act, e.rule, key, words, g, u, y, p, q);
      put_words(out, count, vec, y);
      if (e.slope) {
        __half* factors = static_cast<__half*>(e.slope) + m * 2 * pr.n + n;
        put_words(factors, count, vec, p);
        put_words(factors + pr.n, count, vec, q);
        e.exponents[exponent_at(pr.m, pr.n, 0, m, n)] = static_cast<uint8_t>(exps);
        e.exponents[exponent_at(pr.m, pr.n, 1, m, n)] = static_cast<uint8_t>(exps >> 16);
      }
    }
  }
}

// Whether rows of out and of both halves of the factors are what TMA and vectors of eight columns can address.
bool gated_fits(const Product& pr) {
  const Epilogue& e = pr.epi;
  const int64_t size = pr.dtype == DType::kF32 ? 4 : 2;
  bool ok = aligned16(e.out) && (e.out_ld * size) % 16 == 0;
  if (e.slope) ok = ok && aligned16(e.slope) && (pr.n * size) % 16 == 0;
  return ok;
}

template <typename T, bool kF32>
cudaError_t launch_gated_tile(const Plan& plan, const Maps& maps, const Job& job, int sms, cudaStream_t stream) {
  if constexpr (kF32) {
    if (plan.bn == 128) return launch<128, 2, T, kF32, GatedEpilogue>(maps, job, sms, stream);
  } else {
    if (plan.bn == 256)
      return plan.pair == 2 ? launch<256, 2, T, kF32, GatedEpilogue>(maps, job, sms, stream)
                            : launch<256, 1, T, kF32, GatedEpilogue>(maps, job, sms, stream);
    if (plan.bn == 128) return launch<128, 1, T, kF32, GatedEpilogue>(maps, job, sms, stream);
  }
  return launch<64, 1, T, kF32, GatedEpilogue>(maps, job, sms, stream);
}

}  // namespace

bool gated_apart(const Product& pr, const Plan& plan) { return plan.splits > 1 || pr.k == 0 || !gated_fits(pr); }

cudaError_t launch_gated(const Product& pr, const Plan& plan, cudaStream_t stream) {
  if (pr.m == 0 || pr.n == 0) return cudaSuccess;
  const bool f32 = pr.dtype == DType::kF32;
  Job job{};
  job.pr = pr;
  job.vec = gated_fits(pr);
  job.splits = plan.splits;
  if (!gated_apart(pr, plan)) {
    int sms = 148;
    const cudaError_t err = prepare(job, plan, plan.bn / 2, &sms);
    if (err != cudaSuccess) return err;
    job.box_a = static_cast<int>(std::min<int64_t>(kTileM, ceil_div(pr.m, 8) * 8));
    job.box_b = static_cast<int>(std::min<int64_t>(plan.bn / 2, ceil_div(pr.n, 8) * 8));
    const Epilogue& e = pr.epi;
    const auto type = f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    const int64_t size = f32 ? 4 : 2;
    const int cols = std::max(32, plan.bn / 4) / 2, row_bytes = cols * static_cast<int>(size);
    Maps maps{};
    bool ok = operand_map(&maps.a, pr.a, job.box_a) && operand_map(&maps.b, pr.b, job.box_b) &&
              make_map(&maps.out, type, e.out, pr.n, pr.m, 1, e.out_ld * size, 0, cols, 32, row_bytes);
    if (e.slope)
      ok = ok &&
           make_map(&maps.extra, type, e.slope, pr.n, pr.m, 1, 2 * pr.n * size, 0, cols, 32, row_bytes) &&
           make_map(&maps.slope, type, static_cast<char*>(e.slope) + pr.n * size, pr.n, pr.m, 1, 2 * pr.n * size, 0, cols,
                    32, row_bytes);
    if (!ok) return cudaErrorInvalidValue;
    return f32 ? launch_gated_tile<float, true>(plan, maps, job, sms, stream)
               : launch_gated_tile<bf16, false>(plan, maps, job, sms, stream);
  }
  if (pr.k > 0) {
    Product sums = pr;
    sums.n = 2 * pr.n;
    const cudaError_t err = launch_sums(sums, plan, stream);
    if (err != cudaSuccess) return err;
  } else {
    job.splits = 0;  // an empty sum
  }
  const int64_t groups = pr.m * ((pr.n + 7) / 8);
  const bool spread = job.splits >= 8;
  const int blocks = static_cast<int>(std::min<int64_t>((groups * (spread ? 8 : 1) + 255) / 256, 148 * 8));
  if (f32)
    (spread ? gated_finish_kernel<float, 8> : gated_finish_kernel<float, 1>)<<<blocks, 256, 0, stream>>>(job);
  else
    (spread ? gated_finish_kernel<bf16, 8> : gated_finish_kernel<bf16, 1>)<<<blocks, 256, 0, stream>>>(job);
  return cudaGetLastError();
}

cudaError_t gated_wait_timeouts(unsigned int* count) { return async::read_timeouts(count); }

}  // namespace lin
