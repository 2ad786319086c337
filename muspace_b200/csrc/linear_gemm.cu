// The product D[m, n] = sum_k A(m, k) B(n, k) of the fused linear operator on
// the fifth-generation tensor cores, with the operator's epilogues.
//
// One persistent block per SM (or a pair of them on two SMs) of ten warps:
// a producer thread copies tiles of A and B into a ring of shared-memory stages
// (TMA, 128-byte swizzle), one thread issues tcgen05.mma on them into one of
// two accumulators in tensor memory, and eight warps carry the other
// accumulator through the epilogue meanwhile: tensor memory -> registers ->
// shared memory, turned so that neighbouring lanes hold neighbouring columns ->
// bias, activation, residual -> global memory.
//
// Either operand may be stored along k or across it: the forward reads both
// along k, dx = dz W reads W across it, dW = dz^T x both. Nothing is transposed
// in memory; the instruction and the tile's layout differ.
//
// float32 (three bfloat16 planes an operand): the same loop runs over the six
// products of planes that reach 2^-24 of the result. The tensor core's float32
// accumulator cuts where an FMA would round: 2^-25 of the result per step on
// average, always towards zero. So the small products go first, and the sums
// over 128 of k at a time are added up in registers: relative error 2.9e-6 with
// 256 of k and the large products first, see planes_of.
#include <cuda.h>  // CUtensorMap and its enums only: the encoder comes from cudaGetDriverEntryPoint

#include <algorithm>
#include <atomic>

#include "linear_device.cuh"

namespace lin {
namespace {

constexpr int kTileM = 128;       // rows of a block's tile
constexpr int kBlockK = 64;       // k of a stage: 128 bytes, one swizzle row
constexpr int kEpiWarps = 8;
constexpr int kProducer = kEpiWarps, kIssuer = kEpiWarps + 1;
constexpr int kThreads = 32 * (kEpiWarps + 2);
constexpr int kStageA = kTileM * kBlockK * 2;
constexpr int kStagingBytes = 32 * 32 * 4;  // a warp's 32 x 32 floats
constexpr int kRingBytes = 192 * 1024;
constexpr int kPromote = 2;       // k blocks between additions in registers (float32)
constexpr int kGroupM = 8;        // rows of tiles walked together, for L2
constexpr long long kWaitClocks = 4000000000ll;  // about two seconds

template <int BN, int CG>
struct Shape {
  static constexpr int kRowsB = BN / CG;  // rows of B in one block's stage
  static constexpr int kStageB = kRowsB * kBlockK * 2;
  static constexpr int kStage = kStageA + kStageB;
  static constexpr int kStages = kRingBytes / kStage;
  static constexpr int kBarriers = 2 * kStages + 4;
  // stages, the warps' staging, barriers, the tensor-memory address; and room to start on 1024 bytes
  static constexpr int kSmem = kStages * kStage + kEpiWarps * kStagingBytes + kBarriers * 8 + 16 + 1024;
  static constexpr uint32_t kColumns = 2 * BN < 32 ? 32 : 2 * BN;
  static_assert(kSmem <= 232448, "more shared memory than a block may have");
};

// What a launch needs beside the tensor maps.
struct Job {
  Product pr;
  int64_t tiles_m, tiles_n;
  int splits, kblocks, kblocks_per_split, pairs;
  int box_a, box_b;  // rows of the boxes along k
  int device;
  bool vec;          // rows of bias, extra, out and slope start on 16-byte boundaries
};

__device__ unsigned int g_wait_timeouts;

// ---- PTX ---------------------------------------------------------------------------

__device__ __forceinline__ uint32_t smem_addr(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

__device__ __forceinline__ void barrier_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}

__device__ __forceinline__ void expect_bytes(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}

__device__ __forceinline__ bool try_wait(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
      : "=r"(done)
      : "r"(bar), "r"(parity)
      : "memory");
  return done != 0;
}

// Waits have a limit. One that runs out is counted, and from then on the
// thread polls each barrier once: the kernel ends, with wrong results and a
// count that msda_linear_wait_timeouts reports.
__device__ __forceinline__ void wait(uint32_t bar, uint32_t parity, bool& dead) {
  if (try_wait(bar, parity)) return;
  if (dead) return;
  const long long start = clock64();
  do {
    if (try_wait(bar, parity)) return;
  } while (clock64() - start < kWaitClocks);
  dead = true;
  atomicAdd(&g_wait_timeouts, 1u);
}

// The address of `addr` in block `rank` of the cluster.
__device__ __forceinline__ uint32_t in_block(uint32_t addr, uint32_t rank) {
  uint32_t out;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(out) : "r"(addr), "r"(rank));
  return out;
}

__device__ __forceinline__ void arrive_in(uint32_t cluster_bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}

// Box of `map` at (x, y, plane) into this block's shared memory; the bytes count at `bar`.
template <int CG>
__device__ __forceinline__ void copy_box(uint32_t dst, const CUtensorMap* map, int x, int y, int plane, uint32_t bar) {
  if (CG == 1)
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
        "[%5];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(plane), "r"(bar)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, "
        "{%2, %3, %4}], [%5];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(plane), "r"(bar)
        : "memory");
}

template <int CG>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  const uint32_t acc = accumulate;
  if (CG == 1)
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(
            d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
  else
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(
            d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}

// `bar` (in both blocks of a pair) is arrived at when the products so far are done.
template <int CG>
__device__ __forceinline__ void commit(uint32_t bar) {
  if (CG == 1)
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
  else
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
        "h"(static_cast<uint16_t>(3))
        : "memory");
}

template <int CG>
__device__ __forceinline__ void tmem_alloc(uint32_t dst, uint32_t columns) {
  if (CG == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst), "r"(columns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  } else {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst), "r"(columns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
}

template <int CG>
__device__ __forceinline__ void tmem_free(uint32_t addr, uint32_t columns) {
  if (CG == 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(columns));
  else
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(columns));
}

__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// 16 columns of this warp's 32 lanes of tensor memory, without waiting for them.
__device__ __forceinline__ void tmem_load16(uint32_t addr, uint32_t r[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
      "[%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr)
      : "memory");
}

// The loads so far have arrived; the registers pass through, so none is read before.
__device__ __forceinline__ void tmem_wait(uint32_t r[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}

template <int CG>
__device__ __forceinline__ void block_or_pair_sync() {
  if (CG == 1) {
    __syncthreads();
  } else {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
}

// ---- descriptors ---------------------------------------------------------------------

// A tile in shared memory with 128-byte swizzle. Stored along k, a row is 128
// bytes of k and eight rows follow one another every 1024 bytes. Stored across
// k, a line is 64 rows at one k; eight k follow one another every 1024 bytes,
// and 64 rows on comes the next box of 64 x 64, 8192 bytes later.
__device__ __forceinline__ uint64_t tile_descriptor(uint32_t addr, bool across) {
  const uint64_t lead = across ? 8192 >> 4 : 1, stride = 1024 >> 4;
  return static_cast<uint64_t>((addr >> 4) & 0x3fff) | (lead << 16) | (stride << 32) | (1ull << 46) | (2ull << 61);
}

// Bytes from one 16 of k to the next.
__device__ __forceinline__ uint32_t k_step(bool across) { return across ? 2048 : 32; }

// bfloat16 x bfloat16 -> float32
__device__ __forceinline__ uint32_t instruction(int m, int n, bool a_across, bool b_across) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(a_across) << 15) |
         (static_cast<uint32_t>(b_across) << 16) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>(m >> 4) << 24);
}

// ---- work ------------------------------------------------------------------------------

struct Item {
  int64_t m, n;  // first row and column
  int split, kb0, kb1;
};

template <int BN, int CG>
__device__ __forceinline__ Item item_of(const Job& j, int64_t i) {
  const int64_t tiles = j.tiles_m * j.tiles_n;
  Item t;
  t.split = static_cast<int>(i / tiles);
  const int64_t at = i - t.split * tiles, per_group = kGroupM * j.tiles_n;
  const int64_t group = at / per_group, first = group * kGroupM;
  const int64_t rows = min(static_cast<int64_t>(kGroupM), j.tiles_m - first), local = at - group * per_group;
  t.m = (first + local % rows) * (kTileM * CG);
  t.n = local / rows * BN;
  t.kb0 = t.split * j.kblocks_per_split;
  t.kb1 = min(j.kblocks, t.kb0 + j.kblocks_per_split);
  return t;
}

// The planes of A and B in product `i`, the smallest products first: the
// accumulator cuts at each step by up to 2^-24 of what it holds, and holds
// 2^-8 of the result until the last product of planes begins.
__device__ __forceinline__ void planes_of(const Job& j, int i, int& pa, int& pb) {
  if (j.pairs == 6) {
    pa = (0x010120 >> (4 * i)) & 3;
    pb = (0x001102 >> (4 * i)) & 3;
  } else {
    pa = j.pr.a.planes == 3 ? j.pairs - 1 - i : 0;
    pb = j.pr.b.planes == 3 ? j.pairs - 1 - i : 0;
  }
}

// ---- float32: what planes cannot hold -----------------------------------------------

__device__ __forceinline__ float whole(const Operand& o, bool across, int64_t i, int64_t k) {
  const int64_t at = across ? k * o.ld + i : i * o.ld + k;
  float v = 0.f;
  for (int q = o.planes - 1; q >= 0; --q) v += __bfloat162float(o.p[q * o.plane + at]);
  return v;
}

// An infinity is all in the first plane, and its product with the other
// operand's small planes is an infinity of any sign, or a NaN. So outputs
// whose row or column holds one are summed again, element by element; a NaN
// there makes them NaN.
__device__ __noinline__ float repaired(const Product& pr, uint32_t flags, int64_t m, int64_t n) {
  if (flags & 2u) return __uint_as_float(0x7fc00000u);
  float s = 0.f;
  for (int64_t k = 0; k < pr.k; ++k) s = fmaf(whole(pr.a, pr.a_mn, m, k), whole(pr.b, pr.b_mn, n, k), s);
  return s;
}

// Flags of rows / columns of the output; null where none can be set.
__device__ __forceinline__ const uint32_t* flags_m(const Product& pr) {
  return pr.a_mn ? pr.a.col_flags : pr.a.row_flags;
}
__device__ __forceinline__ const uint32_t* flags_n(const Product& pr) {
  return pr.b_mn ? pr.b.col_flags : pr.b.row_flags;
}

__device__ __noinline__ void repair8(const Product& pr, uint32_t row, float4& lo, float4& hi, int64_t m, int64_t n) {
  float* v[8] = {&lo.x, &lo.y, &lo.z, &lo.w, &hi.x, &hi.y, &hi.z, &hi.w};
  const uint32_t* fb = flags_n(pr);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (n + j >= pr.n) break;
    const uint32_t f = row | (fb ? fb[n + j] : 0u);
    if (f) *v[j] = repaired(pr, f, m, n + j);
  }
}

// ---- the kernel ------------------------------------------------------------------------

// A warp's 32 rows x 32 columns go through shared memory: a lane writes a row,
// and reads eight columns of every eighth row. Both ways the 16-byte units of a
// row are exchanged by its number, so no two lanes of a quarter warp meet in a
// bank.
__device__ __forceinline__ void stage_row(float* stage, const float v[32]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int q = 0; q < 8; ++q)
    *reinterpret_cast<float4*>(stage + lane * 32 + (q ^ (lane & 7)) * 4) =
        make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
}

// What was staged, through the epilogue. The residual of the next rows is
// loaded ahead.
template <typename T, bool kRepair>
__device__ __forceinline__ void drain(const Job& j, const Epilogue& e, const float* stage, int64_t m0, int64_t n0) {
  const int lane = threadIdx.x & 31, sub = lane >> 2, q = (lane & 3) * 2;
  const int64_t n = n0 + (lane & 3) * 8;
  if (n < j.pr.n) {
    const bool vec = j.vec && n + 8 <= j.pr.n;
    float b[8], x[8] = {};
    uint32_t col = 0;
    load_bias8<T>(e, n, j.pr.n, b);
    if (kRepair && flags_n(j.pr)) {
      for (int c = 0; c < 8 && n + c < j.pr.n; ++c) col |= flags_n(j.pr)[n + c];
    }
    const T* extra = static_cast<const T*>(e.extra);
    const bool ahead = vec && extra;
    if (ahead && m0 + sub < j.pr.m) load8(extra + (m0 + sub) * e.extra_ld + n, x);
#pragma unroll 1
    for (int i = 0; i < 4; ++i) {
      const int row = i * 8 + sub;
      const int64_t m = m0 + row;
      if (m >= j.pr.m) break;
      float4 lo = *reinterpret_cast<const float4*>(stage + row * 32 + (q ^ sub) * 4);
      float4 hi = *reinterpret_cast<const float4*>(stage + row * 32 + ((q + 1) ^ sub) * 4);
      if (kRepair) {
        const uint32_t f = flags_m(j.pr) ? flags_m(j.pr)[m] : 0u;
        if (f | col) repair8(j.pr, f, lo, hi, m, n);
      }
      if (vec) {
        float w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w}, y[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) y[c] = x[c];
        if (ahead && i < 3 && m + 8 < j.pr.m) load8(extra + (m + 8) * e.extra_ld + n, x);
        finish8<T>(e, w, y, b, m, n, j.pr.n, 8, true);
      } else {
        finish_some<T>(e, lo, hi, m, n, j.pr.n);
      }
    }
  }
}

// The same as a call: where the sums of the whole tile are held in registers,
// the loop over its parts is unrolled.
template <typename T, bool kRepair>
__device__ __noinline__ void drain_apart(const Job& j, const Epilogue& e, const float* stage, int64_t m0, int64_t n0) {
  drain<T, kRepair>(j, e, stage, m0, n0);
}

template <int BN, int CG, typename T, bool kF32>
__global__ void __launch_bounds__(kThreads, 1)
    product_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                   const __grid_constant__ Job job) {
  using S = Shape<BN, CG>;
  extern __shared__ uint8_t raw[];
  uint8_t* base = raw + ((1024 - (smem_addr(raw) & 1023)) & 1023);
  const uint32_t ring = smem_addr(base);
  float* staging = reinterpret_cast<float*>(base + S::kStages * S::kStage);
  const uint32_t bars = ring + S::kStages * S::kStage + kEpiWarps * kStagingBytes;
  const uint32_t tmem_slot = bars + S::kBarriers * 8;
  const auto full = [&](int s) { return bars + 8 * s; };
  const auto empty = [&](int s) { return bars + 8 * (S::kStages + s); };
  const auto acc_full = [&](int b) { return bars + 8 * (2 * S::kStages + b); };
  const auto acc_empty = [&](int b) { return bars + 8 * (2 * S::kStages + 2 + b); };

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t rank = 0;
  if (CG == 2) asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));

  if (threadIdx.x == 0) {
    for (int s = 0; s < S::kStages; ++s) {
      barrier_init(full(s), 1);
      barrier_init(empty(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      barrier_init(acc_full(b), 1);
      barrier_init(acc_empty(b), kEpiWarps * CG);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kIssuer) tmem_alloc<CG>(tmem_slot, S::kColumns);
  fence_before();
  block_or_pair_sync<CG>();
  fence_after();
  uint32_t tmem;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(tmem_slot));

  const int64_t items = job.tiles_m * job.tiles_n * job.splits;
  const int64_t first = blockIdx.x / CG, step = gridDim.x / CG;
  const int chunk = kF32 ? kPromote : job.kblocks;
  bool dead = false;

  if (warp == kProducer && lane == 0) {
    int s = 0;
    uint32_t phase = 0;
    for (int64_t i = first; i < items; i += step) {
      const Item t = item_of<BN, CG>(job, i);
      // boxes that hold rows of the tile; what a skipped box leaves in its place reaches no row or column that is kept
      const auto boxes = [](int64_t have, int most) {
        return static_cast<int>(have <= 0 ? 0 : have >= most * 64ll ? most : (have + 63) / 64);
      };
      const auto bytes_of = [&](int64_t ma, int64_t nb) {
        return (job.pr.a_mn ? boxes(job.pr.m - ma, kTileM / 64) * 8192 : job.box_a * 128) +
               (job.pr.b_mn ? boxes(job.pr.n - nb, S::kRowsB / 64) * 8192 : job.box_b * 128);
      };
      const int64_t ma = t.m + rank * kTileM, nb = t.n + rank * S::kRowsB;
      const int boxes_a = boxes(job.pr.m - ma, kTileM / 64), boxes_b = boxes(job.pr.n - nb, S::kRowsB / 64);
      uint32_t bytes = bytes_of(t.m, t.n);
      if (CG == 2) bytes += bytes_of(t.m + kTileM, t.n + S::kRowsB);
      for (int c = t.kb0; c < t.kb1; c += chunk) {
        const int c1 = min(c + chunk, t.kb1);
        for (int p = 0; p < job.pairs; ++p) {
          int pa, pb;
          planes_of(job, p, pa, pb);
          for (int kb = c; kb < c1; ++kb) {
            wait(empty(s), phase ^ 1, dead);
            if (rank == 0) expect_bytes(full(s), bytes);
            const uint32_t bar = CG == 2 ? in_block(full(s), 0) : full(s);
            const uint32_t a = ring + s * S::kStage, b = a + kStageA;
            const int k = kb * kBlockK;
            if (job.pr.a_mn) {
              for (int x = 0; x < boxes_a; ++x)
                copy_box<CG>(a + x * 8192, &map_a, static_cast<int>(ma) + x * 64, k, pa, bar);
            } else {
              copy_box<CG>(a, &map_a, k, static_cast<int>(ma), pa, bar);
            }
            if (job.pr.b_mn) {
              for (int x = 0; x < boxes_b; ++x)
                copy_box<CG>(b + x * 8192, &map_b, static_cast<int>(nb) + x * 64, k, pb, bar);
            } else {
              copy_box<CG>(b, &map_b, k, static_cast<int>(nb), pb, bar);
            }
            if (++s == S::kStages) s = 0, phase ^= 1;
          }
        }
      }
    }
    // the copies that are still in flight land before the block's memory goes
    for (int x = 0; x < S::kStages; ++x) {
      wait(empty(s), phase ^ 1, dead);
      if (++s == S::kStages) s = 0, phase ^= 1;
    }
  } else if (warp == kIssuer && rank == 0) {
    // the whole warp walks the loop, one lane issues: the warp stays together for the barriers below
    const uint32_t idesc = instruction(kTileM * CG, BN, job.pr.a_mn, job.pr.b_mn);
    const uint32_t step_a = k_step(job.pr.a_mn) >> 4, step_b = k_step(job.pr.b_mn) >> 4;
    int s = 0, buf = 0;
    uint32_t phase = 0, acc_phase = 0;
    for (int64_t i = first; i < items; i += step) {
      const Item t = item_of<BN, CG>(job, i);
      for (int c = t.kb0; c < t.kb1; c += chunk) {
        const int steps = (min(c + chunk, t.kb1) - c) * job.pairs;
        wait(acc_empty(buf), acc_phase ^ 1, dead);
        fence_after();
        for (int x = 0; x < steps; ++x) {
          wait(full(s), phase, dead);
          fence_after();
          if (lane == 0) {
            const uint32_t a = ring + s * S::kStage;
            const uint64_t da = tile_descriptor(a, job.pr.a_mn), db = tile_descriptor(a + kStageA, job.pr.b_mn);
#pragma unroll
            for (int kk = 0; kk < kBlockK / 16; ++kk)
              mma<CG>(tmem + buf * BN, da + kk * step_a, db + kk * step_b, idesc, x > 0 || kk > 0);
            commit<CG>(empty(s));
          }
          __syncwarp();
          if (++s == S::kStages) s = 0, phase ^= 1;
        }
        if (lane == 0) commit<CG>(acc_full(buf));
        __syncwarp();
        buf ^= 1;
        if (buf == 0) acc_phase ^= 1;
      }
    }
  } else if (warp < kEpiWarps) {
    Epilogue e = job.pr.epi;
    const int quad = warp & 3, half = warp >> 2;
    float* stage = staging + warp * (kStagingBytes / 4);
    int buf = 0;
    uint32_t acc_phase = 0;
    constexpr int kParts = BN / 64;  // of 32 columns
    for (int64_t i = first; i < items; i += step) {
      const Item t = item_of<BN, CG>(job, i);
      if (job.splits > 1) {
        e = Epilogue();
        e.out = job.pr.partial + t.split * job.pr.m * job.pr.n;
        e.out_ld = job.pr.n;
      }
      const int64_t m = t.m + rank * kTileM + quad * 32, n = t.n + half * (BN / 2);
      const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
      if (kF32) {
        float acc[kParts][32] = {};
        for (int c = t.kb0; c < t.kb1; c += chunk) {
          wait(acc_full(buf), acc_phase, dead);
          fence_after();
#pragma unroll
          for (int p = 0; p < kParts; ++p) {
            const uint32_t at = tmem + lanes + buf * BN + half * (BN / 2) + p * 32;
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              uint32_t r[16];
              tmem_load16(at + q * 16, r);
              tmem_wait(r);
#pragma unroll
              for (int x = 0; x < 16; ++x) acc[p][q * 16 + x] += __uint_as_float(r[x]);
            }
          }
          fence_before();
          __syncwarp();
          if (lane == 0) arrive_in(in_block(acc_empty(buf), 0));
          buf ^= 1;
          if (buf == 0) acc_phase ^= 1;
        }
#pragma unroll
        for (int p = 0; p < kParts; ++p) {
          stage_row(stage, acc[p]);
          __syncwarp();
          if (job.splits > 1)
            drain_apart<float, false>(job, e, stage, m, n + p * 32);
          else
            drain_apart<T, true>(job, e, stage, m, n + p * 32);
          __syncwarp();
        }
      } else {
        wait(acc_full(buf), acc_phase, dead);
        fence_after();
#pragma unroll 1
        for (int p = 0; p < kParts; ++p) {
          const uint32_t at = tmem + lanes + buf * BN + half * (BN / 2) + p * 32;
          uint32_t r[2][16];
          tmem_load16(at, r[0]);
          tmem_load16(at + 16, r[1]);
          tmem_wait(r[0]);
          tmem_wait(r[1]);
          float v[32];
#pragma unroll
          for (int x = 0; x < 32; ++x) v[x] = __uint_as_float(r[x / 16][x % 16]);
          if (p + 1 == kParts) {
            fence_before();
            __syncwarp();
            if (lane == 0) arrive_in(in_block(acc_empty(buf), 0));
          }
          stage_row(stage, v);
          __syncwarp();
          drain<T, false>(job, e, stage, m, n + p * 32);
          __syncwarp();
        }
        buf ^= 1;
        if (buf == 0) acc_phase ^= 1;
      }
    }
  }
  __syncwarp();
  fence_before();
  block_or_pair_sync<CG>();
  if (warp == kIssuer) {
    fence_after();
    tmem_free<CG>(tmem, S::kColumns);
  }
}

// Sums the ranges of k in order and runs the epilogue: a thread per eight columns.
template <typename T, bool kF32>
__global__ void __launch_bounds__(256) finish_kernel(const __grid_constant__ Job job) {
  const Product& pr = job.pr;
  const int64_t per_row = (pr.n + 7) / 8, total = pr.m * per_row;
  const bool part_vec = pr.n % 4 == 0;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
    const int64_t m = i / per_row, n = (i - m * per_row) * 8;
    const int count = static_cast<int>(pr.n - n < 8 ? pr.n - n : 8);
    float v[8] = {}, b[8];
    for (int s = 0; s < job.splits; ++s) {
      float w[8];
      load_some(pr.partial + (s * pr.m + m) * pr.n + n, count, part_vec && count == 8, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] += w[j];
    }
    float4 lo = make_float4(v[0], v[1], v[2], v[3]), hi = make_float4(v[4], v[5], v[6], v[7]);
    if (kF32 && pr.k > 0) {
      const uint32_t row = flags_m(pr) ? flags_m(pr)[m] : 0u;
      uint32_t any = row;
      if (flags_n(pr))
        for (int j = 0; j < count; ++j) any |= flags_n(pr)[n + j];
      if (any) repair8(pr, row, lo, hi, m, n);
    }
    if (job.vec && count == 8) {
      float w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w}, x[8] = {};
      load_bias8<T>(pr.epi, n, pr.n, b);
      if (pr.epi.extra) load8(static_cast<const T*>(pr.epi.extra) + m * pr.epi.extra_ld + n, x);
      finish8<T>(pr.epi, w, x, b, m, n, pr.n, 8, true);
    } else {
      finish_some<T>(pr.epi, lo, hi, m, n, pr.n);
    }
  }
}

// ---- host --------------------------------------------------------------------------------

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encoder() {
  static const EncodeTiledFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q = cudaDriverEntryPointSymbolNotFound;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<EncodeTiledFn>(p);
  }();
  return fn;
}

// Boxes of 64 columns (128 bytes, swizzled) and `rows` rows of one plane;
// columns start at multiples of 64, and what lies outside reads as zero.
bool make_map(CUtensorMap* map, const Operand& o, int rows) {
  const EncodeTiledFn encode = encoder();
  if (!encode) return false;
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(o.cols), static_cast<cuuint64_t>(o.rows),
                              static_cast<cuuint64_t>(o.planes)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(o.ld) * 2,
                                 static_cast<cuuint64_t>(o.planes > 1 ? o.plane : o.ld) * 2};
  const cuuint32_t box[3] = {kBlockK, static_cast<cuuint32_t>(rows), 1};
  const cuuint32_t unit[3] = {1, 1, 1};
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<__nv_bfloat16*>(o.p), dims, strides, box, unit,
                CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Whether eight columns at a multiple of eight are one aligned vector everywhere.
bool vectors_fit(const Product& pr) {
  const Epilogue& e = pr.epi;
  const int64_t size = pr.dtype == DType::kF32 ? 4 : 2;
  bool ok = aligned16(e.out) && (e.out_ld * (e.out_plane ? 2 : size)) % 16 == 0 && (e.out_plane * 2) % 16 == 0;
  if (e.extra) ok = ok && aligned16(e.extra) && (e.extra_ld * size) % 16 == 0;
  if (e.slope) ok = ok && aligned16(e.slope) && (pr.n * size) % 16 == 0;
  return ok;
}

template <int BN, int CG, typename T, bool kF32>
cudaError_t launch(const CUtensorMap& a, const CUtensorMap& b, const Job& job, int sms, cudaStream_t stream) {
  using S = Shape<BN, CG>;
  const auto kernel = product_kernel<BN, CG, T, kF32>;
  static std::atomic<uint64_t> ready{0};  // devices (of the first 64) that know the kernel's shared memory
  const uint64_t bit = job.device < 64 ? 1ull << job.device : 0;
  if (!bit || !(ready.load(std::memory_order_relaxed) & bit)) {
    const cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem);
    if (err != cudaSuccess) return err;
    ready.fetch_or(bit, std::memory_order_relaxed);
  }
  const int64_t items = job.tiles_m * job.tiles_n * job.splits;
  const int blocks = static_cast<int>(std::min<int64_t>(items, sms / CG)) * CG;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(blocks);
  config.blockDim = dim3(kThreads);
  config.dynamicSmemBytes = S::kSmem;
  config.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = CG;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  config.attrs = attr;
  config.numAttrs = CG > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&config, kernel, a, b, job);
}

template <typename T, bool kF32>
cudaError_t launch_tile(const Plan& plan, const CUtensorMap& a, const CUtensorMap& b, const Job& job, int sms,
                        cudaStream_t stream) {
  if constexpr (!kF32) {
    if (plan.bn == 256)
      return plan.pair == 2 ? launch<256, 2, T, kF32>(a, b, job, sms, stream)
                            : launch<256, 1, T, kF32>(a, b, job, sms, stream);
  }
  return plan.bn == 128 ? launch<128, 1, T, kF32>(a, b, job, sms, stream)
                        : launch<64, 1, T, kF32>(a, b, job, sms, stream);
}

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

}  // namespace

// The tile and the ranges of k with the shortest estimated time, in clocks of
// one SM: a stage costs the longer of its products (2 clocks per column) and
// its copies (64 bytes a clock), tiles overlap with the epilogue of the one
// before, and partial sums cost their trip through L2 and a second launch.
Plan plan_product(int64_t m, int64_t n, int64_t k, int pairs, bool any_mn, int sms) {
  const int kblocks = static_cast<int>(ceil_div(k, kBlockK));
  Plan best{64, 1, 1, kblocks};
  if (m == 0 || n == 0 || k == 0) return best;
  double best_time = 1e300;
  const struct {
    int bn, pair;
  } shapes[] = {{64, 1}, {128, 1}, {256, 1}, {256, 2}};
  for (const auto& s : shapes) {
    if (pairs > 1 && s.bn == 256) continue;  // float32 holds its sums in registers
    const int64_t tiles = ceil_div(m, kTileM * s.pair) * ceil_div(n, s.bn);
    const int64_t slots = sms / s.pair;
    const double stage = std::max(2.0 * s.bn, (kStageA + s.bn * 128.0 / s.pair) / 64.0) * pairs;
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

cudaError_t launch_product(const Product& pr, const Plan& plan, cudaStream_t stream) {
  if (pr.m == 0 || pr.n == 0) return cudaSuccess;
  Job job{};
  job.pr = pr;
  job.vec = vectors_fit(pr);
  job.splits = plan.splits;
  const bool f32 = pr.dtype == DType::kF32;
  if (pr.k > 0) {
    int device = 0, sms = 148;
    cudaError_t err = cudaGetDevice(&device);
    // binds the device's context to this thread (autograd's threads may have none yet): the encoder needs one
    if (err == cudaSuccess) err = cudaSetDevice(device);
    if (err == cudaSuccess) err = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
    if (err != cudaSuccess) return err;
    job.device = device;
    if (plan.splits > 1) job.vec = pr.n % 4 == 0;  // of the partial sums
    job.tiles_m = ceil_div(pr.m, kTileM * plan.pair);
    job.tiles_n = ceil_div(pr.n, plan.bn);
    job.kblocks = static_cast<int>(ceil_div(pr.k, kBlockK));
    job.kblocks_per_split = plan.kblocks;
    job.pairs = pr.a.planes == 3 ? (pr.b.planes == 3 ? 6 : 3) : (pr.b.planes == 3 ? 3 : 1);
    const int64_t rows_b = plan.bn / plan.pair;
    job.box_a = pr.a_mn ? 64 : static_cast<int>(std::min<int64_t>(kTileM, ceil_div(pr.m, 8) * 8));
    job.box_b = pr.b_mn ? 64 : static_cast<int>(std::min<int64_t>(rows_b, ceil_div(pr.n, 8) * 8));
    CUtensorMap a, b;
    if (!make_map(&a, pr.a, job.box_a) || !make_map(&b, pr.b, job.box_b)) return cudaErrorInvalidValue;
    if (f32) {
      err = launch_tile<float, true>(plan, a, b, job, sms, stream);
    } else if (plan.splits > 1) {
      err = launch_tile<float, false>(plan, a, b, job, sms, stream);
    } else {
      err = launch_tile<bf16, false>(plan, a, b, job, sms, stream);
    }
    if (err != cudaSuccess || plan.splits == 1) return err;
    job.vec = vectors_fit(pr);
  } else {
    job.splits = 0;  // an empty sum
  }
  const int64_t groups = pr.m * ((pr.n + 7) / 8);
  const int blocks = static_cast<int>(std::min<int64_t>((groups + 255) / 256, 148 * 8));
  if (f32)
    finish_kernel<float, true><<<blocks, 256, 0, stream>>>(job);
  else
    finish_kernel<bf16, false><<<blocks, 256, 0, stream>>>(job);
  return cudaGetLastError();
}

cudaError_t wait_timeouts(unsigned int* count) { return cudaMemcpyFromSymbol(count, g_wait_timeouts, sizeof(*count)); }

}  // namespace lin
