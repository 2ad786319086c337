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
#include <cuda.h>  // CUtensorMap and its enums only: the encoder comes from cudaGetDriverEntryPoint

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "async_device.cuh"
#include "linear_device.cuh"

namespace lin {
namespace {

using async::barrier_init;
using async::expect_bytes;
using async::settle;
using async::smem_addr;
using async::wait;

constexpr int kTileM = 128;       // rows of a block's tile
constexpr int kBlockK = 64;       // k of a stage: 128 bytes, one swizzle row
constexpr int kEpiWarps = 16;     // eight issued half the time: gelu, 40000 x 256 x 512, 52 us
constexpr int kProducer = kEpiWarps, kIssuer = kEpiWarps + 1;
constexpr int kThreads = 32 * (kEpiWarps + 2);
constexpr int kStageA = kTileM * kBlockK * 2;
constexpr int kBoxBytes = 32 * 128;  // a box of the epilogue: 32 rows of 128 bytes
constexpr int kRingBytes = 160 * 1024;
// float32: k blocks between additions in registers (4 takes 9 % off 2048^3, with
// twice the steps that cut)
constexpr int kPromote = 2;
constexpr int kFold = 8;          // and how many of those additions to one of the small products' sums
constexpr int kGroupM = 8;        // rows of tiles walked together, for L2

// float32: the order in which a stage's planes are copied, used and given back.
// A plane of A and of B has a slot of the ring to itself. Half the products want
// no third plane, and the second is free again after half of them: so the copies
// of the next stage begin, and its products do, before the stage is whole.
__host__ __device__ constexpr int plane_of(int i) { return i == 0 ? 1 : i == 1 ? 0 : 2; }

template <int BN, int CG, bool kF32>
struct Shape {
  static constexpr int kPlanes = kF32 ? 3 : 1;
  static constexpr int kRowsB = BN / CG;  // rows of B in one block's stage
  static constexpr int kStageB = kRowsB * kBlockK * 2;
  static constexpr int kStage = kStageA + kStageB;  // one plane of both
  static constexpr int kStages = kRingBytes / kStage;
  static constexpr int kBarriers = 2 * kStages + 4 + kEpiWarps + (kF32 ? 2 : 0);
  // stages, the warps' staging, barriers, the tensor-memory address; and room to start on 1024 bytes
  static constexpr int kSmem = kStages * kStage + kEpiWarps * kBoxBytes + kBarriers * 8 + 16 + 1024;
  // tensor memory: two accumulators; float32 has two more behind them, the small products'
  static constexpr int kSmall = 2 * BN;
  static constexpr uint32_t kColumns = kF32 ? 4 * BN : 2 * BN;
  // a warp of the epilogue takes 32 rows and this many columns
  static constexpr int kCols = BN / 4 < 32 ? 32 : BN / 4;
  static constexpr int kWarps = 4 * (BN / kCols);
  static_assert(kSmem <= 232448, "more shared memory than a block may have");
};

// What a launch needs beside the tensor maps.
struct Job {
  Product pr;
  uint32_t tiles_m, tiles_n;
  uint64_t by_tiles, by_group, by_last;  // divided()
  int splits, kblocks, kblocks_per_split;
  int box_a, box_b;  // rows of the boxes along k
  int device;
  bool apart;        // the epilogue leaves sums in pr.partial
  bool vec;          // finishing: rows of extra, out and slope start on 16-byte boundaries
};

// ---- PTX ---------------------------------------------------------------------------

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

// The same with the wait.
__device__ __forceinline__ void tmem_take16(uint32_t addr, float v[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
      "[%16];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
        "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
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

__device__ __forceinline__ void tmem_store16(uint32_t addr, const float v[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15};" ::"f"(v[0]),
      "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "f"(v[8]), "f"(v[9]), "f"(v[10]),
      "f"(v[11]), "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15]), "r"(addr)
      : "memory");
}

// Eight columns, stored; and loaded and waited for.
__device__ __forceinline__ void tmem_store8(uint32_t addr, const uint32_t r[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(addr)
               : "memory");
}

__device__ __forceinline__ void tmem_load8(uint32_t addr, uint32_t r[8]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
      : "r"(addr)
      : "memory");
}

__device__ __forceinline__ void tmem_stored() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

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
  int m, n;  // first row and column
  int split, kb0, kb1;
};

// x / d for 32-bit x: `magic` is floor(2^64 / d) + 1 (0 stands for d = 1). The
// divisions were a tenth of an epilogue's time.
__device__ __forceinline__ uint32_t divided(uint32_t x, uint64_t magic) {
  return magic ? static_cast<uint32_t>(__umul64hi(x, magic)) : x;
}

template <int BN, int CG>
__device__ __forceinline__ Item item_of(const Job& j, uint32_t i) {
  Item t;
  t.split = static_cast<int>(divided(i, j.by_tiles));
  const uint32_t at = i - t.split * j.tiles_m * j.tiles_n;
  const uint32_t group = divided(at, j.by_group), first = group * kGroupM;
  const uint32_t local = at - group * (kGroupM * j.tiles_n);
  const uint32_t rows = j.tiles_m - first;  // of tiles in the group, if fewer than usual
  const uint32_t col = rows >= kGroupM ? local / kGroupM : divided(local, j.by_last);
  t.m = static_cast<int>((first + local - col * min(rows, static_cast<uint32_t>(kGroupM))) * (kTileM * CG));
  t.n = static_cast<int>(col * BN);
  t.kb0 = t.split * j.kblocks_per_split;
  t.kb1 = min(j.kblocks, t.kb0 + j.kblocks_per_split);
  return t;
}

// ---- the epilogue ------------------------------------------------------------------------

// A warp's box in shared memory: 32 rows of 128 or 64 bytes, whose 16-byte units
// are exchanged by the row's number as TMA's swizzle has it; eight neighbouring
// rows' units at one place then lie in different banks.
template <int kRowBytes>
__device__ __forceinline__ uint32_t unit_at(uint32_t box, int row, int unit) {
  return kRowBytes == 128 ? box + row * 128 + ((unit ^ (row & 7)) << 4)
                          : box + row * 64 + ((unit ^ ((row >> 1) & 3)) << 4);
}

__device__ __forceinline__ void put_unit(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

__device__ __forceinline__ void get_unit(uint32_t addr, uint32_t v[4]) {
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
               : "r"(addr)
               : "memory");
}

__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// 16 values of a row into the box from column `col` on.
template <int kRowBytes>
__device__ __forceinline__ void put16(uint32_t box, int row, int col, const float v[16], bf16) {
#pragma unroll
  for (int u = 0; u < 2; ++u)
    put_unit(unit_at<kRowBytes>(box, row, col / 8 + u), pack2(v[8 * u], v[8 * u + 1]), pack2(v[8 * u + 2], v[8 * u + 3]),
             pack2(v[8 * u + 4], v[8 * u + 5]), pack2(v[8 * u + 6], v[8 * u + 7]));
}
template <int kRowBytes>
__device__ __forceinline__ void put16(uint32_t box, int row, int col, const float v[16], __half) {
#pragma unroll
  for (int u = 0; u < 2; ++u)
    put_unit(unit_at<kRowBytes>(box, row, col / 8 + u), pack_half2(v[8 * u], v[8 * u + 1]),
             pack_half2(v[8 * u + 2], v[8 * u + 3]), pack_half2(v[8 * u + 4], v[8 * u + 5]),
             pack_half2(v[8 * u + 6], v[8 * u + 7]));
}
template <int kRowBytes>
__device__ __forceinline__ void put16(uint32_t box, int row, int col, const float v[16], float) {
#pragma unroll
  for (int u = 0; u < 4; ++u)
    put_unit(unit_at<kRowBytes>(box, row, col / 4 + u), __float_as_uint(v[4 * u]), __float_as_uint(v[4 * u + 1]),
             __float_as_uint(v[4 * u + 2]), __float_as_uint(v[4 * u + 3]));
}

template <int kRowBytes>
__device__ __forceinline__ void get16(uint32_t box, int row, int col, float v[16], bf16) {
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    uint32_t w[4];
    get_unit(unit_at<kRowBytes>(box, row, col / 8 + u), w);
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      v[8 * u + 2 * x] = __uint_as_float(w[x] << 16);
      v[8 * u + 2 * x + 1] = __uint_as_float(w[x] & 0xffff0000u);
    }
  }
}
template <int kRowBytes>
__device__ __forceinline__ void get16(uint32_t box, int row, int col, float v[16], float) {
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    uint32_t w[4];
    get_unit(unit_at<kRowBytes>(box, row, col / 4 + u), w);
#pragma unroll
    for (int x = 0; x < 4; ++x) v[4 * u + x] = __uint_as_float(w[x]);
  }
}

// 16 slopes put aside in the tensor memory that their sums came from, and taken back into the box.
__device__ __forceinline__ void put_aside(uint32_t at, const float s[16], __half) {
  uint32_t w[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) w[j] = pack_half2(s[2 * j], s[2 * j + 1]);
  tmem_store8(at, w);
}
__device__ __forceinline__ void put_aside(uint32_t at, const float s[16], float) { tmem_store16(at, s); }
template <int kRowBytes>
__device__ __forceinline__ void take_back(uint32_t box, int row, int col, uint32_t at, __half) {
  uint32_t w[8];
  tmem_load8(at, w);
#pragma unroll
  for (int u = 0; u < 2; ++u)
    put_unit(unit_at<kRowBytes>(box, row, col / 8 + u), w[4 * u], w[4 * u + 1], w[4 * u + 2], w[4 * u + 3]);
}
template <int kRowBytes>
__device__ __forceinline__ void take_back(uint32_t box, int row, int col, uint32_t at, float) {
  uint32_t w[16];
  tmem_load16(at, w);
  tmem_wait(w);
#pragma unroll
  for (int u = 0; u < 4; ++u)
    put_unit(unit_at<kRowBytes>(box, row, col / 4 + u), w[4 * u], w[4 * u + 1], w[4 * u + 2], w[4 * u + 3]);
}

// Bias of columns [n, n + 16), the same for all lanes: asked for before the sums
// it is added to have come.
template <typename T>
struct Bias16 {
  uint4 u[sizeof(T)];
  __device__ __forceinline__ void load(const T* p, bool vec, int count) {
    if (vec && count >= 16) {
#pragma unroll
      for (int k = 0; k < static_cast<int>(sizeof(T)); ++k) u[k] = __ldg(reinterpret_cast<const uint4*>(p) + k);
    } else {
      uint4 few[sizeof(T)];  // only this copy has an address
      copy_few(p, count, reinterpret_cast<T*>(few));
#pragma unroll
      for (int k = 0; k < static_cast<int>(sizeof(T)); ++k) u[k] = few[k];
    }
  }
  static __device__ __noinline__ void copy_few(const T* p, int count, T* out) {
    for (int j = 0; j < 16; ++j) out[j] = j < count ? p[j] : from_float<T>(0.f);
  }
  __device__ __forceinline__ void add(float v[16]) const {
    float b[16];
    load8(reinterpret_cast<const T*>(u), b);
    load8(reinterpret_cast<const T*>(u) + 8, b + 8);
#pragma unroll
    for (int j = 0; j < 16; j += 2) {
      const float2 s = add2(make_float2(v[j], v[j + 1]), make_float2(b[j], b[j + 1]));
      v[j] = s.x, v[j + 1] = s.y;
    }
  }
};

__device__ __forceinline__ void store_box(const CUtensorMap* map, int x, int y, int z, uint32_t src) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(map), "r"(x),
               "r"(y), "r"(z), "r"(src)
               : "memory");
}

__device__ __forceinline__ void stores_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }

// At most N groups of stores still read their boxes.
template <int N>
__device__ __forceinline__ void stores_read() {
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
}

// ---- the kernel ------------------------------------------------------------------------

constexpr int kFwdSlope = 3;  // beside Epilogue::Mode: kFwd that also writes the slope

// float32: what is not finite. An infinity or a NaN is all in an operand's first
// plane, so the product of first planes answers as float32 would (a factor below
// 2^-134 counts as 0 there), and so it does where finite products overflow. The
// small products then are infinities of any sign, or NaNs: a sum of them that is
// not finite is left out.
__device__ __forceinline__ float finite_or_zero(float v) { return fabsf(v) <= 3.402823466e38f ? v : 0.f; }

struct Maps {
  CUtensorMap a, b, out, extra, slope;
};

// Where a block's things are: addresses in tensor and shared memory, and its rank in a pair.
struct Place {
  uint32_t tmem, boxes, bars, rank;
};

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

// NaNs over all that this block's epilogue writes, by the same boxes: a box of ones in every bit.
template <int BN, int CG, typename T, bool kF32>
__device__ __noinline__ void spoil(const Maps& maps, const Job& job, const Place place) {
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

template <int BN, int CG, typename T, bool kF32>
__global__ void __launch_bounds__(kThreads, 1)
    product_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Job job) {
  using S = Shape<BN, CG, kF32>;
  extern __shared__ uint8_t raw[];
  const uint32_t ring = (smem_addr(raw) + 1023) & ~1023u;
  const uint32_t bars = ring + S::kStages * S::kStage + kEpiWarps * kBoxBytes;
  const uint32_t tmem_slot = bars + S::kBarriers * 8, spoilt = tmem_slot + 4;
  const auto full = [&](int s) { return bars + 8 * s; };
  const auto empty = [&](int s) { return bars + 8 * (S::kStages + s); };
  const auto acc_full = [&](int b) { return bars + 8 * (2 * S::kStages + b); };
  const auto acc_empty = [&](int b) { return bars + 8 * (2 * S::kStages + 2 + b); };
  const auto small_empty = [&](int b) { return bars + 8 * (2 * S::kStages + 4 + kEpiWarps + b); };

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
      barrier_init(acc_empty(b), S::kWarps * CG);
      if (kF32) barrier_init(small_empty(b), S::kWarps * CG);
    }
    for (int x = 0; x < kEpiWarps; ++x) barrier_init(bars + 8 * (2 * S::kStages + 4 + x), 1);
    asm volatile("st.shared.u32 [%0], %1;" ::"r"(spoilt), "r"(0) : "memory");
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kIssuer) tmem_alloc<CG>(tmem_slot, S::kColumns);
  fence_before();
  block_or_pair_sync<CG>();
  fence_after();
  uint32_t tmem;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(tmem_slot));

  const uint32_t items = job.tiles_m * job.tiles_n * job.splits;
  const uint32_t first = blockIdx.x / CG, step = gridDim.x / CG;
  const int chunk = kF32 ? kPromote : job.kblocks;
  bool dead = false;

  if (warp == kProducer && lane == 0) {
    int s = 0;
    uint32_t phase = 0;
    const int rows_m = static_cast<int>(job.pr.m), rows_n = static_cast<int>(job.pr.n);
    const uint32_t full0 = CG == 2 ? in_block(full(0), 0) : full(0);  // the pair's copies count in its first block
    for (uint32_t i = first; i < items && !dead; i += step) {
      const Item t = item_of<BN, CG>(job, i);
      // boxes that hold rows of the tile; what a skipped box leaves in its place reaches no row or column that is kept
      const auto boxes = [](int have, int most) { return have <= 0 ? 0 : min(most, (have - 1) / 64 + 1); };
      const auto bytes_a = [&](int ma) { return job.pr.a_mn ? boxes(rows_m - ma, kTileM / 64) * 8192 : job.box_a * 128; };
      const auto bytes_b = [&](int nb) {
        return job.pr.b_mn ? boxes(rows_n - nb, S::kRowsB / 64) * 8192 : job.box_b * 128;
      };
      const int ma = t.m + rank * kTileM, nb = t.n + rank * S::kRowsB;
      const int boxes_a = boxes(rows_m - ma, kTileM / 64), boxes_b = boxes(rows_n - nb, S::kRowsB / 64);
      const uint32_t from_a = bytes_a(t.m) + (CG == 2 ? bytes_a(t.m + kTileM) : 0);
      const uint32_t from_b = bytes_b(t.n) + (CG == 2 ? bytes_b(t.n + S::kRowsB) : 0);
      // One thread issues a stage's copies while the tensor core works on another
      // (512 clocks): the layouts are constants, as counted loops over boxes and
      // planes took longer than that (8192 x 4096 x 8192, dW: 491 us, now 387).
      const auto stages = [&](auto a_across, auto b_across) {
        constexpr bool kA = decltype(a_across)::value, kB = decltype(b_across)::value;
        for (int kb = t.kb0; kb < t.kb1; ++kb) {
          const int k = kb * kBlockK;
#pragma unroll
          for (int u = 0; u < S::kPlanes; ++u) {
            const int p = kF32 ? plane_of(u) : 0;
            const bool has_a = !kF32 || p < job.pr.a.planes, has_b = !kF32 || p < job.pr.b.planes;
            const uint32_t bar = full0 + 8 * s, a = ring + s * S::kStage, b = a + kStageA;
            wait(empty(s), phase ^ 1, dead);
            if (dead) return;
            if (rank == 0) expect_bytes(full(s), (has_a ? from_a : 0) + (has_b ? from_b : 0));
            if (kA) {
#pragma unroll
              for (int x = 0; x < kTileM / 64; ++x)
                if (has_a && x < boxes_a) copy_box<CG>(a + x * 8192, &maps.a, ma + x * 64, k, p, bar);
            } else {
              if (has_a) copy_box<CG>(a, &maps.a, k, ma, p, bar);
            }
            if (kB) {
#pragma unroll
              for (int x = 0; x < S::kRowsB / 64; ++x)
                if (has_b && x < boxes_b) copy_box<CG>(b + x * 8192, &maps.b, nb + x * 64, k, p, bar);
            } else {
              if (has_b) copy_box<CG>(b, &maps.b, k, nb, p, bar);
            }
            if (++s == S::kStages) s = 0, phase ^= 1;
          }
        }
      };
      if (job.pr.a_mn)
        stages(std::true_type(), std::true_type());
      else if (job.pr.b_mn)
        stages(std::false_type(), std::true_type());
      else
        stages(std::false_type(), std::false_type());
    }
    // the copies have landed, and their products are done, before the block's memory goes
    for (int x = 0; x < S::kStages; ++x) {
      if (rank == 0) settle(full(s), phase ^ 1);
      settle(empty(s), phase ^ 1);
      if (++s == S::kStages) s = 0, phase ^= 1;
    }
  } else if (warp == kIssuer && rank == 0) {
    // the whole warp walks the loop, one lane issues (nothing more once a wait of its own ran out): the warp
    // stays together for the barriers below
    const uint32_t idesc = instruction(kTileM * CG, BN, job.pr.a_mn, job.pr.b_mn);
    const uint32_t step_a = k_step(job.pr.a_mn) >> 4, step_b = k_step(job.pr.b_mn) >> 4;
    const uint64_t first_a = tile_descriptor(ring, job.pr.a_mn);
    const uint64_t first_b = tile_descriptor(ring + kStageA, job.pr.b_mn);
    const bool more_a = job.pr.a.planes > 1, more_b = job.pr.b.planes > 1;
    int s = 0, buf = 0, small_buf = 0;
    uint32_t phase = 0, acc_phase = 0, small_phase = 0;
    for (uint32_t i = first; i < items; i += step) {
      const Item t = item_of<BN, CG>(job, i);
      for (int c = t.kb0, n = 1; c < t.kb1; c += chunk, ++n) {
        const int steps = min(c + chunk, t.kb1) - c;
        const bool fresh = n % kFold == 1;  // the small products' sums begin anew
        wait(acc_empty(buf), acc_phase ^ 1, dead);
        if (kF32 && fresh) wait(small_empty(small_buf), small_phase ^ 1, dead);
        fence_after();
        const uint32_t small = tmem + S::kSmall + small_buf * BN;
        const uint32_t acc = tmem + buf * BN;
        // the stage's A of slot sa times its B of slot sb
        const auto product = [&](uint32_t to, int sa, int sb, bool add) {
          const uint64_t da = first_a + sa * (S::kStage >> 4), db = first_b + sb * (S::kStage >> 4);
#pragma unroll
          for (int kk = 0; kk < kBlockK / 16; ++kk) mma<CG>(to, da + kk * step_a, db + kk * step_b, idesc, add || kk > 0);
        };
        const auto arrived = [&] {  // the next slot, once it is full
          const int at = s;
          wait(full(s), phase, dead);
          fence_after();
          if (++s == S::kStages) s = 0, phase ^= 1;
          return at;
        };
        for (int x = 0; x < steps; ++x) {
          if constexpr (kF32) {
            bool add = x > 0 || !fresh;  // in the small products' accumulator
            const int mid = arrived();
            if (lane == 0 && !dead && more_a && more_b) product(small, mid, mid, add), add = true;
            const int hi = arrived();
            if (lane == 0 && !dead) {
              if (more_a) product(small, mid, hi, add), add = true;
              if (more_b) product(small, hi, mid, add);
              commit<CG>(empty(mid));
              product(acc, hi, hi, x > 0);
            }
            const int lo = arrived();
            if (lane == 0 && !dead) {
              if (more_a) product(small, lo, hi, true);
              if (more_b) product(small, hi, lo, true);
              commit<CG>(empty(hi));
              commit<CG>(empty(lo));
            }
          } else {
            const int at = arrived();
            if (lane == 0 && !dead) {
              product(acc, at, at, x > 0);
              commit<CG>(empty(at));
            }
          }
          __syncwarp();
        }
        if (lane == 0 && !dead) commit<CG>(acc_full(buf));
        __syncwarp();
        if (kF32 && (c + chunk >= t.kb1 || n % kFold == 0) && (small_buf ^= 1) == 0) small_phase ^= 1;
        buf ^= 1;
        if (buf == 0) acc_phase ^= 1;
      }
    }
    // the last products are done before their tensor memory goes, also where the epilogue gave up on them
    wait(acc_full(buf ^ 1), buf == 0 ? acc_phase ^ 1 : acc_phase, dead);
  } else if (warp < S::kWarps) {
    const Epilogue& e = job.pr.epi;
    const int mode = job.apart ? Epilogue::kStore : e.mode;
    const bool extra = mode != Epilogue::kStore && e.extra != nullptr;
    const int kind = mode == Epilogue::kFwd && e.slope ? kFwdSlope * 8 + static_cast<int>(e.act) * 2
                     : mode == Epilogue::kStore        ? Epilogue::kStore * 8
                                                       : mode * 8 + static_cast<int>(e.act) * 2 + (extra ? 1 : 0);
    const Place at{tmem, ring + S::kStages * S::kStage, bars, rank};
    if constexpr (sizeof(T) == 4 && !kF32) {  // partial sums
      dead = epilogue<BN, CG, T, kF32, Epilogue::kStore * 8>(maps, job, at);
    } else {
      switch (kind) {
        case Epilogue::kStore * 8: dead = epilogue<BN, CG, T, kF32, Epilogue::kStore * 8>(maps, job, at); break;
        case Epilogue::kFwd * 8: dead = epilogue<BN, CG, T, kF32, Epilogue::kFwd * 8>(maps, job, at); break;
        case Epilogue::kFwd * 8 + 1: dead = epilogue<BN, CG, T, kF32, Epilogue::kFwd * 8 + 1>(maps, job, at); break;
        case Epilogue::kFwd * 8 + 2: dead = epilogue<BN, CG, T, kF32, Epilogue::kFwd * 8 + 2>(maps, job, at); break;
        case Epilogue::kFwd * 8 + 3: dead = epilogue<BN, CG, T, kF32, Epilogue::kFwd * 8 + 3>(maps, job, at); break;
        case Epilogue::kFwd * 8 + 4: dead = epilogue<BN, CG, T, kF32, Epilogue::kFwd * 8 + 4>(maps, job, at); break;
        case Epilogue::kFwd * 8 + 5: dead = epilogue<BN, CG, T, kF32, Epilogue::kFwd * 8 + 5>(maps, job, at); break;
        case Epilogue::kFwd * 8 + 6: dead = epilogue<BN, CG, T, kF32, Epilogue::kFwd * 8 + 6>(maps, job, at); break;
        case Epilogue::kFwd * 8 + 7: dead = epilogue<BN, CG, T, kF32, Epilogue::kFwd * 8 + 7>(maps, job, at); break;
        case Epilogue::kDz * 8 + 3: dead = epilogue<BN, CG, T, kF32, Epilogue::kDz * 8 + 3>(maps, job, at); break;
        case Epilogue::kDz * 8 + 5: dead = epilogue<BN, CG, T, kF32, Epilogue::kDz * 8 + 5>(maps, job, at); break;
        case Epilogue::kDz * 8 + 7: dead = epilogue<BN, CG, T, kF32, Epilogue::kDz * 8 + 7>(maps, job, at); break;
        case kFwdSlope * 8 + 2: dead = epilogue<BN, CG, T, kF32, kFwdSlope * 8 + 2>(maps, job, at); break;
        case kFwdSlope * 8 + 4: dead = epilogue<BN, CG, T, kF32, kFwdSlope * 8 + 4>(maps, job, at); break;
        case kFwdSlope * 8 + 6: dead = epilogue<BN, CG, T, kF32, kFwdSlope * 8 + 6>(maps, job, at); break;
        default: dead = epilogue<BN, CG, T, kF32, kFwdSlope * 8>(maps, job, at);
      }
    }
  }
  if (dead) {
    for (uint32_t r = 0; r < CG; ++r)
      asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(in_block(spoilt, r)), "r"(1) : "memory");
  }
  __syncwarp();
  fence_before();
  block_or_pair_sync<CG>();
  uint32_t bad;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(bad) : "r"(spoilt) : "memory");
  if (bad && warp < S::kWarps)
    spoil<BN, CG, T, kF32>(maps, job, Place{tmem, ring + S::kStages * S::kStage, bars, rank});
  if (warp == kIssuer) {
    fence_after();
    tmem_free<CG>(tmem, S::kColumns);
  }
}

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

// Boxes of `box_cols` columns and `box_rows` rows of one plane, swizzled over
// the box's rows of 128 or 64 bytes; what lies outside the matrix reads as zero
// and is not written.
bool make_map(CUtensorMap* map, CUtensorMapDataType type, const void* p, int64_t cols, int64_t rows, int64_t planes,
              int64_t ld_bytes, int64_t plane_bytes, int box_cols, int box_rows, int row_bytes) {
  const EncodeTiledFn encode = encoder();
  if (!encode) return false;
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows),
                              static_cast<cuuint64_t>(planes)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(ld_bytes),
                                 static_cast<cuuint64_t>(planes > 1 ? plane_bytes : ld_bytes)};
  const cuuint32_t box[3] = {static_cast<cuuint32_t>(box_cols), static_cast<cuuint32_t>(box_rows), 1};
  const cuuint32_t unit[3] = {1, 1, 1};
  return encode(map, type, 3, const_cast<void*>(p), dims, strides, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE,
                row_bytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool operand_map(CUtensorMap* map, const Operand& o, int rows) {
  return make_map(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, o.p, o.cols, o.rows, o.planes, o.ld * 2, o.plane * 2, kBlockK,
                  rows, 128);
}

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

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Whether rows of extra, out and slope are what TMA and vectors of eight columns can address.
bool vectors_fit(const Product& pr) {
  const Epilogue& e = pr.epi;
  const int64_t size = pr.dtype == DType::kF32 ? 4 : 2;
  bool ok = aligned16(e.out) && (e.out_ld * (e.out_plane ? 2 : size)) % 16 == 0 && (e.out_plane * 2) % 16 == 0;
  if (e.extra) ok = ok && aligned16(e.extra) && (e.extra_ld * size) % 16 == 0 && e.extra_ld >= pr.n;
  if (e.slope) ok = ok && aligned16(e.slope) && (pr.n * size) % 16 == 0;
  return ok;
}

template <int BN, int CG, typename T, bool kF32>
cudaError_t launch(const Maps& maps, const Job& job, int sms, cudaStream_t stream) {
  using S = Shape<BN, CG, kF32>;
  const auto kernel = product_kernel<BN, CG, T, kF32>;
  static std::atomic<uint64_t> ready{0};  // devices (of the first 64) that know the kernel's shared memory
  const uint64_t bit = job.device < 64 ? 1ull << job.device : 0;
  if (!bit || !(ready.load(std::memory_order_relaxed) & bit)) {
    const cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem);
    if (err != cudaSuccess) return err;
    ready.fetch_or(bit, std::memory_order_relaxed);
  }
  const int64_t items = static_cast<int64_t>(job.tiles_m) * job.tiles_n * job.splits;
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
  return cudaLaunchKernelEx(&config, kernel, maps, job);
}

template <typename T, bool kF32>
cudaError_t launch_tile(const Plan& plan, const Maps& maps, const Job& job, int sms, cudaStream_t stream) {
  if constexpr (kF32) {
    if (plan.bn == 128) return launch<128, 2, T, kF32>(maps, job, sms, stream);
  } else {
    if (plan.bn == 256)
      return plan.pair == 2 ? launch<256, 2, T, kF32>(maps, job, sms, stream)
                            : launch<256, 1, T, kF32>(maps, job, sms, stream);
    if (plan.bn == 128) return launch<128, 1, T, kF32>(maps, job, sms, stream);
  }
  return launch<64, 1, T, kF32>(maps, job, sms, stream);
}

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

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

cudaError_t launch_product(const Product& pr, const Plan& plan, cudaStream_t stream) {
  if (pr.m == 0 || pr.n == 0) return cudaSuccess;
  Job job{};
  job.pr = pr;
  job.vec = vectors_fit(pr);
  job.splits = plan.splits;
  const bool f32 = pr.dtype == DType::kF32;
  if (pr.k > 0) {
    int sms = 148;
    cudaError_t err = cudaGetDevice(&job.device);
    // binds the device's context to this thread (autograd's threads may have none yet): the encoder needs one
    if (err == cudaSuccess) err = cudaSetDevice(job.device);
    if (err == cudaSuccess) err = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, job.device);
    if (err != cudaSuccess) return err;
    const int64_t tiles_m = ceil_div(pr.m, kTileM * plan.pair), tiles_n = ceil_div(pr.n, plan.bn);
    if (tiles_m * tiles_n * plan.splits >= 1ll << 31) return cudaErrorInvalidValue;
    job.tiles_m = static_cast<uint32_t>(tiles_m);
    job.tiles_n = static_cast<uint32_t>(tiles_n);
    const auto magic = [](uint64_t d) { return d <= 1 ? 0ull : ~0ull / d + 1; };
    job.by_tiles = magic(job.tiles_m * static_cast<uint64_t>(job.tiles_n));
    job.by_group = magic(kGroupM * static_cast<uint64_t>(job.tiles_n));
    job.by_last = magic(job.tiles_m % kGroupM);
    job.kblocks = static_cast<int>(ceil_div(pr.k, kBlockK));
    job.kblocks_per_split = plan.kblocks;
    job.apart = finished_apart(pr, plan);
    const int64_t rows_b = plan.bn / plan.pair;
    job.box_a = pr.a_mn ? 64 : static_cast<int>(std::min<int64_t>(kTileM, ceil_div(pr.m, 8) * 8));
    job.box_b = pr.b_mn ? 64 : static_cast<int>(std::min<int64_t>(rows_b, ceil_div(pr.n, 8) * 8));
    Maps maps{};
    if (!operand_map(&maps.a, pr.a, job.box_a) || !operand_map(&maps.b, pr.b, job.box_b) ||
        !epilogue_maps(maps, pr, plan, job.apart))
      return cudaErrorInvalidValue;
    if (f32)
      err = launch_tile<float, true>(plan, maps, job, sms, stream);
    else if (job.apart)
      err = launch_tile<float, false>(plan, maps, job, sms, stream);
    else
      err = launch_tile<bf16, false>(plan, maps, job, sms, stream);
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
