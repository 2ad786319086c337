// The persistent product of two operands on the tensor cores, without its epilogue:
// tiles, copies, products and barriers, and the pieces that epilogues are made of.
// linear_gemm.cu has the reasons; it and linear_gated.cu bring epilogues of their own.
#pragma once

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

// kGated: a tile's columns are BN / 2 of the gate and, behind them, the BN / 2 of up
// at the same place; its epilogue has three boxes of half a warp's size.
template <int BN, int CG, bool kF32, bool kGated = false>
struct Shape {
  static constexpr int kPlanes = kF32 ? 3 : 1;
  static constexpr int kRowsB = BN / CG;  // rows of B in one block's stage
  static constexpr int kStageB = kRowsB * kBlockK * 2;
  static constexpr int kStage = kStageA + kStageB;  // one plane of both
  static constexpr int kBox = kGated ? kBoxBytes / 2 * 3 : kBoxBytes;  // of a warp's staging
  static constexpr int kRing = kGated ? kRingBytes - kEpiWarps * kBoxBytes / 2 : kRingBytes;
  static constexpr int kStages = kRing / kStage;
  static constexpr int kTileN = kGated ? BN / 2 : BN;  // columns of the output in a tile
  static constexpr int kBarriers = 2 * kStages + 4 + kEpiWarps + (kF32 ? 2 : 0);
  // stages, the warps' staging, barriers, the tensor-memory address; and room to start on 1024 bytes
  static constexpr int kSmem = kStages * kStage + kEpiWarps * kBox + kBarriers * 8 + 16 + 1024;
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

// The i-th item, of tiles of kTileN columns.
template <int kTileN, int CG>
__device__ __forceinline__ Item item_of(const Job& j, uint32_t i) {
  Item t;
  t.split = static_cast<int>(divided(i, j.by_tiles));
  const uint32_t at = i - t.split * j.tiles_m * j.tiles_n;
  const uint32_t group = divided(at, j.by_group), first = group * kGroupM;
  const uint32_t local = at - group * (kGroupM * j.tiles_n);
  const uint32_t rows = j.tiles_m - first;  // of tiles in the group, if fewer than usual
  const uint32_t col = rows >= kGroupM ? local / kGroupM : divided(local, j.by_last);
  t.m = static_cast<int>((first + local - col * min(rows, static_cast<uint32_t>(kGroupM))) * (kTileM * CG));
  t.n = static_cast<int>(col * kTileN);
  t.kb0 = t.split * j.kblocks_per_split;
  t.kb1 = min(j.kblocks, t.kb0 + j.kblocks_per_split);
  return t;
}

// ---- the epilogue ------------------------------------------------------------------------

// A warp's box in shared memory: 32 rows of 128, 64 or 32 bytes, whose 16-byte units
// (of the first two) are exchanged by the row's number as TMA's swizzle has it; eight neighbouring
// rows' units at one place then lie in different banks.
template <int kRowBytes>
__device__ __forceinline__ uint32_t unit_at(uint32_t box, int row, int unit) {
  return kRowBytes == 128  ? box + row * 128 + ((unit ^ (row & 7)) << 4)
         : kRowBytes == 64 ? box + row * 64 + ((unit ^ ((row >> 1) & 3)) << 4)
                           : box + row * 32 + (unit << 4);
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

// Epi: kGated, and for the epilogue's warps run() from the first tile to the last,
// which returns whether a wait ran out, and spoil(), which then writes NaNs over all
// that the block's epilogue writes.
template <int BN, int CG, typename T, bool kF32, typename Epi>
__global__ void __launch_bounds__(kThreads, 1)
    product_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Job job) {
  constexpr bool kGated = Epi::kGated;
  using S = Shape<BN, CG, kF32, kGated>;
  extern __shared__ uint8_t raw[];
  const uint32_t ring = (smem_addr(raw) + 1023) & ~1023u;
  const uint32_t bars = ring + S::kStages * S::kStage + kEpiWarps * S::kBox;
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
      const Item t = item_of<S::kTileN, CG>(job, i);
      // boxes that hold rows of the tile; what a skipped box leaves in its place reaches no row or column that is kept
      const auto boxes = [](int have, int most) { return have <= 0 ? 0 : min(most, (have - 1) / 64 + 1); };
      const auto bytes_a = [&](int ma) { return job.pr.a_mn ? boxes(rows_m - ma, kTileM / 64) * 8192 : job.box_a * 128; };
      const auto bytes_b = [&](int nb) {
        if (kGated) return (CG == 2 ? 1 : 2) * job.box_b * 128;  // a box of each half
        return job.pr.b_mn ? boxes(rows_n - nb, S::kRowsB / 64) * 8192 : job.box_b * 128;
      };
      const int ma = t.m + rank * kTileM;
      const int nb = kGated ? t.n + static_cast<int>(rank) * rows_n : t.n + static_cast<int>(rank) * S::kRowsB;
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
              if (kGated && CG == 1 && has_b) copy_box<CG>(b + BN / 2 * 128, &maps.b, k, rows_n + nb, p, bar);
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
      const Item t = item_of<S::kTileN, CG>(job, i);
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
    dead = Epi::template run<BN, CG, T, kF32>(maps, job, Place{tmem, ring + S::kStages * S::kStage, bars, rank});
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
    Epi::template spoil<BN, CG, T, kF32>(maps, job, Place{tmem, ring + S::kStages * S::kStage, bars, rank});
  if (warp == kIssuer) {
    fence_after();
    tmem_free<CG>(tmem, S::kColumns);
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
// the box's rows of 128 or 64 bytes (32: as they are); what lies outside the matrix reads as zero
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
                row_bytes == 128  ? CU_TENSOR_MAP_SWIZZLE_128B
                : row_bytes == 64 ? CU_TENSOR_MAP_SWIZZLE_64B
                                  : CU_TENSOR_MAP_SWIZZLE_NONE,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool operand_map(CUtensorMap* map, const Operand& o, int rows) {
  return make_map(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, o.p, o.cols, o.rows, o.planes, o.ld * 2, o.plane * 2, kBlockK,
                  rows, 128);
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// The tiles and ranges of k of a launch over the current device: the output
// in tiles of `tile_cols` columns.
cudaError_t prepare(Job& job, const Plan& plan, int64_t tile_cols, int* sms) {
  const Product& pr = job.pr;
  cudaError_t err = cudaGetDevice(&job.device);
  // binds the device's context to this thread (autograd's threads may have none yet): the encoder needs one
  if (err == cudaSuccess) err = cudaSetDevice(job.device);
  if (err == cudaSuccess) err = cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, job.device);
  if (err != cudaSuccess) return err;
  const int64_t tiles_m = ceil_div(pr.m, kTileM * plan.pair), tiles_n = ceil_div(pr.n, tile_cols);
  if (tiles_m * tiles_n * plan.splits >= 1ll << 31) return cudaErrorInvalidValue;
  job.tiles_m = static_cast<uint32_t>(tiles_m);
  job.tiles_n = static_cast<uint32_t>(tiles_n);
  const auto magic = [](uint64_t d) { return d <= 1 ? 0ull : ~0ull / d + 1; };
  job.by_tiles = magic(job.tiles_m * static_cast<uint64_t>(job.tiles_n));
  job.by_group = magic(kGroupM * static_cast<uint64_t>(job.tiles_n));
  job.by_last = magic(job.tiles_m % kGroupM);
  job.kblocks = static_cast<int>(ceil_div(pr.k, kBlockK));
  job.kblocks_per_split = plan.kblocks;
  return cudaSuccess;
}

template <int BN, int CG, typename T, bool kF32, typename Epi>
cudaError_t launch(const Maps& maps, const Job& job, int sms, cudaStream_t stream) {
  using S = Shape<BN, CG, kF32, Epi::kGated>;
  const auto kernel = product_kernel<BN, CG, T, kF32, Epi>;
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

}  // namespace
}  // namespace lin
