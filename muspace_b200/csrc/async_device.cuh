// Barriers and bulk copies in shared memory, shared by the layer kernels.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace async {

constexpr long long kWaitClocks = 4000000000ll;  // about two seconds

// Waits that gave up in this file's kernels.
static __device__ unsigned int g_wait_timeouts;

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

// Waits have a limit. One that runs out is counted (msda_layer_wait_timeouts)
// and leaves `dead` set: from then on the thread polls each barrier once, and
// starts no copies and no products. Its block waits once more, with a limit, for
// what is in flight, and writes NaNs over all of its results.
__device__ __forceinline__ void wait(uint32_t bar, uint32_t parity, bool& dead, long long limit = kWaitClocks) {
  if (try_wait(bar, parity)) return;
  if (dead) return;
  const long long start = clock64();
  do {
    if (try_wait(bar, parity)) return;
  } while (clock64() - start < limit);
  dead = true;
  atomicAdd(&g_wait_timeouts, 1u);
}

// `bytes` (a multiple of 16, both addresses too) into this block's shared memory; they count at `bar`.
__device__ __forceinline__ void copy_bytes(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

// The same once more, whatever ran out before: for copies in flight before their memory goes.
__device__ __forceinline__ void settle(uint32_t bar, uint32_t parity) {
  bool late = false;
  wait(bar, parity, late);
}

inline cudaError_t read_timeouts(unsigned int* count) {
  return cudaMemcpyFromSymbol(count, g_wait_timeouts, sizeof(*count));
}

}  // namespace async
