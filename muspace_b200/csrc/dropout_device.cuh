// Device code of dropout: which elements are kept, from a counter-based generator.
//
// Philox-4x32 with ten rounds (J. Salmon, M. Moraes, R. Dror, D. Shaw, "Parallel
// random numbers: as easy as 1, 2, 3", 2011). The key is the seed; the counter is
// (column / 8, row, sequence), so a mask depends on where an element stands and on
// nothing of how a kernel walks over it, and the backward pass makes it again
// instead of reading it. One call gives eight neighbouring columns 16 bits each; an
// element is kept where its number is at least t, so p is a multiple of 2^-16. With
// 32 bits an element (p to 2^-32) a call covers four columns: the twenty wide
// multiplications then cost what the bytes of a bfloat16 tensor do.
#pragma once

#include <stdint.h>

#include "dropout.h"

namespace drop {

struct Words {
  uint32_t w[4];
};

// A rule as a thread uses it: the key in registers.
struct Key {
  uint32_t k0, k1, s0, s1;
  uint32_t low, high;  // kept where a number, in the upper half of a word, is above these
  float scale;
};

__device__ __forceinline__ Key key_of(const Rule& rule) {
  const uint64_t seed = rule.seed_at ? static_cast<uint64_t>(__ldg(rule.seed_at)) : rule.seed;
  const uint32_t last = (rule.threshold - 1u) << 16;
  return Key{static_cast<uint32_t>(seed),          static_cast<uint32_t>(seed >> 32),
             static_cast<uint32_t>(rule.sequence), static_cast<uint32_t>(rule.sequence >> 32),
             last,                                 last | 0xffffu,
             rule.scale};
}

// The numbers of columns 8 group to 8 group + 7 of a row.
__device__ __forceinline__ Words numbers(const Key& key, uint32_t row, uint32_t group) {
  uint32_t c0 = group, c1 = row, c2 = key.s0, c3 = key.s1, k0 = key.k0, k1 = key.k1;
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t a = static_cast<uint64_t>(0xD2511F53u) * c0, b = static_cast<uint64_t>(0xCD9E8D57u) * c2;
    c0 = static_cast<uint32_t>(b >> 32) ^ c1 ^ k0;
    c1 = static_cast<uint32_t>(b);
    c2 = static_cast<uint32_t>(a >> 32) ^ c3 ^ k1;
    c3 = static_cast<uint32_t>(a);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return Words{{c0, c1, c2, c3}};
}

__device__ __forceinline__ bool kept(const Key& key, const Words& n, int j) {
  return j % 2 ? n.w[j / 2] > key.high : (n.w[j / 2] << 16) > key.low;
}

// D of eight neighbouring values: what is dropped is 0, whatever it was.
__device__ __forceinline__ void apply8(const Key& key, const Words& n, float v[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = kept(key, n, j) ? v[j] * key.scale : 0.f;
}

// The eight as bits of a byte.
__device__ __forceinline__ uint32_t bits8(const Key& key, const Words& n) {
  uint32_t bits = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) bits |= kept(key, n, j) ? 1u << j : 0u;
  return bits;
}

}  // namespace drop
