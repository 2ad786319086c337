// Device code of 8-bit activation checkpoints.
//
// A row is cut into blocks of 32 elements (the last may be short). A block is
// held as integers q = rint(x / 2^e), ties to even, and one byte e + 127, e
// the smallest integer >= -126 with max|x| <= 127 * 2^e. Scaling by a power
// of two is exact, so the only rounding is q's, and q * 2^e is a float32 and a
// bfloat16 alike; only 64 * 2^122 = 2^128 would not be, and is held as 63. A
// block with an infinity or a NaN is held as the byte 255
// and comes back as NaNs: its gradients say so.
#pragma once

#include <stdint.h>

namespace ckpt {

constexpr int kBlock = 32;
constexpr uint32_t kNonFinite = 255;
constexpr uint32_t kTopExponent = 249;  // of the largest finite values

__host__ __device__ __forceinline__ int64_t blocks_of(int64_t cols) { return (cols + kBlock - 1) / kBlock; }

// The byte for a block whose largest |x| has the bits `top` (of a float; NaN
// and infinity are the largest bit patterns). With top = m * 2^p, m in [1, 2):
// m * 2^p <= 127 * 2^e needs e = p - 6 where m <= 127 / 64, and p - 5 above.
__device__ __forceinline__ uint32_t exponent_of(uint32_t top) {
  if (top >= 0x7f800000u) return kNonFinite;
  const int p = static_cast<int>(top >> 23);  // biased; 0 for subnormals
  const int e = p - 6 + ((top & 0x7fffffu) > 0x7e0000u ? 1 : 0);
  return static_cast<uint32_t>(e < 1 ? 1 : e);
}

__device__ __forceinline__ float scale_of(uint32_t e) {
  return e == kNonFinite ? __uint_as_float(0x7fc00000u) : __uint_as_float(e << 23);
}

__device__ __forceinline__ float inverse_scale(uint32_t e) {
  return e == kNonFinite ? 0.f : __uint_as_float((254u - e) << 23);  // e <= 249, so this is normal
}

__device__ __forceinline__ int code_of(float x, uint32_t e, float inverse) {
  const float v = x * inverse;  // exact, or below 2^-126 of a code
  const int q = v == v ? __float2int_rn(v) : 0;
  return e == kTopExponent ? max(-63, min(63, q)) : q;
}

// Up to eight values of one block as codes.
__device__ __forceinline__ void store_codes8(int8_t* p, int count, bool vec, uint32_t e, const float v[8]) {
  const float inv = inverse_scale(e);
  if (vec) {
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j >> 2] |= static_cast<uint32_t>(code_of(v[j], e, inv) & 0xff) << (8 * (j & 3));
    *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < count) p[j] = static_cast<int8_t>(code_of(v[j], e, inv));
  }
}

// Eight codes of one block as numbers.
__device__ __forceinline__ void values_of(uint2 u, uint32_t e, float v[8]) {
  const float s = scale_of(e);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t w = j < 4 ? u.x : u.y;
    v[j] = static_cast<float>(static_cast<int8_t>(w >> (8 * (j & 3)))) * s;
  }
}

// Up to eight codes of one block as numbers.
__device__ __forceinline__ void load_codes8(const int8_t* p, int count, bool vec, uint32_t e, float v[8]) {
  if (vec) {
    values_of(*reinterpret_cast<const uint2*>(p), e, v);
  } else {
    const float s = scale_of(e);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < count ? static_cast<float>(p[j]) * s : 0.f;
  }
}

}  // namespace ckpt
