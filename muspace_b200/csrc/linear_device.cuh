// Device code shared by the fused linear kernels: activations, the split of a
// float32 into three bfloat16, and the epilogue of eight neighbouring outputs.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "linear_act.h"

namespace lin {

using bf16 = __nv_bfloat16;

// ---- activations: value and slope --------------------------------------------------

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float reciprocal_fast(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLog2eLow = 1.9259630e-8f;  // log2(e) - kLog2e
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kInvSqrt2Pi = 0.39894228040143268f;

// Two float32 in one register pair: one instruction for both.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }
__device__ __forceinline__ float2 add2(float2 a, float2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

// Phi(z), the normal distribution function, and exp(-z^2 / 2), for two z. With
// x = |z| / sqrt 2, Phi(-|z|) = exp(-x^2) erfc(x) exp(x^2) / 2, whose factor of
// the exponential falls smoothly from 1/2 to 0 and is taken as a polynomial
// without constant term in t = 1 / (1 + 0.41 x). Its six coefficients were fitted
// for this kernel by a linear programme on 1500 points of |z| <= 13.3: they
// minimise the larger of relative error / 2^-12 and absolute error of Phi / 1e-7,
// which leaves 1.2e-4 and 4.7e-8 (in float32 arithmetic 2e-7). So z Phi(z) keeps
// bfloat16's digits down to where it underflows; five coefficients for the
// absolute error alone were off by 1 % at z = -8. The factor exp(-x^2) is the
// density's too, so the slope costs two more instructions. The bfloat16 kernels
// use it; float32 takes erfcf. It is bound by its reciprocal and exponential (16
// of them a clock on an SM, 2 a value): 20 million values take 9 us.
__device__ __forceinline__ void normal2(float2 z, float2& cdf, float2& bell) {
  const float2 t = make_float2(reciprocal_fast(fmaf(fabsf(z.x), 0.41f * 0.70710678118654752f, 1.f)),
                               reciprocal_fast(fmaf(fabsf(z.y), 0.41f * 0.70710678118654752f, 1.f)));
  const float2 w = mul2(mul2(z, z), both(-0.5f * kLog2e));
  bell = make_float2(exp2_fast(w.x), exp2_fast(w.y));
  float2 p = fma2(both(-0.08969429724f), t, both(0.2883247121f));
  p = fma2(p, t, both(-0.09784740124f));
  p = fma2(p, t, both(0.1824910442f));
  p = fma2(p, t, both(0.09979514776f));
  p = fma2(p, t, both(0.1169307474f));
  const float2 tail = mul2(mul2(p, t), bell);  // Phi(-|z|)
  cdf = make_float2(z.x < 0.f ? tail.x : 1.f - tail.x, z.y < 0.f ? tail.y : 1.f - tail.y);
}

// act(z) in place of z (kY) and act'(z) in `s` (kS), of N values: one branch for
// all of them. relu's slope at 0 is 0; a NaN stays a NaN. kFast: for bfloat16
// results.
template <bool kFast, bool kY, bool kS, int N>
__device__ __forceinline__ void activate(Act act, float* z, float* s) {
  if (act == Act::kGelu) {
#pragma unroll
    for (int j = 0; j < N; j += 2) {
      const float2 x = make_float2(z[j], z[j + 1]);
      float2 cdf, bell;
      if (kFast) {
        normal2(x, cdf, bell);
      } else {
        cdf = make_float2(0.5f * erfcf(-x.x * 0.70710678118654752f), 0.5f * erfcf(-x.y * 0.70710678118654752f));
        if (kS) bell = make_float2(expf(-0.5f * x.x * x.x), expf(-0.5f * x.y * x.y));
      }
      if (kS) {
        const float2 d = fma2(mul2(x, both(kInvSqrt2Pi)), bell, cdf);
        s[j] = d.x, s[j + 1] = d.y;
      }
      if (kY) {
        const float2 y = mul2(x, cdf);
        z[j] = y.x, z[j + 1] = y.y;
      }
    }
  } else if (act == Act::kSilu) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      float e;
      if (kFast) {
        e = exp2_fast(-kLog2e * z[j]);
      } else {
        // float32: with what the exponent lost in its rounding, to first order; below -88 the result is 0
        const float x = fmaxf(z[j], -88.f), t = kLog2e * x;
        const float lost = fmaf(-kLog2e, x, t) - kLog2eLow * x;
        e = exp2_fast(-t);
        e = fmaf(e, kLn2 * fminf(fmaxf(lost, -1.f), 1.f), e);
      }
      const float g = reciprocal_fast(1.f + e);
      if (kS) s[j] = g * fmaf(z[j], 1.f - g, 1.f);
      if (kY) z[j] *= g;
    }
  } else if (act == Act::kRelu) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      // two selects, by name: as nested ?: it became a branch per value, and the lanes parted
      // (forward with slope, 40000 x 256 x 512 bfloat16: 41 us instead of 32)
      if (kS)
        asm("{.reg .pred p; .reg .f32 t; setp.gt.f32 p, %1, 0f00000000; selp.f32 t, 0f3f800000, 0f00000000, p; "
            "setp.nan.f32 p, %1, %1; selp.f32 %0, %1, t, p;}"
            : "=f"(s[j])
            : "f"(z[j]));
      if (kY) asm("max.NaN.f32 %0, %0, 0f00000000;" : "+f"(z[j]));
    }
  } else if (kS) {
#pragma unroll
    for (int j = 0; j < N; ++j) s[j] = 1.f;
  }
}

// The sums over a warp's lanes of 16 values each: lane l gets that of value
// l / 2. Each step halves the values a lane still carries.
__device__ __forceinline__ float lane_sums16(const float v[16]) {
  const int lane = threadIdx.x & 31;
  float w[8];
#pragma unroll
  for (int n = 8, d = 16; n; n >>= 1, d >>= 1) {
    const bool high = lane & d;
#pragma unroll
    for (int j = 0; j < n; ++j) {
      const float lo = n == 8 ? v[j] : w[j], hi = n == 8 ? v[j + 8] : w[j + n];
      w[j] = (high ? hi : lo) + __shfl_xor_sync(0xffffffffu, high ? lo : hi, d);
    }
  }
  return w[0] + __shfl_xor_sync(0xffffffffu, w[0], 1);
}

// ---- float32 as three bfloat16 --------------------------------------------------------

// x = hi + mid + lo to 2^-24 of x or better: each part is the bfloat16 nearest
// to what is left. A finite x above bfloat16's largest value is cut, not
// rounded, to it; a non-finite x is all in hi.
__device__ __forceinline__ void split3(float x, bf16& hi, bf16& mid, bf16& lo) {
  hi = __float2bfloat16_rn(x);
  const uint32_t bits = __float_as_uint(x);
  const bool finite = (bits & 0x7f800000u) != 0x7f800000u;
  if (finite && (__bfloat16_as_ushort(hi) & 0x7f80u) == 0x7f80u)
    hi = __ushort_as_bfloat16(static_cast<unsigned short>(bits >> 16));
  const float r1 = finite ? x - __bfloat162float(hi) : 0.f;
  mid = __float2bfloat16_rn(r1);
  lo = __float2bfloat16_rn(r1 - __bfloat162float(mid));
}

__device__ __forceinline__ uint32_t pack2(bf16 a, bf16 b) {
  return static_cast<uint32_t>(__bfloat16_as_ushort(a)) | (static_cast<uint32_t>(__bfloat16_as_ushort(b)) << 16);
}

__device__ __forceinline__ uint32_t pack2(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

__device__ __forceinline__ float2 unpack2(uint32_t u) {
  return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}

// The largest magnitude's bits among N values; NaNs have the largest.
template <int N>
__device__ __forceinline__ uint32_t top_bits(const float* v) {
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < N; ++j) top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
  return top;
}

// N values as N / 2 pairs in each plane: two at a time where none is so large
// that bfloat16 rounds it to infinity.
template <int N>
__device__ __forceinline__ void split_pairs(const float* v, uint32_t top, uint32_t part[3][N / 2]) {
  if (top < 0x7f7f8000u) {
#pragma unroll
    for (int j = 0; j < N / 2; ++j) {
      const float2 minus = make_float2(-1.f, -1.f);
      float2 left = make_float2(v[2 * j], v[2 * j + 1]);
#pragma unroll
      for (int k = 0; k < 3; ++k) {
        part[k][j] = pack2(left.x, left.y);
        if (k < 2) left = fma2(unpack2(part[k][j]), minus, left);
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < N / 2; ++j) {
      bf16 a[3], b[3];
      split3(v[2 * j], a[0], a[1], a[2]);
      split3(v[2 * j + 1], b[0], b[1], b[2]);
#pragma unroll
      for (int k = 0; k < 3; ++k) part[k][j] = pack2(a[k], b[k]);
    }
  }
}

// ---- eight neighbouring values ----------------------------------------------------------

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(bf16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ bf16 from_float<bf16>(float v) {
  return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ __half from_float<__half>(float v) {
  return __float2half_rn(v);
}

__device__ __forceinline__ void load8(const bf16* p, float v[8]) {
  const uint4 u = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void load8(const float* p, float v[8]) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
  v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
__device__ __forceinline__ void load8(const __half* p, float v[8]) {
  const uint4 u = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void store8(bf16* p, const float v[8]) {
  *reinterpret_cast<uint4*>(p) =
      make_uint4(pack2(v[0], v[1]), pack2(v[2], v[3]), pack2(v[4], v[5]), pack2(v[6], v[7]));
}
__device__ __forceinline__ void store8(float* p, const float v[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void store8(__half* p, const float v[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

// Loads / stores of up to eight elements: one vector access where the caller
// knows that address and length allow it.
template <typename T>
__device__ __forceinline__ void load_some(const T* p, int count, bool vec, float v[8]) {
  if (vec) {
    load8(p, v);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < count ? to_float(p[j]) : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void store_some(T* p, int count, bool vec, const float v[8]) {
  if (vec) {
    store8(p, v);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < count) p[j] = from_float<T>(v[j]);
  }
}

// Splits eight values into the three planes at p, p + plane, p + 2 plane.
__device__ __forceinline__ void store_planes(bf16* p, int64_t plane, int count, bool vec, const float v[8]) {
  uint32_t part[3][4];
  split_pairs<8>(v, top_bits<8>(v), part);
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    if (vec) {
      *reinterpret_cast<uint4*>(p + i * plane) = make_uint4(part[i][0], part[i][1], part[i][2], part[i][3]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < count)
          p[i * plane + j] = __ushort_as_bfloat16(static_cast<unsigned short>(part[i][j / 2] >> (16 * (j % 2))));
    }
  }
}

// ---- eight float16 under one exponent ---------------------------------------------------

// Factors of any size, eight at a time: scaled by the power of two that brings the largest
// finite one into [2^14, 2^15), as halves. Down to 2^-28 of that one they keep 11 bits; below
// that they are off by up to 2^-39 of it, half of the halves' smallest step. The exponent kept
// is the largest one's float32 exponent (15 at least: what is below 2^-112 loses digits).
// Infinities and NaNs are kept as they are.
constexpr uint32_t kFactorShift = 141;  // the exponent of 2^14

// What stands in the place of a dropped element's Q: a NaN that no arithmetic leaves (its NaNs
// are 0x7fff and 0x7fffffff), nor a wait that ran out (all ones).
constexpr uint32_t kDroppedHalf = 0xfffe, kDroppedFloat = 0xfffffffe;

// Eight factors as halves; their exponent.
__device__ __forceinline__ uint32_t pack_factors8(const float v[8], uint32_t w[4]) {
  float most = fabsf(v[0]);
#pragma unroll
  for (int j = 1; j < 8; ++j) most = fmaxf(most, fabsf(v[j]));  // of a NaN and a number it is the number
  uint32_t top = __float_as_uint(most);
  if (top >= 0x7f800000u) {  // rare: no call here, whose registers every other eight would pay for
    top = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t bits = __float_as_uint(v[j]) & 0x7fffffffu;
      top = max(top, bits < 0x7f800000u ? bits : 0u);
    }
  }
  const uint32_t e = max(top >> 23, 15u);
  const float2 scale = both(__uint_as_float((127u + kFactorShift - e) << 23));
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const __half2 h = __float22half2_rn(mul2(make_float2(v[2 * j], v[2 * j + 1]), scale));
    w[j] = *reinterpret_cast<const uint32_t*>(&h);
  }
  return e;
}

// Where the exponent of P (half 0) or Q in row m, columns c to c + 7 lies: neighbouring
// rows' four of 32 columns are neighbours, as a warp of the epilogue writes them (by rows
// of all columns, 40000 x 256 x 512 took 90 us instead of 76: parts of sectors).
__device__ __forceinline__ int64_t exponent_at(int64_t rows, int64_t cols, int half, int64_t m, int64_t c) {
  return ((half * ((cols + 31) / 32) + c / 32) * rows + m) * 4 + c % 32 / 8;
}

__device__ __forceinline__ float factor_scale(uint32_t e) { return __uint_as_float((e + 127u - kFactorShift) << 23); }

// ---- the epilogue -----------------------------------------------------------------------

template <typename T>
struct SlopeOf {
  // Of bfloat16 outputs: a slope lies in [-0.2, 1.2], where float16 keeps 11 bits; one
  // below 2^-14 is kept to 2^-25, which is nothing beside the slopes of other elements.
  using type = __half;
};
template <>
struct SlopeOf<float> {
  using type = float;
};

// Eight neighbouring outputs of row m, of sums that were finished apart.
template <typename T>
__device__ __forceinline__ void finish8(const Epilogue& e, float v[8], const float x[8], const float b[8], int64_t m,
                                        int64_t n, int64_t cols, int count, bool vec) {
  if (e.mode != Epilogue::kStore) {
    float s[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] += b[j];
    activate<sizeof(T) == 2, true, true, 8>(e.act, v, s);
    if (e.mode == Epilogue::kFwd) {
      if (e.slope) store_some(static_cast<typename SlopeOf<T>::type*>(e.slope) + m * cols + n, count, vec, s);
      if (e.extra) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] += x[j];
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = x[j] * s[j];
      if (e.unrounded) store8(e.unrounded + m * partial_ld(cols) + n, v);
      if (sizeof(T) == 4) {
        store_planes(static_cast<bf16*>(e.out) + m * e.out_ld + n, e.out_plane, count, vec, v);
        return;
      }
    }
  }
  store_some(static_cast<T*>(e.out) + m * e.out_ld + n, count, vec, v);
}

// The same where vectors do not fit, out of the way.
template <typename T>
__device__ __noinline__ void finish_some(const Epilogue& e, const float4 lo, const float4 hi, int64_t m, int64_t n,
                                         int64_t cols) {
  const int count = static_cast<int>(cols - n < 8 ? cols - n : 8);
  float v[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w}, x[8] = {}, b[8] = {};
  if (e.extra) load_some(static_cast<const T*>(e.extra) + m * e.extra_ld + n, count, false, x);
  if (e.bias) load_some(static_cast<const T*>(e.bias) + n, count, false, b);
  finish8<T>(e, v, x, b, m, n, cols, count, false);
}

}  // namespace lin
