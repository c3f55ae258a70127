// Symmetric 8-bit quantization with one scale per vector (a token's row, or a token's head in
// the cache):
//
//   s = fl32(max|x| / 127),   c = round_half_even(x / s) clamped to [-127, 127]
//
// with the EXACT quotient x / s deciding the rounding, so that the codes do not depend on how
// the division is evaluated.  q = rint(x * fl(1/s)) is within one of the answer; the residual
// r = x - q s is exact in fp32 (for |x| >= s it is a multiple of ulp(s) no larger than s, for
// |x| < s either q = 0 or Sterbenz applies), so comparing |r| with s / 2 settles the rounding and
// its ties.  Almost every value takes four instructions: the product is rounded by adding
// 1.5 * 2^23, whose low bits then are the code, and |r| < s / 2 confirms it; the others (within
// rounding of a tie) go through code().  A vector of zeros has s = 0 and codes 0; a vector that holds an
// infinity or a NaN has s = NaN and codes 0, so whatever reads it back sees NaN instead of a plausible
// number.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace tfccb200 {

// max |x| is taken on the bit patterns of |x|: an integer maximum orders finite values,
// infinities and NaN in that order and is exact.
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t max_abs_bits(uint32_t m, float4 v) {
  return max(m, max(max(abs_bits(v.x), abs_bits(v.y)), max(abs_bits(v.z), abs_bits(v.w))));
}

struct TokenQuant {
  float scale;  // what is stored
  float up;     // power of two that moves tiny scales (and the values with them) away from the
                // subnormal range, where 1 / s would overflow
  float s, inv;
  bool live;    // false: every code is 0

  __device__ __forceinline__ explicit TokenQuant(uint32_t amax_bits) {
    scale = amax_bits >= 0x7f800000u ? __uint_as_float(0x7fffffffu)
                                     : __fdiv_rn(__uint_as_float(amax_bits), 127.0f);
    live = scale > 0.f;  // false for NaN
    up = scale < 8.6736174e-19f ? 1.2379400e27f : 1.0f;  // 2^-60, 2^90
    s = scale * up;
    inv = live ? __frcp_rn(s) : 0.f;
  }
  __device__ __forceinline__ int code(float x) const {
    const float v = x * up;
    float q = rintf(v * inv);
    const float r = fmaf(-q, s, v), a = fabsf(r), h = 0.5f * s;
    const bool odd = (__float2int_rn(q) & 1) != 0;
    if (a > h || (a == h && odd)) q += copysignf(1.0f, r);
    return live ? __float2int_rn(fminf(fmaxf(q, -127.0f), 127.0f)) : 0;
  }
  __device__ __forceinline__ uint32_t codes4(float4 v) const {
    if (!live) return 0;
    if (up == 1.0f) {
      constexpr float kMagic = 12582912.f;
      const float h = 0.5f * s;
      const float x[4] = {v.x, v.y, v.z, v.w};
      uint32_t q[4];
      bool sure = true;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float t = fmaf(x[i], inv, kMagic);
        q[i] = __float_as_uint(t);
        sure &= fabsf(fmaf(kMagic - t, s, x[i])) < h;
      }
      if (sure) return __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
    }
    const uint32_t a = code(v.x) & 0xff, b = code(v.y) & 0xff, c = code(v.z) & 0xff, d = code(v.w) & 0xff;
    return a | (b << 8) | (c << 16) | (d << 24);
  }
};

}  // namespace tfccb200
