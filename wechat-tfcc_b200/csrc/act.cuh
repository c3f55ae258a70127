// Activations shared by the GEMM epilogues and the stand-alone element-wise kernels.
#pragma once

#include <cuda_runtime.h>

#include "../../include/tfcc_b200.h"

namespace tfccb200 {

// 0.5 * v * (1 + erf(v / sqrt(2))) with the reference's mixed precision
// (tfcc/mkl/kernel/tfcc_mklactivationkernel.hpp:214-220).  There the literal 0.5 is a double,
// so 0.5 * v * e is evaluated in double and rounded to float once.  Both factors are floats
// (e = 1 + erf(float) is a float sum), so their product is exact in double and the single
// rounding equals one float multiplication; halving e first is exact too.  No double
// arithmetic is needed for the same bits.
__device__ __forceinline__ float gelu_erf(float v) {
  const float e = 1.0f + erff(v / 1.4142135623730951f);
  return __fmul_rn(v, 0.5f * e);
}

// The same function where it has to be cheap (an epilogue of four warps per SM): with
// erfc(z) = (a1 t + ... + a5 t^5) exp(-z^2), t = 1 / (1 + p z), the rational approximation 7.1.26 of
// Abramowitz and Stegun, whose error is at most 1.5e-7; v (1 + erf(v / sqrt 2)) / 2 is then off by at
// most 7.5e-8 |v| and the roundings, where erff costs three times the instructions.
__device__ __forceinline__ float gelu_erfc(float v) {
  const float z = fabsf(v) * 0.70710678118654752f;
  float t, e;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(fmaf(0.3275911f, z, 1.0f)));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(z * z * -1.4426950408889634f));
  float q = fmaf(1.061405429f, t, -1.453152027f);
  q = fmaf(q, t, 1.421413741f);
  q = fmaf(q, t, -0.284496736f);
  q = fmaf(q, t, 0.254829592f);
  const float h = 0.5f * q * t * e;  // erfc(z) / 2
  return v * (v >= 0.f ? 1.f - h : h);  // (a factor, not a difference: infinity stays infinity)
}

__device__ __forceinline__ float apply_activation(float v, int activation) {
  return activation == TFCCB200_ACT_GELU_ERF ? gelu_erf(v) : v;
}

}  // namespace tfccb200
