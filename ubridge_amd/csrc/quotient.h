// quotient.h -- v / s, correctly rounded, for many v of one s (a row's scale).
#pragma once
#include <hip/hip_runtime.h>

namespace {

// v r (r = 1 / s, correctly rounded) corrected twice by its exact residual v - q s
// (Markstein's division: the second correction of a faithful q gives the correctly
// rounded one), 5 operations where the IEEE divide takes 11.  For s of ub_exact_scale.  A
// zero comes out as +0.
__device__ __forceinline__ float ub_quotient(float v, float s, float r) {
  float q = v * r;
  q = __builtin_fmaf(__builtin_fmaf(-q, s, v), r, q);
  return __builtin_fmaf(__builtin_fmaf(-q, s, v), r, q);
}
// Where residuals do not underflow, of quotients that 8 bits do not round to zero.
__device__ __forceinline__ bool ub_exact_scale(float s) { return s >= 0x1p-60f && s <= 0x1p60f; }

}  // namespace
