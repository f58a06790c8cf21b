// Epilogue arithmetic of the 4-bit products.
#pragma once

#include <cuda_fp16.h>
#include <cuda_runtime.h>

namespace hom {
namespace mxf4 {

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// erf GELU of two values with one special-function result each: with n = max(-|x|, -6),
//   GELU(x) = max(x, 0) + n * T(n),   T(n) = erfc(-n / sqrt2) / 2 = 2^Q(n),
// Q the degree-7 polynomial of gemm_epilogue.cuh's gelu_erf_fast2 in -n (max abs error 6.2e-7, 4e-6
// relative where |GELU| > 1e-4).  Taking n instead of -n needs no negation in the packed last step;
// NaN passes through the first term; -infinity gives the limit, 0.
__device__ __forceinline__ float2 gelu2(float2 x) {
  const float2 n = make_float2(fmaxf(-fabsf(x.x), -6.0f), fmaxf(-fabsf(x.y), -6.0f));
  float2 q = make_float2(1.889626219e-06f, 1.889626219e-06f);
  q = __ffma2_rn(q, n, make_float2(6.268139987e-05f, 6.268139987e-05f));
  q = __ffma2_rn(q, n, make_float2(9.388679173e-04f, 9.388679173e-04f));
  q = __ffma2_rn(q, n, make_float2(8.539461531e-03f, 8.539461531e-03f));
  q = __ffma2_rn(q, n, make_float2(5.402068794e-02f, 5.402068794e-02f));
  q = __ffma2_rn(q, n, make_float2(-4.584097862e-01f, -4.584097862e-01f));
  q = __ffma2_rn(q, n, make_float2(1.151269197e+00f, 1.151269197e+00f));
  q = __ffma2_rn(q, n, make_float2(-9.999943376e-01f, -9.999943376e-01f));
  float2 t;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(t.x) : "f"(q.x));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(t.y) : "f"(q.y));
  return __ffma2_rn(n, t, make_float2(max_nan(x.x, 0.f), max_nan(x.y, 0.f)));
}

}  // namespace mxf4
}  // namespace hom
