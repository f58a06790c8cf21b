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
// The steps of PAIRS pairs go side by side: one coefficient in registers serves them all, and there is
// something to do while each waits for its own last step.
template <int PAIRS>
__device__ __forceinline__ void gelu2(float2 (&x)[PAIRS]) {
  constexpr float kQ[8] = {1.889626219e-06f, 6.268139987e-05f,  9.388679173e-04f, 8.539461531e-03f,
                           5.402068794e-02f, -4.584097862e-01f, 1.151269197e+00f, -9.999943376e-01f};
  float2 n[PAIRS], q[PAIRS];
#pragma unroll
  for (int i = 0; i < PAIRS; ++i) {
    n[i] = make_float2(fmaxf(-fabsf(x[i].x), -6.0f), fmaxf(-fabsf(x[i].y), -6.0f));
    q[i] = make_float2(kQ[0], kQ[0]);
  }
#pragma unroll
  for (int k = 1; k < 8; ++k)
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) q[i] = __ffma2_rn(q[i], n[i], make_float2(kQ[k], kQ[k]));
#pragma unroll
  for (int i = 0; i < PAIRS; ++i) {
    float2 t;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(t.x) : "f"(q[i].x));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(t.y) : "f"(q[i].y));
    x[i] = __ffma2_rn(n[i], t, make_float2(max_nan(x[i].x, 0.f), max_nan(x[i].y, 0.f)));
  }
}

}  // namespace mxf4
}  // namespace hom
