// Exponentials on the ex2 unit.
#pragma once

namespace fk {

constexpr float kLog2e = 1.4426950408889634f;

// 2^x to 2 ulp; results below 2^-126 are flushed to 0.
__device__ __forceinline__ float ex2f(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float max_or_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// exp(d), d <= 0, in 32 bits: 2^(d log2 e) with the product in two parts, hi + lo (log2 e =
// kLog2e + kLog2eLow, the roundings of the products caught by FMAs), so that the error stays
// that of ex2 for any d: 2^hi * (1 + lo ln 2), lo being below 2^-16.  d is held at -200 from
// below (2^hi is 0 there), so that -inf does not meet its own residual.
constexpr float kLog2eLow = 1.9259629911266174e-8f;
constexpr float kLn2 = 0.69314718055994531f;
__device__ __forceinline__ float exp2_of(float d) {
  d = max_or_nan(d, -200.f);
  const float hi = d * kLog2e;
  const float lo = fmaf(d, kLog2eLow, fmaf(d, kLog2e, -hi));
  const float p = ex2f(hi);
  return fmaf(p * kLn2, lo, p);
}

}  // namespace fk
