// Gate activations of the row passes and of the grouped product's epilogue.
#pragma once

namespace xf {

__device__ __forceinline__ float silu_f(float g) { return __fdividef(g, 1.0f + __expf(-g)); }
// The same by 2^(-g log2 e) and one reciprocal, both approximations flushing subnormals: half the instructions.
// A subnormal exponential adds nothing to 1, and 1 + e^-g = infinity gives -0 as it should.
__device__ __forceinline__ float silu_fast(float g) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(g * -1.4426950408889634f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
  return g * r;
}
// erf-GeLU, g * 0.5 * (1 + erf(g / sqrt 2)), with erf from the five-term rational approximation of
// Abramowitz & Stegun 7.1.26 (absolute error below 1.5e-7): 1 - erf(z) = P(t) exp(-z^2),
// t = 1 / (1 + p z), z >= 0.  For negative g the factor 1 + erf is formed directly as P(t) exp(-z^2),
// so the far tail does not cancel.  A third of the instructions of erff().
__device__ __forceinline__ float gelu_f(float g) {
  const float z = fabsf(g) * 0.7071067811865475f;
  const float t = __fdividef(1.0f, fmaf(0.3275911f, z, 1.0f));
  float p = fmaf(1.061405429f, t, -1.453152027f);
  p = fmaf(p, t, 1.421413741f);
  p = fmaf(p, t, -0.284496736f);
  p = fmaf(p, t, 0.254829592f);
  const float pe = p * t * __expf(-z * z);         // 1 - erf(z)
  return g * 0.5f * (g >= 0.0f ? 2.0f - pe : pe);
}

}  // namespace xf
