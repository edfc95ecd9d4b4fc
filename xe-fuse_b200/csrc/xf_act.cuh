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
// The same within a bounded relative error, for values that are kept in 32 bits or whose block makes its own scale:
// there the absolute bound above is 5e-4 of the result at g = -4 and 2e-2 at -10.  With z = |g| / sqrt 2 and
// t = 1 / (1 + 0.428 z), erfc(z) / 2 = exp(-g^2 / 2) t P(t); P is a minimax fit (degree 7, relative error 1.0e-7) of
// exp(z^2) erfc(z) / 2 t over 0 <= z <= 9.6, where g exp(-g^2 / 2) leaves the range of fp32.  In fp32: 8 x 2^-24 and
// the errors of the reciprocal (2 ulp) and of __expf, 2 + 1.173 g^2 / 2 ulp.
__device__ __forceinline__ float gelu_rel(float g) {
  const float t = __fdividef(1.0f, fmaf(0.3026417f, fabsf(g), 1.0f));
  float p = fmaf(0.03650734f, t, -0.15615574f);
  p = fmaf(p, t, 0.1972657f);
  p = fmaf(p, t, -0.04688882f);
  p = fmaf(p, t, 0.125341f);
  p = fmaf(p, t, 0.101547554f);
  p = fmaf(p, t, 0.12169367f);
  p = fmaf(p, t, 0.12068925f);
  const float tail = p * t * __expf(-0.5f * g * g);   // erfc(z) / 2
  return g * (g >= 0.0f ? 1.0f - tail : tail);
}

}  // namespace xf
