// What linear_sm100.cu shares: with linear_grad.cu, and host functions.
#pragma once

namespace mr {

// Device status word of K13 (0, or MR_ERR_TIMEOUT); synchronizes.
int linear_status(int reset);

// Phi(-|z|) = t 2^(p(t) - z^2 log2(e) / 2) with t = 1 / (1 + |z| / 2) and p the
// quartic of least largest error (fitted for |z| <= 13.2, where the tail leaves
// float32's range): relative error 5.5e-5.
__device__ __forceinline__ float gelu_tail(float z) {
  const float t = __fdividef(1.f, fmaf(0.5f, fabsf(z), 1.f));
  float p = fmaf(0.375025481f, t, -1.147340059f);
  p = fmaf(p, t, 0.711058915f);
  p = fmaf(p, t, 1.383448601f);
  p = fmaf(p, t, -2.322162628f);
  float power;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(power) : "f"(fmaf(-0.72134752f * z, z, p)));
  return t * power;
}

}  // namespace mr
