// The gated activation situ(g) up' of one element and its derivatives, for the row kernels.
#pragma once

namespace imf {

// situ(g) = beta tanh(g/beta) sigmoid(g); up' = lbeta tanh(up/lbeta).  The hyperbolic
// tangent is the hardware approximation (one MUFU op, error below bf16 resolution) and the
// sigmoid is written through it, sigmoid(x) = 0.5 tanh(x / 2) + 0.5: three special-function
// ops per element, so the kernels that use it stay memory-bound.
__device__ __forceinline__ float tanh_fast(float x) {
  float y;
  asm("tanh.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void situ1(float g, float u, float beta, float inv_beta, float lbeta,
                                      float inv_lbeta, int has_lb, float& a, float& da_dg,
                                      float& up, float& dup_du) {
  const float th = tanh_fast(g * inv_beta), sg = fmaf(0.5f, tanh_fast(0.5f * g), 0.5f);
  a = beta * th * sg;
  da_dg = (1.f - th * th) * sg + beta * th * sg * (1.f - sg);
  if (has_lb) {
    const float tu = tanh_fast(u * inv_lbeta);
    up = lbeta * tu;
    dup_du = 1.f - tu * tu;
  } else {
    up = u;
    dup_du = 1.f;
  }
}

}  // namespace imf
