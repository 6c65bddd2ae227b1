// Host-side interface of differential attention (attn_diff_fwd.cu, attn_diff_bwd.cu).
//
// Heads 2j and 2j + 1 of q, k, v (B, L, 2H, 64) form pair j.  Both maps of a pair multiply the pair's
// values side by side, V = [v_2j | v_2j+1] (128 channels):
//   A_m = softmax(scale q_m k_m^T),  O_m = A_m V,  o = O_1 - lam O_2
//
// The backward pass needs delta_m = rowsum(dO .* O_m), and an error of delta moves every dS of its row the same
// way: from o and O_2 in bf16, dQ was 1.1 % of its norm off at 29,140 tokens whose values have an offset (what
// the keys of a row have in common adds up, what tells them apart averages out).  So the forward pass also
// keeps a signed byte for each value, what bf16 dropped in 1/256 of its last place: 16 bits in all.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"

namespace imf {

// The pairs' weights: bf16 or fp32, `stride` elements apart (0: one weight for all pairs).
struct DiffWeights {
  const void* p;
  int64_t stride;
  int is_bf16;
  __device__ __forceinline__ float at(int pair) const {
    return is_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p)[pair * stride])
                   : static_cast<const float*>(p)[pair * stride];
  }
};

// 2^x of two values, x up to 127, on the FMA units, for part of a tile's exponentials (backward pass): the exponential
// unit takes four values a clock and scheduler.  2^x = 2^n 2^f, n the nearest whole number (from the
// low bits of x + 1.5 2^23) and f in [-1/2, 1/2], where a polynomial of degree 4 with p(0) = 1, fitted to the
// smallest relative error, is off by at most 2.9e-6.  Below -126: 2^-126, which rounds away beside anything.  NaN
// stays NaN (in every step: the factor 2^n is multiplied, not added to the exponent).
__device__ __forceinline__ f32x2 ex2_fma2(f32x2 x) {
  float lo = lo2(x), hi = hi2(x);
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(lo) : "f"(-126.f));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(hi) : "f"(-126.f));
  x = pair2(__float_as_uint(lo), __float_as_uint(hi));
  const f32x2 t = add2(x, dup2(12582912.f));
  const f32x2 f = fma2(add2(t, dup2(-12582912.f)), dup2(-1.f), x);
  f32x2 p = fma2(f, dup2(0x1.39f372p-7f), dup2(0x1.c9fb4ep-5f));
  p = fma2(p, f, dup2(0x1.ec03b6p-3f));
  p = fma2(p, f, dup2(0x1.62e132p-1f));
  p = fma2(p, f, dup2(1.f));
  return mul2(p, pair2(((uint32_t)t << 23) + 0x3f800000u, ((uint32_t)(t >> 32) << 23) + 0x3f800000u));
}
__device__ __forceinline__ f32x2 ex2_mufu2(f32x2 x) {
  return pair2(__float_as_uint(ex2(lo2(x))), __float_as_uint(ex2(hi2(x))));
}

// Eight values as bf16 and what that dropped, and back.  The 32-bit patterns of a value and of its rounding differ by at
// most 2^15 whatever the exponent: the byte is that difference over 2^8, rounded (2^7 at the largest: one less).
// Infinities differ by nothing; whatever the byte of a NaN, the sum of both is one.
__device__ __forceinline__ void diff_split8(const float* x, uint4& hi, uint2& low) {
  uint32_t w[4], c[2];
  int t[8];
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[i / 2]) : "f"(x[i + 1]), "f"(x[i]));
#pragma unroll
    for (int u = 0; u < 2; ++u)
      t[i + u] = min((int)(__float_as_uint(x[i + u]) - (u ? w[i / 2] & 0xffff0000u : w[i / 2] << 16) + 128u), 0x7fff);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)            // the second bytes of four
    c[i] = __byte_perm(__byte_perm(t[4 * i], t[4 * i + 1], 0x0051), __byte_perm(t[4 * i + 2], t[4 * i + 3], 0x0051), 0x5410);
  hi = make_uint4(w[0], w[1], w[2], w[3]);
  low = make_uint2(c[0], c[1]);
}
__device__ __forceinline__ void diff_join8(const uint4& hi, const uint2& low, float* x) {
  const uint32_t w[4] = {hi.x, hi.y, hi.z, hi.w}, c[2] = {low.x, low.y};
#pragma unroll
  for (int i = 0; i < 8; ++i)
    x[i] = __uint_as_float(((i & 1) ? w[i / 2] & 0xffff0000u : w[i / 2] << 16) +
                           (uint32_t)((int)(c[i / 4] << (24 - 8 * (i & 3))) >> 24 << 8));
}

}  // namespace imf
