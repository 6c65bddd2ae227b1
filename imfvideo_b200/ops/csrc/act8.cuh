// The 8-bit form of activations that a training step keeps for its backward pass.
//
// A row is cut into groups of 32 channels.  A group has one step byte s and a signed code for every
// channel; the value is code * 2^(s - 127).  With amax the group's largest magnitude,
//     s = clamp(floor(log2 amax) + 127 - 6 (+ 1 where amax would round to 128 steps), 0, 248)
// so the largest code of a step above the smallest is 64 .. 127 and a value is off by half a step at most, amax / 127.5.
// Groups below 64 steps of 2^-127 have that smallest step, half of which is 2^-128 whatever amax is; above the
// largest bf16, 127.5 * 2^121, which only fp32 has, codes stop at 127, up to a step off.  The step is a power of two
// because the value is then exact in bf16 -- 7 bits of significand -- and a tensor core that is fed the
// codes converted to bf16 multiplies what was stored, with no second rounding.
// s = 255: the group held a NaN or an infinity; all of it reads as NaN.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace imf {

constexpr int A8_GROUP = 32;
constexpr uint32_t A8_BAD = 255u, A8_MAX_STEP = 248u;

// step byte of a group whose largest magnitude has these bits (fp32, sign cleared): adding 2^16
// carries into the exponent from 1.9921875 * 2^e = 127.5 / 64 * 2^e on
__device__ __forceinline__ uint32_t a8_step_of(uint32_t amax_bits) {
  if (amax_bits >= 0x7f800000u) return A8_BAD;
  const int s = (int)((amax_bits + 0x10000u) >> 23) - 6;
  return s < 0 ? 0u : s > (int)A8_MAX_STEP ? A8_MAX_STEP : (uint32_t)s;
}
// 2^(127 - s), s <= 248 (as a pair of bf16: s <= 247)
__device__ __forceinline__ float a8_inv_step(uint32_t s) { return __uint_as_float((254u - s) << 23); }
__device__ __forceinline__ __nv_bfloat162 a8_inv_step2(uint32_t s) {
  const uint32_t w = (254u - s) * 0x00800080u;
  return *reinterpret_cast<const __nv_bfloat162*>(&w);
}

// four codes of v[0..3] as one word.  Adding 1.5 * 2^23 leaves the nearest whole number (ties to even)
// in the low bits; the product with a power of two is exact (or below half a step), so the one rounding
// of the fma is that of the code.
__device__ __forceinline__ uint32_t a8_encode4(const float* v, float inv) {
  constexpr float MAGIC = 12582912.f;
  const uint32_t a = __float_as_uint(fmaf(v[0], inv, MAGIC)), b = __float_as_uint(fmaf(v[1], inv, MAGIC));
  const uint32_t c = __float_as_uint(fmaf(v[2], inv, MAGIC)), d = __float_as_uint(fmaf(v[3], inv, MAGIC));
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}
// the same at the largest step, where 127.5 and more would round to 128
__device__ __forceinline__ uint32_t a8_encode4_top(const float* v, float inv) {
  float c[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) c[i] = fminf(fmaxf(v[i] * inv, -127.f), 127.f);
  return a8_encode4(c, 1.f);
}

// four codes of the bf16 pairs a and b, whose magnitudes are ma and mb, times 2^(127 - s) (in both halves of inv), below
// the largest step.  128 + |x| has a spacing of one in bf16, so the one rounding of the fma is that of the code, whose
// magnitude is the result's low byte; negative codes are then ~m + 1, a byte at a time.
__device__ __forceinline__ uint32_t a8_encode4(uint32_t a, uint32_t b, uint32_t ma, uint32_t mb, __nv_bfloat162 inv) {
  const uint32_t one28 = 0x43004300u;
  const auto mag = [&](uint32_t m) {
    const __nv_bfloat162 r = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&m), inv,
                                     *reinterpret_cast<const __nv_bfloat162*>(&one28));
    return *reinterpret_cast<const uint32_t*>(&r);
  };
  uint32_t neg;                        // 0xff where the sign is set: prmt repeats the top bit of bytes 1, 3 of both
  asm("prmt.b32 %0, %1, %2, 0xfdb9;" : "=r"(neg) : "r"(a), "r"(b));
  const uint32_t c = __byte_perm(mag(ma), mag(mb), 0x6420) ^ neg;
  return ((c & 0x7f7f7f7fu) + (neg & 0x01010101u)) ^ (c & 0x80808080u);
}

// the step in both halves, as bf16: the byte is the exponent.  2^-127 is half the smallest normal number
// and 255 a NaN, both of which the upper mantissa bit makes
__device__ __forceinline__ __nv_bfloat162 a8_step2(uint32_t s) {
  uint32_t w = s * 0x00800080u;
  if (s - 1u >= 254u) w |= 0x00400040u;
  return *reinterpret_cast<const __nv_bfloat162*>(&w);
}
// two codes (low bytes of the halves of x) times the step, exact.  The low seven bits of a code are the
// mantissa of 128 + c, its sign bit the exponent step from 128 to 256: c = (128 + low) - (128 or 256).
__device__ __forceinline__ uint32_t a8_decode2(uint32_t x, __nv_bfloat162 step) {
  const uint32_t lo = (x & 0x007f007fu) | 0x43004300u, hi = (x & 0x00800080u) | 0x43004300u;
  const __nv_bfloat162 v = __hmul2(__hsub2(*reinterpret_cast<const __nv_bfloat162*>(&lo),
                                           *reinterpret_cast<const __nv_bfloat162*>(&hi)), step);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint2 a8_decode4(uint32_t codes, __nv_bfloat162 step) {
  return make_uint2(a8_decode2(__byte_perm(codes, 0u, 0x4140), step),
                    a8_decode2(__byte_perm(codes, 0u, 0x4342), step));
}
__device__ __forceinline__ uint4 a8_decode8(uint2 codes, __nv_bfloat162 step) {
  const uint2 a = a8_decode4(codes.x, step), b = a8_decode4(codes.y, step);
  return make_uint4(a.x, a.y, b.x, b.y);
}

// q = n / d for n < 2^31 by one multiplication: with l = ceil(log2 d), m = floor(2^32 (2^l - d) / d) + 1
// gives q = (mulhi(n, m) + n) >> l (the round-up method of Granlund and Montgomery, 1994).
struct FastDiv {
  uint32_t m, l, d;
  FastDiv() = default;
  explicit FastDiv(uint32_t div) : d(div) {
    l = 0;
    while ((1ull << l) < div) ++l;
    m = (uint32_t)((((1ull << l) - div) << 32) / div + 1);
  }
  __device__ __forceinline__ uint32_t div(uint32_t n) const { return (__umulhi(n, m) + n) >> l; }
};

}  // namespace imf
