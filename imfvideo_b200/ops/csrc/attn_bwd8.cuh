// What the dense attention backward wants before its main kernel, made from 8-bit checkpoints in one launch (short
// sequences are all launches): the values of q, k and v in bf16, exact; delta = rowsum(dO .* O) from dO and an O in 8
// bits or bf16; the row constants in the form of either head_dim; and zeros for the dQ additions.
#pragma once
#include "act8.cuh"
#include "common.cuh"
#include "host_util.h"

namespace imf {

// a checkpoint of a (B, L, H, head_dim) tensor: contiguous rows of head_dim codes and 4 step bytes
struct Bwd8Tensor {
  const int8_t* codes;
  const uint8_t* steps;
};
struct Bwd8Packed {
  Bwd8Tensor q, k, v, o;     // v, o: codes null where they come in bf16
};
struct Bwd8Rows {
  const void *q, *k, *v;     // where the values go (v: only where it is packed), contiguous bf16
  const void *o, *d_o;       // bf16, 16-byte aligned rows (o: where it is not packed)
  const float* lse;          // (B, H, L)
  float* dq_acc;             // (B, L, H, head_dim), zeroed here
  int B, L, H, Lp;           // Lp: rows of the constants per (b, h)
  const int64_t *o_strides, *g_strides;
};

// head_dim 64: c1, c2 = bands of 16 bf16 a row that the tensor core adds up, -lse / scale and -delta in three parts and
// zeros (padding rows: the exponent -30000); inv_exp_scale = 1 / (scale * log2 e).  head_dim 128: c1, c2 = lse * log2 e (padding: infinity) and
// delta, one fp32 a row.  head_dim / 8 lanes a row, 8-byte accesses to codes and 16-byte ones besides.
template <int HD, bool V8, bool O8>
__global__ void attn_bwd_prep8_kernel(Bwd8Packed p, __nv_bfloat16* __restrict__ q, __nv_bfloat16* __restrict__ k,
                                      __nv_bfloat16* __restrict__ v, const __nv_bfloat16* __restrict__ o,
                                      const __nv_bfloat16* __restrict__ d_o, const float* __restrict__ lse,
                                      uint32_t* __restrict__ c1, uint32_t* __restrict__ c2, float* __restrict__ dq_acc,
                                      int B, int L, int H, int Lp, int64_t o_sb, int64_t o_sl, int64_t o_sh, int64_t g_sb,
                                      int64_t g_sl, int64_t g_sh, float inv_exp_scale) {
  constexpr int LANES = HD / 8;
  const int lane = threadIdx.x & 31, part = lane % LANES, c0 = part * 8;
  const long u = (((long)blockIdx.x * blockDim.x + threadIdx.x) >> 5) * (32 / LANES) + lane / LANES;
  const bool in = u < (long)B * H * Lp;          // no early exit: the shuffles below need every lane
  int h = 0, l = 0, b = 0;
  if (in) {
    h = (int)(u % H);
    l = (int)((u / H) % Lp);
    b = (int)(u / ((long)H * Lp));
  }
  const bool live = in && l < L;
  float d = 0.f;
  if (live) {
    const int64_t r = ((int64_t)b * L + l) * H + h, at = r * HD + c0;
    const auto value = [&](const Bwd8Tensor& t) {
      return a8_decode8(*reinterpret_cast<const uint2*>(t.codes + at), a8_step2(t.steps[r * 4 + part / 4]));
    };
    const uint4 a = O8 ? value(p.o) : *reinterpret_cast<const uint4*>(o + b * o_sb + (int64_t)l * o_sl + h * o_sh + c0);
    const uint4 g = *reinterpret_cast<const uint4*>(d_o + b * g_sb + (int64_t)l * g_sl + h * g_sh + c0);
    *reinterpret_cast<uint4*>(q + at) = value(p.q);
    *reinterpret_cast<uint4*>(k + at) = value(p.k);
    if (V8) *reinterpret_cast<uint4*>(v + at) = value(p.v);
    const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
    reinterpret_cast<float4*>(dq_acc + at)[0] = zero;
    reinterpret_cast<float4*>(dq_acc + at)[1] = zero;
    const uint32_t aw[4] = {a.x, a.y, a.z, a.w}, gw[4] = {g.x, g.y, g.z, g.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) d += bf16_lo(aw[i]) * bf16_lo(gw[i]) + bf16_hi(aw[i]) * bf16_hi(gw[i]);
  }
#pragma unroll
  for (int off = LANES / 2; off > 0; off >>= 1) d += __shfl_xor_sync(0xffffffffu, d, off);
  if (!in) return;
  const long row = ((long)b * H + h) * Lp + l;
  float x = live ? lse[((long)b * H + h) * L + l] * 1.4426950408889634f : 0.f;
  if (HD == 128) {
    if (part == 0) {
      reinterpret_cast<float*>(c1)[row] = live ? x : INFINITY;
      reinterpret_cast<float*>(c2)[row] = d;
    }
    return;
  }
  // (infinities become what is still finite over the smallest scale, 1e-30)
  x = (live ? fminf(fmaxf(x, -1e8f), 1e8f) : 30000.f) * inv_exp_scale;
  uint32_t wq = 0u, wd = 0u;                     // 16 bf16 = 8 words per row, one per lane of the row
  if (part < 2) {                                // three parts of 8 bits each hold all 24 of a 32-bit number
    const auto word = [part](float v) {
      const float hi = bf16_lo(pack_bf16(v, 0.f)), mid = bf16_lo(pack_bf16(v - hi, 0.f));
      return part == 0 ? pack_bf16(hi, mid) : pack_bf16(v - hi - mid, 0.f);
    };
    wq = word(-x);
    wd = word(-d);
  }
  c1[row * 8 + part] = wq;
  c2[row * 8 + part] = wd;
}

template <int HD>
static int attn_bwd_prep8(const Bwd8Packed& p, const Bwd8Rows& r, void* c1, void* c2, float inv_exp_scale,
                          cudaStream_t st) {
  typedef __nv_bfloat16 bf;
  const bool v8 = p.v.codes != nullptr, o8 = p.o.codes != nullptr;
  auto kern = v8 ? (o8 ? attn_bwd_prep8_kernel<HD, true, true> : attn_bwd_prep8_kernel<HD, true, false>)
                 : (o8 ? attn_bwd_prep8_kernel<HD, false, true> : attn_bwd_prep8_kernel<HD, false, false>);
  const long threads = (long)r.B * r.H * r.Lp * (HD / 8), blocks = (threads + 255) / 256;
  kern<<<(unsigned)blocks, 256, 0, st>>>(
      p, static_cast<bf*>(const_cast<void*>(r.q)), static_cast<bf*>(const_cast<void*>(r.k)),
      static_cast<bf*>(const_cast<void*>(r.v)), static_cast<const bf*>(r.o), static_cast<const bf*>(r.d_o), r.lse,
      static_cast<uint32_t*>(c1), static_cast<uint32_t*>(c2), r.dq_acc, r.B, r.L, r.H, r.Lp, r.o_strides[0],
      r.o_strides[1], r.o_strides[2], r.g_strides[0], r.g_strides[1], r.g_strides[2], inv_exp_scale);
  return cudaGetLastError() == cudaSuccess ? IMF_OK : IMF_ERR_LAUNCH;
}

}  // namespace imf
