// Activations into 8-bit checkpoints and back, and the gated activation's reverse mode from one
// (format: act8.cuh).
//
// imf_store8 / imf_restore8 take several tensors at once: a transformer block keeps a dozen, and a
// launch for each would cost more than the data of a short clip.  A thread owns eight channels, four
// neighbouring threads a group: 16-byte loads and stores of the 16-bit side, 8-byte ones of the codes,
// every warp access a contiguous run.  The group's maximum takes two shuffles.
#include "act8.cuh"
#include "host_util.h"
#include "situ.cuh"

namespace imf {

constexpr int A8_THREADS = 256;
constexpr int A8_MAX_RECS = 16;
constexpr int A8_VEC = 8;              // channels per thread and step

// One tensor: rows = n0 * n1 * n2 at (i0 * s0 + i1 * s1 + i2 * s2), `cols` channels of stride 1; codes
// [rows][pitch], pitch = cols rounded up to 32; steps [rows][spitch], spitch = groups rounded up to 4.
struct A8Rec {
  void* x;                             // bf16 or fp32
  int8_t* codes;
  uint8_t* steps;
  int64_t s0, s1, s2;
  uint32_t cols, pitch, spitch;
  uint32_t units, chunk0;              // units of eight channels; first chunk of this tensor
  FastDiv upr, gpr, n1, n2;            // units and groups per row; dims
  uint32_t fp32, flat, plain;          // flat: one row stride (s2); plain: no gaps, whole words of steps
};
struct A8Args {
  A8Rec r[A8_MAX_RECS];
  int n;
};

__device__ __forceinline__ const A8Rec& a8_find(const A8Args& a) {
  int i = 0;
  while (i + 1 < a.n && blockIdx.x >= a.r[i + 1].chunk0) ++i;
  return a.r[i];
}
__device__ __forceinline__ int64_t a8_row_offset(const A8Rec& r, uint32_t row) {
  if (r.flat) return (int64_t)row * r.s2;
  const uint32_t t = r.n2.div(row), i2 = row - t * r.n2.d, i0 = r.n1.div(t), i1 = t - i0 * r.n1.d;
  return (int64_t)i0 * r.s0 + (int64_t)i1 * r.s1 + (int64_t)i2 * r.s2;
}
__device__ __forceinline__ uint32_t abs2(uint32_t w) { return w & 0x7fff7fffu; }
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {     // of both halves
  uint32_t r;
  asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ void halves(uint32_t w, float* v) {
  v[0] = __uint_as_float(w << 16);
  v[1] = __uint_as_float(w & 0xffff0000u);
}

// A chunk is UNITS * 256 units of eight channels.  A tensor whose rows are 16-byte aligned is read and
// written by whole units (a thread owns one, loads first); any other one, in a launch of its own, by the channel:
// a warp takes eight groups at a time, a lane a channel of each, so that its accesses are contiguous whatever the
// alignment.
//
// PLAIN: the tensor has no gaps and whole words of steps (a multiple of 128 channels), so unit u is 16 (32) bytes at
// 16 u, its codes are at 8 u and its step at u / 4: no division, one address computation each.  Storing is bound by the
// instructions: 574 M channels in 13 tensors 313 us with two units a thread, 330 with four, 318 with codes rounded in fp32,
// 356 with divisions besides; a copy's rate would be 282.  Restoring is at it: 270 us with four, 305 with two.
template <int UNITS, bool FP32, bool PLAIN>
__device__ __forceinline__ void store_units(const A8Rec& r, uint32_t u0) {
  constexpr int ES = FP32 ? 4 : 2;
  const char* const x = static_cast<const char*>(r.x);
  int8_t* const codes = r.codes;
  uint8_t* const steps = r.steps;
  const int64_t ld = r.s2 * ES;
  const uint32_t spitch = r.spitch, units = r.units, cols = r.cols;
  const FastDiv upr = r.upr;
  const uint32_t gpr = r.gpr.d;
  const bool words = PLAIN || gpr % 4 == 0 || gpr <= 2;
  uint4 w[UNITS][FP32 ? 2 : 1];
  uint32_t row[UNITS], c[UNITS];
#pragma unroll
  for (int k = 0; k < UNITS; ++k) {
    const uint32_t u = u0 + k * A8_THREADS;
    bool in = u < units;
    const char* src;
    if (PLAIN) {
      src = x + (uint64_t)u * (A8_VEC * ES);
    } else {
      row[k] = upr.div(u);
      c[k] = (u - row[k] * upr.d) * A8_VEC;
      in = in && c[k] < cols;
      src = x + row[k] * ld + c[k] * ES;
    }
#pragma unroll
    for (int h = 0; h < (FP32 ? 2 : 1); ++h)
      w[k][h] = in ? __ldcs(reinterpret_cast<const uint4*>(src) + h) : make_uint4(0u, 0u, 0u, 0u);
  }
#pragma unroll
  for (int k = 0; k < UNITS; ++k) {
    float v[A8_VEC];
    uint32_t m, mag[4];                // bits of the largest magnitude, as fp32; bf16: the pairs' magnitudes
    if (FP32) {
      const uint4 a = w[k][0], b = w[k][FP32 ? 1 : 0];
      const uint32_t ww[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
      m = 0u;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        m = max(m, ww[i] & 0x7fffffffu);
        v[i] = __uint_as_float(ww[i]);
      }
      m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
      m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
    } else {
      const uint4 a = w[k][0];
      mag[0] = abs2(a.x); mag[1] = abs2(a.y); mag[2] = abs2(a.z); mag[3] = abs2(a.w);
      uint32_t h = max2(max2(mag[0], mag[1]), max2(mag[2], mag[3]));
      h = max2(h, __shfl_xor_sync(0xffffffffu, h, 1));
      h = max2(h, __shfl_xor_sync(0xffffffffu, h, 2));
      m = max(h << 16, h & 0xffff0000u);
    }
    const uint32_t s = a8_step_of(m);
    // the steps of four groups are one word, which the first of them writes, where a warp holds whole words (by
    // the byte, a d=1024 block's thirteen tensors, three of them with rows of two groups, took 580 us instead of 358)
    uint32_t word = s;
    if (words) {                       // the same for the whole launch's tensor: every lane shuffles
      const uint32_t s1 = __shfl_down_sync(0xffffffffu, s, 4), s2 = __shfl_down_sync(0xffffffffu, s, 8),
                     s3 = __shfl_down_sync(0xffffffffu, s, 12);
      if (PLAIN || gpr > 1) word |= s1 << 8;
      if (PLAIN || gpr > 2) word |= s2 << 16 | s3 << 24;
    }
    const uint32_t u = u0 + k * A8_THREADS;
    if (u < units) {
      uint2 out;
      if (s < A8_MAX_STEP) {
        if (FP32) {
          const float inv = a8_inv_step(s);
          out = make_uint2(a8_encode4(v, inv), a8_encode4(v + 4, inv));
        } else {
          const uint4 a = w[k][0];
          const __nv_bfloat162 inv = a8_inv_step2(s);
          out = make_uint2(a8_encode4(a.x, a.y, mag[0], mag[1], inv), a8_encode4(a.z, a.w, mag[2], mag[3], inv));
        }
      } else if (s == A8_MAX_STEP) {
        const float inv = a8_inv_step(s);
        if (!FP32) {
          const uint4 a = w[k][0];
          halves(a.x, v); halves(a.y, v + 2); halves(a.z, v + 4); halves(a.w, v + 6);
        }
        out = make_uint2(a8_encode4_top(v, inv), a8_encode4_top(v + 4, inv));
      } else {
        out = make_uint2(0u, 0u);
      }
      *reinterpret_cast<uint2*>(codes + (uint64_t)u * A8_VEC) = out;
      if (PLAIN) {
        if (u % 16 == 0) *reinterpret_cast<uint32_t*>(steps + u / 4) = word;
      } else {
        const uint32_t g = c[k] / A8_GROUP;
        uint8_t* st = steps + (int64_t)row[k] * spitch + g;
        if (words) {
          if (c[k] % (4 * A8_GROUP) == 0) *reinterpret_cast<uint32_t*>(st) = word;
        } else if (c[k] % A8_GROUP == 0) {
          *st = (uint8_t)s;
          if (g + 1 == gpr)            // the last group's thread also clears the bytes that pad the row
            for (uint32_t j = gpr; j < spitch; ++j) *++st = 0;
        }
      }
    }
  }
}

template <int UNITS, bool FP32>
__device__ __forceinline__ void store_channels(const A8Rec& r, uint32_t chunk) {
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t groups = r.units / 4, gpr = r.gpr.d, cols = r.cols, pitch = r.pitch, spitch = r.spitch;
  int8_t* const codes = r.codes;
  uint8_t* const steps = r.steps;
#pragma unroll 1
  for (int k = 0; k < UNITS; ++k) {
    const uint32_t g0 = (chunk * UNITS + k) * (A8_THREADS / 4) + warp * 8;
    if (g0 >= groups) return;
    const uint32_t row0 = r.gpr.div(g0), c0 = g0 - row0 * gpr;
    uint32_t bits[8], row = row0, g = c0;
    int64_t off = a8_row_offset(r, row) + lane;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t c = g * A8_GROUP + lane;
      bits[j] = 0u;
      if (g0 + j < groups && c < cols)
        bits[j] = FP32 ? __ldg(static_cast<const uint32_t*>(r.x) + off + g * A8_GROUP)
                       : (uint32_t)__ldg(static_cast<const uint16_t*>(r.x) + off + g * A8_GROUP) << 16;
      if (++g == gpr) {
        g = 0;
        off = a8_row_offset(r, ++row) + lane;
      }
    }
    row = row0;
    g = c0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t s = a8_step_of(__reduce_max_sync(0xffffffffu, bits[j] & 0x7fffffffu));
      if (g0 + j >= groups) break;
      int code = 0;
      if (s < A8_MAX_STEP)
        code = (int)__float_as_uint(fmaf(__uint_as_float(bits[j]), a8_inv_step(s), 12582912.f));     // its low byte
      else if (s == A8_MAX_STEP)
        code = __float2int_rn(fminf(fmaxf(__uint_as_float(bits[j]) * a8_inv_step(s), -127.f), 127.f));
      codes[(int64_t)row * pitch + g * A8_GROUP + lane] = (int8_t)code;
      uint8_t* st = steps + (int64_t)row * spitch + g;
      if (lane == 0) *st = (uint8_t)s;
      if (++g == gpr) {
        if (lane > 0 && gpr - 1 + lane < spitch) st[lane] = 0;                                       // pads the row
        g = 0;
        ++row;
      }
    }
  }
}

template <int UNITS, bool VEC>
__global__ void __launch_bounds__(A8_THREADS) store8_kernel(const __grid_constant__ A8Args args) {
  const A8Rec& r = a8_find(args);
  const uint32_t chunk = blockIdx.x - r.chunk0, u0 = chunk * (UNITS * A8_THREADS) + threadIdx.x;
  if (!VEC) {
    if (r.fp32) store_channels<UNITS, true>(r, chunk);
    else store_channels<UNITS, false>(r, chunk);
  } else if (r.plain) {
    if (r.fp32) store_units<UNITS, true, true>(r, u0);
    else store_units<UNITS, false, true>(r, u0);
  } else {
    if (r.fp32) store_units<UNITS, true, false>(r, u0);
    else store_units<UNITS, false, false>(r, u0);
  }
}

template <int UNITS, bool FP32, bool PLAIN>
__device__ __forceinline__ void restore_units(const A8Rec& r, uint32_t u0) {
  constexpr int ES = FP32 ? 4 : 2;
  char* const x = static_cast<char*>(r.x);
  const int8_t* const src = r.codes;
  const uint8_t* const sts = r.steps;
  const int64_t ld = r.s2 * ES;
  const uint32_t spitch = r.spitch, units = r.units, cols = r.cols;
  const FastDiv upr = r.upr;
  uint2 codes[UNITS];
  uint32_t step[UNITS], row[UNITS], c[UNITS];
#pragma unroll
  for (int k = 0; k < UNITS; ++k) {
    const uint32_t u = u0 + k * A8_THREADS;
    bool in = u < units;
    if (!PLAIN) {
      row[k] = upr.div(u);
      c[k] = (u - row[k] * upr.d) * A8_VEC;
      if (!in) c[k] = cols;                            // nothing to do
      in = c[k] < cols;
    }
    if (in) {
      codes[k] = __ldcs(reinterpret_cast<const uint2*>(src + (uint64_t)u * A8_VEC));
      step[k] = __ldg(PLAIN ? sts + u / 4 : sts + (int64_t)row[k] * spitch + c[k] / A8_GROUP);
    }
  }
#pragma unroll
  for (int k = 0; k < UNITS; ++k) {
    const uint32_t u = u0 + k * A8_THREADS;
    if (PLAIN ? u >= units : c[k] >= cols) continue;
    const uint4 w = a8_decode8(codes[k], a8_step2(step[k]));
    char* dst = PLAIN ? x + (uint64_t)u * (A8_VEC * ES) : x + row[k] * ld + c[k] * ES;
    if (FP32) {
      float v[8];
      halves(w.x, v); halves(w.y, v + 2); halves(w.z, v + 4); halves(w.w, v + 6);
      reinterpret_cast<float4*>(dst)[0] = make_float4(v[0], v[1], v[2], v[3]);
      reinterpret_cast<float4*>(dst)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      *reinterpret_cast<uint4*>(dst) = w;
    }
  }
}

template <int UNITS, bool FP32>
__device__ __forceinline__ void restore_channels(const A8Rec& r, uint32_t chunk) {
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t groups = r.units / 4, gpr = r.gpr.d, cols = r.cols, pitch = r.pitch, spitch = r.spitch;
#pragma unroll 1
  for (int k = 0; k < UNITS; ++k) {
    const uint32_t g0 = (chunk * UNITS + k) * (A8_THREADS / 4) + warp * 8;
    if (g0 >= groups) return;
    const uint32_t row0 = r.gpr.div(g0), c0 = g0 - row0 * gpr;
    uint32_t code[8], step[8], row = row0, g = c0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (g0 + j < groups) {                           // codes are there up to the pitch
        code[j] = (uint8_t)__ldg(r.codes + (int64_t)row * pitch + g * A8_GROUP + lane);
        step[j] = __ldg(r.steps + (int64_t)row * spitch + g);
      }
      if (++g == gpr) {
        g = 0;
        ++row;
      }
    }
    row = row0;
    g = c0;
    int64_t off = a8_row_offset(r, row) + lane;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (g0 + j < groups && g * A8_GROUP + lane < cols) {
        const uint32_t w = a8_decode2(code[j], a8_step2(step[j]));
        if (FP32) static_cast<float*>(r.x)[off + g * A8_GROUP] = __uint_as_float(w << 16);
        else static_cast<uint16_t*>(r.x)[off + g * A8_GROUP] = (uint16_t)w;
      }
      if (++g == gpr) {
        g = 0;
        off = a8_row_offset(r, ++row) + lane;
      }
    }
  }
}

template <int UNITS, bool VEC>
__global__ void __launch_bounds__(A8_THREADS) restore8_kernel(const __grid_constant__ A8Args args) {
  const A8Rec& r = a8_find(args);
  const uint32_t chunk = blockIdx.x - r.chunk0, u0 = chunk * (UNITS * A8_THREADS) + threadIdx.x;
  if (!VEC) {
    if (r.fp32) restore_channels<UNITS, true>(r, chunk);
    else restore_channels<UNITS, false>(r, chunk);
  } else if (r.plain) {
    if (r.fp32) restore_units<UNITS, true, true>(r, u0);
    else restore_units<UNITS, false, true>(r, u0);
  } else {
    if (r.fp32) restore_units<UNITS, true, false>(r, u0);
    else restore_units<UNITS, false, false>(r, u0);
  }
}

// Reverse mode of y = situ(gate) up' from the checkpoint of [gate | up] (width 2F), and y itself, which the
// next weight gradient multiplies: one pass over 8-bit input instead of restoring it (write and
// read back 4 bytes a pair), the bf16 backward and a second forward.
struct Situ8Args {
  const int8_t* codes;
  const uint8_t* steps;
  const __nv_bfloat16* gout;
  __nv_bfloat16 *g_gu, *act;
  uint32_t pitch, spitch, F, units;
  int64_t ld_gout, ld_ggu, ld_act;
  FastDiv upr;
  float beta, lbeta;
  int has_lbeta;
};

template <int VEC, int UNITS>
__global__ void __launch_bounds__(A8_THREADS) situ_bwd8_kernel(const __grid_constant__ Situ8Args a) {
  const float inv_beta = 1.f / a.beta, inv_lbeta = a.has_lbeta ? 1.f / a.lbeta : 0.f;
  const uint32_t u0 = blockIdx.x * (UNITS * A8_THREADS) + threadIdx.x;
  uint2 cg[UNITS], cu[UNITS];
  uint4 go[UNITS];
  uint32_t sg[UNITS], su[UNITS], row[UNITS], c[UNITS];
#pragma unroll
  for (int k = 0; k < UNITS; ++k) {
    const uint32_t u = u0 + k * A8_THREADS;
    if (u >= a.units) break;
    row[k] = a.upr.div(u);
    c[k] = (u - row[k] * a.upr.d) * VEC;
    const int8_t* pc = a.codes + (int64_t)row[k] * a.pitch;
    const uint8_t* ps = a.steps + (int64_t)row[k] * a.spitch;
    const uint32_t cup = a.F + c[k];
    sg[k] = __ldg(ps + c[k] / A8_GROUP);
    su[k] = __ldg(ps + cup / A8_GROUP);
    const __nv_bfloat16* pg = a.gout + (int64_t)row[k] * a.ld_gout + c[k];
    if constexpr (VEC == 8) {
      cg[k] = __ldg(reinterpret_cast<const uint2*>(pc + c[k]));
      cu[k] = __ldg(reinterpret_cast<const uint2*>(pc + cup));
      go[k] = __ldg(reinterpret_cast<const uint4*>(pg));
    } else {
      cg[k] = make_uint2((uint8_t)pc[c[k]], 0u);
      cu[k] = make_uint2((uint8_t)pc[cup], 0u);
      go[k] = make_uint4(*reinterpret_cast<const uint16_t*>(pg), 0u, 0u, 0u);
    }
  }
#pragma unroll
  for (int k = 0; k < UNITS; ++k) {
    if (u0 + k * A8_THREADS >= a.units) break;
    const uint4 gw = a8_decode8(cg[k], a8_step2(sg[k])), uw = a8_decode8(cu[k], a8_step2(su[k]));
    const uint32_t g_[4] = {gw.x, gw.y, gw.z, gw.w}, u_[4] = {uw.x, uw.y, uw.z, uw.w};
    const uint32_t o_[4] = {go[k].x, go[k].y, go[k].z, go[k].w};
    uint32_t rg[4], ru[4], ry[4];
#pragma unroll
    for (int i = 0; i < (VEC + 1) / 2; ++i) {
      float gg[2], gu[2], y[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const auto half = [e](uint32_t w) { return __uint_as_float(e ? w & 0xffff0000u : w << 16); };
        float av, dav, up, dup;
        situ1(half(g_[i]), half(u_[i]), a.beta, inv_beta, a.lbeta, inv_lbeta, a.has_lbeta, av, dav, up, dup);
        const float gout = half(o_[i]);
        gg[e] = gout * dav * up;
        gu[e] = gout * av * dup;
        y[e] = av * up;
      }
      const __nv_bfloat162 a2 = __floats2bfloat162_rn(gg[0], gg[1]), b2 = __floats2bfloat162_rn(gu[0], gu[1]),
                           y2 = __floats2bfloat162_rn(y[0], y[1]);
      rg[i] = *reinterpret_cast<const uint32_t*>(&a2);
      ru[i] = *reinterpret_cast<const uint32_t*>(&b2);
      ry[i] = *reinterpret_cast<const uint32_t*>(&y2);
    }
    __nv_bfloat16* dg = a.g_gu + (int64_t)row[k] * a.ld_ggu + c[k];
    __nv_bfloat16* dy = a.act + (int64_t)row[k] * a.ld_act + c[k];
    if constexpr (VEC == 8) {
      *reinterpret_cast<uint4*>(dg) = make_uint4(rg[0], rg[1], rg[2], rg[3]);
      *reinterpret_cast<uint4*>(dg + a.F) = make_uint4(ru[0], ru[1], ru[2], ru[3]);
      *reinterpret_cast<uint4*>(dy) = make_uint4(ry[0], ry[1], ry[2], ry[3]);
    } else {
      *reinterpret_cast<uint16_t*>(dg) = (uint16_t)rg[0];
      *reinterpret_cast<uint16_t*>(dg + a.F) = (uint16_t)ru[0];
      *reinterpret_cast<uint16_t*>(dy) = (uint16_t)ry[0];
    }
  }
}

// what the host passes for one tensor (all 8-byte fields)
struct A8HostRec {
  void* x;
  void* codes;
  void* steps;
  int64_t n0, n1, n2, s0, s1, s2, cols, fp32;
};

// Checks the records and sorts them into a[0] (rows of aligned units) and a[1] (the others).  A thread takes `many`
// steps where that still gives every SM several blocks, else one.
static int a8_build(const void* recs, int n, A8Args* a, int many, int& per_thread, uint32_t* chunks) {
  if (n <= 0 || n > A8_MAX_RECS) return IMF_ERR_ARG;
  const A8HostRec* h = static_cast<const A8HostRec*>(recs);
  a[0].n = a[1].n = 0;
  uint64_t all = 0;
  for (int i = 0; i < n; ++i) {
    if (h[i].n0 <= 0 || h[i].n1 <= 0 || h[i].n2 <= 0 || h[i].cols <= 0 || !h[i].x || !h[i].codes || !h[i].steps)
      return IMF_ERR_ARG;
    if (h[i].n0 > 0x7fffffff || h[i].n1 > 0x7fffffff || h[i].n2 > 0x7fffffff || h[i].cols > 0x7fffffc0 ||
        h[i].n0 * h[i].n1 > 0x7fffffff || h[i].n0 * h[i].n1 * h[i].n2 > 0x7fffffff)
      return IMF_ERR_TOO_LARGE;
    const int64_t rows = h[i].n0 * h[i].n1 * h[i].n2;
    const uint64_t pitch = ((uint64_t)h[i].cols + A8_GROUP - 1) / A8_GROUP * A8_GROUP;
    const uint64_t units = (uint64_t)rows * (pitch / A8_VEC);
    if (units > 0x7ffffff0u) return IMF_ERR_TOO_LARGE;
    if ((reinterpret_cast<uintptr_t>(h[i].codes) & 15u) || (reinterpret_cast<uintptr_t>(h[i].steps) & 3u))
      return IMF_ERR_ARG;
    const int es = h[i].fp32 ? 4 : 2;
    const bool flat = h[i].n0 == 1 && h[i].n1 == 1;
    const bool vec = flat && (reinterpret_cast<uintptr_t>(h[i].x) & 15u) == 0 && (h[i].s2 * es & 15) == 0 &&
                     h[i].cols % A8_VEC == 0;
    A8Args& t = a[vec ? 0 : 1];
    A8Rec& r = t.r[t.n++];
    r.x = h[i].x;
    r.codes = static_cast<int8_t*>(h[i].codes);
    r.steps = static_cast<uint8_t*>(h[i].steps);
    r.s0 = h[i].s0; r.s1 = h[i].s1; r.s2 = h[i].s2;
    r.cols = (uint32_t)h[i].cols;
    r.pitch = (uint32_t)pitch;
    r.spitch = (uint32_t)((pitch / A8_GROUP + 3) / 4 * 4);
    r.units = (uint32_t)units;
    r.upr = FastDiv((uint32_t)(pitch / A8_VEC));
    r.gpr = FastDiv((uint32_t)(pitch / A8_GROUP));
    r.n1 = FastDiv((uint32_t)h[i].n1);
    r.n2 = FastDiv((uint32_t)h[i].n2);
    r.fp32 = h[i].fp32 != 0;
    r.flat = flat;
    r.plain = flat && h[i].s2 == h[i].cols && h[i].cols % (4 * A8_GROUP) == 0;
    all += units;
  }
  per_thread = all >= 4ull * A8_THREADS * 148 * many ? many : 1;
  for (int k = 0; k < 2; ++k) {
    uint64_t c = 0;
    for (int i = 0; i < a[k].n; ++i) {
      a[k].r[i].chunk0 = (uint32_t)c;
      c += (a[k].r[i].units + (uint64_t)per_thread * A8_THREADS - 1) / ((uint64_t)per_thread * A8_THREADS);
    }
    if (c > 0x7fffffffu) return IMF_ERR_TOO_LARGE;
    chunks[k] = (uint32_t)c;
  }
  return IMF_OK;
}

typedef void (*A8Kernel)(const A8Args);
// kernels: units by `many` and by one a thread, channels likewise
static int a8_run(const void* recs, int n, void* stream, int many, const A8Kernel (&kernels)[2][2]) {
  A8Args a[2];
  int per = 1;
  uint32_t chunks[2] = {0, 0};
  const int rc = a8_build(recs, n, a, many, per, chunks);
  if (rc) return rc;
  for (int k = 0; k < 2; ++k) {
    if (!chunks[k]) continue;
    kernels[k][per == 1]<<<chunks[k], A8_THREADS, 0, static_cast<cudaStream_t>(stream)>>>(a[k]);
    if (cudaGetLastError() != cudaSuccess) return IMF_ERR_LAUNCH;
  }
  return IMF_OK;
}

}  // namespace imf

// n (1 .. 16) records {x, codes, steps, n0, n1, n2, s0, s1, s2, cols, fp32} of 8 bytes a field: rows
// n0 x n1 x n2 of `cols` bf16 (fp32) channels at element strides s0, s1, s2 into codes and steps, or back.
extern "C" int imf_store8(const void* recs, int n, void* stream) {
  using namespace imf;
  static const A8Kernel kernels[2][2] = {{store8_kernel<2, true>, store8_kernel<1, true>},
                                         {store8_kernel<2, false>, store8_kernel<1, false>}};
  return a8_run(recs, n, stream, 2, kernels);
}

extern "C" int imf_restore8(const void* recs, int n, void* stream) {
  using namespace imf;
  static const A8Kernel kernels[2][2] = {{restore8_kernel<4, true>, restore8_kernel<1, true>},
                                         {restore8_kernel<4, false>, restore8_kernel<1, false>}};
  return a8_run(recs, n, stream, 4, kernels);
}

// codes / steps: checkpoint of [gate | up], rows x 2F; gout rows x F, g_gu rows x 2F, act rows x F (bf16, row
// pitches in elements)
extern "C" int imf_situ_bwd8(const void* codes, const void* steps, const void* gout, void* g_gu, void* act,
                             long rows, int F, int64_t ld_gout, int64_t ld_ggu, int64_t ld_act, float beta,
                             float lbeta, int has_lbeta, void* stream) {
  using namespace imf;
  if (rows <= 0 || F <= 0 || !codes || !steps || !gout || !g_gu || !act) return IMF_ERR_ARG;
  if (rows > 0x7fffffffL || F > 0x3fffffe0) return IMF_ERR_TOO_LARGE;
  if ((reinterpret_cast<uintptr_t>(codes) & 15u) || (reinterpret_cast<uintptr_t>(steps) & 3u)) return IMF_ERR_ARG;
  Situ8Args a;
  a.codes = static_cast<const int8_t*>(codes);
  a.steps = static_cast<const uint8_t*>(steps);
  a.gout = static_cast<const __nv_bfloat16*>(gout);
  a.g_gu = static_cast<__nv_bfloat16*>(g_gu);
  a.act = static_cast<__nv_bfloat16*>(act);
  a.pitch = (uint32_t)((2 * F + A8_GROUP - 1) / A8_GROUP * A8_GROUP);
  a.spitch = (a.pitch / A8_GROUP + 3) / 4 * 4;
  a.F = (uint32_t)F;
  a.ld_gout = ld_gout; a.ld_ggu = ld_ggu; a.ld_act = ld_act;
  a.beta = beta; a.lbeta = lbeta; a.has_lbeta = has_lbeta;
  auto al16 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
  const bool v8 = F % 8 == 0 && ld_gout % 8 == 0 && ld_ggu % 8 == 0 && ld_act % 8 == 0 && al16(gout) &&
                  al16(g_gu) && al16(act);
  const uint64_t units = (uint64_t)rows * (v8 ? F / 8 : F);
  if (units > 0x7fffffffu) return IMF_ERR_TOO_LARGE;
  a.units = (uint32_t)units;
  a.upr = FastDiv((uint32_t)(v8 ? F / 8 : F));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool wide = units >= 2ull * A8_THREADS * 148 * 4;
  const uint64_t per = (uint64_t)A8_THREADS * (wide ? 2 : 1);
  const unsigned blocks = (unsigned)((units + per - 1) / per);
  if (v8 && wide) situ_bwd8_kernel<8, 2><<<blocks, A8_THREADS, 0, st>>>(a);
  else if (v8) situ_bwd8_kernel<8, 1><<<blocks, A8_THREADS, 0, st>>>(a);
  else if (wide) situ_bwd8_kernel<1, 2><<<blocks, A8_THREADS, 0, st>>>(a);
  else situ_bwd8_kernel<1, 1><<<blocks, A8_THREADS, 0, st>>>(a);
  return cudaGetLastError() == cudaSuccess ? IMF_OK : IMF_ERR_LAUNCH;
}
