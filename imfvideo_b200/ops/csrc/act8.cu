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
  FastDiv upr, n1, n2;                 // units per row; dims
  uint32_t fp32, flat, vec;            // flat: one row stride (s2); vec: 16-byte accesses
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

// UNITS steps per thread, loads first
template <int UNITS>
__global__ void __launch_bounds__(A8_THREADS) store8_kernel(const __grid_constant__ A8Args args) {
  const A8Rec& r = a8_find(args);
  const uint32_t u0 = (blockIdx.x - r.chunk0) * (UNITS * A8_THREADS) + threadIdx.x;
  float v[UNITS][A8_VEC];
  uint32_t row[UNITS], c[UNITS];
#pragma unroll
  for (int k = 0; k < UNITS; ++k) {
    const uint32_t u = u0 + k * A8_THREADS;
    const bool in = u < r.units;
    row[k] = in ? r.upr.div(u) : 0u;
    c[k] = in ? (u - row[k] * r.upr.d) * A8_VEC : 0u;
#pragma unroll
    for (int i = 0; i < A8_VEC; ++i) v[k][i] = 0.f;
    if (!in) continue;
    const int64_t off = a8_row_offset(r, row[k]) + c[k];
    if (r.vec && c[k] + A8_VEC <= r.cols) {
      if (r.fp32) {
        const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(r.x) + off);
        const float4 a = __ldcs(p), b = __ldcs(p + 1);
        v[k][0] = a.x; v[k][1] = a.y; v[k][2] = a.z; v[k][3] = a.w;
        v[k][4] = b.x; v[k][5] = b.y; v[k][6] = b.z; v[k][7] = b.w;
      } else {
        const uint4 w = __ldg(reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(r.x) + off));
        const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[k][2 * i] = __uint_as_float(ww[i] << 16);
          v[k][2 * i + 1] = __uint_as_float(ww[i] & 0xffff0000u);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < A8_VEC; ++i)
        if (c[k] + i < r.cols)
          v[k][i] = r.fp32 ? static_cast<const float*>(r.x)[off + i]
                           : __bfloat162float(static_cast<const __nv_bfloat16*>(r.x)[off + i]);
    }
  }
#pragma unroll
  for (int k = 0; k < UNITS; ++k) {
    uint32_t m = 0u;
#pragma unroll
    for (int i = 0; i < A8_VEC; ++i) m = max(m, __float_as_uint(v[k][i]) & 0x7fffffffu);
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
    if (u0 + k * A8_THREADS >= r.units) continue;
    const uint32_t s = a8_step_of(m);
    uint2 w = make_uint2(0u, 0u);
    if (s < A8_MAX_STEP) {
      const float inv = a8_inv_step(s);
      w = make_uint2(a8_encode4(v[k], inv), a8_encode4(v[k] + 4, inv));
    } else if (s == A8_MAX_STEP) {
      const float inv = a8_inv_step(s);
      w = make_uint2(a8_encode4_top(v[k], inv), a8_encode4_top(v[k] + 4, inv));
    }
    *reinterpret_cast<uint2*>(r.codes + (int64_t)row[k] * r.pitch + c[k]) = w;
    // one byte a group; the last group's thread also clears the bytes that pad the row
    if ((c[k] & (A8_GROUP - 1)) == 0) {
      uint8_t* st = r.steps + (int64_t)row[k] * r.spitch + c[k] / A8_GROUP;
      *st = (uint8_t)s;
      if (c[k] + A8_GROUP == r.pitch)
        for (uint32_t g = r.pitch / A8_GROUP; g < r.spitch; ++g) *++st = 0;
    }
  }
}

template <int UNITS>
__global__ void __launch_bounds__(A8_THREADS) restore8_kernel(const __grid_constant__ A8Args args) {
  const A8Rec& r = a8_find(args);
  const uint32_t u0 = (blockIdx.x - r.chunk0) * (UNITS * A8_THREADS) + threadIdx.x;
  uint2 codes[UNITS];
  uint32_t step[UNITS], row[UNITS], c[UNITS];
#pragma unroll
  for (int k = 0; k < UNITS; ++k) {
    const uint32_t u = u0 + k * A8_THREADS;
    if (u >= r.units) break;
    row[k] = r.upr.div(u);
    c[k] = (u - row[k] * r.upr.d) * A8_VEC;
    codes[k] = __ldg(reinterpret_cast<const uint2*>(r.codes + (int64_t)row[k] * r.pitch + c[k]));
    step[k] = __ldg(r.steps + (int64_t)row[k] * r.spitch + c[k] / A8_GROUP);
  }
#pragma unroll
  for (int k = 0; k < UNITS; ++k) {
    if (u0 + k * A8_THREADS >= r.units) break;
    if (c[k] >= r.cols) continue;
    const uint4 w = a8_decode8(codes[k], a8_step2(step[k]));
    const int64_t off = a8_row_offset(r, row[k]) + c[k];
    const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
    const bool whole = r.vec && c[k] + A8_VEC <= r.cols;
    if (r.fp32) {
      float* dst = static_cast<float*>(r.x) + off;
      float f[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        f[2 * i] = __uint_as_float(ww[i] << 16);
        f[2 * i + 1] = __uint_as_float(ww[i] & 0xffff0000u);
      }
      if (whole) {
        reinterpret_cast<float4*>(dst)[0] = make_float4(f[0], f[1], f[2], f[3]);
        reinterpret_cast<float4*>(dst)[1] = make_float4(f[4], f[5], f[6], f[7]);
      } else {
#pragma unroll
        for (int i = 0; i < A8_VEC; ++i)
          if (c[k] + i < r.cols) dst[i] = f[i];
      }
    } else {
      uint16_t* dst = static_cast<uint16_t*>(r.x) + off;
      if (whole) {
        *reinterpret_cast<uint4*>(dst) = w;
      } else {
#pragma unroll
        for (int i = 0; i < A8_VEC; ++i)
          if (c[k] + i < r.cols) dst[i] = (uint16_t)(ww[i / 2] >> (16 * (i & 1)));
      }
    }
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

// a thread takes four steps where that still gives every SM several blocks, else one
static bool a8_wide(uint64_t units) { return units >= 4ull * A8_THREADS * 148 * 4; }

static int a8_build(const void* recs, int n, A8Args& a, int& per_thread, uint32_t& chunks) {
  if (n <= 0 || n > A8_MAX_RECS) return IMF_ERR_ARG;
  const A8HostRec* h = static_cast<const A8HostRec*>(recs);
  a.n = 0;
  uint64_t all = 0;
  for (int i = 0; i < n; ++i) {
    const int64_t rows = h[i].n0 * h[i].n1 * h[i].n2;
    if (h[i].n0 <= 0 || h[i].n1 <= 0 || h[i].n2 <= 0 || h[i].cols <= 0 || !h[i].x || !h[i].codes || !h[i].steps)
      return IMF_ERR_ARG;
    if (h[i].n0 > 0x7fffffff || h[i].n1 > 0x7fffffff || h[i].n2 > 0x7fffffff || h[i].cols > 0x7fffffc0 ||
        rows > 0x7fffffff)
      return IMF_ERR_TOO_LARGE;
    const uint64_t pitch = ((uint64_t)h[i].cols + A8_GROUP - 1) / A8_GROUP * A8_GROUP;
    const uint64_t units = (uint64_t)rows * (pitch / A8_VEC);
    if (units > 0x7fffffffu) return IMF_ERR_TOO_LARGE;
    if ((reinterpret_cast<uintptr_t>(h[i].codes) & 15u) || (reinterpret_cast<uintptr_t>(h[i].steps) & 3u))
      return IMF_ERR_ARG;
    A8Rec& r = a.r[a.n++];
    const int es = h[i].fp32 ? 4 : 2;
    r.x = h[i].x;
    r.codes = static_cast<int8_t*>(h[i].codes);
    r.steps = static_cast<uint8_t*>(h[i].steps);
    r.s0 = h[i].s0; r.s1 = h[i].s1; r.s2 = h[i].s2;
    r.cols = (uint32_t)h[i].cols;
    r.pitch = (uint32_t)pitch;
    r.spitch = (uint32_t)((pitch / A8_GROUP + 3) / 4 * 4);
    r.units = (uint32_t)units;
    r.upr = FastDiv((uint32_t)(pitch / A8_VEC));
    r.n1 = FastDiv((uint32_t)h[i].n1);
    r.n2 = FastDiv((uint32_t)h[i].n2);
    r.fp32 = h[i].fp32 != 0;
    r.flat = h[i].n0 == 1 && h[i].n1 == 1;
    const int64_t q = 16 / es - 1;
    r.vec = (reinterpret_cast<uintptr_t>(h[i].x) & 15u) == 0 && (r.s2 & q) == 0 &&
            (r.flat || ((r.s0 & q) == 0 && (r.s1 & q) == 0));
    all += units;
  }
  per_thread = a8_wide(all) ? 4 : 1;
  uint64_t c = 0;
  for (int i = 0; i < a.n; ++i) {
    a.r[i].chunk0 = (uint32_t)c;
    c += (a.r[i].units + (uint64_t)per_thread * A8_THREADS - 1) / ((uint64_t)per_thread * A8_THREADS);
  }
  if (c > 0x7fffffffu) return IMF_ERR_TOO_LARGE;
  chunks = (uint32_t)c;
  return IMF_OK;
}

}  // namespace imf

// n (1 .. 16) records {x, codes, steps, n0, n1, n2, s0, s1, s2, cols, fp32} of 8 bytes a field: rows
// n0 x n1 x n2 of `cols` bf16 (fp32) channels at element strides s0, s1, s2 into codes and steps, or back.
extern "C" int imf_store8(const void* recs, int n, void* stream) {
  using namespace imf;
  A8Args a;
  int per = 1;
  uint32_t chunks = 0;
  const int rc = a8_build(recs, n, a, per, chunks);
  if (rc) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (per == 4) store8_kernel<4><<<chunks, A8_THREADS, 0, st>>>(a);
  else store8_kernel<1><<<chunks, A8_THREADS, 0, st>>>(a);
  return cudaGetLastError() == cudaSuccess ? IMF_OK : IMF_ERR_LAUNCH;
}

extern "C" int imf_restore8(const void* recs, int n, void* stream) {
  using namespace imf;
  A8Args a;
  int per = 1;
  uint32_t chunks = 0;
  const int rc = a8_build(recs, n, a, per, chunks);
  if (rc) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (per == 4) restore8_kernel<4><<<chunks, A8_THREADS, 0, st>>>(a);
  else restore8_kernel<1><<<chunks, A8_THREADS, 0, st>>>(a);
  return cudaGetLastError() == cudaSuccess ? IMF_OK : IMF_ERR_LAUNCH;
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
