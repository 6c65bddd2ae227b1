// Residual update whose branch is normed before it is added, with the norm that the next branch begins
// with, its forward-mode tangent and its gradient:
//
//   yh = y iy, iy = rsqrt(mean y^2 + eps);   x = r .* res + gate .* post .* yh      (fp32)
//   xh = x ix, ix = rsqrt(mean x^2 + eps);   n = pre .* xh                          (y's type)
//   dx = r .* dres + gate .* post .* iy (dy - yh mean(yh dy)),  dn = pre .* ix (dx - xh mean(xh dx))
//   a = pre .* gn,  g = gx + ix (a - xh mean(a xh));   g_res = r .* g,  b = gate .* post .* g,
//   g_y = iy (b - yh mean(b yh));   column sums  g_pre: gn xh,  g_r: g res,  g_gate: post g yh,  g_post: gate g yh
//
// Memory-bound: every row is read once and held in registers through its two norms.  A row belongs to W
// warps, a lane to 8 adjacent channels of each of NV chunks (16-byte accesses to bf16), W chosen so
// that NV is 2 from 257 to 4,096 channels: more chunks a lane leave too few warps in flight beside the
// column sums of the backward pass (48 registers).  The backward pass makes x again from res and y, of
// which it needs both anyway, instead of reading it.  Row sums add in a fixed order; column sums go through
// one partial row a CTA, added up in a fixed order by imf_colsum.
#include "host_util.h"
#include "rowops_common.cuh"

namespace imf {
namespace pn {

struct Args {
  const float *res, *dres;               // null: the stream begins here / stands still
  const void *y, *dy;
  const float *post, *gate, *r, *pre;    // r null: 1; pre null: no second norm
  float *x, *dx;
  void *n, *dn;
  const float* gx;                       // null: no gradient of x
  const void* gn;
  float* g_res;                          // null: not wanted
  void* g_y;
  float* partial;                        // [grid][4][D]: pre, r, gate, post
  int rows, D;
  float eps;
};

struct V8 {
  float v[8];
};
__device__ __forceinline__ V8 zero8() {
  V8 r;
#pragma unroll
  for (int i = 0; i < 8; ++i) r.v[i] = 0.f;
  return r;
}
__device__ __forceinline__ V8 load8(const float* p) {
  const float4 a = ld4(p), b = ld4(p + 4);
  return {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
}
__device__ __forceinline__ V8 load8(const __nv_bfloat16* p) {
  const uint4 u = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  V8 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    r.v[2 * i] = __uint_as_float(w[i] << 16);
    r.v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
  return r;
}
__device__ __forceinline__ void store8(float* p, const V8& a) {
  st4(p, make_float4(a.v[0], a.v[1], a.v[2], a.v[3]));
  st4(p + 4, make_float4(a.v[4], a.v[5], a.v[6], a.v[7]));
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const V8& a) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a.v[2 * i], a.v[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

// Sums over a row, which W warps hold (group `g` of the CTA's ROW_WARPS / W; `slot` alternates, so that a
// sum's values are read before the one after the next is written).
template <int W>
struct RowSum {
  float2 (*red)[ROW_WARPS];              // [2][ROW_WARPS]
  int warp, slot;
  __device__ __forceinline__ float2 operator()(float a, float b) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      a += __shfl_xor_sync(0xffffffffu, a, o);
      b += __shfl_xor_sync(0xffffffffu, b, o);
    }
    if (W == 1) return make_float2(a, b);
    if ((threadIdx.x & 31) == 0) red[slot][warp] = make_float2(a, b);
    asm volatile("bar.sync %0, %1;" ::"r"(1 + warp / W), "n"(32 * W) : "memory");
    float2 t = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const float2 e = red[slot][warp / W * W + i];
      t.x += e.x;
      t.y += e.y;
    }
    slot ^= 1;
    return t;
  }
};

template <typename TY, int NV, int W, bool T>
__global__ void __launch_bounds__(ROW_THREADS, T ? 2 : 3) fwd_kernel(const Args a) {
  __shared__ float2 red[2][ROW_WARPS];
  constexpr int GROUPS = ROW_WARPS / W;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const float inv_d = 1.f / a.D;
  const TY *y = static_cast<const TY*>(a.y), *dy = static_cast<const TY*>(a.dy);
  RowSum<W> sum{red, warp, 0};
  int col[NV];
  bool in[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    col[i] = ((i * W + warp % W) * 32 + lane) * 8;
    in[i] = col[i] < a.D;
  }
  for (int row = blockIdx.x * GROUPS + warp / W; row < a.rows; row += gridDim.x * GROUPS) {
    const size_t at = (size_t)row * a.D;
    V8 v[NV], dv[T ? NV : 1], x[NV], dx[T ? NV : 1];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      v[i] = in[i] ? load8(y + at + col[i]) : zero8();
      x[i] = in[i] && a.res ? load8(a.res + at + col[i]) : zero8();
      if (T) {
        dv[i] = in[i] ? load8(dy + at + col[i]) : zero8();
        dx[i] = in[i] && a.dres ? load8(a.dres + at + col[i]) : zero8();
      }
    }
    float s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        s0 = fmaf(v[i].v[e], v[i].v[e], s0);
        if (T) s1 = fmaf(v[i].v[e], dv[i].v[e], s1);
      }
    float2 t = sum(s0, s1);
    const float iy = rsqrtf(t.x * inv_d + a.eps), cy = t.y * inv_d * iy * iy;     // (dy - y cy) iy
    s0 = s1 = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (!in[i]) continue;
      const V8 p = load8(a.post + col[i]), g = load8(a.gate + col[i]);
      V8 r;
      if (a.r) r = load8(a.r + col[i]);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float w = g.v[e] * p.v[e] * iy, re = a.r ? r.v[e] : 1.f;
        x[i].v[e] = fmaf(w, v[i].v[e], x[i].v[e] * re);
        s0 = fmaf(x[i].v[e], x[i].v[e], s0);
        if (T) {
          dx[i].v[e] = fmaf(w, fmaf(-cy, v[i].v[e], dv[i].v[e]), dx[i].v[e] * re);
          s1 = fmaf(x[i].v[e], dx[i].v[e], s1);
        }
      }
      store8(a.x + at + col[i], x[i]);
      if (T) store8(a.dx + at + col[i], dx[i]);
    }
    if (!a.pre) continue;
    t = sum(s0, s1);
    const float ix = rsqrtf(t.x * inv_d + a.eps), cx = t.y * inv_d * ix * ix;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (!in[i]) continue;
      const V8 p = load8(a.pre + col[i]);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (T) dx[i].v[e] = fmaf(-cx, x[i].v[e], dx[i].v[e]) * ix * p.v[e];
        x[i].v[e] *= ix * p.v[e];
      }
      store8(static_cast<TY*>(a.n) + at + col[i], x[i]);
      if (T) store8(static_cast<TY*>(a.dn) + at + col[i], dx[i]);
    }
  }
}

template <typename TY, int NV, int W>
__global__ void __launch_bounds__(ROW_THREADS, NV <= 2 ? 2 : 1) bwd_kernel(const Args a) {
  __shared__ float2 red[2][ROW_WARPS];
  constexpr int GROUPS = ROW_WARPS / W, COLS = NV * W * 256;
  __shared__ float flush[GROUPS > 1 ? GROUPS * COLS : 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, grp = warp / W;
  const float inv_d = 1.f / a.D;
  const TY *y = static_cast<const TY*>(a.y), *gn = static_cast<const TY*>(a.gn);
  RowSum<W> sum{red, warp, 0};
  int col[NV];
  bool in[NV];
  V8 c_pre[NV], c_r[NV], c_s[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    col[i] = ((i * W + warp % W) * 32 + lane) * 8;
    in[i] = col[i] < a.D;
    c_pre[i] = c_r[i] = c_s[i] = zero8();
  }
  for (int row = blockIdx.x * GROUPS + grp; row < a.rows; row += gridDim.x * GROUPS) {
    const size_t at = (size_t)row * a.D;
    V8 v[NV], x[NV], g[NV], h[NV];
    const bool need_res = a.res && (a.pre || a.r);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      v[i] = in[i] ? load8(y + at + col[i]) : zero8();
      x[i] = in[i] && need_res ? load8(a.res + at + col[i]) : zero8();
      g[i] = in[i] && a.gx ? load8(a.gx + at + col[i]) : zero8();
      h[i] = in[i] && a.pre ? load8(gn + at + col[i]) : zero8();
    }
    float s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) s0 = fmaf(v[i].v[e], v[i].v[e], s0);
    const float iy = rsqrtf(sum(s0, 0.f).x * inv_d + a.eps);
    V8 z[NV];                            // x again; `x` keeps res for the gradient of r
    float ix = 0.f, cx = 0.f;
    if (a.pre) {
      s0 = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (!in[i]) {
          z[i] = zero8();
          continue;
        }
        const V8 p = load8(a.post + col[i]), w = load8(a.gate + col[i]), q = load8(a.pre + col[i]);
        V8 r;
        if (a.r) r = load8(a.r + col[i]);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          z[i].v[e] = fmaf(w.v[e] * p.v[e] * iy, v[i].v[e], x[i].v[e] * (a.r ? r.v[e] : 1.f));
          s0 = fmaf(z[i].v[e], z[i].v[e], s0);
          s1 = fmaf(z[i].v[e], h[i].v[e] * q.v[e], s1);
        }
      }
      const float2 t = sum(s0, s1);
      ix = rsqrtf(t.x * inv_d + a.eps);
      cx = t.y * inv_d * ix * ix;        // g = gx + ix (pre gn - x cx)
    }
    s0 = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (!in[i]) continue;
      if (a.pre) {
        const V8 q = load8(a.pre + col[i]);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          c_pre[i].v[e] = fmaf(h[i].v[e] * ix, z[i].v[e], c_pre[i].v[e]);
          g[i].v[e] = fmaf(ix, fmaf(-cx, z[i].v[e], h[i].v[e] * q.v[e]), g[i].v[e]);
        }
      }
      const V8 p = load8(a.post + col[i]), w = load8(a.gate + col[i]);
      V8 r;
      if (a.r) r = load8(a.r + col[i]);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float yh = v[i].v[e] * iy;
        if (a.r) c_r[i].v[e] = fmaf(g[i].v[e], x[i].v[e], c_r[i].v[e]);
        c_s[i].v[e] = fmaf(g[i].v[e], yh, c_s[i].v[e]);
        h[i].v[e] = g[i].v[e] * w.v[e] * p.v[e];
        s0 = fmaf(h[i].v[e], yh, s0);
        if (a.r) g[i].v[e] *= r.v[e];
      }
      if (a.g_res) pn::store8(a.g_res + at + col[i], g[i]);
    }
    const float cy = sum(s0, 0.f).x * inv_d * iy;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (!in[i]) continue;
#pragma unroll
      for (int e = 0; e < 8; ++e) h[i].v[e] = fmaf(-cy, v[i].v[e], h[i].v[e]) * iy;
      pn::store8(static_cast<TY*>(a.g_y) + at + col[i], h[i]);
    }
  }
  // column sums of the CTA: groups in a fixed order; s becomes the gradients of gate and post
  float* out = a.partial + (size_t)blockIdx.x * 4 * a.D;
  auto write = [&](const V8(&acc)[NV], int which) {
    if (GROUPS == 1) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (!in[i]) continue;
        if (which < 2) {
          pn::store8(out + which * a.D + col[i], acc[i]);
        } else {
          const V8 p = load8(a.post + col[i]), w = load8(a.gate + col[i]);
          V8 u, t;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            u.v[e] = acc[i].v[e] * p.v[e];
            t.v[e] = acc[i].v[e] * w.v[e];
          }
          pn::store8(out + 2 * a.D + col[i], u);
          pn::store8(out + 3 * a.D + col[i], t);
        }
      }
      return;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NV; ++i) pn::store8(flush + grp * COLS + col[i], acc[i]);
    __syncthreads();
    for (int c = threadIdx.x; c < a.D; c += ROW_THREADS) {
      float t = 0.f;
#pragma unroll
      for (int k = 0; k < GROUPS; ++k) t += flush[k * COLS + c];
      if (which < 2) {
        out[which * a.D + c] = t;
      } else {
        out[2 * a.D + c] = t * a.post[c];
        out[3 * a.D + c] = t * a.gate[c];
      }
    }
  };
  if (a.pre) write(c_pre, 0);
  if (a.r) write(c_r, 1);
  write(c_s, 2);
}

// CTAs: every one of them works on rows from its start on, and the partial rows stay few.
template <int W>
static int grid(int rows, int ctas_per_sm) {
  const int groups = ROW_WARPS / W, most = 148 * ctas_per_sm, want = (rows + groups - 1) / groups;
  return want < most ? want : most;
}

constexpr int BWD_CTAS = 2;              // per SM

template <typename TY, int NV, int W>
static int launch(const Args& a, int mode, cudaStream_t st) {
  if (mode == 0)
    fwd_kernel<TY, NV, W, false><<<grid<W>(a.rows, 6), ROW_THREADS, 0, st>>>(a);
  else if (mode == 1)
    fwd_kernel<TY, NV, W, true><<<grid<W>(a.rows, 4), ROW_THREADS, 0, st>>>(a);
  else
    bwd_kernel<TY, NV, W><<<grid<W>(a.rows, BWD_CTAS), ROW_THREADS, 0, st>>>(a);
  return cudaGetLastError() == cudaSuccess ? IMF_OK : IMF_ERR_LAUNCH;
}

template <typename TY>
static int by_width(const Args& a, int mode, cudaStream_t st) {
  if (a.D <= 256) return launch<TY, 1, 1>(a, mode, st);
  if (a.D <= 512) return launch<TY, 2, 1>(a, mode, st);
  if (a.D <= 1024) return launch<TY, 2, 2>(a, mode, st);
  if (a.D <= 2048) return launch<TY, 2, 4>(a, mode, st);
  if (a.D <= 4096) return launch<TY, 2, 8>(a, mode, st);
  return launch<TY, 4, 8>(a, mode, st);
}

}  // namespace pn
}  // namespace imf

// Partial rows of column sums that mode 2 of imf_norm_add_norm writes.
extern "C" int imf_norm_add_norm_grid(int rows, int D) {
  using namespace imf::pn;
  if (D <= 512) return grid<1>(rows, BWD_CTAS);
  if (D <= 1024) return grid<2>(rows, BWD_CTAS);
  if (D <= 2048) return grid<4>(rows, BWD_CTAS);
  return grid<8>(rows, BWD_CTAS);
}

// mode 0 primal, 1 with tangent, 2 gradients.  p: 0 res, 1 dres, 2 y, 3 dy, 4 post, 5 gate, 6 r, 7 pre, 8 x, 9 dx,
// 10 n, 11 dn, 12 gx, 13 gn, 14 g_res, 15 g_y, 16 partial.  Rows contiguous, D a multiple of 8 up to 8,192, all
// addresses 16-byte aligned; y, dy, n, dn, gn, g_y bf16 or (y_fp32) fp32, the rest fp32.
extern "C" int imf_norm_add_norm(void** p, int rows, int D, float eps, int y_fp32, int mode, void* stream) {
  using namespace imf;
  if (rows <= 0 || D <= 0 || D % 8 || D > 8192 || mode < 0 || mode > 2) return IMF_ERR_ARG;
  for (int i = 0; i < 17; ++i)
    if (reinterpret_cast<uintptr_t>(p[i]) & 15) return IMF_ERR_ARG;
  if (!p[2] || !p[4] || !p[5] || (p[6] && !p[0])) return IMF_ERR_ARG;
  if (mode < 2 ? (!p[8] || (p[7] && !p[10])) : (!p[15] || !p[16] || (p[7] && !p[13]))) return IMF_ERR_ARG;
  if (mode == 1 && (!p[3] || !p[9] || (p[7] && !p[11]))) return IMF_ERR_ARG;
  pn::Args a;
  auto f = [&](int i) { return static_cast<float*>(p[i]); };
  a.res = f(0); a.dres = f(1); a.y = p[2]; a.dy = p[3];
  a.post = f(4); a.gate = f(5); a.r = f(6); a.pre = f(7);
  a.x = f(8); a.dx = f(9); a.n = p[10]; a.dn = p[11];
  a.gx = f(12); a.gn = p[13]; a.g_res = f(14); a.g_y = p[15]; a.partial = f(16);
  a.rows = rows; a.D = D; a.eps = eps;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return y_fp32 ? pn::by_width<float>(a, mode, st) : pn::by_width<__nv_bfloat16>(a, mode, st);
}
