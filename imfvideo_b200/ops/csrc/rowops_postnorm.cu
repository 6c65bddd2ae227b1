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
// warps, a lane to 8 adjacent channels of each of NV chunks; NV is 1 up to 2,048 channels, so that the column
// sums of the backward pass (24 registers a chunk) leave two CTAs of eight warps their place.  Rows come through
// shared memory, each group of W warps keeping the next STAGES rows on their way by bulk copies: loads from
// the warps themselves left too few bytes in flight (an earlier form, 32,780 x 1,024, gradients: 221 us with two chunks a
// lane, 174 with one; 104 this way).  The backward pass makes x again from res and y, of which it needs both anyway, instead of
// reading it.  Row sums add in a fixed order; column sums go through one partial row a CTA, added up in a fixed
// order by imf_colsum.
//
// Measured, 32,780 x 1,024, bf16 branch, cold, on the device: forward 66 us (342 of 402 MB reach DRAM by the end: 5.2
// TB/s, copy 6.55), with tangent 136 (746 of 806 MB, 5.5 TB/s), gradients 104 (563 of 604 MB, 5.4 TB/s).  From 1,025
// channels on a CTA has one row at a time, some 1.8 us each for gradients whatever its width: two or three
// exchanges between its warps, one behind the other, with two or three rows on an SM at a time (enough bytes
// are on their way: 72 to 192 KB an SM).  7,820 x 1,536 gradients 50 us, 4.3 TB/s; 20,000 x 2,048 133 us, 5.5
// TB/s.  One exchange less between a row's warps, the next row's sum over y going with this row's last, changes
// nothing there and costs the tangent 10 % at 2,048.  Column sums take 4 to 6 us more.
#include "common.cuh"
#include "host_util.h"
#include "rowops_common.cuh"

#include <type_traits>

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
  int stages;                            // rows of a group on their way
  int* status;
};

// eight channels, in pairs
struct V8 {
  f32x2 v[4];
};
__device__ __forceinline__ V8 zero8() { return {{0ull, 0ull, 0ull, 0ull}}; }
__device__ __forceinline__ V8 load8(const float* p) {
  const ulonglong2 a = reinterpret_cast<const ulonglong2*>(p)[0], b = reinterpret_cast<const ulonglong2*>(p)[1];
  return {{a.x, a.y, b.x, b.y}};
}
__device__ __forceinline__ V8 load8(const __nv_bfloat16* p) {
  const uint4 u = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  V8 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r.v[i] = pair2(w[i] << 16, w[i] & 0xffff0000u);
  return r;
}
// to global memory
__device__ __forceinline__ void store8(float* p, const V8& a) {
  reinterpret_cast<ulonglong2*>(p)[0] = make_ulonglong2(a.v[0], a.v[1]);
  reinterpret_cast<ulonglong2*>(p)[1] = make_ulonglong2(a.v[2], a.v[3]);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const V8& a) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = pack_bf16(lo2(a.v[i]), hi2(a.v[i]));
  *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ float sum2(f32x2 v) { return lo2(v) + hi2(v); }

// Warps of a CTA and CTAs of an SM.  From 1,025 channels on a CTA has one row at a time and as many warps as that takes;
// where registers leave room (five warps, or six without column sums), three such CTAs share an SM.  7,820 rows forward
// and gradients, against eight warps and two CTAs: 1,032 channels 33 -> 25 and 53 -> 39 us, 1,280 33 -> 29 and 53 -> 39,
// 1,536 35 -> 31 and 56 -> 49, 1,792 the same.
constexpr int cta_warps(int W) { return W > 4 ? W : ROW_WARPS; }
constexpr int ctas(int NV, int W, bool bwd) { return NV > 1 ? 1 : W == 5 || (W == 6 && !bwd) ? 3 : 2; }

// Sums over a row, which W warps hold (group `g` of the CTA's cta_warps(W) / W; `slot` alternates, so that a
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
    return across(a, b);
  }
  __device__ __forceinline__ float operator()(float a) { return across(warp_sum(a), 0.f).x; }
  __device__ __forceinline__ float2 across(float a, float b) {
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

// Rows of a group of W warps on their way from global memory: `n` tensors of `bytes` a row each.
struct Source {
  const uint8_t* p[4];
  uint32_t bytes[4];
};
constexpr int MAX_STAGES = 8;
template <int W>
struct Ring {
  uint64_t* full;                        // [stages] of this group
  uint8_t* buf;
  volatile int* abort_flag;
  Source src;
  uint32_t row_bytes;
  int stages, step, rows, next, st;      // next: the row to be asked for
  uint32_t par;
  bool issuer;

  __device__ __forceinline__ void ask(int stage) {
    if (issuer && next < rows) {
      mbar_arrive_expect_tx(full + stage, row_bytes);
      uint8_t* dst = buf + (size_t)stage * row_bytes;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        if (!src.p[t]) continue;
        asm volatile(
            "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
            ::"r"(smem_u32(dst)), "l"(src.p[t] + (size_t)next * src.bytes[t]), "r"(src.bytes[t]), "r"(smem_u32(full + stage))
            : "memory");
        dst += src.bytes[t];
      }
    }
    next += step;
  }
  // The current row's tensors are in shared memory.  A wait that runs out is recorded in the status word and the
  // row is made from what is there: a warp that left would leave the others of its group at their barrier.
  __device__ __forceinline__ void wait(int* status) { mbar_wait(full + st, par, abort_flag, status, STATUS_TIMEOUT_TMA); }
  __device__ __forceinline__ const uint8_t* row() const { return buf + (size_t)st * row_bytes; }
  // every warp of the group has the row in registers: its place goes to the row `stages` further
  __device__ __forceinline__ void pass() {
    if (W == 1) __syncwarp();            // (a row's sum over several warps has a barrier)
    ask(st);
    if (++st == stages) {
      st = 0;
      par ^= 1;
    }
  }
};

// Shared memory: barriers, flag, then the rows of the groups.
constexpr int HEAD = ROW_WARPS * MAX_STAGES * 8 + 64;
template <int W>
__device__ __forceinline__ Ring<W> make_ring(uint8_t* smem, const Args& a, const Source& src) {
  constexpr int GROUPS = cta_warps(W) / W;
  const int warp = threadIdx.x >> 5, grp = warp / W;
  Ring<W> r;
  r.full = reinterpret_cast<uint64_t*>(smem) + grp * MAX_STAGES;
  r.abort_flag = reinterpret_cast<volatile int*>(smem + ROW_WARPS * MAX_STAGES * 8);
  r.src = src;
  r.row_bytes = 0;
#pragma unroll
  for (int t = 0; t < 4; ++t) r.row_bytes += src.p[t] ? src.bytes[t] : 0;
  r.stages = a.stages;
  r.buf = smem + HEAD + (size_t)grp * a.stages * r.row_bytes;
  r.step = gridDim.x * GROUPS;
  r.rows = a.rows;
  r.next = blockIdx.x * GROUPS + grp;
  r.st = 0;
  r.par = 0;
  r.issuer = warp % W == 0 && (threadIdx.x & 31) == 0;
  if (threadIdx.x == 0) *const_cast<int*>(r.abort_flag) = 0;
  if (r.issuer) {
    for (int i = 0; i < a.stages; ++i) mbar_init(r.full + i, 1);
    fence_barrier_init();
  }
  __syncthreads();
  for (int i = 0; i < a.stages; ++i) r.ask(i);
  return r;
}

template <typename TY, int NV, int W, bool T>
__global__ void __launch_bounds__(32 * cta_warps(W), ctas(NV, W, false)) fwd_kernel(const Args a) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float2 red[2][ROW_WARPS];
  constexpr int GROUPS = cta_warps(W) / W;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const float inv_d = 1.f / a.D;
  const uint32_t by = a.D * (uint32_t)sizeof(TY), bf = a.D * 4u;
  typedef const uint8_t* ptr;
  Ring<W> ring = make_ring<W>(smem, a, Source{{(ptr)a.y, (ptr)a.res, T ? (ptr)a.dy : nullptr, T ? (ptr)a.dres : nullptr},
                                              {by, bf, by, bf}});
  RowSum<W> sum{red, warp, 0};
  int col[NV];
  bool in[NV];
  V8 gp[NV], r[NV], pre[NV];             // gate * post, the residual's scale, the second norm's gain
  const V8 one = {{dup2(1.f), dup2(1.f), dup2(1.f), dup2(1.f)}};
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    col[i] = ((i * W + warp % W) * 32 + lane) * 8;
    in[i] = col[i] < a.D;
    const V8 p = in[i] ? load8(a.post + col[i]) : zero8(), g = in[i] ? load8(a.gate + col[i]) : zero8();
#pragma unroll
    for (int e = 0; e < 4; ++e) gp[i].v[e] = mul2(p.v[e], g.v[e]);
    r[i] = in[i] && a.r ? load8(a.r + col[i]) : one;
    pre[i] = in[i] && a.pre ? load8(a.pre + col[i]) : zero8();
  }
  for (int row = blockIdx.x * GROUPS + warp / W; row < a.rows; row += gridDim.x * GROUPS) {
    const size_t at = (size_t)row * a.D;
    ring.wait(a.status);
    const uint8_t* sy = ring.row();
    const float* sr = reinterpret_cast<const float*>(sy + by);
    const uint8_t* sdy = sy + by + (a.res ? bf : 0);
    const float* sdr = reinterpret_cast<const float*>(sdy + by);
    V8 v[NV], dv[T ? NV : 1], x[NV], dx[T ? NV : 1];
    f32x2 s0 = 0ull, s1 = 0ull;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      v[i] = in[i] ? load8(reinterpret_cast<const TY*>(sy) + col[i]) : zero8();
      x[i] = in[i] && a.res ? load8(sr + col[i]) : zero8();
      if (T) {
        dv[i] = in[i] ? load8(reinterpret_cast<const TY*>(sdy) + col[i]) : zero8();
        dx[i] = in[i] && a.dres ? load8(sdr + col[i]) : zero8();
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s0 = fma2(v[i].v[e], v[i].v[e], s0);
        if (T) s1 = fma2(v[i].v[e], dv[i].v[e], s1);
      }
    }
    float2 t = T ? sum(sum2(s0), sum2(s1)) : make_float2(sum(sum2(s0)), 0.f);
    ring.pass();
    const float iy = rsqrtf(t.x * inv_d + a.eps);
    const f32x2 iy2 = dup2(iy), cy2 = dup2(-t.y * inv_d * iy * iy);              // (dy - y cy) iy
    s0 = s1 = 0ull;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (!in[i]) continue;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const f32x2 w = mul2(gp[i].v[e], iy2);
        x[i].v[e] = fma2(w, v[i].v[e], mul2(x[i].v[e], r[i].v[e]));
        s0 = fma2(x[i].v[e], x[i].v[e], s0);
        if (T) {
          dx[i].v[e] = fma2(w, fma2(cy2, v[i].v[e], dv[i].v[e]), mul2(dx[i].v[e], r[i].v[e]));
          s1 = fma2(x[i].v[e], dx[i].v[e], s1);
        }
      }
      pn::store8(a.x + at + col[i], x[i]);
      if (T) pn::store8(a.dx + at + col[i], dx[i]);
    }
    if (!a.pre) continue;
    t = T ? sum(sum2(s0), sum2(s1)) : make_float2(sum(sum2(s0)), 0.f);
    const float ix = rsqrtf(t.x * inv_d + a.eps);
    const f32x2 ix2 = dup2(ix), cx2 = dup2(-t.y * inv_d * ix * ix);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (!in[i]) continue;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const f32x2 w = mul2(pre[i].v[e], ix2);
        if (T) dx[i].v[e] = mul2(fma2(cx2, x[i].v[e], dx[i].v[e]), w);
        x[i].v[e] = mul2(x[i].v[e], w);
      }
      pn::store8(static_cast<TY*>(a.n) + at + col[i], x[i]);
      if (T) pn::store8(static_cast<TY*>(a.dn) + at + col[i], dx[i]);
    }
  }
}

template <typename TY, int NV, int W>
__global__ void __launch_bounds__(32 * cta_warps(W), ctas(NV, W, true)) bwd_kernel(const Args a) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float2 red[2][ROW_WARPS];
  constexpr int GROUPS = cta_warps(W) / W, COLS = NV * W * 256;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, grp = warp / W;
  const float inv_d = 1.f / a.D;
  const bool need_res = a.res && (a.pre || a.r);
  const uint32_t by = a.D * (uint32_t)sizeof(TY), bf = a.D * 4u;
  typedef const uint8_t* ptr;
  Ring<W> ring = make_ring<W>(smem, a, Source{{(ptr)a.y, need_res ? (ptr)a.res : nullptr, (ptr)a.gx, a.pre ? (ptr)a.gn : nullptr},
                                              {by, bf, bf, by}});
  RowSum<W> sum{red, warp, 0};
  int col[NV];
  bool in[NV];
  V8 gp[NV], r[NV], pre[NV];             // gate * post, the residual's scale, the second norm's gain
  V8 c_pre[NV], c_r[NV], c_s[NV];
  const V8 one = {{dup2(1.f), dup2(1.f), dup2(1.f), dup2(1.f)}};
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    col[i] = ((i * W + warp % W) * 32 + lane) * 8;
    in[i] = col[i] < a.D;
    const V8 p = in[i] ? load8(a.post + col[i]) : zero8(), g = in[i] ? load8(a.gate + col[i]) : zero8();
#pragma unroll
    for (int e = 0; e < 4; ++e) gp[i].v[e] = mul2(p.v[e], g.v[e]);
    r[i] = in[i] && a.r ? load8(a.r + col[i]) : one;
    c_pre[i] = c_r[i] = c_s[i] = zero8();
    pre[i] = in[i] && a.pre ? load8(a.pre + col[i]) : zero8();
  }
  for (int row = blockIdx.x * GROUPS + grp; row < a.rows; row += gridDim.x * GROUPS) {
    const size_t at = (size_t)row * a.D;
    ring.wait(a.status);
    const uint8_t* sy = ring.row();
    const uint8_t* sr = sy + by;
    const uint8_t* sg = sr + (need_res ? bf : 0);
    const uint8_t* sn = sg + (a.gx ? bf : 0);
    V8 v[NV], x[NV], g[NV], h[NV];
    f32x2 s0 = 0ull, s1 = 0ull;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      v[i] = in[i] ? load8(reinterpret_cast<const TY*>(sy) + col[i]) : zero8();
      x[i] = in[i] && need_res ? load8(reinterpret_cast<const float*>(sr) + col[i]) : zero8();
      g[i] = in[i] && a.gx ? load8(reinterpret_cast<const float*>(sg) + col[i]) : zero8();
      h[i] = in[i] && a.pre ? load8(reinterpret_cast<const TY*>(sn) + col[i]) : zero8();
#pragma unroll
      for (int e = 0; e < 4; ++e) s0 = fma2(v[i].v[e], v[i].v[e], s0);
    }
    const float iy = rsqrtf(sum(sum2(s0)) * inv_d + a.eps);
    const f32x2 iy2 = dup2(iy);
    ring.pass();
    if (a.pre) {
      s0 = 0ull;
      V8 z[NV];                          // x again; `x` keeps res for the gradient of r
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          z[i].v[e] = fma2(mul2(gp[i].v[e], iy2), v[i].v[e], mul2(x[i].v[e], r[i].v[e]));
          s0 = fma2(z[i].v[e], z[i].v[e], s0);
          s1 = fma2(z[i].v[e], mul2(h[i].v[e], pre[i].v[e]), s1);
        }
      const float2 t = sum(sum2(s0), sum2(s1));
      const float ix = rsqrtf(t.x * inv_d + a.eps);
      const f32x2 ix2 = dup2(ix), cx2 = dup2(-t.y * inv_d * ix * ix);      // g = gx + ix (pre gn - x cx)
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          c_pre[i].v[e] = fma2(mul2(h[i].v[e], ix2), z[i].v[e], c_pre[i].v[e]);
          g[i].v[e] = fma2(ix2, fma2(cx2, z[i].v[e], mul2(h[i].v[e], pre[i].v[e])), g[i].v[e]);
        }
    }
    s0 = 0ull;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const f32x2 yh = mul2(v[i].v[e], iy2);
        c_r[i].v[e] = fma2(g[i].v[e], x[i].v[e], c_r[i].v[e]);
        c_s[i].v[e] = fma2(g[i].v[e], yh, c_s[i].v[e]);
        h[i].v[e] = mul2(g[i].v[e], gp[i].v[e]);
        s0 = fma2(h[i].v[e], yh, s0);
        g[i].v[e] = mul2(g[i].v[e], r[i].v[e]);
      }
      if (a.g_res && in[i]) pn::store8(a.g_res + at + col[i], g[i]);
    }
    const f32x2 cy2 = dup2(-sum(sum2(s0)) * inv_d * iy);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
      for (int e = 0; e < 4; ++e) h[i].v[e] = mul2(fma2(cy2, v[i].v[e], h[i].v[e]), iy2);
      if (in[i]) pn::store8(static_cast<TY*>(a.g_y) + at + col[i], h[i]);
    }
  }
  // column sums of the CTA: groups in a fixed order; s becomes the gradients of gate and post
  float* out = a.partial + (size_t)blockIdx.x * 4 * a.D;
  float* flush = reinterpret_cast<float*>(smem + HEAD);
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
          for (int e = 0; e < 4; ++e) {
            u.v[e] = mul2(acc[i].v[e], p.v[e]);
            t.v[e] = mul2(acc[i].v[e], w.v[e]);
          }
          pn::store8(out + 2 * a.D + col[i], u);
          pn::store8(out + 3 * a.D + col[i], t);
        }
      }
      return;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) reinterpret_cast<f32x2*>(flush + grp * COLS + col[i])[e] = acc[i].v[e];
    __syncthreads();
    for (int c = threadIdx.x; c < a.D; c += 32 * cta_warps(W)) {
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

// CTAs: every one of them works on rows from its start on, and the partial rows stay few.  (Three or four CTAs an SM of the
// forward pass, with fewer rows each on their way, change nothing: 32,780 x 1,024 77 and 78 us instead of 77, with
// tangent 147 and 148 to 152 instead of 147, launch included.)
static int grid(int rows, int groups, int ctas_per_sm) {
  const int most = 148 * ctas_per_sm, want = (rows + groups - 1) / groups;
  return want < most ? want : most;
}

template <typename TY, int NV, int W>
static int launch(Args a, int mode, cudaStream_t st) {
  const int per_sm = ctas(NV, W, mode == 2), groups = cta_warps(W) / W;
  const size_t ty = sizeof(TY);
  const size_t row = a.D * (mode == 0 ? ty + (a.res ? 4 : 0)
                            : mode == 1 ? 2 * ty + (a.res ? 4 : 0) + (a.dres ? 4 : 0)
                                        : ty + (a.res && (a.pre || a.r) ? 4 : 0) + (a.gx ? 4 : 0) + (a.pre ? ty : 0));
  // as many rows on their way as fit beside the other CTAs of an SM
  const int fit = (int)((216 * 1024 / per_sm - HEAD - 1024) / (groups * row));
  a.stages = fit < 1 ? 1 : fit > MAX_STAGES ? MAX_STAGES : fit;
  size_t smem = HEAD + groups * a.stages * row;
  const size_t flush = HEAD + (mode == 2 && groups > 1 ? (size_t)groups * NV * W * 256 * 4 : 0);
  if (smem < flush) smem = flush;
  auto kern = mode == 0 ? fwd_kernel<TY, NV, W, false> : mode == 1 ? fwd_kernel<TY, NV, W, true> : bwd_kernel<TY, NV, W>;
  static bool smem_set[3][HOST_MAX_DEVICES] = {{false}};
  if (!allow_smem((const void*)kern, 225 * 1024, smem_set[mode])) return IMF_ERR_LAUNCH;
  kern<<<grid(a.rows, groups, per_sm), 32 * cta_warps(W), smem, st>>>(a);
  return cudaGetLastError() == cudaSuccess ? IMF_OK : IMF_ERR_LAUNCH;
}

// f(chunks a lane, warps a row) for rows of D channels
template <typename F>
static int by_width(int D, F f) {
  using std::integral_constant;
  #define IMF_WIDTH(NV, W) \
  if (D <= NV * W * 256) return f(integral_constant<int, NV>(), integral_constant<int, W>())
  IMF_WIDTH(1, 1);
  IMF_WIDTH(1, 2);
  IMF_WIDTH(1, 4);
  IMF_WIDTH(1, 5);
  IMF_WIDTH(1, 6);
  IMF_WIDTH(1, 7);
  IMF_WIDTH(1, 8);
  IMF_WIDTH(2, 8);
  return f(integral_constant<int, 4>(), integral_constant<int, 8>());
#undef IMF_WIDTH
}

template <typename TY>
static int run(const Args& a, int mode, cudaStream_t st) {
  return by_width(a.D, [&](auto nv, auto w) { return launch<TY, nv.value, w.value>(a, mode, st); });
}

}  // namespace pn
}  // namespace imf

// Partial rows of column sums that mode 2 of imf_norm_add_norm writes.
extern "C" int imf_norm_add_norm_grid(int rows, int D) {
  using namespace imf::pn;
  return by_width(D, [&](auto nv, auto w) {
    return grid(rows, cta_warps(w.value) / w.value, ctas(nv.value, w.value, true));
  });
}

extern "C" int imf_colsum(const void* entries, int n, void* stream);

// mode 0 primal, 1 with tangent, 2 gradients.  p: 0 res, 1 dres, 2 y, 3 dy, 4 post, 5 gate, 6 r, 7 pre, 8 x, 9 dx,
// 10 n, 11 dn, 12 gx, 13 gn, 14 g_res, 15 g_y, 16 partial, 17 gradients of pre, r, gate, post ([4][D], null: the caller
// adds the partial rows up).  Rows contiguous, D a multiple of 8 up to 8,192, all
// addresses 16-byte aligned; y, dy, n, dn, gn, g_y bf16 or (y_fp32) fp32, the rest fp32.
extern "C" int imf_norm_add_norm(void** p, int rows, int D, float eps, int y_fp32, int mode, int* status, void* stream) {
  using namespace imf;
  // (a row's number, and that of a row some steps further, in 32 bits)
  if (rows <= 0 || rows >= 1 << 30 || D <= 0 || D % 8 || D > 8192 || mode < 0 || mode > 2) return IMF_ERR_ARG;
  for (int i = 0; i < 18; ++i)
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
  a.stages = 0; a.status = status;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int rc = y_fp32 ? pn::run<float>(a, mode, st) : pn::run<__nv_bfloat16>(a, mode, st);
  if (rc != IMF_OK || mode != 2 || !p[17]) return rc;
  struct {
    const float* part;
    float* dst;
    int g, D, stride, accumulate;
  } e[4];
  int n = 0;
  for (int i = 0; i < 4; ++i)
    if ((i != 0 || a.pre) && (i != 1 || a.r))
      e[n++] = {a.partial + (size_t)i * D, f(17) + (size_t)i * D, imf_norm_add_norm_grid(rows, D), D, 4 * D, 0};
  return imf_colsum(e, n, stream);
}
