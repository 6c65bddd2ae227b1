// Differential attention backward (reverse mode) on tcgen05 / TMEM (see attn_diff.h for the pairing of
// heads; w_1 = 1, w_2 = -lam):
//
//   S_m^T = K_m Q_m^T,  P_m^T = w_m exp2(S_m^T * scale*log2e - lse2_m),  dP^T = V dO^T,
//   dS_m^T = P_m^T .* (dP^T - delta_m),   delta_m = rowsum(dO .* O_m)
//   dV = sum_m P_m^T dO,   dK_m = scale * dS_m^T Q_m,   dQ_m = scale * dS_m K_m,   dlam = -sum delta_2
//
// From o = O_1 - lam O_2 and O_2, which the forward pass keeps to 16 bits: delta_1 = rowsum(dO .* o) + lam delta_2.
//
// CTA = one 128-row K/V tile of one (batch, pair).  It walks over the 128-row query tiles twice, for map 1
// and then for map 2; dV (128 columns) adds up over both walks, dK (64) is stored between them.  As in
// attn_bwd.cu everything is computed transposed (K/V rows on the TMEM lanes), P^T and dS^T are the A
// operands of dV and dK from TMEM, dS^T goes through shared memory for dQ, and dQ tiles are added to fp32
// in global memory by TMA.
//
// TMEM: S^T 128 columns, dP^T 128, dK 64, dV 128, dQ 64 are all 512, so P^T lies over the S^T and dS^T over
// the dP^T that it is made from, and S^T of the next step follows dV of this one.  The tensor core then
// works in two stretches, dV and the next S^T (768 clocks) while the math warps are at dS^T, dK, dQ and the
// next dP^T (1,280) while they take exponentials.  Both maps at once would share dP^T but take 64 columns
// more.
//
// The constants of a query row ride on the tensor core: a band of 16 columns a row holds -lse / scale and
// -delta as three bf16 parts each (24 bits), and one more K-step against a tile of ones in the columns
// that are meant makes S^T - lse / scale and dP^T - delta.  Reading them from shared memory instead costs the
// math warps 1,024 clocks of its 128 B a clock per step, every lane of a warp the same 16 bytes.
// Shared memory: both K, V, two stages each of Q and dO, dS^T, half a dQ tile, bands and ones: 225 of 227 KB.
//
// Roundings: P^T and dS^T go to the tensor core in bf16 (each off by at most 2^-8 of its value); dP, delta,
// the exponents and all sums are in 32 bits (delta and the log-sum-exp as three bf16 parts, 24 bits).
//
// What bounds it: shared memory moves 361 KB a step, 2,820 clocks at 128 B a clock, and a step takes some
// 2,800 to 2,900; the tensor pipe is 69 % busy.  Measured, 1 x 7,820 rows, 8 pairs: 730 to 745 us, with
// preparation and conversion 780; 1 x 29,140 rows, 2 pairs: 2.5 to 2.7 ms.  Before: row constants from shared
// memory, all exponentials on their unit and whole dQ tiles behind a barrier of four warps 926 us; a quarter of the
// exponentials on the FMA units 838 -> 817.  Slower: P^T and dS^T both over dP^T, with S^T a step ahead (1,130); dQ
// added from registers (1,135); V as dP^T's operand in TMEM, 329 KB a step, for which dQ has to lie over dP^T (798
// for 780).  Both maps at once on 64-row steps would need one dP^T and one dV, but each map has a delta of its own,
// to be read from shared memory again: 346 KB for what are 361 now.
#include "attn_bwd_split.h"
#include "attn_diff.h"
#include "common.cuh"
#include "host_util.h"

namespace imf {
namespace diffb {

constexpr int HD = 64;
constexpr int VD = 128;
constexpr int T = 128;               // rows of a K/V tile and of a query tile
constexpr int THREADS = 512;         // 16 warps (setmaxnreg works on whole warpgroups; 14, 15 idle)
constexpr int STAGES = 2;            // of Q (with the rows' constants) and of dO, each a ring of its own
constexpr int PANEL = T * 128;       // bytes of 64 bf16 (or 32 fp32) columns of a tile
constexpr float LOG2E = 1.4426950408889634f;

// TMEM columns
constexpr int C_S = 0, C_DP = 128, C_DK = 256, C_DV = 320, C_DQ = 448;
// column of the bf16 A operand of k-step `ks` (16 query rows): query columns 0-63 become columns 0-31,
// query columns 64-127 columns 64-95 (each half is read and written by one warp group only)
__device__ __forceinline__ constexpr int step_col(int ks) { return (ks >> 2) * 64 + (ks & 3) * 8; }

struct Smem {
  uint8_t k[2][PANEL];               // K_1, K_2
  uint8_t v[2][PANEL];               // the two halves of V
  uint8_t q[STAGES][PANEL];
  uint8_t d_o[STAGES][2][PANEL];
  uint8_t ds[2][PANEL];              // dS^T: [kv 128][q 128] as two 64-column panels
  uint8_t dq_stage[4][PANEL / 4];    // by warp: 32 rows of 32 columns of a dQ tile [q 128][64] fp32
  uint8_t band[STAGES][T * 32];      // [q 128][16] bf16: -lse / scale, -delta in three parts each, zeros
  uint8_t ones[2][T * 32];           // [kv 128][16] bf16: ones in columns 0-2, in columns 3-5
  uint64_t kv_full;
  uint64_t q_full[STAGES], q_empty[STAGES], do_full[STAGES], do_empty[STAGES];
  uint64_t s_full, p_ready, dp_full, ds_ready, dq_full, dq_free, dk_free, final_bar;
  uint32_t tmem_base;
  int abort_flag;
};
static_assert(sizeof(Smem) <= 232448, "shared memory of an SM");

struct Params {
  DiffWeights lam;
  __nv_bfloat16* dk;
  __nv_bfloat16* dv;
  int B, H, L, Lp;        // H pairs
  int64_t dk_sb, dk_sl, dk_sh, dv_sb, dv_sl, dv_sh;
  float scale;
  int* status;
  int n_t, group;         // K/V tiles of a chain; chains that are worked on at a time (bwd_item)
  // the steps of each K/V tile from n_whole on are split over `parts` CTAs to even out the last wave
  // (attn_bwd_split.h); each writes fp32 partials to part[(tile - n_whole) * parts + r] =
  // [dK_1 | dK_2 | dV] ([128][64], [128][64], [128][128], dK unscaled) and the last kernel adds them up
  int n_whole, parts;
  float* part;
  // fixed-order dQ (null = arrival order): one counter per (batch, head, 32 query rows), zeroed before the
  // launch; the CTA of K/V tile j adds when the counter shows j
  int* turn;
};
constexpr size_t PART = (size_t)T * (2 * HD + VD);       // floats of a partial result
static_assert(PART % (4 * 256) == 0, "blocks of the merge lie within a tile");

// which of a row's pairs of columns take their exponentials on the FMA units
__device__ __forceinline__ constexpr bool fma_pair(int i) { return (i & 3) == 1; }

IMF_DEVICE void tma_reduce_add_4d(const CUtensorMap* m, const void* src, int c0, int c1, int c2, int c3) {
  asm volatile(
      "cp.reduce.async.bulk.tensor.4d.global.shared::cta.add.tile.bulk_group"
      " [%0, {%2, %3, %4, %5}], [%1];"
      ::"l"(reinterpret_cast<uint64_t>(m)), "r"(smem_u32(src)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}

__global__ void __launch_bounds__(THREADS, 1)
attn_diff_bwd_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                     const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_do,
                     const __grid_constant__ CUtensorMap tm_dq, const __grid_constant__ CUtensorMap tm_band,
                     const Params p) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  auto& s = *reinterpret_cast<Smem*>(smem_raw);
  if (smem_u32(smem_raw) & 1023u) {      // the swizzled tiles need it; there is no room to align here
    if (threadIdx.x == 0 && p.status) atomicCAS(p.status, 0, STATUS_BAD_ARG);
    return;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int idx = (int)blockIdx.x;
  const bool split = idx >= p.n_whole;
  const int item = split ? p.n_whole + (idx - p.n_whole) / p.parts : idx;
  const int qpart = split ? (idx - p.n_whole) % p.parts : 0, parts = split ? p.parts : 1;
  int chain, kvb;
  bwd_item(item, p.B * p.H, p.n_t, p.group, chain, kvb);
  const int h = chain % p.H, b = chain / p.H;
  // Step i of this CTA is step first + i of the tile: map 1 for the first n_qt of these, then map 2.
  const int n_qt = (p.L + T - 1) / T;
  const int first = (int)((long)qpart * 2 * n_qt / parts);
  const int n = (int)((long)(qpart + 1) * 2 * n_qt / parts) - first;
  auto map_of = [&](int i) { return first + i >= n_qt ? 1 : 0; };
  auto tile_of = [&](int i) { return first + i >= n_qt ? first + i - n_qt : first + i; };
  int* turn = p.turn ? p.turn + ((size_t)b * p.H + h) * 2 * n_qt * 4 : nullptr;     // by step of the tile and warp

  if (threadIdx.x == 0) {
    mbar_init(&s.kv_full, 1);
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&s.q_full[i], 1);
      mbar_init(&s.q_empty[i], 1);
      mbar_init(&s.do_full[i], 1);
      mbar_init(&s.do_empty[i], 1);
    }
    mbar_init(&s.s_full, 1);
    mbar_init(&s.p_ready, 8);      // one arrival per math warp
    mbar_init(&s.dp_full, 1);
    mbar_init(&s.ds_ready, 8);
    mbar_init(&s.dq_full, 1);
    mbar_init(&s.dq_free, 4);
    mbar_init(&s.dk_free, 4);
    mbar_init(&s.final_bar, 1);
    s.abort_flag = 0;
    fence_barrier_init();
  }
  // rows of 16 bf16, 32 bytes, whose two halves SWIZZLE_32B exchanges in every other group of four rows
  for (int i = threadIdx.x; i < 2 * T * 2; i += THREADS) {
    const int which = i / (2 * T), r = i / 2 % T, half = i & 1;
    const uint4 w = half ? make_uint4(0u, 0u, 0u, 0u)
                         : which == 0 ? make_uint4(0x3f803f80u, 0x00003f80u, 0u, 0u)
                                      : make_uint4(0u, 0x3f800000u, 0x3f803f80u, 0u);
    *reinterpret_cast<uint4*>(s.ones[which] + r * 32 + ((half ^ ((r >> 2) & 1)) << 4)) = w;
  }
  fence_proxy_async_smem();
  if (warp == 12) {
    tmem_alloc(&s.tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s.tmem_base;
  volatile int* abort_flag = &s.abort_flag;

  if (warp >= 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
    if (warp == 13) {
      // ------------------------------------------------------ TMA producer --
      if (elect_one()) {
        prefetch_tmap(&tm_q);
        prefetch_tmap(&tm_k);
        prefetch_tmap(&tm_v);
        prefetch_tmap(&tm_do);
        mbar_arrive_expect_tx(&s.kv_full, 4 * PANEL);
        for (int m = 0; m < 2; ++m) {
          tma_load_4d(s.k[m], &tm_k, &s.kv_full, 0, 2 * h + m, kvb * T, b);
          tma_load_4d(s.v[m], &tm_v, &s.kv_full, 0, 2 * h + m, kvb * T, b);
        }
        for (int i = 0; i < n; ++i) {
          const int st = i & 1, m = map_of(i), qt = tile_of(i);
          const uint32_t par = (uint32_t)((i >> 1) & 1) ^ 1;
          // (the dO of a step has its last reader well before its Q has)
          if (i >= STAGES && !mbar_wait(&s.do_empty[st], par, abort_flag, p.status, STATUS_TIMEOUT_EMPTY)) break;
          mbar_arrive_expect_tx(&s.do_full[st], 2 * PANEL);
          for (int c = 0; c < 2; ++c) tma_load_4d(s.d_o[st][c], &tm_do, &s.do_full[st], 0, 2 * h + c, qt * T, b);
          if (i >= STAGES && !mbar_wait(&s.q_empty[st], par, abort_flag, p.status, STATUS_TIMEOUT_EMPTY)) break;
          mbar_arrive_expect_tx(&s.q_full[st], PANEL + T * 32);
          tma_load_4d(s.q[st], &tm_q, &s.q_full[st], 0, 2 * h + m, qt * T, b);
          tma_load_3d(s.band[st], &tm_band, &s.q_full[st], 0, qt * T, b * 2 * p.H + 2 * h + m);
        }
      }
    } else if (warp == 12) {
      // -------------------------------------------------------- MMA issuer --
      if (elect_one()) {
        constexpr uint32_t id_st = idesc_bf16(T, T, 0, 0);       // S^T, dP^T: [kv 128][q 128] (SS)
        constexpr uint32_t id_dv = idesc_bf16(T, VD, 0, 1);      // dV: [kv 128][128] (TS)
        constexpr uint32_t id_dk = idesc_bf16(T, HD, 0, 1);      // dK: [kv 128][64] (TS)
        constexpr uint32_t id_dq = idesc_bf16(T, HD, 1, 1);      // dQ: [q 128][64] (SS, A MN-major)
        const uint32_t ka = smem_u32(s.k[0]), va = smem_u32(s.v[0]), dsa = smem_u32(s.ds[0]);
        auto issue_s = [&](int i) {
          const uint32_t a = ka + map_of(i) * PANEL, qa = smem_u32(s.q[i & 1]);
#pragma unroll
          for (int ks = 0; ks < HD / 16; ++ks)
            mma_ss(tmem + C_S, sdesc_kmajor(a + ks * 32), sdesc_kmajor(qa + ks * 32), id_st, ks != 0);
          mma_ss(tmem + C_S, sdesc_kmajor_sw32(smem_u32(s.ones[0])), sdesc_kmajor_sw32(smem_u32(s.band[i & 1])), id_st, 1);
          tc_commit(&s.s_full);
        };
        auto issue_dp = [&](int i) {
          const uint32_t doa = smem_u32(s.d_o[i & 1][0]);
#pragma unroll
          for (int ks = 0; ks < VD / 16; ++ks)
            mma_ss(tmem + C_DP, sdesc_kmajor(va + (ks / 4) * PANEL + (ks % 4) * 32),
                   sdesc_kmajor(doa + (ks / 4) * PANEL + (ks % 4) * 32), id_st, ks != 0);
          mma_ss(tmem + C_DP, sdesc_kmajor_sw32(smem_u32(s.ones[1])), sdesc_kmajor_sw32(smem_u32(s.band[i & 1])), id_st, 1);
          tc_commit(&s.dp_full);
        };
        bool ok = n > 0 && mbar_wait(&s.kv_full, 0, abort_flag, p.status, STATUS_TIMEOUT_TMA) &&
                  mbar_wait(&s.q_full[0], 0, abort_flag, p.status, STATUS_TIMEOUT_TMA) &&
                  mbar_wait(&s.do_full[0], 0, abort_flag, p.status, STATUS_TIMEOUT_TMA);
        if (ok) {
          tc_fence_after();
          issue_s(0);
          issue_dp(0);
        }
        for (int i = 0; i < n && ok; ++i) {
          const int st = i & 1;
          const uint32_t par = (uint32_t)(i & 1), nph = (uint32_t)(((i + 1) >> 1) & 1);
          const uint32_t qa = smem_u32(s.q[st]), doa = smem_u32(s.d_o[st][0]);
          const bool new_map = i > 0 && map_of(i) != map_of(i - 1);
          // dV += P^T dO, and S^T of the next step over that P^T, while the math warps work on dS^T
          ok = mbar_wait(&s.p_ready, par, abort_flag, p.status, STATUS_TIMEOUT_SOFTMAX);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int ks = 0; ks < T / 16; ++ks)
            mma_ts(tmem + C_DV, tmem + C_S + step_col(ks), sdesc_mnmajor(doa + ks * 2048, PANEL), id_dv, (i | ks) != 0);
          tc_commit(&s.do_empty[st]);
          if (i + 1 < n) {
            ok = mbar_wait(&s.q_full[st ^ 1], nph, abort_flag, p.status, STATUS_TIMEOUT_TMA);
            if (!ok) break;
            tc_fence_after();
            issue_s(i + 1);
          }
          // dK += dS^T Q, dQ = dS K, the next dP^T over that dS^T, while the math warps take the next
          // exponentials
          ok = mbar_wait(&s.ds_ready, par, abort_flag, p.status, STATUS_TIMEOUT_SOFTMAX) &&
               (!new_map || mbar_wait(&s.dk_free, 0, abort_flag, p.status, STATUS_TIMEOUT_SOFTMAX));
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int ks = 0; ks < T / 16; ++ks)
            mma_ts(tmem + C_DK, tmem + C_DP + step_col(ks), sdesc_mnmajor(qa + ks * 2048, PANEL), id_dk,
                   !((i == 0 || new_map) && ks == 0));
          tc_commit(&s.q_empty[st]);
          if (i > 0) {
            ok = mbar_wait(&s.dq_free, par ^ 1, abort_flag, p.status, STATUS_TIMEOUT_SOFTMAX);
            if (!ok) break;
            tc_fence_after();
          }
          const uint32_t a = ka + map_of(i) * PANEL;
#pragma unroll
          for (int ks = 0; ks < T / 16; ++ks)
            mma_ss(tmem + C_DQ, sdesc_mnmajor(dsa + ks * 2048, PANEL), sdesc_mnmajor(a + ks * 2048, PANEL), id_dq, ks != 0);
          tc_commit(&s.dq_full);
          // behind dQ, so that dp_full also says that dS^T in shared memory has been read
          if (i + 1 < n) {
            ok = mbar_wait(&s.do_full[st ^ 1], nph, abort_flag, p.status, STATUS_TIMEOUT_TMA);
            if (!ok) break;
            tc_fence_after();
            issue_dp(i + 1);
          }
        }
        if (ok) tc_commit(&s.final_bar);
      }
    }
  } else if (warp >= 8) {
    // ------------------------------- dQ tiles -> global reduction; dK stores --
    asm volatile("setmaxnreg.dec.sync.aligned.u32 96;");
    const int wl = warp & 3;
    const int row = wl * 32 + lane;
    const uint32_t tb = tmem_addr(tmem, wl * 32, 0);
    const int kv_row = kvb * T + row;
    float* const part = split ? p.part + (size_t)(idx - p.n_whole) * PART : nullptr;
    // dK of a map from TMEM (or zeros, a map that this part has no step of)
    auto store_dk = [&](int m, bool zero) {
#pragma unroll 1
      for (int c = 0; c < HD; c += 32) {
        uint32_t r[32];
        tmem_ld32(tb + C_DK + c, r);
        tc_wait_ld();
        if (zero) {
#pragma unroll
          for (int e = 0; e < 32; ++e) r[e] = 0u;
        }
        if (kv_row >= p.L) {
        } else if (part) {
          uint4* dst = reinterpret_cast<uint4*>(part + ((size_t)m * T + row) * HD + c);
#pragma unroll
          for (int e = 0; e < 8; ++e) dst[e] = make_uint4(r[4 * e], r[4 * e + 1], r[4 * e + 2], r[4 * e + 3]);
        } else {
          uint4* dst = reinterpret_cast<uint4*>(p.dk + (int64_t)b * p.dk_sb + (int64_t)kv_row * p.dk_sl +
                                                (int64_t)(2 * h + m) * p.dk_sh + c);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint32_t o[4];
#pragma unroll
            for (int u = 0; u < 4; ++u)
              o[u] = pack_bf16(__uint_as_float(r[8 * e + 2 * u]) * p.scale, __uint_as_float(r[8 * e + 2 * u + 1]) * p.scale);
            dst[e] = make_uint4(o[0], o[1], o[2], o[3]);
          }
        }
      }
    };
    bool ok = true;
    bool turn_live = true;          // false once a turn wait gave up (the status word says so)
    for (int i = 0; i < n && ok; ++i) {
      ok = __all_sync(0xffffffffu, mbar_wait(&s.dq_full, (uint32_t)(i & 1), abort_flag, p.status,
                                             STATUS_TIMEOUT_MMA));
      if (!ok) break;
      tc_fence_after();
      uint32_t r[64];
      tmem_ld32(tb + C_DQ, r);
      tmem_ld32(tb + C_DQ + 32, r + 32);
      tc_wait_ld();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&s.dq_free);
      // Each warp adds its 32 rows for itself, 32 columns at a time, by TMA from shared memory to the fp32
      // accumulator (rows >= L clipped; a box that begins behind them is left out)
      const int r0 = tile_of(i) * T + wl * 32;
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        if (i > 0 || hf > 0) {
          if (lane == 0) {
            if (turn && turn_live && hf == 0) {
              // the previous tile's adds have been performed: pass its query rows on
              asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
              turn_pass(turn + (first + i - 1) * 4 + wl, kvb + 1);
            } else {
              asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
            }
          }
          __syncwarp();
        }
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          const int x = hf * 32 + 4 * c;
          *reinterpret_cast<uint4*>(s.dq_stage[wl] + lane * 128 + ((c ^ (lane & 7)) << 4)) =
              make_uint4(r[x], r[x + 1], r[x + 2], r[x + 3]);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          if (turn && turn_live && hf == 0) turn_live = turn_wait(turn + (first + i) * 4 + wl, kvb, abort_flag, p.status);
          if ((!turn || turn_live) && r0 < p.L)
            tma_reduce_add_4d(&tm_dq, s.dq_stage[wl], hf * 32, 2 * h + map_of(i), r0, b);
          asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        }
        __syncwarp();
      }
      // dQ of a map's last step is behind its last dK
      if (i + 1 == n || map_of(i + 1) != map_of(i)) {
        store_dk(map_of(i), false);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.dk_free);
      }
    }
    if (lane == 0) {
      asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
      if (turn && turn_live && ok && n > 0) turn_pass(turn + (first + n - 1) * 4 + wl, kvb + 1);
    }
    __syncwarp();
    if (part && ok) {
      if (map_of(0) == 1) store_dk(0, true);
      if (map_of(n - 1) == 0) store_dk(1, true);
    }
    tc_fence_before();
  } else {
    // ------------------------------------------------------ exp / dS math ----
    asm volatile("setmaxnreg.inc.sync.aligned.u32 168;");
    const int wg = warp >> 2;           // query columns [64 wg, 64 wg + 64)
    const int wl = warp & 3;
    const int row = wl * 32 + lane;     // kv row of this thread (TMEM lane)
    const uint32_t tb = tmem_addr(tmem, wl * 32, 0);
    const int kv_row = kvb * T + row;
    // rows behind the last key take no part: their score is zero, and exp(-lse) would be infinite from lse = -89
    // on, dQ infinity times a key of zeros
    const bool key = kv_row < p.L;
    const f32x2 to_exp = dup2(key ? p.scale * LOG2E : 0.f);
    const float w1 = key ? 1.f : 0.f, w2 = key ? -p.lam.at(h) : 0.f;
    bool ok = true;
    for (int i = 0; i < n && ok; ++i) {
      const uint32_t par = (uint32_t)(i & 1);
      ok = __all_sync(0xffffffffu, mbar_wait(&s.s_full, par, abort_flag, p.status, STATUS_TIMEOUT_MMA));
      if (!ok) break;
      tc_fence_after();
      uint32_t sv[64];                  // S - lse / scale, then P^T
      tmem_ld32(tb + C_S + wg * 64, sv);
      tmem_ld32(tb + C_S + wg * 64 + 32, sv + 32);
      tc_wait_ld();
      const f32x2 w = dup2(map_of(i) ? w2 : w1);
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        uint32_t pk[16];
#pragma unroll
        for (int c = 0; c < 32; c += 2) {
          const int cg = hh * 32 + c;
          const f32x2 x = mul2(pair2(sv[cg], sv[cg + 1]), to_exp);
          const f32x2 e = mul2(w, fma_pair(c / 2) ? ex2_fma2(x) : ex2_mufu2(x));
          sv[cg] = __float_as_uint(lo2(e));
          sv[cg + 1] = __float_as_uint(hi2(e));
          pk[c / 2] = pack_bf16(lo2(e), hi2(e));
        }
        tmem_st16(tb + C_S + wg * 64 + hh * 16, pk);
      }
      tc_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&s.p_ready);
      // dS^T = P^T .* (dP^T - delta), the bracket straight from the tensor core: to TMEM for dK and to shared
      // memory for dQ (dP^T was issued behind the dQ product of the previous step)
      ok = __all_sync(0xffffffffu, mbar_wait(&s.dp_full, par, abort_flag, p.status, STATUS_TIMEOUT_MMA));
      if (!ok) break;
      tc_fence_after();
      uint8_t* dsb = s.ds[wg] + row * 128;
      uint32_t dp[2][32];
      tmem_ld32(tb + C_DP + wg * 64, dp[0]);
      tc_wait_ld();
      tmem_ld32(tb + C_DP + wg * 64 + 32, dp[1]);
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        uint32_t dk_[16];
        if (hh == 1) tc_wait_ld();
#pragma unroll
        for (int c = 0; c < 32; c += 2) {
          const int cg = hh * 32 + c;
          const f32x2 d = mul2(pair2(sv[cg], sv[cg + 1]), pair2(dp[hh][c], dp[hh][c + 1]));
          dk_[c / 2] = pack_bf16(lo2(d), hi2(d));
        }
        tmem_st16(tb + C_DP + wg * 64 + hh * 16, dk_);     // (columns that hh = 0 has read)
#pragma unroll
        for (int cc = 0; cc < 4; ++cc) {
          const int chunk = hh * 4 + cc;
          uint4 val = make_uint4(dk_[4 * cc], dk_[4 * cc + 1], dk_[4 * cc + 2], dk_[4 * cc + 3]);
          *reinterpret_cast<uint4*>(dsb + ((chunk ^ (row & 7)) << 4)) = val;
        }
      }
      tc_wait_st();
      fence_proxy_async_smem();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&s.ds_ready);
    }
    // ---- epilogue: group wg stores the dV of head 2h + wg ----
    if (ok && n > 0) ok = mbar_wait(&s.final_bar, 0, abort_flag, p.status, STATUS_TIMEOUT_MMA);
    ok = __all_sync(0xffffffffu, ok);
    if (ok && n > 0) {
      tc_fence_after();
#pragma unroll 1
      for (int c = 0; c < VD / 2; c += 32) {
        uint32_t r[32];
        tmem_ld32(tb + C_DV + wg * (VD / 2) + c, r);
        tc_wait_ld();
        if (kv_row >= p.L) {
        } else if (split) {
          uint4* dst = reinterpret_cast<uint4*>(p.part + (size_t)(idx - p.n_whole) * PART + (size_t)2 * T * HD +
                                                (size_t)row * VD + wg * (VD / 2) + c);
#pragma unroll
          for (int e = 0; e < 8; ++e) dst[e] = make_uint4(r[4 * e], r[4 * e + 1], r[4 * e + 2], r[4 * e + 3]);
        } else {
          uint4* dst = reinterpret_cast<uint4*>(p.dv + (int64_t)b * p.dv_sb + (int64_t)kv_row * p.dv_sl +
                                                (int64_t)(2 * h + wg) * p.dv_sh + c);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint32_t o[4];
#pragma unroll
            for (int u = 0; u < 4; ++u)
              o[u] = pack_bf16(__uint_as_float(r[8 * e + 2 * u]), __uint_as_float(r[8 * e + 2 * u + 1]));
            dst[e] = make_uint4(o[0], o[1], o[2], o[3]);
          }
        }
      }
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == 12) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Per (b, l, pair), 16 lanes of 8 channels: the bands of both maps (padding rows: the exponent -30000, so
// P = 0), delta_2 for dlam, and zeros for the dQ additions.
__global__ void attn_diff_bwd_prep_kernel(const __nv_bfloat16* __restrict__ o, const __nv_bfloat16* __restrict__ o2,
                                          const uint8_t* __restrict__ low,
                                          const __nv_bfloat16* __restrict__ d_o, const float* __restrict__ lse,
                                          const DiffWeights lam, uint4* __restrict__ band, float* __restrict__ delta2,
                                          float* __restrict__ dq_acc, int B, int L, int H, int Lp, int64_t o_sb,
                                          int64_t o_sl, int64_t o_sh, int64_t g_sb, int64_t g_sl, int64_t g_sh,
                                          float inv_exp_scale) {
  const int lane = threadIdx.x & 31, part = lane & 15, c = (part & 7) * 8;
  const long u = (((long)blockIdx.x * blockDim.x + threadIdx.x) >> 5) * 2 + (lane >> 4);
  const bool in = u < (long)B * H * Lp;          // no early exit: the shuffles below need every lane
  int h = 0, l = 0, b = 0;
  if (in) {
    h = (int)(u % H);
    l = (int)((u / H) % Lp);
    b = (int)(u / ((long)H * Lp));
  }
  const bool live = in && l < L;
  const int head = 2 * h + (part >> 3);
  float d = 0.f, d2 = 0.f;
  if (live) {
    const int64_t at = b * o_sb + l * o_sl + head * o_sh + c;
    const uint4 g = *reinterpret_cast<const uint4*>(d_o + b * g_sb + l * g_sl + head * g_sh + c);
    const uint32_t gw[4] = {g.x, g.y, g.z, g.w};
    float x[8], y[8];
    const uint4 lo = *reinterpret_cast<const uint4*>(low + 2 * at);
    diff_join8(*reinterpret_cast<const uint4*>(o + at), make_uint2(lo.x, lo.y), x);
    diff_join8(*reinterpret_cast<const uint4*>(o2 + at), make_uint2(lo.z, lo.w), y);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float ge = (i & 1) ? bf16_hi(gw[i / 2]) : bf16_lo(gw[i / 2]);
      d = fmaf(x[i], ge, d);
      d2 = fmaf(y[i], ge, d2);
    }
    float4* acc = reinterpret_cast<float4*>(dq_acc + (((int64_t)b * L + l) * 2 * H + head) * HD + c);
    acc[0] = acc[1] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
#pragma unroll
  for (int off = 8; off > 0; off >>= 1) {
    d += __shfl_xor_sync(0xffffffffu, d, off);
    d2 += __shfl_xor_sync(0xffffffffu, d2, off);
  }
  if (!in || part >= 2) return;
  const long row = ((long)b * 2 * H + 2 * h + part) * Lp + l;
  float x = live ? lse[((long)b * 2 * H + 2 * h + part) * L + l] * LOG2E : 0.f;
  // (infinities become what is still finite over the smallest scale, 1e-30; NaN stays)
  if (x == x) x = fminf(fmaxf(x, -1e8f), 1e8f);
  x = -(live ? x : 30000.f) * inv_exp_scale;
  const float y = live ? -(part ? d2 : fmaf(lam.at(h), d2, d)) : 0.f;
  const float x1 = bf16_lo(pack_bf16(x, 0.f)), x2 = bf16_lo(pack_bf16(x - x1, 0.f));
  const float y1 = bf16_lo(pack_bf16(y, 0.f)), y2 = bf16_lo(pack_bf16(y - y1, 0.f));
  band[2 * row] = make_uint4(pack_bf16(x1, x2), pack_bf16(x - x1 - x2, y1), pack_bf16(y2, y - y1 - y2), 0u);
  band[2 * row + 1] = make_uint4(0u, 0u, 0u, 0u);
  if (part) delta2[((long)b * H + h) * Lp + l] = d2;
}

// dK_m = scale * sum_r part[r].dK_m, dV = sum_r part[r].dV (fixed order) of the split K/V tiles.  One
// thread (i) per 4 channels of a row.
IMF_DEVICE void combine4(const Params& p, int i) {
  constexpr int TILE4 = (int)(PART / 4);
  const int t = i / TILE4, e = (i % TILE4) * 4;           // e: first float of the thread in a partial result
  const bool is_dk = e < 2 * T * HD;
  const int e2 = is_dk ? e : e - 2 * T * HD;
  const int row = is_dk ? (e2 / HD) % T : e2 / VD;
  const int c = is_dk ? e2 % HD : e2 % VD;                // channel; dV: of both heads
  int chain, kv_ord;
  bwd_item(p.n_whole + t, p.B * p.H, p.n_t, p.group, chain, kv_ord);
  const int h = chain % p.H, b = chain / p.H;
  const int kv_row = kv_ord * T + row;
  if (kv_row >= p.L) return;
  const float* src = p.part + (size_t)t * p.parts * PART + e;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int r = 0; r < p.parts; ++r) {
    const float4 x = *reinterpret_cast<const float4*>(src + (size_t)r * PART);
    a.x += x.x; a.y += x.y; a.z += x.z; a.w += x.w;
  }
  const float mul = is_dk ? p.scale : 1.f;
  const int head = 2 * h + (is_dk ? e2 / (T * HD) : c / HD);
  __nv_bfloat16* dst = is_dk ? p.dk + (int64_t)b * p.dk_sb + (int64_t)kv_row * p.dk_sl + (int64_t)head * p.dk_sh
                             : p.dv + (int64_t)b * p.dv_sb + (int64_t)kv_row * p.dv_sl + (int64_t)head * p.dv_sh;
  *reinterpret_cast<uint2*>(dst + c % HD) = make_uint2(pack_bf16(a.x * mul, a.y * mul), pack_bf16(a.z * mul, a.w * mul));
}

// What is left when the sums are there, in one launch, longest first: in H blocks dlam = -sum of delta_2, in a fixed
// order; in n_merge the split K/V tiles; then dq = bf16(acc * scale).
__global__ void __launch_bounds__(256)
attn_diff_bwd_post_kernel(const float* __restrict__ acc, __nv_bfloat16* __restrict__ dq, long n4, float scale,
                          const float* __restrict__ delta2, void* dlam, int dlam_bf16, int B, int H, int L, int Lp,
                          int n_merge, const Params p) {
  const int h = (int)blockIdx.x;
  if (h >= H) {
    if (h < H + n_merge) {
      combine4(p, (h - H) * 256 + threadIdx.x);
      return;
    }
    const long i = (long)(h - H - n_merge) * 256 + threadIdx.x;
    if (i >= n4) return;
    const float4 v = reinterpret_cast<const float4*>(acc)[i];
    reinterpret_cast<uint2*>(dq)[i] = make_uint2(pack_bf16(v.x * scale, v.y * scale), pack_bf16(v.z * scale, v.w * scale));
    return;
  }
  __shared__ double sum[256];
  double t = 0.0;
  for (int b = 0; b < B; ++b) {
    const float* d = delta2 + ((long)b * H + h) * Lp;
#pragma unroll 8
    for (int l = threadIdx.x; l < L; l += 256) t += d[l];
  }
  sum[threadIdx.x] = t;
  for (int k = 128; k > 0; k >>= 1) {
    __syncthreads();
    if (threadIdx.x < k) sum[threadIdx.x] += sum[threadIdx.x + k];
  }
  if (threadIdx.x == 0) {
    if (dlam_bf16)
      static_cast<__nv_bfloat16*>(dlam)[h] = __double2bfloat16(-sum[0]);
    else
      static_cast<float*>(dlam)[h] = (float)-sum[0];
  }
}

static int make_map(CUtensorMap* m, const void* ptr, int B, int L, int heads, const int64_t* st) {
  uint64_t dims[4] = {(uint64_t)HD, (uint64_t)heads, (uint64_t)L, (uint64_t)B};
  uint64_t str[4] = {2, (uint64_t)st[2] * 2, (uint64_t)st[1] * 2, (uint64_t)st[0] * 2};
  uint32_t box[4] = {(uint32_t)HD, 1, (uint32_t)T, 1};
  return make_tmap(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(ptr), dims, str, box);
}

// Where the parts of the scratch begin, in bytes, and its whole size.
struct Layout {
  size_t turn, turn_bytes, band, delta2, part, all;
};
static Layout layout(int B, int L, int H, const BwdSplit& sp) {
  const size_t Lp = (size_t)(L + T - 1) / T * T;
  auto up = [](size_t x) { return (x + 255) & ~size_t(255); };
  Layout y;
  y.turn = up((size_t)B * L * 2 * H * HD * 4);                // fp32 dQ first
  y.turn_bytes = up((size_t)B * 2 * H * (Lp / 32) * 4);
  y.band = y.turn + y.turn_bytes;
  y.delta2 = y.band + up((size_t)B * 2 * H * Lp * 32);
  y.part = y.delta2 + up((size_t)B * H * Lp * 4);
  y.all = y.part + (size_t)sp.n_split * sp.parts * PART * 4;
  return y;
}

// A CTA's start, pipeline fill and epilogue cost about 2.5 of its steps (128 query rows of one map).
static BwdSplit split_for(int B, int L, int H) {
  const int n_t = (L + T - 1) / T;
  return bwd_split((long)n_t * H * B, 2 * n_t, bwd_sm_count(), 2.5f);
}

}  // namespace diffb
}  // namespace imf

extern "C" long imf_attn_diff_bwd_scratch_bytes(int B, int L, int H) {
  using namespace imf::diffb;
  if (B <= 0 || L <= 0 || H <= 0 || (long)B * H * ((L + T - 1) / T) > 0x3fffffffL) return 0;
  return (long)layout(B, L, H, split_for(B, L, H)).all;
}

// q, k, v, d_o: (B, L, 2H, 64) bf16, (batch, row, head) element strides in strides[0..11]; o, o2 and their low
// bytes and lse as imf_attn_diff_fwd wrote them; dq contiguous, dk and dv with strides of their own;
// dlam: H values, in the type of lam.  All with 16-byte aligned rows.
extern "C" int imf_attn_diff_bwd(const void* q, const void* k, const void* v, const void* o, const void* o2,
                                 const void* low, const void* d_o, const float* lse, const void* lam,
                                 int64_t lam_stride, int lam_bf16, void* dq, void* dk, void* dv, void* dlam, int B,
                                 int L, int H, const int64_t* strides,
                                 const int64_t* o_strides, const int64_t* dk_strides, const int64_t* dv_strides,
                                 float scale, void* scratch, long scratch_bytes, int fixed_order, int* status,
                                 void* stream) {
  using namespace imf;
  using namespace imf::diffb;
  for (const void* x : {q, k, v, o, o2, low, d_o, (const void*)lse, lam, (const void*)dq, (const void*)dk, (const void*)dv,
                        (const void*)dlam})
    if (!x) return IMF_ERR_ARG;
  if (B <= 0 || L <= 0 || H <= 0 || !(scale > 0.f) || scale > 1e30f) return IMF_ERR_ARG;
  if ((long)B * H * ((L + T - 1) / T) > 0x3fffffffL) return IMF_ERR_TOO_LARGE;
  const BwdSplit sp = split_for(B, L, H);
  const Layout y = layout(B, L, H, sp);
  if (scratch == nullptr || scratch_bytes < (long)y.all || (reinterpret_cast<uintptr_t>(scratch) & 255)) return IMF_ERR_ARG;
  for (const void* x : {q, k, v, o, o2, low, d_o, (const void*)dq, (const void*)dk, (const void*)dv})
    if (reinterpret_cast<uintptr_t>(x) & 15) return IMF_ERR_ARG;
  for (int i = 0; i < 3; ++i)
    if ((dk_strides[i] & 7) || (dv_strides[i] & 7) || (o_strides[i] & 7) || (strides[9 + i] & 7))
      return IMF_ERR_ARG;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  uint8_t* base = static_cast<uint8_t*>(scratch);
  const int Lp = (L + T - 1) / T * T;
  float* dq_acc = reinterpret_cast<float*>(base);
  uint4* band = reinterpret_cast<uint4*>(base + y.band);
  float* delta2 = reinterpret_cast<float*>(base + y.delta2);
  const bool ordered = fixed_order && status != nullptr;
  if (ordered && cudaMemsetAsync(base + y.turn, 0, y.turn_bytes, st) != cudaSuccess) return IMF_ERR_LAUNCH;
  const DiffWeights w{lam, lam_stride, lam_bf16};
  typedef const __nv_bfloat16 cbf;
  const long threads = (long)B * H * Lp * 16;
  attn_diff_bwd_prep_kernel<<<(unsigned)((threads + 255) / 256), 256, 0, st>>>(
      static_cast<cbf*>(o), static_cast<cbf*>(o2), static_cast<const uint8_t*>(low), static_cast<cbf*>(d_o), lse, w,
      band, delta2, dq_acc, B, L, H, Lp, o_strides[0], o_strides[1], o_strides[2], strides[9], strides[10], strides[11],
      1.f / (scale * LOG2E));
  if (cudaGetLastError() != cudaSuccess) return IMF_ERR_LAUNCH;
  CUtensorMap mq, mk, mv, mdo, mdq, mb;
  int rc;
  if ((rc = make_map(&mq, q, B, L, 2 * H, strides))) return rc;
  if ((rc = make_map(&mk, k, B, L, 2 * H, strides + 3))) return rc;
  if ((rc = make_map(&mv, v, B, L, 2 * H, strides + 6))) return rc;
  if ((rc = make_map(&mdo, d_o, B, L, 2 * H, strides + 9))) return rc;
  {
    const uint64_t row = (uint64_t)2 * H * HD * 4;
    uint64_t dims[4] = {(uint64_t)HD, (uint64_t)2 * H, (uint64_t)L, (uint64_t)B};
    uint64_t str[4] = {4, (uint64_t)HD * 4, row, row * L};
    uint32_t box[4] = {32, 1, 32, 1};
    if ((rc = make_tmap(&mdq, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, dq_acc, dims, str, box))) return rc;
  }
  {
    uint64_t dims[3] = {16, (uint64_t)Lp, (uint64_t)B * 2 * H};
    uint64_t str[3] = {2, 32, (uint64_t)Lp * 32};
    uint32_t box[3] = {16, (uint32_t)T, 1};
    if ((rc = make_tmap(&mb, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, band, dims, str, box, CU_TENSOR_MAP_SWIZZLE_32B)))
      return rc;
  }
  Params prm;
  prm.lam = w;
  prm.dk = static_cast<__nv_bfloat16*>(dk);
  prm.dv = static_cast<__nv_bfloat16*>(dv);
  prm.B = B; prm.H = H; prm.L = L; prm.Lp = Lp;
  prm.dk_sb = dk_strides[0]; prm.dk_sl = dk_strides[1]; prm.dk_sh = dk_strides[2];
  prm.dv_sb = dv_strides[0]; prm.dv_sl = dv_strides[1]; prm.dv_sh = dv_strides[2];
  prm.scale = scale;
  prm.status = status;
  prm.n_t = (L + T - 1) / T;
  // a walk reads 64 channels of Q and 128 of dO and adds to 64 of dQ: 640 bytes a row, 8 for each of 80 channels
  prm.group = bwd_group(B * H, L, 80, ordered);
  prm.n_whole = sp.n_whole;
  prm.parts = sp.parts;
  prm.part = sp.n_split ? reinterpret_cast<float*>(base + y.part) : nullptr;
  prm.turn = ordered ? reinterpret_cast<int*>(base + y.turn) : nullptr;
  static bool smem_set[HOST_MAX_DEVICES] = {false};
  if (!allow_smem((const void*)attn_diff_bwd_kernel, sizeof(Smem), smem_set)) return IMF_ERR_LAUNCH;
  attn_diff_bwd_kernel<<<sp.ctas(), THREADS, sizeof(Smem), st>>>(mq, mk, mv, mdo, mdq, mb, prm);
  if (cudaGetLastError() != cudaSuccess) return IMF_ERR_LAUNCH;
  const long n4 = (long)B * L * 2 * H * HD / 4;
  const int n_merge = (int)(sp.n_split * (PART / 4 / 256));
  attn_diff_bwd_post_kernel<<<(unsigned)(H + n_merge + (n4 + 255) / 256), 256, 0, st>>>(
      dq_acc, static_cast<__nv_bfloat16*>(dq), n4, scale, delta2, dlam, lam_bf16, B, H, L, Lp, n_merge, prm);
  return cudaGetLastError() == cudaSuccess ? IMF_OK : IMF_ERR_LAUNCH;
}
