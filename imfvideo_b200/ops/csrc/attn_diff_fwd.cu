// Differential attention forward on tcgen05 / TMEM, primal and fused forward-mode tangent
// (see attn_diff.h for the pairing of heads):
//
//   S_m = Q_m K_m^T * scale,  A_m = softmax(S_m),  O_m = A_m V,  o = O_1 - lam O_2
//   dS_m = (dQ_m K_m^T + Q_m dK_m^T) * scale,  T_m = A_m .* (dS_m - rowsum(A_m dS_m)),
//   do = (T_1 V + A_1 dV) - lam (T_2 V + A_2 dV)
//
// Each map is a flash attention of its own, q and k 64 wide and V 128, with its own running maximum
// and sum; what they share is V.  O_1 and O_2 are divided and subtracted in 32 bits and rounded once.
//
// TMEM (512 columns of fp32 per SM) decides the shapes:
//   primal  : an item is 128 query rows of a pair.  Each map has O (128) and two buffers of S (64) with P
//             over it, so K_1, K_2 and V are read once for both maps, and the epilogue reads both O (the
//             warps of a lane quadrant see its lanes in every column).
//   tangent : O | dO of one map (256) and two S | dS buffers leave no room for the other map.  A segment
//             runs map 1, then map 2, over the same K/V tiles; map 1's finished rows wait in global
//             memory (128 KB a CTA, in L2) and come back to the thread that wrote them.
// Scheduling, shares and records of split items are those of attn_fwd_split.h, with a record for each
// map; the kernel that merges the parts also subtracts.
//
// Roundings: P and P .* dS go to the tensor core in bf16 (each off by at most 2^-8 of its value,
// independently from key to key), o and do are rounded once; scores, maxima, sums and both O are in 32 bits.
//
// Measured, 1 x 29,140 rows, 2 pairs: primal 1.13 to 1.30 ms, 1,000 to 1,150 TFLOP/s; with tangent 2.61 to 2.74 ms alone and
// 2.85 to 3.09 in a loop under the power cap, 1,430 to 1,500 and 1,270 to 1,370.  1 x 7,820 rows, 8 pairs: 343 to 375
// and 850 to 910 us.
// Primal: the exponential unit sets the pace (72 % busy, the tensor pipe 53 %); a sixteenth of the
// exponentials on the FMA units takes registers that are not there (371 -> 404 us).  Four groups of softmax warps, by
// map and parity of the step, against two: 427 -> 371.  Tangent: the tensor pipe is 76 % busy, the rest the
// chain from scores to products at a segment's ends and between steps.
#include "attn_diff.h"
#include "attn_fwd_split.h"
#include "common.cuh"
#include "host_util.h"

#include <math.h>

namespace imf {
namespace diff {

constexpr int HD = 64;               // channels of a query or key
constexpr int VD = 128;              // channels of a pair's values
constexpr int TM = 128;              // query rows per item
constexpr int BN = 64;               // K/V rows per tile
constexpr int QPANEL = TM * 128;     // bytes of a query tile (64 columns)
constexpr int KPANEL = BN * 128;     // bytes of 64 columns of a K/V tile
constexpr int SOFT_WARPS = 8;
constexpr int WARP_MMA = 8, WARP_TMA = 9;
constexpr int THREADS = 12 * 32;
constexpr int REG_SOFT = 216, REG_OTHER = 72, REG_LAUNCH = 168;
static_assert(SOFT_WARPS * 32 * REG_SOFT + (THREADS - SOFT_WARPS * 32) * REG_OTHER <= THREADS * REG_LAUNCH,
              "register pool exceeded");
constexpr float LOG2E = 1.4426950408889634f;

// A record of a partial segment, for each map: accumulators [column][row] (o, then do), m of the scaled
// scores, l, mu.
template <bool TANGENT>
struct Rec {
  static constexpr int ACC = TANGENT ? 2 * VD : VD;
  static constexpr int STATS = ACC * TM;
  static constexpr size_t MAP = (size_t)TM * (ACC + 3), ALL = 2 * MAP;
};
constexpr size_t HOLD = (size_t)TM * 2 * VD;      // floats a CTA holds of map 1 (tangent)

struct Params {
  __nv_bfloat16 *o, *dout, *o2;      // o2: O_2 for the backward pass, or null
  int8_t* low;                       // what bf16 dropped of eight channels of o, then of the same of o2; null with o2
  float* lse;                        // (B, 2H, L) or null
  float* scratch;                    // records of split items
  float* hold;                       // tangent: the held rows of map 1, HOLD a CTA
  DiffWeights lam;
  int B, H, L;                       // H pairs
  int n_qblk;
  FwdShares sh;
  int64_t o_sb, o_sl, o_sh;          // o, dout and o2
  float scale;
  int* status;
};

IMF_DEVICE void item_coords(const Params& p, int item, int& q0, int& h, int& b) {
  q0 = (item % p.n_qblk) * TM;
  h = (item / p.n_qblk) % p.H;
  b = item / (p.n_qblk * p.H);
}

// Eight channels of o and, where they are kept, of O_2 (z) at element `at`, with the bytes that both lost.
IMF_DEVICE void store_out8(const Params& p, int64_t at, const float* y, const float* z) {
  uint4 hi;
  uint2 ly, lz;
  diff_split8(y, hi, ly);
  *reinterpret_cast<uint4*>(p.o + at) = hi;
  if (!p.o2) return;
  diff_split8(z, hi, lz);
  *reinterpret_cast<uint4*>(p.o2 + at) = hi;
  *reinterpret_cast<uint4*>(p.low + 2 * at) = make_uint4(ly.x, ly.y, lz.x, lz.y);
}

// The row's reference maximum as step `n` of its map left it goes to the warp of the other group in one
// 64-bit word, the step's number in its upper half.  One scalar access each way: a vector of two words is
// two accesses in no order, and the number could be seen before the maximum that it stands for.
IMF_DEVICE uint64_t ref_word(float m, int n) { return (uint64_t)(uint32_t)n << 32 | __float_as_uint(m); }
IMF_DEVICE void publish_ref(uint64_t* addr, float m, int n) {
  asm volatile("st.volatile.shared.b64 [%0], %1;" ::"r"(smem_u32(addr)), "l"(ref_word(m, n)) : "memory");
}
// From the other group's warp, which decided long before as a rule.  Bounded; false: gave up.
IMF_DEVICE bool ref_of_step(const uint64_t* addr, int n, float& m, volatile int* abort_flag, int* status) {
  uint64_t t0 = 0;
  for (uint32_t spins = 1;; ++spins) {
    uint64_t word;
    asm volatile("ld.volatile.shared.b64 %0, [%1];" : "=l"(word) : "r"(smem_u32(addr)) : "memory");
    m = __uint_as_float((uint32_t)word);
    if (__all_sync(0xffffffffu, (int)(word >> 32) >= n)) return true;
    if ((spins & 63u) == 0) {
      if (__any_sync(0xffffffffu, *abort_flag)) return false;
      const uint64_t now = globaltimer_ns();
      if (t0 == 0) t0 = now;
      if (__any_sync(0xffffffffu, now - t0 > IMF_WAIT_LIMIT_NS)) {
        *abort_flag = 1;
        if (status) atomicCAS(status, 0, STATUS_TIMEOUT_SOFTMAX);
        return false;
      }
    }
  }
}

// ------------------------------------------------------------------ primal ---
constexpr int P_STAGES = 4;
constexpr int P_SOFT_WARPS = 16;       // by map and parity of the step, four each
constexpr int P_WARP_MMA = 16, P_WARP_TMA = 18;        // a warp that issues products for either map; loads
constexpr int P_THREADS = 20 * 32;
// setmaxnreg.inc draws from what the CTA was launched with; a request beyond that pool blocks for ever
constexpr int P_REG_SOFT = 104, P_REG_OTHER = 64, P_REG_LAUNCH = 96;
static_assert(P_SOFT_WARPS * 32 * P_REG_SOFT + (P_THREADS - P_SOFT_WARPS * 32) * P_REG_OTHER <= P_THREADS * P_REG_LAUNCH,
              "register pool exceeded");
// TMEM columns of a map: O, then S of even and of odd steps, P over the S that it is made from
constexpr int P_MAP = 256, P_COL_O = 0;
__host__ __device__ constexpr int p_col_s(int g) { return VD + g * BN; }
static_assert(p_col_s(2) <= P_MAP, "TMEM budget");

struct PSmem {
  alignas(1024) uint8_t q[2][2][QPANEL];             // of two segments: Q_1, Q_2
  alignas(1024) uint8_t k[P_STAGES][2][KPANEL];      // K_1, K_2
  alignas(1024) uint8_t v[P_STAGES][2][KPANEL];      // the two halves of V
  uint64_t m_ref[2][TM];       // by map: reference maximum of the row as of the last step decided | that step's number
  // of two segments (a group without a step in the next one may be there already), by map and group: l and
  // reference maximum at the segment's end
  float xst[2][2][2][2][TM];
  uint64_t q_full[2], q_empty[2];
  uint64_t k_full[P_STAGES], k_empty[P_STAGES];
  uint64_t v_full[P_STAGES], v_empty[P_STAGES];
  uint64_t s_full[2][2], p_full[2][2], o_done[2][2];   // by map and group
  uint64_t o_final[2];         // the last P V of a segment (one phase per segment, never skipped)
  uint64_t o_free, sums;
  uint32_t tmem_base;
  int abort_flag;
};

__global__ void __launch_bounds__(P_THREADS, 1)
attn_diff_fwd_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                     const __grid_constant__ CUtensorMap tm_v, const Params p) {
  extern __shared__ uint8_t smem_raw[];
  auto& s = *reinterpret_cast<PSmem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int cta = blockIdx.x, G = gridDim.x;

  if (threadIdx.x == 0) {
    for (int i = 0; i < P_STAGES; ++i) {
      mbar_init(&s.k_full[i], 1);
      mbar_init(&s.k_empty[i], 2);         // read for either map
      mbar_init(&s.v_full[i], 1);
      mbar_init(&s.v_empty[i], 2);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&s.q_full[t], 1);
      mbar_init(&s.q_empty[t], 2);
      for (int g = 0; g < 2; ++g) {
        mbar_init(&s.s_full[t][g], 1);
        mbar_init(&s.p_full[t][g], 4);
        mbar_init(&s.o_done[t][g], 1);
      }
      mbar_init(&s.o_final[t], 1);
    }
    mbar_init(&s.o_free, P_SOFT_WARPS);
    mbar_init(&s.sums, P_SOFT_WARPS);
    s.abort_flag = 0;
    fence_barrier_init();
  }
  if (threadIdx.x < 2 * TM) s.m_ref[threadIdx.x / TM][threadIdx.x % TM] = ref_word(0.f, -1);
  if (warp == P_WARP_MMA) {
    tmem_alloc(&s.tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s.tmem_base;
  volatile int* abort_flag = &s.abort_flag;

  if (warp >= P_SOFT_WARPS) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(P_REG_OTHER));
    if (warp == P_WARP_TMA) {
      // ------------------------------------------------------ TMA producer --
      if (elect_one()) {
        prefetch_tmap(&tm_q);
        prefetch_tmap(&tm_k);
        prefetch_tmap(&tm_v);
        int st = 0;
        uint32_t par = 1;                    // an "empty" wait passes in the first round of a ring
        Segment sg;
        bool ok = true;
        for (int si = 0; ok && get_segment(p.sh, cta, G, si, sg); ++si) {
          int q0, h, b;
          item_coords(p, sg.item, q0, h, b);
          const int qs = si & 1;
          ok = mbar_wait(&s.q_empty[qs], (uint32_t)((si >> 1) & 1) ^ 1, abort_flag, p.status, STATUS_TIMEOUT_EMPTY);
          if (!ok) break;
          mbar_arrive_expect_tx(&s.q_full[qs], 2 * QPANEL);
          for (int m = 0; m < 2; ++m) tma_load_4d(s.q[qs][m], &tm_q, &s.q_full[qs], 0, 2 * h + m, q0, b);
          for (int j = sg.j0; j < sg.j1; ++j) {
            ok = mbar_wait(&s.k_empty[st], par, abort_flag, p.status, STATUS_TIMEOUT_EMPTY);
            if (!ok) break;
            mbar_arrive_expect_tx(&s.k_full[st], 2 * KPANEL);
            for (int m = 0; m < 2; ++m) tma_load_4d(s.k[st][m], &tm_k, &s.k_full[st], 0, 2 * h + m, j * BN, b);
            ok = mbar_wait(&s.v_empty[st], par, abort_flag, p.status, STATUS_TIMEOUT_EMPTY);
            if (!ok) break;
            mbar_arrive_expect_tx(&s.v_full[st], 2 * KPANEL);
            for (int m = 0; m < 2; ++m) tma_load_4d(s.v[st][m], &tm_v, &s.v_full[st], 0, 2 * h + m, j * BN, b);
            if (++st == P_STAGES) {
              st = 0;
              par ^= 1;
            }
          }
        }
      }
    } else if (warp < P_WARP_TMA) {
      // ------------------------------------------- MMA issuer of a map --
      // scores of step n + 2 right behind P V of step n, whose P they overwrite
      const int t = warp - P_WARP_MMA;
      if (elect_one()) {
        constexpr uint32_t idesc_qk = idesc_bf16(TM, BN, 0, 0);
        constexpr uint32_t idesc_pv = idesc_bf16(TM, VD, 0, 1);
        const uint64_t q_desc = sdesc_kmajor(smem_u32(s.q[0][t])), k_desc = sdesc_kmajor(smem_u32(s.k[0][t]));
        const uint64_t v_desc = sdesc_mnmajor(smem_u32(s.v[0][0]), KPANEL);
        const uint32_t tb = tmem + t * P_MAP;
        int kst = 0, kg = 0, vst = 0, vg = 0;
        uint32_t kpar = 0, vpar = 0, ppar = 0;
        Segment sg;
        bool ok = true;
        for (int si = 0; ok && get_segment(p.sh, cta, G, si, sg); ++si) {
          const int n_j = sg.j1 - sg.j0, qs = si & 1;
          ok = mbar_wait(&s.q_full[qs], (uint32_t)((si >> 1) & 1), abort_flag, p.status, STATUS_TIMEOUT_TMA);
          const uint64_t qd = q_desc + (uint32_t)(qs * (2 * QPANEL >> 4));
          auto scores = [&](int jj) {
            if (!mbar_wait(&s.k_full[kst], kpar, abort_flag, p.status, STATUS_TIMEOUT_TMA)) return false;
            tc_fence_after();
            const uint64_t kd = k_desc + (uint32_t)(kst * (2 * KPANEL >> 4));
#pragma unroll
            for (int ks = 0; ks < HD / 16; ++ks)
              mma_ss(tb + p_col_s(kg), qd + ks * 2, kd + ks * 2, idesc_qk, ks != 0);
            tc_commit(&s.s_full[t][kg]);
            tc_commit(&s.k_empty[kst]);
            if (jj + 1 == n_j) tc_commit(&s.q_empty[qs]);
            if (++kst == P_STAGES) {
              kst = 0;
              kpar ^= 1;
            }
            kg ^= 1;
            return true;
          };
          ok = ok && scores(0) && (n_j == 1 || scores(1));
          if (ok && si > 0)        // epilogue of the previous segment has drained both O
            ok = mbar_wait(&s.o_free, (uint32_t)((si - 1) & 1), abort_flag, p.status, STATUS_TIMEOUT_SOFTMAX);
          for (int jj = 0; jj < n_j && ok; ++jj) {
            ok = mbar_wait(&s.v_full[vst], vpar, abort_flag, p.status, STATUS_TIMEOUT_TMA) &&
                 mbar_wait(&s.p_full[t][vg], ppar, abort_flag, p.status, STATUS_TIMEOUT_SOFTMAX);
            if (!ok) break;
            tc_fence_after();
            const uint64_t vd = v_desc + (uint32_t)(vst * (2 * KPANEL >> 4));
#pragma unroll
            for (int ks = 0; ks < BN / 16; ++ks)
              mma_ts(tb + P_COL_O, tb + p_col_s(vg) + ks * 8, vd + 128 * ks, idesc_pv, !(jj == 0 && ks == 0));
            tc_commit(&s.o_done[t][vg]);
            tc_commit(&s.v_empty[vst]);
            if (jj + 1 == n_j) tc_commit(&s.o_final[t]);
            if (++vst == P_STAGES) {
              vst = 0;
              vpar ^= 1;
            }
            vg ^= 1;
            if (vg == 0) ppar ^= 1;
            if (jj + 2 < n_j) ok = scores(jj + 2);
          }
        }
      }
    }
  } else {
    // --------------------------------------- softmax / correction / epilogue --
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(P_REG_SOFT));
    // Group g of map t takes the steps (K/V tiles) of parity g.  The row's reference maximum goes from one
    // group of a map to the other before the exponentials, as in the tangent kernel below.
    const int t = warp >> 3, g = (warp >> 2) & 1, wl = warp & 3;
    const int row = wl * 32 + lane;
    const uint32_t tq = tmem_addr(tmem, wl * 32, 0), tb = tq + t * P_MAP, sc = tb + p_col_s(g);
    const float scale_log2 = p.scale * LOG2E;
    uint32_t par = 0;                               // phase of this group's buffer
    int n0 = 0;                                     // number of the segment's first step
    Segment sg;
    bool ok = true;
    for (int si = 0; ok && get_segment(p.sh, cta, G, si, sg); ++si) {
      float m_used = -INFINITY, l_sum = 0.f, l_sum2 = 0.f;
      const int j_own = sg.j0 + ((n0 ^ g) & 1);     // this group's first step of the segment
      for (int j = j_own; j < sg.j1 && ok; j += 2) {
        const int n = n0 + j - sg.j0;
        // (the O product of this group's step before first, as in the tangent kernel below)
        ok = mbar_wait(&s.o_done[t][g], par ^ 1, abort_flag, p.status, STATUS_TIMEOUT_MMA) &&
             mbar_wait(&s.s_full[t][g], par, abort_flag, p.status, STATUS_TIMEOUT_MMA);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        const int kv_rem = p.L - j * BN;
        if (kv_rem < BN) {                          // scores of keys past the end: -inf
          int c = kv_rem;
          for (; c & 7; ++c) tmem_st1(sc + c, 0xff800000u);
#pragma unroll 1
          for (; c < BN; c += 8) tmem_fill8(sc + c, 0xff800000u);
          tc_wait_st();
        }
        uint32_t sv[BN];
        tmem_ld32(sc, sv);
        tmem_ld32(sc + 32, sv + 32);
        tc_wait_ld();
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < BN; i += 2)
          asm("max.f32 %0, %0, %1, %2;" : "+f"(mx[(i / 2) & 3]) : "f"(__uint_as_float(sv[i])), "f"(__uint_as_float(sv[i + 1])));
        mx[0] = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
        // The reference moves only when a row has outgrown it by more than 2^8 (or has none yet).
        float m_prev;
        ok = ref_of_step(&s.m_ref[t][row], n - 1, m_prev, abort_flag, p.status);
        if (!ok) break;
        if (j == sg.j0) m_prev = mx[0];
        const bool need = (mx[0] - m_prev) * scale_log2 > 8.0f;
        const float m_new = need ? mx[0] : m_prev;
        publish_ref(&s.m_ref[t][row], m_new, n);
        if (__any_sync(0xffffffffu, m_new != m_used)) {
          if (__any_sync(0xffffffffu, need)) {      // O, as of the step before, to the new reference
            ok = __all_sync(0xffffffffu, mbar_wait(&s.o_done[t][g ^ 1], g == 0 ? par ^ 1 : par, abort_flag, p.status,
                                                   STATUS_TIMEOUT_MMA));
            if (!ok) break;
            tc_fence_after();
            const float alpha = ex2((m_prev - m_new) * scale_log2);
#pragma unroll 1
            for (int c = 0; c < VD; c += 8) {
              uint32_t ov[8];
              tmem_ld8(tb + P_COL_O + c, ov);
              tc_wait_ld();
#pragma unroll
              for (int i = 0; i < 8; ++i) ov[i] = __float_as_uint(__uint_as_float(ov[i]) * alpha);
              tmem_st8(tb + P_COL_O + c, ov);
            }
          }
          if (j != j_own) {                         // the sums so far to the new reference
            const float alpha = ex2((m_used - m_new) * scale_log2);
            l_sum *= alpha;
            l_sum2 *= alpha;
          }
          m_used = m_new;
        }
        const f32x2 neg_m2 = dup2(-m_used * scale_log2);
        f32x2 l_new = dup2(0.f);
#pragma unroll
        for (int c = 0; c < BN; c += 32) {
          uint32_t pk[32 / 2];
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            const f32x2 e = fma2(pair2(sv[c + i], sv[c + i + 1]), dup2(scale_log2), neg_m2);
            const f32x2 pp = ex2_mufu2(e);
            pk[i / 2] = pack_bf16(lo2(pp), hi2(pp));
            l_new = add2(l_new, pp);
          }
          tmem_st16(sc + c / 2, pk);
        }
        l_sum += lo2(l_new);
        l_sum2 += hi2(l_new);
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.p_full[t][g]);
        par ^= 1;
      }
      // ---- epilogue of this segment ----
      auto& xst = s.xst[si & 1];
      xst[t][g][0][row] = l_sum + l_sum2;
      xst[t][g][1][row] = m_used;
      __syncwarp();
      if (lane == 0) mbar_arrive(&s.sums);
      if (ok)
        ok = mbar_wait(&s.sums, (uint32_t)(si & 1), abort_flag, p.status, STATUS_TIMEOUT_SOFTMAX) &&
             mbar_wait(&s.o_final[0], (uint32_t)(si & 1), abort_flag, p.status, STATUS_TIMEOUT_MMA) &&
             mbar_wait(&s.o_final[1], (uint32_t)(si & 1), abort_flag, p.status, STATUS_TIMEOUT_MMA);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      // the group of the last step has the final reference
      const int n_j = sg.j1 - sg.j0, gl = (n0 + n_j - 1) & 1;
      n0 += n_j;
      float m_fin[2], l_tot[2];
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        m_fin[m] = xst[m][gl][1][row];
        l_tot[m] = xst[m][gl][0][row];
        if (n_j > 1) l_tot[m] += ex2((xst[m][gl ^ 1][1][row] - m_fin[m]) * scale_log2) * xst[m][gl ^ 1][0][row];
      }
      int q0, h, b;
      item_coords(p, sg.item, q0, h, b);
      const int q_row = q0 + row;
      const bool live = q_row < p.L;
      const float m_score = (t ? m_fin[1] : m_fin[0]) * p.scale, l_own = t ? l_tot[1] : l_tot[0];
      if (sg.rec < 0) {
        // this thread takes 32 channels of the pair, of both O: half g of head 2h + t
        const float w1 = 1.f / l_tot[0], inv_l2 = 1.f / l_tot[1], w2 = p.lam.at(h) * inv_l2;
        const int64_t off = (int64_t)b * p.o_sb + (int64_t)q_row * p.o_sl + (int64_t)(2 * h + t) * p.o_sh + g * 32;
#pragma unroll 1
        for (int c = 0; c < 32; c += 8) {
          uint32_t a[8], e[8];
          tmem_ld8(tq + P_COL_O + t * HD + g * 32 + c, a);
          tmem_ld8(tq + P_MAP + P_COL_O + t * HD + g * 32 + c, e);
          tc_wait_ld();
          if (live) {
            float y[8], z[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
              y[u] = __uint_as_float(a[u]) * w1 - __uint_as_float(e[u]) * w2;
              z[u] = __uint_as_float(e[u]) * inv_l2;
            }
            store_out8(p, off + c, y, z);
          }
        }
        if (live && p.lse && g == 0)
          p.lse[((int64_t)b * 2 * p.H + 2 * h + t) * p.L + q_row] = m_score + __logf(l_own);
      } else {
        // partial result of a split item: raw accumulators, [column][row] so that a warp stores 128
        // consecutive bytes, + (m, l, mu); a group stores half the columns of its map
        float* part = p.scratch + (size_t)sg.rec * Rec<false>::ALL + t * Rec<false>::MAP;
#pragma unroll 1
        for (int c = g * HD; c < (g + 1) * HD; c += 16) {
          uint32_t ov[16];
          tmem_ld16(tb + P_COL_O + c, ov);
          tc_wait_ld();
          float* acc = part + (size_t)c * TM + row;
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[i * TM] = __uint_as_float(ov[i]);
        }
        if (g == 0) {
          float* stats = part + Rec<false>::STATS;
          stats[row] = m_score;
          stats[TM + row] = l_own;
          stats[2 * TM + row] = 0.f;
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&s.o_free);
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == P_WARP_MMA) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ----------------------------------------------------------------- tangent ---
constexpr int T_KSTAGES = 3, T_VSTAGES = 3;
constexpr int T_COL_O = 0, T_COL_DO = VD;
__host__ __device__ constexpr int t_col_s(int buf) { return 2 * VD + buf * 2 * BN; }      // S, dS; then P and T over them

struct TSmem {
  alignas(1024) uint8_t q[2][2][QPANEL];             // of two walks: q, dq
  alignas(1024) uint8_t k[T_KSTAGES][2][KPANEL];     // k, dk
  alignas(1024) uint8_t v[T_VSTAGES][4][KPANEL];     // V, dV
  uint64_t m_ref[TM];       // reference maximum of the row as of the last step decided | that step's number
  float xst[2][3][TM];      // l, mu and reference maximum of either group, at a walk's end
  uint64_t q_full[2], q_empty[2];
  // Queries scaled, a barrier for each of the two walks: a group without a step in a walk of one tile scales the
  // next walk's at once, and must not be counted for a warp that has not scaled its share of this one's.
  uint64_t q_ready[2];
  uint64_t k_full[T_KSTAGES], k_empty[T_KSTAGES];
  uint64_t v_full[T_VSTAGES], v_empty[T_VSTAGES];
  uint64_t s_full[2], p_full[2];
  uint64_t o_done[2];       // every O product
  uint64_t o_final;         // the last one of a walk (one phase per walk, never skipped)
  uint64_t o_free, sums;
  uint32_t tmem_base;
  int abort_flag;
};

// q and dq times a power of two, in place, by the softmax warps
IMF_DEVICE void scale_queries(uint8_t (&q)[2][QPANEL], float f) {
  uint4* qs = reinterpret_cast<uint4*>(q);
#pragma unroll 4
  for (int i = threadIdx.x; i < (int)(sizeof(q) / 16); i += SOFT_WARPS * 32) {
    uint4 x = qs[i];
    x.x = pack_bf16(bf16_lo(x.x) * f, bf16_hi(x.x) * f);
    x.y = pack_bf16(bf16_lo(x.y) * f, bf16_hi(x.y) * f);
    x.z = pack_bf16(bf16_lo(x.z) * f, bf16_hi(x.z) * f);
    x.w = pack_bf16(bf16_lo(x.w) * f, bf16_hi(x.w) * f);
    qs[i] = x;
  }
  fence_proxy_async_smem();
  __syncwarp();
}

// UNIT: the scale is a power of two, which is multiplied into q and dq in shared memory, exactly, instead
// of into every T.
template <bool UNIT>
__global__ void __launch_bounds__(THREADS, 1)
attn_diff_jvp_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                     const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_dq,
                     const __grid_constant__ CUtensorMap tm_dk, const __grid_constant__ CUtensorMap tm_dv,
                     const Params p) {
  extern __shared__ uint8_t smem_raw[];
  auto& s = *reinterpret_cast<TSmem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int cta = blockIdx.x, G = gridDim.x;

  if (threadIdx.x == 0) {
    for (int i = 0; i < T_KSTAGES; ++i) {
      mbar_init(&s.k_full[i], 1);
      mbar_init(&s.k_empty[i], 1);
    }
    for (int i = 0; i < T_VSTAGES; ++i) {
      mbar_init(&s.v_full[i], 1);
      mbar_init(&s.v_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s.q_full[i], 1);
      mbar_init(&s.q_empty[i], 1);
      mbar_init(&s.q_ready[i], SOFT_WARPS);
      mbar_init(&s.s_full[i], 1);
      mbar_init(&s.p_full[i], SOFT_WARPS / 2);
      mbar_init(&s.o_done[i], 1);
    }
    mbar_init(&s.o_final, 1);
    mbar_init(&s.o_free, SOFT_WARPS);
    mbar_init(&s.sums, SOFT_WARPS);
    s.abort_flag = 0;
    fence_barrier_init();
  }
  if (threadIdx.x < TM) s.m_ref[threadIdx.x] = ref_word(0.f, -1);
  if (warp == WARP_MMA) {
    tmem_alloc(&s.tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s.tmem_base;
  volatile int* abort_flag = &s.abort_flag;

  // A walk is one map over the K/V tiles of a segment: walk 2 si + m of the CTA.
  if (warp >= SOFT_WARPS) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REG_OTHER));
    if (warp == WARP_TMA) {
      // ------------------------------------------------------ TMA producer --
      if (elect_one()) {
        prefetch_tmap(&tm_q);
        prefetch_tmap(&tm_k);
        prefetch_tmap(&tm_v);
        prefetch_tmap(&tm_dq);
        prefetch_tmap(&tm_dk);
        prefetch_tmap(&tm_dv);
        int kst = 0, vst = 0, walk = 0;
        uint32_t kpar = 1, vpar = 1;         // an "empty" wait passes in the first round of a ring
        Segment sg;
        bool ok = true;
        for (int si = 0; ok && get_segment(p.sh, cta, G, si, sg); ++si) {
          int q0, h, b;
          item_coords(p, sg.item, q0, h, b);
          for (int m = 0; m < 2 && ok; ++m, ++walk) {
            const int qs = walk & 1;
            ok = mbar_wait(&s.q_empty[qs], (uint32_t)((walk >> 1) & 1) ^ 1, abort_flag, p.status, STATUS_TIMEOUT_EMPTY);
            if (!ok) break;
            mbar_arrive_expect_tx(&s.q_full[qs], 2 * QPANEL);
            tma_load_4d(s.q[qs][0], &tm_q, &s.q_full[qs], 0, 2 * h + m, q0, b);
            tma_load_4d(s.q[qs][1], &tm_dq, &s.q_full[qs], 0, 2 * h + m, q0, b);
            for (int j = sg.j0; j < sg.j1; ++j) {
              ok = mbar_wait(&s.k_empty[kst], kpar, abort_flag, p.status, STATUS_TIMEOUT_EMPTY);
              if (!ok) break;
              mbar_arrive_expect_tx(&s.k_full[kst], 2 * KPANEL);
              tma_load_4d(s.k[kst][0], &tm_k, &s.k_full[kst], 0, 2 * h + m, j * BN, b);
              tma_load_4d(s.k[kst][1], &tm_dk, &s.k_full[kst], 0, 2 * h + m, j * BN, b);
              if (++kst == T_KSTAGES) {
                kst = 0;
                kpar ^= 1;
              }
              ok = mbar_wait(&s.v_empty[vst], vpar, abort_flag, p.status, STATUS_TIMEOUT_EMPTY);
              if (!ok) break;
              mbar_arrive_expect_tx(&s.v_full[vst], 4 * KPANEL);
              for (int i = 0; i < 2; ++i) {
                tma_load_4d(s.v[vst][i], &tm_v, &s.v_full[vst], 0, 2 * h + i, j * BN, b);
                tma_load_4d(s.v[vst][2 + i], &tm_dv, &s.v_full[vst], 0, 2 * h + i, j * BN, b);
              }
              if (++vst == T_VSTAGES) {
                vst = 0;
                vpar ^= 1;
              }
            }
          }
        }
      }
    } else if (warp == WARP_MMA) {
      // -------------------------------------------------------- MMA issuer --
      // One thread issues both products, the scores of step n + 2 right behind the O product of step n, whose
      // P and T they overwrite: that keeps the groups half a period apart.  With a warp for each product the
      // O products of two steps came one behind the other, the scores of the next two behind those, and both
      // groups waited at the same time (2 pairs of 29,140 tokens: 3.24 ms).
      if (elect_one()) {
        // Q [K | dK]^T -> S | dS and P [V | dV] -> O | dO are one product each (operands adjacent in
        // shared memory, accumulators in TMEM): an SM reads 128 B of operands per clock, just what
        // M = N = 128 from shared memory asks for
        constexpr uint32_t idesc_qk = idesc_bf16(TM, 2 * BN, 0, 0);
        constexpr uint32_t idesc_dqk = idesc_bf16(TM, BN, 0, 0);
        constexpr uint32_t idesc_pv = idesc_bf16(TM, 2 * VD, 0, 1);
        constexpr uint32_t idesc_tv = idesc_bf16(TM, VD, 0, 1);
        const uint64_t q_desc = sdesc_kmajor(smem_u32(s.q[0][0])), k_desc = sdesc_kmajor(smem_u32(s.k[0][0]));
        const uint64_t v_desc = sdesc_mnmajor(smem_u32(s.v[0][0]), KPANEL);
        int kst = 0, kbuf = 0, vst = 0, vbuf = 0, walk = 0;
        uint32_t kpar = 0, vpar = 0, ppar = 0;
        Segment sg;
        bool ok = true;
        for (int si = 0; ok && get_segment(p.sh, cta, G, si, sg); ++si) {
          const int n_j = sg.j1 - sg.j0;
          for (int m = 0; m < 2 && ok; ++m, ++walk) {
            const int qs = walk & 1;
            ok = UNIT ? mbar_wait(&s.q_ready[qs], (uint32_t)((walk >> 1) & 1), abort_flag, p.status, STATUS_TIMEOUT_SOFTMAX)
                      : mbar_wait(&s.q_full[qs], (uint32_t)((walk >> 1) & 1), abort_flag, p.status, STATUS_TIMEOUT_TMA);
            const uint64_t qd = q_desc + (uint32_t)(qs * (2 * QPANEL >> 4)), dqd = qd + (QPANEL >> 4);
            // scores of step jj of the walk
            auto scores = [&](int jj) {
              if (!mbar_wait(&s.k_full[kst], kpar, abort_flag, p.status, STATUS_TIMEOUT_TMA)) return false;
              tc_fence_after();
              const uint64_t kd = k_desc + (uint32_t)(kst * (2 * KPANEL >> 4));
              const uint32_t sc = tmem + t_col_s(kbuf);
#pragma unroll
              for (int ks = 0; ks < HD / 16; ++ks) mma_ss(sc, qd + 2 * ks, kd + 2 * ks, idesc_qk, ks != 0);
#pragma unroll
              for (int ks = 0; ks < HD / 16; ++ks) mma_ss(sc + BN, dqd + 2 * ks, kd + 2 * ks, idesc_dqk, 1);
              tc_commit(&s.s_full[kbuf]);
              tc_commit(&s.k_empty[kst]);
              if (jj + 1 == n_j) tc_commit(&s.q_empty[qs]);
              if (++kst == T_KSTAGES) {
                kst = 0;
                kpar ^= 1;
              }
              kbuf ^= 1;
              return true;
            };
            ok = ok && scores(0) && (n_j == 1 || scores(1));
            if (ok && walk > 0)      // epilogue of the previous walk has drained O
              ok = mbar_wait(&s.o_free, (uint32_t)((walk - 1) & 1), abort_flag, p.status, STATUS_TIMEOUT_SOFTMAX);
            for (int jj = 0; jj < n_j && ok; ++jj) {
              ok = mbar_wait(&s.v_full[vst], vpar, abort_flag, p.status, STATUS_TIMEOUT_TMA) &&
                   mbar_wait(&s.p_full[vbuf], ppar, abort_flag, p.status, STATUS_TIMEOUT_SOFTMAX);
              if (!ok) break;
              tc_fence_after();
              const uint64_t vd = v_desc + (uint32_t)(vst * (4 * KPANEL >> 4));
              const uint32_t pc = tmem + t_col_s(vbuf);
#pragma unroll
              for (int ks = 0; ks < BN / 16; ++ks)
                mma_ts(tmem + T_COL_O, pc + ks * 8, vd + 128 * ks, idesc_pv, !(jj == 0 && ks == 0));
#pragma unroll
              for (int ks = 0; ks < BN / 16; ++ks)
                mma_ts(tmem + T_COL_DO, pc + BN / 2 + ks * 8, vd + 128 * ks, idesc_tv, 1);
              tc_commit(&s.o_done[vbuf]);
              tc_commit(&s.v_empty[vst]);
              if (jj + 1 == n_j) tc_commit(&s.o_final);
              if (++vst == T_VSTAGES) {
                vst = 0;
                vpar ^= 1;
              }
              vbuf ^= 1;
              if (vbuf == 0) ppar ^= 1;
              if (jj + 2 < n_j) ok = scores(jj + 2);
            }
          }
        }
      }
    }
  } else {
    // ------------------------------------- softmax / correction / epilogue --
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REG_SOFT));
    // Group g takes the steps (K/V tiles) of parity g, with buffer g.  Either warp of a row pair needs
    // the row's reference maximum as the step before left it: it is handed from one to the other,
    // before the exponentials.
    const int g = warp >> 2, wl = warp & 3;
    const int row = wl * 32 + lane;
    const uint32_t tb = tmem_addr(tmem, wl * 32, 0);
    const uint32_t sc = tb + t_col_s(g);
    const float scale_log2 = (UNIT ? 1.f : p.scale) * LOG2E;
    // 64 columns of o, then of do, of this thread's head: [column][row]
    float* const hold = p.hold + (size_t)cta * HOLD + (size_t)g * VD * TM + row;
    uint32_t par = 0;                               // phase of this group's buffer
    int n0 = 0;                                     // number of the walk's first step
    int walk = 0;
    auto scale_for = [&](int w) {                   // UNIT: the queries of walk w
      if (!__all_sync(0xffffffffu, mbar_wait(&s.q_full[w & 1], (uint32_t)((w >> 1) & 1), abort_flag, p.status,
                                             STATUS_TIMEOUT_TMA)))
        return false;
      scale_queries(s.q[w & 1], p.scale);
      if (lane == 0) mbar_arrive(&s.q_ready[w & 1]);
      return true;
    };
    Segment sg;
    bool ok = true;
    for (int si = 0; ok && get_segment(p.sh, cta, G, si, sg); ++si) {
      int q0, h, b;
      item_coords(p, sg.item, q0, h, b);
      const int q_row = q0 + row;
      const bool live = q_row < p.L;
#pragma unroll 1
      for (int m = 0; m < 2 && ok; ++m, ++walk) {
        float m_used = -INFINITY, l_sum = 0.f, l_sum2 = 0.f, mu_sum = 0.f, mu_sum2 = 0.f;
        const int j_own = sg.j0 + ((n0 ^ g) & 1);     // this group's first step of the walk
        if (UNIT && walk == 0) ok = scale_for(0);
        for (int j = j_own; j < sg.j1 && ok; j += 2) {
          const int n = n0 + j - sg.j0;
          // The O product of this group's step before, n - 2, is seen to be over before the reference of step n is
          // published: whoever has that reference and asks o_done for the O product of step n then finds the
          // barrier in that phase or one further.  (A wait by parity on a barrier still two phases back returns at
          // once.  The scores of step n are made behind that product, but nothing says that arrivals on two
          // barriers are seen in their order.)
          ok = mbar_wait(&s.o_done[g], par ^ 1, abort_flag, p.status, STATUS_TIMEOUT_MMA) &&
               mbar_wait(&s.s_full[g], par, abort_flag, p.status, STATUS_TIMEOUT_MMA);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          tc_fence_after();
          const int kv_rem = p.L - j * BN;
          if (kv_rem < BN) {                          // scores of keys past the end: -inf
            int c = kv_rem;
            for (; c & 7; ++c) tmem_st1(sc + c, 0xff800000u);
#pragma unroll 1
            for (; c < BN; c += 8) tmem_fill8(sc + c, 0xff800000u);
            tc_wait_st();
          }
          uint32_t sv[BN];
          tmem_ld32(sc, sv);
          tmem_ld32(sc + 32, sv + 32);
          tc_wait_ld();
          float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int i = 0; i < BN; i += 2)
            asm("max.f32 %0, %0, %1, %2;" : "+f"(mx[(i / 2) & 3]) : "f"(__uint_as_float(sv[i])), "f"(__uint_as_float(sv[i + 1])));
          mx[0] = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
          // The reference is moved only when a row has outgrown it by more than 2^8 (or has none yet).
          float m_prev;
          ok = ref_of_step(&s.m_ref[row], n - 1, m_prev, abort_flag, p.status);
          if (!ok) break;
          if (j == sg.j0) m_prev = mx[0];
          const bool need = (mx[0] - m_prev) * scale_log2 > 8.0f;
          const float m_new = need ? mx[0] : m_prev;
          publish_ref(&s.m_ref[row], m_new, n);
          if (__any_sync(0xffffffffu, m_new != m_used)) {
            if (__any_sync(0xffffffffu, need)) {      // O, as of the step before, to the new reference
              ok = __all_sync(0xffffffffu, mbar_wait(&s.o_done[g ^ 1], g == 0 ? par ^ 1 : par, abort_flag,
                                                     p.status, STATUS_TIMEOUT_MMA));
              if (!ok) break;
              tc_fence_after();
              const float alpha = ex2((m_prev - m_new) * scale_log2);
#pragma unroll 1
              for (int c = 0; c < 2 * VD; c += 16) {
                uint32_t ov[16];
                tmem_ld16(tb + T_COL_O + c, ov);
                tc_wait_ld();
#pragma unroll
                for (int i = 0; i < 16; ++i) ov[i] = __float_as_uint(__uint_as_float(ov[i]) * alpha);
                tmem_st16(tb + T_COL_O + c, ov);
              }
            }
            if (j != j_own) {                         // the sums so far to the new reference
              const float alpha = ex2((m_used - m_new) * scale_log2);
              l_sum *= alpha;
              l_sum2 *= alpha;
              mu_sum *= alpha;
              mu_sum2 *= alpha;
            }
            m_used = m_new;
          }
          const f32x2 neg_m2 = dup2(-m_used * scale_log2);
          f32x2 l_new = dup2(0.f), mu_new = dup2(0.f);
          uint32_t dsv[2][32];
          tmem_ld32(sc + BN, dsv[0]);
          tmem_ld32(sc + BN + 32, dsv[1]);
          tc_wait_ld();
#pragma unroll
          for (int c = 0; c < BN; c += 32) {
            uint32_t pk[16], tk[16];
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              const int i = c + e;
              const f32x2 x = fma2(pair2(sv[i], sv[i + 1]), dup2(scale_log2), neg_m2);
              const float p0 = ex2(lo2(x)), p1 = ex2(hi2(x));
              const f32x2 pp = pair2(__float_as_uint(p0), __float_as_uint(p1));
              pk[e / 2] = pack_bf16(p0, p1);
              l_new = add2(l_new, pp);
              f32x2 tt = mul2(pp, pair2(dsv[i >> 5][i & 31], dsv[i >> 5][(i & 31) + 1]));
              if (!UNIT) tt = mul2(tt, dup2(p.scale));
              mu_new = add2(mu_new, tt);
              tk[e / 2] = pack_bf16(lo2(tt), hi2(tt));
            }
            tmem_st16(sc + c / 2, pk);
            tmem_st16(sc + BN / 2 + c / 2, tk);
          }
          l_sum += lo2(l_new);
          l_sum2 += hi2(l_new);
          mu_sum += lo2(mu_new);
          mu_sum2 += hi2(mu_new);
          tc_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&s.p_full[g]);
          par ^= 1;
        }
        // the next walk's scores are made during this one's epilogue
        Segment next;
        if (UNIT && ok && (m == 0 || get_segment(p.sh, cta, G, si + 1, next))) ok = scale_for(walk + 1);
        // ---- epilogue of this walk ----
        if (ok) ok = mbar_wait(&s.o_final, (uint32_t)(walk & 1), abort_flag, p.status, STATUS_TIMEOUT_MMA);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        s.xst[g][0][row] = l_sum + l_sum2;
        s.xst[g][1][row] = mu_sum + mu_sum2;
        s.xst[g][2][row] = m_used;
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.sums);
        ok = __all_sync(0xffffffffu, mbar_wait(&s.sums, (uint32_t)(walk & 1), abort_flag, p.status,
                                               STATUS_TIMEOUT_SOFTMAX));
        if (!ok) break;
        // the group of the last step has the final reference
        const int n_j = sg.j1 - sg.j0, gl = (n0 + n_j - 1) & 1;
        const float m_fin = s.xst[gl][2][row];
        float l_tot = s.xst[gl][0][row], mu_tot = s.xst[gl][1][row];
        if (n_j > 1) {
          const float alpha = ex2((s.xst[gl ^ 1][2][row] - m_fin) * scale_log2);
          l_tot += alpha * s.xst[gl ^ 1][0][row];
          mu_tot += alpha * s.xst[gl ^ 1][1][row];
        }
        n0 += n_j;
        const float m_score = UNIT ? m_fin : m_fin * p.scale;      // of the scaled scores
        if (sg.rec < 0) {
          // this thread takes the 64 channels of head 2h + g, of o and of do
          const float inv_l = 1.f / l_tot, mul = mu_tot * inv_l, lam = p.lam.at(h);
          const int64_t off = (int64_t)b * p.o_sb + (int64_t)q_row * p.o_sl + (int64_t)(2 * h + g) * p.o_sh;
#pragma unroll 1
          for (int c = 0; c < VD / 2; c += 32) {
            uint32_t ov[32], dv_[32];
            tmem_ld32(tb + T_COL_O + g * (VD / 2) + c, ov);
            tmem_ld32(tb + T_COL_DO + g * (VD / 2) + c, dv_);
            tc_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              const float o = __uint_as_float(ov[i]) * inv_l;
              ov[i] = __float_as_uint(o);
              dv_[i] = __float_as_uint(__uint_as_float(dv_[i]) * inv_l - mul * o);
            }
            float* ho = hold + (size_t)c * TM;
            float* hd = ho + (size_t)(VD / 2) * TM;
            if (m == 0) {
#pragma unroll
              for (int i = 0; i < 32; ++i) {
                ho[i * TM] = __uint_as_float(ov[i]);
                hd[i * TM] = __uint_as_float(dv_[i]);
              }
            } else if (live) {
#pragma unroll
              for (int i = 0; i < 32; i += 8) {
                float r[8], z[8];
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                  z[u] = __uint_as_float(ov[i + u]);
                  r[u] = ho[(i + u) * TM] - lam * z[u];
                }
                store_out8(p, off + c + i, r, z);
#pragma unroll
                for (int u = 0; u < 8; ++u) r[u] = hd[(i + u) * TM] - lam * __uint_as_float(dv_[i + u]);
                *reinterpret_cast<uint4*>(p.dout + off + c + i) =
                    make_uint4(pack_bf16(r[0], r[1]), pack_bf16(r[2], r[3]), pack_bf16(r[4], r[5]), pack_bf16(r[6], r[7]));
              }
            }
          }
          if (live && p.lse && g == 0)
            p.lse[((int64_t)b * 2 * p.H + 2 * h + m) * p.L + q_row] = m_score + __logf(l_tot);
        } else {
          // group 0 stores the O accumulators (columns 0-127), group 1 those of dO (128-255)
          float* part = p.scratch + (size_t)sg.rec * Rec<true>::ALL + m * Rec<true>::MAP;
          for (int c = 0; c < VD; c += 32) {
            uint32_t ov[32];
            tmem_ld32(tb + T_COL_O + g * VD + c, ov);
            tc_wait_ld();
            float* acc = part + (size_t)(c + g * VD) * TM + row;
#pragma unroll
            for (int i = 0; i < 32; ++i) acc[i * TM] = __uint_as_float(ov[i]);
          }
          if (g == 0) {
            float* stats = part + Rec<true>::STATS;
            stats[row] = m_score;
            stats[TM + row] = l_tot;
            stats[2 * TM + row] = mu_tot;
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.o_free);
      }
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == WARP_MMA) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ------------------------------------------------------------------- merge ---
// Merge the parts of every split item and subtract map 2 (as combine_split_items, a record for each
// map).  A CTA takes 32 query rows (a lane each), a warp 8 of the 128 columns.
template <bool TANGENT>
__global__ void __launch_bounds__(32 * VD / COMBINE_COLS) attn_diff_combine_kernel(const Params p, int G) {
  using R = Rec<TANGENT>;
  const int c = blockIdx.x;
  int item, parts;
  if (!split_item(p.sh, c, G, item, parts)) return;
  int q0, h, b;
  item_coords(p, item, q0, h, b);
  const float lam = p.lam.at(h);
  const int r = blockIdx.y * COMBINE_ROWS + (threadIdx.x & 31);
  const int col = (threadIdx.x >> 5) * COMBINE_COLS;
  const int q_row = q0 + r;
  if (q_row >= p.L) return;
  const int64_t off = (int64_t)b * p.o_sb + (int64_t)q_row * p.o_sl + (int64_t)(2 * h + col / HD) * p.o_sh + col % HD;
  const float* x = p.scratch + (size_t)(2 * c + 1) * R::ALL + r;   // then records 2c + 2, 2c + 4, ...
  float m[2] = {x[R::STATS], x[R::MAP + R::STATS]}, l[2] = {0.f, 0.f}, mu[2] = {0.f, 0.f};
  float o[2][COMBINE_COLS], d[2][COMBINE_COLS];
#pragma unroll
  for (int i = 0; i < COMBINE_COLS; ++i) o[0][i] = o[1][i] = d[0][i] = d[1][i] = 0.f;
  // All of it is latency: with a tangent both maps' loads at once (1 x 1,100 rows, 2 pairs 41 -> 33 us in all), without
  // one map after the other (24, at once 28).
  if constexpr (TANGENT) {
#pragma unroll 2
    for (int k = 0; k < parts; ++k, x += k == 1 ? R::ALL : 2 * R::ALL) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const float* z = x + t * R::MAP;
        const float mk = z[R::STATS], mn = fmaxf(m[t], mk);
        const float w0 = ex2((m[t] - mn) * LOG2E), w1 = ex2((mk - mn) * LOG2E);
        m[t] = mn;
        l[t] = l[t] * w0 + z[R::STATS + TM] * w1;
        mu[t] = mu[t] * w0 + z[R::STATS + 2 * TM] * w1;
#pragma unroll
        for (int i = 0; i < COMBINE_COLS; ++i) {
          o[t][i] = o[t][i] * w0 + z[(col + i) * TM] * w1;
          d[t][i] = d[t][i] * w0 + z[(VD + col + i) * TM] * w1;
        }
      }
    }
  } else {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const float* z = x + t * R::MAP;
#pragma unroll 2
      for (int k = 0; k < parts; ++k, z += k == 1 ? R::ALL : 2 * R::ALL) {
        const float mk = z[R::STATS], mn = fmaxf(m[t], mk);
        const float w0 = ex2((m[t] - mn) * LOG2E), w1 = ex2((mk - mn) * LOG2E);
        m[t] = mn;
        l[t] = l[t] * w0 + z[R::STATS + TM] * w1;
#pragma unroll
        for (int i = 0; i < COMBINE_COLS; ++i) o[t][i] = o[t][i] * w0 + z[(col + i) * TM] * w1;
      }
    }
  }
  float y[COMBINE_COLS], dy[COMBINE_COLS];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const float inv_l = 1.f / l[t], mul = mu[t] * inv_l;
#pragma unroll
    for (int i = 0; i < COMBINE_COLS; ++i) {
      o[t][i] *= inv_l;
      d[t][i] = d[t][i] * inv_l - mul * o[t][i];
      y[i] = t == 0 ? o[t][i] : y[i] - lam * o[t][i];
      dy[i] = t == 0 ? d[t][i] : dy[i] - lam * d[t][i];
    }
    if (p.lse && col == 0) p.lse[((int64_t)b * 2 * p.H + 2 * h + t) * p.L + q_row] = m[t] + __logf(l[t]);
  }
  store_out8(p, off, y, o[1]);
  if (TANGENT)
    *reinterpret_cast<uint4*>(p.dout + off) =
        make_uint4(pack_bf16(dy[0], dy[1]), pack_bf16(dy[2], dy[3]), pack_bf16(dy[4], dy[5]), pack_bf16(dy[6], dy[7]));
}

// 4-D map over a (B, L, 2H, 64) bf16 tensor whose box is `rows` rows of one head
static int make_map(CUtensorMap* m, const void* ptr, int B, int L, int heads, const int64_t* st, int rows) {
  uint64_t dims[4] = {(uint64_t)HD, (uint64_t)heads, (uint64_t)L, (uint64_t)B};
  uint64_t str[4] = {2, (uint64_t)st[2] * 2, (uint64_t)st[1] * 2, (uint64_t)st[0] * 2};
  uint32_t box[4] = {(uint32_t)HD, 1, (uint32_t)rows, 1};
  return make_tmap(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(ptr), dims, str, box);
}

static FwdShares shares(int B, int L, int H) {
  FwdShares sh;
  sh.n_items = (L + TM - 1) / TM * H * B;
  sh.n_kv = (L + BN - 1) / BN;
  sh.total = (long)sh.n_items * sh.n_kv;
  return sh;
}

// Floats of scratch of a grid of G CTAs: with a tangent the held rows, then the records if items are split.
template <bool TANGENT>
static size_t scratch_floats(int G, bool split) {
  return (TANGENT ? (size_t)G * HOLD : 0) + (split ? (size_t)G * 2 * Rec<TANGENT>::ALL : 0);
}

// CTAs.  Fewer items than SMs: shares of at least two K/V tiles, if that shortens a CTA's walk by more than the
// second kernel, the partial results and the second segment cost: 12 us at 148 CTAs (16 tiles of 0.74 us) or 16
// (11 of 1.54) with a tangent, less with fewer records.  Measured whole / in shares, us, pairs of one batch
// entry: 532 rows, 2 pairs 14.8 / 18.5 and 31.1 / 29.2; 1,100 rows, 2 pairs 21.7 / 23.7 and 45 / 34; 1,500
// rows, 3 pairs 27.1 / 25.8 and 55 / 42; 4,116 rows, 1 pair 56 / 33 and 117 / 56.
template <bool TANGENT>
static int grid(const FwdShares& sh) {
  const int sms = fwd_sm_count();
  if (sh.n_items >= sms) return sms;
  const long g = sh.total / 2 < sms ? sh.total / 2 : sms;
  if (g <= sh.n_items) return sh.n_items;
  const float saved = (float)(sh.n_kv - (sh.total + g - 1) / g);
  return saved < (TANGENT ? 5.f : 10.5f) + 0.04f * (float)g ? sh.n_items : (int)g;
}

}  // namespace diff
}  // namespace imf

// Bytes of scratch that imf_attn_diff_fwd needs (0: none).
extern "C" long imf_attn_diff_fwd_scratch_bytes(int B, int L, int H, int tangent) {
  using namespace imf;
  using namespace imf::diff;
  if (B <= 0 || L <= 0 || H <= 0 || (long)B * H * ((L + TM - 1) / TM) > 0x3fffffffL) return 0;
  const FwdShares sh = shares(B, L, H);
  const int G = tangent ? grid<true>(sh) : grid<false>(sh);
  return 4L * (long)(tangent ? scratch_floats<true>(G, G != sh.n_items) : scratch_floats<false>(G, G != sh.n_items));
}

// q, k, v (, dq, dk, dv): (B, L, 2H, 64) bf16 with (batch, row, head) element strides in strides[0..17]; o, dout, o2
// share (batch, row, head) strides o_strides; dout null without a tangent.  Where a backward pass follows: o2, lse
// (B, 2H, L) and low, 16 bytes at twice o's offsets, of eight channels of o and then of o2 (see attn_diff.h).  lam: H
// weights, lam_stride elements apart.
extern "C" int imf_attn_diff_fwd(const void* q, const void* k, const void* v, const void* dq, const void* dk,
                                 const void* dv, const void* lam, int64_t lam_stride, int lam_bf16, void* o, void* dout,
                                 void* o2, void* low, float* lse, int B, int L, int H, const int64_t* strides,
                                 const int64_t* o_strides, float scale, void* scratch, long scratch_bytes, int* status,
                                 void* stream) {
  using namespace imf;
  using namespace imf::diff;
  const bool tangent = dq != nullptr;
  if (!q || !k || !v || !lam || !o || B <= 0 || L <= 0 || H <= 0) return IMF_ERR_ARG;
  if (tangent != (dk != nullptr) || tangent != (dv != nullptr) || tangent != (dout != nullptr)) return IMF_ERR_ARG;
  if ((o2 != nullptr) != (low != nullptr) || (reinterpret_cast<uintptr_t>(low) & 15)) return IMF_ERR_ARG;
  if (!(scale > 0.f) || scale > 1e30f) return IMF_ERR_ARG;
  if ((long)B * H * ((L + TM - 1) / TM) > 0x3fffffffL) return IMF_ERR_TOO_LARGE;
  for (const void* x : {(const void*)o, (const void*)dout, (const void*)o2})
    if (reinterpret_cast<uintptr_t>(x) & 15) return IMF_ERR_ARG;
  for (int i = 0; i < 3; ++i)
    if (o_strides[i] & 7) return IMF_ERR_ARG;
  Params prm;
  prm.o = static_cast<__nv_bfloat16*>(o);
  prm.dout = static_cast<__nv_bfloat16*>(dout);
  prm.o2 = static_cast<__nv_bfloat16*>(o2);
  prm.low = static_cast<int8_t*>(low);
  prm.lse = lse;
  prm.lam = {lam, lam_stride, lam_bf16};
  prm.B = B; prm.H = H; prm.L = L;
  prm.n_qblk = (L + TM - 1) / TM;
  prm.sh = shares(B, L, H);
  prm.o_sb = o_strides[0]; prm.o_sl = o_strides[1]; prm.o_sh = o_strides[2];
  prm.scale = scale;
  prm.status = status;
  const int G = tangent ? grid<true>(prm.sh) : grid<false>(prm.sh);
  const bool split = G != prm.sh.n_items;
  const size_t need = 4 * (tangent ? scratch_floats<true>(G, split) : scratch_floats<false>(G, split));
  if (need && (scratch == nullptr || (size_t)scratch_bytes < need || (reinterpret_cast<uintptr_t>(scratch) & 15)))
    return IMF_ERR_ARG;
  prm.hold = static_cast<float*>(scratch);
  prm.scratch = prm.hold + (tangent ? (size_t)G * HOLD : 0);
  CUtensorMap mq, mk, mv, mdq, mdk, mdv;
  int rc;
  if ((rc = make_map(&mq, q, B, L, 2 * H, strides, TM))) return rc;
  if ((rc = make_map(&mk, k, B, L, 2 * H, strides + 3, BN))) return rc;
  if ((rc = make_map(&mv, v, B, L, 2 * H, strides + 6, BN))) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  static bool smem_set[3][HOST_MAX_DEVICES] = {{false}};
  if (tangent) {
    if ((rc = make_map(&mdq, dq, B, L, 2 * H, strides + 9, TM))) return rc;
    if ((rc = make_map(&mdk, dk, B, L, 2 * H, strides + 12, BN))) return rc;
    if ((rc = make_map(&mdv, dv, B, L, 2 * H, strides + 15, BN))) return rc;
    const size_t smem = sizeof(TSmem) + 1024;
    int e;
    // (a power of two so far below one that queries times it might leave bf16's normal numbers is not taken)
    const bool unit = scale > 0x1p-9f && scale <= 1.f && frexpf(scale, &e) == 0.5f;
    auto kern = unit ? attn_diff_jvp_kernel<true> : attn_diff_jvp_kernel<false>;
    if (!allow_smem((const void*)kern, smem, smem_set[unit ? 2 : 1])) return IMF_ERR_LAUNCH;
    kern<<<G, THREADS, smem, st>>>(mq, mk, mv, mdq, mdk, mdv, prm);
  } else {
    const size_t smem = sizeof(PSmem) + 1024;
    if (!allow_smem((const void*)attn_diff_fwd_kernel, smem, smem_set[0])) return IMF_ERR_LAUNCH;
    attn_diff_fwd_kernel<<<G, P_THREADS, smem, st>>>(mq, mk, mv, prm);
  }
  if (cudaGetLastError() != cudaSuccess) return IMF_ERR_LAUNCH;
  if (split) {
    const dim3 g(G - 1, TM / COMBINE_ROWS);
    if (tangent)
      attn_diff_combine_kernel<true><<<g, 32 * VD / COMBINE_COLS, 0, st>>>(prm, G);
    else
      attn_diff_combine_kernel<false><<<g, 32 * VD / COMBINE_COLS, 0, st>>>(prm, G);
    if (cudaGetLastError() != cudaSuccess) return IMF_ERR_LAUNCH;
  }
  return IMF_OK;
}
