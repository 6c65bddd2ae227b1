// Weight gradient of a linear layer whose input was kept in 8 bits (format: act8.cuh):
//
//   dW[N, C] (+)= dY^T X,   dY [R, N] bf16,  X [R, C] = codes * 2^(step - 127),  fp32 result
//
// on tcgen05 with the accumulator in TMEM.  Both operands are consumed MN-major as they lie in memory
// (the contraction runs over the rows).  The step belongs to 32 channels of ONE row, so it cannot be taken
// out of the sum; the codes are converted on their way from shared memory to shared memory instead,
// and exactly (bf16 holds code * 2^k), so the product is that of the stored values.
//
// Two CTAs (a cluster) share a 256 (N) x BN (C) tile and its products (cta_group::2): each holds 128 of the
// rows of dY^T and half of X's columns, so each converts half a tile for 256 rows of products.  k-blocks are
// 64 rows of R.  Warps 0-3: epilogue; warp 4: loads of dY; warp 5: tcgen05.mma in the first CTA, word of the
// other's dY in the second; warp 6: loads of the codes (TMA) and steps (cp.async: their rows
// are no 16-byte multiples); then CONV groups of warps that convert a k-block each.  dY and the codes have rings
// of their own: dY's stages wait for products alone, those of the codes for the conversion.
// R is cut into slices (split-K) where that fills the SMs; a second kernel adds their planes up
// in a fixed order, so results repeat bit for bit.
//
// The tensor core's fp32 accumulator drops bits with every k-step, more the longer the chain (of the result's norm,
// 32,780 rows of activations with outliers: 1.2e-5 in one chain, 4.0e-6 in chains of 103 k-blocks, 1.9e-6 of
// 52, 0.8e-6 of 35); so a slice is cut into equal chains of CHAIN k-blocks at most, and the TMA unit adds the
// next one's sum to the stored one (one CTA owns the place, and waits for one addition before the next: the order is
// fixed).  Storing a chain's sum runs under the next one's products where TMEM holds two accumulators; with BN 512
// it holds one, whose halves are stored and begun again one after the other, at some 4 us a chain.
//
// What bounds it.  For a k-block of BN 256 a CTA moves 24 KB in by TMA, 24 KB through the conversion and 32 KB into the
// tensor core, 640 clocks of shared memory at 128 bytes, against 512 of tcgen05.mma (BN 512, whose two accumulators share
// the rows of dY^T: 1,152 against 1,024); 900 and 1,230 are measured.  Neither sets the pace alone: without the
// converted tile's stores it takes 12 % less, without three of four products 6 %.  What makes up the rest is not known;
// rings of five or seven stages and fewer or more polls of the barriers do not change it.
// 32,780 rows x 5,472 x 1,024: 334 us alone (1,100 TFLOP/s; among other passes, at the power cap, 380 to 410), of which
// the ends of the chains are 20 and the kernel that adds the planes up 20 to 27; restoring X to bf16 first and the bf16
// kernel of gemm.cu 428.  29,140 x 1,376 x 256: 37 us, the bf16 kernel alone 45.  Into a gradient buffer 4 and 2 us more.
// Tried and slower: one ring and one loading warp for dY, codes and steps (2 to 6 %); codes loaded into registers by
// the converting warps (594 us: the proxy fence waits for the loads) or by cp.async (463); the k-blocks of all tiles
// dealt to the pairs in equal runs (9 %: pairs at different rows share nothing in L2); sums added from registers (10 %).
#include "act8.cuh"
#include "common.cuh"
#include "host_util.h"
#include <stddef.h>

namespace imf {
namespace w8 {

constexpr int BM = 128, BK = 64;           // rows of dY^T per CTA; rows of a k-block

template <int BN>
struct Smem {
  static constexpr int BNL = BN / 2;                 // columns of this CTA
  static constexpr int NH = BN == 512 ? 2 : 1;       // products of 256 columns
  static constexpr int STAGES = BN == 512 ? 4 : BN == 256 ? 6 : 8;
  static constexpr int CONV = BN == 512 ? 2 : 3;     // converted tiles in flight, one group of warps each
  static constexpr int GROUP_WARPS = BN == 512 ? 8 : 4;
  static constexpr int THREADS = (7 + CONV * GROUP_WARPS) * 32;
  static constexpr int CHAIN = BN == 512 ? 44 : 20;  // k-blocks that one chain of accumulations runs over at most
  static constexpr int WORDS = BNL > 128 ? 2 : 1;    // 4-byte words of steps per row
  alignas(1024) uint8_t a[STAGES][BM * BK * 2];      // dY: two panels [64 rows][128 bytes], swizzled
  alignas(1024) uint8_t b[CONV][BNL * BK * 2];       // X as bf16: BNL / 64 such panels
  alignas(1024) uint8_t c[4][2][32 * 128];           // per epilogue warp: 32 rows x 32 fp32, swizzled, twice
  alignas(1024) uint8_t b8[STAGES][BK * BNL];        // codes [64 rows][BNL]
  alignas(16) uint8_t st[STAGES][BK * 4 * WORDS];    // step bytes [64 rows][4 WORDS]
  uint64_t full_a[STAGES], empty_a[STAGES], full_8[STAGES], empty_8[STAGES];
  uint64_t conv_full[CONV], conv_empty[CONV], acc_full[2], acc_empty[2];
  uint32_t tmem_base;
  int abort_flag;
};
// what a launch asks for: the members, and room to align them as far as an SM has it (the window starts on a
// multiple of 1,024 bytes in practice; the kernel checks)
template <int BN>
constexpr size_t smem_bytes() {
  const size_t used = (offsetof(Smem<BN>, abort_flag) + sizeof(int) + 15) / 16 * 16;
  return used + 1024 < 232448 ? used + 1024 : 232448;
}

struct Params {
  const uint8_t* steps;
  int64_t spitch;
  int R, N, C;
  int n_c, tiles, num_kb, kb_per, chain;
  int run, runs, rest;     // slices of an owner's piece, such pieces and single slices of a tile
  int accumulate;          // what is stored is added to what the result holds
  int* status;
};

// k-blocks [kb0, kb1) of a tile, whose sum goes to a plane
struct Piece {
  int tile, plane, kb0, kb1;
};
// The pieces of a pair of CTAs.  Where the slices of all tiles take `run` rounds of the pairs, a pair of the first
// runs * tiles ones takes that many slices of one tile, one after the other, into one plane; what slices are left the
// others take, all tiles of a slice before the next one's, a plane a slice.  So at any time the pairs read few
// different rows, and planes are few (32,780 x 5,472 x 1,024: three for five slices, 356 us against 361 in a row).
struct Walk {
  const Params& p;
  int64_t pos;
  int pairs;
  IMF_DEVICE Walk(const Params& prm, int pair, int n) : p(prm), pos(pair), pairs(n) {}
  IMF_DEVICE bool next(Piece& w) {
    const int64_t owners = (int64_t)p.runs * p.tiles;
    if (pos >= owners + (int64_t)p.tiles * p.rest) return false;
    const int64_t row = pos / p.tiles;
    w.tile = (int)(pos - row * p.tiles);
    w.plane = (int)row;
    const bool owner = pos < owners;
    const int first = owner ? (int)row * p.run : p.runs * p.run + (int)(row - p.runs);
    w.kb0 = first * p.kb_per;
    w.kb1 = min(w.kb0 + (owner ? p.run * p.kb_per : p.kb_per), p.num_kb);
    pos += owner ? owners + (int64_t)p.tiles * p.rest : pairs - owners;
    return true;
  }
};

IMF_DEVICE void cp_async4(void* dst, const void* src, bool in) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(in ? 4 : 0)
               : "memory");
}
IMF_DEVICE void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
IMF_DEVICE void tma_reduce_add_3d(const CUtensorMap* m, const void* src, int c0, int c1, int c2) {
  asm volatile("cp.reduce.async.bulk.tensor.3d.global.shared::cta.add.tile.bulk_group [%0, {%2, %3, %4}], [%1];"
               ::"l"(reinterpret_cast<uint64_t>(m)), "r"(smem_u32(src)), "r"(c0), "r"(c1), "r"(c2)
               : "memory");
}
// all but the newest bulk store have read their source
IMF_DEVICE void tma_store_wait_read1() { asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory"); }

// given up after `it` k-blocks: see the copies in flight land (bounded)
IMF_DEVICE void see_landed(uint64_t* full, uint32_t stages, uint32_t it) {
  for (uint32_t j = it < stages ? 0 : it - stages; j < it; ++j)
    for (int spin = 0; spin < 100000 && !mbar_test(&full[j % stages], (j / stages) & 1); ++spin) {
    }
}

// ---- the pair of CTAs
IMF_DEVICE uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
IMF_DEVICE void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
IMF_DEVICE void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
// Arrive on the first CTA's barrier, for what the arriving thread's own CTA is read by: products that take this CTA's dY
// and converted tile from its shared memory through the async proxy.  The writes are in place before the arrival leaves:
// dY's by the barrier that this thread has waited for, the tile's by its writers' proxy fences and the warp's barrier.
// No thread of the other CTA reads anything that this one wrote, so the order that the arrival gives within this
// CTA is enough (a release at cluster scope here waits for everything the thread has in flight: 627 us for 322).
IMF_DEVICE void arrive_first(uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .b32 ra;\n\t"
      "mapa.shared::cluster.u32 ra, %0, 0;\n\t"
      "mbarrier.arrive.shared::cluster.b64 _, [ra];\n\t}" ::"r"(smem_u32(bar))
      : "memory");
}
// The same, ordered over the cluster, and its waiter's part: an accumulator has been read, once a chain of products
// (32,780 x 5,472 x 1,024: 334 us; without the order 328, and 338 behind the last store instead of the last read).
IMF_DEVICE void arrive_first_cluster(uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .b32 ra;\n\t"
      "mapa.shared::cluster.u32 ra, %0, 0;\n\t"
      "mbarrier.arrive.release.cluster.shared::cluster.b64 _, [ra];\n\t}" ::"r"(smem_u32(bar))
      : "memory");
}
IMF_DEVICE bool acquire_cluster(uint64_t* bar, uint32_t parity) {     // a phase that has ended
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.b32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
// the arrival, in both CTAs, of this thread's products so far
IMF_DEVICE void commit_both(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"((uint16_t)3)
      : "memory");
}
IMF_DEVICE void mma_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

template <int BN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(Smem<BN>::THREADS, 1)
wgrad8_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
              const __grid_constant__ CUtensorMap tm_c, const __grid_constant__ Params p) {
  extern __shared__ uint8_t smem_raw[];
  using S = Smem<BN>;
  constexpr int STAGES = S::STAGES, BNL = S::BNL, CONV = S::CONV, GROUP_WARPS = S::GROUP_WARPS,
                NH = S::NH, WORDS = S::WORDS, PN = BN / NH;      // PN: columns of a product
  // the same offset in both CTAs, whose windows start alike: the products address them by one descriptor
  const uint32_t pad = (1024 - (smem_u32(smem_raw) & 1023)) % 1024;
  if (pad + offsetof(S, abort_flag) + sizeof(int) > smem_bytes<BN>()) {
    if (threadIdx.x == 0 && p.status) atomicCAS(p.status, 0, STATUS_BAD_ARG);
    return;
  }
  auto& s = *reinterpret_cast<S*>(smem_raw + pad);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)cluster_rank(), pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  if (threadIdx.x == 0) {
    prefetch_tmap(&tm_a);
    prefetch_tmap(&tm_b);
    prefetch_tmap(&tm_c);
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&s.full_8[i], 1 + 32);               // the bytes' announcement, and each lane's step bytes
      mbar_init(&s.empty_8[i], GROUP_WARPS);
      mbar_init(&s.full_a[i], rank == 0 ? 2 : 1);    // the bytes' announcement; in the first CTA: the other has its own
      mbar_init(&s.empty_a[i], 1);
    }
    for (int i = 0; i < CONV; ++i) {
      mbar_init(&s.conv_full[i], 2 * GROUP_WARPS);   // one arrival per warp of the group, from both CTAs
      mbar_init(&s.conv_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s.acc_full[i], 1);
      mbar_init(&s.acc_empty[i], 2 * 4);
    }
    s.abort_flag = 0;
    fence_barrier_init();
  }
  __syncthreads();
  if (warp == 5) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s.tmem_base)),
                 "r"(512u)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  cluster_arrive();
  // the loading warps touch nothing of the other CTA, nor TMEM: they begin, and wait for it at their end
  const bool loads = warp == 4 || warp == 6;
  if (!loads) cluster_wait();
  tc_fence_after();
  const uint32_t tmem = loads ? 0u : s.tmem_base;
  volatile int* abort_flag = &s.abort_flag;
  Walk walk(p, pair, pairs);
  Piece w;
  const auto m_of = [&](int tile) { return tile / p.n_c * (2 * BM) + rank * BM; };     // first row of this CTA
  const auto n_of = [&](int tile) { return tile % p.n_c * BN; };

  if (warp == 4) {
    // ---------------------------------------------------------------- dY --
    if (elect_one()) {
      uint32_t it = 0;
      bool ok = true;
      while (ok && walk.next(w)) {
        const int m0 = m_of(w.tile);
        for (int kb = w.kb0; kb < w.kb1; ++kb, ++it) {
          const int st = it % STAGES, k0 = kb * BK;
          if (it >= STAGES)
            ok = mbar_wait(&s.empty_a[st], ((it / STAGES) & 1) ^ 1, abort_flag, p.status, STATUS_TIMEOUT_EMPTY);
          if (!ok) break;
          mbar_arrive_expect_tx(&s.full_a[st], BM * BK * 2);
          tma_load_2d(s.a[st], &tm_a, &s.full_a[st], m0, k0);
          tma_load_2d(s.a[st] + BK * 128, &tm_a, &s.full_a[st], m0 + 64, k0);
        }
      }
      if (!ok) see_landed(s.full_a, STAGES, it);
    }
  } else if (warp == 6) {
    // --------------------------------------------------- codes and steps --
    uint32_t it = 0;
    bool ok = true;
    while (ok && walk.next(w)) {
      const int n0 = n_of(w.tile) + rank * BNL;
      const int64_t g = n0 / 128 * 4;                // the word with the steps of these columns
      for (int kb = w.kb0; kb < w.kb1; ++kb, ++it) {
        const int st = it % STAGES, k0 = kb * BK;
        if (it >= STAGES)
          ok = __all_sync(0xffffffffu, mbar_wait(&s.empty_8[st], ((it / STAGES) & 1) ^ 1, abort_flag, p.status,
                                                    STATUS_TIMEOUT_EMPTY));
        if (!ok) break;
        if (lane == 0) {
          mbar_arrive_expect_tx(&s.full_8[st], BK * BNL);
          tma_load_2d(s.b8[st], &tm_b, &s.full_8[st], n0, k0);
        }
#pragma unroll
        for (int i = 0; i < 2 * WORDS; ++i) {        // rows and words past the end: zeros, nothing is read
          const int r = i / WORDS * 32 + lane, w4 = i % WORDS;
          const bool in = k0 + r < p.R && g + 4 * w4 < p.spitch;
          cp_async4(s.st[st] + (r * WORDS + w4) * 4, in ? p.steps + (int64_t)(k0 + r) * p.spitch + g + 4 * w4 : p.steps,
                    in);
        }
        cp_async_arrive(&s.full_8[st]);
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (!ok) see_landed(s.full_8, STAGES, it);
  } else if (warp == 5 && rank == 1) {
    // ------------------------------------ tells the first CTA of its dY --
    if (elect_one()) {
      uint32_t it = 0;
      bool ok = true;
      while (ok && walk.next(w))
        for (int kb = w.kb0; kb < w.kb1 && ok; ++kb, ++it) {
          ok = mbar_wait(&s.full_a[it % STAGES], (it / STAGES) & 1, abort_flag, p.status, STATUS_TIMEOUT_TMA);
          if (ok) arrive_first(&s.full_a[it % STAGES]);
        }
    }
  } else if (warp == 5) {
    // --------------------------------------------------------------- MMA --
    if (elect_one()) {
      constexpr uint32_t idesc = idesc_bf16(2 * BM, PN, 1, 1);
      uint32_t it = 0, ch = 0, total = 0;            // k-blocks and chains so far, k-blocks in all
      for (Walk all = walk; all.next(w);) total += w.kb1 - w.kb0;
      bool ok = true;
      while (ok && walk.next(w)) {
        for (int c0 = w.kb0; c0 < w.kb1 && ok; c0 += p.chain, ++ch) {
          const int c1 = min(c0 + p.chain, w.kb1);
          for (int kb = c0; kb < c1; ++kb, ++it) {
            const int st = it % STAGES, cs = it % CONV;
            ok = mbar_wait(&s.full_a[st], (it / STAGES) & 1, abort_flag, p.status, STATUS_TIMEOUT_TMA) &&
                 mbar_wait(&s.conv_full[cs], (it / CONV) & 1, abort_flag, p.status, STATUS_TIMEOUT_TMA);
            if (!ok) break;
            const uint32_t a_base = smem_u32(s.a[st]), b_base = smem_u32(s.b[cs]);
#pragma unroll
            for (int h = 0; h < NH; ++h) {
              // the accumulator: one of two that take turns, or the half of the only one
              const uint32_t acc = NH == 2 ? h : ch & 1, turns = NH == 2 ? ch : ch >> 1;
              if (kb == c0 && turns > 0)
                ok = mbar_wait(&s.acc_empty[acc], (turns - 1) & 1, abort_flag, p.status, STATUS_TIMEOUT_SOFTMAX) &&
                     acquire_cluster(&s.acc_empty[acc], (turns - 1) & 1);
              if (!ok) break;
              tc_fence_after();
#pragma unroll
              for (int ks = 0; ks < BK / 16; ++ks)
                mma_pair(tmem + acc * 256, sdesc_mnmajor(a_base + ks * 2048, BK * 128),
                         sdesc_mnmajor(b_base + h * (PN / 2 * BK * 2) + ks * 2048, BK * 128), idesc,
                         kb != c0 || ks != 0);
              if (kb + 1 == c1) commit_both(&s.acc_full[acc]);
            }
            if (!ok) break;
            // slots that are used again; nobody would wait for the other arrivals, which might then find the other
            // CTA gone
            if (it + CONV < total) commit_both(&s.conv_empty[cs]);
            if (it + STAGES < total) commit_both(&s.empty_a[st]);
          }
        }
      }
    }
  } else if (warp >= 7) {
    // -------------------------------------------------------- conversion --
    // a lane owns eight codes of a row: a warp reads whole rows, and eight lanes write the eight 16-byte
    // chunks of a panel's line, no bank twice.  Its rows are a multiple of eight apart, so its place in a
    // line, and every address but for a constant, stays the same
    constexpr int LANES = BNL / 8, ROWS = 32 / LANES;    // lanes of a row, rows a warp takes at a time
    constexpr int STEP = GROUP_WARPS * ROWS, UNITS = BK / STEP;
    static_assert(STEP % 8 == 0, "rows of a lane keep their place in the swizzle");
    const int grp = (warp - 7) / GROUP_WARPS, col = lane % LANES;
    const int r0 = ((warp - 7) % GROUP_WARPS) * ROWS + lane / LANES;
    uint8_t* const dst = s.b[grp] + (col / 8) * (BK * 128) + r0 * 128 + (((col & 7) ^ (r0 & 7)) << 4);
    uint32_t it = 0;
    bool ok = true;
    while (ok && walk.next(w)) {
      const int st0 = r0 * 4 * WORDS + ((n_of(w.tile) + rank * BNL) / 32 & 3) + col / 4;
      for (int kb = w.kb0; kb < w.kb1; ++kb, ++it) {
        if ((int)(it % CONV) != grp) continue;
        const int st = it % STAGES;
        ok = __all_sync(0xffffffffu, mbar_wait(&s.full_8[st], (it / STAGES) & 1, abort_flag, p.status,
                                               STATUS_TIMEOUT_TMA));
        if (!ok) break;
        // converted into registers while products still read the tile; what is left between their end
        // and the next ones are the stores
        const uint8_t *src = s.b8[st] + r0 * BNL + col * 8, *steps = s.st[st] + st0;
        uint2 codes[UNITS];
        uint32_t step[UNITS];
        uint4 v[UNITS];
#pragma unroll
        for (int j = 0; j < UNITS; ++j) {
          codes[j] = *reinterpret_cast<const uint2*>(src + j * STEP * BNL);
          step[j] = steps[j * STEP * 4 * WORDS];
        }
#pragma unroll
        for (int j = 0; j < UNITS; ++j) {
          v[j] = a8_decode8(codes[j], a8_step2(step[j]));
          asm volatile("" : "+r"(v[j].x), "+r"(v[j].y), "+r"(v[j].z), "+r"(v[j].w));   // here, not behind the wait
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.empty_8[st]);
        if (it >= CONV)
          ok = __all_sync(0xffffffffu, mbar_wait(&s.conv_empty[grp], ((it / CONV) & 1) ^ 1, abort_flag,
                                                    p.status, STATUS_TIMEOUT_MMA));
        if (!ok) break;
#pragma unroll
        for (int j = 0; j < UNITS; ++j) *reinterpret_cast<uint4*>(dst + j * STEP * 128) = v[j];
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) arrive_first(&s.conv_full[grp]);
      }
    }
  } else {
    // ---------------------------------------------------------- epilogue --
    uint32_t ch = 0, step = 0, chains = 0;           // chains so far, in all
    for (Walk all = walk; all.next(w);) chains += (w.kb1 - w.kb0 + p.chain - 1) / p.chain;
    bool ok = true;
    while (ok && walk.next(w)) {
      const int row0 = m_of(w.tile) + warp * 32, n0 = n_of(w.tile);
      for (int c0 = w.kb0; c0 < w.kb1 && ok; c0 += p.chain, ++ch) {
        const bool add = p.accumulate || c0 != w.kb0;
        if (c0 != w.kb0 && lane == 0) tma_store_wait_all();          // the chain before is in memory
#pragma unroll 1
        for (int h = 0; h < NH; ++h) {
          const uint32_t acc = NH == 2 ? h : ch & 1, turns = NH == 2 ? ch : ch >> 1;
          ok = __all_sync(0xffffffffu, mbar_wait(&s.acc_full[acc], turns & 1, abort_flag, p.status, STATUS_TIMEOUT_MMA));
          if (!ok) break;
          tc_fence_after();
          bool read = false;                         // told that the accumulator is free
          const auto done = [&] {
            tc_fence_before();
            __syncwarp();
            if (lane == 1 && ch + (NH == 2 ? 1 : 2) < chains) arrive_first_cluster(&s.acc_empty[acc]);   // used again
            read = true;
          };
#pragma unroll 1
          for (int c = 0; c < PN && row0 < p.N; c += 32) {
            // column of the product -> of the tile: its first half is the first CTA's
            const int n = n0 + (NH == 1 ? c : (c & 128) * 2 + h * 128 + (c & 127));
            if (n >= p.C) continue;
            uint32_t r[32];
            tmem_ld32(tmem_addr(tmem + acc * 256, warp * 32, c), r);
            if (lane == 0) tma_store_wait_read1();
            __syncwarp();
            tc_wait_ld();
            if (c + 32 == PN) done();
            uint8_t *stage = s.c[warp][step++ & 1], *line = stage + lane * 128;
#pragma unroll
            for (int i = 0; i < 8; ++i)
              *reinterpret_cast<uint4*>(line + ((i ^ (lane & 7)) << 4)) =
                  make_uint4(r[4 * i], r[4 * i + 1], r[4 * i + 2], r[4 * i + 3]);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              if (add) tma_reduce_add_3d(&tm_c, stage, n, row0, w.plane);
              else tma_store_3d(&tm_c, stage, n, row0, w.plane);
              tma_store_commit();
            }
          }
          if (!read) done();
        }
      }
    }
    if (lane == 0) tma_store_wait_all();
    tc_fence_before();
  }
  if (loads) cluster_wait();
  __syncthreads();
  cluster_arrive();
  cluster_wait();            // the other CTA's products have read this one's tiles
  if (warp == 5) {
    __syncwarp();
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
}

static int sm_count() {
  static int sms_of[HOST_MAX_DEVICES] = {0};
  int dev = 0;
  cudaGetDevice(&dev);
  int sms = (dev >= 0 && dev < HOST_MAX_DEVICES) ? sms_of[dev] : 0;
  if (!sms) {
    if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms <= 0) sms = 148;
    if (dev >= 0 && dev < HOST_MAX_DEVICES) sms_of[dev] = sms;
  }
  return sms;
}

struct Plan {
  int bn, kb_per, pairs;
  int run, runs, rest;     // see Walk
  int planes() const { return runs + rest; }
};

// Tile width and slices: the least time among the counts that fill one, two or three rounds of pairs (and one
// slice).  In us, measured on full clips and short ones: a k-block, what a tile costs besides (the
// store of its accumulator above all), and 5 + 0.22 a MB for planes and the kernel that adds them up.  Widths against
// each other: 32,780 x 2,064 x 1,024 141 us (512) and 162 (256); 32,780 x 1,024 x 512 53 and 49; 2,068 x 1,376
// x 256 20.5 (256) and 18.4 (128).
static Plan plan(int R, int N, int C, int sms) {
  const int num_kb = (R + BK - 1) / BK, most = sms > 1 ? sms / 2 : 1;
  Plan best{128, num_kb, 1, 1, 1, 0};
  double least = 1e30;
  for (int bn = 128; bn <= 512; bn *= 2) {
    const double kb_us = bn == 512 ? 0.82 : bn == 256 ? 0.50 : 0.45, tile_us = bn == 512 ? 6 : bn == 256 ? 3.5 : 2.5;
    const int64_t tiles = (int64_t)((N + 2 * BM - 1) / (2 * BM)) * ((C + bn - 1) / bn);
    for (int rounds = 0; rounds <= 3; ++rounds) {
      int64_t want = rounds ? rounds * most / tiles : 1;
      if (want > num_kb / 2) want = num_kb / 2;        // two k-blocks a slice at least
      if (want < 1) want = 1;
      const int per = (int)((num_kb + want - 1) / want), sp = (num_kb + per - 1) / per;
      const int64_t pieces = tiles * sp, lines = (pieces + most - 1) / most;
      const int run = (int)(lines < sp ? lines : sp), runs = tiles <= most ? sp / run : 0, rest = sp - runs * run;
      double cost = (double)lines * (per * kb_us + tile_us);
      if (runs + rest > 1) cost += 5.0 + 0.22 * ((runs + rest) * (4e-6 * N * C));
      if (cost < least) {
        least = cost;
        const int64_t walks = tiles * (runs + rest);
        best = Plan{bn, per, (int)(walks < most ? walks : most), run, runs, rest};
      }
    }
  }
  return best;
}

template <int BN>
static int launch(const void* dy, int64_t ld_dy, const void* codes, const void* steps, int R, int N, int C,
                  float* dst, int64_t ld_dst, int64_t plane, int accumulate, const Plan& pl, int* status, cudaStream_t st) {
  CUtensorMap ta, tb, tc;
  int rc;
  {
    uint64_t dims[2] = {(uint64_t)N, (uint64_t)R}, str[2] = {2, (uint64_t)ld_dy * 2};
    uint32_t box[2] = {64, BK};
    if ((rc = make_tmap(&ta, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(dy), dims, str, box))) return rc;
  }
  const uint64_t pitch = ((uint64_t)C + 31) / 32 * 32;
  {
    uint64_t dims[2] = {pitch, (uint64_t)R}, str[2] = {1, pitch};
    uint32_t box[2] = {BN / 2, BK};
    if ((rc = make_tmap(&tb, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(codes), dims, str, box,
                        CU_TENSOR_MAP_SWIZZLE_NONE)))
      return rc;
  }
  {
    uint64_t dims[3] = {(uint64_t)C, (uint64_t)N, (uint64_t)pl.planes()};
    uint64_t str[3] = {4, (uint64_t)ld_dst * 4, (uint64_t)plane * 4};
    uint32_t box[3] = {32, 32, 1};
    if ((rc = make_tmap(&tc, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, dst, dims, str, box))) return rc;
  }
  Params p;
  p.steps = static_cast<const uint8_t*>(steps);
  p.spitch = (int64_t)(pitch / 32 + 3) / 4 * 4;
  p.R = R; p.N = N; p.C = C;
  p.n_c = (C + BN - 1) / BN;
  p.tiles = (N + 2 * BM - 1) / (2 * BM) * p.n_c;
  p.num_kb = (R + BK - 1) / BK;
  p.run = pl.run;
  p.runs = pl.runs;
  p.rest = pl.rest;
  p.kb_per = pl.kb_per;
  const int chains = (pl.kb_per + Smem<BN>::CHAIN - 1) / Smem<BN>::CHAIN;
  p.chain = (pl.kb_per + chains - 1) / chains;
  p.accumulate = accumulate;
  p.status = status;
  const size_t smem = smem_bytes<BN>();
  static bool allowed[HOST_MAX_DEVICES] = {false};
  if (!allow_smem((const void*)wgrad8_kernel<BN>, smem, allowed)) return IMF_ERR_LAUNCH;
  wgrad8_kernel<BN><<<(unsigned)pl.pairs * 2, Smem<BN>::THREADS, smem, st>>>(ta, tb, tc, p);
  return cudaGetLastError() == cudaSuccess ? IMF_OK : IMF_ERR_LAUNCH;
}

static int64_t plane_floats(int N, int C) { return (int64_t)N * (((int64_t)C + 3) & ~int64_t(3)); }

}  // namespace w8
}  // namespace imf

// Whether TMA may write a result in place: 16-byte rows, and a width of whole 16 bytes, for it writes those of the last
// columns whole (what lies behind a band's 738 columns was overwritten up to 740).
static bool in_place(const float* out, int64_t ldo, int C) {
  return (ldo & 3) == 0 && (C & 3) == 0 && (reinterpret_cast<uintptr_t>(out) & 15u) == 0;
}

// Floats of workspace that imf_wgrad8 wants for these sizes and this result.
extern "C" int64_t imf_wgrad8_work(int R, int N, int C, const float* out, int64_t ldo) {
  using namespace imf;
  if (R <= 0 || N <= 0 || C <= 0) return 0;
  const w8::Plan pl = w8::plan(R, N, C, w8::sm_count());
  return pl.planes() > 1 || !in_place(out, ldo, C) ? pl.planes() * w8::plane_floats(N, C) : 0;
}

extern "C" int imf_splitk_reduce_ld(const float* partial, int splits, int M, int N, int64_t ldp, int64_t plane, float* out,
                                    int64_t ldo, float alpha, int accumulate, void* stream);

// dy [R, N] bf16 (row pitch ld_dy), codes / steps: checkpoint of X [R, C]; out [N, C] fp32 (row pitch ldo).
extern "C" int imf_wgrad8(const void* dy, int64_t ld_dy, const void* codes, const void* steps, int R, int N, int C,
                          float* out, int64_t ldo, int accumulate, float* work, int64_t work_floats, int* status,
                          void* stream) {
  using namespace imf;
  if (R <= 0 || N <= 0 || C <= 0 || !dy || !codes || !steps || !out || (ld_dy & 7)) return IMF_ERR_ARG;
  if (R > 0x7fffff00 || N > 0x7fffff00 || C > 0x7ffffe00) return IMF_ERR_TOO_LARGE;
  if ((reinterpret_cast<uintptr_t>(codes) & 15u) || (reinterpret_cast<uintptr_t>(steps) & 3u)) return IMF_ERR_ARG;
  const w8::Plan pl = w8::plan(R, N, C, w8::sm_count());
  if ((int64_t)((N + 255) / 256) * ((C + pl.bn - 1) / pl.bn) * pl.planes() > 0x7fffffff) return IMF_ERR_TOO_LARGE;
  const bool direct = pl.planes() == 1 && in_place(out, ldo, C);
  const int64_t plane = w8::plane_floats(N, C), cp = plane / N;
  if (!direct && (!work || work_floats < pl.planes() * plane || (reinterpret_cast<uintptr_t>(work) & 15u)))
    return IMF_ERR_ARG;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto go = pl.bn == 512 ? w8::launch<512> : pl.bn == 256 ? w8::launch<256> : w8::launch<128>;
  const int rc = direct ? go(dy, ld_dy, codes, steps, R, N, C, out, ldo, (int64_t)N * ldo, accumulate, pl, status, st)
                        : go(dy, ld_dy, codes, steps, R, N, C, work, cp, plane, 0, pl, status, st);
  if (rc || direct) return rc;
  return imf_splitk_reduce_ld(work, pl.planes(), N, C, cp, plane, out, ldo, 1.f, accumulate, stream);
}
