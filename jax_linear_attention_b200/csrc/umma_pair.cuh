// Tensor-core primitives beyond umma.cuh: products of e4m3 operands, clusters of CTAs, and pairs of CTAs that work on
// one tile (cta_group::2).
//
// A pair computes D (256 x N) = A B: each CTA holds 128 rows of A and the accumulators of those rows (its own TMEM), and
// half of B (N / 2 of its rows, or columns in the MN-major view); the tensor core reads the other half of B from the other
// CTA's shared memory at the same offset. One thread of CTA 0 (the leader) issues the instructions for both.
#pragma once

#include "umma.cuh"

namespace jla {
namespace umma {

// ---- clusters --------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {  // every thread of every CTA of the cluster
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
// The same in two halves: what must have happened before, and where it must have. Once each for every thread, in this order.
__device__ __forceinline__ void cluster_arrive() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  __syncwarp();
  asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
// shared::cluster address of what lies at `addr` in this CTA, in the CTA of rank `rank`
__device__ __forceinline__ uint32_t map_rank(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
// `bytes` (a multiple of 16) of this CTA's shared memory to `dst` in another CTA's, counted on a barrier of that CTA; the
// source has to be fenced (fence_async_smem) and to stay as it is until they have arrived.
__device__ __forceinline__ void copy_cluster(uint32_t dst, uint32_t src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n" ::"r"(dst),
               "r"(src), "r"(bytes), "r"(bar)
               : "memory");
}
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];\n" ::"r"(bar) : "memory");
}

// ---- roles of one warp -----------------------------------------------------------------------------------------
// A warp that issues copies or products runs its loop with all lanes, so that its counters and addresses stay in uniform
// registers, and lets one lane issue; a loop that one lane runs alone takes about three times as long a step.
__device__ __forceinline__ bool elect_one() {
  uint32_t mine;
  asm volatile(
      "{\n.reg .pred p;\n"
      "elect.sync _|p, 0xffffffff;\n"
      "selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(mine));
  return mine != 0;
}
// mbar_wait by a whole warp: false, for all lanes alike, where the phase did not complete within the spin limit.
__device__ __forceinline__ bool mbar_wait_warp(uint32_t bar, uint32_t parity) {
  for (uint32_t spin = 0; spin < kSpinLimit; ++spin) {
    uint32_t done;
    asm volatile(
        "{\n.reg .pred p;\n"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
        "selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    if (__all_sync(0xffffffffu, done)) return true;
  }
  return false;
}

// ---- instruction descriptor of kind::f8f6f4 with e4m3 operands, fp32 accumulators; both operands K-major -------------
__host__ __device__ constexpr uint32_t instr_desc_e4m3(int M, int N) {
  return (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

// ---- one CTA ----------------------------------------------------------------------------------------------------
// 32 bytes of each operand row's contraction a step: 16 elements of kind::f16, 32 of kind::f8f6f4.
template <bool FP8>
__device__ __forceinline__ void mma_any(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, bool accumulate) {
  if constexpr (!FP8) {
    mma(d_tmem, a_desc, b_desc, idesc, accumulate);
  } else {
    asm volatile(
        "{\n.reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}\n" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"((uint32_t)accumulate)
        : "memory");
  }
}

// ---- sums in TMEM ------------------------------------------------------------------------------------------------
// 16 columns of the 32 lanes of a warp: sum = part, or sum += part.
__device__ __forceinline__ void ld_32x32b_x16(uint32_t (&r)[16], uint32_t taddr) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void join_x16(uint32_t sum, uint32_t part, bool first) {
  uint32_t v[16], t[16];
  ld_32x32b_x16(v, part);
  if (!first) ld_32x32b_x16(t, sum);
  wait_ld();
  if (!first) {
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) + __uint_as_float(t[j]));
  }
  st_32x32b_x16(sum, v);
}

// ---- a pair of CTAs -----------------------------------------------------------------------------------------------
// One warp of EACH CTA allocates (and at the end frees) the same number of columns.
__device__ __forceinline__ void tmem_alloc_pair(uint32_t* slot, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_addr(slot)), "r"(cols)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc_pair(uint32_t base, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;\n" ::"r"(base), "r"(cols) : "memory");
}
template <bool FP8>
__device__ __forceinline__ void mma_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, bool accumulate) {
  if constexpr (!FP8) {
    asm volatile(
        "{\n.reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"((uint32_t)accumulate)
        : "memory");
  } else {
    asm volatile(
        "{\n.reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n}\n" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"((uint32_t)accumulate)
        : "memory");
  }
}
// Arrive on the barrier at this offset in BOTH CTAs once all products issued so far by this thread have completed.
__device__ __forceinline__ void commit_pair(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n" ::"r"(
          smem_addr(bar)),
      "h"((uint16_t)3)
      : "memory");
}

}  // namespace umma
}  // namespace jla
