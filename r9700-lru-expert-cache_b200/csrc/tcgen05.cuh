// tcgen05, tensor-map and thread-block-cluster primitives (sm_100a) of the scoring kernels.
#pragma once
#include <cuda.h>
#include "common.cuh"

namespace b200 {

// ---- ordering, descriptors, MMA --------------------------------------------------------------

B200_DEVINL void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
B200_DEVINL void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// Shared-memory matrix descriptor: K-major rows of 128 B, 128-byte swizzle, 8-row groups 1024 B apart.
B200_DEVINL uint64_t sw128_desc(uint32_t saddr) {
  uint64_t d = (uint64_t)((saddr & 0x3FFFFu) >> 4);      // start address, bits [0, 14)
  d |= (uint64_t)1 << 16;                                // leading byte offset (unused with this swizzle)
  d |= (uint64_t)(1024 >> 4) << 32;                      // stride byte offset
  d |= (uint64_t)1 << 46;                                // descriptor version
  d |= (uint64_t)2 << 61;                                // 128-byte swizzle
  return d;
}

// True in one lane of a converged warp.
B200_DEVINL bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(p));
  return p != 0;
}

// D (f32, TMEM) = or += A B^T for one K = 32 step, A and B e4m3 in shared memory. CG CTAs share the tile.
template <int CG>
B200_DEVINL void tc_mma_f8(uint32_t tmem_d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if constexpr (CG == 1)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(tmem_d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate));
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(tmem_d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate));
}

// One arrival on `bar` (for CG = 2: on the barrier at the same place in both CTAs) once every MMA that
// this thread has issued is complete.
template <int CG>
B200_DEVINL void tc_commit(uint64_t* bar) {
  if constexpr (CG == 1)
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                 : "memory");
  else
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            smem_u32(bar)),
        "h"((uint16_t)3)
        : "memory");
}

template <int CG>
B200_DEVINL void tmem_alloc_512(uint32_t* slot) {
  if constexpr (CG == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(slot)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  } else {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(slot)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
}

template <int CG>
B200_DEVINL void tmem_dealloc_512(uint32_t tmem) {
  if constexpr (CG == 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  else
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

// 16 fp32 columns of the warp's 32 TMEM lanes.
B200_DEVINL void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}

// Waits for the warp's TMEM loads. The values are tied to the wait, so that none is used before it.
B200_DEVINL void tmem_wait_ld16(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]),
                 "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                 "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}

// (a.x, a.y) += (v0 s, v1 s) in one instruction.
B200_DEVINL void fma2_scaled(float2& a, uint32_t v0, uint32_t v1, float s) {
  unsigned long long acc = ((unsigned long long)__float_as_uint(a.y) << 32) | __float_as_uint(a.x);
  const unsigned long long v = ((unsigned long long)v1 << 32) | v0;
  const unsigned long long c = ((unsigned long long)__float_as_uint(s) << 32) | __float_as_uint(s);
  asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc) : "l"(v), "l"(c));
  a.x = __uint_as_float((uint32_t)acc);
  a.y = __uint_as_float((uint32_t)(acc >> 32));
}

// ---- clusters ----------------------------------------------------------------------------------

B200_DEVINL uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
B200_DEVINL uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
B200_DEVINL void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
B200_DEVINL void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
B200_DEVINL void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
B200_DEVINL void st_cluster(uint32_t cluster_addr, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cluster_addr), "r"(v) : "memory");
}
// The shared::cluster address of this CTA's shared address in CTA `rank` of the cluster.
B200_DEVINL uint32_t map_to_rank(uint32_t saddr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(saddr), "r"(rank));
  return r;
}
// Arrival on another CTA's barrier. Of CTA scope: it orders nothing in memory across the CTAs (the caller's
// TMEM loads are complete before it); a release of cluster scope cost about 2000 clocks each.
B200_DEVINL void mbar_arrive_remote(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
B200_DEVINL void st_cluster_f4(uint32_t cluster_addr, float4 v) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1,%2,%3,%4};" ::"r"(cluster_addr), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w)
               : "memory");
}

// ---- bounded waits -----------------------------------------------------------------------------
//
// A wait on a barrier that is already there takes 110 to 160 clocks, and a try that fails suspends its thread
// for up to 7800 (4 us) unless the phase completes: so a loop of tries is bounded by their number, and warps that
// need two barriers wait for both at once, on different lanes.

constexpr uint32_t WAIT_TRIES = 1u << 18;            // about a second
// Waits for a phase, with `tries` tries. false: it did not come (or tries is 0), and the caller records an error and
// leaves.
B200_DEVINL bool mbar_wait_limited(uint64_t* bar, uint32_t parity, uint32_t tries) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .u32 n;\n\tmov.u32 n, 0;\n"
      "TRY_%=:\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t@p bra DONE_%=;\n\t"
      "add.u32 n, n, 1;\n\tsetp.lt.u32 q, n, %3;\n\t@q bra TRY_%=;\n"
      "DONE_%=:\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity), "r"(tries)
      : "memory");
  return ok != 0 && tries != 0;
}
// The warp waits for `bar` and, where `both`, for `other` too. Uniform. What either barrier guards is there for
// every lane, although each lane waited for one of them: the vote alone would let a load be moved ahead of it.
B200_DEVINL bool warp_wait(uint64_t* bar, uint32_t parity, uint64_t* other, uint32_t other_parity, bool both,
                           uint32_t tries) {
  const bool second = both && (lane_id() & 1);
  const bool ok = __all_sync(0xffffffffu, mbar_wait_limited(second ? other : bar, second ? other_parity : parity, tries));
  __syncwarp();
  return ok;
}
B200_DEVINL bool warp_wait(uint64_t* bar, uint32_t parity, uint32_t tries) {
  return __all_sync(0xffffffffu, mbar_wait_limited(bar, parity, tries));
}

// ---- tensor-map copies -------------------------------------------------------------------------

B200_DEVINL void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

// One box global -> this CTA's shared memory, its bytes counted on the barrier at `bar` (a shared::cluster
// address; for CG = 2 it may be the peer's).
template <int CG>
B200_DEVINL void tma_load_2d(uint32_t dst, const CUtensorMap* map, int c0, int c1, uint32_t bar) {
  if constexpr (CG == 1)
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
            dst),
        "l"(map), "r"(c0), "r"(c1), "r"(bar)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, "
        "%3}], [%4];" ::"r"(dst),
        "l"(map), "r"(c0), "r"(c1), "r"(bar)
        : "memory");
}
template <int CG>
B200_DEVINL void tma_load_4d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, int c3, uint32_t bar) {
  if constexpr (CG == 1)
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
        "[%6];" ::"r"(dst),
        "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3, "
        "%4, %5}], [%6];" ::"r"(dst),
        "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar)
        : "memory");
}

// One box of this CTA's shared memory -> global, in the thread's current bulk group. The shared writes must be
// fenced for the async proxy before it.
B200_DEVINL void tma_store_2d(const CUtensorMap* map, int c0, int c1, uint32_t src) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map), "r"(c0), "r"(c1),
               "r"(src)
               : "memory");
}
B200_DEVINL void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
// All but the thread's last N bulk groups have read their shared memory.
template <int N>
B200_DEVINL void bulk_wait_read() {
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
}
B200_DEVINL void bulk_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

}  // namespace b200
