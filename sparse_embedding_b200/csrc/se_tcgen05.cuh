// Tensor-core plumbing for sm_100a: tcgen05 matrix instructions with
// accumulators in tensor memory, operand descriptors, tiled TMA loads, and
// barrier waits that give up. Loads are local to a CTA (no multicast); with
// CG = 2 two CTAs of a cluster form one matrix unit (cta_group::2), each
// loading its own half of both operands.
#pragma once

#include <cuda.h>

#include "se_common.cuh"

namespace se_gpu {

// A wait gives up after `limit` clocks (kWaitClocks unless se_set_wait_limit
// changed it: seconds), or this many tries. In a healthy launch a wait takes
// microseconds. (Clocks, since a read of the nanosecond timer is slow enough
// to show in every wait.) The limit is looked at after a first look that failed:
// before it, its load would be in every wait (4096 x 1024 fp32 370 -> 383 us).
constexpr uint32_t kWaitTries = 1u << 30;
// Limits below this are kept by looking: a try suspends the thread for a time of its own choice.
constexpr long long kBriefClocks = 10000000ll;
// What a launch that gave up allows its copies and matrix instructions in flight, in all.
constexpr long long kDrainClocks = 2000000000ll;

__device__ __forceinline__ bool mbar_test_wait(uint64_t *bar, uint32_t parity) {
  uint32_t done;
  asm volatile("{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n"
               " selp.u32 %0, 1, 0, p;\n}"
               : "=r"(done)
               : "r"(smem_u32(bar)), "r"(parity)
               : "memory");
  return done != 0u;
}
// Waits for a barrier's phase; false when the limit ran out or another role
// of the CTA gave up (*given_up). The caller then leaves its loop. CALL: all but
// the first look as a call of a function, which leaves the caller's loop short
// (1000 x 517 fp32 159.7 us in place, 156.5 by call; but the matrices on chip 25.1
// and 26.6 at 128 x 64, and normalisation backward 173 and 175 at 32,768 x 4,096).
__device__ __forceinline__ bool wait_on(uint64_t *bar, uint32_t parity, volatile uint32_t *given_up, long long limit) {
  const bool brief = limit < kBriefClocks;
  const long long start = clock64();
  for (uint32_t n = 0; n < kWaitTries; ++n) {
    if (brief ? mbar_test_wait(bar, parity) : mbar_try_wait(bar, parity)) return true;
    if (*given_up || clock64() - start > limit) break;
  }
  *given_up = 1u;
  return false;
}
static __device__ __noinline__ bool wait_by_call(uint64_t *bar, uint32_t parity, volatile uint32_t *given_up, long long limit) {
  return wait_on(bar, parity, given_up, limit);
}
template <bool CALL>
__device__ __forceinline__ bool wait_or_give_up(uint64_t *bar, uint32_t parity, volatile uint32_t *given_up,
                                                long long limit) {
  if (mbar_test_wait(bar, parity)) return true;
  if constexpr (CALL) return wait_by_call(bar, parity, given_up, limit);
  else return wait_on(bar, parity, given_up, limit);
}
// A wait for what is in flight when a launch has given up: until clock `end`.
__device__ __forceinline__ void wait_until(uint64_t *bar, uint32_t parity, long long end) {
  while (!mbar_try_wait(bar, parity) && clock64() < end) {
  }
}
// One lane of the converged warp, the same one every time.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(p));
  return p != 0u;
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The address of this CTA's shared variable in the cluster's CTA `rank`.
__device__ __forceinline__ uint32_t mapa(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
// (Releases at the CTA's scope only: what it orders is tensor memory, by the
// tcgen05 fences; a wider release would wait for the thread's stores.)
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}

__device__ __forceinline__ void prefetch_map(const CUtensorMap *map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

// A box of a 3-D tensor map into shared memory, counted on `bar` (a shared::cluster address).
template <int CG>
__device__ __forceinline__ void tma_load(void *dst, const CUtensorMap *map, int x, int y, int z, uint32_t bar) {
  if constexpr (CG == 1) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
                 " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_u32(dst)), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
                 : "memory");
  } else {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2"
                 " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_u32(dst)), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
                 : "memory");
  }
}

// Descriptor of an operand tile in shared memory with 128-byte swizzle, 16-bit
// values. K-major: rows of 64 k-values (128 bytes), groups of 8 rows 1,024
// bytes apart. MN-major: rows of 64 mn-values, one per k; groups of 8 k-rows
// 1,024 bytes apart and the next 64 mn-values `mn_step` bytes on.
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr, uint32_t mn_step) {
  return uint64_t((addr & 0x3ffffu) >> 4) | (uint64_t(mn_step >> 4) << 16) | (uint64_t(1024u >> 4) << 32) |
         (uint64_t(1) << 46) | (uint64_t(2) << 61);
}
// Instruction descriptor: f16 operands, fp32 accumulators, M x N; b_mn: B is MN-major.
constexpr __host__ __device__ uint32_t mma_desc(int m, int n, bool b_mn) {
  return (1u << 4) | (b_mn ? 1u << 16 : 0u) | (uint32_t(n >> 3) << 17) | (uint32_t(m >> 4) << 24);
}

template <int CG>
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t desc, bool add) {
  if constexpr (CG == 1) {
    asm volatile("{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
                 " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a), "l"(b), "r"(desc),
                 "r"(uint32_t(add)));
  } else {
    asm volatile("{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
                 " tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a), "l"(b), "r"(desc),
                 "r"(uint32_t(add)));
  }
}
// Arrives on the barrier (in both CTAs with CG = 2) when the thread's matrix instructions are done.
template <int CG>
__device__ __forceinline__ void mma_commit(uint64_t *bar) {
  if constexpr (CG == 1) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                 : "memory");
  } else {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::
                     "r"(smem_u32(bar)),
                 "h"(uint16_t(3))
                 : "memory");
  }
}
template <int CG>
__device__ __forceinline__ void tmem_alloc(uint32_t *out, uint32_t columns) {
  if constexpr (CG == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(out)), "r"(columns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  } else {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(out)), "r"(columns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
}
template <int CG>
__device__ __forceinline__ void tmem_free(uint32_t addr, uint32_t columns) {
  if constexpr (CG == 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(columns));
  else
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(columns));
}
__device__ __forceinline__ void tmem_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// 32 accumulator columns of the warp's 32 rows: thread = row, register = column.
__device__ __forceinline__ void tmem_load32(uint32_t addr, float (&v)[32]) {
  uint32_t *r = reinterpret_cast<uint32_t *>(v);
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
               "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
               "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                 "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
                 "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
                 "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
               : "r"(addr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

}  // namespace se_gpu
