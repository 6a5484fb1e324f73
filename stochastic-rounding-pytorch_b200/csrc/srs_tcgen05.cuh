// The sm_100a instructions the matrix products are made of (tcgen05 MMA and TMEM,
// TMA box loads, mbarriers with bounded waits), as small inline functions.
//
// Every wait is bounded: a role that waits longer than kWaitCycles records where
// in a status word (in host memory, so that the host sees it without a copy), stops, and
// its CTA leaves after its copies had time to land.
#pragma once

#include <cstdint>
#include <cuda.h>
#include <cuda_runtime.h>

namespace srs {

constexpr int kSliceBytes = 128;  // bytes of k per pipeline stage and row (one swizzle row)
constexpr int kPanelBytes = 128 * kSliceBytes;   // 128 rows of an operand per stage
constexpr long long kWaitCycles = 4000000000ll;  // about 2 s

__device__ __forceinline__ uint32_t smem_address(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}

// The warp's index as a warp-uniform value, and one elected lane of the warp.  The
// load and MMA roles run with the whole warp in uniform control flow, and only the
// instruction itself is under the election: descriptors then stay in uniform
// registers (with the loop itself under `lane == 0`, moving them there for every
// MMA took 745 cycles a slice instead of the 512 of its FP8 MMAs).
__device__ __forceinline__ int warp_index() {
  return __shfl_sync(0xFFFFFFFFu, (int)(threadIdx.x >> 5), 0);
}

__device__ __forceinline__ bool elect_lane() {
  uint32_t chosen;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(chosen));
  return chosen != 0;
}

// shared::cluster address of `addr` (a shared::cta address) in CTA `rank`.
__device__ __forceinline__ uint32_t map_to_rank(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::
                   : "memory");
}

__device__ __forceinline__ void barrier_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}

__device__ __forceinline__ void barrier_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes)
               : "memory");
}

// Arrive on a barrier given by its shared::cluster address.
__device__ __forceinline__ void barrier_arrive(uint32_t cluster_bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar)
               : "memory");
}

// The same without ordering this thread's stores before it, which would wait for them:
// for giving back an accumulator, whose loads are complete and fenced.
__device__ __forceinline__ void barrier_arrive_relaxed(uint32_t cluster_bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar)
               : "memory");
}

__device__ __forceinline__ bool barrier_try(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(bar), "r"(parity)
      : "memory");
  return done != 0;
}

__device__ __forceinline__ void record_wait(unsigned int* status, unsigned int where) {
  asm volatile("st.relaxed.sys.global.u32 [%0], %1;" ::"l"(status), "r"(where) : "memory");
}

// Bounded wait for the completion of the phase of `parity`; false (and `where`
// recorded) when it did not come.
__device__ __forceinline__ bool barrier_wait(uint32_t bar, uint32_t parity, unsigned int* status,
                                             unsigned int where, long long limit = kWaitCycles) {
  if (barrier_try(bar, parity)) return true;
  const long long start = clock64();
  while (!barrier_try(bar, parity)) {
    if (clock64() - start > limit) {
      record_wait(status, where);
      return false;
    }
  }
  return true;
}

__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

template <int CG>
__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap* map, int x, int y, int z,
                                         uint32_t cluster_bar) {
  if constexpr (CG == 2) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::"
        "bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(cluster_bar)
        : "memory");
  } else {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], "
        "[%1, {%2, %3, %4}], [%5];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(cluster_bar)
        : "memory");
  }
}

template <int CG>
__device__ __forceinline__ void tmem_alloc(uint32_t dst, uint32_t columns) {
  if constexpr (CG == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst),
                 "r"(columns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  } else {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst),
                 "r"(columns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
}

template <int CG>
__device__ __forceinline__ void tmem_free(uint32_t tmem, uint32_t columns) {
  if constexpr (CG == 2)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns));
  else
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns));
}

// Arrive on `bar` (same offset in every CTA of the group) once all MMAs and
// copies issued so far by this thread are done.
template <int CG>
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  if constexpr (CG == 2) {
    const uint16_t both = 3;
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 "
        "[%0], %1;" ::"r"(bar),
        "h"(both)
        : "memory");
  } else {
    asm volatile(
        "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar)
        : "memory");
  }
}

template <int CG>
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                        uint32_t accumulate) {
  if constexpr (CG == 2) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
  } else {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
  }
}

template <int CG>
__device__ __forceinline__ void mma_f8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                       uint32_t scale_a, uint32_t scale_b, uint32_t accumulate) {
  if constexpr (CG == 2) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale [%0], %1, %2, %3, [%4], [%5], "
        "p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(scale_a), "r"(scale_b), "r"(accumulate)
        : "memory");
  } else {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale [%0], %1, %2, %3, [%4], [%5], "
        "p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(scale_a), "r"(scale_b), "r"(accumulate)
        : "memory");
  }
}

// 32 lanes x 16 bytes of shared memory into 4 TMEM columns, repeated for the
// four groups of 32 lanes (the layout block scales are read in).
template <int CG>
__device__ __forceinline__ void copy_scales(uint32_t tmem, uint64_t desc) {
  if constexpr (CG == 2)
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc)
                 : "memory");
  else
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc)
                 : "memory");
}

// 32 accumulator columns of this warp's 32 lanes: r[c] = D[lane, column + c].  The
// registers are valid after tmem_wait(r).
__device__ __forceinline__ void tmem_load32(uint32_t addr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
        "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
        "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}

// Waits for this warp's TMEM loads; naming the registers keeps their uses behind it.
__device__ __forceinline__ void tmem_wait(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]),
                 "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]),
                 "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]),
                 "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]),
                 "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}

__device__ __forceinline__ void tmem_fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tmem_fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}

// Shared-memory matrix descriptors (sm_100 format: version 1 at bit 46, the
// swizzle mode at bits 61-63, addresses and offsets in 16-byte units).
//
// k contiguous: rows of 128 bytes, 128-byte swizzle; groups of 8 rows are 1024
// bytes apart.  Row index contiguous: 64 rows (128 bytes) x 64 k per box; groups
// of 8 k are 1024 bytes apart (stride offset), boxes 8192 bytes (leading offset).
__device__ __forceinline__ uint64_t operand_descriptor(bool rows_inner) {
  const uint64_t lead = rows_inner ? 8192u >> 4 : 1u;
  return (lead << 16) | (uint64_t(1024u >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// Scale blocks: unswizzled 8 x 16-byte core matrices, 128 bytes apart.
__device__ __forceinline__ uint64_t scale_descriptor(uint32_t addr) {
  return uint64_t((addr >> 4) & 0x3FFFu) | (1ull << 16) | (uint64_t(128u >> 4) << 32) |
         (1ull << 46);
}

// Bounded wait until `counter` has reached `count` (arrivals of a whole grid).
__device__ __forceinline__ bool counter_wait(const unsigned int* counter, unsigned int count,
                                             unsigned int* status, unsigned int where) {
  const long long start = clock64();
  for (;;) {
    unsigned int seen;
    asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(seen) : "l"(counter) : "memory");
    if (seen >= count) return true;
    if (clock64() - start > kWaitCycles) {
      record_wait(status, where);
      return false;
    }
  }
}

// Adds one to a counter in shared memory, ordered after and before the CTA's accesses
// (the count before it is returned).
__device__ __forceinline__ unsigned int shared_count(unsigned int* counter) {
  unsigned int before;
  asm volatile("atom.acq_rel.cta.shared::cta.add.u32 %0, [%1], 1;"
               : "=r"(before)
               : "r"(smem_address(counter))
               : "memory");
  return before;
}

__device__ __forceinline__ void counter_arrive(unsigned int* counter) {
  asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(counter) : "memory");
}

}  // namespace srs
