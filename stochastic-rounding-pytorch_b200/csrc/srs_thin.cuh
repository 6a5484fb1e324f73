// FP8 block products with one thin side (up to 64 rows: decoded tokens):
//
//   D[i, j] = sum_k A[i, k] * B[j, k],   A: m x k (the weights), B: n x k, n <= 64
//
// What bounds it: A's bytes, read once, and about 6 us of launch, first loads and last
// sums.  The weights take the 128-row side of the MMA and the thin operand the column
// side, so that no MMA row is idle, and k is split over a cluster of up to 8 CTAs so
// that all SMs stream: 4096 rows are only 32 tiles.  The split sums meet in distributed
// shared memory and are added in rank order (FP32), so results do not depend on
// timing.  Two CTAs share an SM, each with 72 KB of slices on their way in tiles of 128 rows
// and up to 85 KB in smaller ones.
// 14336 x 4096 by one token (58.7 MB): 16.7 us a call; 28672 x 8192: 42.9 us, 5.5 TB/s.
//
// Launched behind the quantisation of its B (srs_linear_blocks) the kernel may start
// while that one runs: it loads A first and waits for the other kernel before it
// touches B.
//
// Roles, barriers and bounded waits as in the large product (one tile per CTA).
#pragma once

#include "srs_product.cuh"

namespace srs {

constexpr int kThinThreads = 256;

constexpr int kThinMaxStages = 12;
constexpr int kThinSlots = 8;    // scale groups on their way
constexpr int kThinLoaders = 6;  // warps that bring them

struct ThinArgs {
  CUtensorMap map_a, map_b;
  int m, n;             // rows of A and of B
  int rows;             // of a tile
  int panel_bytes;      // of A in a stage (whole 8-row groups)
  int stages;
  int slices;           // of 128 along k
  const uint8_t* scale_a;
  const uint8_t* scale_b;
  int64_t scale_a_pitch, scale_b_pitch;
  int scale_a_shift, scale_b_shift;
  uint32_t idesc;
  void* out;
  int out_format;
  int64_t row_stride, col_stride;  // of D, elements
  unsigned int* status;
};

template <int BN>
struct ThinShape {
  static constexpr int kColumns = BN <= 16 ? 32 : BN <= 32 ? 64 : 128;  // TMEM
  static constexpr int kScaleColumn = BN;  // two groups of 8 columns (A, B)
  static constexpr int kScaleBytes = 1024;
  static constexpr int kFixed = 1024 + kThinSlots * kScaleBytes;  // alignment, scales
  // Two CTAs fit an SM.  The MMA reads 128 rows of A whatever the tile has: behind the
  // last stage's panel a whole one stays inside the CTA's memory.
  static constexpr int kBudget = 110 * 1024 - kFixed;
  static constexpr int kSums = 128 * BN * 4;  // split sums, in the stages' place
  static_assert(BN + 16 <= kColumns, "accumulator and scales fit");
  static_assert(kSums <= kBudget, "split sums fit the stages");
};

__device__ __forceinline__ void tmem_load16(uint32_t addr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]),
                 "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                 "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}

__device__ __forceinline__ void store_value(void* out, int format, int64_t at, float v) {
  if (format == SRS_FMT_F32) static_cast<float*>(out)[at] = v;
  else if (format == SRS_FMT_BF16) static_cast<__nv_bfloat16*>(out)[at] = __float2bfloat16_rn(v);
  else static_cast<__half*>(out)[at] = __float2half_rn(v);
}

template <int BN>
__global__ void __launch_bounds__(kThinThreads, 2)
thin_product_kernel(const __grid_constant__ ThinArgs a) {
  using S = ThinShape<BN>;
  extern __shared__ uint8_t raw[];
  __shared__ __align__(8) uint64_t bars[2 * kThinMaxStages + 1 + 2 * kThinSlots];
  __shared__ uint32_t tmem_slot;

  const int warp = warp_index(), lane = threadIdx.x & 31;
  uint32_t splits;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(splits));
  const uint32_t rank = cluster_rank();
  const int row0 = (int)(blockIdx.x / splits) * a.rows;
  const int first = (int)((int64_t)a.slices * rank / splits);
  const int last = (int)((int64_t)a.slices * (rank + 1) / splits);
  const uint32_t scales0 = (smem_address(raw) + 1023u) & ~1023u;
  const uint32_t stage0 = scales0 + kThinSlots * S::kScaleBytes;
  const int stages = a.stages;
  const uint32_t panel_bytes = (uint32_t)a.panel_bytes;
  const uint32_t stage_bytes = panel_bytes + BN * kSliceBytes;
  const uint32_t load_bytes = (uint32_t)a.rows * kSliceBytes + BN * kSliceBytes;
  const uint32_t bar0 = smem_address(bars);
  const auto full = [&](int s) { return bar0 + 8u * s; };
  const auto empty = [&](int s) { return bar0 + 8u * (kThinMaxStages + s); };
  const uint32_t done = bar0 + 8u * (2 * kThinMaxStages);
  const auto scale_full = [&](int i) { return bar0 + 8u * (2 * kThinMaxStages + 1 + i); };
  const auto scale_empty = [&](int i) {
    return bar0 + 8u * (2 * kThinMaxStages + 1 + kThinSlots + i);
  };

  // The loading warp sets up its barriers and sends for its first slices of A at once,
  // before TMEM is there.
  const int ahead = min(stages, last - first);
  if (warp == 4) {
    if (elect_lane()) {
      for (int s = 0; s < stages; ++s) {
        barrier_init(full(s), 1);
        barrier_init(empty(s), 1);
      }
      barrier_init(done, 1);
      for (int i = 0; i < kThinSlots; ++i) {
        barrier_init(scale_full(i), 1);
        barrier_init(scale_empty(i), 1);
      }
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      for (int i = 0; i < ahead; ++i) {
        barrier_expect(full(i), load_bytes);
        load_box<1>(stage0 + i * stage_bytes, &a.map_a, (first + i) * kSliceBytes, row0, 0,
                    full(i));
      }
    }
    __syncwarp();
  }
  if (warp == 5) tmem_alloc<1>(smem_address(&tmem_slot), S::kColumns);
  tmem_fence_before();
  __syncthreads();
  tmem_fence_after();
  const uint32_t tmem = tmem_slot;
  bool ok = true;

  if (warp == 4) {
    const bool leader = elect_lane();
    // B may come from the kernel this one overlaps.
    asm volatile("griddepcontrol.wait;" ::: "memory");
    int s = 0;
    uint32_t phase = 0;
    for (int i = first; i < last; ++i) {
      const uint32_t pa = stage0 + s * stage_bytes;
      const bool sent = i - first < ahead;
      if (!sent) ok = barrier_wait(empty(s), phase ^ 1u, a.status, 1u << 8);
      if (!ok) break;
      if (leader) {
        if (!sent) {
          barrier_expect(full(s), load_bytes);
          load_box<1>(pa, &a.map_a, i * kSliceBytes, row0, 0, full(s));
        }
        load_box<1>(pa + panel_bytes, &a.map_b, i * kSliceBytes, 0, 0, full(s));
      }
      __syncwarp();
      if (++s == stages) {
        s = 0;
        phase ^= 1u;
      }
    }
    // Every stage given back before the CTA can leave.
    for (int i = 0; i < stages && ok; ++i) {
      ok = barrier_wait(empty(s), phase ^ 1u, a.status, 1u << 14);
      if (++s == stages) {
        s = 0;
        phase ^= 1u;
      }
    }
  } else if (warp == 5) {
    const bool leader = elect_lane();
    const uint64_t desc = operand_descriptor(false);
    int s = 0, slot = 0, last_slot = -1;
    uint32_t phase = 0, slot_phase = 0, last_phase = 0, group = 0;
    for (int i = first; i < last && ok; ++i) {
      const int j0 = i - first;
      const uint32_t scale_tmem = tmem + S::kScaleColumn + 8u * (group & 1u);
      if ((j0 & 3) == 0) {
        // (see the large product: the columns' last readers are done after this)
        if (last_slot >= 0) ok = barrier_wait(scale_empty(last_slot), last_phase, a.status, 1u << 9);
        ok = ok && barrier_wait(scale_full(slot), slot_phase, a.status, 1u << 10);
        if (!ok) break;
        tmem_fence_after();
        const uint32_t src = scales0 + slot * S::kScaleBytes;
        if (leader) {
          copy_scales<1>(scale_tmem, scale_descriptor(src));
          copy_scales<1>(scale_tmem + 4, scale_descriptor(src + 512));
          mma_commit<1>(scale_empty(slot));
        }
        __syncwarp();
        last_slot = slot;
        last_phase = slot_phase;
        if (++slot == kThinSlots) {
          slot = 0;
          slot_phase ^= 1u;
        }
      }
      ok = barrier_wait(full(s), phase, a.status, 1u << 11);
      if (!ok) break;
      tmem_fence_after();
      const uint32_t pa = stage0 + s * stage_bytes;
      const uint64_t da = desc | uint64_t((pa >> 4) & 0x3FFFu);
      const uint64_t db = desc | uint64_t(((pa + panel_bytes) >> 4) & 0x3FFFu);
      const uint32_t id = (uint32_t)(j0 & 3), idesc = a.idesc | (id << 29) | (id << 4);
      if (leader) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          mma_f8<1>(tmem, da + 2 * j, db + 2 * j, idesc, scale_tmem, scale_tmem + 4,
                    (j0 | j) != 0 ? 1u : 0u);
        mma_commit<1>(empty(s));
      }
      __syncwarp();
      if (++s == stages) {
        s = 0;
        phase ^= 1u;
      }
      if ((j0 & 3) == 3) ++group;
    }
    if (ok && leader) mma_commit<1>(done);
    __syncwarp();
  } else {
    // ---- block scales: the writing warps and two more take a group each in turn, as a
    // group's loads take microseconds behind the weights' in DRAM (one warp, a group
    // after the other, held a product of 58.7 MB at 18.6 us)
    const bool words_a = scale_words(a.scale_a, a.scale_a_pitch, first);
    const bool words_b = scale_words(a.scale_b, a.scale_b_pitch, first);
    ScaleRows from_a, from_b;
    from_a.at(a.scale_a, a.scale_a_pitch, a.scale_a_shift, row0, a.m, lane);
    from_b.at(a.scale_b, a.scale_b_pitch, a.scale_b_shift, 0, a.n, lane);
    const int groups = (last - first + 3) >> 2;
    bool waited = false;
    for (int g = warp < 4 ? warp : warp - 2; g < groups; g += kThinLoaders) {
      const int slot = g % kThinSlots, kb = first + 4 * g;
      uint32_t w[2][4];
      from_a.read(kb, last, words_a, w[0]);
      if (!waited) asm volatile("griddepcontrol.wait;" ::: "memory");
      waited = true;
      from_b.read<true>(kb, last, words_b, w[1]);
      ok = barrier_wait(scale_empty(slot), ((uint32_t)(g / kThinSlots) & 1u) ^ 1u, a.status,
                        1u << 12);
      ok = __all_sync(0xFFFFFFFFu, ok);
      if (!ok) break;
      const uint32_t dst = scales0 + slot * S::kScaleBytes + 16u * lane;
#pragma unroll
      for (int c = 0; c < 2; ++c)
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst + 512 * c),
                     "r"(w[c][0]), "r"(w[c][1]), "r"(w[c][2]), "r"(w[c][3])
                     : "memory");
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) barrier_arrive(map_to_rank(scale_full(slot), rank));
    }
    if (warp == 6) {
      for (int i = 0; i < kThinSlots && i < groups && ok; ++i) {
        // the last copy out of every slot
        const int g = groups - 1 - i;
        ok = barrier_wait(scale_empty(g % kThinSlots), (uint32_t)(g / kThinSlots) & 1u, a.status,
                          1u << 15);
      }
    }
  }
  __syncwarp();
  // Every warp waits for the last MMA: all loads and commits of this CTA are done
  // then, and the stages are free for the split sums.
  const bool finished = barrier_wait(done, 0u, a.status, 1u << 13);
  ok = __all_sync(0xFFFFFFFFu, ok && finished);
  if (!ok) {
    const long long start = clock64();
    while (clock64() - start < 4000000ll) {
    }
  }
  tmem_fence_after();
  const uint32_t acc = tmem + ((uint32_t)(warp * 32) << 16);
  const int row = row0 + 32 * warp + lane, row_end = min(a.m, row0 + a.rows);
  if (splits == 1) {
    if (warp < 4 && ok) {
#pragma unroll
      for (int c0 = 0; c0 < BN; c0 += 16) {
        if (c0 >= a.n) break;
        uint32_t v[16];
        tmem_load16(acc + c0, v);
#pragma unroll
        for (int c = 0; c < 16; ++c)
          if (row < row_end && c0 + c < a.n)
            store_value(a.out, a.out_format, row * a.row_stride + (c0 + c) * a.col_stride,
                        __uint_as_float(v[c]));
      }
    }
  } else {
    // column c of this CTA's sum at 512 * c bytes, one word a row
    if (warp < 4) {
#pragma unroll
      for (int c0 = 0; c0 < BN; c0 += 16) {
        if (c0 >= a.n) break;
        uint32_t v[16];
        tmem_load16(acc + c0, v);
#pragma unroll
        for (int c = 0; c < 16; ++c)
          asm volatile("st.shared.b32 [%0], %1;" ::"r"(stage0 + 512 * (c0 + c) + 128 * warp +
                                                       4 * lane),
                       "r"(v[c])
                       : "memory");
      }
    }
    cluster_sync();
    // columns rank, rank + splits, ...: half of the CTA's threads a column
    const int half = threadIdx.x >> 7, at = threadIdx.x & 127;
    const int out_row = row0 + at;
    for (int c = (int)rank + half * (int)splits; c < a.n; c += 2 * (int)splits) {
      float part[8];
#pragma unroll
      for (uint32_t r = 0; r < 8; ++r) {
        part[r] = 0.0f;
        if (r < splits)
          asm volatile("ld.shared::cluster.f32 %0, [%1];"
                       : "=f"(part[r])
                       : "r"(map_to_rank(stage0 + 512 * c + 4 * at, r))
                       : "memory");
      }
      float sum = part[0];
#pragma unroll
      for (int r = 1; r < 8; ++r)
        if (r < (int)splits) sum = __fadd_rn(sum, part[r]);
      if (out_row < row_end && ok)
        store_value(a.out, a.out_format, out_row * a.row_stride + c * a.col_stride, sum);
    }
    cluster_sync();  // the others have read this CTA's sums
  }
  tmem_fence_before();
  __syncthreads();
  tmem_fence_after();
  if (warp == 5) tmem_free<1>(tmem, S::kColumns);
}

}  // namespace srs
