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
//
// GROUPED: the rows of B are in groups, each with a matrix A of its own.  A CTA's tile is 128
// rows of one group's A by up to BN of its rows; which, it finds from the ends (all its warps
// do, so that nothing waits for a barrier).  Grids are sized by a bound: the CTAs left over write
// zeros for the rows of no group, as the others do behind their tile, and leave.
//
// ADAPTERS: B's rows are tokens, and token t of adapter a gets U_a low_t more, as MMAs of 16-bit
// operands (see the large product with adapters): an item of low parts, zero but for its adapter's
// tokens, by the adapter's U; the CTAs of a cluster take the adapters in turn.  Their sums are apart
// from the projection's, as zero times an infinity is NaN and an item's zeros are in other tokens'
// columns, which an MMA cannot leave out: a row where an adapter's U is not finite has such sums in
// every column.  The adapters' part of a sum that is not finite is computed again, from the token's
// own adapter alone (sums_again, out of line: in the epilogue's own code it took a microsecond for 64
// tokens, used or not; a look at U in shared memory ahead of the MMAs took three).
// (In a kernel of its own behind this one that part took 5 us for one token and 10 for 64 with
// 41 adapters, nearly all of it launch and dependent loads; in this one's epilogue as much.)
// Ranks up to 16 take narrow boxes, three adapters a stage: with one a stage, of boxes of 128 bytes
// that were mostly fill, 64 tokens of 40 adapters waited for four loads in flight (14336 x 4096:
// 34 us a call in a graph, 30.8 with three).  The product of the projection does not wait for the low
// part, which the kernels ahead arrange: 29.7 us, and of one adapter 24.6 -> 22.1; without any 17.6.
// What is left is mostly the items: 40 of 64 tokens a CTA's tile, of which one or two are not zero.
#pragma once

#include "srs_groups.cuh"
#include "srs_product.cuh"

namespace srs {

constexpr int kThinThreads = 256;

constexpr int kThinMaxStages = 12;
constexpr int kThinSlots = 8;    // scale groups on their way
constexpr int kThinLoaders = 6;  // warps that bring them

template <int N>
struct Constant {
  static constexpr int value = N;
};

// What else a thin product does.
enum : int { kThinPlain = 0, kThinGrouped = 1, kThinAdapters = 2 };

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
  // GROUPED: m is the rows of one group's A, n those of all of B
  const int32_t* ends;
  int groups;
  int64_t scale_a_group;  // bytes of scales from one group's A to the next
  // ADAPTERS (`ends`, `groups`: those of the tokens' adapters)
  CUtensorMap map_h, map_u;
  int rank, item_slices, rest_at;
  bool up_rows_inner;  // U is stored rank x rows
  // Ranks up to 16: adapters a stage (0: see item_slices), boxes of 32 bytes a row of U, and behind
  // them, from pack_at on, of 64 bytes a token of the pairs.
  int pack, pack_at;
  const int32_t* exponents;  // of FP16 pairs, one a token (null: BF16)
  uint32_t extra_idesc;
  // for own_part: low parts and U as the maps have them, and the tokens' order
  const uint16_t* pairs;
  const uint16_t* up;
  int64_t up_pitch, up_stride;  // elements
  int pair_pitch;
  const int32_t* order;
};

template <int BN>
struct ThinShape {
  static constexpr int kColumns = BN <= 16 ? 32 : BN <= 32 ? 64 : 128;  // TMEM
  static constexpr int kScaleColumn = BN;  // two groups of 8 columns (A, B)
  // ADAPTERS: their sums behind the scales (two CTAs an SM still fit its 512 columns)
  static constexpr int kAdapterColumn = BN + 16;
  static constexpr int kAllColumns = BN <= 16 ? 64 : BN <= 32 ? 128 : 256;
  static constexpr int kScaleBytes = 1024;
  static constexpr int kFixed = 1024 + kThinSlots * kScaleBytes;  // alignment, scales
  // Two CTAs fit an SM.  The MMA reads 128 rows of A whatever the tile has: behind the
  // last stage's panel a whole one stays inside the CTA's memory.
  static constexpr int kBudget = 110 * 1024 - kFixed;
  static constexpr int kSums = 128 * BN * 4;  // split sums, in the stages' place
  static_assert(BN + 16 <= kColumns && 2 * BN + 16 <= kAllColumns, "accumulators and scales fit");
  static_assert(kSums <= kBudget, "split sums fit the stages");
};

__device__ __forceinline__ void store_value(void* out, int format, int64_t at, float v) {
  if (format == SRS_FMT_F32) static_cast<float*>(out)[at] = v;
  else if (format == SRS_FMT_BF16) static_cast<__nv_bfloat16*>(out)[at] = __float2bfloat16_rn(v);
  else static_cast<__half*>(out)[at] = __float2half_rn(v);
}

// Zeros in the rows of D (B's rows) that belong to no group, by all threads of the grid.
__device__ __forceinline__ void zero_ungrouped(const ThinArgs& a) {
  // the last end as the groups' own reading of them has it
  const int lane = threadIdx.x & 31;
  const EndsAhead ahead(a.ends, a.groups, lane);
  int carry = 0;
  for (int base = 0; base < a.groups; base += 32) {
    int start, end;
    group_span(a.ends, ahead, a.groups, a.n, base, lane, &carry, &start, &end);
  }
  const int64_t last = (int64_t)a.n * a.m;
  for (int64_t i = (int64_t)carry * a.m + (int64_t)blockIdx.x * kThinThreads + threadIdx.x;
       i < last; i += (int64_t)gridDim.x * kThinThreads)
    store_value(a.out, a.out_format, i, 0.0f);
}

// ADAPTERS: those with tokens, in order; active[e] has the places first[e] .. first[e + 1] - 1.
struct ThinAdapters {
  int active[kThinRows], actives;
  int first[kThinRows + 1];
};

// Row `row` of U low for one token (its pairs are held times a power of two), if its adapter is one
// of every `step`-th from e on; else 0.
template <int BN>
__device__ __noinline__ float own_part(const ThinArgs& a, const ThinAdapters& given, int e, int step,
                                       int token, int row) {
  for (; e < given.actives; e += step) {
    int p = given.first[e];
    while (p < given.first[e + 1] && token_at(a.order, p, a.n) != token) ++p;
    if (p < given.first[e + 1]) break;
  }
  if (e >= given.actives) return 0.0f;
  const uint16_t* const low = a.pairs + ((int64_t)e * BN + token) * a.pair_pitch;
  const uint16_t* const up = a.up + given.active[e] * a.up_stride +
                             (a.up_rows_inner ? row : row * a.up_pitch);
  const int64_t up_step = a.up_rows_inner ? a.up_pitch : 1;
  const auto decode = [&](uint16_t v) {
    return a.out_format == SRS_FMT_BF16 ? __uint_as_float((uint32_t)v << 16)
                                        : __half2float(__ushort_as_half(v));
  };
  float sum = 0.0f;
  for (int r = 0; r < a.rank; ++r) {
    const float h = decode(__ldcg(low + r)) + decode(__ldcg(low + a.rest_at + r));
    sum = fmaf(h, decode(__ldg(up + r * up_step)), sum);
  }
  return sum;
}

// Times the power of two that a token's FP16 pairs, and with them its sums, do not have.
__device__ __forceinline__ float unscaled(const ThinArgs& a, float sum, int token) {
  return a.exponents != nullptr ? sum * two_to(-__ldcg(a.exponents + token)) : sum;
}

// The sums of this thread's row whose adapters' part is not finite, with their own adapter's part
// instead: to D (`last`), or to `words` in shared memory, 512 bytes a column.  By whole warps.
template <int BN>
__device__ __noinline__ void sums_again(const ThinArgs& a, const ThinAdapters& given, uint32_t acc,
                                        uint32_t words, int e, int step, int row, bool last) {
#pragma unroll 1
  for (int c0 = 0; c0 < a.n; c0 += 16) {
    uint32_t v[16], u[16];
    tmem_load16(acc + c0, v, acc + ThinShape<BN>::kAdapterColumn + c0, u);
    unsigned odd = 0u;
#pragma unroll
    for (int c = 0; c < 16; ++c) {
      if (row < 0 || c0 + c >= a.n || (u[c] & 0x7F800000u) != 0x7F800000u) continue;
      odd |= 1u << c;
      asm volatile("st.shared.b32 [%0], %1;" ::"r"(words + 512 * (c0 + c)), "r"(v[c]) : "memory");
    }
    for (; odd != 0u; odd &= odd - 1u) {
      const int c = c0 + __ffs(odd) - 1;
      const float sum = __uint_as_float(staged_read(words + 512 * c)) +
                        own_part<BN>(a, given, e, step, c, row);
      if (last)
        store_value(a.out, a.out_format, row * a.row_stride + c * a.col_stride, unscaled(a, sum, c));
      else
        asm volatile("st.shared.f32 [%0], %1;" ::"r"(words + 512 * c), "f"(sum) : "memory");
    }
    __syncwarp();
  }
}

template <int BN, int FORM>
__global__ void __launch_bounds__(kThinThreads, 2)
thin_product_kernel(const __grid_constant__ ThinArgs a) {
  constexpr bool GROUPED = FORM == kThinGrouped;
  constexpr bool ADAPTERS = FORM == kThinAdapters;
  using S = ThinShape<BN>;
  constexpr uint32_t kColumns = ADAPTERS ? S::kAllColumns : S::kColumns;
  __shared__ ThinAdapters given;
  // A kernel launched to overlap this one may start (and wait for it).
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  extern __shared__ uint8_t raw[];
  __shared__ __align__(8) uint64_t bars[2 * kThinMaxStages + 1 + 2 * kThinSlots];
  __shared__ uint32_t tmem_slot;

  const int warp = warp_index(), lane = threadIdx.x & 31;
  uint32_t splits;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(splits));
  const uint32_t rank = cluster_rank();
  int row0 = (int)(blockIdx.x / splits) * a.rows;
  // first row of A in its map, first row of B and of D's columns, and how many of them
  int map_row = row0, b_row0 = 0, n = a.n;
  const uint8_t* scale_a = a.scale_a;
  if constexpr (GROUPED) {
    const int row_tiles = (a.m + a.rows - 1) / a.rows, t = (int)(blockIdx.x / splits);
    const GroupTile tile =
        find_group_tile(a.ends, a.groups, a.n, BN, t / row_tiles, lane);
    row0 = t % row_tiles * a.rows;
    map_row = tile.group * a.m + row0;
    b_row0 = tile.row0;
    n = tile.group < 0 ? 0 : min(BN, tile.end - tile.row0);
    scale_a += (int64_t)tile.group * a.scale_a_group;
    if (tile.group < 0) {
      // the same for all CTAs of the cluster; no later kernel before the one ahead is done
      asm volatile("griddepcontrol.wait;" ::: "memory");
      zero_ungrouped(a);
      return;
    }
  }
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
        load_box<1>(stage0 + i * stage_bytes, &a.map_a, (first + i) * kSliceBytes, map_row, 0,
                    full(i));
      }
    }
    __syncwarp();
  }
  if (warp == 5) tmem_alloc<1>(smem_address(&tmem_slot), kColumns);
  tmem_fence_before();
  __syncthreads();
  tmem_fence_after();
  const uint32_t tmem = tmem_slot;
  bool ok = true;
  if (warp == 4) {
    const bool leader = elect_lane();
    // B may come from the kernel this one overlaps (of adapters: only from the one ahead of that,
    // which was done before this kernel could start).
    if constexpr (!ADAPTERS) asm volatile("griddepcontrol.wait;" ::: "memory");
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
          load_box<1>(pa, &a.map_a, i * kSliceBytes, map_row, 0, full(s));
        }
        load_box<1>(pa + panel_bytes, &a.map_b, i * kSliceBytes, b_row0, 0, full(s));
      }
      __syncwarp();
      if (++s == stages) {
        s = 0;
        phase ^= 1u;
      }
    }
    if constexpr (ADAPTERS) {
      asm volatile("griddepcontrol.wait;" ::: "memory");  // the low part
      asm volatile("bar.sync 1, 96;" ::: "memory");       // the list of adapters
      const int slices = a.pack != 0 ? 0 : a.item_slices, chunks = (slices + 1) / 2;
      const int actives = given.actives;
      for (int e0 = (int)rank; a.pack != 0 && e0 < actives && ok; e0 += (int)splits * a.pack) {
        const uint32_t pa = stage0 + s * stage_bytes;
        ok = barrier_wait(empty(s), phase ^ 1u, a.status, 1u << 8);
        if (!ok) break;
        if (leader) {
          const int count = min(a.pack, (actives - e0 + (int)splits - 1) / (int)splits);
          barrier_expect(full(s), (uint32_t)(count * (a.rows * 32 + BN * 64)));
          for (int i = 0; i < count; ++i) {
            const int e = e0 + i * (int)splits;
            load_box<1>(pa + i * (panel_bytes / 4), &a.map_u, 0, row0, given.active[e], full(s));
            load_box<1>(pa + a.pack_at + i * (BN * 64), &a.map_h, 0, e * BN, 0, full(s));
          }
        }
        __syncwarp();
        if (++s == stages) {
          s = 0;
          phase ^= 1u;
        }
      }
      for (int e = (int)rank; e < actives && ok; e += (int)splits) {
        for (int q = 0; q < slices && ok; ++q) {
          const uint32_t pa = stage0 + s * stage_bytes;
          ok = barrier_wait(empty(s), phase ^ 1u, a.status, 1u << 8);
          if (!ok) break;
          if (leader) {
            const int k = 64 * (q < chunks ? q : q - chunks);
            barrier_expect(full(s), load_bytes);
            if (a.up_rows_inner) {
              load_box<1>(pa, &a.map_u, row0, k, given.active[e], full(s));
              load_box<1>(pa + kPanelBytes / 2, &a.map_u, row0 + 64, k, given.active[e], full(s));
            } else {
              load_box<1>(pa, &a.map_u, k, row0, given.active[e], full(s));
            }
            load_box<1>(pa + panel_bytes, &a.map_h, 64 * q, e * BN, 0, full(s));
          }
          __syncwarp();
          if (++s == stages) {
            s = 0;
            phase ^= 1u;
          }
        }
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
    if constexpr (ADAPTERS) {
      asm volatile("bar.sync 1, 96;" ::: "memory");
      const int slices = a.pack != 0 ? 0 : a.item_slices, chunks = (slices + 1) / 2;
      const int actives = given.actives;
      const uint32_t sums = tmem + S::kAdapterColumn;
      uint32_t more = 0u;  // 0: the first MMA writes the sums
      const bool inner = a.up_rows_inner;
      const uint64_t desc_u = operand_descriptor(inner);
      const uint32_t step_u = (inner ? 2048u : 32u) >> 4;
      const uint32_t idesc = a.extra_idesc | (inner ? 1u << 15 : 0u);
      for (int e0 = (int)rank; a.pack != 0 && e0 < actives && ok; e0 += (int)splits * a.pack) {
        ok = barrier_wait(full(s), phase, a.status, 1u << 11);
        if (!ok) break;
        tmem_fence_after();
        const uint32_t pa = stage0 + s * stage_bytes;
        if (leader) {
          const int count = min(a.pack, (actives - e0 + (int)splits - 1) / (int)splits);
          for (int i = 0; i < count; ++i) {
            const uint64_t du = short_row_descriptor(32) |
                                uint64_t(((pa + i * (panel_bytes / 4)) >> 4) & 0x3FFFu);
            const uint64_t dh = short_row_descriptor(64) |
                                uint64_t(((pa + a.pack_at + i * (BN * 64)) >> 4) & 0x3FFFu);
            mma_f16<1>(sums, du, dh, idesc, more | (uint32_t)i);
            mma_f16<1>(sums, du, dh + 2, idesc, 1u);  // the pairs' second parts
          }
          mma_commit<1>(empty(s));
        }
        __syncwarp();
        more = 1u;
        if (++s == stages) {
          s = 0;
          phase ^= 1u;
        }
      }
      for (int e = (int)rank; e < actives && ok; e += (int)splits) {
        for (int q = 0; q < slices && ok; ++q) {
          ok = barrier_wait(full(s), phase, a.status, 1u << 11);
          if (!ok) break;
          tmem_fence_after();
          const uint32_t pa = stage0 + s * stage_bytes;
          const uint64_t du = desc_u | uint64_t((pa >> 4) & 0x3FFFu);
          const uint64_t dh = desc | uint64_t(((pa + panel_bytes) >> 4) & 0x3FFFu);
          const int chunk = q < chunks ? q : q - chunks;
          const int steps = (min(a.rank - 64 * chunk, 64) + 15) / 16;
          if (leader) {
            for (int j = 0; j < steps; ++j)
              mma_f16<1>(sums, du + j * step_u, dh + 2 * j, idesc, more | (uint32_t)j);
            if (slices == 1) {
              for (int j = 0; j < steps; ++j)
                mma_f16<1>(sums, du + j * step_u, dh + 2 * (a.rest_at / 16 + j), idesc, 1u);
            }
            mma_commit<1>(empty(s));
          }
          __syncwarp();
          more = 1u;
          if (++s == stages) {
            s = 0;
            phase ^= 1u;
          }
        }
      }
    }
    if (ok && leader) mma_commit<1>(done);
    __syncwarp();
  } else {
    // ---- block scales: the writing warps and two more take a group each in turn, as a
    // group's loads take microseconds behind the weights' in DRAM (one warp, a group
    // after the other, held a product of 58.7 MB at 18.6 us)
    const bool words_a = scale_words(scale_a, a.scale_a_pitch, first);
    const bool words_b = scale_words(a.scale_b, a.scale_b_pitch, first);
    ScaleRows from_a, from_b;
    from_a.at(scale_a, a.scale_a_pitch, a.scale_a_shift, row0, a.m, lane);
    from_b.at(a.scale_b, a.scale_b_pitch, a.scale_b_shift, b_row0, a.n, lane);
    if constexpr (ADAPTERS) {
      if (warp == 7) {
        // the adapters with tokens, for the loads and MMAs (at most as many as tokens)
        const EndsAhead ahead(a.ends, a.groups, lane);
        int carry = 0, count = 0;
        for (int base = 0; base < a.groups; base += 32) {
          int start, end;
          group_span(a.ends, ahead, a.groups, a.n, base, lane, &carry, &start, &end);
          const unsigned some = __ballot_sync(0xFFFFFFFFu, end > start);
          if (end > start) {
            const int e = count + __popc(some & ((1u << lane) - 1u));
            given.active[e] = base + lane;
            given.first[e] = start;
          }
          count += __popc(some);
        }
        if (lane == 0) {
          given.actives = count;
          given.first[count] = carry;
        }
        __syncwarp();
        asm volatile("bar.arrive 1, 96;" ::: "memory");
      }
    }
    const int groups = (last - first + 3) >> 2;
    bool waited = false;
    uint32_t more[4] = {0u, 0u, 0u, 0u};  // ADAPTERS: for B's scales
    for (int g = warp < 4 ? warp : warp - 2; g < groups; g += kThinLoaders) {
      const int slot = g % kThinSlots, kb = first + 4 * g;
      uint32_t w[2][4];
      from_a.read(kb, last, words_a, w[0]);
      if (!waited && (!ADAPTERS || a.exponents != nullptr)) {
        asm volatile("griddepcontrol.wait;" ::: "memory");
        if constexpr (ADAPTERS) {
          // (written ahead of this kernel, as the pairs are)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            more[j] = in_every_byte(__ldcg(a.exponents + min(lane + 32 * j, a.n - 1)));
        }
      }
      waited = true;
      from_b.read<true>(kb, last, words_b, w[1]);
      if constexpr (ADAPTERS) {
#pragma unroll
        for (int j = 0; j < 4; ++j) w[1][j] = __vadd4(w[1][j], more[j]);
      }
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
  bool with = false;  // this CTA has adapters' sums
  if constexpr (ADAPTERS) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    __syncthreads();  // (the list of adapters)
    with = (int)rank < given.actives;
  }
  // This thread's row among sums in shared memory: column c at 512 * c bytes, one word a row.
  const uint32_t words = stage0 + 128 * warp + 4 * lane;
  // 16 columns of this thread's row.
  uint32_t top = 0u;  // largest size of the adapters' sums among them
  const auto sums_of = [&](int c0, uint32_t (&v)[16]) {
    if (!ADAPTERS || !with) {
      tmem_load16(acc + c0, v);
    } else {
      uint32_t u[16];
      tmem_load16(acc + c0, v, acc + S::kAdapterColumn + c0, u);
#pragma unroll
      for (int c = 0; c < 16; ++c) {
        v[c] = __float_as_uint(__uint_as_float(v[c]) + __uint_as_float(u[c]));
        top = max(top, c0 + c < n ? u[c] & 0x7FFFFFFFu : 0u);
      }
    }
  };
  const auto result = [&](float sum, int c) {
    if constexpr (ADAPTERS) return unscaled(a, sum, c);
    return sum;
  };
  const auto look_again = [&]() {
    if constexpr (ADAPTERS) {
      if (__any_sync(0xFFFFFFFFu, top >= 0x7F800000u && row < row_end))
        sums_again<BN>(a, given, acc, words, (int)rank, (int)splits, row < row_end ? row : -1,
                       splits == 1);
    }
  };
  if (splits == 1) {
    if (warp < 4 && ok) {
#pragma unroll
      for (int c0 = 0; c0 < BN; c0 += 16) {
        if (c0 >= n) break;
        uint32_t v[16];
        sums_of(c0, v);
#pragma unroll
        for (int c = 0; c < 16; ++c)
          if (row < row_end && c0 + c < n)
            store_value(a.out, a.out_format,
                        row * a.row_stride + (b_row0 + c0 + c) * a.col_stride,
                        result(__uint_as_float(v[c]), c0 + c));
      }
      look_again();
    }
  } else {
    if (warp < 4) {
#pragma unroll
      for (int c0 = 0; c0 < BN; c0 += 16) {
        if (c0 >= n) break;
        uint32_t v[16];
        sums_of(c0, v);
#pragma unroll
        for (int c = 0; c < 16; ++c)
          asm volatile("st.shared.b32 [%0], %1;" ::"r"(words + 512 * (c0 + c)), "r"(v[c])
                       : "memory");
      }
      look_again();
    }
    cluster_sync();
    // columns rank, rank + splits, ...: half of the CTA's threads a column
    const int half = threadIdx.x >> 7, at = threadIdx.x & 127;
    const int out_row = row0 + at;
    const bool write = out_row < row_end && ok;
    // `columns` of `parts` words in flight, then their stores: one column after the other took a
    // microsecond more for 64 columns of two parts.
    const auto join = [&](auto parts, auto columns) {
      constexpr int P = decltype(parts)::value, C = decltype(columns)::value;
      for (int c0 = (int)rank + half * P; c0 < n; c0 += 2 * P * C) {
        float part[C][P];
#pragma unroll
        for (int i = 0; i < C; ++i) {
          const int c = min(c0 + 2 * P * i, n - 1);
#pragma unroll
          for (int r = 0; r < P; ++r)
            asm volatile("ld.shared::cluster.f32 %0, [%1];"
                         : "=f"(part[i][r])
                         : "r"(map_to_rank(stage0 + 512 * c + 4 * at, (uint32_t)r))
                         : "memory");
        }
#pragma unroll
        for (int i = 0; i < C; ++i) {
          const int c = c0 + 2 * P * i;
          float sum = part[i][0];
#pragma unroll
          for (int r = 1; r < P; ++r) sum = __fadd_rn(sum, part[i][r]);
          if (write && c < n)
            store_value(a.out, a.out_format,
                        out_row * a.row_stride + (b_row0 + c) * a.col_stride,
                        result(sum, c));
        }
      }
    };
    if (splits == 2) join(Constant<2>{}, Constant<4>{});
    else if (splits == 4) join(Constant<4>{}, Constant<4>{});
    else join(Constant<8>{}, Constant<1>{});
    cluster_sync();  // the others have read this CTA's sums
  }
  tmem_fence_before();
  __syncthreads();
  tmem_fence_after();
  if (warp == 5) tmem_free<1>(tmem, kColumns);
  if constexpr (GROUPED) zero_ungrouped(a);
}

}  // namespace srs
