// Matrix products on the sm_100a tensor cores (tcgen05, accumulators in TMEM):
//
//   D[i, j] = sum_k A[i, k] * B[j, k]      (A: M x K, B: N x K, FP32 accumulation)
//
// for FP16 operands, each stored with k or with its row index contiguous, and
// for FP8 operands (k contiguous) whose blocks of 128 along k carry a
// power-of-two scale that the tensor core applies (block-scaled MMA).
//
// What bounds it: the MMA rate for large products, and the bytes a tile pulls
// through L2.  A tile of R x C costs (R + C) * 128 B of loads per 128-byte
// slice of k, so the large form pairs two CTAs (cta_group::2) on a 256 x 256
// tile: each CTA loads 128 rows of A and 128 rows of B per slice, 32 KB for
// 512 cycles of MMA.  The small form (one CTA, 128 x 128) keeps the SMs busy
// when there are too few large tiles; the launcher chooses by tile count.
//
// A CTA has 8 warps: warps 0-3 read the accumulator and write the result
// (warp w owns TMEM lanes 32w..32w+31, one row of the tile per lane), warp 4
// issues the TMA loads, warp 5 the MMAs, warp 6 stages the FP8 block scales.
// Grids are persistent; the accumulator is double-buffered in TMEM so that one
// tile's result is written while the next is computed.
//
// Every wait is bounded: a role that waits longer than kWaitCycles records
// where in *status, stops, and the CTA leaves after its copies had time to land.
#pragma once

#include <cstdint>
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "srs_common.cuh"

namespace srs {

constexpr int kSliceBytes = 128;        // bytes of k per pipeline stage and row (one swizzle row)
constexpr int kProductThreads = 256;
constexpr int kStages = 6;
constexpr int kScaleSlots = 3;          // ring of scale groups (each covers 4 slices)
constexpr int kPanelBytes = 128 * kSliceBytes;  // 128 rows of an operand per stage
constexpr int kPieceBytes = 32 * 128;   // a warp's piece of results on its way out
constexpr long long kWaitCycles = 4000000000ll;  // about 2 s

enum : int { kOperandF16 = 0, kOperandF8 = 1 };
enum : int { kEpilogueSymmetric = 0, kEpilogueStore = 1, kEpilogueMuon = 2 };

// What happens to the accumulator.
struct ProductEpilogue {
  const float* rho;  // per batch entry: the operand X stands for X / rho (null: 1)
  int rho_power;     // 1 or 2
  float alpha;       // factor of the accumulator
  float beta;        // symmetric: factor of `addend`
  float diagonal;    // symmetric: added where i == j
  const __half* addend;  // symmetric: M x M, row pitch ldd (null: none)
  void* out;
  int out_format;     // SRS_FMT_F32, SRS_FMT_BF16 or SRS_FMT_F16
  int64_t ldd;        // row pitch of out (elements)
  int64_t batch_stride;  // batch pitch of out (elements)
  const srs_row* rows;   // Muon: one row per batch entry (param address, dtype flag)
  float decay;        // Muon: p' = fma(step, D, p * decay)
  float step;
};

struct ProductArgs {
  int m, n, k;        // elements
  int tiles_m, tiles_n;  // tiles per batch entry
  int64_t n_tiles;    // over the batch
  int64_t tiles_per_entry;
  int symmetric;      // only tiles on and below the diagonal are computed
  uint32_t idesc;     // MMA instruction descriptor without scale ids
  int a_rows_inner;   // operand A is stored with its row index contiguous
  int b_rows_inner;
  // FP8: scales of A and B (UE8M0), row pitch in blocks; shift 7 when one scale
  // covers 128 rows, else 0
  const uint8_t* scale_a;
  const uint8_t* scale_b;
  int64_t scale_a_pitch, scale_b_pitch;
  int scale_a_shift, scale_b_shift;
  unsigned int* status;
  ProductEpilogue e;
};

// ------------------------------------------------------------ PTX wrappers --

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

// Bounded wait for the completion of the phase of `parity`; false (and `where`
// recorded) when it did not come.
__device__ __forceinline__ bool barrier_wait(uint32_t bar, uint32_t parity, unsigned int* status,
                                             unsigned int where) {
  if (barrier_try(bar, parity)) return true;
  const long long start = clock64();
  while (!barrier_try(bar, parity)) {
    if (clock64() - start > kWaitCycles) {
      atomicOr(status, where);
      return false;
    }
  }
  return true;
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

// Scales of one operand for a warp: rows row0 + lane + 32 j (j < 4), blocks kb ..
// kb + 3 of each, one byte a block.  Rows outside the matrix read its last row
// instead (their data are zeros and their results are not stored); blocks from
// `last` on give 1 (127).  Rows on 4-byte boundaries are read a word at a time.
struct ScaleRows {
  const uint8_t* row[4];
  __device__ __forceinline__ void at(const uint8_t* scale, int64_t pitch, int shift, int first,
                                     int rows, int lane) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      row[j] = scale + (int64_t)(min(first + lane + 32 * j, rows - 1) >> shift) * pitch;
  }
  __device__ __forceinline__ void read(int kb, int last, bool words, uint32_t (&w)[4]) const {
    if (words && kb + 4 <= last) {
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = __ldg(reinterpret_cast<const uint32_t*>(row[j] + kb));
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        w[j] = 0x7F7F7F7Fu;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (kb + i < last)
            w[j] = (w[j] & ~(0xFFu << (8 * i))) | ((uint32_t)__ldg(row[j] + kb + i) << (8 * i));
      }
    }
  }
};

__device__ __forceinline__ bool scale_words(const uint8_t* scale, int64_t pitch, int kb) {
  return ((reinterpret_cast<uint64_t>(scale) | (uint64_t)pitch | (uint64_t)kb) & 3) == 0;
}

// ------------------------------------------------------------------- tiles --

struct TileAt {
  int batch, m, n;  // tile coordinates
};

// Tiles of an entry in bands of 8 tile rows, column by column within a band, so
// that the CTAs running at one time share rows of A and B in L2.
__device__ __forceinline__ TileAt tile_at(const ProductArgs& a, int64_t t) {
  TileAt r;
  r.batch = (int)(t / a.tiles_per_entry);
  const int64_t i = t - (int64_t)r.batch * a.tiles_per_entry;
  if (a.symmetric) {
    int row = (int)((sqrtf(8.0f * (float)i + 1.0f) - 1.0f) * 0.5f);
    while ((int64_t)(row + 1) * (row + 2) / 2 <= i) ++row;
    while ((int64_t)row * (row + 1) / 2 > i) --row;
    r.m = row;
    r.n = (int)(i - (int64_t)row * (row + 1) / 2);
  } else {
    const int64_t band = 8ll * a.tiles_n;
    const int first = (int)(i / band) * 8;
    const int rows = min(8, a.tiles_m - first);
    const int j = (int)(i % band);
    r.m = first + j % rows;
    r.n = j / rows;
  }
  return r;
}

// ---------------------------------------------------------------- epilogue --

// Results leave in pieces of 32 rows x 128 bytes: a lane holds one row's piece (32
// words), the warp turns it through shared memory (16-byte slots, slot index xor
// row so that both sides are conflict-free), and 8 lanes then store one row's 128
// bytes.  Rows that are not on 16-byte boundaries are stored by words, and 16-bit
// results of odd pitch by elements.
__device__ __forceinline__ uint32_t staged_slot(uint32_t base, int row, int slot) {
  return base + row * 128 + 16 * (slot ^ (row & 7));
}

__device__ __forceinline__ void stage_row(uint32_t base, int lane, const uint32_t (&w)[32]) {
#pragma unroll
  for (int j = 0; j < 8; ++j)
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(staged_slot(base, lane, j)),
                 "r"(w[4 * j]), "r"(w[4 * j + 1]), "r"(w[4 * j + 2]), "r"(w[4 * j + 3])
                 : "memory");
}

__device__ __forceinline__ uint4 staged_read4(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

__device__ __forceinline__ uint32_t staged_read(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

// Staged piece to rows of `size`-byte elements: `out` is the piece's first element,
// `pitch` and `cols` count elements, `rows` <= 32.
__device__ __forceinline__ void store_piece(uint32_t base, char* out, int size, int64_t pitch,
                                            int rows, int cols, int lane) {
  const uint64_t align = reinterpret_cast<uint64_t>(out) | (uint64_t)(pitch * size);
  const int bytes = min(cols * size, 128);
  const int64_t step = pitch * size;
  if ((align & 15) == 0 && (bytes & 15) == 0) {
    const int slot = lane & 7, row0 = lane >> 3;
    char* p = out + row0 * step + 16 * slot;
    if (16 * slot < bytes) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int row = 4 * i + row0;
        const uint4 v = staged_read4(staged_slot(base, row, slot));
        if (row < rows) *reinterpret_cast<uint4*>(p + 4 * i * step) = v;
      }
    }
  } else if ((align & 3) == 0) {
    const bool whole = 4 * lane + 4 <= bytes, half = !whole && 4 * lane < bytes;
    char* p = out + 4 * lane;
#pragma unroll 8
    for (int row = 0; row < rows; ++row, p += step) {
      const uint32_t v = staged_read(staged_slot(base, row, lane >> 2) + 4 * (lane & 3));
      if (whole) *reinterpret_cast<uint32_t*>(p) = v;
      else if (half) *reinterpret_cast<uint16_t*>(p) = (uint16_t)v;
    }
  } else {
    char* p = out + 2 * lane;
#pragma unroll 4
    for (int row = 0; row < rows; ++row, p += step) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int e = lane + 32 * h;
        const uint32_t v = staged_read(staged_slot(base, row, e >> 3) + 4 * ((e >> 1) & 3));
        if (2 * e < bytes)
          *reinterpret_cast<uint16_t*>(p + 64 * h) = (uint16_t)(v >> (16 * (e & 1)));
      }
    }
  }
}

__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// p' = fma(step, D, p * decay) for the staged 32 x 32 FP32 piece of D.
template <bool BF16>
__device__ __forceinline__ void update_piece(uint32_t base, char* param, int64_t pitch, int rows,
                                             int cols, float step, float decay, int lane) {
  constexpr int kSize = BF16 ? 2 : 4;
  const auto next = [&](float p, uint32_t d) {
    return fmaf(step, __uint_as_float(d), __fmul_rn(p, decay));
  };
  const uint64_t align = reinterpret_cast<uint64_t>(param) | (uint64_t)(pitch * kSize);
  if ((align & (4 * kSize - 1)) == 0 && cols >= 32) {
    // 4 columns a lane, 4 rows at a time; all loads first
    const int slot = lane & 7, row0 = lane >> 3;
    char* p = param + (row0 * pitch + 4 * slot) * kSize;
    uint4 old[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      old[i] = make_uint4(0u, 0u, 0u, 0u);
      if (4 * i + row0 < rows) {
        const char* q = p + 4 * i * pitch * kSize;
        if constexpr (BF16) {
          const uint2 t = *reinterpret_cast<const uint2*>(q);
          old[i] = make_uint4(t.x << 16, t.x & 0xFFFF0000u, t.y << 16, t.y & 0xFFFF0000u);
        } else {
          old[i] = *reinterpret_cast<const uint4*>(q);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int row = 4 * i + row0;
      const uint4 d = staged_read4(staged_slot(base, row, slot));
      if (row >= rows) continue;
      char* q = p + 4 * i * pitch * kSize;
      const float a = next(__uint_as_float(old[i].x), d.x), b = next(__uint_as_float(old[i].y), d.y);
      const float c = next(__uint_as_float(old[i].z), d.z), e = next(__uint_as_float(old[i].w), d.w);
      if constexpr (BF16) *reinterpret_cast<uint2*>(q) = make_uint2(pack_bf16(a, b), pack_bf16(c, e));
      else *reinterpret_cast<float4*>(q) = make_float4(a, b, c, e);
    }
  } else if (lane < cols) {
    char* p = param + lane * kSize;
#pragma unroll 8
    for (int row = 0; row < rows; ++row, p += pitch * kSize) {
      const uint32_t d = staged_read(staged_slot(base, row, lane >> 2) + 4 * (lane & 3));
      if constexpr (BF16) {
        __nv_bfloat16* q = reinterpret_cast<__nv_bfloat16*>(p);
        *q = __float2bfloat16_rn(next(__bfloat162float(*q), d));
      } else {
        float* q = reinterpret_cast<float*>(p);
        *q = next(*q, d);
      }
    }
  }
}

// Where a warp's 32 accumulator rows go.
struct TileRows {
  int batch, row0, lane;
  int col_end;    // end of the tile's columns inside the matrix
  bool mirror;    // symmetric: also store the transposed tile
  float factor;
  uint32_t staged;
};

// This lane's row of the addend, 64 columns from col0 on (the pitch is a multiple of 8).
__device__ __forceinline__ void load_addend(const ProductArgs& a, const TileRows& t, int col0,
                                            uint4 (&add)[8]) {
  const ProductEpilogue& e = a.e;
  const int row = t.row0 + t.lane;
  const __half* from = e.addend + (int64_t)t.batch * e.batch_stride + (int64_t)row * e.ldd + col0;
#pragma unroll
  for (int j = 0; j < 8; ++j)
    add[j] = (row < a.m && col0 + 8 * j < e.ldd) ? __ldg(reinterpret_cast<const uint4*>(from) + j)
                                                 : make_uint4(0u, 0u, 0u, 0u);
}

// 64 accumulator columns from col0 on: v[0][c] and v[1][c] are columns c and 32 + c.
// `add` holds the addend's piece; the next piece's (next_col, -1: none) is requested
// before this one is stored.
template <int EPILOGUE>
__device__ __forceinline__ void write_columns(const ProductArgs& a, const TileRows& t, int col0,
                                              uint32_t (&v)[2][32], uint4 (&add)[8],
                                              int next_col) {
  const ProductEpilogue& e = a.e;
  const int row = t.row0 + t.lane, rows = min(32, a.m - t.row0);
  const int64_t at = (int64_t)t.batch * e.batch_stride;
  if constexpr (EPILOGUE == kEpilogueSymmetric) {
    __half* out = static_cast<__half*>(e.out) + at;
    uint32_t w[32];
    if (e.addend != nullptr) {
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        const uint4 q = add[i >> 2];
        const uint32_t pair = (i & 3) == 0 ? q.x : (i & 3) == 1 ? q.y : (i & 3) == 2 ? q.z : q.w;
        const float2 g = f16x2_to_float2(pair);
        const float x = __uint_as_float(v[i >> 4][(2 * i) & 31]) * t.factor;
        const float y = __uint_as_float(v[i >> 4][(2 * i + 1) & 31]) * t.factor;
        const int col = col0 + 2 * i;
        w[i] = pack_half(fmaf(e.beta, g.x, x) + (row == col ? e.diagonal : 0.0f),
                         fmaf(e.beta, g.y, y) + (row == col + 1 ? e.diagonal : 0.0f));
      }
      if (next_col >= 0) load_addend(a, t, next_col, add);
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i)
        w[i] = pack_half(__uint_as_float(v[i >> 4][(2 * i) & 31]) * t.factor,
                         __uint_as_float(v[i >> 4][(2 * i + 1) & 31]) * t.factor);
    }
    if (t.mirror) {
      // Lane pairs swap halves: the even lane gets two rows of an even column, the
      // odd lane of the next one, so a store covers 2 x 64 bytes.  (An odd last
      // row writes one padding element beside it.)
      const bool odd = (t.lane & 1) != 0;
      __half* to = out + (int64_t)(col0 + (odd ? 1 : 0)) * e.ldd + (row & ~1);
#pragma unroll
      for (int i = 0; i < 32; ++i, to += 2 * e.ldd) {
        const uint32_t other = __shfl_xor_sync(0xFFFFFFFFu, w[i], 1);
        const uint32_t pair =
            odd ? __byte_perm(other, w[i], 0x7632u) : __byte_perm(w[i], other, 0x5410u);
        if ((row & ~1) < a.m && col0 + 2 * i + (odd ? 1 : 0) < a.n)
          *reinterpret_cast<uint32_t*>(to) = pair;
      }
    }
    stage_row(t.staged, t.lane, w);
    __syncwarp();
    store_piece(t.staged, reinterpret_cast<char*>(out + (int64_t)t.row0 * e.ldd + col0), 2, e.ldd,
                rows, (int)e.ldd - col0, t.lane);
    __syncwarp();
  } else if (EPILOGUE == kEpilogueStore && e.out_format != SRS_FMT_F32) {
    uint32_t w[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const float x = __uint_as_float(v[i >> 4][(2 * i) & 31]) * t.factor;
      const float y = __uint_as_float(v[i >> 4][(2 * i + 1) & 31]) * t.factor;
      w[i] = e.out_format == SRS_FMT_BF16 ? pack_bf16(x, y) : pack_half(x, y);
    }
    stage_row(t.staged, t.lane, w);
    __syncwarp();
    store_piece(t.staged,
                static_cast<char*>(e.out) + 2 * (at + (int64_t)t.row0 * e.ldd + col0), 2, e.ldd,
                rows, t.col_end - col0, t.lane);
    __syncwarp();
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int col = col0 + 32 * h;
      if (col >= t.col_end) break;
#pragma unroll
      for (int c = 0; c < 32; ++c)
        v[h][c] = __float_as_uint(__uint_as_float(v[h][c]) * t.factor);
      stage_row(t.staged, t.lane, v[h]);
      __syncwarp();
      if constexpr (EPILOGUE == kEpilogueMuon) {
        const srs_row& target = e.rows[t.batch];
        const int64_t first = (int64_t)t.row0 * a.n + col;
        if (target.flags & SRS_ROW_PARAM_BF16)
          update_piece<true>(t.staged, reinterpret_cast<char*>(target.param) + 2 * first, a.n,
                             rows, t.col_end - col, e.step, e.decay, t.lane);
        else
          update_piece<false>(t.staged, reinterpret_cast<char*>(target.param) + 4 * first, a.n,
                              rows, t.col_end - col, e.step, e.decay, t.lane);
      } else {
        store_piece(t.staged,
                    static_cast<char*>(e.out) + 4 * (at + (int64_t)t.row0 * e.ldd + col), 4, e.ldd,
                    rows, t.col_end - col, t.lane);
      }
      __syncwarp();
    }
  }
}

// ------------------------------------------------------------------ kernel --

template <int KIND, int CG>
struct ProductShape {
  static constexpr int kTileRows = 128 * CG;  // over the CTA group
  static constexpr int kTileCols = 128 * CG;
  // Accumulator 1 starts after accumulator 0, except that for FP8 pairs both
  // accumulators and two groups of scales do not fit the 512 columns of TMEM: the
  // accumulators then share 32 columns, which the writing warps drain first, and a
  // tile starts once the one before is drained that far.  (Tiles of 240 columns
  // need no sharing and take fewer cycles, 17.0k instead of 18.6k for k = 4096, but
  // load more bytes per operation and were 4-7 % slower in time under the power
  // cap: 8192 x 14336 x 4096 429 us, with 256 columns 412 us.)
  static constexpr int kShared = KIND == kOperandF8 && CG == 2 ? 32 : 0;
  static constexpr int kSecond = kTileCols - kShared;
  static constexpr int kScaleBytes = KIND == kOperandF8 ? 512 * (1 + CG) : 0;  // per slot
  static constexpr int kScaleColumn = 480;  // 2 groups of 12 columns (pitch 16)
  static constexpr int kStageBytes = 2 * kPanelBytes;
  static constexpr int kSmem = 1024 + kStages * kStageBytes + kScaleSlots * kScaleBytes +
                               4 * kPieceBytes;
};

template <int KIND, int CG, int EPILOGUE>
__global__ void __launch_bounds__(kProductThreads, 1)
product_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
               const __grid_constant__ ProductArgs a) {
  using S = ProductShape<KIND, CG>;
  extern __shared__ uint8_t raw[];
  __shared__ __align__(8) uint64_t bars[2 * kStages + 4 + 2 * kScaleSlots];
  __shared__ uint32_t tmem_slot;

  const int warp = warp_index(), lane = threadIdx.x & 31;
  const uint32_t rank = CG == 2 ? cluster_rank() : 0u;
  const uint32_t stage0 = (smem_address(raw) + 1023u) & ~1023u;
  const uint32_t scales0 = stage0 + kStages * S::kStageBytes;
  const uint32_t staged0 = scales0 + kScaleSlots * S::kScaleBytes;

  const uint32_t bar0 = smem_address(bars);
  const auto full = [&](int s) { return bar0 + 8u * s; };
  const auto empty = [&](int s) { return bar0 + 8u * (kStages + s); };
  const auto acc_full = [&](int i) { return bar0 + 8u * (2 * kStages + i); };
  const auto acc_empty = [&](int i) { return bar0 + 8u * (2 * kStages + 2 + i); };
  const auto scale_full = [&](int i) { return bar0 + 8u * (2 * kStages + 4 + i); };
  const auto scale_empty = [&](int i) { return bar0 + 8u * (2 * kStages + 4 + kScaleSlots + i); };

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      barrier_init(full(s), 1);
      barrier_init(empty(s), 1);
    }
    for (int i = 0; i < 2; ++i) {
      barrier_init(acc_full(i), 1);
      barrier_init(acc_empty(i), 4 * CG);
    }
    for (int i = 0; i < kScaleSlots; ++i) {
      barrier_init(scale_full(i), CG);
      barrier_init(scale_empty(i), 1);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 5) tmem_alloc<CG>(smem_address(&tmem_slot), 512);
  tmem_fence_before();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync();
  tmem_fence_after();
  const uint32_t tmem = tmem_slot;

  const int64_t first = blockIdx.x / CG, step = gridDim.x / CG;
  constexpr int kSliceK = KIND == kOperandF8 ? 128 : 64;  // elements of k per stage
  const int slices = (a.k + kSliceK - 1) / kSliceK;
  bool ok = true;

  if (warp == 4) {
    const bool leader = elect_lane();
    // ---- TMA loads: this CTA's 128 rows of A and of B per slice
    int s = 0;
    uint32_t phase = 0;
    for (int64_t t = first; t < a.n_tiles && ok; t += step) {
      const TileAt at = tile_at(a, t);
      const int ra = at.m * S::kTileRows + 128 * (int)rank;
      const int rb = at.n * S::kTileCols + 128 * (int)rank;
      for (int i = 0; i < slices; ++i) {
        ok = barrier_wait(empty(s), phase ^ 1u, a.status, 1u);
        if (!ok) break;
        const uint32_t bar = CG == 2 ? map_to_rank(full(s), 0) : full(s);
        const uint32_t pa = stage0 + s * S::kStageBytes, pb = pa + kPanelBytes;
        const int k = i * kSliceK;
        if (leader) {
          if (rank == 0) barrier_expect(full(s), CG * S::kStageBytes);
          if (a.a_rows_inner) {
            load_box<CG>(pa, &map_a, ra, k, at.batch, bar);
            load_box<CG>(pa + kPanelBytes / 2, &map_a, ra + 64, k, at.batch, bar);
          } else {
            load_box<CG>(pa, &map_a, k, ra, at.batch, bar);
          }
          if (a.b_rows_inner) {
            load_box<CG>(pb, &map_b, rb, k, at.batch, bar);
            load_box<CG>(pb + kPanelBytes / 2, &map_b, rb + 64, k, at.batch, bar);
          } else {
            load_box<CG>(pb, &map_b, k, rb, at.batch, bar);
          }
        }
        __syncwarp();
        if (++s == kStages) {
          s = 0;
          phase ^= 1u;
        }
      }
    }
    // Every stage given back (its commit has reached this CTA) before leaving.
    for (int i = 0; i < kStages && ok; ++i) {
      ok = barrier_wait(empty(s), phase ^ 1u, a.status, 2u);
      if (++s == kStages) {
        s = 0;
        phase ^= 1u;
      }
    }
  } else if (warp == 5 && rank == 0) {
    const bool leader = elect_lane();
    // ---- MMAs (the pair's leader issues for both CTAs)
    const uint64_t desc_a = operand_descriptor(a.a_rows_inner != 0);
    const uint64_t desc_b = operand_descriptor(a.b_rows_inner != 0);
    // bytes per MMA step of k (32 bytes; 16 rows of 128 bytes when rows are inner)
    const uint32_t step_a = (a.a_rows_inner ? 2048u : 32u) >> 4;
    const uint32_t step_b = (a.b_rows_inner ? 2048u : 32u) >> 4;
    int s = 0, slot = 0, count = 0;
    uint32_t phase = 0, slot_phase = 0;
    // Scales go to TMEM one group ahead: the copy of group h is issued behind the
    // second slice of group h - 1, so that no MMA waits for it.  Its columns were
    // last read by group h - 2, whose last slice gave back stage done_stage.
    uint32_t group = 0, done_phase = 0;
    int done_stage = -1;
    const int groups = (slices + 3) >> 2;
    const auto copy_group = [&](uint32_t h) {
      if (done_stage >= 0) ok = barrier_wait(empty(done_stage), done_phase, a.status, 8u);
      ok = ok && barrier_wait(scale_full(slot), slot_phase, a.status, 8u);
      if (!ok) return;
      tmem_fence_after();
      const uint32_t src = scales0 + slot * S::kScaleBytes;
      const uint32_t dst = tmem + S::kScaleColumn + 16u * (h & 1u);
      if (leader) {
#pragma unroll
        for (int c = 0; c < 1 + CG; ++c)
          copy_scales<CG>(dst + 4 * c, scale_descriptor(src + 512 * c));
        mma_commit<CG>(scale_empty(slot));
      }
      __syncwarp();
      if (++slot == kScaleSlots) {
        slot = 0;
        slot_phase ^= 1u;
      }
    };
    if (KIND == kOperandF8 && first < a.n_tiles) copy_group(0);
    for (int64_t t = first; t < a.n_tiles && ok; t += step, ++count) {
      const int acc = count & 1;
      const uint32_t d = tmem + acc * S::kSecond;
      // The tile before the previous one has left this accumulator; with shared
      // columns, the previous tile has left those (and so has the one before it).
      if (S::kShared == 0) {
        if (count >= 2) ok = barrier_wait(acc_empty(acc), ((count >> 1) - 1) & 1u, a.status, 4u);
      } else {
        if (count >= 1) ok = barrier_wait(acc_empty(acc ^ 1), ((count - 1) >> 1) & 1u, a.status, 4u);
      }
      tmem_fence_after();
      for (int i = 0; i < slices && ok; ++i) {
        ok = barrier_wait(full(s), phase, a.status, 16u);
        if (!ok) break;
        tmem_fence_after();
        const uint32_t scale_tmem = tmem + S::kScaleColumn + 16u * (group & 1u);
        const uint32_t pa = stage0 + s * S::kStageBytes;
        const uint64_t da = desc_a | uint64_t((pa >> 4) & 0x3FFFu);
        const uint64_t db = desc_b | uint64_t(((pa + kPanelBytes) >> 4) & 0x3FFFu);
        const uint32_t id = (uint32_t)(i & 3);
        const uint32_t idesc = KIND == kOperandF8 ? a.idesc | (id << 29) | (id << 4) : a.idesc;
        if (leader) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t accumulate = (i | j) != 0 ? 1u : 0u;
            if constexpr (KIND == kOperandF8)
              mma_f8<CG>(d, da + j * step_a, db + j * step_b, idesc, scale_tmem, scale_tmem + 4,
                         accumulate);
            else
              mma_f16<CG>(d, da + j * step_a, db + j * step_b, idesc, accumulate);
          }
          mma_commit<CG>(empty(s));
        }
        __syncwarp();
        if constexpr (KIND == kOperandF8) {
          const bool last = id == 3 || i == slices - 1;
          if (id == 1 || (last && id == 0)) {
            if ((i >> 2) + 1 < groups || t + step < a.n_tiles) copy_group(group + 1);
          }
          if (last) {
            ++group;
            done_stage = s;
            done_phase = phase;
          }
        }
        if (++s == kStages) {
          s = 0;
          phase ^= 1u;
        }
      }
      if (ok && leader) mma_commit<CG>(acc_full(acc));
      __syncwarp();
    }
  } else if (KIND == kOperandF8 && warp == 6) {
    // ---- block scales: words of 4 consecutive scales (512 elements of k) per
    // row, row r at 16 * (r % 32) + 4 * (r / 32) of its 512-byte group, the order
    // in which the tensor core reads them from 4 TMEM columns
    const bool words_a = scale_words(a.scale_a, a.scale_a_pitch, 0);
    const bool words_b = scale_words(a.scale_b, a.scale_b_pitch, 0);
    int slot = 0;
    uint32_t phase = 0;
    // One group ahead: the next group's scales are requested before this one's
    // slot is waited for.
    int64_t t = first;
    int kb = 0;
    ScaleRows from[1 + CG];
    uint32_t next[1 + CG][4];
    const auto request = [&]() {
      if (kb == 0) {
        const TileAt at = tile_at(a, t);
        from[0].at(a.scale_a, a.scale_a_pitch, a.scale_a_shift,
                   at.m * S::kTileRows + 128 * (int)rank, a.m, lane);
#pragma unroll
        for (int c = 0; c < CG; ++c)
          from[1 + c].at(a.scale_b, a.scale_b_pitch, a.scale_b_shift,
                         at.n * S::kTileCols + 128 * c, a.n, lane);
      }
      from[0].read(kb, slices, words_a, next[0]);
#pragma unroll
      for (int c = 0; c < CG; ++c) from[1 + c].read(kb, slices, words_b, next[1 + c]);
      kb += 4;
      if (kb >= slices) {
        kb = 0;
        t += step;
      }
    };
    bool more = t < a.n_tiles;
    if (more) request();
    while (more) {
      uint32_t w[1 + CG][4];
#pragma unroll
      for (int c = 0; c < 1 + CG; ++c) {
#pragma unroll
        for (int j = 0; j < 4; ++j) w[c][j] = next[c][j];
      }
      more = t < a.n_tiles;
      if (more) request();
      ok = barrier_wait(scale_empty(slot), phase ^ 1u, a.status, 32u);
      ok = __all_sync(0xFFFFFFFFu, ok);
      if (!ok) break;
      const uint32_t dst = scales0 + slot * S::kScaleBytes + 16u * lane;
#pragma unroll
      for (int c = 0; c < 1 + CG; ++c)
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst + 512 * c), "r"(w[c][0]),
                     "r"(w[c][1]), "r"(w[c][2]), "r"(w[c][3])
                     : "memory");
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) barrier_arrive(map_to_rank(scale_full(slot), 0));
      if (++slot == kScaleSlots) {
        slot = 0;
        phase ^= 1u;
      }
    }
    for (int i = 0; i < kScaleSlots && ok; ++i) {
      ok = barrier_wait(scale_empty(slot), phase ^ 1u, a.status, 64u);
      if (++slot == kScaleSlots) {
        slot = 0;
        phase ^= 1u;
      }
    }
  } else if (warp < 4) {
    // ---- results
    int count = 0;
    for (int64_t t = first; t < a.n_tiles && ok; t += step, ++count) {
      const TileAt at = tile_at(a, t);
      const int acc = count & 1;
      float factor = a.e.alpha;
      if (a.e.rho != nullptr) {
        const float r = __ldg(a.e.rho + at.batch);
        factor = __fdiv_rn(factor, a.e.rho_power == 2 ? __fmul_rn(r, r) : r);
      }
      TileRows rows;
      rows.batch = at.batch;
      rows.row0 = at.m * S::kTileRows + 128 * (int)rank + 32 * warp;
      rows.lane = lane;
      rows.mirror = a.symmetric != 0 && at.m != at.n;
      rows.factor = factor;
      rows.staged = staged0 + warp * kPieceBytes;
      const int col0 = at.n * S::kTileCols;
      constexpr int kPieces = S::kTileCols / 64;
      rows.col_end = min(a.n, col0 + S::kTileCols);
      uint4 add[8];
      if (EPILOGUE == kEpilogueSymmetric && a.e.addend != nullptr) load_addend(a, rows, col0, add);
      ok = barrier_wait(acc_full(acc), (count >> 1) & 1u, a.status, 128u);
      ok = __all_sync(0xFFFFFFFFu, ok);
      if (!ok) break;
      tmem_fence_after();
      const uint32_t src = tmem + acc * S::kSecond + ((uint32_t)(warp * 32) << 16);
#pragma unroll 1
      for (int i = 0; i < kPieces; ++i) {
        // accumulator 0 gives its last (shared) columns first
        const int c = (S::kShared != 0 && acc == 0) ? kPieces - 1 - i : i;
        uint32_t v[2][32];
        tmem_load32(src + 64 * c, v[0]);
        tmem_load32(src + 64 * c + 32, v[1]);
        tmem_wait(v[0]);
        tmem_wait(v[1]);
        if (i == (S::kShared != 0 ? 0 : kPieces - 1)) {
          tmem_fence_before();
          __syncwarp();
          if (lane == 0) barrier_arrive(map_to_rank(acc_empty(acc), 0));
        }
        if (rows.row0 < a.m && col0 + 64 * c < rows.col_end)
          write_columns<EPILOGUE>(a, rows, col0 + 64 * c, v, add,
                                  c + 1 < kPieces ? col0 + 64 * (c + 1) : -1);
      }
    }
  }
  __syncwarp();
  if (!ok) {
    // A wait ran out: give copies and MMAs already issued time to finish before
    // shared memory and TMEM are given up.
    const long long start = clock64();
    while (clock64() - start < 4000000ll) {
    }
  }
  tmem_fence_before();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync();
  tmem_fence_after();
  if (warp == 5) tmem_free<CG>(tmem, 512);
}

// An operand in global memory: `rows` x `k` per batch entry.  k contiguous: row
// pitch `pitch` elements; rows_inner: element (i, k) at k * pitch + i.
struct ProductOperand {
  const void* base;
  int64_t rows, k, pitch, batch_stride;  // elements
  bool rows_inner;
};

// Enqueues D = A B^T of FP8 blocks where B has at most kThinRows rows (srs_product.cu);
// element (i, j) of D goes to i * row_stride + j * col_stride.
constexpr int kThinRows = 64;
int launch_thin(const ProductOperand& a, const ProductOperand& b, int a_format, int b_format,
                const ProductArgs& scales, void* out, int out_format, int64_t row_stride,
                int64_t col_stride, cudaStream_t stream);

// Enqueues D = A B^T with the given epilogue over `batch` entries (srs_product.cu).
// `args` carries the epilogue, the scales and the symmetric flag; the rest is
// filled in.  Returns SRS_OK or an error code with its text set.
int launch_product(int kind, int epilogue, const ProductOperand& a, const ProductOperand& b,
                   int64_t batch, int a_format, int b_format, ProductArgs args,
                   cudaStream_t stream);

}  // namespace srs
