// Matrix products on the sm_100a tensor cores (tcgen05, accumulators in TMEM):
//
//   D[i, j] = sum_k A[i, k] * B[j, k]      (A: M x K, B: N x K, FP32 accumulation)
//
// for FP16 operands, each stored with k or with its row index contiguous, and
// for FP8 operands (k contiguous) whose blocks of 128 along k carry a
// power-of-two scale that the tensor core applies (block-scaled MMA).
//
// What bounds it: the MMA rate for large products (and, after some milliseconds
// of them, the power limit), and the bytes a tile pulls through L2.  A tile of
// R x C costs (R + C) * 128 B of loads per 128-byte slice of k, so the large form
// pairs two CTAs (cta_group::2) on a 256 x 256 tile: each CTA loads 128 rows of A
// and 128 rows of B per slice, 32 KB for 512 cycles of MMA.  The small form (one
// CTA, 128 x 128) keeps the SMs busy when there are too few large tiles.
//
// A CTA has 8 warps that read the accumulator and write the result (warp w owns
// TMEM lanes 32 (w % 4) .., one row of the tile per lane, and its part of the
// columns), then one that issues the TMA loads, one for the MMAs and one that stages the
// FP8 block scales.  Grids are persistent; the accumulator is double-buffered in TMEM
// so that one tile's result is written while the next is computed.
//
// The work comes from a Source: one list of tiles, or several lists (phases), each
// of which reads what the one before has written.  Between phases all CTAs of the
// grid meet at a counter in global memory, one for each phase, as a CTA without
// tiles may report several phases ahead (such a grid is launched cooperatively).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "srs_common.cuh"
#include "srs_tcgen05.cuh"

namespace srs {

constexpr int kMaxPhases = 3 * SRS_NEWTON_MAX_STEPS;
constexpr int kScaleSlots = 3;          // ring of scale groups (each covers 4 slices)
constexpr int kPieceBytes = 32 * 128;   // a warp's piece of results on its way out

enum : int { kOperandF16 = 0, kOperandF8 = 1 };

// What the loading and multiplying warps need of a tile.
struct TileLoad {
  const CUtensorMap* map_a;
  const CUtensorMap* map_b;
  int row0, col0;  // first row of A and of B
  int batch;
  int slices;      // of 128 bytes along k
  bool a_rows_inner, b_rows_inner;
  // A symmetric operand is stored on and below its diagonal tiles alone: slices of k
  // past the tile's rows are read from the transposed tiles, with the row index
  // contiguous (maps map_a_t, map_b_t).
  bool a_symmetric, b_symmetric;
  const CUtensorMap* map_a_t;
  const CUtensorMap* map_b_t;
  // SPLIT: an operand is the sum of two FP16 matrices, high and low, whose maps lie
  // beside one another ([0] and [1] of every pointer above).  `slices` counts k three
  // times: low by high, high by low, then high by high parts.  (The tensor core truncates
  // its FP32 sums at every step: the small parts go first, while the sum is small;
  // 4096 x 14336 to FP32 was 1.3e-4 off so, with the high parts first 2.5e-4.)
};

// What happens to a tile's accumulator.
struct TileStore {
  int row0, col0;  // in the matrix
  int m, n;        // size of the matrix
  int update;      // 1: Muon's parameter update instead of a store
  float factor;    // of the accumulator
  const float* late;  // multiplies factor and beta (null: nothing), read while the sum runs
  float beta;      // of `addend`
  float diagonal;  // added where i == j
  const __half* addend;  // m x n, row pitch `pitch` (null: none)
  int addend_phase;      // the phase that wrote it (negative: an earlier kernel)
  char* out;       // first element of the matrix (update: of the parameter)
  int64_t low;     // bytes from a 16-bit result (SPLIT: and its addend) to its low part; 0: none
  int format;      // SRS_FMT_F32, SRS_FMT_BF16 or SRS_FMT_F16
  int64_t pitch;   // elements
  float step, decay;  // update: p' = fma(step, D, p * decay)
};

// Scales of one operand for a warp: rows row0 + lane + 32 j (j < 4), blocks kb ..
// kb + 3 of each, one byte a block.  Rows outside the matrix read its last row
// instead (their data are zeros and their results are not stored); blocks from
// `last` on give 1 (127).  Rows on 4-byte boundaries are read a word at a time.
//
// FRESH: the kernel ahead in the stream may write the scales while this one runs; they are
// then read (behind the wait for that kernel) through L2, never through the non-coherent
// path, which may hold what an earlier call left at their address.
struct ScaleRows {
  const uint8_t* row[4];
  __device__ __forceinline__ void at(const uint8_t* scale, int64_t pitch, int shift, int first,
                                     int rows, int lane) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      row[j] = scale + (int64_t)(min(first + lane + 32 * j, rows - 1) >> shift) * pitch;
  }
  template <bool FRESH = false, class T>
  __device__ static __forceinline__ T load(const T* p) {
    if constexpr (FRESH) return __ldcg(p);
    return __ldg(p);
  }
  template <bool FRESH = false>
  __device__ __forceinline__ void read(int kb, int last, bool words, uint32_t (&w)[4]) const {
    if (words && kb + 4 <= last) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        w[j] = load<FRESH>(reinterpret_cast<const uint32_t*>(row[j] + kb));
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        w[j] = 0x7F7F7F7Fu;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (kb + i < last)
            w[j] = (w[j] & ~(0xFFu << (8 * i))) |
                   ((uint32_t)load<FRESH>(row[j] + kb + i) << (8 * i));
      }
    }
  }
};

__device__ __forceinline__ bool scale_words(const uint8_t* scale, int64_t pitch, int kb) {
  return ((reinterpret_cast<uint64_t>(scale) | (uint64_t)pitch | (uint64_t)kb) & 3) == 0;
}

// Division of a 31-bit number by a number the host knows: with 2^(s-1) < d <= 2^s and
// mul = floor(2^(31+s) / d) + 1, n / d = floor(n * mul / 2^(31+s)) for n < 2^31, as
// the excess mul * d - 2^(31+s) is at most 2^s.
struct Divider {
  uint32_t d, mul;
  int shift;  // s - 1; -1: d == 1
  __device__ __forceinline__ uint32_t quotient(uint32_t n) const {
    return shift < 0 ? n : __umulhi(n, mul) >> shift;
  }
};

inline Divider make_divider(uint32_t d) {
  Divider r{d, 0u, -1};
  if (d > 1) {
    int s = 1;
    while (s < 32 && (1ull << s) < d) ++s;
    r.mul = (uint32_t)((1ull << (31 + s)) / d + 1);
    r.shift = s - 1;
  }
  return r;
}

// Tiles of a matrix in bands of 8 tile rows, column by column within a band, so that
// the CTAs running at one time share rows of A and B in L2.
struct TileGrid {
  uint32_t rows, cols;
  Divider band;  // 8 * cols
  Divider last;  // rows of the last band
  __device__ __forceinline__ void at(uint32_t i, int* row, int* col) const {
    const uint32_t b = band.quotient(i), j = i - b * band.d;
    if (8u * b + 8u <= rows) {
      *row = (int)(8u * b + (j & 7u));
      *col = (int)(j >> 3);
    } else {
      const uint32_t c = last.quotient(j);
      *row = (int)(8u * b + (j - c * last.d));
      *col = (int)c;
    }
  }
};

inline TileGrid make_grid(uint32_t rows, uint32_t cols) {
  return {rows, cols, make_divider(8u * cols), make_divider(rows % 8u ? rows % 8u : 8u)};
}

// Tile i of those on and below the diagonal, row by row.
__device__ __forceinline__ void triangle_tile(uint32_t i, int* row, int* col) {
  int r = (int)((sqrtf(8.0f * (float)i + 1.0f) - 1.0f) * 0.5f);
  while ((uint32_t)(r + 1) * (uint32_t)(r + 2) / 2u <= i) ++r;
  while ((uint32_t)r * (uint32_t)(r + 1) / 2u > i) --r;
  *row = r;
  *col = (int)(i - (uint32_t)r * (uint32_t)(r + 1) / 2u);
}

// ---------------------------------------------------------------- epilogue --

// Results leave in pieces of 32 rows x 32 columns: a lane holds one row's piece, the
// warp turns it through shared memory (16-byte slots, xored so that both sides are
// conflict-free), and the lanes then store whole rows, 64 bytes of 16-bit results or
// 128 of FP32 ones.  Rows that are not on 16-byte boundaries are stored by words,
// and 16-bit results of odd pitch by elements.  (Pieces and loops are small on
// purpose: a phase of few tiles runs this code once, from a cold instruction cache.)
//
// SLOTS: 16-byte slots of a row, 4 (16-bit results) or 8 (FP32).
template <int SLOTS>
__device__ __forceinline__ uint32_t staged_slot(uint32_t base, int row, int slot) {
  const int turn = SLOTS == 8 ? row & 7 : (row >> 1) & 3;
  return base + row * 16 * SLOTS + 16 * (slot ^ turn);
}

__device__ __forceinline__ void staged_write4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c,
                                              uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c),
               "r"(d)
               : "memory");
}

// A lane's row of a piece: words FIRST, FIRST + STEP, ... of `w`.
template <int SLOTS, int FIRST = 0, int STEP = 1>
__device__ __forceinline__ void stage_row(uint32_t base, int lane, const uint32_t (&w)[32]) {
#pragma unroll
  for (int j = 0; j < SLOTS; ++j) {
    const int i = FIRST + 4 * STEP * j;
    staged_write4(staged_slot<SLOTS>(base, lane, j), w[i], w[i + STEP], w[i + 2 * STEP],
                  w[i + 3 * STEP]);
  }
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

// Staged piece to rows of elements of SLOTS / 2 bytes: `out` is the piece's first
// element, `pitch` and `cols` count elements, `rows` <= 32.
template <int SLOTS>
__device__ __forceinline__ void store_piece(uint32_t base, char* out, int64_t pitch, int rows,
                                            int cols, int lane) {
  constexpr int kSize = SLOTS / 2, kAtOnce = 32 / SLOTS;  // element bytes; rows a pass
  const int64_t step = pitch * kSize;
  const uint64_t align = reinterpret_cast<uint64_t>(out) | (uint64_t)step;
  const int bytes = min(cols * kSize, 16 * SLOTS);
  if ((align & 15) == 0 && (bytes & 15) == 0) {
    const int slot = lane % SLOTS, row0 = lane / SLOTS;
    char* p = out + row0 * step + 16 * slot;
    if (16 * slot < bytes) {
#pragma unroll
      for (int i = 0; i < SLOTS; ++i) {
        const int row = kAtOnce * i + row0;
        const uint4 v = staged_read4(staged_slot<SLOTS>(base, row, slot));
        if (row < rows) *reinterpret_cast<uint4*>(p) = v;
        p += kAtOnce * step;
      }
    }
  } else if ((align & 3) == 0) {
    // 4 * SLOTS words a row: a warp takes one row of 32 words, or two of 16
    constexpr int kRows = SLOTS == 8 ? 1 : 2;
    const int word = lane % (4 * SLOTS), row0 = lane / (4 * SLOTS);
    const bool whole = 4 * word + 4 <= bytes, half = !whole && 4 * word < bytes;
    char* p = out + row0 * step + 4 * word;
#pragma unroll 4
    for (int row = row0; row < rows; row += kRows, p += kRows * step) {
      const uint32_t v = staged_read(staged_slot<SLOTS>(base, row, word >> 2) + 4 * (word & 3));
      if (whole) *reinterpret_cast<uint32_t*>(p) = v;
      else if (half) *reinterpret_cast<uint16_t*>(p) = (uint16_t)v;
    }
  } else {
    char* p = out + 2 * lane;
#pragma unroll 4
    for (int row = 0; row < rows; ++row, p += step) {
      const uint32_t v =
          staged_read(staged_slot<SLOTS>(base, row, lane >> 3) + 4 * ((lane >> 1) & 3));
      if (2 * lane < bytes) *reinterpret_cast<uint16_t*>(p) = (uint16_t)(v >> (16 * (lane & 1)));
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
      const uint4 d = staged_read4(staged_slot<8>(base, row, slot));
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
      const uint32_t d = staged_read(staged_slot<8>(base, row, lane >> 2) + 4 * (lane & 3));
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

// The addend's piece of 32 rows and columns from (row0, col0) on, whole rows at a time (the
// pitch is a multiple of 8): columns 8 (lane % 4) .. of rows lane / 4 + 8 i.  Written by an
// earlier phase of the same kernel: never through the non-coherent path.
__device__ __forceinline__ void load_addend(const TileStore& t, int row0, int col0, int lane,
                                            uint4 (&add)[4], int64_t bytes = 0) {
  const int row = row0 + (lane >> 2), col = col0 + 8 * (lane & 3);
  const char* from = reinterpret_cast<const char*>(t.addend + (int64_t)row * t.pitch + col) + bytes;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    add[i] = (row + 8 * i < t.m && col < t.pitch)
                 ? __ldcg(reinterpret_cast<const uint4*>(from + 16 * i * t.pitch))
                 : make_uint4(0u, 0u, 0u, 0u);
}

// v += beta * that piece, turned to this lane's row in the staging memory.
__device__ __forceinline__ void add_piece(const uint4 (&add)[4], float beta, uint32_t staged,
                                          int lane, uint32_t (&v)[32]) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    staged_write4(staged_slot<4>(staged, 8 * i + (lane >> 2), lane & 3), add[i].x, add[i].y,
                  add[i].z, add[i].w);
  __syncwarp();
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint4 q = staged_read4(staged_slot<4>(staged, lane, j));
    const uint32_t pairs[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 g = f16x2_to_float2(pairs[i]);
      uint32_t* to = v + 8 * j + 2 * i;
      to[0] = __float_as_uint(fmaf(beta, g.x, __uint_as_float(to[0])));
      to[1] = __float_as_uint(fmaf(beta, g.y, __uint_as_float(to[1])));
    }
  }
  __syncwarp();
}

// 32 accumulator columns from col0 on for a warp's 32 rows from row0 on: v[c] is
// column col0 + c of row row0 + lane.  `add` holds the addend's piece; the next piece's
// (next_col, -1: none) is requested before this one is stored.
template <bool NEWTON, bool SPLIT>
__device__ __forceinline__ void write_columns(const TileStore& t, int row0, int col0, int lane,
                                              uint32_t staged, uint32_t (&v)[32],
                                              uint4 (&add)[4], int next_col) {
  const int row = row0 + lane, rows = min(32, t.m - row0);
  const int64_t at = (int64_t)row0 * t.pitch + col0;
#pragma unroll
  for (int c = 0; c < 32; ++c) v[c] = __float_as_uint(__uint_as_float(v[c]) * t.factor);
  const auto value = [&](int c) { return __uint_as_float(v[c]); };
  if (t.format != SRS_FMT_F32 && !(NEWTON && t.update != 0)) {
    if (NEWTON && t.addend != nullptr) {
      add_piece(add, t.beta, staged, lane, v);
      if (SPLIT) {
        load_addend(t, row0, col0, lane, add, t.low);
        add_piece(add, t.beta, staged, lane, v);
      }
      if (next_col >= 0) load_addend(t, row0, next_col, lane, add);
      if (t.diagonal != 0.0f) {
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (row == col0 + i) v[i] = __float_as_uint(value(i) + t.diagonal);
      }
    }
    // Pairs in place: the rounded pair at 2 i and what it leaves (exact in FP32) at 2 i + 1.
    const bool low = NEWTON && t.low != 0;
    if (t.format == SRS_FMT_BF16) {
#pragma unroll
      for (int i = 0; i < 32; i += 2) v[i] = pack_bf16(value(i), value(i + 1));
    } else if (low) {
#pragma unroll
      for (int i = 0; i < 32; i += 2) {
        const uint32_t pair = pack_half(value(i), value(i + 1));
        const float2 high = f16x2_to_float2(pair);
        v[i + 1] = pack_half(value(i) - high.x, value(i + 1) - high.y);
        v[i] = pair;
      }
      stage_row<4, 1, 2>(staged + kPieceBytes / 2, lane, v);
    } else {
#pragma unroll
      for (int i = 0; i < 32; i += 2) v[i] = pack_half(value(i), value(i + 1));
    }
    stage_row<4, 0, 2>(staged, lane, v);
    __syncwarp();
    store_piece<4>(staged, t.out + 2 * at, t.pitch, rows, t.n - col0, lane);
    if (low)
      store_piece<4>(staged + kPieceBytes / 2, t.out + t.low + 2 * at, t.pitch, rows, t.n - col0,
                     lane);
  } else {
    stage_row<8>(staged, lane, v);
    __syncwarp();
    if (NEWTON && t.update != 0) {
      if (t.format == SRS_FMT_BF16)
        update_piece<true>(staged, t.out + 2 * at, t.pitch, rows, t.n - col0, t.step, t.decay,
                           lane);
      else
        update_piece<false>(staged, t.out + 4 * at, t.pitch, rows, t.n - col0, t.step, t.decay,
                            lane);
    } else {
      store_piece<8>(staged, t.out + 4 * at, t.pitch, rows, t.n - col0, lane);
    }
  }
  __syncwarp();
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
  // Writing warps.  16 leave 96 registers a thread, too few for a piece, its addend and its
  // low part: orthogonalising 768^2 took 141 us with 16 (single-CTA tiles) and 143 with 8,
  // 2048^2 252 and 242, 12 x 768^2 231 and 218, 4 x (1024 x 4096) 438 and 416.
  static constexpr int kWriters = 8;
  static constexpr int kThreads = 32 * (kWriters + 4);
  static constexpr int kStages = KIND == kOperandF16 && CG == 2 ? 6 : 5;  // 4 to 6 measure the same
  static constexpr int kScaleBytes = KIND == kOperandF8 ? 512 * (1 + CG) : 0;  // per slot
  static constexpr int kScaleColumn = 480;  // 2 groups of 12 columns (pitch 16)
  static constexpr int kStageBytes = 2 * kPanelBytes;
  static constexpr int kSmem = 1024 + kStages * kStageBytes + kScaleSlots * kScaleBytes +
                               kWriters * kPieceBytes;
  // Instruction descriptor: N / 8, M / 16 and, for FP16, FP32 accumulation; for FP8,
  // UE8M0 scales.  Operand formats and orders are added.
  static constexpr uint32_t kInstruction = (uint32_t)(kTileCols >> 3) << 17 |
                                           (uint32_t)(kTileRows >> 4) << 24 |
                                           (KIND == kOperandF8 ? 1u << 23 : 1u << 4);
};

// The CTA's work.  Source gives: phases(), tiles(phase), load(phase, tile),
// store(phase, tile), formats() (bits of the instruction descriptor), counter(phase),
// status() and longest() (slices of a tile, where they can take seconds); for FP8 also
// scales(): the operands' block scales.
template <int KIND, int CG, bool NEWTON, bool SPLIT, class Source>
__device__ __forceinline__ void run_products(const Source& src) {
  using S = ProductShape<KIND, CG>;
  constexpr int kStages = S::kStages;
  extern __shared__ uint8_t raw[];
  __shared__ __align__(8) uint64_t bars[2 * kStages + 4 + 2 * kScaleSlots];
  __shared__ uint32_t tmem_slot;
  __shared__ unsigned int phase_warps[NEWTON ? kMaxPhases : 1];  // writing warps done with each

  const int warp = warp_index(), lane = threadIdx.x & 31;
  const uint32_t rank = CG == 2 ? cluster_rank() : 0u;
  const uint32_t stage0 = (smem_address(raw) + 1023u) & ~1023u;
  const uint32_t scales0 = stage0 + kStages * S::kStageBytes;
  const uint32_t staged0 = scales0 + kScaleSlots * S::kScaleBytes;
  unsigned int* const status = src.status();

  const uint32_t bar0 = smem_address(bars);
  const auto full = [&](int s) { return bar0 + 8u * s; };
  const auto empty = [&](int s) { return bar0 + 8u * (kStages + s); };
  const auto acc_full = [&](int i) { return bar0 + 8u * (2 * kStages + i); };
  const auto acc_empty = [&](int i) { return bar0 + 8u * (2 * kStages + 2 + i); };
  const auto scale_full = [&](int i) { return bar0 + 8u * (2 * kStages + 4 + i); };
  const auto scale_empty = [&](int i) { return bar0 + 8u * (2 * kStages + 4 + kScaleSlots + i); };

  if (NEWTON && threadIdx.x < kMaxPhases) phase_warps[threadIdx.x] = 0u;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      barrier_init(full(s), 1);
      barrier_init(empty(s), 1);
    }
    for (int i = 0; i < 2; ++i) {
      barrier_init(acc_full(i), 1);
      barrier_init(acc_empty(i), S::kWriters * CG);
    }
    for (int i = 0; i < kScaleSlots; ++i) {
      barrier_init(scale_full(i), CG);
      barrier_init(scale_empty(i), 1);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == S::kWriters + 1) tmem_alloc<CG>(smem_address(&tmem_slot), 512);
  tmem_fence_before();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync();
  tmem_fence_after();
  const uint32_t tmem = tmem_slot;

  const uint32_t first = blockIdx.x / CG, step = gridDim.x / CG;
  constexpr int kSliceK = KIND == kOperandF8 ? 128 : 64;  // elements of k per stage
  const int phases = src.phases();
  bool ok = true;

  if (warp == S::kWriters) {
    // ---- TMA loads: this CTA's 128 rows of A and of B per slice
    const bool leader = elect_lane();
    int s = 0;
    uint32_t parity = 0;
    for (int p = 0; p < phases && ok; ++p) {
      const uint32_t tiles = src.tiles(p);
      TileLoad at{};
      if (first < tiles) {
        at = src.load(p, first);
        prefetch_map(at.map_a);
        prefetch_map(at.map_b);
      }
      if (p > 0) {
        // what the earlier phase wrote, seen by the copies that follow
        if (lane == 0) ok = counter_wait(src.counter(p - 1), gridDim.x, status, 1u << 16);
        ok = __all_sync(0xFFFFFFFFu, ok);
        __syncwarp();  // a vote orders no memory: what lane 0 has acquired, for the others
        asm volatile("fence.proxy.async;" ::: "memory");
      }
      for (uint32_t t = first; t < tiles && ok; t += step) {
        if (t != first) at = src.load(p, t);
        const int ra = at.row0 + 128 * (int)rank, rb = at.col0 + 128 * (int)rank;
        const int third = SPLIT ? at.slices / 3 : 0;
        for (int i = 0; i < at.slices; ++i) {
          ok = barrier_wait(empty(s), parity ^ 1u, status, 1u);
          if (!ok) break;
          const uint32_t bar = CG == 2 ? map_to_rank(full(s), 0) : full(s);
          const uint32_t pa = stage0 + s * S::kStageBytes, pb = pa + kPanelBytes;
          const int part = SPLIT ? (i >= third) + (i >= 2 * third) : 0;
          const int k = (i - part * third) * kSliceK;
          const int low_a = SPLIT && part == 0 ? 1 : 0, low_b = SPLIT && part == 1 ? 1 : 0;
          if (leader) {
            if (rank == 0) barrier_expect(full(s), CG * S::kStageBytes);
            const bool past_a = NEWTON && at.a_symmetric && k >= at.row0 + S::kTileRows;
            const bool past_b = NEWTON && at.b_symmetric && k >= at.col0 + S::kTileCols;
            if (NEWTON && (at.a_rows_inner || past_a)) {
              const CUtensorMap* map = (past_a ? at.map_a_t : at.map_a) + low_a;
              load_box<CG>(pa, map, ra, k, at.batch, bar);
              load_box<CG>(pa + kPanelBytes / 2, map, ra + 64, k, at.batch, bar);
            } else {
              load_box<CG>(pa, at.map_a + low_a, k, ra, at.batch, bar);
            }
            if (NEWTON && (at.b_rows_inner || past_b)) {
              const CUtensorMap* map = (past_b ? at.map_b_t : at.map_b) + low_b;
              load_box<CG>(pb, map, rb, k, at.batch, bar);
              load_box<CG>(pb + kPanelBytes / 2, map, rb + 64, k, at.batch, bar);
            } else {
              load_box<CG>(pb, at.map_b + low_b, k, rb, at.batch, bar);
            }
          }
          __syncwarp();
          if (++s == kStages) {
            s = 0;
            parity ^= 1u;
          }
        }
      }
    }
    // Every stage given back (its commit has reached this CTA) before leaving.
    for (int i = 0; i < kStages && ok; ++i) {
      ok = barrier_wait(empty(s), parity ^ 1u, status, 2u);
      if (++s == kStages) {
        s = 0;
        parity ^= 1u;
      }
    }
  } else if (warp == S::kWriters + 1 && rank == 0) {
    // ---- MMAs (the pair's leader issues for both CTAs)
    const bool leader = elect_lane();
    int s = 0, slot = 0, count = 0;
    uint32_t parity = 0, slot_parity = 0;
    // Scales go to TMEM one group ahead: the copy of group h is issued behind the
    // second slice of group h - 1, so that no MMA waits for it.  Its columns were
    // last read by group h - 2, whose last slice gave back stage done_stage.
    uint32_t group = 0, done_parity = 0;
    int done_stage = -1;
    const auto copy_group = [&](uint32_t h) {
      if (done_stage >= 0) ok = barrier_wait(empty(done_stage), done_parity, status, 8u);
      ok = ok && barrier_wait(scale_full(slot), slot_parity, status, 8u);
      if (!ok) return;
      tmem_fence_after();
      const uint32_t from = scales0 + slot * S::kScaleBytes;
      const uint32_t to = tmem + S::kScaleColumn + 16u * (h & 1u);
      if (leader) {
#pragma unroll
        for (int c = 0; c < 1 + CG; ++c)
          copy_scales<CG>(to + 4 * c, scale_descriptor(from + 512 * c));
        mma_commit<CG>(scale_empty(slot));
      }
      __syncwarp();
      if (++slot == kScaleSlots) {
        slot = 0;
        slot_parity ^= 1u;
      }
    };
    if (KIND == kOperandF8 && first < src.tiles(0)) copy_group(0);
    for (int p = 0; p < phases && ok; ++p) {
      const uint32_t tiles = src.tiles(p);
      for (uint32_t t = first; t < tiles && ok; t += step, ++count) {
        const TileLoad at = src.load(p, t);
        const int third = SPLIT ? at.slices / 3 : 0;
        const int groups = (at.slices + 3) >> 2;
        const int acc = count & 1;
        const uint32_t d = tmem + acc * S::kSecond;
        // The tile before the previous one has left this accumulator; with shared
        // columns, the previous tile has left those (and so has the one before it).
        if (S::kShared == 0) {
          if (count >= 2) ok = barrier_wait(acc_empty(acc), ((count >> 1) - 1) & 1u, status, 4u);
        } else {
          if (count >= 1) ok = barrier_wait(acc_empty(acc ^ 1), ((count - 1) >> 1) & 1u, status, 4u);
        }
        tmem_fence_after();
        for (int i = 0; i < at.slices && ok; ++i) {
          ok = barrier_wait(full(s), parity, status, 16u);
          if (!ok) break;
          tmem_fence_after();
          const uint32_t scale_tmem = tmem + S::kScaleColumn + 16u * (group & 1u);
          const uint32_t pa = stage0 + s * S::kStageBytes;
          const int part = SPLIT ? (i >= third) + (i >= 2 * third) : 0;
          const int k = (i - part * third) * kSliceK;
          const bool a_inner = NEWTON && (at.a_rows_inner ||
                                          (at.a_symmetric && k >= at.row0 + S::kTileRows));
          const bool b_inner = NEWTON && (at.b_rows_inner ||
                                          (at.b_symmetric && k >= at.col0 + S::kTileCols));
          const uint64_t da = operand_descriptor(a_inner) | uint64_t((pa >> 4) & 0x3FFFu);
          const uint64_t db =
              operand_descriptor(b_inner) | uint64_t(((pa + kPanelBytes) >> 4) & 0x3FFFu);
          // 16-byte units per MMA step of k (32 bytes; 16 rows of 128 bytes when rows are inner)
          const uint32_t step_a = (a_inner ? 2048u : 32u) >> 4, step_b = (b_inner ? 2048u : 32u) >> 4;
          const uint32_t base = S::kInstruction | src.formats() | (a_inner ? 1u << 15 : 0u) |
                                (b_inner ? 1u << 16 : 0u);
          const uint32_t id = (uint32_t)(i & 3);
          const uint32_t idesc = KIND == kOperandF8 ? base | (id << 29) | (id << 4) : base;
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
            const bool last = id == 3 || i == at.slices - 1;
            if (id == 1 || (last && id == 0)) {
              if ((i >> 2) + 1 < groups || t + step < tiles) copy_group(group + 1);
            }
            if (last) {
              ++group;
              done_stage = s;
              done_parity = parity;
            }
          }
          if (++s == kStages) {
            s = 0;
            parity ^= 1u;
          }
        }
        if (ok && leader) mma_commit<CG>(acc_full(acc));
        __syncwarp();
      }
    }
  } else if (warp == S::kWriters + 2) {
    if constexpr (KIND == kOperandF8) {
      // ---- block scales: words of 4 consecutive scales (512 elements of k) per row,
      // row r at 16 * (r % 32) + 4 * (r / 32) of its 512-byte group, the order in
      // which the tensor core reads them from 4 TMEM columns.  One group ahead: the
      // next group's scales are requested before this one's slot is waited for.
      const auto scales = src.scales();
      int slot = 0;
      uint32_t parity = 0;
      uint32_t t = first;
      int kb = 0, slices = 0;
      ScaleRows from[1 + CG];
      uint32_t next[1 + CG][4];
      const uint32_t tiles = src.tiles(0);
      const auto request = [&]() {
        if (kb == 0) {
          const TileLoad at = src.load(0, t);
          slices = at.slices;
          from[0].at(scales.a, scales.a_pitch, scales.a_shift, at.row0 + 128 * (int)rank, scales.m,
                     lane);
#pragma unroll
          for (int c = 0; c < CG; ++c)
            from[1 + c].at(scales.b, scales.b_pitch, scales.b_shift, at.col0 + 128 * c, scales.n,
                           lane);
        }
        from[0].read(kb, slices, scales.a_words, next[0]);
#pragma unroll
        for (int c = 0; c < CG; ++c) from[1 + c].read(kb, slices, scales.b_words, next[1 + c]);
        kb += 4;
        if (kb >= slices) {
          kb = 0;
          t += step;
        }
      };
      bool more = t < tiles;
      if (more) request();
      while (more) {
        uint32_t w[1 + CG][4];
#pragma unroll
        for (int c = 0; c < 1 + CG; ++c) {
#pragma unroll
          for (int j = 0; j < 4; ++j) w[c][j] = next[c][j];
        }
        more = t < tiles;
        if (more) request();
        ok = barrier_wait(scale_empty(slot), parity ^ 1u, status, 32u);
        ok = __all_sync(0xFFFFFFFFu, ok);
        if (!ok) break;
        const uint32_t to = scales0 + slot * S::kScaleBytes + 16u * lane;
#pragma unroll
        for (int c = 0; c < 1 + CG; ++c)
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to + 512 * c),
                       "r"(w[c][0]), "r"(w[c][1]), "r"(w[c][2]), "r"(w[c][3])
                       : "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) barrier_arrive(map_to_rank(scale_full(slot), 0));
        if (++slot == kScaleSlots) {
          slot = 0;
          parity ^= 1u;
        }
      }
      for (int i = 0; i < kScaleSlots && ok; ++i) {
        ok = barrier_wait(scale_empty(slot), parity ^ 1u, status, 64u);
        if (++slot == kScaleSlots) {
          slot = 0;
          parity ^= 1u;
        }
      }
    }
  } else if (warp < S::kWriters) {
    // ---- results: this warp's 32 rows, its part of the tile's 32-column pieces
    constexpr int kPieces = S::kTileCols / (8 * S::kWriters);
    const int part = warp >> 2, quarter = warp & 3;
    const uint32_t staged = staged0 + warp * kPieceBytes;
    int count = 0, met = -1;  // met: the last phase known to be complete
    // These warps wait for whole tiles: beyond the limit of other waits, 4096 cycles a slice
    // of k.  (A tile alone on the GPU takes 700 to 840: 3 s for 2^30 of k.)
    const long long patience = kWaitCycles + 4096ll * src.longest();
    for (int p = 0; p < phases && ok; ++p) {
      const uint32_t tiles = src.tiles(p);
      for (uint32_t t = first; t < tiles && ok; t += step, ++count) {
        TileStore at = src.store(p, t);
        const int acc = count & 1;
        const int row0 = at.row0 + 128 * (int)rank + 32 * quarter;
        uint4 add[4];
        if (NEWTON && at.addend != nullptr) {
          // the one thing these warps read of an earlier phase
          if (met < at.addend_phase) {
            if (lane == 0)
              ok = counter_wait(src.counter(at.addend_phase), gridDim.x, status, 1u << 17);
            ok = __all_sync(0xFFFFFFFFu, ok);
            __syncwarp();  // what lane 0 has acquired, for the other lanes' loads
            if (!ok) break;
            met = at.addend_phase;
          }
          load_addend(at, row0, at.col0 + 32 * part * kPieces, lane, add);
        }
        float late = 1.0f;
        if (NEWTON && at.late != nullptr) late = __ldg(at.late);
        ok = barrier_wait(acc_full(acc), (count >> 1) & 1u, status, 128u, patience);
        ok = __all_sync(0xFFFFFFFFu, ok);
        if (!ok) break;
        tmem_fence_after();
        if (NEWTON) {
          at.factor *= late;
          at.beta *= late;
        }
        const uint32_t from = tmem + acc * S::kSecond + ((uint32_t)(quarter * 32) << 16);
#pragma unroll 1
        for (int i = 0; i < kPieces; ++i) {
          // accumulator 0 gives its last (shared) columns first
          const int c = part * kPieces + ((S::kShared != 0 && acc == 0) ? kPieces - 1 - i : i);
          uint32_t v[32];
          tmem_load32(from + 32 * c, v);
          tmem_wait(v);
          if (i == (S::kShared != 0 ? 0 : kPieces - 1)) {
            tmem_fence_before();
            __syncwarp();
            if (lane == 0) barrier_arrive_relaxed(map_to_rank(acc_empty(acc), 0));
          }
          if (row0 < at.m && at.col0 + 32 * c < at.n)
            write_columns<NEWTON, SPLIT>(at, row0, at.col0 + 32 * c, lane, staged, v, add,
                                  i + 1 < kPieces ? at.col0 + 32 * (c + 1) : -1);
        }
      }
      if (NEWTON && p + 1 < phases && ok) {
        // This CTA's results of the phase: each warp's stores, passed on inside the CTA,
        // then released to the grid by the last warp.  (The reading side orders them
        // before its copies.)
        __syncwarp();
        if (lane == 0 && shared_count(&phase_warps[p]) == S::kWriters - 1u)
          counter_arrive(src.counter(p));
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
  if (warp == S::kWriters + 1) tmem_free<CG>(tmem, 512);
}

}  // namespace srs
