// FP8 blocks: quantisation with a power-of-two scale for every 128 elements (or
// 128 x 128), and the products of such matrices.
//
// Why powers of two: scaling is then exact, so an element is rounded once, and
// the tensor core's block-scaled MMA applies the scales itself (UE8M0), so the
// product loop has no FP32 work of its own.
#include "srs_host.h"
#include "srs_common.cuh"
#include "srs_groups.cuh"
#include "srs_launch.h"

namespace srs {
namespace {

constexpr int kBlock = 128;

struct QuantizeArgs {
  const void* x;
  int64_t rows, cols, x_pitch;
  int vec;  // x's rows start on 16-byte boundaries
  int rule;
  uint32_t ctr, ctr_t;  // counters of element 0 of the copy and of the transposed copy
  uint8_t* data;
  uint8_t* scale;
  uint8_t* data_t;
  uint8_t* scale_t;
  int64_t data_pitch, scale_pitch, data_t_pitch, scale_t_pitch;
  // kStack: elements (scales: bytes) from one matrix to the next
  int64_t x_stride, data_stride, scale_stride, data_t_stride, scale_t_stride;
  // kGroups: see below
  const int32_t* ends;
  int groups;
  const int32_t* order;  // rows kernel: row i of the copy is row order[i] of x (null: i)
  bool overlap;          // host: launched beside the kernel ahead
};

// What a tile kernel's grid covers: one matrix; a stack of them (blockIdx.z), whose counters
// go on from one to the next; or the rows of groups, tiles counted from a group's first
// row.  The transposed copy of groups has the columns of tile i of all groups' tiles at
// 128 i, zeros behind a group's last row; its scales are words of 4 blocks, the words of all its
// rows one after the other, and a group starts with a new word.  Rows of no group are not written.
enum : int { kMatrix = 0, kStack = 1, kGroups = 2 };

// k of a block whose largest finite |x| has FP32 encoding u: the largest values of
// both formats are 1.75 * 2^TOP, so k = exponent - TOP, plus one where the
// significand exceeds 1.75 (adding 0x1FFFFF carries exactly then).
template <int OF>
__device__ __forceinline__ int block_exponent(uint32_t u) {
  constexpr int kTop = OF == SRS_FMT_E4M3 ? 8 : 15;
  if (u == 0u) return 0;
  return max((int)((u + 0x1FFFFFu) >> 23) - 127 - kTop, -127);
}

__device__ __forceinline__ float power_of_two(int k) {  // -126 <= k <= 127
  return __uint_as_float((uint32_t)(k + 127) << 23);
}

// Sizes are compared as encodings without their sign, two 16-bit ones to a word.
template <int XF>
struct Size {
  static constexpr bool kPacked = Fmt<XF>::kBytes == 2;
  static constexpr uint32_t kMask = kPacked ? 0x7FFF7FFFu : 0x7FFFFFFFu;
  // first encoding that is not a finite number
  static constexpr uint32_t kInfinite =
      XF == SRS_FMT_F32 ? 0x7F800000u : XF == SRS_FMT_BF16 ? 0x7F80u : 0x7C00u;
  __device__ static uint32_t of(uint32_t word) { return word & kMask; }
  __device__ static uint32_t larger(uint32_t a, uint32_t b) {
    if constexpr (kPacked) {
      uint32_t r;
      asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
      return r;
    } else {
      return max(a, b);
    }
  }
  // sizes with those that are not of finite numbers taken as zero
  __device__ static uint32_t finite(uint32_t u) {
    if (!kPacked) return u < kInfinite ? u : 0u;
    return ((u & 0xFFFFu) < kInfinite ? u & 0xFFFFu : 0u) |
           ((u >> 16) < kInfinite ? u & 0xFFFF0000u : 0u);
  }
  // larger half of a word / FP32 encoding of one size
  __device__ static uint32_t single(uint32_t a) {
    return kPacked ? max(a & 0xFFFFu, a >> 16) : a;
  }
  __device__ static uint32_t as_f32(uint32_t u) {
    if (XF == SRS_FMT_F32) return u;
    if (XF == SRS_FMT_BF16) return u << 16;
    return __float_as_uint(__half2float(__ushort_as_half((unsigned short)u)));
  }
};

template <int XF>
__device__ __forceinline__ void load_words(const QuantizeArgs& a, int64_t row, int64_t row_end,
                                           int64_t col, uint32_t (&w)[kWords<XF>]) {
  const int64_t left = a.cols - col;
  if (row >= row_end || left <= 0) {
#pragma unroll
    for (int j = 0; j < kWords<XF>; ++j) w[j] = 0u;
  } else if (a.vec && left >= 8) {
    load_raw8<XF>(a.x, row * a.x_pitch + col, w);
  } else {
    load_raw_partial<XF>(a.x, row * a.x_pitch + col, left < 8 ? (int)left : 8, w);
  }
}

// `to`: the sizes in `w`, those of infinities and NaN set to zero.
template <int XF, int N>
__device__ __forceinline__ void only_finite(const uint32_t (&w)[N][kWords<XF>],
                                            uint32_t (&to)[N][kWords<XF>]) {
  using Z = Size<XF>;
#pragma unroll
  for (int i = 0; i < N; ++i) {
#pragma unroll
    for (int j = 0; j < kWords<XF>; ++j) to[i][j] = Z::finite(Z::of(w[i][j]));
  }
}

// Largest sizes of N rows of 128 elements, 8 of each row a lane of 16: lane l is given that
// of row l % N.  Two rows of 16-bit elements share a word, and each exchange between lanes
// halves the words that a lane keeps: 5 shuffles for 8 such rows instead of 32.
template <int XF, int N>
__device__ __forceinline__ uint32_t row_sizes(const uint32_t (&w)[N][kWords<XF>], int lane16) {
  using Z = Size<XF>;
  constexpr int kHeld = Z::kPacked ? N / 2 : N;
  uint32_t r[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    r[i] = Z::of(w[i][0]);
#pragma unroll
    for (int j = 1; j < kWords<XF>; ++j) r[i] = Z::larger(r[i], Z::of(w[i][j]));
  }
  if constexpr (Z::kPacked) {
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
      r[i] = Z::larger(__byte_perm(r[i], r[i + kHeld], 0x5410u),
                       __byte_perm(r[i], r[i + kHeld], 0x7632u));
  }
#pragma unroll
  for (int d = kHeld / 2; d > 0; d >>= 1) {
    const bool upper = (lane16 & d) != 0;
#pragma unroll
    for (int i = 0; i < d; ++i) {
      const uint32_t keep = upper ? r[i + d] : r[i], give = upper ? r[i] : r[i + d];
      r[i] = Z::larger(keep, __shfl_xor_sync(0xFFFFFFFFu, give, d));
    }
  }
#pragma unroll
  for (int d = kHeld; d < 16; d <<= 1)
    r[0] = Z::larger(r[0], __shfl_xor_sync(0xFFFFFFFFu, r[0], d));
  if constexpr (Z::kPacked) return (lane16 & kHeld) != 0 ? r[0] >> 16 : r[0] & 0xFFFFu;
  return r[0];
}

// Rounds 8 scaled values to 8 bytes.  Values of a block are finite and at most the
// format's largest after scaling unless the block held infinities or NaN: `plain` says
// that it did not, and the stochastic rule then needs no screen.  The general form (any
// value, toward zero) is kept out of line: compiled into every row, it left each warp of
// the stochastic form waiting 4.3 cycles an instruction for the instruction cache.
template <int OF>
__device__ __forceinline__ uint2 encode_plain(const float (&y)[kVec], uint32_t ctr, bool nearest) {
  uint32_t w[2];
  if (nearest) encode8<OF>(y, 0u, SRS_RULE_NEAREST, w);
  else encode8_stochastic_fast<OF>(y, ctr, w);
  return make_uint2(w[0], w[1]);
}

template <int OF>
__device__ __noinline__ uint2 encode_general(float4 a, float4 b, uint32_t ctr, int rule) {
  const float y[kVec] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  uint32_t w[2];
  encode8<OF>(y, ctr, rule, w);
  return make_uint2(w[0], w[1]);
}

template <int OF>
__device__ __forceinline__ uint2 encode_values(const float (&y)[kVec], uint32_t ctr, int rule,
                                               bool plain) {
  if (plain) return encode_plain<OF>(y, ctr, rule == SRS_RULE_NEAREST);
  return encode_general<OF>(make_float4(y[0], y[1], y[2], y[3]),
                            make_float4(y[4], y[5], y[6], y[7]), ctr, rule);
}

// `left` of the bytes in `w` (all, or those up to the end of a row): nothing is written outside
// the matrix, so that a copy may be columns of a wider buffer.
__device__ __forceinline__ void store_bytes(uint8_t* out, uint2 w, int left) {
  if (left >= 8) {
    *reinterpret_cast<uint2*>(out) = w;
  } else {
    uint64_t bytes = (uint64_t)w.y << 32 | w.x;
#pragma unroll 1
    for (int j = 0; j < left; ++j, bytes >>= 8) out[j] = (uint8_t)bytes;
  }
}

// Rows alone, 1 x 128 blocks: 16 lanes to a block, kAhead blocks of one column a
// half-warp with all their loads first.  HBM-bound when rounding to nearest (8192 x
// 4096: 20.5 us a call among others; 3 bytes an element at 6.5 TB/s would be 15), by the
// integer units for the stochastic rule's hashes (37 us).
constexpr int kAhead = 4;
static_assert(kMaxQuantizedRows <= 65535ll * 16 * kAhead, "the rows fit a grid's height");

__device__ __forceinline__ int64_t ordered_row(const QuantizeArgs& a, int64_t row) {
  const int64_t from = __ldg(a.order + row);
  return from >= 0 && from < a.rows ? from : 0;
}

template <int OF, int XF, bool ORDERED>
__global__ void __launch_bounds__(kThreads) quantize_rows_kernel(const QuantizeArgs a) {
  // A product launched to overlap this kernel (srs_linear_blocks) may start.
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int lane16 = threadIdx.x & 15;
  const int64_t col = (int64_t)blockIdx.x * kBlock + 8 * lane16;
  const int64_t row0 = ((int64_t)blockIdx.y * 16 + (threadIdx.x >> 4)) * kAhead;
  uint32_t raw[kAhead][kWords<XF>];
#pragma unroll
  for (int i = 0; i < kAhead; ++i) {
    int64_t row = row0 + i;
    // an entry of `order` that names no row of x reads its first
    if (ORDERED && row < a.rows) row = ordered_row(a, row);
    load_words<XF>(a, ORDERED && row0 + i >= a.rows ? a.rows : row, a.rows, col, raw[i]);
  }
  uint32_t top = row_sizes<XF, kAhead>(raw, lane16);
  bool plain = !__any_sync(0xFFFFFFFFu, top >= Size<XF>::kInfinite);
  if (!plain) {
    uint32_t sizes[kAhead][kWords<XF>];
    only_finite<XF>(raw, sizes);
    top = row_sizes<XF, kAhead>(sizes, lane16);
  }
  const int own_k = block_exponent<OF>(Size<XF>::as_f32(top));
  if (lane16 < kAhead && row0 + lane16 < a.rows)
    a.scale[(row0 + lane16) * a.scale_pitch + blockIdx.x] = (uint8_t)(own_k + 127);
  const float own_factor = power_of_two(-own_k);
  plain = plain && a.rule != SRS_RULE_TOWARD_ZERO;
  const int cols_left = (int)min(a.cols - col, (int64_t)kVec);
#pragma unroll
  for (int i = 0; i < kAhead; ++i) {
    const int64_t row = row0 + i;
    const float factor = __shfl_sync(0xFFFFFFFFu, own_factor, i, 16);
    if (row >= a.rows) continue;
    float y[kVec];
    decode8<XF>(raw[i], y);
#pragma unroll
    for (int j = 0; j < kVec; ++j) y[j] *= factor;
    const int64_t from = ORDERED ? ordered_row(a, row) : row;
    const uint2 w =
        encode_values<OF>(y, a.ctr + (uint32_t)(from * a.cols + col), a.rule, plain);
    store_bytes(a.data + row * a.data_pitch + col, w, cols_left);
  }
  // Launched beside the kernel ahead: done only when that one is.
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// One CTA quantises one 128 x 128 tile of x, read once into shared memory.  Thread t has
// columns 8 * (t % 16) .. of rows 8 * (t / 16) ..: a row's block maximum is a reduction
// over 16 lanes, a column's one over the 16 row groups.  The transposed copy's bytes
// are kept by rows (32-bit words rotated by 4 * (row / 16), so that both sides are
// conflict-free) and leave as 4 x 4 byte transposes, 128 bytes of a column at a time.
// Nearest: bound by waits for the loads and at the barriers (integer pipe 51 % busy);
// stochastic both ways: by the hashes (two an element, about 25 integer operations).
// 8192 x 4096 from BF16, both ways: 39 us to nearest, 72 us stochastic; the bytes alone
// would take 20.  128 x 128 blocks: 21 us rows, 31 both ways; stochastic 37 and 65.  A
// reduction of 4 shuffles for every row and 16 partial maxima a column instead of 8 took
// a fifth more.
template <int OF, int XF, bool ROWS, bool COLS, bool SQUARE, int COVER>
__global__ void __launch_bounds__(kThreads, Fmt<XF>::kBytes == 2 ? 4 : 2)
quantize_tile_kernel(const __grid_constant__ QuantizeArgs args) {
  QuantizeArgs a = args;
  if constexpr (COVER == kStack) {
    const int64_t z = blockIdx.z;
    a.x = static_cast<const char*>(a.x) + z * a.x_stride * Fmt<XF>::kBytes;
    a.data += z * a.data_stride;
    a.scale += z * a.scale_stride;
    a.data_t += z * a.data_t_stride;
    a.scale_t += z * a.scale_t_stride;
    a.ctr += (uint32_t)(z * a.rows * a.cols);
    a.ctr_t += (uint32_t)(z * a.rows * a.cols);
  }
  using Z = Size<XF>;
  constexpr int kW = kWords<XF>;
  extern __shared__ __align__(16) uint8_t tile_raw[];  // 128 x 128 elements of x
  __shared__ __align__(16) uint32_t tops[COLS && !SQUARE ? 8 * 16 * kW : 8];
  __shared__ float row_factor[kBlock];
  __shared__ __align__(16) uint32_t turned[COLS ? kBlock * 32 : 4];
  const int lane16 = threadIdx.x & 15, group = threadIdx.x >> 4;
  int64_t row0 = (int64_t)blockIdx.y * kBlock, row_end = a.rows;
  const int64_t col0 = (int64_t)blockIdx.x * kBlock;
  int64_t scale_t_at = blockIdx.y;  // column of the transposed copy's scales
  if constexpr (COVER == kGroups) {
    const GroupTile tile = find_group_tile(a.ends, a.groups, (int)a.rows, kBlock,
                                           (int)blockIdx.y, (int)(threadIdx.x & 31));
    if (tile.group < 0) return;
    row0 = tile.row0;
    row_end = tile.end;
    scale_t_at = tile.quads;
  }
  const int64_t row_base = row0 + 8 * group, col = col0 + 8 * lane16;
  // this thread's words of row i of its group: kW / 4 vectors of 16 bytes, 256 threads apart
  uint4* const mine = reinterpret_cast<uint4*>(tile_raw) + threadIdx.x;
  const auto slot = [&](int i, int v) { return (i * (kW / 4) + v) * kThreads; };

  bool plain = a.rule != SRS_RULE_TOWARD_ZERO;
  int tile_k = 0;          // SQUARE: the block's exponent
  float col_factor[kVec];  // else: the columns' factors
  {
    uint32_t raw[8][kW];
#pragma unroll
    for (int i = 0; i < 8; ++i) load_words<XF>(a, row_base + i, row_end, col, raw[i]);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
#pragma unroll
      for (int v = 0; v < kW / 4; ++v)
        mine[slot(i, v)] =
            make_uint4(raw[i][4 * v], raw[i][4 * v + 1], raw[i][4 * v + 2], raw[i][4 * v + 3]);
#pragma unroll
      for (int j = 0; j < kW; ++j) raw[i][j] = Z::of(raw[i][j]);  // from here on: the sizes
    }
    if constexpr (SQUARE) {
      uint32_t top;
#pragma unroll 1
      while (true) {
        top = 0u;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
#pragma unroll
          for (int j = 0; j < kW; ++j) top = Z::larger(top, raw[i][j]);
        }
        top = __reduce_max_sync(0xFFFFFFFFu, Z::single(top));
        __syncthreads();
        if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kThreads / 32; ++w) top = max(top, tops[w]);
        if (top < Z::kInfinite) break;  // the same for the whole CTA
        plain = false;
        only_finite<XF>(raw, raw);
      }
      tile_k = block_exponent<OF>(Z::as_f32(top));
    } else {
      if constexpr (ROWS) {
        uint32_t top;
#pragma unroll 1
        while (__any_sync(0xFFFFFFFFu,
                          (top = row_sizes<XF, 8>(raw, lane16)) >= Z::kInfinite)) {
          plain = false;
          only_finite<XF>(raw, raw);
        }
        const int k = block_exponent<OF>(Z::as_f32(top));
        if (lane16 < 8) {
          row_factor[8 * group + lane16] = power_of_two(-k);
          if (row_base + lane16 < row_end)
            a.scale[(row_base + lane16) * a.scale_pitch + blockIdx.x] = (uint8_t)(k + 127);
        }
      }
      if constexpr (COLS) {
        uint32_t col_top[kVec];
#pragma unroll 1
        while (true) {
          uint32_t top[kW];
#pragma unroll
          for (int j = 0; j < kW; ++j) {
            top[j] = raw[0][j];
#pragma unroll
            for (int i = 1; i < 8; ++i) top[j] = Z::larger(top[j], raw[i][j]);
            top[j] = Z::larger(top[j], __shfl_xor_sync(0xFFFFFFFFu, top[j], 16));
          }
          uint4* const all = reinterpret_cast<uint4*>(tops) + lane16;
          if ((group & 1) == 0) {
#pragma unroll
            for (int v = 0; v < kW / 4; ++v)
              all[((group >> 1) * (kW / 4) + v) * 16] =
                  make_uint4(top[4 * v], top[4 * v + 1], top[4 * v + 2], top[4 * v + 3]);
          }
          __syncthreads();
#pragma unroll
          for (int v = 0; v < kW / 4; ++v) {
#pragma unroll
            for (int g = 0; g < 8; ++g) {
              const uint4 q = all[(g * (kW / 4) + v) * 16];
              top[4 * v] = Z::larger(top[4 * v], q.x);
              top[4 * v + 1] = Z::larger(top[4 * v + 1], q.y);
              top[4 * v + 2] = Z::larger(top[4 * v + 2], q.z);
              top[4 * v + 3] = Z::larger(top[4 * v + 3], q.w);
            }
          }
          bool infinite = false;
#pragma unroll
          for (int j = 0; j < kW; ++j) {
            if (Z::kPacked) {
              col_top[2 * j % kVec] = top[j] & 0xFFFFu;
              col_top[(2 * j + 1) % kVec] = top[j] >> 16;
            } else {
              col_top[j] = top[j];
            }
            infinite = infinite || Z::single(top[j]) >= Z::kInfinite;
          }
          if (!__syncthreads_or(infinite)) break;
          plain = false;
          only_finite<XF>(raw, raw);
        }
#pragma unroll
        for (int j = 0; j < kVec; ++j) {
          const int k = block_exponent<OF>(Z::as_f32(col_top[j]));
          col_factor[j] = power_of_two(-k);
          if (group == 0 && col + j < a.cols)
            a.scale_t[COVER == kGroups
                          ? ((scale_t_at >> 2) * a.cols + col + j) * 4 + (scale_t_at & 3)
                          : (col + j) * a.scale_t_pitch + scale_t_at] = (uint8_t)(k + 127);
        }
      }
    }
  }
  __syncwarp();

  uint32_t ctr = a.ctr + (uint32_t)(row_base * a.cols + col);
  uint32_t ctr_t = a.ctr_t + (uint32_t)(row_base * a.cols + col);
  const float tile_factor = power_of_two(-tile_k);
  const int rows_left = (int)min(row_end - row_base, (int64_t)8);
  const int cols_left = (int)min(a.cols - col, (int64_t)kVec);
  uint8_t* out = a.data + row_base * a.data_pitch + col;
  uint32_t* turn = turned + (COLS ? 8 * group * 32 + ((2 * lane16 + 4 * (group >> 1)) & 31) : 0);
#pragma unroll 1
  for (int i = 0; i < 8; ++i) {
    uint32_t raw[kW];
#pragma unroll
    for (int v = 0; v < kW / 4; ++v) {
      const uint4 q = mine[slot(i, v)];
      raw[4 * v] = q.x;
      raw[4 * v + 1] = q.y;
      raw[4 * v + 2] = q.z;
      raw[4 * v + 3] = q.w;
    }
    float x[kVec], y[kVec];
    decode8<XF>(raw, x);
    if constexpr (ROWS) {
      const float factor = SQUARE ? tile_factor : row_factor[8 * group + i];
#pragma unroll
      for (int j = 0; j < kVec; ++j) y[j] = x[j] * factor;
      const uint2 w = encode_values<OF>(y, ctr, a.rule, plain);
      if (i < rows_left) store_bytes(out, w, cols_left);
      out += a.data_pitch;
    }
    if constexpr (COLS) {
#pragma unroll
      for (int j = 0; j < kVec; ++j) y[j] = x[j] * (SQUARE ? tile_factor : col_factor[j]);
      *reinterpret_cast<uint2*>(turn) = encode_values<OF>(y, ctr_t, a.rule, plain);
      turn += 32;
    }
    ctr += (uint32_t)a.cols;
    ctr_t += (uint32_t)a.cols;
  }
  if (SQUARE && threadIdx.x == 0) {
    if (ROWS)
      a.scale[(int64_t)blockIdx.y * a.scale_pitch + blockIdx.x] = (uint8_t)(tile_k + 127);
    if (COLS)
      a.scale_t[(int64_t)blockIdx.x * a.scale_t_pitch + scale_t_at] = (uint8_t)(tile_k + 127);
  }

  if constexpr (COLS) {
    __syncthreads();
    // 16 rows of 4 columns a thread
    const int h = threadIdx.x & 7, word = threadIdx.x >> 3;
    uint32_t out[4][4];  // column, 4 rows a word
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      uint32_t w[4];
#pragma unroll
      for (int r = 0; r < 4; ++r)
        w[r] = turned[(16 * h + 4 * q + r) * 32 + ((word + 4 * h) & 31)];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const uint32_t pick = (uint32_t)c | ((uint32_t)(c + 4) << 4);
        out[c][q] = __byte_perm(__byte_perm(w[0], w[1], pick), __byte_perm(w[2], w[3], pick),
                                0x5410u);
      }
    }
    // of groups: whole tiles, the rows behind a group's last are the zeros that were loaded
    const int64_t at = (int64_t)blockIdx.y * kBlock + 16 * h;
    const int left = COVER == kGroups ? 16 : (int)min(a.rows - at, (int64_t)16);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int64_t to = col0 + 4 * word + c;
      if (to >= a.cols) continue;
      uint8_t* const dst = a.data_t + to * a.data_t_pitch + at;
      if (left >= 16) {
        *reinterpret_cast<uint4*>(dst) = make_uint4(out[c][0], out[c][1], out[c][2], out[c][3]);
      } else {
        store_bytes(dst, make_uint2(out[c][0], out[c][1]), left);
        store_bytes(dst + 8, make_uint2(out[c][2], out[c][3]), left - 8);
      }
    }
  }
}

template <int OF, int XF, bool ROWS, bool COLS, bool SQUARE, int COVER = kMatrix>
cudaError_t launch_tile(const QuantizeArgs& a, dim3 grid, cudaStream_t stream) {
  constexpr int kTileBytes = kBlock * kBlock * Fmt<XF>::kBytes;
  const auto kernel = &quantize_tile_kernel<OF, XF, ROWS, COLS, SQUARE, COVER>;
  if (kTileBytes + (COLS ? 24 * 1024 : 0) > 40 * 1024) {
    const cudaError_t e =
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kTileBytes);
    if (e != cudaSuccess) return e;
  }
  kernel<<<grid, kThreads, kTileBytes, stream>>>(a);
  return cudaGetLastError();
}

// One form of block and of copies, for a matrix, a stack or groups.
template <int OF, int XF, int COVER>
cudaError_t launch_tiles(const QuantizeArgs& a, bool square, dim3 tiles, cudaStream_t stream) {
  const bool rows = a.data != nullptr, cols = a.data_t != nullptr;
  if constexpr (COVER != kGroups) {
    if (square) {
      if (rows && cols) return launch_tile<OF, XF, true, true, true, COVER>(a, tiles, stream);
      return rows ? launch_tile<OF, XF, true, false, true, COVER>(a, tiles, stream)
                  : launch_tile<OF, XF, false, true, true, COVER>(a, tiles, stream);
    }
    if (COVER == kStack && !cols)
      return launch_tile<OF, XF, true, false, false, COVER>(a, tiles, stream);
  }
  return rows ? launch_tile<OF, XF, true, true, false, COVER>(a, tiles, stream)
              : launch_tile<OF, XF, false, true, false, COVER>(a, tiles, stream);
}

template <int OF, int XF>
cudaError_t launch_quantize(const QuantizeArgs& a, bool square, int matrices,
                            cudaStream_t stream) {
  const unsigned columns = (unsigned)((a.cols + kBlock - 1) / kBlock);
  const dim3 tiles(columns, (unsigned)((a.rows + kBlock - 1) / kBlock));
  if (a.ends != nullptr) {
    const dim3 grid(columns, (unsigned)most_group_tiles(a.rows, a.groups, kBlock));
    return launch_tiles<OF, XF, kGroups>(a, false, grid, stream);
  }
  if (matrices > 1)
    return launch_tiles<OF, XF, kStack>(a, square, dim3(tiles.x, tiles.y, (unsigned)matrices),
                                        stream);
  if (square || a.data_t != nullptr) return launch_tiles<OF, XF, kMatrix>(a, square, tiles, stream);
  const dim3 grid(columns, (unsigned)((a.rows + 16 * kAhead - 1) / (16 * kAhead)));
  const auto kernel = a.order != nullptr ? &quantize_rows_kernel<OF, XF, true>
                                         : &quantize_rows_kernel<OF, XF, false>;
  if (!a.overlap) {
    kernel<<<grid, kThreads, 0, stream>>>(a);
    return cudaGetLastError();
  }
  cudaLaunchConfig_t config{};
  cudaLaunchAttribute attribute{};
  attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute.val.programmaticStreamSerializationAllowed = 1;
  config.gridDim = grid;
  config.blockDim = dim3(kThreads);
  config.stream = stream;
  config.attrs = &attribute;
  config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, kernel, a);
}

template <int OF>
cudaError_t launch_quantize(const QuantizeArgs& a, int x_format, bool square, int matrices,
                            cudaStream_t stream) {
  if (x_format == SRS_FMT_F32)
    return launch_quantize<OF, SRS_FMT_F32>(a, square, matrices, stream);
  if (x_format == SRS_FMT_BF16)
    return launch_quantize<OF, SRS_FMT_BF16>(a, square, matrices, stream);
  return launch_quantize<OF, SRS_FMT_F16>(a, square, matrices, stream);
}

// 16 bytes of the copy a thread, from any source alignment.
__global__ void __launch_bounds__(kThreads)
copy_rows_kernel(const uint8_t* __restrict__ src, int64_t src_pitch, int64_t rows, int64_t cols,
                 uint8_t* __restrict__ dst, int64_t dst_pitch) {
  const int64_t chunks = dst_pitch / 16;
  const int64_t stride = (int64_t)gridDim.x * kThreads;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < rows * chunks; i += stride) {
    const int64_t row = i / chunks, col = (i - row * chunks) * 16;
    const uint8_t* from = src + row * src_pitch + col;
    const int64_t left = cols - col;
    uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (j < left) w[j >> 2] |= (uint32_t)__ldg(from + j) << (8 * (j & 3));
    *reinterpret_cast<uint4*>(dst + row * dst_pitch + col) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

uint32_t host_h32(uint32_t x) {
  x ^= x >> 16;
  x *= 0x7FEB352Du;
  x ^= x >> 15;
  x *= 0x846CA68Bu;
  return x ^ (x >> 16);
}

int64_t blocks_of(int64_t x) { return (x + kBlock - 1) / kBlock; }

int check_copy(const char* what, const srs_block_copy& c, int64_t cols, int64_t blocks,
               int64_t matrices) {
  if (c.scale == 0) return fail(SRS_ERR_INVALID_ARGUMENT, "%s has data but no scale", what);
  if (c.data % 16 != 0 || c.pitch % 16 != 0 || c.pitch < cols ||
      (matrices > 1 && c.stride % 16 != 0))
    return fail(SRS_ERR_INVALID_ARGUMENT,
                "%s needs a 16-byte aligned address and a row pitch that is a multiple of 16 and "
                "at least the row length (%lld, %lld)",
                what, (long long)c.pitch, (long long)cols);
  if (c.scale_pitch < blocks)
    return fail(SRS_ERR_INVALID_ARGUMENT, "%s: scale pitch %lld, %lld blocks a row", what,
                (long long)c.scale_pitch, (long long)blocks);
  return SRS_OK;
}

}  // namespace

int check_groups(const int32_t* ends, int groups) {
  if (groups < 1 || groups > kMaxGroups)
    return fail(SRS_ERR_INVALID_ARGUMENT, "groups must be in [1, %d], got %d", kMaxGroups, groups);
  if (ends == nullptr || reinterpret_cast<uintptr_t>(ends) % 4 != 0)
    return fail(SRS_ERR_INVALID_ARGUMENT, "null or misaligned ends");
  return SRS_OK;
}

int check_operand(const char* what, const srs_blocks* b, int64_t k) {
  if (b == nullptr) return fail(SRS_ERR_INVALID_ARGUMENT, "null operand %s", what);
  if (b->format != SRS_FMT_E4M3 && b->format != SRS_FMT_E5M2)
    return fail(SRS_ERR_INVALID_ARGUMENT, "operand %s: unknown format %d", what, b->format);
  if (b->rows < 0 || b->rows > (1ll << 30))
    return fail(SRS_ERR_INVALID_ARGUMENT, "operand %s: %lld rows", what, (long long)b->rows);
  if (b->rows == 0 || k == 0) return SRS_OK;
  if (b->data == 0 || b->scale == 0)
    return fail(SRS_ERR_INVALID_ARGUMENT, "operand %s: null address", what);
  if (b->data % 16 != 0 || b->pitch % 16 != 0 || b->pitch < k)
    return fail(SRS_ERR_INVALID_ARGUMENT,
                "operand %s needs a 16-byte aligned address and a row pitch that is a multiple "
                "of 16 and at least k (%lld, %lld)",
                what, (long long)b->pitch, (long long)k);
  if (b->scale_pitch < blocks_of(k))
    return fail(SRS_ERR_INVALID_ARGUMENT, "operand %s: scale pitch %lld, %lld blocks a row", what,
                (long long)b->scale_pitch, (long long)blocks_of(k));
  return SRS_OK;
}

}  // namespace srs

using namespace srs;

int srs::quantize(const QuantizeCall& q, cudaStream_t stream) {
  if (q.x_format < SRS_FMT_F32 || q.x_format > SRS_FMT_F16)
    return fail(SRS_ERR_INVALID_ARGUMENT, "unsupported input format %d", q.x_format);
  if (q.out_format != SRS_FMT_E4M3 && q.out_format != SRS_FMT_E5M2)
    return fail(SRS_ERR_INVALID_ARGUMENT, "unknown output format %d (E4M3 or E5M2)", q.out_format);
  if (!valid_rule(q.rule)) return fail(SRS_ERR_INVALID_ARGUMENT, "unknown rounding rule %d", q.rule);
  if (q.rows < 0 || q.cols < 0 || q.x_pitch < 0 || q.matrices < 0)
    return fail(SRS_ERR_INVALID_ARGUMENT, "negative size or pitch");
  if (q.rows > kMaxQuantizedRows || q.cols > (1ll << 30) || q.matrices > 65535)
    return fail(SRS_ERR_INVALID_ARGUMENT, "%lld x %lld is too large", (long long)q.rows,
                (long long)q.cols);
  const srs_block_copy &copy = q.copy, &turned = q.turned;
  if (copy.data == 0 && turned.data == 0) return fail(SRS_ERR_INVALID_ARGUMENT, "null outputs");
  if (q.rows == 0 || q.cols == 0 || q.matrices == 0) return SRS_OK;
  if (q.x == nullptr) return fail(SRS_ERR_INVALID_ARGUMENT, "null input pointer");
  if (reinterpret_cast<uintptr_t>(q.x) % fmt_bytes(q.x_format) != 0)
    return fail(SRS_ERR_INVALID_ARGUMENT, "input pointer is not element aligned");
  const int64_t tiles = q.ends == nullptr ? 0 : most_group_tiles(q.rows, q.groups, kBlock);
  if (copy.data != 0)
    if (int rc = check_copy("the copy", copy, q.cols, blocks_of(q.cols), q.matrices)) return rc;
  if (turned.data != 0) {
    const int64_t cols = q.ends == nullptr ? q.rows : tiles * kBlock;
    const int64_t scales = q.ends == nullptr ? blocks_of(q.rows) : srs_group_scales(q.rows, q.groups);
    if (int rc = check_copy("the transposed copy", turned, cols, scales, q.matrices)) return rc;
  }
  if (int rc = check_device()) return rc;
  if (q.for_product)
    if (int rc = check_products()) return rc;
  QuantizeArgs a{};
  a.x = q.x;
  a.rows = q.rows;
  a.cols = q.cols;
  a.x_pitch = q.x_pitch;
  a.x_stride = q.x_stride;
  a.vec = reinterpret_cast<uintptr_t>(q.x) % 16 == 0 && q.x_pitch % 8 == 0 &&
          (q.matrices == 1 || q.x_stride % 8 == 0);
  a.rule = q.rule;
  a.ctr = q.offset + host_h32(q.seed);
  a.ctr_t = q.offset + host_h32(q.seed ^ 1u);
  a.data = reinterpret_cast<uint8_t*>(copy.data);
  a.scale = reinterpret_cast<uint8_t*>(copy.scale);
  a.data_t = reinterpret_cast<uint8_t*>(turned.data);
  a.scale_t = reinterpret_cast<uint8_t*>(turned.scale);
  a.data_pitch = copy.pitch;
  a.scale_pitch = copy.scale_pitch;
  a.data_stride = copy.stride;
  a.scale_stride = copy.scale_stride;
  a.data_t_pitch = turned.pitch;
  a.scale_t_pitch = turned.scale_pitch;
  a.data_t_stride = turned.stride;
  a.scale_t_stride = turned.scale_stride;
  a.ends = q.ends;
  a.groups = q.groups;
  a.order = q.order;
  a.overlap = q.overlap;
  const cudaError_t e =
      q.out_format == SRS_FMT_E4M3
          ? launch_quantize<SRS_FMT_E4M3>(a, q.x_format, q.square, (int)q.matrices, stream)
          : launch_quantize<SRS_FMT_E5M2>(a, q.x_format, q.square, (int)q.matrices, stream);
  return e == cudaSuccess ? SRS_OK : cuda_fail(e, "FP8 block quantisation launch");
}

extern "C" int srs_quantize_blocks(const void* x, int x_format, int64_t rows, int64_t cols,
                                   int64_t x_pitch, int out_format, int rule, int square,
                                   uint32_t seed, uint32_t offset, void* data, int64_t data_pitch,
                                   void* scale, int64_t scale_pitch, void* data_t,
                                   int64_t data_t_pitch, void* scale_t, int64_t scale_t_pitch,
                                   void* stream) {
  clear_error();
  QuantizeCall q{x, x_format, rows, cols, x_pitch, out_format, rule, square != 0, seed, offset};
  q.copy = {reinterpret_cast<uint64_t>(data), reinterpret_cast<uint64_t>(scale), data_pitch,
            scale_pitch, 0, 0};
  q.turned = {reinterpret_cast<uint64_t>(data_t), reinterpret_cast<uint64_t>(scale_t),
              data_t_pitch, scale_t_pitch, 0, 0};
  return quantize(q, static_cast<cudaStream_t>(stream));
}

extern "C" int srs_quantize_stack(const void* x, int x_format, int64_t matrices, int64_t rows,
                                  int64_t cols, int64_t x_pitch, int64_t x_stride, int out_format,
                                  int rule, int square, uint32_t seed, uint32_t offset,
                                  const srs_block_copy* copy, const srs_block_copy* copy_t,
                                  void* stream) {
  clear_error();
  QuantizeCall q{x, x_format, rows, cols, x_pitch, out_format, rule, square != 0, seed, offset};
  q.matrices = matrices;
  q.x_stride = x_stride;
  if (copy != nullptr) q.copy = *copy;
  if (copy_t != nullptr) q.turned = *copy_t;
  return quantize(q, static_cast<cudaStream_t>(stream));
}

extern "C" int64_t srs_group_columns(int64_t rows, int groups) {
  return rows <= 0 || groups <= 0 ? 0 : kBlock * most_group_tiles(rows, groups, kBlock);
}

extern "C" int64_t srs_group_scales(int64_t rows, int groups) {
  // every group with rows takes a multiple of 4
  if (rows <= 0 || groups <= 0) return 0;
  return (most_group_tiles(rows, groups, kBlock) + 3 * (groups < rows ? groups : rows) + 3) / 4 * 4;
}

extern "C" int srs_quantize_groups(const void* x, int x_format, int64_t rows, int64_t cols,
                                   int64_t x_pitch, const int32_t* ends, int groups,
                                   int out_format, int rule, uint32_t seed, uint32_t offset,
                                   const srs_block_copy* copy, const srs_block_copy* copy_t,
                                   void* stream) {
  clear_error();
  if (int rc = check_groups(ends, groups)) return rc;
  if (copy_t == nullptr || copy_t->data == 0)
    return fail(SRS_ERR_INVALID_ARGUMENT, "groups need the transposed copy");
  QuantizeCall q{x, x_format, rows, cols, x_pitch, out_format, rule, false, seed, offset};
  q.ends = ends;
  q.groups = groups;
  if (copy != nullptr) q.copy = *copy;
  q.turned = *copy_t;
  return quantize(q, static_cast<cudaStream_t>(stream));
}

extern "C" int srs_copy_rows(const void* src, int64_t src_pitch, int64_t rows, int64_t cols,
                             void* dst, int64_t dst_pitch, void* stream) {
  clear_error();
  if (rows < 0 || cols < 0 || src_pitch < 0)
    return fail(SRS_ERR_INVALID_ARGUMENT, "negative size or pitch");
  if (rows == 0 || cols == 0) return SRS_OK;
  if (src == nullptr || dst == nullptr)
    return fail(SRS_ERR_INVALID_ARGUMENT, "null input or output pointer");
  if (reinterpret_cast<uintptr_t>(dst) % 16 != 0 || dst_pitch % 16 != 0 || dst_pitch < cols)
    return fail(SRS_ERR_INVALID_ARGUMENT,
                "the copy needs a 16-byte aligned address and a row pitch that is a multiple of "
                "16 and at least the row length (%lld, %lld)",
                (long long)dst_pitch, (long long)cols);
  if (int rc = check_device()) return rc;
  const int64_t work = (rows * (dst_pitch / 16) + kThreads - 1) / kThreads;
  const int64_t most = 8ll * sm_count();
  copy_rows_kernel<<<(unsigned)(work < most ? work : most), kThreads, 0,
                     static_cast<cudaStream_t>(stream)>>>(
      static_cast<const uint8_t*>(src), src_pitch, rows, cols, static_cast<uint8_t*>(dst),
      dst_pitch);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? SRS_OK : cuda_fail(e, "srs_copy_rows launch");
}

extern "C" int srs_matmul_blocks(const srs_blocks* a, const srs_blocks* b, int64_t k, void* d,
                                 int d_format, void* stream) {
  clear_error();
  if (d_format < SRS_FMT_F32 || d_format > SRS_FMT_F16)
    return fail(SRS_ERR_INVALID_ARGUMENT, "unsupported result format %d", d_format);
  if (k < 0 || k > (1ll << 30))
    return fail(SRS_ERR_INVALID_ARGUMENT, "k must be in [0, 2^30], got %lld", (long long)k);
  if (int rc = check_operand("a", a, k)) return rc;
  if (int rc = check_operand("b", b, k)) return rc;
  if (a->rows == 0 || b->rows == 0) return SRS_OK;
  if (d == nullptr || reinterpret_cast<uintptr_t>(d) % fmt_bytes(d_format) != 0)
    return fail(SRS_ERR_INVALID_ARGUMENT, "null or misaligned result pointer");
  if (int rc = check_device()) return rc;
  if (int rc = check_products()) return rc;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (k == 0) {
    const cudaError_t e =
        cudaMemsetAsync(d, 0, (size_t)a->rows * b->rows * fmt_bytes(d_format), st);
    return e == cudaSuccess ? SRS_OK : cuda_fail(e, "srs_matmul_blocks");
  }
  // Few rows on one side: the other side's bytes bound the product.
  if (b->rows <= kThinRows && a->rows >= b->rows)
    return launch_thin(*a, *b, k, d, d_format, b->rows, 1, false, st);
  if (a->rows <= kThinRows) return launch_thin(*b, *a, k, d, d_format, 1, b->rows, false, st);
  return launch_block_product(*a, *b, k, d, d_format, st);
}

extern "C" int64_t srs_linear_workspace(int64_t tokens, int64_t k) {
  if (tokens <= 0 || k <= 0) return 0;
  const int64_t pitch = (k + 15) / 16 * 16;
  return tokens * (pitch + blocks_of(k));
}

extern "C" int srs_linear_blocks(const void* x, int x_format, int64_t tokens, int64_t k,
                                 int64_t x_pitch, int block_format, const srs_blocks* w, void* d,
                                 void* workspace, int64_t workspace_bytes, void* stream) {
  clear_error();
  if (int rc = check_operand("w", w, k)) return rc;
  if (tokens < 0 || k < 0)
    return fail(SRS_ERR_INVALID_ARGUMENT, "negative size (%lld, %lld)", (long long)tokens,
                (long long)k);
  if (tokens == 0 || w->rows == 0) return SRS_OK;
  if (workspace_bytes < srs_linear_workspace(tokens, k) ||
      (k > 0 && (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 16 != 0)))
    return fail(SRS_ERR_INVALID_ARGUMENT,
                "workspace of %lld bytes, %lld needed at a 16-byte aligned address",
                (long long)workspace_bytes, (long long)srs_linear_workspace(tokens, k));
  srs_blocks rows{};
  rows.data = reinterpret_cast<uint64_t>(workspace);
  rows.rows = tokens;
  rows.pitch = (k + 15) / 16 * 16;
  rows.scale = rows.data + (uint64_t)(tokens * rows.pitch);
  rows.scale_pitch = blocks_of(k);
  rows.format = block_format;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (k == 0) return srs_matmul_blocks(&rows, w, k, d, x_format, stream);
  QuantizeCall q{x,     x_format, tokens, k, x_pitch, block_format, SRS_RULE_NEAREST,
                 false, 0u,       0u};
  q.copy = {rows.data, rows.scale, rows.pitch, rows.scale_pitch, 0, 0};
  q.for_product = true;
  if (int rc = quantize(q, st)) return rc;
  // With few tokens the product starts beside the quantisation and streams the
  // weights, which that kernel does not write, before it needs the tokens.
  if (tokens <= kThinRows && w->rows >= tokens) {
    if (d == nullptr || reinterpret_cast<uintptr_t>(d) % fmt_bytes(x_format) != 0)
      return fail(SRS_ERR_INVALID_ARGUMENT, "null or misaligned result pointer");
    return launch_thin(*w, rows, k, d, x_format, 1, w->rows, true, st);
  }
  return srs_matmul_blocks(&rows, w, k, d, x_format, stream);
}
