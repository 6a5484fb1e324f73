// Low-rank adapters of many requests beside a projection in FP8 blocks:
//
//   h_t = s_a A_a x_t                 (rank numbers a token, "low")
//   d_t = W x_t + B_a h_t             a: the token's adapter
//
// and the adapters' gradients, sums over the tokens of one adapter:
//
//   dA_a = sum_t g_t x_t^T,  g_t = s_a B_a^T dy_t;      dB_a = sum_t dy_t h_t^T
//
// The backward pass is the same operator with the roles turned: g is the low part of dy with
// B^T for A, and dx_t = W^T dy_t + A_a^T g_t.
//
// Tokens are taken in the order of their adapters (srs_group_rows), gathered where they are
// read and scattered where results are written.  h and g are FP32; where a tensor core takes them
// they are split into a pair of 16-bit numbers, so that only the results are rounded.
#include <cooperative_groups.h>

#include "srs_common.cuh"
#include "srs_groups.cuh"
#include "srs_host.h"
#include "srs_launch.h"

namespace srs {
namespace {

namespace cg = cooperative_groups;

__device__ __forceinline__ int64_t token_at(const int32_t* order, int place, int tokens) {
  const int t = __ldg(order + place);
  return t >= 0 && t < tokens ? t : 0;  // an entry that names no token reads the first
}

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ uint32_t shared_at(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

template <bool TURN>
__device__ __forceinline__ void load_matrices(uint32_t at, uint32_t (&r)[4]) {
  if constexpr (TURN)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(at)
                 : "memory");
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(at)
                 : "memory");
}

// c += a b: 16 x 8 += (16 x 16) (16 x 8)
template <int F>
__device__ __forceinline__ void multiply(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  if constexpr (F == SRS_FMT_BF16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <int F>
__device__ __forceinline__ float decode16(uint32_t bits) {
  if constexpr (F == SRS_FMT_BF16) return __uint_as_float(bits << 16);
  return __half2float(__ushort_as_half((unsigned short)bits));
}

template <int F>
__device__ __forceinline__ uint32_t encode16(float x) {
  if constexpr (F == SRS_FMT_BF16) return __bfloat16_as_ushort(__float2bfloat16_rn(x));
  return __half_as_ushort(__float2half_rn(x));
}

// ------------------------------------------------------------------ low part --
//
// A CTA takes up to 128 tokens of one adapter (tiles counted from the adapter's first), up to
// 64 of the rank and a part of the sum; the parts of a cluster's CTAs are added through
// distributed shared memory in rank order.  x's bytes, read once, bound it: mma.sync is far
// faster than they arrive (4096 tokens, 4096 -> 64: 2 GFLOP).  Sums are FP32.
constexpr int kLowTokens = 128, kLowRank = 64, kLowStep = 64, kLowStages = 4;
constexpr int kLowWarps = kLowTokens / 16;
constexpr int kLowX = kLowTokens * kLowStep * 2, kLowW = kLowRank * kLowStep * 2;
constexpr int kLowSmem = kLowStages * (kLowX + kLowW);
static_assert(kLowTokens * (kLowRank + 1) * 4 <= kLowSmem, "the sums fit the stages");

struct LowArgs {
  const char* x;  // 16-bit, rows of x_pitch elements
  const char* w;  // KINNER: rank x k a matrix; else k x rank
  int64_t x_pitch, w_pitch, w_stride;  // elements
  int tokens, k, rank, adapters;
  const int32_t* order;
  const int32_t* ends;
  const float* scale;  // null: `factor` alone
  float factor;
  float* low;             // tokens (in order) x rank (null: not wanted)
  uint16_t* pairs;        // items for a large product (null: not wanted)
  int edge, pitch, rest_at;
  unsigned int* largest;  // of an adapter's |low|, as encodings (null: not wanted)
};

// 16-byte slot `slot` of a row of 128 bytes, turned so that 8 rows at one slot and 8 slots of a
// row both reach all banks.
__device__ __forceinline__ uint32_t turned_slot(int row, int slot) {
  return (uint32_t)(row * 128 + ((slot ^ (row & 7)) << 4));
}

template <int F, bool KINNER>
__global__ void __launch_bounds__(32 * kLowWarps, 2) low_kernel(const LowArgs a) {
  extern __shared__ __align__(128) uint8_t raw[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t splits, split;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(splits));
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(split));
  const GroupTile tile = find_group_tile(a.ends, a.adapters, a.tokens, kLowTokens,
                                         (int)(blockIdx.x / splits), lane);
  if (tile.group < 0) return;  // the whole cluster
  const int count = min(kLowTokens, tile.end - tile.row0);
  const int rank0 = (int)blockIdx.y * kLowRank, ranks = min(kLowRank, a.rank - rank0);
  const int steps = (a.k + kLowStep - 1) / kLowStep;
  const int first = (int)((int64_t)steps * split / splits);
  const int last = (int)((int64_t)steps * (split + 1) / splits);
  const uint32_t base = shared_at(raw);
  const auto x_at = [&](int s) { return base + (uint32_t)(s * (kLowX + kLowW)); };

  // this thread's rows of x: threadIdx.x / 8 + 32 i, slot threadIdx.x % 8
  const int slot = threadIdx.x & 7, row = threadIdx.x >> 3;
  const char* from[kLowTokens / 32];
#pragma unroll
  for (int i = 0; i < kLowTokens / 32; ++i) {
    const int r = row + 32 * i;
    from[i] = a.x + (r < count ? token_at(a.order, tile.row0 + r, a.tokens) : 0) * a.x_pitch * 2;
  }
  const char* const w = a.w + (int64_t)tile.group * a.w_stride * 2;
  const auto load = [&](int step, int s) {
    const int k = step * kLowStep + 8 * slot, bytes = min(max(a.k - k, 0) * 2, 16);
    const uint32_t to = x_at(s);
#pragma unroll
    for (int i = 0; i < kLowTokens / 32; ++i) {
      const int r = row + 32 * i;
      if (32 * i < count)  // rows that no warp multiplies stay as they are
        copy16(to + turned_slot(r, slot), bytes > 0 ? from[i] + 2 * k : a.x, r < count ? bytes : 0);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = row + 32 * i;
      if (KINNER) {
        const bool in = r < ranks && bytes > 0;
        if (32 * i < ((ranks + 15) & ~15))
          copy16(to + kLowX + turned_slot(r, slot),
                 in ? w + ((int64_t)(rank0 + r) * a.w_pitch + k) * 2 : w, in ? bytes : 0);
      } else {
        // rows are k, slots 8 of the rank
        const int kk = step * kLowStep + r, left = min(max(ranks - 8 * slot, 0) * 2, 16);
        const bool in = kk < a.k && left > 0;
        copy16(to + kLowX + turned_slot(r, slot),
               in ? w + ((int64_t)kk * a.w_pitch + rank0 + 8 * slot) * 2 : w, in ? left : 0);
      }
    }
  };

  float sum[kLowRank / 8][4];
#pragma unroll
  for (int i = 0; i < kLowRank / 8; ++i) {
#pragma unroll
    for (int j = 0; j < 4; ++j) sum[i][j] = 0.0f;
  }
  for (int i = 0; i < kLowStages - 1; ++i) {
    if (first + i < last) load(first + i, i);
    copies_done();
  }
  const bool busy = 16 * warp < count;
  for (int step = first; step < last; ++step) {
    const int s = (step - first) % kLowStages;
    copies_wait<kLowStages - 2>();
    __syncthreads();
    if (step + kLowStages - 1 < last)
      load(step + kLowStages - 1, (step - first + kLowStages - 1) % kLowStages);
    copies_done();
    if (!busy) continue;
    const uint32_t xs = x_at(s), ws = xs + kLowX;
#pragma unroll
    for (int kk = 0; kk < kLowStep / 16; ++kk) {
      uint32_t m[4];
      load_matrices<false>(xs + turned_slot(16 * warp + (lane & 15), 2 * kk + (lane >> 4)), m);
#pragma unroll
      for (int j = 0; j < kLowRank / 16; ++j) {
        if (16 * j >= ranks) break;
        uint32_t b[4];
        if (KINNER)  // ranks 16 j + (0..15) x k 16 kk ..
          load_matrices<false>(ws + turned_slot(16 * j + (lane & 7) + ((lane >> 4) << 3),
                                                2 * kk + ((lane >> 3) & 1)), b);
        else         // k 16 kk + (0..15) x ranks 16 j ..
          load_matrices<true>(ws + turned_slot(16 * kk + (lane & 15), 2 * j + (lane >> 4)), b);
        multiply<F>(sum[2 * j], m, b[0], b[1]);
        multiply<F>(sum[2 * j + 1], m, b[2], b[3]);
      }
    }
  }
  // sums to shared memory, [token][rank]
  copies_wait<0>();
  __syncthreads();
  float* const sums = reinterpret_cast<float*>(raw);
  constexpr int kPitch = kLowRank + 1;
  if (busy) {
#pragma unroll
    for (int j = 0; j < kLowRank / 8; ++j) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        sums[(16 * warp + (lane >> 2) + 8 * (i >> 1)) * kPitch + 8 * j + 2 * (lane & 3) + (i & 1)] =
            sum[j][i];
    }
  }
  if (splits > 1) cg::this_cluster().sync();
  else __syncthreads();
  const float factor = a.factor * (a.scale != nullptr ? __ldg(a.scale + tile.group) : 1.0f);
  float most = 0.0f;
  // token t of the tile by CTA t % splits
  const int whole = (ranks + 15) & ~15;
  for (int i = threadIdx.x; i < kLowTokens / (int)splits * kLowRank; i += 32 * kLowWarps) {
    const int t = i / kLowRank * (int)splits + (int)split, r = i % kLowRank;
    if (t >= count || r >= whole) continue;
    float v = 0.0f;
    if (r < ranks) {
      for (uint32_t p = 0; p < splits; ++p) {
        const float* const theirs = splits > 1 ? cg::this_cluster().map_shared_rank(sums, p) : sums;
        v += theirs[t * kPitch + r];
      }
      v *= factor;
      if (a.low != nullptr) a.low[(int64_t)(tile.row0 + t) * a.rank + rank0 + r] = v;
      most = fmaxf(most, isfinite(v) ? fabsf(v) : 0.0f);
    }
    if (a.pairs != nullptr) {
      const int place = tile.row0 + t;
      uint16_t* const to = a.pairs + ((int64_t)(place / a.edge + tile.rank) * a.edge +
                                      place % a.edge) * a.pitch + rank0 + r;
      const uint32_t high = encode16<F>(v);
      const float left = v - decode16<F>(high);
      to[0] = (uint16_t)high;
      to[a.rest_at] = (uint16_t)encode16<F>(isfinite(left) ? left : 0.0f);
    }
  }
  if (a.pairs != nullptr) {
    // zeros in the rows of the adapter's first and last item that are not its own
    const int words = whole / 2;
    const auto clear = [&](int item, int from, int to) {
      const int rows = to - from;
      for (int i = threadIdx.x + 32 * kLowWarps * (int)split; i < rows * words;
           i += 32 * kLowWarps * (int)splits) {
        uint16_t* const p = a.pairs + ((int64_t)item * a.edge + from + i / words) * a.pitch +
                            rank0 + 2 * (i % words);
        *reinterpret_cast<uint32_t*>(p) = 0u;
        *reinterpret_cast<uint32_t*>(p + a.rest_at) = 0u;
      }
    };
    if (tile.row0 == tile.start) clear(tile.start / a.edge + tile.rank, 0, tile.start % a.edge);
    const int last = tile.end - 1;
    if (last - tile.row0 < kLowTokens)
      clear(last / a.edge + tile.rank, last % a.edge + 1, a.edge);
  }
  if (a.largest != nullptr) {
    const unsigned int top = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(most));
    if (lane == 0 && top != 0u) atomicMax(a.largest + tile.group, top);  // the order is no matter
  }
  if (splits > 1) cg::this_cluster().sync();  // the others have read this CTA's sums
}

// -------------------------------------------------------------- few tokens --
//
// d_t = base_t + U_a low_t with the base in FP32: a CTA takes 256 columns of up to 64 tokens of
// one adapter, a thread a column, whose row of U it keeps in registers 8 of the rank at a time.
// U's bytes bound it.  The last tiles of the grid hold the tokens of no adapter.
constexpr int kExpandTokens = 64, kExpandThreads = 256;

struct ExpandArgs {
  const float* base;  // tokens x n
  const char* u;      // RINNER: n x rank a matrix; else rank x n
  int64_t u_pitch, u_stride;
  const float* low;
  int tokens, n, rank, adapters;
  const int32_t* order;
  const int32_t* ends;
  void* out;  // tokens x n
};

template <int F, bool RINNER>
__global__ void __launch_bounds__(kExpandThreads) expand_kernel(const ExpandArgs a) {
  extern __shared__ float lows[];  // [token][rank, whole 8s]
  __shared__ int32_t rows[kExpandTokens];
  const int lane = threadIdx.x & 31, ranks = (a.rank + 7) & ~7;
  GroupTile tile = find_group_tile(a.ends, a.adapters, a.tokens, kExpandTokens, (int)blockIdx.y,
                                   lane);
  if (tile.group < 0) {
    // tokens without an adapter, from the last of the grid's tiles backwards
    int carry = 0;
    for (int base = 0; base < a.adapters; base += 32) {
      int start, end;
      group_span(a.ends, a.adapters, a.tokens, base, lane, &carry, &start, &end);
    }
    const int64_t at = carry + (int64_t)kExpandTokens * (gridDim.y - 1 - blockIdx.y);
    if (at >= a.tokens) return;
    tile.row0 = (int)at;
    tile.end = a.tokens;
  }
  const int count = min(kExpandTokens, tile.end - tile.row0);
  if (threadIdx.x < count)
    rows[threadIdx.x] = (int32_t)token_at(a.order, tile.row0 + threadIdx.x, a.tokens);
  if (tile.group >= 0) {
    for (int i = threadIdx.x; i < count * ranks; i += kExpandThreads) {
      const int t = i / ranks, r = i % ranks;
      lows[i] = r < a.rank ? a.low[(int64_t)(tile.row0 + t) * a.rank + r] : 0.0f;
    }
  }
  __syncthreads();
  const int col = (int)blockIdx.x * kExpandThreads + threadIdx.x;
  if (col >= a.n) return;
  const char* const u = a.u + (int64_t)(tile.group < 0 ? 0 : tile.group) * a.u_stride * 2;
  for (int t0 = 0; t0 < count; t0 += 8) {
    float sum[8];
#pragma unroll
    for (int t = 0; t < 8; ++t)
      sum[t] = t0 + t < count ? a.base[(int64_t)rows[t0 + t] * a.n + col] : 0.0f;
    if (tile.group >= 0) {
      for (int r = 0; r < ranks; r += 8) {
        float v[8];
        if (RINNER) {
          const uint4 q = __ldg(reinterpret_cast<const uint4*>(u + ((int64_t)col * a.u_pitch + r) * 2));
          const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
          for (int i = 0; i < 8; ++i)
            v[i] = r + i < a.rank ? decode16<F>((w[i >> 1] >> (16 * (i & 1))) & 0xFFFFu) : 0.0f;
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            v[i] = r + i < a.rank
                       ? decode16<F>(__ldg(reinterpret_cast<const unsigned short*>(u) +
                                           (int64_t)(r + i) * a.u_pitch + col))
                       : 0.0f;
        }
#pragma unroll
        for (int t = 0; t < 8; ++t) {
          if (t0 + t >= count) break;
          const float4* const l = reinterpret_cast<const float4*>(lows + (t0 + t) * ranks + r);
          const float4 p = l[0], q = l[1];
          sum[t] = fmaf(v[0], p.x, sum[t]);
          sum[t] = fmaf(v[1], p.y, sum[t]);
          sum[t] = fmaf(v[2], p.z, sum[t]);
          sum[t] = fmaf(v[3], p.w, sum[t]);
          sum[t] = fmaf(v[4], q.x, sum[t]);
          sum[t] = fmaf(v[5], q.y, sum[t]);
          sum[t] = fmaf(v[6], q.z, sum[t]);
          sum[t] = fmaf(v[7], q.w, sum[t]);
        }
      }
    }
#pragma unroll
    for (int t = 0; t < 8; ++t)
      if (t0 + t < count)
        static_cast<uint16_t*>(a.out)[(int64_t)rows[t0 + t] * a.n + col] =
            (uint16_t)encode16<F>(sum[t]);
  }
}

// ---------------------------------------------------------------- gradients --
//
// out_a = sum over an adapter's tokens of z_t (cols) by low_t (rank).  A CTA takes 128 columns,
// up to 64 of the rank and a chunk of up to kSumTokens tokens of one adapter (counted from
// its first); adapters of several chunks leave FP32 parts, which another kernel adds in
// order.  z's bytes, read once for every 64 of the rank, bound it.  `low` enters as a pair of
// 16-bit numbers (high and what it leaves); in FP16 both are scaled by a power of two that
// brings the adapter's largest to 2^11 .. 2^12, so that small gradients keep their digits.
constexpr int kSumCols = 128, kSumRank = 64, kSumStep = 64, kSumStages = 3, kSumTokens = 512;
constexpr int kSumWarps = kSumCols / 16;
constexpr int kSumZ = kSumStep * kSumCols * 2, kSumLow = kSumStep * kSumRank * 2;
constexpr int kSumSmem = kSumStages * kSumZ + 2 * 2 * kSumLow;

struct SumArgs {
  const char* z;
  int64_t z_pitch;
  const float* low;
  const unsigned int* largest;
  int tokens, cols, rank, adapters;
  const int32_t* order;
  const int32_t* ends;
  void* out;
  float* parts;  // [chunk][rank][cols]
  int turned;    // out: cols x rank instead of rank x cols
};

__device__ __forceinline__ float pair_scale(const unsigned int* largest, int group) {
  if (largest == nullptr) return 1.0f;
  const unsigned int top = __ldg(largest + group);
  // 2^11 <= top * 2^k < 2^12; an encoding of zero or below the normal range: the largest factor
  const int k = 11 - ((int)(top >> 23) - 127);
  return __uint_as_float((uint32_t)(min(max(k, -126), 126) + 127) << 23);
}

__device__ __forceinline__ uint32_t wide_slot(int row, int slot) {  // rows of 256 bytes
  return (uint32_t)(row * 256 + ((slot ^ (row & 7)) << 4));
}

template <int F>
__global__ void __launch_bounds__(32 * kSumWarps, 2) sum_kernel(const SumArgs a) {
  extern __shared__ __align__(128) uint8_t raw[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const GroupTile tile =
      find_group_tile(a.ends, a.adapters, a.tokens, kSumTokens, (int)blockIdx.y, lane);
  if (tile.group < 0) return;
  const int count = min(kSumTokens, tile.end - tile.row0);
  const int rank0 = (int)blockIdx.z * kSumRank, ranks = min(kSumRank, a.rank - rank0);
  const int col0 = (int)blockIdx.x * kSumCols;
  const float scale = pair_scale(a.largest, tile.group);
  const uint32_t z0 = shared_at(raw), low0 = z0 + kSumStages * kSumZ;

  const int slot = threadIdx.x & 15, row = threadIdx.x >> 4;  // 16 rows at a time
  const int col = col0 + 8 * slot, bytes = min(max(a.cols - col, 0) * 2, 16);
  const auto load = [&](int step, int s) {
#pragma unroll
    for (int i = 0; i < kSumStep / 16; ++i) {
      const int r = row + 16 * i, t = step * kSumStep + r;
      const bool in = t < count && bytes > 0;
      const char* from =
          in ? a.z + (token_at(a.order, tile.row0 + t, a.tokens) * a.z_pitch + col) * 2 : a.z;
      copy16(z0 + s * kSumZ + wide_slot(r, slot), from, in ? bytes : 0);
    }
  };
  // low: thread t has 16 of the rank of token t / 4
  const int low_row = threadIdx.x >> 2, low_col = (threadIdx.x & 3) * 16;
  float held[16];
  const auto fetch = [&](int step) {
    const int t = step * kSumStep + low_row;
    const float* from = a.low + (int64_t)(tile.row0 + t) * a.rank + rank0 + low_col;
#pragma unroll
    for (int i = 0; i < 16; ++i)
      held[i] = t < count && low_col + i < ranks ? __ldg(from + i) * scale : 0.0f;
  };
  const auto split = [&](int b) {
    const uint32_t to = low0 + b * 2 * kSumLow;
    if (low_col >= ((ranks + 15) & ~15)) return;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t high[4], rest[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = held[8 * h + 2 * i], y = held[8 * h + 2 * i + 1];
        const uint32_t hx = encode16<F>(x), hy = encode16<F>(y);
        high[i] = hx | hy << 16;
        rest[i] = encode16<F>(x - decode16<F>(hx)) | encode16<F>(y - decode16<F>(hy)) << 16;
      }
      const uint32_t at = to + turned_slot(low_row, (low_col >> 3) + h);
      asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(high[0]), "r"(high[1]),
                   "r"(high[2]), "r"(high[3])
                   : "memory");
      asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at + kSumLow), "r"(rest[0]),
                   "r"(rest[1]), "r"(rest[2]), "r"(rest[3])
                   : "memory");
    }
  };

  float sum[kSumRank / 8][4];
#pragma unroll
  for (int i = 0; i < kSumRank / 8; ++i) {
#pragma unroll
    for (int j = 0; j < 4; ++j) sum[i][j] = 0.0f;
  }
  const int steps = (count + kSumStep - 1) / kSumStep;
  for (int i = 0; i < kSumStages - 1; ++i) {
    if (i < steps) load(i, i);
    copies_done();
  }
  fetch(0);
  for (int step = 0; step < steps; ++step) {
    split(step & 1);
    copies_wait<kSumStages - 2>();
    __syncthreads();
    if (step + kSumStages - 1 < steps) load(step + kSumStages - 1, (step + kSumStages - 1) % kSumStages);
    copies_done();
    if (step + 1 < steps) fetch(step + 1);
    const uint32_t zs = z0 + step % kSumStages * kSumZ, ls = low0 + (step & 1) * 2 * kSumLow;
#pragma unroll
    for (int kk = 0; kk < kSumStep / 16; ++kk) {
      // columns 16 warp .. by tokens 16 kk ..: matrices of 8 tokens x 8 columns, turned
      uint32_t m[4];
      load_matrices<true>(zs + wide_slot(16 * kk + (lane & 7) + ((lane >> 4) << 3),
                                         2 * warp + ((lane >> 3) & 1)), m);
#pragma unroll
      for (int j = 0; j < kSumRank / 16; ++j) {
        if (16 * j >= ranks) break;
        uint32_t b[4];
        const uint32_t at = ls + turned_slot(16 * kk + (lane & 15), 2 * j + (lane >> 4));
        load_matrices<true>(at, b);
        multiply<F>(sum[2 * j], m, b[0], b[1]);
        multiply<F>(sum[2 * j + 1], m, b[2], b[3]);
        load_matrices<true>(at + kSumLow, b);
        multiply<F>(sum[2 * j], m, b[0], b[1]);
        multiply<F>(sum[2 * j + 1], m, b[2], b[3]);
      }
    }
  }
  copies_wait<0>();
  const float back = 1.0f / scale;  // a power of two: exact
#pragma unroll
  for (int j = 0; j < kSumRank / 8; ++j) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = col0 + 16 * warp + (lane >> 2) + 8 * (i >> 1);
      const int r = 8 * j + 2 * (lane & 3) + (i & 1);
      if (c >= a.cols || r >= ranks) continue;
      a.parts[((int64_t)blockIdx.y * a.rank + rank0 + r) * a.cols + c] = sum[j][i] * back;
    }
  }
}

// out_a = the sum of its chunks' parts, in order; zeros without tokens.
template <int F>
__global__ void __launch_bounds__(256) join_kernel(const SumArgs a) {
  const int lane = threadIdx.x & 31, group = (int)blockIdx.y;
  int carry = 0, chunks_before = 0, first = 0, chunks = 0;
  for (int base = 0; base <= group; base += 32) {
    int start, end;
    group_span(a.ends, a.adapters, a.tokens, base, lane, &carry, &start, &end);
    const int n = (end - start + kSumTokens - 1) / kSumTokens;
    const int upto = chunks_before + warp_scan_sum(n, lane);
    if (group - base < 32) {
      first = __shfl_sync(0xFFFFFFFFu, upto - n, group - base);
      chunks = __shfl_sync(0xFFFFFFFFu, n, group - base);
    }
    chunks_before = __shfl_sync(0xFFFFFFFFu, upto, 31);
  }
  const int64_t each = (int64_t)a.rank * a.cols;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < each; i += (int64_t)gridDim.x * 256) {
    // i runs over the result's order
    const int64_t at = a.turned ? i % a.rank * a.cols + i / a.rank : i;
    float v = 0.0f;
    for (int c = 0; c < chunks; ++c) v += a.parts[(first + c) * each + at];
    static_cast<uint16_t*>(a.out)[group * each + i] = (uint16_t)encode16<F>(v);
  }
}

// --------------------------------------------------------------------- host --

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
int64_t whole(int64_t bytes) { return ceil_div(bytes, 256) * 256; }

template <int F, bool KINNER>
int launch_low(const LowArgs& args, cudaStream_t stream) {
  const auto kernel = &low_kernel<F, KINNER>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kLowSmem);
  if (e != cudaSuccess) return cuda_fail(e, "low part");
  const int64_t busy = args.adapters < args.tokens ? args.adapters : args.tokens;
  const int64_t tiles = most_group_tiles(args.tokens, args.adapters, kLowTokens);
  const int64_t blocks = ceil_div(args.rank, kLowRank), steps = ceil_div(args.k, kLowStep);
  // Parts of the sum while the tiles that are likely leave SMs idle, at least 4 steps each.
  const int64_t likely = (args.tokens / kLowTokens + (busy + 1) / 2) * blocks;
  int splits = 1;
  while (splits < 8 && likely * splits < 2 * sm_count() && steps >= 8 * splits) splits *= 2;
  cudaLaunchConfig_t config{};
  cudaLaunchAttribute cluster{};
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = (unsigned)splits;
  cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
  config.gridDim = dim3((unsigned)(tiles * splits), (unsigned)blocks);
  config.blockDim = dim3(32 * kLowWarps);
  config.dynamicSmemBytes = kLowSmem;
  config.stream = stream;
  config.attrs = &cluster;
  config.numAttrs = 1;
  e = cudaLaunchKernelEx(&config, kernel, args);
  return e == cudaSuccess ? SRS_OK : cuda_fail(e, "low part launch");
}

template <int F, bool RINNER>
int launch_expand(const ExpandArgs& args, cudaStream_t stream) {
  const auto kernel = &expand_kernel<F, RINNER>;
  const int bytes = kExpandTokens * (int)ceil_div(args.rank, 8) * 8 * 4;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       kExpandTokens * SRS_ADAPTER_MAX_RANK * 4);
  if (e != cudaSuccess) return cuda_fail(e, "expansion");
  // one more tile than adapters' tokens can take: tokens of none in a last, partial one
  const int64_t tiles = most_group_tiles(args.tokens, args.adapters, kExpandTokens) + 1;
  const dim3 grid((unsigned)ceil_div(args.n, kExpandThreads), (unsigned)tiles);
  kernel<<<grid, kExpandThreads, bytes, stream>>>(args);
  e = cudaGetLastError();
  return e == cudaSuccess ? SRS_OK : cuda_fail(e, "expansion launch");
}

int check_adapters(const srs_adapters* a, int64_t tokens, int64_t k, int64_t n, bool turned) {
  if (a == nullptr) return fail(SRS_ERR_INVALID_ARGUMENT, "null adapters");
  if (int rc = check_groups(reinterpret_cast<const int32_t*>(a->ends), a->count)) return rc;
  if (a->format != SRS_FMT_BF16 && a->format != SRS_FMT_F16)
    return fail(SRS_ERR_INVALID_ARGUMENT, "adapters are BF16 or FP16, got format %d", a->format);
  if (a->rank < 1 || a->rank > SRS_ADAPTER_MAX_RANK)
    return fail(SRS_ERR_INVALID_ARGUMENT, "the rank must be in [1, %d], got %d",
                SRS_ADAPTER_MAX_RANK, a->rank);
  if (tokens < 0 || tokens > (1ll << 22) || k < 0 || n < 0 || k > (1ll << 30) || n > (1ll << 30))
    return fail(SRS_ERR_INVALID_ARGUMENT, "sizes out of range (%lld tokens, %lld -> %lld)",
                (long long)tokens, (long long)k, (long long)n);
  if (tokens == 0) return SRS_OK;
  if (a->order == 0 || a->order % 4 != 0)
    return fail(SRS_ERR_INVALID_ARGUMENT, "null or misaligned order");
  const int64_t in = turned ? n : k, out = turned ? k : n;  // of the adapters
  const auto bad = [](uint64_t at, int64_t pitch, int64_t stride, int64_t least) {
    return at == 0 || at % 16 != 0 || pitch % 8 != 0 || stride % 8 != 0 || pitch < least;
  };
  if ((in > 0 && bad(a->down, a->down_pitch, a->down_stride, in)) ||
      (out > 0 && bad(a->up, a->up_pitch, a->up_stride, a->rank)))
    return fail(SRS_ERR_INVALID_ARGUMENT,
                "adapter matrices need 16-byte aligned addresses, pitches and strides");
  return SRS_OK;
}

}  // namespace
}  // namespace srs

using namespace srs;

// Few tokens: the projection's thin form with an FP32 result and the expansion; else the adapters
// enter the large product.
static bool few(int64_t tokens) { return tokens <= kThinRows; }

// Parts of a call's workspace, each on a 256-byte boundary.
struct AdapterSpace {
  int64_t rows, low, base, total;  // rows: quantised tokens; low: FP32 or pairs; base: FP32
};

static AdapterSpace adapter_space(int64_t tokens, int64_t k, int64_t n, int adapters, int rank) {
  AdapterSpace s{};
  int64_t at = whole(srs_linear_workspace(tokens, k));
  s.low = at;
  if (few(tokens)) {
    at += whole(tokens * rank * 4);
    s.base = at;
    at += whole(tokens * n * 4);
  } else if (n > 0) {
    const int64_t edge = adapter_edge(tokens, n, k);
    at += whole(pair_items(tokens, adapters, edge) * edge * pair_shape(rank).pitch * 2);
  }
  s.total = at;
  return s;
}

extern "C" int64_t srs_adapter_workspace(int64_t tokens, int64_t k, int64_t n, int adapters,
                                         int rank) {
  if (tokens <= 0 || k < 0 || n < 0 || adapters < 1 || rank < 1) return 0;
  return adapter_space(tokens, k, n, adapters, rank).total;
}

extern "C" int srs_adapter_linear(const void* x, int64_t tokens, int64_t k, int64_t x_pitch,
                                  int block_format, int rule, uint32_t seed, const srs_blocks* w,
                                  const srs_adapters* a, int turned, void* d, float* low,
                                  uint32_t* largest, void* workspace, int64_t workspace_bytes,
                                  void* stream) {
  clear_error();
  const int64_t n = w == nullptr || d == nullptr ? 0 : w->rows;
  if (d != nullptr)
    if (int rc = check_operand("w", w, k)) return rc;
  if (int rc = check_adapters(a, tokens, k, n, turned != 0)) return rc;
  if (tokens == 0 || (n == 0 && low == nullptr)) return SRS_OK;
  if (k > 0 && (x == nullptr || reinterpret_cast<uintptr_t>(x) % 16 != 0 || x_pitch % 8 != 0 ||
                x_pitch < k))
    return fail(SRS_ERR_INVALID_ARGUMENT, "x needs a 16-byte aligned address and row pitch");
  if (n > 0 && reinterpret_cast<uintptr_t>(d) % 2 != 0)
    return fail(SRS_ERR_INVALID_ARGUMENT, "misaligned result pointer");
  const AdapterSpace space = adapter_space(tokens, k, n, a->count, a->rank);
  if (workspace_bytes < space.total ||
      (space.total > 0 &&
       (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 256 != 0)))
    return fail(SRS_ERR_INVALID_ARGUMENT,
                "workspace of %lld bytes, %lld needed at a 256-byte aligned address",
                (long long)workspace_bytes, (long long)space.total);
  if (int rc = check_device()) return rc;
  if (int rc = check_products()) return rc;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  char* const at = static_cast<char*>(workspace);
  const bool bf16 = a->format == SRS_FMT_BF16, thin = few(tokens);

  cudaError_t e = cudaSuccess;
  if (largest != nullptr) e = cudaMemsetAsync(largest, 0, (size_t)a->count * 4, st);
  // without a sum there is neither a projection nor a low part
  if (e == cudaSuccess && n > 0 && k == 0) e = cudaMemsetAsync(d, 0, (size_t)(tokens * n * 2), st);
  if (e != cudaSuccess) return cuda_fail(e, "srs_adapter_linear");
  const int edge = thin || n == 0 ? 0 : adapter_edge(tokens, n, k);
  const PairShape pairs = pair_shape(a->rank);
  LowArgs l{};
  l.x = static_cast<const char*>(x);
  l.w = reinterpret_cast<const char*>(turned ? a->up : a->down);
  l.x_pitch = x_pitch;
  l.w_pitch = turned ? a->up_pitch : a->down_pitch;
  l.w_stride = turned ? a->up_stride : a->down_stride;
  l.tokens = (int)tokens;
  l.k = (int)k;
  l.rank = a->rank;
  l.adapters = a->count;
  l.order = reinterpret_cast<const int32_t*>(a->order);
  l.ends = reinterpret_cast<const int32_t*>(a->ends);
  l.scale = reinterpret_cast<const float*>(a->scale);
  l.factor = a->factor;
  l.low = low != nullptr ? low : thin ? reinterpret_cast<float*>(at + space.low) : nullptr;
  l.largest = largest;
  if (edge != 0) {
    l.pairs = reinterpret_cast<uint16_t*>(at + space.low);
    l.edge = edge;
    l.pitch = pairs.pitch;
    l.rest_at = pairs.rest_at;
  }
  if (int rc = turned ? (bf16 ? launch_low<SRS_FMT_BF16, false>(l, st)
                              : launch_low<SRS_FMT_F16, false>(l, st))
                      : (bf16 ? launch_low<SRS_FMT_BF16, true>(l, st)
                              : launch_low<SRS_FMT_F16, true>(l, st)))
    return rc;
  if (n == 0 || k == 0) return SRS_OK;

  srs_blocks rows{};
  rows.data = reinterpret_cast<uint64_t>(workspace);
  rows.rows = tokens;
  rows.pitch = ceil_div(k, 16) * 16;
  rows.scale = rows.data + (uint64_t)(tokens * rows.pitch);
  rows.scale_pitch = ceil_div(k, 128);
  rows.format = block_format;
  QuantizeCall q{x, a->format, tokens, k, x_pitch, block_format, rule, false, seed, 0u};
  q.copy = {rows.data, rows.scale, rows.pitch, rows.scale_pitch, 0, 0};
  q.order = thin ? nullptr : l.order;
  if (int rc = quantize(q, st)) return rc;
  const void* const up = reinterpret_cast<const void*>(turned ? a->down : a->up);
  const int64_t up_pitch = turned ? a->down_pitch : a->up_pitch;
  const int64_t up_stride = turned ? a->down_stride : a->up_stride;
  if (!thin) {
    const AdapterCall call{l.pairs,  up,       up_pitch,  up_stride, turned != 0,
                           a->count, a->rank,  a->format, l.order,   l.ends};
    return launch_adapter_product(rows, *w, k, call, edge, d, st);
  }
  float* const base = reinterpret_cast<float*>(at + space.base);
  if (int rc = srs_matmul_blocks(&rows, w, k, base, SRS_FMT_F32, stream)) return rc;
  ExpandArgs x_args{};
  x_args.base = base;
  x_args.u = static_cast<const char*>(up);
  x_args.u_pitch = up_pitch;
  x_args.u_stride = up_stride;
  x_args.low = l.low;
  x_args.tokens = (int)tokens;
  x_args.n = (int)n;
  x_args.rank = a->rank;
  x_args.adapters = a->count;
  x_args.order = l.order;
  x_args.ends = l.ends;
  x_args.out = d;
  return turned ? (bf16 ? launch_expand<SRS_FMT_BF16, false>(x_args, st)
                        : launch_expand<SRS_FMT_F16, false>(x_args, st))
                : (bf16 ? launch_expand<SRS_FMT_BF16, true>(x_args, st)
                        : launch_expand<SRS_FMT_F16, true>(x_args, st));
}

extern "C" int64_t srs_adapter_gradient_workspace(int64_t tokens, int64_t cols, int adapters,
                                                  int rank) {
  if (tokens <= 0 || cols <= 0 || adapters < 1 || rank < 1) return 0;
  return most_group_tiles(tokens, adapters, kSumTokens) * rank * cols * 4;
}

extern "C" int srs_adapter_gradient(const void* z, int format, int64_t tokens, int64_t cols,
                                    int64_t z_pitch, const float* low, const uint32_t* largest,
                                    int adapters, int rank, const int32_t* order,
                                    const int32_t* ends, int turned, void* out, void* workspace,
                                    int64_t workspace_bytes, void* stream) {
  clear_error();
  if (int rc = check_groups(ends, adapters)) return rc;
  if (format != SRS_FMT_BF16 && format != SRS_FMT_F16)
    return fail(SRS_ERR_INVALID_ARGUMENT, "adapters are BF16 or FP16, got format %d", format);
  if (rank < 1 || rank > SRS_ADAPTER_MAX_RANK || tokens < 0 || tokens > (1ll << 22) || cols < 0 ||
      cols > (1ll << 30))
    return fail(SRS_ERR_INVALID_ARGUMENT, "sizes out of range (%lld tokens, %lld columns, rank %d)",
                (long long)tokens, (long long)cols, rank);
  if (cols == 0) return SRS_OK;
  if (out == nullptr || reinterpret_cast<uintptr_t>(out) % 2 != 0)
    return fail(SRS_ERR_INVALID_ARGUMENT, "null or misaligned result pointer");
  if (int rc = check_device()) return rc;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (tokens == 0) {
    const cudaError_t e = cudaMemsetAsync(out, 0, (size_t)(2 * cols * rank * adapters), st);
    return e == cudaSuccess ? SRS_OK : cuda_fail(e, "srs_adapter_gradient");
  }
  if (z == nullptr || low == nullptr || order == nullptr || z_pitch < cols || z_pitch % 8 != 0 ||
      reinterpret_cast<uintptr_t>(z) % 16 != 0)
    return fail(SRS_ERR_INVALID_ARGUMENT, "z needs a 16-byte aligned address and row pitch");
  if (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 16 != 0 ||
      workspace_bytes < srs_adapter_gradient_workspace(tokens, cols, adapters, rank))
    return fail(SRS_ERR_INVALID_ARGUMENT, "workspace of %lld bytes, %lld needed",
                (long long)workspace_bytes,
                (long long)srs_adapter_gradient_workspace(tokens, cols, adapters, rank));
  SumArgs a{};
  a.z = static_cast<const char*>(z);
  a.z_pitch = z_pitch;
  a.low = low;
  a.largest = format == SRS_FMT_F16 ? largest : nullptr;
  a.tokens = (int)tokens;
  a.cols = (int)cols;
  a.rank = rank;
  a.adapters = adapters;
  a.order = order;
  a.ends = ends;
  a.out = out;
  a.parts = static_cast<float*>(workspace);
  a.turned = turned != 0;
  const auto kernel = format == SRS_FMT_BF16 ? &sum_kernel<SRS_FMT_BF16> : &sum_kernel<SRS_FMT_F16>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSumSmem);
  if (e != cudaSuccess) return cuda_fail(e, "adapter gradient");
  const dim3 grid((unsigned)ceil_div(cols, kSumCols),
                  (unsigned)most_group_tiles(tokens, adapters, kSumTokens),
                  (unsigned)ceil_div(rank, kSumRank));
  kernel<<<grid, 32 * kSumWarps, kSumSmem, st>>>(a);
  e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "adapter gradient launch");
  const int64_t blocks = ceil_div((int64_t)rank * cols, 1024);
  const dim3 joins((unsigned)(blocks < 1024 ? blocks : 1024), (unsigned)adapters);
  if (format == SRS_FMT_BF16) join_kernel<SRS_FMT_BF16><<<joins, 256, 0, st>>>(a);
  else join_kernel<SRS_FMT_F16><<<joins, 256, 0, st>>>(a);
  e = cudaGetLastError();
  return e == cudaSuccess ? SRS_OK : cuda_fail(e, "adapter gradient launch");
}
