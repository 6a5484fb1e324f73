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
  asm volatile("cp.async.cg.shared.global.L2::256B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes)
               : "memory");
}
// Rows of SLOTS (2 or 4) 16-byte slots, turned as rows of 8 are.
template <int SLOTS>
__device__ __forceinline__ uint32_t narrow_slot(int row, int slot) {
  return (uint32_t)(row * 16 * SLOTS + ((slot ^ ((row / (8 / SLOTS)) & (SLOTS - 1))) << 4));
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
// A CTA takes up to TOKENS tokens of one adapter (tiles counted from the adapter's first), up to
// 16 RT of the rank and a part of the sum; the parts of a cluster's CTAs are added through
// distributed shared memory in rank order.  x's bytes, read once, bound it: mma.sync is far
// faster than they arrive (4096 tokens, 4096 -> 64: 2 GFLOP).  Sums are FP32.
//
// TOKENS = 128: 8 warps of 16 tokens each.  TOKENS = 16, for calls of few tokens where most
// adapters have one or two: 4 warps that share a stage's four steps of 16 of k.
constexpr int kLowStep = 64;  // of k a stage: 128 bytes of a row

template <int TOKENS, int RT>
struct LowShape {
  static constexpr int kWarps = TOKENS == 16 ? 4 : TOKENS / 16;
  static constexpr int kThreads = 32 * kWarps;
  static constexpr bool kShared = TOKENS == 16;  // warps share the steps of a stage
  static constexpr int kRank = 16 * RT;
  static constexpr int kX = TOKENS * kLowStep * 2, kW = kRank * kLowStep * 2;
  // bytes on their way: 6 stages for ranks up to 16; two CTAs an SM fit with all of these
  static constexpr int kStages = TOKENS == 16 ? 8 : RT == 1 ? 6 : RT == 2 ? 5 : 4;
  static constexpr int kPitch = kRank + 1;
  static constexpr int kSums = (kShared ? kWarps : 1) * TOKENS * kPitch * 4;
  static constexpr int kStageBytes = kStages * (kX + kW);
  static constexpr int kSmem = kStageBytes > kSums ? kStageBytes : kSums;
};

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
  bool spread;            // items of a thin product: rows are the batch's
  unsigned int* largest;  // of an adapter's |low|, as encodings (null: not wanted)
};

// 16-byte slot `slot` of a row of 128 bytes, turned so that 8 rows at one slot and 8 slots of a
// row both reach all banks.
__device__ __forceinline__ uint32_t turned_slot(int row, int slot) {
  return (uint32_t)(row * 128 + ((slot ^ (row & 7)) << 4));
}

template <int F, bool KINNER, int TOKENS, int RT>
__global__ void __launch_bounds__(LowShape<TOKENS, RT>::kThreads, TOKENS == 16 ? 4 : 2)
low_kernel(const LowArgs a) {
  using S = LowShape<TOKENS, RT>;
  // The quantisation behind this kernel reads nothing of it and waits for it at its end.
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  extern __shared__ __align__(128) uint8_t raw[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t splits, split;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(splits));
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(split));
  const GroupTile tile = find_group_tile(a.ends, a.adapters, a.tokens, TOKENS,
                                         (int)(blockIdx.x / splits), lane);
  if (tile.group < 0) return;  // the whole cluster
  const int count = min(TOKENS, tile.end - tile.row0);
  const int rank0 = (int)blockIdx.y * S::kRank, ranks = min(S::kRank, a.rank - rank0);
  const int steps = (a.k + kLowStep - 1) / kLowStep;
  const int first = (int)((int64_t)steps * split / splits);
  const int last = (int)((int64_t)steps * (split + 1) / splits);
  const uint32_t base = shared_at(raw);
  const auto x_at = [&](int s) { return base + (uint32_t)(s * (S::kX + S::kW)); };

  // this thread's rows of x: threadIdx.x / 8 + kRows i, slot threadIdx.x % 8
  constexpr int kRows = S::kThreads / 8, kEach = TOKENS / kRows, kOfW = (S::kRank + kRows - 1) / kRows;
  const int slot = threadIdx.x & 7, row = threadIdx.x >> 3;
  const char* from[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int r = row + kRows * i;
    from[i] = a.x + (r < count ? token_at(a.order, tile.row0 + r, a.tokens) : 0) * a.x_pitch * 2;
  }
  const char* const w = a.w + (int64_t)tile.group * a.w_stride * 2;
  const auto load = [&](int step, int s) {
    const int k = step * kLowStep + 8 * slot, bytes = min(max(a.k - k, 0) * 2, 16);
    const uint32_t to = x_at(s);
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int r = row + kRows * i;
      if (kRows * i < count)  // rows that no warp multiplies stay as they are
        copy16(to + turned_slot(r, slot), bytes > 0 ? from[i] + 2 * k : a.x, r < count ? bytes : 0);
    }
    if (KINNER) {
#pragma unroll
      for (int i = 0; i < kOfW; ++i) {
        const int r = row + kRows * i;
        const bool in = r < ranks && bytes > 0;
        if (r < S::kRank)
          copy16(to + S::kX + turned_slot(r, slot),
                 in ? w + ((int64_t)(rank0 + r) * a.w_pitch + k) * 2 : w, in ? bytes : 0);
      }
    } else {
      // 64 rows of k, 2 RT slots of 8 of the rank each (the others are not read)
#pragma unroll
      for (int i = threadIdx.x; i < kLowStep * 2 * RT; i += S::kThreads) {
        const int r = i / (2 * RT), c = i % (2 * RT), kk = step * kLowStep + r;
        const int left = min(max(ranks - 8 * c, 0) * 2, 16);
        const bool in = kk < a.k && left > 0;
        copy16(to + S::kX + (RT == 4 ? turned_slot(r, c) : narrow_slot<2 * RT>(r, c)),
               in ? w + ((int64_t)kk * a.w_pitch + rank0 + 8 * c) * 2 : w, in ? left : 0);
      }
    }
  };

  float sum[2 * RT][4];
#pragma unroll
  for (int i = 0; i < 2 * RT; ++i) {
#pragma unroll
    for (int j = 0; j < 4; ++j) sum[i][j] = 0.0f;
  }
  for (int i = 0; i < S::kStages - 1; ++i) {
    if (first + i < last) load(first + i, i);
    copies_done();
  }
  const int my_rows = S::kShared ? 0 : 16 * warp;
  const bool busy = my_rows < count;
  int s = 0;
  for (int step = first; step < last; ++step) {
    copies_wait<S::kStages - 2>();
    __syncthreads();
    if (step + S::kStages - 1 < last) load(step + S::kStages - 1, s == 0 ? S::kStages - 1 : s - 1);
    copies_done();
    const uint32_t xs = x_at(s), ws = xs + S::kX;
    if (++s == S::kStages) s = 0;
    if (!busy) continue;
#pragma unroll
    for (int q = 0; q < (S::kShared ? 1 : kLowStep / 16); ++q) {
      const int kk = S::kShared ? warp : q;
      uint32_t m[4];
      load_matrices<false>(xs + turned_slot(my_rows + (lane & 15), 2 * kk + (lane >> 4)), m);
#pragma unroll
      for (int j = 0; j < RT; ++j) {
        uint32_t b[4];
        if (KINNER) {  // ranks 16 j + (0..15) x k 16 kk ..
          load_matrices<false>(ws + turned_slot(16 * j + (lane & 7) + ((lane >> 4) << 3),
                                                2 * kk + ((lane >> 3) & 1)), b);
        } else {       // k 16 kk + (0..15) x ranks 16 j ..
          const int r = 16 * kk + (lane & 15), c = 2 * j + (lane >> 4);
          load_matrices<true>(ws + (RT == 4 ? turned_slot(r, c) : narrow_slot<2 * RT>(r, c)), b);
        }
        multiply<F>(sum[2 * j], m, b[0], b[1]);
        multiply<F>(sum[2 * j + 1], m, b[2], b[3]);
      }
    }
  }
  // sums to shared memory, [token][rank] (of every warp, where they share the steps)
  copies_wait<0>();
  __syncthreads();
  float* const sums = reinterpret_cast<float*>(raw);
  if (busy) {
    float* const mine = sums + (S::kShared ? warp * TOKENS * S::kPitch : 0);
#pragma unroll
    for (int j = 0; j < 2 * RT; ++j) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        mine[(my_rows + (lane >> 2) + 8 * (i >> 1)) * S::kPitch + 8 * j + 2 * (lane & 3) + (i & 1)] =
            sum[j][i];
    }
  }
  const float factor = a.factor * (a.scale != nullptr ? __ldg(a.scale + tile.group) : 1.0f);
  if (splits > 1) cg::this_cluster().sync();
  else __syncthreads();
  float most = 0.0f;
  // token t of the tile by CTA t % splits
  const int whole = (ranks + 15) & ~15;
  for (int i = threadIdx.x; i < (TOKENS + (int)splits - 1) / (int)splits * S::kRank;
       i += S::kThreads) {
    const int t = i / S::kRank * (int)splits + (int)split, r = i % S::kRank;
    if (t >= count || r >= whole) continue;
    float v = 0.0f;
    if (r < ranks) {
      for (uint32_t p = 0; p < splits; ++p) {
        const float* const theirs =
            (splits > 1 ? cg::this_cluster().map_shared_rank(sums, p) : sums) + t * S::kPitch + r;
#pragma unroll
        for (int q = 0; q < (S::kShared ? S::kWarps : 1); ++q) v += theirs[q * TOKENS * S::kPitch];
      }
      v *= factor;
      if (a.low != nullptr) a.low[(int64_t)(tile.row0 + t) * a.rank + rank0 + r] = v;
      most = fmaxf(most, isfinite(v) ? fabsf(v) : 0.0f);
    }
    if (a.pairs != nullptr) {
      const int place = tile.row0 + t;
      const int64_t at =
          a.spread ? (int64_t)tile.rank * a.edge + token_at(a.order, place, a.tokens)
                   : (int64_t)(place / a.edge + tile.rank) * a.edge + place % a.edge;
      uint16_t* const to = a.pairs + at * a.pitch + rank0 + r;
      const uint32_t high = encode16<F>(v);
      const float left = v - decode16<F>(high);
      to[0] = (uint16_t)high;
      to[a.rest_at] = (uint16_t)encode16<F>(isfinite(left) ? left : 0.0f);
    }
  }
  if (a.pairs != nullptr) {
    // zeros in the rows of the adapter's first and last item that are not its own
    const int words = whole / 2;
    // (spread: in those of all tokens that are not this adapter's)
    if (a.spread && tile.row0 == tile.start) {
      const int others = a.tokens - (tile.end - tile.start);
      for (int i = threadIdx.x + S::kThreads * (int)split; i < others * words;
           i += S::kThreads * (int)splits) {
        const int o = i / words, place = o < tile.start ? o : o + tile.end - tile.start;
        uint16_t* const p =
            a.pairs + ((int64_t)tile.rank * a.edge + token_at(a.order, place, a.tokens)) * a.pitch +
            rank0 + 2 * (i % words);
        *reinterpret_cast<uint32_t*>(p) = 0u;
        *reinterpret_cast<uint32_t*>(p + a.rest_at) = 0u;
      }
    }
    const auto clear = [&](int item, int from_row, int to_row) {
      const int rows = to_row - from_row;
      for (int i = threadIdx.x + S::kThreads * (int)split; i < rows * words;
           i += S::kThreads * (int)splits) {
        uint16_t* const p = a.pairs + ((int64_t)item * a.edge + from_row + i / words) * a.pitch +
                            rank0 + 2 * (i % words);
        *reinterpret_cast<uint32_t*>(p) = 0u;
        *reinterpret_cast<uint32_t*>(p + a.rest_at) = 0u;
      }
    };
    if (!a.spread && tile.row0 == tile.start) clear(tile.start / a.edge + tile.rank, 0, tile.start % a.edge);
    const int final_row = tile.end - 1;
    if (!a.spread && final_row - tile.row0 < TOKENS)
      clear(final_row / a.edge + tile.rank, final_row % a.edge + 1, a.edge);
  }
  if (a.largest != nullptr) {
    const unsigned int top = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(most));
    if (lane == 0 && top != 0u) atomicMax(a.largest + tile.group, top);  // the order is no matter
  }
  if (splits > 1) cg::this_cluster().sync();  // the others have read this CTA's sums
}

// ---------------------------------------------------------------- gradients --
//
// out_a = sum over an adapter's tokens of z_t (cols) by low_t (rank).  A CTA takes 128 columns,
// up to 64 of the rank and a chunk of up to kSumTokens tokens of one adapter (counted from
// its first); adapters of several chunks leave FP32 parts, which another kernel adds in
// order.  z's bytes, read once for every 64 of the rank, bound it.  `low` enters as a pair of
// 16-bit numbers (high and what it leaves); in FP16 both are scaled by a power of two that
// brings the adapter's largest to 2^11 .. 2^12, so that small gradients keep their digits.
constexpr int kSumCols = 128, kSumStep = 64, kSumTokens = 512;
constexpr int kSumWarps = kSumCols / 16, kSumThreads = 32 * kSumWarps;

template <int RT>  // 16 RT of the rank
struct SumShape {
  static constexpr int kRank = 16 * RT;
  static constexpr int kZ = kSumStep * kSumCols * 2, kLow = kSumStep * kRank * 2;
  static constexpr int kStages = 5 - RT / 2;  // with them two CTAs an SM fit
  static constexpr int kSmem = kStages * kZ + 2 * 2 * kLow;
};

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

template <int F, int RT>
__global__ void __launch_bounds__(kSumThreads, 2) sum_kernel(const SumArgs a) {
  using S = SumShape<RT>;
  extern __shared__ __align__(128) uint8_t raw[];
  __shared__ int32_t places[kSumTokens];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const GroupTile tile =
      find_group_tile(a.ends, a.adapters, a.tokens, kSumTokens, (int)blockIdx.y, lane);
  if (tile.group < 0) return;
  const int count = min(kSumTokens, tile.end - tile.row0);
  for (int i = threadIdx.x; i < count; i += kSumThreads)
    places[i] = (int32_t)token_at(a.order, tile.row0 + i, a.tokens);
  const int rank0 = (int)blockIdx.z * S::kRank, ranks = min(S::kRank, a.rank - rank0);
  const int col0 = (int)blockIdx.x * kSumCols;
  const float scale = pair_scale(a.largest, tile.group);
  const uint32_t z0 = shared_at(raw), low0 = z0 + S::kStages * S::kZ;
  __syncthreads();

  const int slot = threadIdx.x & 15, row = threadIdx.x >> 4;  // 16 rows at a time
  const int col = col0 + 8 * slot, bytes = min(max(a.cols - col, 0) * 2, 16);
  const char* const z = a.z + (int64_t)col * 2;
  const auto load = [&](int step, int s) {
#pragma unroll
    for (int i = 0; i < kSumStep / 16; ++i) {
      const int r = row + 16 * i, t = step * kSumStep + r;
      const bool in = t < count && bytes > 0;
      copy16(z0 + s * S::kZ + wide_slot(r, slot), in ? z + places[t] * a.z_pitch * 2 : a.z,
             in ? bytes : 0);
    }
  };
  // low: thread t has ranks 4 (t % 4) + 16 j of token t / 4
  const int low_row = threadIdx.x >> 2, low_col = (threadIdx.x & 3) * 4;
  const bool whole = (a.rank & 3) == 0;  // rows of whole 16 bytes
  float held[RT][4];
  const auto fetch = [&](int step) {
    const int t = step * kSumStep + low_row;
    const float* const from = a.low + (int64_t)(tile.row0 + t) * a.rank + rank0 + low_col;
#pragma unroll
    for (int j = 0; j < RT; ++j) {
      if (whole && t < count && low_col + 16 * j < ranks) {
        const float4 v = __ldg(reinterpret_cast<const float4*>(from + 16 * j));
        held[j][0] = v.x;
        held[j][1] = v.y;
        held[j][2] = v.z;
        held[j][3] = v.w;
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          held[j][i] = t < count && low_col + 16 * j + i < ranks ? __ldg(from + 16 * j + i) : 0.0f;
      }
    }
  };
  const auto low_slot = [](int r, int c) {
    return RT == 4 ? turned_slot(r, c) : narrow_slot<2 * RT>(r, c);
  };
  const auto split = [&](int b) {
    const uint32_t to = low0 + b * 2 * S::kLow;
#pragma unroll
    for (int j = 0; j < RT; ++j) {
      uint32_t high[2], rest[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float x = held[j][2 * i] * scale, y = held[j][2 * i + 1] * scale;
        const uint32_t hx = encode16<F>(x), hy = encode16<F>(y);
        high[i] = hx | hy << 16;
        rest[i] = encode16<F>(x - decode16<F>(hx)) | encode16<F>(y - decode16<F>(hy)) << 16;
      }
      // 8 of the 16 bytes of a slot
      const uint32_t at = to + low_slot(low_row, 2 * j + (low_col >> 3)) + 2 * (low_col & 7);
      asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(at), "r"(high[0]), "r"(high[1])
                   : "memory");
      asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(at + S::kLow), "r"(rest[0]),
                   "r"(rest[1])
                   : "memory");
    }
  };

  float sum[2 * RT][4];
#pragma unroll
  for (int i = 0; i < 2 * RT; ++i) {
#pragma unroll
    for (int j = 0; j < 4; ++j) sum[i][j] = 0.0f;
  }
  const int steps = (count + kSumStep - 1) / kSumStep;
  for (int i = 0; i < S::kStages - 1; ++i) {
    if (i < steps) load(i, i);
    copies_done();
  }
  fetch(0);
  int s = 0;
  for (int step = 0; step < steps; ++step) {
    split(step & 1);
    copies_wait<S::kStages - 2>();
    __syncthreads();
    if (step + S::kStages - 1 < steps)
      load(step + S::kStages - 1, s == 0 ? S::kStages - 1 : s - 1);
    copies_done();
    if (step + 1 < steps) fetch(step + 1);
    const uint32_t zs = z0 + s * S::kZ, ls = low0 + (step & 1) * 2 * S::kLow;
    if (++s == S::kStages) s = 0;
#pragma unroll
    for (int kk = 0; kk < kSumStep / 16; ++kk) {
      // columns 16 warp .. by tokens 16 kk ..: matrices of 8 tokens x 8 columns, turned
      uint32_t m[4];
      load_matrices<true>(zs + wide_slot(16 * kk + (lane & 7) + ((lane >> 4) << 3),
                                         2 * warp + ((lane >> 3) & 1)), m);
#pragma unroll
      for (int j = 0; j < RT; ++j) {
        uint32_t b[4];
        const uint32_t at = ls + low_slot(16 * kk + (lane & 15), 2 * j + (lane >> 4));
        load_matrices<true>(at, b);
        multiply<F>(sum[2 * j], m, b[0], b[1]);
        multiply<F>(sum[2 * j + 1], m, b[2], b[3]);
        load_matrices<true>(at + S::kLow, b);
        multiply<F>(sum[2 * j], m, b[0], b[1]);
        multiply<F>(sum[2 * j + 1], m, b[2], b[3]);
      }
    }
  }
  copies_wait<0>();
  const float back = 1.0f / scale;  // a power of two: exact
#pragma unroll
  for (int j = 0; j < 2 * RT; ++j) {
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
  const EndsAhead ahead(a.ends, a.adapters, lane);
  int carry = 0, chunks_before = 0, first = 0, chunks = 0;
  for (int base = 0; base <= group; base += 32) {
    int start, end;
    group_span(a.ends, ahead, a.adapters, a.tokens, base, lane, &carry, &start, &end);
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

// Opt-in shared memory of a kernel, once a device.
int allow_shared(const void* kernel, int bytes) {
  int resident = 0;
  return prepare_kernel(kernel, 1, 32, bytes, &resident);
}

template <int F, bool KINNER, int TOKENS, int RT>
int launch_low_as(const LowArgs& args, cudaStream_t stream) {
  using S = LowShape<TOKENS, RT>;
  const auto kernel = &low_kernel<F, KINNER, TOKENS, RT>;
  if (int rc = allow_shared(reinterpret_cast<const void*>(kernel), S::kSmem)) return rc;
  const int64_t busy = args.adapters < args.tokens ? args.adapters : args.tokens;
  const int64_t tiles = most_group_tiles(args.tokens, args.adapters, TOKENS);
  const int64_t blocks = ceil_div(args.rank, S::kRank), steps = ceil_div(args.k, kLowStep);
  // Parts of the sum while all likely CTAs run at once (two an SM; four of the small), at least
  // four stages each.  A second round costs as much as the first: 16 prompts of 4096 tokens in
  // all, 4096 -> 64, took 30 us in 384 CTAs.
  const int64_t likely = (args.tokens / TOKENS + (busy + 1) / 2) * blocks;
  const int64_t room = (TOKENS == 16 ? 4 : 2) * sm_count();
  int64_t splits = likely > 0 ? room / likely : 8;
  if (splits > steps / 4) splits = steps / 4;
  splits = splits < 1 ? 1 : splits > 8 ? 8 : splits;
  cudaLaunchConfig_t config{};
  cudaLaunchAttribute cluster{};
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = (unsigned)splits;
  cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
  config.gridDim = dim3((unsigned)(tiles * splits), (unsigned)blocks);
  config.blockDim = dim3(S::kThreads);
  config.dynamicSmemBytes = S::kSmem;
  config.stream = stream;
  config.attrs = &cluster;
  config.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&config, kernel, args);
  return e == cudaSuccess ? SRS_OK : cuda_fail(e, "low part launch");
}

template <int F, bool KINNER>
int launch_low(const LowArgs& args, bool thin, cudaStream_t stream) {
  if (args.rank <= 16)
    return thin ? launch_low_as<F, KINNER, 16, 1>(args, stream)
                : launch_low_as<F, KINNER, 128, 1>(args, stream);
  if (args.rank <= 32)
    return thin ? launch_low_as<F, KINNER, 16, 2>(args, stream)
                : launch_low_as<F, KINNER, 128, 2>(args, stream);
  return thin ? launch_low_as<F, KINNER, 16, 4>(args, stream)
              : launch_low_as<F, KINNER, 128, 4>(args, stream);
}

template <int F, int RT>
int launch_sum_as(const SumArgs& args, cudaStream_t stream) {
  using S = SumShape<RT>;
  const auto kernel = &sum_kernel<F, RT>;
  if (int rc = allow_shared(reinterpret_cast<const void*>(kernel), S::kSmem)) return rc;
  const dim3 grid((unsigned)ceil_div(args.cols, kSumCols),
                  (unsigned)most_group_tiles(args.tokens, args.adapters, kSumTokens),
                  (unsigned)ceil_div(args.rank, S::kRank));
  kernel<<<grid, kSumThreads, S::kSmem, stream>>>(args);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? SRS_OK : cuda_fail(e, "adapter gradient launch");
}

template <int F>
int launch_sum(const SumArgs& args, cudaStream_t stream) {
  if (args.rank <= 16) return launch_sum_as<F, 1>(args, stream);
  if (args.rank <= 32) return launch_sum_as<F, 2>(args, stream);
  return launch_sum_as<F, 4>(args, stream);
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

// Few tokens: the projection's thin form.
static bool few(int64_t tokens) { return tokens <= kThinRows; }

// Parts of a call's workspace, each on a 256-byte boundary.
struct AdapterSpace {
  int64_t low, total;  // quantised tokens first, then the pairs of the low part
};

static AdapterSpace adapter_space(int64_t tokens, int64_t k, int64_t n, int adapters, int rank) {
  AdapterSpace s{};
  int64_t at = whole(srs_linear_workspace(tokens, k));
  s.low = at;
  if (n > 0) {
    const int64_t rows = few(tokens)
                             ? (adapters < tokens ? adapters : tokens) * thin_columns(tokens)
                             : pair_items(tokens, adapters, adapter_edge(tokens, n, k)) *
                                   adapter_edge(tokens, n, k);
    at += whole(rows * pair_shape(rank).pitch * 2);
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
  const int edge = n == 0 ? 0 : thin ? thin_columns(tokens) : adapter_edge(tokens, n, k);
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
  l.low = low;
  l.largest = largest;
  if (edge != 0) {
    l.pairs = reinterpret_cast<uint16_t*>(at + space.low);
    l.edge = edge;
    l.pitch = pairs.pitch;
    l.rest_at = pairs.rest_at;
    l.spread = thin;
  }
  if (int rc = turned ? (bf16 ? launch_low<SRS_FMT_BF16, false>(l, thin, st)
                              : launch_low<SRS_FMT_F16, false>(l, thin, st))
                      : (bf16 ? launch_low<SRS_FMT_BF16, true>(l, thin, st)
                              : launch_low<SRS_FMT_F16, true>(l, thin, st)))
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
  q.overlap = true;  // beside the low part
  if (int rc = quantize(q, st)) return rc;
  const AdapterCall call{l.pairs,
                         reinterpret_cast<const void*>(turned ? a->down : a->up),
                         turned ? a->down_pitch : a->up_pitch,
                         turned ? a->down_stride : a->up_stride,
                         turned != 0,
                         a->count,
                         a->rank,
                         a->format,
                         l.order,
                         l.ends};
  // (with few tokens beside the quantisation: the weights are streamed first)
  return thin ? launch_thin(*w, rows, k, d, a->format, 1, n, true, st, &call)
              : launch_adapter_product(rows, *w, k, call, edge, d, st);
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
  if (int rc = format == SRS_FMT_BF16 ? launch_sum<SRS_FMT_BF16>(a, st)
                                      : launch_sum<SRS_FMT_F16>(a, st))
    return rc;
  const int64_t blocks = ceil_div((int64_t)rank * cols, 1024);
  const dim3 joins((unsigned)(blocks < 1024 ? blocks : 1024), (unsigned)adapters);
  if (format == SRS_FMT_BF16) join_kernel<SRS_FMT_BF16><<<joins, 256, 0, st>>>(a);
  else join_kernel<SRS_FMT_F16><<<joins, 256, 0, st>>>(a);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? SRS_OK : cuda_fail(e, "adapter gradient launch");
}
