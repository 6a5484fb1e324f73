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
// they are split into a pair of 16-bit numbers.  A pair loses 2^-17 of them in BF16 and 2^-22 in
// FP16, a 512th and a 2048th of what the result's own rounding may: with three BF16 numbers in the
// gradients' sums the results' distance from FP64 was the same to five digits (0.001654 of their
// size), and calls were 1 to 4 % slower.
#include <cooperative_groups.h>

#include "srs_common.cuh"
#include "srs_groups.cuh"
#include "srs_host.h"
#include "srs_launch.h"
#include "srs_product.cuh"

namespace srs {
namespace {

namespace cg = cooperative_groups;

// 16 bytes to shared memory, those behind the first `bytes` zero.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global.L2::256B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes)
               : "memory");
}

// Rows of SLOTS (2, 4 or 8) 16-byte slots, turned so that 8 rows at one slot reach all banks: the
// order of 32-, 64- and 128-byte swizzled boxes.
template <int SLOTS>
__device__ __forceinline__ uint32_t narrow_slot(int row, int slot) {
  return (uint32_t)(row * 16 * SLOTS + ((slot ^ ((row / (8 / SLOTS)) & (SLOTS - 1))) << 4));
}

// Descriptor of such an operand with 16 RT rows side by side: groups of 8 of k are 256 RT bytes
// apart.
template <int RT>
__device__ __forceinline__ uint64_t narrow_descriptor() {
  constexpr uint64_t kMode = RT == 4 ? 2 : RT == 2 ? 4 : 6;  // 128-, 64-, 32-byte swizzle
  return (1ull << 16) | (uint64_t((256u * RT) >> 4) << 32) | (1ull << 46) | (kMode << 61);
}

__device__ __forceinline__ void copies_done() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
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
// A CTA takes up to 128 (or 16) tokens of one adapter (tiles counted from the adapter's first), up
// to 16 RT of the rank and a part of the sum; the parts of a cluster's CTAs are added through
// distributed shared memory in rank order.  x's bytes, read once, bound it.  Sums are FP32.
constexpr int kLowStep = 64;  // of k a stage: 128 bytes of a row

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
  uint16_t* pairs;        // items for a product (null: not wanted)
  int edge, pitch, rest_at;
  bool spread;            // items of a thin product: rows are the batch's
  unsigned int* largest;  // of an adapter's |low|, as encodings (null: not wanted)
  int32_t* exponents;     // of the tokens' pairs (FP16)
  unsigned int* status;
};

// 16-byte slot `slot` of a row of 128 bytes, turned so that 8 rows at one slot and 8 slots of a
// row both reach all banks: the order of 128-byte swizzled boxes.
__device__ __forceinline__ uint32_t turned_slot(int row, int slot) {
  return (uint32_t)(row * 128 + ((slot ^ (row & 7)) << 4));
}

// The CTA's part of a sum.
struct LowTile {
  GroupTile tile;
  int count, rank0, ranks, first, last;  // tokens, ranks, stages of k
  uint32_t splits, split;
};

__device__ __forceinline__ LowTile low_tile(const LowArgs& a, int most, int rank_block, int lane) {
  LowTile t;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(t.splits));
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(t.split));
  t.tile = find_group_tile(a.ends, a.adapters, a.tokens, most, (int)(blockIdx.x / t.splits), lane);
  t.count = min(most, t.tile.end - t.tile.row0);
  t.rank0 = (int)blockIdx.y * rank_block;
  t.ranks = min(rank_block, a.rank - t.rank0);
  const int steps = (a.k + kLowStep - 1) / kLowStep;
  t.first = (int)((int64_t)steps * t.split / t.splits);
  t.last = (int)((int64_t)steps * (t.split + 1) / t.splits);
  return t;
}

// Token at place `place`, rank r of the low part as a pair.
template <int F>
__device__ __forceinline__ void write_pair(const LowArgs& a, const GroupTile& tile, int place, int r,
                                           float v) {
  const int64_t at = a.spread ? (int64_t)tile.rank * a.edge + token_at(a.order, place, a.tokens)
                              : (int64_t)(place / a.edge + tile.rank) * a.edge + place % a.edge;
  uint16_t* const to = a.pairs + at * a.pitch + r;
  const uint32_t high = encode16<F>(v);
  const float left = v - decode16<F>(high);
  to[0] = (uint16_t)high;
  to[a.rest_at] = (uint16_t)encode16<F>(isfinite(left) ? left : 0.0f);
}

// Zeros in the rows of a thin product's item that are not its adapter's (`whole` of the rank from
// rank0 on), by the threads from, from + step, .. of those that have the adapter's first tile.
__device__ __forceinline__ void clear_item(const LowArgs& a, const GroupTile& tile, int rank0,
                                           int whole, int from, int step) {
  if (tile.row0 != tile.start) return;
  const int words = whole / 2, others = a.tokens - (tile.end - tile.start);
  for (int i = from; i < others * words; i += step) {
    const int o = i / words, place = o < tile.start ? o : o + tile.end - tile.start;
    uint16_t* const p =
        a.pairs + ((int64_t)tile.rank * a.edge + token_at(a.order, place, a.tokens)) * a.pitch +
        rank0 + 2 * (i % words);
    *reinterpret_cast<uint32_t*>(p) = 0u;
    *reinterpret_cast<uint32_t*>(p + a.rest_at) = 0u;
  }
}

// Sums of the cluster's CTAs (`sums`: [token][rank], rows of `pitch`, PARTS of them `part` apart
// in every CTA) added, scaled and written: token t of the tile by CTA t % splits.
template <int F, int RANK, int PARTS>
__device__ __forceinline__ void write_low(const LowArgs& a, const LowTile& l, float* sums, int pitch,
                                          int part, int most, int threads) {
  const GroupTile& tile = l.tile;
  const int splits = (int)l.splits, split = (int)l.split;
  const float factor = a.factor * (a.scale != nullptr ? __ldg(a.scale + tile.group) : 1.0f);
  if (splits > 1) cg::this_cluster().sync();
  else __syncthreads();
  float top_size = 0.0f;
  const int whole = (l.ranks + 15) & ~15;
  for (int i = threadIdx.x; i < (most + splits - 1) / splits * RANK; i += threads) {
    const int t = i / RANK * splits + split, r = i % RANK;
    if (t >= l.count || r >= whole) continue;
    float v = 0.0f;
    if (r < l.ranks) {
      for (int p = 0; p < splits; ++p) {
        const float* const theirs =
            (splits > 1 ? cg::this_cluster().map_shared_rank(sums, p) : sums) + t * pitch + r;
#pragma unroll
        for (int q = 0; q < PARTS; ++q) v += theirs[q * part];
      }
      v *= factor;
      if (a.low != nullptr) a.low[(int64_t)(tile.row0 + t) * a.rank + l.rank0 + r] = v;
      top_size = fmaxf(top_size, isfinite(v) ? fabsf(v) : 0.0f);
    }
    if (a.pairs != nullptr) write_pair<F>(a, tile, tile.row0 + t, l.rank0 + r, v);
  }
  if (a.pairs != nullptr && a.spread)
    clear_item(a, tile, l.rank0, whole, (int)threadIdx.x + threads * split, threads * splits);
  if (a.largest != nullptr) {
    const unsigned int top = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(top_size));
    // (the order is no matter)
    if ((threadIdx.x & 31) == 0 && top != 0u) atomicMax(a.largest + tile.group, top);
  }
  if (splits > 1) cg::this_cluster().sync();  // the others have read this CTA's sums
}

// FP16 pairs, of the finished FP32 low part: what they are scaled by depends on all of a token's.  A
// warp a token.
constexpr int kPairTokens = 32, kPairThreads = 256;

__global__ void __launch_bounds__(kPairThreads) pairs_kernel(const LowArgs a) {
  // A thin product launched to overlap this kernel may start.
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const GroupTile tile = find_group_tile(a.ends, a.adapters, a.tokens, kPairTokens,
                                         (int)blockIdx.x, (int)(threadIdx.x & 31));
  const int lane = threadIdx.x & 31;
  const auto exponent_of = [&](int place) {
    return a.exponents + (a.spread ? token_at(a.order, place, a.tokens) : place);
  };
  {
    // tokens of no adapter, by all threads of the grid
    const EndsAhead ahead(a.ends, a.adapters, lane);
    int last = 0;
    for (int base = 0; base < a.adapters; base += 32) {
      int start, end;
      group_span(a.ends, ahead, a.adapters, a.tokens, base, lane, &last, &start, &end);
    }
    for (int i = last + (int)(blockIdx.x * kPairThreads + threadIdx.x); i < a.tokens;
         i += (int)gridDim.x * kPairThreads)
      *exponent_of(i) = 0;
  }
  if (tile.group < 0) return;
  const int count = min(kPairTokens, tile.end - tile.row0), whole = (a.rank + 15) & ~15;
  for (int t = threadIdx.x >> 5; t < count; t += kPairThreads / 32) {
    const int place = tile.row0 + t;
    const float* const from = a.low + (int64_t)place * a.rank;
    float top_size = 0.0f;
    for (int r = lane; r < a.rank; r += 32) {
      const float size = fabsf(__ldcg(from + r));
      top_size = fmaxf(top_size, isfinite(size) ? size : 0.0f);
    }
    const int k =
        pair_exponent(__reduce_max_sync(0xFFFFFFFFu, __float_as_uint(top_size)));
    const float factor = two_to(k);
    for (int r = lane; r < whole; r += 32)
      write_pair<SRS_FMT_F16>(a, tile, place, r, r < a.rank ? __ldcg(from + r) * factor : 0.0f);
    if (lane == 0) *exponent_of(place) = k;
  }
  if (a.spread) clear_item(a, tile, 0, whole, (int)threadIdx.x, kPairThreads);
}

// Calls of few tokens, where most adapters have one or two: 16 tokens, and 4 warps that share a
// stage's four steps of 16 of k with mma.sync.  Latency bounds them: launch, the ends, the order and
// the first bytes one after the other, and the cluster's meeting.
template <int RT>
struct FewShape {
  static constexpr int kTokens = 16, kWarps = 4, kThreads = 128, kRank = 16 * RT, kStages = 8;
  static constexpr int kX = kTokens * kLowStep * 2, kW = kRank * kLowStep * 2;
  static constexpr int kPitch = kRank + 1;
  static constexpr int kSums = kWarps * kTokens * kPitch * 4;
  static constexpr int kSmem = kStages * (kX + kW) > kSums ? kStages * (kX + kW) : kSums;
};

template <int F, bool KINNER, int RT>
__global__ void __launch_bounds__(FewShape<RT>::kThreads, 4) low_few_kernel(const LowArgs a) {
  using S = FewShape<RT>;
  extern __shared__ __align__(128) uint8_t raw[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const LowTile l = low_tile(a, S::kTokens, S::kRank, lane);
  // This kernel runs beside the quantisation, of which it reads nothing, but no CTA of it lets the
  // product behind start, or leaves, before that is done: the product starts with the tokens'
  // blocks there and waits for the low part alone, when it comes to the adapters.
  if (l.tile.group < 0) {  // the whole cluster
    asm volatile("griddepcontrol.wait;" ::: "memory");
    return;
  }
  const uint32_t base = smem_address(raw);
  const int slot = threadIdx.x & 7, row = threadIdx.x >> 3;
  const char* const from =
      a.x + (row < l.count ? token_at(a.order, l.tile.row0 + row, a.tokens) : 0) * a.x_pitch * 2;
  const char* const w = a.w + (int64_t)l.tile.group * a.w_stride * 2;
  const auto load = [&](int step, int s) {
    const int k = step * kLowStep + 8 * slot, bytes = min(max(a.k - k, 0) * 2, 16);
    const uint32_t to = base + (uint32_t)(s * (S::kX + S::kW));
    copy16(to + turned_slot(row, slot), bytes > 0 ? from + 2 * k : a.x, row < l.count ? bytes : 0);
    if (KINNER) {
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        const int r = row + 16 * i;
        const bool in = r < l.ranks && bytes > 0;
        copy16(to + S::kX + turned_slot(r, slot),
               in ? w + ((int64_t)(l.rank0 + r) * a.w_pitch + k) * 2 : w, in ? bytes : 0);
      }
    } else {
      // 64 rows of k, 2 RT slots of 8 of the rank each
#pragma unroll
      for (int i = threadIdx.x; i < kLowStep * 2 * RT; i += S::kThreads) {
        const int r = i / (2 * RT), c = i % (2 * RT), kk = step * kLowStep + r;
        const int left = min(max(l.ranks - 8 * c, 0) * 2, 16);
        const bool in = kk < a.k && left > 0;
        copy16(to + S::kX + narrow_slot<2 * RT>(r, c),
               in ? w + ((int64_t)kk * a.w_pitch + l.rank0 + 8 * c) * 2 : w, in ? left : 0);
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
    if (l.first + i < l.last) load(l.first + i, i);
    copies_done();
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  int s = 0;
  for (int step = l.first; step < l.last; ++step) {
    copies_wait<S::kStages - 2>();
    __syncthreads();
    if (step + S::kStages - 1 < l.last) load(step + S::kStages - 1, s == 0 ? S::kStages - 1 : s - 1);
    copies_done();
    const uint32_t xs = base + (uint32_t)(s * (S::kX + S::kW)), ws = xs + S::kX;
    if (++s == S::kStages) s = 0;
    uint32_t m[4];
    load_matrices<false>(xs + turned_slot(lane & 15, 2 * warp + (lane >> 4)), m);
#pragma unroll
    for (int j = 0; j < RT; ++j) {
      uint32_t b[4];
      if (KINNER) {  // ranks 16 j + (0..15) x k 16 warp ..
        load_matrices<false>(ws + turned_slot(16 * j + (lane & 7) + ((lane >> 4) << 3),
                                              2 * warp + ((lane >> 3) & 1)), b);
      } else {       // k 16 warp + (0..15) x ranks 16 j ..
        const int r = 16 * warp + (lane & 15), c = 2 * j + (lane >> 4);
        load_matrices<true>(ws + narrow_slot<2 * RT>(r, c), b);
      }
      multiply<F>(sum[2 * j], m, b[0], b[1]);
      multiply<F>(sum[2 * j + 1], m, b[2], b[3]);
    }
  }
  // every warp's sums to shared memory
  copies_wait<0>();
  __syncthreads();
  float* const sums = reinterpret_cast<float*>(raw);
  float* const mine = sums + warp * S::kTokens * S::kPitch;
#pragma unroll
  for (int j = 0; j < 2 * RT; ++j) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      mine[((lane >> 2) + 8 * (i >> 1)) * S::kPitch + 8 * j + 2 * (lane & 3) + (i & 1)] = sum[j][i];
  }
  write_low<F, S::kRank, S::kWarps>(a, l, sums, S::kPitch, S::kTokens * S::kPitch, S::kTokens,
                                    S::kThreads);
}

// Many tokens: 128 of one adapter (the rows of an MMA), gathered with cp.async into the layout that
// the tensor core reads, so that a stage's four MMAs need nothing of the warps.  A stage is loaded
// again once the MMAs of two stages before have read theirs.  4096 tokens, 4096 -> 64, 16 adapters,
// beside the quantisation: 24 us; x's bytes would take 5, some 9 are launch, dependent first loads and
// the cluster's meeting.  4096 tokens, 14336 -> 16, behind a kernel that left 117 MB to write back:
// 49 us for 117 MB.  (ldmatrix and mma.sync in 8 warps read shared memory five times as often and
// took as long, 25 and 44 us; one kernel for this and the quantisation, x read once, took 36 and
// 113 us, these two side by side 33 and 112.)
constexpr int kManyTokens = 128, kManyThreads = 256;

template <int RT>
struct ManyShape {
  static constexpr int kRank = 16 * RT;
  static constexpr int kX = kManyTokens * 128, kW = kLowStep * kRank * 2;
  static constexpr int kStages = RT == 1 ? 6 : RT == 2 ? 5 : 4;  // two CTAs an SM fit
  static constexpr int kPitch = kRank + 1;
  static constexpr int kSmem = 1024 + kStages * (kX + kW);
  static constexpr uint32_t kColumns = RT == 4 ? 64 : 32;  // of TMEM
  static_assert(kManyTokens * kPitch * 4 <= kStages * (kX + kW), "the sums fit the stages");
};

template <int F, bool KINNER, int RT>
__global__ void __launch_bounds__(kManyThreads, 2) low_many_kernel(const LowArgs a) {
  using S = ManyShape<RT>;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  extern __shared__ uint8_t raw[];
  __shared__ __align__(8) uint64_t bars[S::kStages];
  __shared__ uint32_t tmem_slot;
  const int lane = threadIdx.x & 31, warp = warp_index();
  const LowTile l = low_tile(a, kManyTokens, S::kRank, lane);
  if (l.tile.group < 0) return;  // the whole cluster
  const uint32_t base = (smem_address(raw) + 1023u) & ~1023u, bar0 = smem_address(bars);
  if (threadIdx.x == 0) {
    for (int i = 0; i < S::kStages; ++i) barrier_init(bar0 + 8 * i, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) tmem_alloc<1>(smem_address(&tmem_slot), S::kColumns);

  // this thread's rows of x: threadIdx.x / 8 + 32 i, slot threadIdx.x % 8
  const int slot = threadIdx.x & 7, row = threadIdx.x >> 3;
  const char* from[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = row + 32 * i;
    from[i] = a.x + (r < l.count ? token_at(a.order, l.tile.row0 + r, a.tokens) : 0) * a.x_pitch * 2;
  }
  const char* const w = a.w + (int64_t)l.tile.group * a.w_stride * 2;
  const auto load = [&](int step, int s) {
    const int k = step * kLowStep + 8 * slot, bytes = min(max(a.k - k, 0) * 2, 16);
    const uint32_t to = base + (uint32_t)(s * (S::kX + S::kW));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = row + 32 * i;
      if (32 * i < l.count)  // sums of the rows behind are not read
        copy16(to + turned_slot(r, slot), bytes > 0 ? from[i] + 2 * k : a.x,
               r < l.count ? bytes : 0);
    }
    if (KINNER) {
#pragma unroll
      for (int i = 0; i < (S::kRank + 31) / 32; ++i) {
        const int r = row + 32 * i;
        const bool in = r < l.ranks && bytes > 0;
        if (r < S::kRank)
          copy16(to + S::kX + turned_slot(r, slot),
                 in ? w + ((int64_t)(l.rank0 + r) * a.w_pitch + k) * 2 : w, in ? bytes : 0);
      }
    } else {
      // 64 rows of k, 2 RT slots of 8 of the rank each
#pragma unroll
      for (int i = threadIdx.x; i < kLowStep * 2 * RT; i += kManyThreads) {
        const int r = i / (2 * RT), c = i % (2 * RT), kk = step * kLowStep + r;
        const int left = min(max(l.ranks - 8 * c, 0) * 2, 16);
        const bool in = kk < a.k && left > 0;
        copy16(to + S::kX + narrow_slot<2 * RT>(r, c),
               in ? w + ((int64_t)kk * a.w_pitch + l.rank0 + 8 * c) * 2 : w, in ? left : 0);
      }
    }
  };
  for (int i = 0; i < S::kStages - 2; ++i) {
    if (l.first + i < l.last) load(l.first + i, i);
    copies_done();
  }
  tmem_fence_before();
  __syncthreads();
  tmem_fence_after();
  const uint32_t tmem = tmem_slot;
  constexpr uint32_t kInstruction = (uint32_t)(S::kRank >> 3) << 17 | (128u >> 4) << 24 | 1u << 4 |
                                    (F == SRS_FMT_BF16 ? 1u << 7 | 1u << 10 : 0u) |
                                    (KINNER ? 0u : 1u << 16);
  bool ok = true;
  const int steps = l.last - l.first;
  for (int i = 0; i < steps; ++i) {
    const int s = i % S::kStages;
    // what the threads have copied, for the tensor core
    copies_wait<S::kStages - 3>();
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncthreads();
    if (warp == 0) {
      if (elect_lane()) {
        const uint32_t xs = base + (uint32_t)(s * (S::kX + S::kW));
        const uint64_t dx = operand_descriptor(false) | uint64_t((xs >> 4) & 0x3FFFu);
        const uint64_t dw = (KINNER ? operand_descriptor(false) : narrow_descriptor<RT>()) |
                            uint64_t(((xs + S::kX) >> 4) & 0x3FFFu);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          mma_f16<1>(tmem, dx + 2 * j, dw + j * (KINNER ? 2u : 32u * RT), kInstruction,
                     (i | j) != 0 ? 1u : 0u);
        mma_commit<1>(bar0 + 8 * s);
      }
      __syncwarp();
    }
    // stage s - 2 for step i + kStages - 2
    if (i + S::kStages - 2 < steps) {
      if (ok && i >= 2)
        ok = barrier_wait(bar0 + 8 * ((i - 2) % S::kStages), ((i - 2) / S::kStages) & 1, a.status,
                          1u << 18);
      if (ok) load(l.first + i + S::kStages - 2, (i + S::kStages - 2) % S::kStages);
    }
    copies_done();
  }
  copies_wait<0>();
  // the last MMAs (those before are done with them)
  if (ok && steps > 0)
    barrier_wait(bar0 + 8 * ((steps - 1) % S::kStages), ((steps - 1) / S::kStages) & 1, a.status,
                 1u << 18);
  tmem_fence_after();
  __syncthreads();  // no thread still copies or reads a stage
  float* const sums = reinterpret_cast<float*>(raw + (base - smem_address(raw)));
  if (warp < 4) {
    const int t = 32 * warp + lane;
#pragma unroll
    for (int j = 0; j < RT; ++j) {
      uint32_t v[16];
      tmem_load16(tmem + ((uint32_t)(32 * warp) << 16) + 16 * j, v);
#pragma unroll
      for (int i = 0; i < 16; ++i)
        sums[t * S::kPitch + 16 * j + i] = steps > 0 ? __uint_as_float(v[i]) : 0.0f;
    }
  }
  tmem_fence_before();
  write_low<F, S::kRank, 1>(a, l, sums, S::kPitch, 0, kManyTokens, kManyThreads);
  __syncthreads();
  tmem_fence_after();
  if (warp == 1) tmem_free<1>(tmem, S::kColumns);
}

// ---------------------------------------------------------------- gradients --
//
// out_a = sum over an adapter's tokens of z_t (cols) by low_t (rank).  A CTA takes 128 columns (the
// rows of an MMA), up to 16 RT of the rank and a chunk of tokens of one adapter (counted from its
// first); an adapter of one chunk is finished here, one of several leaves FP32 parts, which another
// kernel adds in order.  z's bytes, read once for every 64 of the rank, bound it: rows are gathered
// with cp.async into the layout in which the tensor core reads tokens as k (4096 tokens, 4096 + 14336
// columns, rank 16: 61 us for 151 MB, and 9 to join).  `low` enters as a
// pair of 16-bit numbers (high and what it leaves); in FP16 both are scaled by a power of two that
// brings the adapter's largest to 2^11 .. 2^12, so that small gradients keep their digits.
constexpr int kSumCols = 128, kSumStep = 64, kSumThreads = 256;
constexpr int kSumChunk = 1024;  // most tokens of a chunk
constexpr int kSumZ = kSumStep * kSumCols * 2;

template <int RT>
struct SumShape {
  static constexpr int kRank = 16 * RT, kLow = kSumStep * kRank * 2;
  // two CTAs an SM for ranks up to 16 and above 32 (what shared memory has room for), else three
  static constexpr int kStages = RT == 2 ? 3 : 4, kResident = RT == 2 ? 3 : 2;
  static constexpr int kSmem = 1024 + kStages * kSumZ + 2 * 2 * kLow;
};

struct SumJob {
  const char* z;
  int64_t z_pitch;
  const float* low;
  const unsigned int* largest;
  int cols, turned;  // turned: out is cols x rank instead of rank x cols
  void* out;
  float* parts;  // [part][rank][cols]: the chunks of the adapters that have several, in order
  int blocks;    // of the grid's width (of sums; of joins)
};

// Both gradients of a call in one launch: their CTAs fill the SMs' last round together.
struct SumArgs {
  SumJob job[2];
  int tokens, rank, adapters;
  int chunk;  // tokens
  const int32_t* order;
  const int32_t* ends;
  unsigned int* status;
};

// An adapter's chunks, and the parts ahead of its own; by a warp.
struct SumParts {
  int first, chunks;
};

__device__ __forceinline__ SumParts parts_of(const SumArgs& a, int group, int lane) {
  const EndsAhead ahead(a.ends, a.adapters, lane);
  SumParts p{0, 0};
  int carry = 0, before = 0;
  for (int base = 0; base <= group; base += 32) {
    int start, end;
    group_span(a.ends, ahead, a.adapters, a.tokens, base, lane, &carry, &start, &end);
    const int n = (end - start + a.chunk - 1) / a.chunk, parts = n > 1 ? n : 0;
    const int upto = before + warp_scan_sum(parts, lane);
    if (group - base < 32) {
      p.first = __shfl_sync(0xFFFFFFFFu, upto - parts, group - base);
      p.chunks = __shfl_sync(0xFFFFFFFFu, n, group - base);
    }
    before = __shfl_sync(0xFFFFFFFFu, upto, 31);
  }
  return p;
}

__device__ __forceinline__ float pair_scale(const unsigned int* largest, int group) {
  if (largest == nullptr) return 1.0f;
  const unsigned int top = __ldg(largest + group);
  // 2^11 <= top * 2^k < 2^12; an encoding of zero or below the normal range: the largest factor
  const int k = 11 - ((int)(top >> 23) - 127);
  return __uint_as_float((uint32_t)(min(max(k, -126), 126) + 127) << 23);
}

template <int F, int RT>
__global__ void __launch_bounds__(kSumThreads, SumShape<RT>::kResident)
sum_kernel(const __grid_constant__ SumArgs a) {
  constexpr int kRank = 16 * RT, kSumStages = SumShape<RT>::kStages, kSumLow = SumShape<RT>::kLow;
  constexpr uint32_t kColumns = RT == 4 ? 64 : 32;
  extern __shared__ uint8_t raw[];
  __shared__ int32_t places[kSumChunk];
  __shared__ __align__(8) uint64_t bars[kSumStages];
  __shared__ uint32_t tmem_slot;
  const int lane = threadIdx.x & 31, warp = warp_index();
  const GroupTile tile =
      find_group_tile(a.ends, a.adapters, a.tokens, a.chunk, (int)blockIdx.y, lane);
  if (tile.group < 0) return;
  const int count = min(a.chunk, tile.end - tile.row0);
  for (int i = threadIdx.x; i < count; i += kSumThreads)
    places[i] = (int32_t)token_at(a.order, tile.row0 + i, a.tokens);
  const bool second = (int)blockIdx.x >= a.job[0].blocks;
  const SumJob& job = a.job[second ? 1 : 0];
  const int rank0 = (int)blockIdx.z * kRank, ranks = min(kRank, a.rank - rank0);
  const int col0 = ((int)blockIdx.x - (second ? a.job[0].blocks : 0)) * kSumCols;
  const float scale = pair_scale(job.largest, tile.group);
  const uint32_t z0 = (smem_address(raw) + 1023u) & ~1023u, low0 = z0 + kSumStages * kSumZ;
  const uint32_t bar0 = smem_address(bars);
  if (threadIdx.x == 0) {
    for (int i = 0; i < kSumStages; ++i) barrier_init(bar0 + 8 * i, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) tmem_alloc<1>(smem_address(&tmem_slot), kColumns);
  tmem_fence_before();
  __syncthreads();
  tmem_fence_after();
  const uint32_t tmem = tmem_slot;

  // z: two boxes of 64 columns, a token's 128 bytes a row; 16 tokens at a time
  const int slot = threadIdx.x & 15, row = threadIdx.x >> 4;
  const int col = col0 + 8 * slot, bytes = min(max(job.cols - col, 0) * 2, 16);
  const char* const z = job.z + (int64_t)col * 2;
  const int64_t z_step = job.z_pitch * 2;
  const uint32_t box = (uint32_t)(slot >> 3) * (kSumZ / 2);
  const auto load = [&](int step, int s) {
#pragma unroll
    for (int i = 0; i < kSumStep / 16; ++i) {
      const int r = row + 16 * i, t = step * kSumStep + r;
      const bool in = t < count && bytes > 0;
      copy16(z0 + s * kSumZ + box + turned_slot(r, slot & 7),
             in ? z + places[t] * z_step : job.z, in ? bytes : 0);
    }
  };
  // low: thread t has ranks 4 (t % 4) + 16 j of token t / 4
  const int low_row = threadIdx.x >> 2, low_col = (threadIdx.x & 3) * 4;
  const bool whole = (a.rank & 3) == 0;  // rows of whole 16 bytes
  const float* const low = job.low;
  float held[RT][4];
  const auto fetch = [&](int step) {
    const int t = step * kSumStep + low_row;
    const float* const from = low + (int64_t)(tile.row0 + t) * a.rank + rank0 + low_col;
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
  const auto split = [&](int b) {
    const uint32_t to = low0 + b * 2 * kSumLow;
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
      const uint32_t at = to + narrow_slot<2 * RT>(low_row, 2 * j + (low_col >> 3)) + 2 * (low_col & 7);
      asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(at), "r"(high[0]), "r"(high[1])
                   : "memory");
      asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(at + kSumLow), "r"(rest[0]),
                   "r"(rest[1])
                   : "memory");
    }
  };
  // both operands have their rows (columns of z, ranks) side by side
  constexpr uint32_t kInstruction = (uint32_t)(kRank >> 3) << 17 | (128u >> 4) << 24 | 1u << 4 |
                                    (F == SRS_FMT_BF16 ? 1u << 7 | 1u << 10 : 0u) | 1u << 15 |
                                    1u << 16;
  const int steps = (count + kSumStep - 1) / kSumStep;
  for (int i = 0; i < kSumStages - 2; ++i) {
    if (i < steps) load(i, i);
    copies_done();
  }
  fetch(0);
  const bool alone = tile.end - tile.start <= a.chunk;
  const int part = alone ? 0 : parts_of(a, tile.group, lane).first + (tile.row0 - tile.start) / a.chunk;
  bool ok = true;
  for (int i = 0; i < steps; ++i) {
    const int s = i % kSumStages;
    // the MMAs of step i - 2 have read this step's buffer of low, and the stage loaded below
    if (ok && i >= 2)
      ok = barrier_wait(bar0 + 8 * ((i - 2) % kSumStages), ((i - 2) / kSumStages) & 1, a.status,
                        1u << 19);
    split(i & 1);
    copies_wait<kSumStages - 3>();
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncthreads();
    if (warp == 0) {
      if (elect_lane()) {
        const uint32_t zs = z0 + s * kSumZ, ls = low0 + (i & 1) * 2 * kSumLow;
        const uint64_t dz = operand_descriptor(true) | uint64_t((zs >> 4) & 0x3FFFu);
        const uint64_t dl = narrow_descriptor<RT>() | uint64_t((ls >> 4) & 0x3FFFu);
        const uint64_t dr = narrow_descriptor<RT>() | uint64_t(((ls + kSumLow) >> 4) & 0x3FFFu);
#pragma unroll
        for (int j = 0; j < kSumStep / 16; ++j) {
          mma_f16<1>(tmem, dz + 128 * j, dr + 32 * RT * j, kInstruction, (i | j) != 0 ? 1u : 0u);
          mma_f16<1>(tmem, dz + 128 * j, dl + 32 * RT * j, kInstruction, 1u);
        }
        mma_commit<1>(bar0 + 8 * s);
      }
      __syncwarp();
    }
    if (i + kSumStages - 2 < steps && ok)
      load(i + kSumStages - 2, (i + kSumStages - 2) % kSumStages);
    copies_done();
    if (i + 1 < steps) fetch(i + 1);
  }
  copies_wait<0>();
  if (ok)
    barrier_wait(bar0 + 8 * ((steps - 1) % kSumStages), ((steps - 1) / kSumStages) & 1, a.status,
                 1u << 19);
  tmem_fence_after();
  if (warp < 4) {
    const float back = 1.0f / scale;  // a power of two: exact
    const int c = col0 + 32 * warp + lane;
#pragma unroll
    for (int j = 0; j < RT; ++j) {
      uint32_t v[16];
      tmem_load16(tmem + ((uint32_t)(32 * warp) << 16) + 16 * j, v);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int r = 16 * j + i;
        if (c >= job.cols || r >= ranks) continue;
        const float value = __uint_as_float(v[i]) * back;
        if (!alone)
          job.parts[((int64_t)part * a.rank + rank0 + r) * job.cols + c] = value;
        else
          static_cast<uint16_t*>(job.out)[(int64_t)tile.group * a.rank * job.cols +
                                          (job.turned ? (int64_t)c * a.rank + rank0 + r
                                                      : (int64_t)(rank0 + r) * job.cols + c)] =
              (uint16_t)encode16<F>(value);
      }
    }
  }
  tmem_fence_before();
  __syncthreads();
  tmem_fence_after();
  if (warp == 1) tmem_free<1>(tmem, kColumns);
}

// out_a = the sum of its chunks' parts, in order, where there are several; zeros without tokens.
template <int F>
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ SumArgs a) {
  const int lane = threadIdx.x & 31, group = (int)blockIdx.y;
  const SumParts own = parts_of(a, group, lane);
  if (own.chunks == 1) return;
  const bool second = (int)blockIdx.x >= a.job[0].blocks;
  const SumJob& job = a.job[second ? 1 : 0];
  const int block = (int)blockIdx.x - (second ? a.job[0].blocks : 0);
  const int64_t each = (int64_t)a.rank * job.cols;
  for (int64_t i = (int64_t)block * 256 + threadIdx.x; i < each; i += (int64_t)job.blocks * 256) {
    // i runs over the result's order
    const int64_t at = job.turned ? i % a.rank * job.cols + i / a.rank : i;
    float v = 0.0f;
    for (int c = 0; c < own.chunks; ++c) v += job.parts[(own.first + c) * each + at];
    static_cast<uint16_t*>(job.out)[group * each + i] = (uint16_t)encode16<F>(v);
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

// `room`: CTAs that run at once.  `overlap`: may start beside the kernel ahead.
int launch_low_kernel(const void* kernel, const LowArgs& args, int most, int rank_block, int threads,
                      int smem, int64_t room, bool overlap, cudaStream_t stream) {
  if (int rc = allow_shared(kernel, smem)) return rc;
  const int64_t busy = args.adapters < args.tokens ? args.adapters : args.tokens;
  const int64_t tiles = most_group_tiles(args.tokens, args.adapters, most);
  const int64_t blocks = ceil_div(args.rank, rank_block), steps = ceil_div(args.k, kLowStep);
  // Parts of the sum while all likely CTAs run at once, at least four stages each.  A second round
  // costs as much as the first: 16 prompts of 4096 tokens in all, 4096 -> 64, took 30 us in 384 CTAs.
  const int64_t likely = (args.tokens / most + (busy + 1) / 2) * blocks;
  int64_t splits = likely > 0 ? room / likely : 8;
  if (splits > steps / 4) splits = steps / 4;
  splits = splits < 1 ? 1 : splits > 8 ? 8 : splits;
  cudaLaunchConfig_t config{};
  cudaLaunchAttribute attributes[2]{};
  attributes[0].id = cudaLaunchAttributeClusterDimension;
  attributes[0].val.clusterDim.x = (unsigned)splits;
  attributes[0].val.clusterDim.y = attributes[0].val.clusterDim.z = 1;
  attributes[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attributes[1].val.programmaticStreamSerializationAllowed = 1;
  config.gridDim = dim3((unsigned)(tiles * splits), (unsigned)blocks);
  config.blockDim = dim3((unsigned)threads);
  config.dynamicSmemBytes = (size_t)smem;
  config.stream = stream;
  config.attrs = attributes;
  config.numAttrs = overlap ? 2 : 1;
  LowArgs copy = args;
  void* arguments[1] = {&copy};
  const cudaError_t e = cudaLaunchKernelExC(&config, kernel, arguments);
  return e == cudaSuccess ? SRS_OK : cuda_fail(e, "low part launch");
}

template <int F, bool KINNER, int RT>
int launch_low_as(const LowArgs& args, bool thin, bool overlap, cudaStream_t stream) {
  const int64_t sms = sm_count();
  if (thin)
    return launch_low_kernel(reinterpret_cast<const void*>(&low_few_kernel<F, KINNER, RT>), args,
                             FewShape<RT>::kTokens, FewShape<RT>::kRank, FewShape<RT>::kThreads,
                             FewShape<RT>::kSmem, (RT == 4 ? 2 : 4) * sms, overlap, stream);
  return launch_low_kernel(reinterpret_cast<const void*>(&low_many_kernel<F, KINNER, RT>), args,
                           kManyTokens, ManyShape<RT>::kRank, kManyThreads, ManyShape<RT>::kSmem,
                           2 * sms, overlap, stream);
}

template <int F, bool KINNER>
int launch_low(const LowArgs& args, bool thin, bool overlap, cudaStream_t stream) {
  if (args.rank <= 16) return launch_low_as<F, KINNER, 1>(args, thin, overlap, stream);
  if (args.rank <= 32) return launch_low_as<F, KINNER, 2>(args, thin, overlap, stream);
  return launch_low_as<F, KINNER, 4>(args, thin, overlap, stream);
}

template <int F, int RT>
int launch_sum_as(SumArgs& args, cudaStream_t stream) {
  const auto kernel = &sum_kernel<F, RT>;
  if (int rc = allow_shared(reinterpret_cast<const void*>(kernel), SumShape<RT>::kSmem)) return rc;
  for (SumJob& job : args.job) job.blocks = (int)ceil_div(job.cols, kSumCols);
  const dim3 grid((unsigned)(args.job[0].blocks + args.job[1].blocks),
                  (unsigned)most_group_tiles(args.tokens, args.adapters, args.chunk),
                  (unsigned)ceil_div(args.rank, 16 * RT));
  kernel<<<grid, kSumThreads, SumShape<RT>::kSmem, stream>>>(args);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? SRS_OK : cuda_fail(e, "adapter gradient launch");
}

template <int F>
int launch_sum(SumArgs& args, cudaStream_t stream) {
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
  if (tokens < 0 || tokens > kMaxQuantizedRows || k < 0 || n < 0 || k > (1ll << 30) ||
      n > (1ll << 30))
    return fail(SRS_ERR_INVALID_ARGUMENT, "sizes out of range (%lld tokens, %lld -> %lld)",
                (long long)tokens, (long long)k, (long long)n);
  if (tokens == 0) return SRS_OK;
  if (a->order == 0 || a->order % 4 != 0)
    return fail(SRS_ERR_INVALID_ARGUMENT, "null or misaligned order");
  if (a->scale % 4 != 0) return fail(SRS_ERR_INVALID_ARGUMENT, "misaligned scales");
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

// Few tokens: the projection's thin form.  (4096 -> 4096, rank 16, 5 adapters for every 8 tokens: 64
// tokens 25 us a call, 65 in the large form 43: nothing splits k there, and a tile has as many
// adapters as a thin one.)
static bool few(int64_t tokens) { return tokens <= kThinRows; }

// Parts of a call's workspace, each on a 256-byte boundary: the quantised tokens first; FP16 alone
// needs `low` and `exponents` (for both formats there is room).
struct AdapterSpace {
  int64_t pairs, low, exponents, total;
};

static AdapterSpace adapter_space(int64_t tokens, int64_t k, int64_t n, int adapters, int rank) {
  AdapterSpace s{};
  s.pairs = whole(srs_linear_workspace(tokens, k));
  int64_t rows = 0;
  if (n > 0)
    rows = few(tokens) ? (adapters < tokens ? adapters : tokens) * thin_columns(tokens)
                       : pair_items(tokens, adapters, adapter_edge(tokens, n, k)) *
                             adapter_edge(tokens, n, k);
  s.low = s.pairs + whole(rows * pair_shape(rank).pitch * 2);
  s.exponents = s.low + (n > 0 ? whole(tokens * rank * 4) : 0);
  s.total = s.exponents + (n > 0 ? whole(tokens * 4) : 0);
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
  if ((n > 0 && reinterpret_cast<uintptr_t>(d) % 2 != 0) ||
      reinterpret_cast<uintptr_t>(low) % 4 != 0 || reinterpret_cast<uintptr_t>(largest) % 4 != 0)
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
  if (bf16) largest = nullptr;
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
  l.low = low != nullptr ? low : bf16 ? nullptr : reinterpret_cast<float*>(at + space.low);
  l.largest = largest;
  l.exponents = reinterpret_cast<int32_t*>(at + space.exponents);
  if (int rc = status_word(&l.status)) return rc;
  if (edge != 0) {
    if (bf16) l.pairs = reinterpret_cast<uint16_t*>(at + space.pairs);
    l.edge = edge;
    l.pitch = pairs.pitch;
    l.rest_at = pairs.rest_at;
    l.spread = thin;
  }
  // Quantisation and low part run beside each other: with few tokens the quantisation first, as the
  // product waits for the low part only when it comes to the adapters; with many the longer one.
  const bool project = n > 0 && k > 0;
  const auto low_part = [&](bool overlap) {
    return turned ? (bf16 ? launch_low<SRS_FMT_BF16, false>(l, thin, overlap, st)
                          : launch_low<SRS_FMT_F16, false>(l, thin, overlap, st))
                  : (bf16 ? launch_low<SRS_FMT_BF16, true>(l, thin, overlap, st)
                          : launch_low<SRS_FMT_F16, true>(l, thin, overlap, st));
  };
  if (!thin || !project)
    if (int rc = low_part(false)) return rc;
  if (!project) return SRS_OK;

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
  q.overlap = !thin;
  if (int rc = quantize(q, st)) return rc;
  if (thin)
    if (int rc = low_part(true)) return rc;
  if (!bf16) {
    l.pairs = reinterpret_cast<uint16_t*>(at + space.pairs);
    pairs_kernel<<<(unsigned)most_group_tiles(tokens, a->count, kPairTokens), kPairThreads, 0, st>>>(l);
    e = cudaGetLastError();
    if (e != cudaSuccess) return cuda_fail(e, "pairs of the low part");
  }
  const AdapterCall call{l.pairs,
                         reinterpret_cast<const void*>(turned ? a->down : a->up),
                         turned ? a->down_pitch : a->up_pitch,
                         turned ? a->down_stride : a->up_stride,
                         turned != 0,
                         a->count,
                         a->rank,
                         a->format,
                         l.order,
                         l.ends,
                         bf16 ? nullptr : l.exponents};
  // (with few tokens beside the low part or its pairs: weights and tokens' blocks are streamed first)
  return thin ? launch_thin(*w, rows, k, d, a->format, 1, n, true, st, &call)
              : launch_adapter_product(rows, *w, k, call, edge, d, st);
}

// Tokens of a chunk for `cols` columns in all: long ones leave fewer parts, short ones keep the SMs
// busy (as if with three CTAs each).
static int sum_chunk(int64_t tokens, int64_t cols, int rank) {
  const int64_t each = ceil_div(cols, kSumCols) * ceil_div(rank, 64);
  int64_t chunk = tokens * each / (3 * sm_count());
  chunk = ceil_div(chunk < 256 ? 256 : chunk, kSumStep) * kSumStep;
  return (int)(chunk > kSumChunk ? kSumChunk : chunk);
}

// Most chunks of the adapters that have more than one: two of every chunk + 1 tokens, as many such
// adapters as there can be, and one more of a chunk that is left.
static int64_t sum_parts(int64_t tokens, int64_t chunk) {
  const int64_t adapters = tokens / (chunk + 1);
  return adapters == 0 ? 0 : 2 * adapters + (tokens - adapters * (chunk + 1)) / chunk;
}

extern "C" int64_t srs_adapter_gradient_workspace(int64_t tokens, int64_t cols, int adapters,
                                                  int rank) {
  if (tokens <= 0 || cols <= 0 || adapters < 1 || rank < 1) return 0;
  return sum_parts(tokens, sum_chunk(tokens, cols, rank)) * rank * cols * 4;
}

extern "C" int srs_adapter_gradient(const srs_adapter_sum* sums, int n_sums, int format,
                                    int64_t tokens, int adapters, int rank, const int32_t* order,
                                    const int32_t* ends, void* workspace, int64_t workspace_bytes,
                                    void* stream) {
  clear_error();
  if (int rc = check_groups(ends, adapters)) return rc;
  if (sums == nullptr || n_sums < 1 || n_sums > 2)
    return fail(SRS_ERR_INVALID_ARGUMENT, "one or two sums a call, got %d", n_sums);
  if (format != SRS_FMT_BF16 && format != SRS_FMT_F16)
    return fail(SRS_ERR_INVALID_ARGUMENT, "adapters are BF16 or FP16, got format %d", format);
  if (rank < 1 || rank > SRS_ADAPTER_MAX_RANK || tokens < 0 || tokens > kMaxQuantizedRows)
    return fail(SRS_ERR_INVALID_ARGUMENT, "sizes out of range (%lld tokens, rank %d)",
                (long long)tokens, rank);
  SumArgs a{};
  int64_t cols = 0;
  int jobs = 0;
  for (int i = 0; i < n_sums; ++i) {
    const srs_adapter_sum& s = sums[i];
    if (s.cols < 0 || s.cols > (1ll << 30))
      return fail(SRS_ERR_INVALID_ARGUMENT, "%lld columns are out of range", (long long)s.cols);
    if (s.cols == 0) continue;
    if (s.out == 0 || s.out % 2 != 0)
      return fail(SRS_ERR_INVALID_ARGUMENT, "null or misaligned result pointer");
    if (tokens > 0 && (s.z == 0 || s.z_pitch < s.cols || s.z_pitch % 8 != 0 || s.z % 16 != 0))
      return fail(SRS_ERR_INVALID_ARGUMENT, "z needs a 16-byte aligned address and row pitch");
    if (tokens > 0 && (s.low == 0 || s.low % 16 != 0 || s.largest % 4 != 0))
      return fail(SRS_ERR_INVALID_ARGUMENT,
                  "low needs a 16-byte aligned address, the largest a multiple of 4");
    if (tokens > 0 && (order == nullptr || reinterpret_cast<uintptr_t>(order) % 4 != 0))
      return fail(SRS_ERR_INVALID_ARGUMENT, "null or misaligned order");
    SumJob& job = a.job[jobs++];
    job.z = reinterpret_cast<const char*>(s.z);
    job.z_pitch = s.z_pitch;
    job.low = reinterpret_cast<const float*>(s.low);
    job.largest =
        format == SRS_FMT_F16 ? reinterpret_cast<const unsigned int*>(s.largest) : nullptr;
    job.cols = (int)s.cols;
    job.turned = s.turned != 0;
    job.out = reinterpret_cast<void*>(s.out);
    cols += s.cols;
  }
  if (jobs == 0) return SRS_OK;
  if (int rc = check_device()) return rc;
  if (int rc = check_products()) return rc;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (tokens == 0) {
    for (int i = 0; i < jobs; ++i) {
      const cudaError_t e = cudaMemsetAsync(
          a.job[i].out, 0, (size_t)(2ll * a.job[i].cols * rank * adapters), st);
      if (e != cudaSuccess) return cuda_fail(e, "srs_adapter_gradient");
    }
    return SRS_OK;
  }
  const int64_t least = srs_adapter_gradient_workspace(tokens, cols, adapters, rank);
  if (workspace_bytes < least ||
      (least > 0 && (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 16 != 0)))
    return fail(SRS_ERR_INVALID_ARGUMENT, "workspace of %lld bytes, %lld needed",
                (long long)workspace_bytes, (long long)least);
  a.tokens = (int)tokens;
  a.rank = rank;
  a.adapters = adapters;
  a.order = order;
  a.ends = ends;
  a.chunk = sum_chunk(tokens, cols, rank);
  if (int rc = status_word(&a.status)) return rc;
  a.job[0].parts = static_cast<float*>(workspace);
  a.job[1].parts = a.job[0].parts + sum_parts(tokens, a.chunk) * rank * a.job[0].cols;
  if (int rc = format == SRS_FMT_BF16 ? launch_sum<SRS_FMT_BF16>(a, st)
                                      : launch_sum<SRS_FMT_F16>(a, st))
    return rc;
  for (SumJob& job : a.job) {
    const int64_t blocks = ceil_div((int64_t)rank * job.cols, 1024);
    job.blocks = (int)(blocks < 512 ? blocks : 512);
  }
  const dim3 joins((unsigned)(a.job[0].blocks + a.job[1].blocks), (unsigned)adapters);
  if (format == SRS_FMT_BF16) join_kernel<SRS_FMT_BF16><<<joins, 256, 0, st>>>(a);
  else join_kernel<SRS_FMT_F16><<<joins, 256, 0, st>>>(a);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? SRS_OK : cuda_fail(e, "adapter gradient launch");
}
