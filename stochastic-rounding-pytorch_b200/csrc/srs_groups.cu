// Rows sorted by their group: a stable counting sort of small whole numbers.
//
//   order: rows of group 0 in order, then those of group 1, .. , then rows of no group
//   ends[g] = rows whose group is at most g
//
// What bounds it: latency.  4 bytes a row in and out are nothing (65536 rows: 0.1 us at
// the HBM's rate); a launch, two walks over the rows and the sums between them are what
// there is.  One launch: each warp takes a run of consecutive rows, counts its rows of
// each group in shared memory, the counts are added over the warps (and over the cluster's
// CTAs through distributed shared memory), and the warp then places its rows one batch of
// 32 after the other, a row's rank in its batch from a vote over equal groups.  No atomic
// decides an order, so the result does not depend on timing.
//
// In a cluster, up to 4096 rows of a CTA are put in order in shared memory first and leave in runs.
#include <cooperative_groups.h>

#include "srs_groups.cuh"
#include "srs_host.h"
#include "srs_launch.h"

namespace srs {
namespace {

namespace cg = cooperative_groups;

constexpr int kSortAhead = 8;     // batches of a warp loaded together
// Rows up to kSortSmall: one CTA of 32 warps, 128 rows each.  More: a cluster of 16 CTAs of 16
// warps (its meetings and remote counts cost about 2 us).  The instructions of 200 a batch bound
// it: 65536 rows took 12.2 us on eight SMs, 9.6 on these.  Beyond 65536 rows (16 x 4096) they do not
// fit the registers and shared memory: the index is read twice and rows leave one by one, 14.6 us a
// call for 2^17 rows, 21.9 for 2^18, 66 for 2^20, 240 for 2^22.
constexpr int kSortCluster = 16;
constexpr int64_t kSortSmall = 4096;

struct SortArgs {
  const void* index;
  int64_t rows, segment;  // rows of a warp
  int groups, bits;  // bits: of groups + 1
  int32_t* order;
  int32_t* ends;
};

template <class I>
__device__ __forceinline__ int group_of(const SortArgs& a, int64_t row, int64_t end) {
  if (row >= end) return a.groups + 1;  // no row
  const I g = static_cast<const I*>(a.index)[row];
  return g >= 0 && g < (I)a.groups ? (int)g : a.groups;
}

// Lanes whose value of `bits` bits is this lane's: a vote a bit (match.any takes longer the more
// values differ: with it 65536 rows in 64 groups took 2 us more).
__device__ __forceinline__ unsigned equal_lanes(int value, int bits) {
  unsigned same = 0xFFFFFFFFu;
  for (int b = 0; b < bits; ++b) {
    const bool set = (value >> b & 1) != 0;
    const unsigned vote = __ballot_sync(0xFFFFFFFFu, set);
    same &= set ? vote : ~vote;
  }
  return same;
}

// values[0 .. wide): their sums before each, by the whole CTA (at most 1025 values).
template <int THREADS>
__device__ __forceinline__ void sums_before(int* values, int wide, int* warp_sums) {
  constexpr int kEach = (kMaxGroups + THREADS) / THREADS;  // values a thread
  const int at = kEach * threadIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int n[kEach], sum = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    n[i] = at + i < wide ? values[at + i] : 0;
    sum += n[i];
  }
  const int upto = warp_scan_sum(sum, lane);
  __syncthreads();  // (warp_sums may still be read)
  if (lane == 31) warp_sums[warp] = upto;
  __syncthreads();
  int start = upto - sum;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) start += w < warp ? warp_sums[w] : 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    if (at + i < wide) values[at + i] = start;
    start += n[i];
  }
  __syncthreads();
}

// `totals` again in `to`, for their sums.
__device__ __forceinline__ int* totals_copy(const int* totals, int* to, int wide) {
  __syncthreads();
  for (int q = threadIdx.x; q < wide; q += blockDim.x) to[q] = totals[q];
  __syncthreads();
  return to;
}

template <int C>
struct SortShape {
  static constexpr int kWarps = C > 1 ? 16 : 32, kThreads = 32 * kWarps;
  static constexpr int kLocal = kWarps * 32 * kSortAhead;  // rows of a CTA put in order locally
  static constexpr int kMostBytes = (kWarps + 3) * (kMaxGroups + 1) * 4 + kLocal * 6;
};

template <class I, int C>
__global__ void __launch_bounds__(SortShape<C>::kThreads, 1) sort_rows_kernel(const SortArgs a) {
  constexpr int kSortWarps = SortShape<C>::kWarps, kSortThreads = SortShape<C>::kThreads;
  constexpr int kSortLocal = SortShape<C>::kLocal;
  extern __shared__ int counts[];  // [warp][group], group `groups`: rows of none
  __shared__ int sums[kSortWarps];
  const int wide = a.groups + 1, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int* const totals = counts + kSortWarps * wide;  // of this CTA
  int* const before = totals + wide;               // of the CTAs before it
  int* const all = before + wide;                  // of all, then their sums
  const int rank = C > 1 ? (int)cg::this_cluster().block_rank() : 0;
  int* const mine = counts + warp * wide;
  for (int i = threadIdx.x; i < kSortWarps * wide; i += kSortThreads) counts[i] = 0;
  __syncthreads();

  const int64_t first = min(((int64_t)rank * kSortWarps + warp) * a.segment, a.rows);
  const int64_t end = min(first + a.segment, a.rows);
  int g[kSortAhead];  // the groups of the batches at hand: for short segments, of all
  for (int64_t r = first; r < end; r += 32 * kSortAhead) {
#pragma unroll
    for (int i = 0; i < kSortAhead; ++i) g[i] = group_of<I>(a, r + 32 * i + lane, end);
#pragma unroll
    for (int i = 0; i < kSortAhead; ++i)
      if (g[i] < wide) atomicAdd(mine + g[i], 1);
  }
  __syncthreads();
  // counts of the warps before, a warp to a group
  for (int q = warp; q < wide; q += kSortWarps) {
    int* const at = counts + (lane < kSortWarps ? lane : 0) * wide + q;
    const int n = lane < kSortWarps ? *at : 0, upto = warp_scan_sum(n, lane);
    __syncwarp();
    if (lane < kSortWarps) *at = upto - n;
    if (lane == 31) totals[q] = upto;
  }
  if constexpr (C > 1) {
    cg::this_cluster().sync();
    for (int q = threadIdx.x; q < wide; q += kSortThreads) {
      int sum = 0, prior = 0;
#pragma unroll
      for (int r = 0; r < C; ++r) {
        const int n = cg::this_cluster().map_shared_rank(totals, r)[q];
        if (r < rank) prior += n;
        sum += n;
      }
      before[q] = prior;
      all[q] = sum;
    }
  } else {
    __syncthreads();
    for (int q = threadIdx.x; q < wide; q += kSortThreads) {
      before[q] = 0;
      all[q] = totals[q];
    }
  }
  __syncthreads();
  // the first place of every group
  sums_before<kSortThreads>(all, wide, sums);
  if (rank == 0) {
    for (int q = threadIdx.x; q < a.groups; q += kSortThreads) a.ends[q] = all[q + 1];
  }
  // (few rows go straight to their places)
  const bool at_hand = a.segment <= 32 * kSortAhead, local = C > 1 && at_hand;
  int* const rows = all + wide;  // local: the CTA's rows in order, and their groups
  uint16_t* const groups = reinterpret_cast<uint16_t*>(rows + kSortLocal);
  if (local) {
    // `before`: from a place among the CTA's rows to the place among all
    for (int q = threadIdx.x; q < wide; q += kSortThreads) before[q] += all[q];
    sums_before<kSortThreads>(totals_copy(totals, all, wide), wide, sums);
    for (int q = threadIdx.x; q < wide; q += kSortThreads) before[q] -= all[q];
    for (int q = warp; q < wide; q += kSortWarps)
      if (lane < kSortWarps) counts[lane * wide + q] += all[q];
  } else {
    for (int q = warp; q < wide; q += kSortWarps)
      if (lane < kSortWarps) counts[lane * wide + q] += all[q] + before[q];
  }
  __syncthreads();

  for (int64_t r = first; r < end; r += 32 * kSortAhead) {
    if (!at_hand) {
#pragma unroll
      for (int i = 0; i < kSortAhead; ++i) g[i] = group_of<I>(a, r + 32 * i + lane, end);
    }
#pragma unroll
    for (int i = 0; i < kSortAhead; ++i) {
      if (r + 32 * i >= end) break;
      const unsigned same = equal_lanes(g[i], a.bits);
      const int place = __popc(same & ((1u << lane) - 1u));
      const bool is_row = g[i] < wide;
      const int base = is_row ? mine[g[i]] : 0;
      __syncwarp();
      if (is_row) {
        const int32_t at = (int32_t)(r + 32 * i + lane);
        if (local) {
          rows[base + place] = at;
          groups[base + place] = (uint16_t)g[i];
        } else {
          a.order[base + place] = at;
        }
        if (place == 0) mine[g[i]] = base + __popc(same);
      }
      __syncwarp();
    }
  }
  if (local) {
    __syncthreads();
    const int64_t mine0 = min((int64_t)rank * kSortWarps * a.segment, a.rows);
    const int count = (int)(min(mine0 + kSortWarps * a.segment, a.rows) - mine0);
    for (int i = threadIdx.x; i < count; i += kSortThreads) a.order[i + before[groups[i]]] = rows[i];
  }
  // no CTA leaves while others may still read its totals
  if constexpr (C > 1) cg::this_cluster().sync();
}

template <class I, int C>
int launch_sort(SortArgs& a, cudaStream_t stream) {
  const auto kernel = &sort_rows_kernel<I, C>;
  using S = SortShape<C>;
  int resident = 0;
  if (int rc = prepare_kernel(reinterpret_cast<const void*>(kernel), 1, S::kThreads, S::kMostBytes,
                              &resident))
    return rc;
  if (C > 8) {
    // (an attribute of the kernel; set again it costs half a microsecond)
    const cudaError_t e =
        cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return cuda_fail(e, "srs_group_rows");
  }
  const int64_t warps = (int64_t)C * S::kWarps;
  a.segment = ((a.rows + warps - 1) / warps + 31) / 32 * 32;
  const bool local = C > 1 && a.segment <= 32 * kSortAhead;
  const size_t bytes =
      (size_t)(S::kWarps + 3) * (a.groups + 1) * sizeof(int) + (local ? S::kLocal * 6 : 0);
  cudaLaunchConfig_t config{};
  cudaLaunchAttribute cluster{};
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = C;
  cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
  config.gridDim = dim3(C);
  config.blockDim = dim3(S::kThreads);
  config.dynamicSmemBytes = bytes;
  config.stream = stream;
  config.attrs = &cluster;
  config.numAttrs = C > 1 ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&config, kernel, static_cast<const SortArgs&>(a));
  return e == cudaSuccess ? SRS_OK : cuda_fail(e, "srs_group_rows launch");
}

}  // namespace
}  // namespace srs

extern "C" int srs_group_rows(const void* index, int index_bytes, int64_t rows, int groups,
                              int32_t* order, int32_t* ends, void* stream) {
  using namespace srs;
  clear_error();
  if (index_bytes != 4 && index_bytes != 8)
    return fail(SRS_ERR_INVALID_ARGUMENT, "indices are 4 or 8 bytes, got %d", index_bytes);
  if (groups < 1 || groups > kMaxGroups)
    return fail(SRS_ERR_INVALID_ARGUMENT, "groups must be in [1, %d], got %d", kMaxGroups, groups);
  if (rows < 0 || rows > (1ll << 30))
    return fail(SRS_ERR_INVALID_ARGUMENT, "rows must be in [0, 2^30], got %lld", (long long)rows);
  if (ends == nullptr || (rows > 0 && (index == nullptr || order == nullptr)))
    return fail(SRS_ERR_INVALID_ARGUMENT, "null index, order or ends");
  if (reinterpret_cast<uintptr_t>(index) % index_bytes != 0 ||
      reinterpret_cast<uintptr_t>(order) % 4 != 0 || reinterpret_cast<uintptr_t>(ends) % 4 != 0)
    return fail(SRS_ERR_INVALID_ARGUMENT, "index, order or ends is not element aligned");
  if (int rc = check_device()) return rc;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  SortArgs a{index, rows, 0, groups, 1, order, ends};
  while ((groups + 1) >> a.bits != 0) ++a.bits;
  const bool small = rows <= kSortSmall;
  return index_bytes == 4
             ? (small ? launch_sort<int32_t, 1>(a, st) : launch_sort<int32_t, kSortCluster>(a, st))
             : (small ? launch_sort<int64_t, 1>(a, st) : launch_sort<int64_t, kSortCluster>(a, st));
}
