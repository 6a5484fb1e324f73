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
#include <cooperative_groups.h>

#include "srs_groups.cuh"
#include "srs_host.h"

namespace srs {
namespace {

namespace cg = cooperative_groups;

constexpr int kSortThreads = 1024, kSortWarps = kSortThreads / 32;
constexpr int kSortAhead = 4;     // batches of a warp loaded together
constexpr int kSortCluster = 8;   // CTAs of a large sort
// One CTA places 65536 rows in 64 batches a warp; from 4096 rows (4 batches) on eight CTAs
// are used.
constexpr int64_t kSortSmall = 4096;

struct SortArgs {
  const void* index;
  int64_t rows, segment;  // rows of a warp
  int groups;
  int32_t* order;
  int32_t* ends;
};

template <class I>
__device__ __forceinline__ int group_of(const SortArgs& a, int64_t row, int64_t end) {
  if (row >= end) return a.groups + 1;  // no row
  const I g = static_cast<const I*>(a.index)[row];
  return g >= 0 && g < (I)a.groups ? (int)g : a.groups;
}

template <class I, int C>
__global__ void __launch_bounds__(kSortThreads, 1) sort_rows_kernel(const SortArgs a) {
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
  for (int64_t r = first; r < end; r += 32 * kSortAhead) {
    int g[kSortAhead];
#pragma unroll
    for (int i = 0; i < kSortAhead; ++i) g[i] = group_of<I>(a, r + 32 * i + lane, end);
#pragma unroll
    for (int i = 0; i < kSortAhead; ++i)
      if (g[i] < wide) atomicAdd(mine + g[i], 1);
  }
  __syncthreads();
  for (int g = threadIdx.x; g < wide; g += kSortThreads) {
    int sum = 0;
    for (int w = 0; w < kSortWarps; ++w) {
      const int n = counts[w * wide + g];
      counts[w * wide + g] = sum;
      sum += n;
    }
    totals[g] = sum;
  }
  if constexpr (C > 1) {
    cg::this_cluster().sync();
    for (int g = threadIdx.x; g < wide; g += kSortThreads) {
      int sum = 0, prior = 0;
#pragma unroll
      for (int r = 0; r < C; ++r) {
        const int n = cg::this_cluster().map_shared_rank(totals, r)[g];
        if (r < rank) prior += n;
        sum += n;
      }
      before[g] = prior;
      all[g] = sum;
    }
  } else {
    __syncthreads();
    for (int g = threadIdx.x; g < wide; g += kSortThreads) {
      before[g] = 0;
      all[g] = totals[g];
    }
  }
  __syncthreads();
  // the first place of every group: at most 1025 numbers, two a thread
  const int at = 2 * threadIdx.x;
  const int n0 = at < wide ? all[at] : 0, n1 = at + 1 < wide ? all[at + 1] : 0;
  const int pair = warp_scan_sum(n0 + n1, lane);
  if (lane == 31) sums[warp] = pair;
  __syncthreads();
  if (warp == 0) sums[lane] = warp_scan_sum(sums[lane], lane);
  __syncthreads();
  const int start = pair - n0 - n1 + (warp > 0 ? sums[warp - 1] : 0);
  if (at < wide) all[at] = start;
  if (at + 1 < wide) all[at + 1] = start + n0;
  if (rank == 0) {
    if (at < a.groups) a.ends[at] = start + n0;
    if (at + 1 < a.groups) a.ends[at + 1] = start + n0 + n1;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < kSortWarps * wide; i += kSortThreads)
    counts[i] += all[i % wide] + before[i % wide];
  __syncthreads();

  for (int64_t r = first; r < end; r += 32 * kSortAhead) {
    int g[kSortAhead];
#pragma unroll
    for (int i = 0; i < kSortAhead; ++i) g[i] = group_of<I>(a, r + 32 * i + lane, end);
#pragma unroll
    for (int i = 0; i < kSortAhead; ++i) {
      const unsigned same = __match_any_sync(0xFFFFFFFFu, g[i]);
      const int place = __popc(same & ((1u << lane) - 1u));
      const bool is_row = g[i] < wide;
      const int base = is_row ? mine[g[i]] : 0;
      __syncwarp();
      if (is_row) {
        a.order[base + place] = (int32_t)(r + 32 * i + lane);
        if (place == 0) mine[g[i]] = base + __popc(same);
      }
      __syncwarp();
    }
  }
  // no CTA leaves while others may still read its totals
  if constexpr (C > 1) cg::this_cluster().sync();
}

template <class I, int C>
cudaError_t launch_sort(SortArgs& a, cudaStream_t stream) {
  const auto kernel = &sort_rows_kernel<I, C>;
  const int64_t warps = (int64_t)C * kSortWarps;
  a.segment = ((a.rows + warps - 1) / warps + 31) / 32 * 32;
  const size_t bytes = (size_t)(kSortWarps + 3) * (a.groups + 1) * sizeof(int);
  if (bytes > 40 * 1024) {
    const cudaError_t e =
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e != cudaSuccess) return e;
  }
  cudaLaunchConfig_t config{};
  cudaLaunchAttribute cluster{};
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = C;
  cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
  config.gridDim = dim3(C);
  config.blockDim = dim3(kSortThreads);
  config.dynamicSmemBytes = bytes;
  config.stream = stream;
  config.attrs = &cluster;
  config.numAttrs = C > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&config, kernel, a);
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
  SortArgs a{index, rows, 0, groups, order, ends};
  const bool small = rows <= kSortSmall;
  const cudaError_t e =
      index_bytes == 4
          ? (small ? launch_sort<int32_t, 1>(a, st) : launch_sort<int32_t, kSortCluster>(a, st))
          : (small ? launch_sort<int64_t, 1>(a, st) : launch_sort<int64_t, kSortCluster>(a, st));
  return e == cudaSuccess ? SRS_OK : cuda_fail(e, "srs_group_rows launch");
}
