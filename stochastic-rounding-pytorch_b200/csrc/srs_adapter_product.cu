// The large FP8 product with low-rank adapters added to its sums:
//
//   D[order[i], :] = A[i, :] W^T + H_a[i, :] U_a^T       a: the adapter of row i
//
// A and H have the tokens in their adapters' order, D in the batch's.  A tile runs its FP8 slices
// and then, for every adapter with rows in it, one slice of 16-bit products for ranks up to 32
// (two for every 64 above), H as a pair of 16-bit numbers, so that the sum stays FP32 all through
// and the result is rounded once.  These MMAs write the adapter's own rows of the accumulator alone:
// what other adapters' matrices hold, infinities and NaN too, never reaches a token.  At rank 16 that is 2 to 3
// slices beside the 32 of k = 4096; adding the adapters' part in a pass of its own took as long
// as the product (4096 tokens, 4096 -> 14336, rank 16: 147 us beside 178).  MMA-bound, then by
// the power limit.
#include "srs_groups.cuh"
#include "srs_host.h"
#include "srs_launch.h"
#include "srs_product.cuh"

namespace srs {
namespace {

struct AdapterProduct {
  CUtensorMap map_a, map_b, map_h, map_u;
  const int32_t* ends;
  const int32_t* order;
  int adapters;
  int m, n, slices, edge;
  TileGrid grid;
  uint32_t instruction_formats, extra_formats;
  const uint8_t* scale_a;
  const uint8_t* scale_b;
  int64_t scale_a_pitch, scale_b_pitch;
  int scale_b_shift;
  char* out;
  int format;
  int rank, extra_slices, rest_at;
  const int32_t* exponents;  // of FP16 pairs, one a row (null: BF16)
  bool rows_inner;
  unsigned int* status_at;
};

// The adapters with tokens, in order.
struct AdapterPlan {
  int start[kMaxGroups + 1];  // first row of each; behind the last, the end of all
  int group[kMaxGroups];
  int count;
};

__device__ __forceinline__ void plan_adapters(AdapterPlan& p, const int32_t* ends, int adapters,
                                              int rows) {
  const int lane = threadIdx.x & 31;
  const EndsAhead ahead(ends, adapters, lane);
  int carry = 0, count = 0;
  for (int base = 0; base < adapters; base += 32) {
    int start, end;
    group_span(ends, ahead, adapters, rows, base, lane, &carry, &start, &end);
    const unsigned some = __ballot_sync(0xFFFFFFFFu, end > start);
    if (end > start) {
      const int at = count + __popc(some & ((1u << lane) - 1u));
      p.start[at] = start;
      p.group[at] = base + lane;
    }
    count += __popc(some);
  }
  if (lane == 0) {
    p.start[count] = carry;
    p.count = count;
  }
}

struct AdapterSource {
  static constexpr bool kExtras = true, kPadded = false;
  const AdapterProduct& w;
  const AdapterPlan& p;
  __device__ int phases() const { return 1; }
  __device__ uint32_t tiles(int) const { return w.grid.rows * w.grid.cols; }
  __device__ uint32_t formats() const { return w.instruction_formats; }
  __device__ uint32_t extra_formats() const { return w.extra_formats; }
  __device__ unsigned int* counter(int) const { return nullptr; }
  __device__ unsigned int* status() const { return w.status_at; }
  __device__ int longest() const { return w.slices; }
  __device__ TileLoad load(int, uint32_t t) const {
    int row, col;
    w.grid.at(t, &row, &col);
    TileLoad l{};
    l.map_a = &w.map_a;
    l.map_b = &w.map_b;
    l.row0 = row * w.edge;
    l.col0 = col * w.edge;
    l.slices = w.slices;
    return l;
  }
  __device__ TileStore store(int, uint32_t t) const {
    int row, col;
    w.grid.at(t, &row, &col);
    TileStore s{};
    s.row0 = row * w.edge;
    s.col0 = col * w.edge;
    s.m = w.m;
    s.n = w.n;
    s.factor = 1.0f;
    s.out = w.out;
    s.format = w.format;
    s.pitch = w.n;
    s.order = w.order;
    s.exponents = w.exponents;
    return s;
  }
  __device__ BlockScales scales(uint32_t t) const {
    int row, col;
    w.grid.at(t, &row, &col);
    return {w.scale_a,        w.scale_b,    w.scale_a_pitch, w.scale_b_pitch, 0,
            w.scale_b_shift,  row * w.edge, col * w.edge,    w.m,             w.n,
            w.slices,         4,            4,               w.exponents};
  }
  __device__ void spare(int) const {}
  // The first adapter whose rows reach past `row`.
  __device__ __forceinline__ int first_past(int row) const {
    int lo = 0, hi = p.count;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (p.start[mid + 1] > row) hi = mid;
      else lo = mid + 1;
    }
    return lo;
  }
  __device__ ExtraSet extras(uint32_t t) const {
    int row, col;
    w.grid.at(t, &row, &col);
    if (row * w.edge >= p.start[p.count]) return {row, 0, 0};
    const int first = first_past(row * w.edge);
    const int last = first_past(min((row + 1) * w.edge, p.start[p.count]) - 1);
    return {row, first, (last - first + 1) * w.extra_slices};
  }
  __device__ ExtraLoad extra(const ExtraSet& set, int i) const {
    const int row = set.row, row0 = row * w.edge;
    const int ahead = w.extra_slices == 1 ? i : i / w.extra_slices;
    const int adapter = set.first + ahead, slice = i - ahead * w.extra_slices;
    ExtraLoad e;
    e.map_a = &w.map_h;
    e.map_b = &w.map_u;
    e.row_a = (row + adapter) * w.edge;
    e.batch_b = p.group[adapter];
    e.b_rows_inner = w.rows_inner;
    e.k_a = 64 * slice;
    const int chunks = (w.extra_slices + 1) / 2, chunk = slice < chunks ? slice : slice - chunks;
    e.k_b = 64 * chunk;
    e.steps = (min(w.rank - 64 * chunk, 64) + 15) / 16;
    e.again = w.extra_slices == 1 ? w.rest_at / 16 : 0;
    e.first = p.start[adapter] - row0;
    e.end = p.start[adapter + 1] - row0;
    return e;
  }
};

template <int CG>
__global__ void __launch_bounds__(ProductShape<kOperandF8, CG>::kThreads, 1)
adapter_kernel(const __grid_constant__ AdapterProduct w) {
  __shared__ AdapterPlan plan;
  if (threadIdx.x < 32) plan_adapters(plan, w.ends, w.adapters, w.m);
  __syncthreads();
  run_products<kOperandF8, CG, false, false>(AdapterSource{w, plan});
}

template <int CG>
int launch(AdapterProduct& w, cudaStream_t stream) {
  const void* kernel = reinterpret_cast<const void*>(&adapter_kernel<CG>);
  using S = ProductShape<kOperandF8, CG>;
  int resident = 0;
  if (int rc = prepare_kernel(kernel, CG, S::kThreads, S::kSmem, &resident)) return rc;
  const int64_t tiles = (int64_t)w.grid.rows * w.grid.cols;
  return launch_groups(kernel, tiles < resident ? tiles : resident, CG, S::kThreads, S::kSmem,
                       false, &w, stream, "adapter product launch");
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

}  // namespace

int adapter_edge(int64_t tokens, int64_t n, int64_t k) {
  // rough times as for a plain product (launch_block_product)
  const int64_t sms = sm_count(), pairs = sms / 2, slices = ceil_div(k, kSliceBytes);
  const auto tiles = [&](int64_t edge) { return ceil_div(tokens, edge) * ceil_div(n, edge); };
  const double time_small = (350.0 * slices + 2000.0) * (double)ceil_div(tiles(128), sms);
  const double time_large = (512.0 * slices + 5000.0) * (double)ceil_div(tiles(256), pairs);
  return time_large <= time_small ? 256 : 128;
}

int launch_adapter_product(const srs_blocks& rows, const srs_blocks& w, int64_t k,
                           const AdapterCall& a, int edge, void* d, cudaStream_t stream) {
  const int64_t high = ceil_div(rows.rows, edge), across = ceil_div(w.rows, edge);
  if (high * across >= (1ll << 31))
    return fail(SRS_ERR_INVALID_ARGUMENT, "a result of %lld x %lld is too large",
                (long long)rows.rows, (long long)w.rows);
  const PairShape pairs = pair_shape(a.rank);
  AdapterProduct p{};
  const ProductOperand left{reinterpret_cast<const void*>(rows.data), rows.rows, k, rows.pitch, 0,
                            false};
  const ProductOperand right{reinterpret_cast<const void*>(w.data), w.rows, k, w.pitch, 0, false};
  const ProductOperand items{a.pairs, pair_items(rows.rows, a.count, edge) * edge, pairs.pitch,
                             pairs.pitch, 0, false};
  const ProductOperand up{a.up, w.rows, a.rank, a.pitch, a.stride, a.rows_inner};
  if (int rc = encode_operand(left, 1, 1, 128, &p.map_a)) return rc;
  if (int rc = encode_operand(right, 1, 1, 128, &p.map_b)) return rc;
  if (int rc = encode_operand(items, 2, 1, 128, &p.map_h)) return rc;
  if (int rc = encode_operand(up, 2, a.count, 128, &p.map_u)) return rc;
  if (int rc = status_word(&p.status_at)) return rc;
  p.ends = a.ends;
  p.order = a.order;
  p.adapters = a.count;
  p.m = (int)rows.rows;
  p.n = (int)w.rows;
  p.slices = (int)ceil_div(k, kSliceBytes);
  p.edge = edge;
  p.grid = make_grid((uint32_t)high, (uint32_t)across);
  p.instruction_formats = (rows.format == SRS_FMT_E5M2 ? 1u : 0u) << 7 |
                          (w.format == SRS_FMT_E5M2 ? 1u : 0u) << 10;
  p.extra_formats = a.format == SRS_FMT_BF16 ? 1u << 7 | 1u << 10 : 0u;
  p.scale_a = reinterpret_cast<const uint8_t*>(rows.scale);
  p.scale_b = reinterpret_cast<const uint8_t*>(w.scale);
  p.scale_a_pitch = rows.scale_pitch;
  p.scale_b_pitch = w.scale_pitch;
  p.scale_b_shift = w.square ? 7 : 0;
  p.out = static_cast<char*>(d);
  p.format = a.format;
  p.rank = a.rank;
  p.exponents = a.exponents;
  p.extra_slices = pairs.slices;
  p.rest_at = pairs.rest_at;
  p.rows_inner = a.rows_inner;
  return edge == 256 ? launch<2>(p, stream) : launch<1>(p, stream);
}

}  // namespace srs
