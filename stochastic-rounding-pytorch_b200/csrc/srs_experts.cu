// FP8 block products whose rows are in groups, one weight a group (a mixture of experts):
//
//   forward, dx:  D[i, :] = A[i, :] W_e^T           for the rows i of group e
//   dW:           D_e = A_e^T B_e                   sums over the rows of group e
//
// The host does not know where groups end, so a grid is sized by a bound and every CTA finds
// its tiles from the ends.  Three forms:
//
// * Few rows a group (thin, srs_thin.cuh): the weights' bytes bound it.  A CTA takes 128 rows of
//   one group's weight and up to 64 of its rows.
// * Ragged rows: the tiles of the large product, counted from each group's first row.  A tile
//   that reaches past its group's end loads rows of the next group and does not store them.
// * Ragged sums: blocks of 128 rows are counted from the group's first one as well, so that a
//   group's sum is a run of whole slices of k of the transposed copies and its scales are its
//   own.  Those lie in words of four blocks, a word of every row one after the other: a warp then
//   reads its 128 rows in whole lines.  Groups without rows have no tiles; their zeros are written by the warp that has no role
//   in a product, as are the zeros of rows without a group.
//
// MMA-bound when groups are large (and then by the power limit), by the weights' bytes when they
// are small.
#include "srs_groups.cuh"
#include "srs_host.h"
#include "srs_launch.h"
#include "srs_product.cuh"
#include "srs_thin.cuh"

namespace srs {
namespace {

struct ExpertProduct {
  CUtensorMap map_a, map_b;
  const int32_t* ends;
  int experts;
  int rows;        // of A and D (ragged rows), of what is summed (ragged sums)
  int m, n;        // ragged sums: size of D_e; ragged rows: n columns of D
  int slices;      // ragged rows
  int edge;        // of a tile
  int tile_cols;   // tiles across D
  int tile_rows;   // ragged sums: tiles down D_e
  uint32_t instruction_formats;
  const uint8_t* scale_a;
  const uint8_t* scale_b;
  int64_t scale_a_pitch, scale_b_pitch, scale_b_expert;
  int scale_b_shift;
  char* out;
  int format;
  unsigned int* status_at;
};

// Where groups are, in shared memory: of group e its first row, and the tiles (ragged sums:
// slices, words of scales, groups with rows) before it.
struct GroupPlan {
  int start[kMaxGroups + 1];
  int before[kMaxGroups + 1];
  int quads[kMaxGroups + 1];
  int active[kMaxGroups + 1];  // active[i]: the i-th group with rows
  int count;                   // of groups with rows
};

// By the first warp; `edge` rows a tile.
template <bool SUMS>
__device__ __forceinline__ void plan_groups(GroupPlan& p, const int32_t* ends, int groups, int rows,
                                            int edge) {
  const int lane = threadIdx.x & 31;
  const EndsAhead ahead(ends, groups, lane);
  int carry = 0, tiles_before = 0, quads_before = 0, count = 0;
  for (int base = 0; base < groups; base += 32) {
    const int g = base + lane;
    int start, end;
    group_span(ends, ahead, groups, rows, base, lane, &carry, &start, &end);
    const int tiles = (end - start + edge - 1) / edge;
    const int upto = tiles_before + warp_scan_sum(tiles, lane);
    if (g < groups) {
      p.start[g] = start;
      p.before[g] = upto - tiles;
    }
    tiles_before = __shfl_sync(0xFFFFFFFFu, upto, 31);
    if (SUMS) {
      const int quads = (tiles + 3) & ~3;
      const int quads_upto = quads_before + warp_scan_sum(quads, lane);
      if (g < groups) p.quads[g] = quads_upto - quads;
      quads_before = __shfl_sync(0xFFFFFFFFu, quads_upto, 31);
      const unsigned some = __ballot_sync(0xFFFFFFFFu, tiles > 0);
      if (tiles > 0) p.active[count + __popc(some & ((1u << lane) - 1u))] = g;
      count += __popc(some);
    }
  }
  if (lane == 0) {
    p.start[groups] = carry;
    p.before[groups] = tiles_before;
    p.count = count;
  }
}

// Zeros over `count` elements of `size` bytes from `out` on, by one warp of every CTA.
__device__ __forceinline__ void spread_zeros(char* out, int64_t count, int size, int lane) {
  char* const end = out + count * size;
  const int64_t step = (int64_t)gridDim.x * 32 * 16;
  char* const first = reinterpret_cast<char*>((reinterpret_cast<uint64_t>(out) + 15) & ~15ull);
  if (blockIdx.x == 0) {
    // what lies before the first whole 16 bytes, by elements
    for (char* p = out + lane * size; p < first && p < end; p += 32 * size) {
      if (size == 4) *reinterpret_cast<uint32_t*>(p) = 0u;
      else *reinterpret_cast<uint16_t*>(p) = 0;
    }
  }
  for (char* p = first + ((int64_t)blockIdx.x * 32 + lane) * 16; p < end; p += step) {
    if (p + 16 <= end) {
      *reinterpret_cast<uint4*>(p) = make_uint4(0u, 0u, 0u, 0u);
    } else {
      for (char* q = p; q < end; q += 2) *reinterpret_cast<uint16_t*>(q) = 0;
    }
  }
}

struct RowSource {
  static constexpr bool kExtras = false, kPadded = false;
  const ExpertProduct& w;
  const GroupPlan& p;
  struct At {
    int expert, row, col;  // tile row and column inside the expert
  };
  // Tiles of an expert in bands of 8 tile rows, column by column within a band.
  __device__ __forceinline__ At at(uint32_t t) const {
    int lo = 0, hi = w.experts - 1;  // the last expert with tiles before it <= t
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if ((uint32_t)p.before[mid] * (uint32_t)w.tile_cols <= t) lo = mid;
      else hi = mid - 1;
    }
    const uint32_t rows = (uint32_t)(p.before[lo + 1] - p.before[lo]);
    const uint32_t j = t - (uint32_t)p.before[lo] * (uint32_t)w.tile_cols;
    const uint32_t band = j / (8u * (uint32_t)w.tile_cols);
    const uint32_t in = j - band * 8u * (uint32_t)w.tile_cols, high = min(rows - 8u * band, 8u);
    return {lo, (int)(8u * band + in % high), (int)(in / high)};
  }
  __device__ int phases() const { return 1; }
  __device__ uint32_t tiles(int) const {
    return (uint32_t)p.before[w.experts] * (uint32_t)w.tile_cols;
  }
  __device__ uint32_t formats() const { return w.instruction_formats; }
  __device__ unsigned int* counter(int) const { return nullptr; }
  __device__ unsigned int* status() const { return w.status_at; }
  __device__ int longest() const { return w.slices; }
  __device__ TileLoad load(int, uint32_t t) const {
    const At i = at(t);
    TileLoad l{};
    l.map_a = &w.map_a;
    l.map_b = &w.map_b;
    l.row0 = p.start[i.expert] + i.row * w.edge;
    l.col0 = i.expert * w.n + i.col * w.edge;
    l.slices = w.slices;
    return l;
  }
  __device__ TileStore store(int, uint32_t t) const {
    const At i = at(t);
    TileStore s{};
    s.row0 = p.start[i.expert] + i.row * w.edge;
    s.col0 = i.col * w.edge;
    s.m = p.start[i.expert + 1];
    s.n = w.n;
    s.factor = 1.0f;
    s.out = w.out;
    s.format = w.format;
    s.pitch = w.n;
    return s;
  }
  __device__ BlockScales scales(uint32_t t) const {
    const At i = at(t);
    return {w.scale_a,
            w.scale_b + i.expert * w.scale_b_expert,
            w.scale_a_pitch,
            w.scale_b_pitch,
            0,
            w.scale_b_shift,
            p.start[i.expert] + i.row * w.edge,
            i.col * w.edge,
            w.rows,
            w.n,
            w.slices};
  }
  __device__ void spare(int lane) const {
    const int64_t from = (int64_t)p.start[w.experts] * w.n;
    const int size = w.format == SRS_FMT_F32 ? 4 : 2;
    spread_zeros(w.out + from * size, (int64_t)w.rows * w.n - from, size, lane);
  }
};

struct SumSource {
  static constexpr bool kExtras = false, kPadded = true;
  const ExpertProduct& w;
  const GroupPlan& p;
  struct At {
    int expert, row, col;
  };
  // Group after group: a tile of every group in turn, so that short sums (bound by the bytes of
  // their results) run beside long ones, was slower (8192 rows in 8 uneven groups, 14336 x 4096
  // each: 629 us instead of 559), as the groups' operands then share the L2.
  __device__ __forceinline__ At at(uint32_t t) const {
    const uint32_t each = (uint32_t)w.tile_rows * (uint32_t)w.tile_cols, i = t / each;
    const uint32_t j = t - i * each;
    const uint32_t band = j / (8u * (uint32_t)w.tile_cols);
    const uint32_t in = j - band * 8u * (uint32_t)w.tile_cols;
    const uint32_t high = min((uint32_t)w.tile_rows - 8u * band, 8u);
    return {p.active[i], (int)(8u * band + in % high), (int)(in / high)};
  }
  __device__ __forceinline__ int slices(int expert) const {
    return p.before[expert + 1] - p.before[expert];
  }
  __device__ int phases() const { return 1; }
  __device__ uint32_t tiles(int) const {
    return (uint32_t)p.count * (uint32_t)w.tile_rows * (uint32_t)w.tile_cols;
  }
  __device__ uint32_t formats() const { return w.instruction_formats; }
  __device__ unsigned int* counter(int) const { return nullptr; }
  __device__ unsigned int* status() const { return w.status_at; }
  __device__ int longest() const { return w.rows / kSliceBytes + 1; }
  __device__ TileLoad load(int, uint32_t t) const {
    const At i = at(t);
    TileLoad l{};
    l.map_a = &w.map_a;
    l.map_b = &w.map_b;
    l.row0 = i.row * w.edge;
    l.col0 = i.col * w.edge;
    l.slices = slices(i.expert);
    l.k0 = p.before[i.expert] * kSliceBytes;
    return l;
  }
  __device__ TileStore store(int, uint32_t t) const {
    const At i = at(t);
    TileStore s{};
    s.row0 = i.row * w.edge;
    s.col0 = i.col * w.edge;
    s.m = w.m;
    s.n = w.n;
    s.factor = 1.0f;
    s.out = w.out + (int64_t)i.expert * w.m * w.n * (w.format == SRS_FMT_F32 ? 4 : 2);
    s.format = w.format;
    s.pitch = w.n;
    return s;
  }
  __device__ BlockScales scales(uint32_t t) const {
    const At i = at(t);
    // words of four scales, all rows of one k after the other
    const int64_t a_quad = 4ll * w.m, b_quad = 4ll * w.n, quad = p.quads[i.expert] >> 2;
    return {w.scale_a + quad * a_quad,
            w.scale_b + quad * b_quad,
            4,
            4,
            0,
            0,
            i.row * w.edge,
            i.col * w.edge,
            w.m,
            w.n,
            slices(i.expert),
            a_quad,
            b_quad};
  }
  __device__ void spare(int lane) const {
    const int size = w.format == SRS_FMT_F32 ? 4 : 2;
    const int64_t each = (int64_t)w.m * w.n;
    for (int e = 0; e < w.experts; ++e)
      if (slices(e) == 0) spread_zeros(w.out + e * each * size, each, size, lane);
  }
};

template <int CG, bool SUMS>
__global__ void __launch_bounds__(ProductShape<kOperandF8, CG>::kThreads, 1)
expert_kernel(const __grid_constant__ ExpertProduct w) {
  __shared__ GroupPlan plan;
  if (threadIdx.x < 32)
    plan_groups<SUMS>(plan, w.ends, w.experts, w.rows, SUMS ? kSliceBytes : w.edge);
  __syncthreads();
  if constexpr (SUMS)
    run_products<kOperandF8, CG, false, false>(SumSource{w, plan});
  else
    run_products<kOperandF8, CG, false, false>(RowSource{w, plan});
}

template <int CG, bool SUMS>
int launch_experts(ExpertProduct& w, int64_t tiles, cudaStream_t stream) {
  const void* kernel = reinterpret_cast<const void*>(&expert_kernel<CG, SUMS>);
  using S = ProductShape<kOperandF8, CG>;
  int resident = 0;
  if (int rc = prepare_kernel(kernel, CG, S::kThreads, S::kSmem, &resident)) return rc;
  return launch_groups(kernel, tiles < resident ? tiles : resident, CG, S::kThreads, S::kSmem,
                       false, &w, stream, "expert product launch");
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

int expert_map(const srs_blocks& b, int64_t k, CUtensorMap* map) {
  const ProductOperand o{reinterpret_cast<const void*>(b.data), b.rows, k, b.pitch, 0, false};
  return encode_operand(o, 1, 1, 128, map);
}

uint32_t formats_of(const srs_blocks& a, const srs_blocks& b) {
  return (a.format == SRS_FMT_E5M2 ? 1u : 0u) << 7 | (b.format == SRS_FMT_E5M2 ? 1u : 0u) << 10;
}

int launch_ragged_rows(const srs_blocks& a, const srs_blocks& w, int experts, const int32_t* ends,
                       int64_t k, void* d, int d_format, cudaStream_t stream) {
  const int64_t n = w.rows / experts, slices = ceil_div(k, kSliceBytes);
  const int64_t busy = experts < a.rows ? experts : a.rows;
  // As for one product (launch_block_product); of every group with rows half a tile is
  // counted on top, as its last tile is half full in the mean.
  const int64_t sms = sm_count(), pairs = sms / 2;
  const auto rounds = [&](int64_t edge, int64_t at_once) {
    const double tiles = ((double)a.rows / edge + 0.5 * busy) * ceil_div(n, edge);
    return tiles < at_once ? 1.0 : tiles / at_once;
  };
  const double time_small = (350.0 * slices + 2000.0) * rounds(128, sms);
  const double time_large = (512.0 * slices + 5000.0) * rounds(256, pairs);
  const int cg = time_large <= time_small ? 2 : 1;
  ExpertProduct p{};
  p.edge = 128 * cg;
  p.tile_cols = (int)ceil_div(n, p.edge);
  const int64_t tiles = most_group_tiles(a.rows, experts, p.edge) * p.tile_cols;
  if (tiles >= (1ll << 31))
    return fail(SRS_ERR_INVALID_ARGUMENT, "a result of %lld x %lld is too large",
                (long long)a.rows, (long long)n);
  if (int rc = expert_map(a, k, &p.map_a)) return rc;
  if (int rc = expert_map(w, k, &p.map_b)) return rc;
  if (int rc = status_word(&p.status_at)) return rc;
  p.ends = ends;
  p.experts = experts;
  p.rows = (int)a.rows;
  p.n = (int)n;
  p.slices = (int)slices;
  p.instruction_formats = formats_of(a, w);
  p.scale_a = reinterpret_cast<const uint8_t*>(a.scale);
  p.scale_b = reinterpret_cast<const uint8_t*>(w.scale);
  p.scale_a_pitch = a.scale_pitch;
  p.scale_b_pitch = w.scale_pitch;
  p.scale_b_shift = w.square ? 7 : 0;
  p.scale_b_expert = (w.square ? ceil_div(n, 128) : n) * w.scale_pitch;
  p.out = static_cast<char*>(d);
  p.format = d_format;
  return cg == 2 ? launch_experts<2, false>(p, tiles, stream)
                 : launch_experts<1, false>(p, tiles, stream);
}

int check_weights(const srs_blocks* w, int experts, const int32_t* ends, int64_t k) {
  if (int rc = check_groups(ends, experts)) return rc;
  if (int rc = check_operand("w", w, k)) return rc;
  if (w->rows % experts != 0)
    return fail(SRS_ERR_INVALID_ARGUMENT, "w has %lld rows, not a multiple of %d experts",
                (long long)w->rows, experts);
  if (k < 0 || k > (1ll << 30))
    return fail(SRS_ERR_INVALID_ARGUMENT, "k must be in [0, 2^30], got %lld", (long long)k);
  return SRS_OK;
}

int check_result(const void* d, int d_format) {
  if (d_format < SRS_FMT_F32 || d_format > SRS_FMT_F16)
    return fail(SRS_ERR_INVALID_ARGUMENT, "unsupported result format %d", d_format);
  if (d == nullptr || reinterpret_cast<uintptr_t>(d) % fmt_bytes(d_format) != 0)
    return fail(SRS_ERR_INVALID_ARGUMENT, "null or misaligned result pointer");
  return SRS_OK;
}

int zeros(void* d, int64_t count, int format, cudaStream_t stream) {
  const cudaError_t e = cudaMemsetAsync(d, 0, (size_t)(count * fmt_bytes(format)), stream);
  return e == cudaSuccess ? SRS_OK : cuda_fail(e, "zeros of an empty sum");
}

// Checked operands; `overlap`: the quantisation of `a` is the kernel ahead.
int expert_matmul(const srs_blocks& a, const srs_blocks& w, int experts, const int32_t* ends,
                  int64_t k, void* d, int d_format, bool overlap, cudaStream_t stream) {
  const int64_t busy = experts < a.rows ? experts : a.rows;
  // Up to 32 rows a group in the mean the weights' bytes bound the product.  Both forms, thin first, us
  // a call: 64 experts, 2048 -> 1024, of 16 rows each 37 and 43, of 32 43.3 and 44.0, of 40 47.4 and
  // 45.5, of 64 57 and 49; 8 experts, 4096 -> 14336, 91 and 107, 98 and 109, 103 and 110, 124 and 111.
  if (a.rows <= 32 * busy)
    return launch_expert_thin(a, w, experts, ends, k, d, d_format, overlap, stream);
  return launch_ragged_rows(a, w, experts, ends, k, d, d_format, stream);
}

}  // namespace
}  // namespace srs

using namespace srs;

extern "C" int srs_expert_matmul(const srs_blocks* a, const srs_blocks* w, int experts,
                                 const int32_t* ends, int64_t k, void* d, int d_format,
                                 void* stream) {
  clear_error();
  if (int rc = check_weights(w, experts, ends, k)) return rc;
  if (int rc = check_operand("a", a, k)) return rc;
  if (a->square) return fail(SRS_ERR_INVALID_ARGUMENT, "rows in groups have blocks of 1 x 128");
  if (a->rows == 0 || w->rows == 0) return SRS_OK;
  if (int rc = check_result(d, d_format)) return rc;
  if (int rc = check_device()) return rc;
  if (int rc = check_products()) return rc;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (k == 0) return zeros(d, a->rows * (w->rows / experts), d_format, st);
  return expert_matmul(*a, *w, experts, ends, k, d, d_format, false, st);
}

extern "C" int srs_expert_linear(const void* x, int x_format, int64_t rows, int64_t k,
                                 int64_t x_pitch, int block_format, const srs_blocks* w,
                                 int experts, const int32_t* ends, void* d, void* workspace,
                                 int64_t workspace_bytes, void* stream) {
  clear_error();
  if (int rc = check_weights(w, experts, ends, k)) return rc;
  if (rows < 0) return fail(SRS_ERR_INVALID_ARGUMENT, "negative size (%lld)", (long long)rows);
  if (rows == 0 || w->rows == 0) return SRS_OK;
  if (int rc = check_result(d, x_format)) return rc;
  if (workspace_bytes < srs_linear_workspace(rows, k) ||
      (k > 0 && (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 16 != 0)))
    return fail(SRS_ERR_INVALID_ARGUMENT,
                "workspace of %lld bytes, %lld needed at a 16-byte aligned address",
                (long long)workspace_bytes, (long long)srs_linear_workspace(rows, k));
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (k == 0) {
    if (int rc = check_device()) return rc;
    return zeros(d, rows * (w->rows / experts), x_format, st);
  }
  srs_blocks a{};
  a.data = reinterpret_cast<uint64_t>(workspace);
  a.rows = rows;
  a.pitch = (k + 15) / 16 * 16;
  a.scale = a.data + (uint64_t)(rows * a.pitch);
  a.scale_pitch = ceil_div(k, 128);
  a.format = block_format;
  QuantizeCall q{x, x_format, rows, k, x_pitch, block_format, SRS_RULE_NEAREST, false, 0u, 0u};
  q.copy = {a.data, a.scale, a.pitch, a.scale_pitch, 0, 0};
  q.for_product = true;
  if (int rc = quantize(q, st)) return rc;
  return expert_matmul(a, *w, experts, ends, k, d, x_format, true, st);
}

extern "C" int srs_expert_gradient(const srs_blocks* a_t, const srs_blocks* b_t, int64_t rows,
                                   int experts, const int32_t* ends, void* d, int d_format,
                                   void* stream) {
  clear_error();
  if (int rc = check_groups(ends, experts)) return rc;
  if (rows < 0 || rows > kMaxQuantizedRows)
    return fail(SRS_ERR_INVALID_ARGUMENT, "rows must be in [0, %lld], got %lld",
                (long long)kMaxQuantizedRows, (long long)rows);
  const int64_t columns = srs_group_columns(rows, experts);
  for (const srs_blocks* b : {a_t, b_t}) {
    if (int rc = check_operand(b == a_t ? "a_t" : "b_t", b, columns)) return rc;
    if (rows == 0) continue;
    if (b->square || b->scale_pitch < srs_group_scales(rows, experts) || b->scale % 4 != 0)
      return fail(SRS_ERR_INVALID_ARGUMENT,
                  "operand %s: not the transposed copy of rows in groups, or its scales' address "
                  "is no multiple of 4",
                  b == a_t ? "a_t" : "b_t");
  }
  const int64_t m = a_t->rows, n = b_t->rows;
  if (m == 0 || n == 0) return SRS_OK;
  if (int rc = check_result(d, d_format)) return rc;
  if (int rc = check_device()) return rc;
  if (int rc = check_products()) return rc;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (rows == 0) return zeros(d, experts * m * n, d_format, st);
  const int64_t busy = experts < rows ? experts : rows;
  const int64_t sms = sm_count(), pairs = sms / 2, slices = ceil_div(rows / busy + 64, kSliceBytes);
  const auto tiles_of = [&](int64_t edge) { return ceil_div(m, edge) * ceil_div(n, edge); };
  const double time_small =
      (350.0 * slices + 2000.0) * (double)ceil_div(busy * tiles_of(128), sms);
  const double time_large =
      (512.0 * slices + 5000.0) * (double)ceil_div(busy * tiles_of(256), pairs);
  const int cg = time_large <= time_small ? 2 : 1;
  ExpertProduct p{};
  p.edge = 128 * cg;
  if (busy * tiles_of(p.edge) >= (1ll << 31))
    return fail(SRS_ERR_INVALID_ARGUMENT, "results of %lld x %lld are too large", (long long)m,
                (long long)n);
  if (int rc = expert_map(*a_t, columns, &p.map_a)) return rc;
  if (int rc = expert_map(*b_t, columns, &p.map_b)) return rc;
  if (int rc = status_word(&p.status_at)) return rc;
  p.ends = ends;
  p.experts = experts;
  p.rows = (int)rows;
  p.m = (int)m;
  p.n = (int)n;
  p.tile_rows = (int)ceil_div(m, p.edge);
  p.tile_cols = (int)ceil_div(n, p.edge);
  p.instruction_formats = formats_of(*a_t, *b_t);
  p.scale_a = reinterpret_cast<const uint8_t*>(a_t->scale);
  p.scale_b = reinterpret_cast<const uint8_t*>(b_t->scale);
  p.out = static_cast<char*>(d);
  p.format = d_format;
  // (without a group with rows a grid of one still writes the zeros)
  const int64_t tiles = busy * tiles_of(p.edge);
  return cg == 2 ? launch_experts<2, true>(p, tiles, st) : launch_experts<1, true>(p, tiles, st);
}
