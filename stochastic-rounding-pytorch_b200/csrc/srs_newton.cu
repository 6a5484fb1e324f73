// Orthogonalised updates: Newton-Schulz steps on the tensor cores, and the
// momentum step whose update they orthogonalise (Muon).
//
//   X_0 = V / (|V|_F + eps)
//   repeat: G = X X^T;  P = a I + b G + c G^2;  X = P X      (smaller side inside)
//
// V is a tensor (srs_orthogonalize) or, for an optimizer step, computed from the
// gradient and the stored momentum (srs_muon_multi):
//   u' = u * momentum + g;  V = nesterov ? u' * momentum + g : u'
// u' is stored in its format; p' = p * decay + step * X.
//
// Matrices taller than wide use G = X^T X and X P instead, with the same storage:
// the products read either operand with k or with its row index contiguous, so
// nothing is ever transposed.
//
// Number formats.  G, P and X are held in FP16, accumulated in FP32: 11 significant bits
// where BF16 would keep 8.  Errors of G and P act on X from the side of its shorter
// dimension: they turn directions that X has.  Those of X itself are different: they have
// directions that X has not (a gradient of few tokens has few), where P is a I, and a
// step multiplies them by a, five of them by a^5 = 485 (rank 1: 15 % of the result).  So X
// is carried with what its FP16 leaves, in a second FP16 matrix, until the last step, and
// the epilogue of X = P X adds a times that second matrix: P acts as a I where it
// matters, and the product needs no MMA more.  The norms of errors are then 1e-3 to 3e-3 of
// the result's for noise, low ranks and spectra that fall by any power, 6e-3 for a few
// orthogonal rows (restated in FP64 and measured; rounding to BF16 adds 1.7e-3).  At sides of
// ten thousand the truncation below adds to low ranks: rank 2, 8192 x 8192 4.6e-3.
//
// X_0 is held as V * 2^j with a power of two that puts |V * 2^j|_F between 2^14 and 2^15;
// the remaining factor rho enters the first products in FP32.  The norm is summed in FP64,
// so no input in range overflows or vanishes in it.  The later X are held times 2^12, far
// from FP16's smallest numbers.  Where eps dwarfs the norm the X_k are small: while their
// bound |V| / (|V| + eps) * (|a| + |b| + |c|)^k is below 1, they are held times a power of
// two more (at most 2^100) that it leaves room for.  (Singular values up to 15 fit; the default coefficients keep them below
// 1.3.)
//
// Results in FP32 or FP16 hold more digits than that.  For them (SPLIT) every held
// matrix is the sum of two FP16 matrices, what the first leaves of a value in the
// second, and a product of two such is low by high + high by low + high by high: three
// times the MMAs, errors for noise from 4e-6 (128 x 512) to 7e-5 (4096 x 14336).  The
// tensor core truncates its FP32 sums, so errors grow with the sides, and with few
// directions, as above, to more: rank 2 4e-5 (128 x 128), 2.5e-4 (768 x 768), 1.4e-3
// (4096 x 4096), 2.8e-3 (8192 x 8192); FP32 sums rounded to nearest 5e-5 at 768.  So P is held without its
// a I, and the epilogue adds all of a X: shorter sums to truncate (with a I in P: noise
// 9e-5, rank 8 at 768 1.7e-4 instead of 8e-5).  (Sums of the first two steps in parts of
// 512 of k, joined in the epilogue: rank 1 worse, 15 % more time at 4096 x 14336; not kept.)
//
// Three launches: the norm, X_0, and one cooperative grid that runs the 3 * steps
// products of all matrices, whatever their shapes, as phases with a grid-wide meeting
// between them (a launch a product took 7 us each where the products themselves take 1
// to 3).  G and P are symmetric: only tiles on and below the diagonal are computed and
// stored; products read the others from their transposes.
//
// What bounds it: the MMAs and the power they draw for large matrices (4096 x 14336:
// 3.55 ms among other calls, 1.11 PFLOP/s of the 3 m^2 n + m^3 a step needs, 3.35 before X
// had a low part), about 4 us a phase of meeting, first loads and results for small ones
// (768 x 768: 126 us in 15 phases), and the tiles of G alone for long, narrow ones: G has
// one tile for every 128 x 128 of the shorter side, and a tile's sum runs over the whole
// longer side on one CTA or pair.
//
// Reads of V: one for the norm and one for X_0.  For an optimizer step both passes
// compute V from the gradient and the momentum (8 or fewer bytes an element) rather than
// keeping V in FP32 (8 bytes more of traffic and 4 of memory); the second pass stores
// u'.  4096 x 14336 from BF16: 44 us and, with two matrices to write, 62: 3 % of the whole.
#include <cmath>

#include "srs_host.h"
#include "srs_launch.h"
#include "srs_product.cuh"

namespace srs {
namespace {

constexpr int kMaxClasses = SRS_MUON_MAX_CLASSES;
constexpr int kMaxMatrices = SRS_MUON_MAX_MATRICES;
static_assert(kMaxPhases <= kThreads, "one CTA zeroes the counters");
constexpr int kSumChunks = 1024;  // most partial sums of a matrix
constexpr int kPlain = -1;        // source template value: a plain tensor
// G and P are held times 2^8: their small elements (1 / m and less in the first
// steps) then stay among FP16's normal numbers, and eigenvalues up to 255 fit.  (P is held
// times less where the coefficients are larger than that: see hold_of_p.)
constexpr float kHeld = 256.0f;
// X_0 is held with a norm below 2^kTarget, the later X times kHeldX.
constexpr int kTarget = 15;
constexpr float kHeldX = 4096.0f;
constexpr int kFactors = 2 * SRS_NEWTON_MAX_STEPS;  // of a matrix: two a step (G, X)

// A matrix of an optimizer step.
struct MuonMatrix {
  uint64_t param, grad, state;
  uint32_t key, offset, flags, unused;  // key or parameter index; SRS_ROW_* bits
};

// Where the matrices of one shape come from and go to.
struct NewtonSource {
  const void* x;      // plain: the tensor
  int x_format;       // plain: SRS_FMT_F32, SRS_FMT_BF16 or SRS_FMT_F16
  int64_t row_pitch, batch_stride;
  int vec;            // plain: rows start on 16-byte boundaries
  int m, n;           // rows, columns
  uint32_t units;     // vectors of 8 per matrix: m * ceil(n / 8)
  uint32_t row_units;
  int first;          // number of this shape's first matrix among all
  int chunks;         // partial sums of one matrix
  __half* x0;
  int64_t low;        // elements from X_0 to its low part
  int64_t ld, x_elems;
  float* factors;
};

// One launch over the matrices of several shapes (blockIdx.y: the matrix).
struct NewtonPlan {
  NewtonSource source[kMaxClasses];
  MuonMatrix matrix[kMaxMatrices];  // Muon: by place among all matrices
  int classes;
  double* partial;    // kSumChunks for each matrix
  unsigned int* counters;  // of the product grid's phases, set to zero here
  double eps;
  double growth;  // log2(|a| + |b| + |c|), at least 0: of X in a step
  int steps;
  float hold_p;   // P is held times this
  srs_rng rng;
  float momentum;
  int nesterov;
  int u_rule;
};

struct Unit {
  int64_t at;  // element offset of the vector in its matrix
  int row, col, count;
};

__device__ __forceinline__ Unit unit_of(const NewtonSource& s, uint32_t u, int64_t pitch) {
  Unit r;
  r.row = (int)(u / s.row_units);
  r.col = (int)(u - (uint32_t)r.row * s.row_units) * 8;
  r.count = min(8, s.n - r.col);
  r.at = (int64_t)r.row * pitch + r.col;
  return r;
}

// 8 elements of V at `u` (elements beyond the row: zero).  With STORE the new
// momentum is written back as well.
template <int U, bool STORE>
__device__ __forceinline__ void source8(const NewtonPlan& plan, const NewtonSource& s,
                                        const MuonMatrix& row, uint32_t ctr, int batch, uint32_t u,
                                        float (&v)[kVec]) {
  if constexpr (U == kPlain) {
    const Unit w = unit_of(s, u, s.row_pitch);
    const bool vec = s.vec && w.count == 8;
    const int64_t at = (int64_t)batch * s.batch_stride + w.at;
    if (s.x_format == SRS_FMT_F32) load_state8<SRS_FMT_F32>(s.x, at, w.count, vec, v);
    else if (s.x_format == SRS_FMT_BF16) load_state8<SRS_FMT_BF16>(s.x, at, w.count, vec, v);
    else load_state8<SRS_FMT_F16>(s.x, at, w.count, vec, v);
  } else {
    const Unit w = unit_of(s, u, s.n);
    const bool vec = (row.flags & SRS_ROW_VECTOR_OK) != 0u && s.n % 8 == 0;
    float g[kVec], old[kVec];
    const void* grad = reinterpret_cast<const void*>(row.grad);
    if (row.flags & SRS_ROW_GRAD_BF16) load_param8<true>(grad, w.at, w.count, vec, g);
    else load_param8<false>(grad, w.at, w.count, vec, g);
    load_state8<U>(reinterpret_cast<const void*>(row.state), w.at, w.count, vec, old);
    float next[kVec];
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      next[j] = __fadd_rn(__fmul_rn(old[j], plan.momentum), g[j]);
      v[j] = plan.nesterov ? __fadd_rn(__fmul_rn(next[j], plan.momentum), g[j]) : next[j];
    }
    if constexpr (STORE)
      store_state8<U>(reinterpret_cast<void*>(row.state), w.at, w.count, vec, next,
                      ctr + (uint32_t)w.at, plan.u_rule);
  }
}

template <int U>
__device__ __forceinline__ void open_row(const NewtonPlan& plan, int matrix, MuonMatrix* row,
                                         uint32_t* ctr) {
  if constexpr (U != kPlain) {
    *row = plan.matrix[matrix];
    const uint32_t key =
        (plan.rng.key_mode == SRS_KEY_GIVEN) ? row->key : update_key(plan.rng, row->key);
    *ctr = row->offset + state_key(key, 0u);
  }
}

__device__ __forceinline__ int class_of(const NewtonPlan& plan, int matrix) {
  int c = 0;
  while (c + 1 < plan.classes && matrix >= plan.source[c + 1].first) ++c;
  return c;
}

__device__ __forceinline__ double block_sum(double x, double* shared) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) x += __shfl_xor_sync(0xFFFFFFFFu, x, d);
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = x;
  __syncthreads();
  double total = 0.0;
  for (int w = 0; w < kThreads / 32; ++w) total += shared[w];
  return total;
}

// Partial sums of squares, in an order that depends on the sizes, the number of matrices and
// that of SMs.
template <int U>
__global__ void __launch_bounds__(kThreads)
newton_sum_kernel(const __grid_constant__ NewtonPlan plan) {
  __shared__ double shared[kThreads / 32];
  if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x < kMaxPhases)
    plan.counters[threadIdx.x] = 0u;
  const NewtonSource& s = plan.source[class_of(plan, (int)blockIdx.y)];
  if ((int)blockIdx.x >= s.chunks) return;
  const int batch = (int)blockIdx.y - s.first;
  MuonMatrix row{};
  uint32_t ctr = 0;
  open_row<U>(plan, (int)blockIdx.y, &row, &ctr);
  double sum = 0.0;
  const uint32_t stride = (uint32_t)s.chunks * kThreads;
#pragma unroll 2
  for (uint32_t u = blockIdx.x * kThreads + threadIdx.x; u < s.units; u += stride) {
    float v[kVec];
    source8<U, false>(plan, s, row, ctr, batch, u, v);
#pragma unroll
    for (int j = 0; j < kVec; ++j) sum = fma((double)v[j], (double)v[j], sum);
  }
  const double total = block_sum(sum, shared);
  if (threadIdx.x == 0) plan.partial[(int64_t)blockIdx.y * kSumChunks + blockIdx.x] = total;
}

// X_0 = V * 2^j in two FP16 matrices (row pitch `ld`, padding zero) and the factors of the
// products' sums: X_0 stands for X times rho = (|V|_F + eps) * 2^j, the later X_k for X times
// kHeldX or, while a bound on X_k is below 1, more.
template <int U>
__global__ void __launch_bounds__(kThreads)
newton_scale_kernel(const __grid_constant__ NewtonPlan plan) {
  __shared__ double shared[kThreads / 32];
  const NewtonSource& s = plan.source[class_of(plan, (int)blockIdx.y)];
  if ((int)blockIdx.x >= s.chunks) return;
  const int batch = (int)blockIdx.y - s.first;
  double part = 0.0;
  for (int i = threadIdx.x; i < s.chunks; i += kThreads)
    part += plan.partial[(int64_t)blockIdx.y * kSumChunks + i];
  const double length = sqrt(block_sum(part, shared)), norm = length + plan.eps;
  int exponent = 0;
  const bool finite = norm < INFINITY;  // false for NaN
  if (finite) frexp(length, &exponent);
  const int j = kTarget - exponent;
  // Two exact factors, as 2^j itself may not be an FP32 number.
  const float scale0 = finite ? (float)ldexp(1.0, j / 2) : __int_as_float(0x7FC00000);
  const float scale1 = (float)ldexp(1.0, j - j / 2);
  if (blockIdx.x == 0 && threadIdx.x < plan.steps) {
    const int step = threadIdx.x;
    const double below = finite && length > 0.0 ? log2(norm / length) : 0.0;
    const auto held = [&](int k) {
      return ldexp((double)kHeldX, (int)fmin(fmax(floor(below - k * plan.growth), 0.0), 100.0));
    };
    const double rho = !finite ? (double)NAN : step == 0 ? ldexp(norm, j) : held(step);
    const double next = step + 1 < plan.steps ? held(step + 1) : 1.0;
    float* const to = s.factors + kFactors * batch + 2 * step;
    to[0] = (float)(kHeld / rho / rho);
    to[1] = (float)(next / plan.hold_p / rho);
  }

  MuonMatrix row{};
  uint32_t ctr = 0;
  open_row<U>(plan, (int)blockIdx.y, &row, &ctr);
  __half* out = s.x0 + (int64_t)batch * s.x_elems;
  const uint32_t stride = (uint32_t)s.chunks * kThreads;
#pragma unroll 2
  for (uint32_t u = blockIdx.x * kThreads + threadIdx.x; u < s.units; u += stride) {
    float v[kVec];
    source8<U, true>(plan, s, row, ctr, batch, u, v);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < kVec; ++i) v[i] = v[i] * scale0 * scale1;
    encode8<SRS_FMT_F16>(v, 0u, SRS_RULE_NEAREST, w);
    const Unit at = unit_of(s, u, s.ld);
    *reinterpret_cast<uint4*>(out + at.at) = make_uint4(w[0], w[1], w[2], w[3]);
    float high[kVec];
    decode8<SRS_FMT_F16>(w, high);
#pragma unroll
    for (int i = 0; i < kVec; ++i) v[i] -= high[i];
    encode8<SRS_FMT_F16>(v, 0u, SRS_RULE_NEAREST, w);
    *reinterpret_cast<uint4*>(out + s.low + at.at) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// ------------------------------------------------------------------ products --

// Matrices of one shape in the product grid.  SPLIT: every map is followed by that of
// the matrix's low part.
template <bool SPLIT>
struct NewtonClass {
  static constexpr int kParts = SPLIT ? 2 : 1;
  CUtensorMap along[2][kParts];   // X, both copies, as the operands of G
  CUtensorMap across[2][kParts];  // X as the operand of X = P X
  CUtensorMap g[kParts], p[kParts];      // by rows
  CUtensorMap g_t[kParts], p_t[kParts];  // by columns
  int m, n, small, tall;
  int long_slices, small_slices;
  TileGrid grid;          // tiles of X
  Divider each_triangle;  // tiles of one G or P
  Divider each_grid;      // tiles of one X
  int64_t ld, x_elems, small_ld, small_elems;
  int64_t x_low, small_low;  // bytes from a matrix to its low part (G, P: SPLIT alone)
  __half* x[2];
  __half* g_at;
  __half* p_at;
  const float* factors;  // of each matrix and step
  char* out;             // orthogonalize: the result, contiguous matrices
  int out_format;
  int update;            // Muon: the result updates parameters
  int first;             // their place among all matrices
  float step, decay;
};

template <bool SPLIT>
struct NewtonWork {
  static constexpr int kClasses = SPLIT ? 1 : kMaxClasses;
  NewtonClass<SPLIT> shape[kClasses];
  uint64_t param[SPLIT ? 1 : kMaxMatrices];       // Muon: the parameters
  uint8_t param_bf16[SPLIT ? 1 : kMaxMatrices];
  uint32_t triangles[kClasses + 1];  // first tile of each class in a G or P phase
  uint32_t grids[kClasses + 1];      // ... in an X phase
  int classes, steps, edge;
  float a, b, c, hold_p;
  unsigned int* counters;  // one a phase
  unsigned int* status_at;
};

// Phase 3 i: G = X X^T; 3 i + 1: P = a I + b G + c G G; 3 i + 2: X = P X.  (SPLIT: a X by
// itself, so that P has no a I, except in the last step, whose result is not in FP16.)
template <bool SPLIT>
struct NewtonProducts {
  static constexpr bool kExtras = false;
  const NewtonWork<SPLIT>& w;
  struct Place {
    int shape, batch, row, col;
  };
  __device__ int phases() const { return 3 * w.steps; }
  __device__ uint32_t tiles(int p) const {
    return p % 3 == 2 ? w.grids[w.classes] : w.triangles[w.classes];
  }
  __device__ uint32_t formats() const { return 0u; }
  __device__ unsigned int* counter(int p) const { return w.counters + p; }
  __device__ unsigned int* status() const { return w.status_at; }
  __device__ int longest() const { return 0; }  // at most 2^18 slices, three times
  __device__ Place place(int p, uint32_t t) const {
    const bool grid = p % 3 == 2;
    const uint32_t* begin = grid ? w.grids : w.triangles;
    Place r;
    r.shape = 0;
    while (t >= begin[r.shape + 1]) ++r.shape;
    t -= begin[r.shape];
    const NewtonClass<SPLIT>& s = w.shape[r.shape];
    const Divider& each = grid ? s.each_grid : s.each_triangle;
    const uint32_t batch = each.quotient(t);
    r.batch = (int)batch;
    t -= batch * each.d;
    if (grid) s.grid.at(t, &r.row, &r.col);
    else triangle_tile(t, &r.row, &r.col);
    r.row *= w.edge;
    r.col *= w.edge;
    return r;
  }
  __device__ TileLoad load(int p, uint32_t t) const {
    const Place at = place(p, t);
    const NewtonClass<SPLIT>& s = w.shape[at.shape];
    const int step = p / 3, kind = p - 3 * step;
    const bool tall = s.tall != 0;
    TileLoad r{};
    r.row0 = at.row;
    r.col0 = at.col;
    r.batch = at.batch;
    if (kind == 0) {
      r.map_a = r.map_b = s.along[step & 1];
      r.slices = s.long_slices;
      r.a_rows_inner = r.b_rows_inner = tall;
    } else if (kind == 1) {
      r.map_a = r.map_b = s.g;
      r.map_a_t = r.map_b_t = s.g_t;
      r.slices = s.small_slices;
      r.a_symmetric = r.b_symmetric = true;
    } else {
      // P X: P by its rows, X with its row index (the summed one) outer; X P: X by
      // its rows, and P's columns are its rows
      r.map_a = tall ? s.across[step & 1] : s.p;
      r.map_b = tall ? s.p : s.across[step & 1];
      r.map_a_t = r.map_b_t = s.p_t;
      r.slices = s.small_slices;
      r.a_symmetric = !tall;
      r.b_symmetric = tall;
      r.b_rows_inner = !tall;
    }
    if (SPLIT) r.slices *= 3;
    return r;
  }
  __device__ TileStore store(int p, uint32_t t) const {
    const Place at = place(p, t);
    const NewtonClass<SPLIT>& s = w.shape[at.shape];
    const int step = p / 3, kind = p - 3 * step;
    TileStore r{};
    r.row0 = at.row;
    r.col0 = at.col;
    r.factor = 1.0f;
    if (kind != 1) r.late = s.factors + kFactors * at.batch + 2 * step + (kind >> 1);
    r.format = SRS_FMT_F16;
    if (kind != 2) {
      const int64_t from = (int64_t)at.batch * s.small_elems;
      r.m = r.n = s.small;
      r.pitch = s.small_ld;
      r.low = s.small_low;
      if (kind == 0) {
        r.out = reinterpret_cast<char*>(s.g_at + from);
      } else {
        r.factor = w.c * (w.hold_p / (kHeld * kHeld));
        r.beta = w.b * (w.hold_p / kHeld);
        if (!SPLIT || step + 1 == w.steps) r.diagonal = w.a * w.hold_p;
        r.addend = s.g_at + from;
        r.addend_phase = p - 1;
        r.out = reinterpret_cast<char*>(s.p_at + from);
      }
    } else {
      r.m = s.m;
      r.n = s.n;
      if (step + 1 < w.steps) {
        r.pitch = s.ld;
        // a times X (SPLIT) or its low part; the last step's X has none
        const __half* const x = s.x[step & 1] + (int64_t)at.batch * s.x_elems;
        r.addend = SPLIT ? x
                         : reinterpret_cast<const __half*>(reinterpret_cast<const char*>(x) +
                                                           s.x_low);
        r.addend_phase = p - 3;  // (below 0: the kernel before this one)
        r.beta = w.a * w.hold_p;  // (times the sum's factor)
        if (SPLIT || step + 2 < w.steps) r.low = s.x_low;
        r.out = reinterpret_cast<char*>(s.x[(step + 1) & 1] + (int64_t)at.batch * s.x_elems);
      } else if (!SPLIT && s.update != 0) {
        r.update = 1;
        r.format = w.param_bf16[s.first + at.batch] ? SRS_FMT_BF16 : SRS_FMT_F32;
        r.out = reinterpret_cast<char*>(w.param[s.first + at.batch]);
        r.pitch = s.n;
        r.step = s.step;
        r.decay = s.decay;
      } else {
        r.format = s.out_format;
        r.pitch = s.n;
        r.out = s.out + (int64_t)at.batch * s.m * s.n * (s.out_format == SRS_FMT_F32 ? 4 : 2);
      }
    }
    return r;
  }
};

template <int CG, bool SPLIT>
__global__ void __launch_bounds__(ProductShape<kOperandF16, CG>::kThreads, 1)
newton_kernel(const __grid_constant__ NewtonWork<SPLIT> w) {
  run_products<kOperandF16, CG, true, SPLIT>(NewtonProducts<SPLIT>{w});
}

int64_t round_up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }

// The matrices of one shape and their part of the workspace: factors, two copies of X
// and G and P, each aligned to 256 bytes.
struct NewtonShape {
  int64_t batch, m, n, small, ld, small_ld, x_elems, small_elems;
  int64_t x_low, small_low;  // bytes from a matrix to its low part (small_low 0: none)
  int64_t factors, x[2], g, p;  // byte offsets
};

// Rows on 128-byte boundaries, so that a box's 128-byte rows are whole cache lines
// (3000 x 3000 with a pitch of 3000: 754 us, of 3008: 574 us); narrow matrices only need
// the 16 bytes of a copy.
int64_t row_pitch_of(int64_t n) { return round_up(n, n >= 64 ? 64 : 8); }

int64_t take(int64_t* at, int64_t bytes) {
  const int64_t here = *at;
  *at += round_up(bytes, 256);
  return here;
}

NewtonShape lay_out(int64_t batch, int64_t m, int64_t n, bool split, int64_t* at) {
  NewtonShape s{};
  s.batch = batch;
  s.m = m;
  s.n = n;
  s.small = m < n ? m : n;
  s.ld = row_pitch_of(n);
  s.small_ld = row_pitch_of(s.small);
  s.x_elems = m * s.ld;
  s.small_elems = s.small * s.small_ld;
  const int64_t x_bytes = round_up(batch * s.x_elems * 2, 256);
  const int64_t small_bytes = round_up(batch * s.small_elems * 2, 256);
  s.x_low = x_bytes;
  s.small_low = split ? small_bytes : 0;
  s.factors = take(at, batch * kFactors * 4);
  s.x[0] = take(at, x_bytes + s.x_low);
  s.x[1] = take(at, x_bytes + s.x_low);
  s.g = take(at, small_bytes + s.small_low);
  s.p = take(at, small_bytes + s.small_low);
  return s;
}

// Shared by all shapes of a call: the grid's counters and the partial sums.
int64_t lay_out_head(int64_t matrices, int64_t* at) {
  take(at, kMaxPhases * 4);
  return take(at, matrices * kSumChunks * 8);
}

template <int U>
int launch_prepare(const NewtonPlan& plan, int64_t matrices, int chunks, cudaStream_t stream) {
  const dim3 grid((unsigned)chunks, (unsigned)matrices);
  newton_sum_kernel<U><<<grid, kThreads, 0, stream>>>(plan);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "newton_sum_kernel launch");
  newton_scale_kernel<U><<<grid, kThreads, 0, stream>>>(plan);
  e = cudaGetLastError();
  return e == cudaSuccess ? SRS_OK : cuda_fail(e, "newton_scale_kernel launch");
}

// Where results go, per class.
struct NewtonResult {
  void* out;
  int out_format;
  bool update;
  int first;
  float decay, step;
};

// What P is held times: 2^8, or the largest power of two with which the eigenvalues of P
// for singular values up to 1.4 stay below 60000 (FP16 ends at 65504).
float hold_of_p(const srs_newton& h) {
  const double a = h.coefficients[0], b = h.coefficients[1], c = h.coefficients[2];
  double most = std::fmax(std::fabs(a), std::fabs(a + 2.0 * b + 4.0 * c));
  const double vertex = -b / (2.0 * c);  // of a + b l + c l^2
  if (vertex > 0.0 && vertex < 2.0) most = std::fmax(most, std::fabs(a + 0.5 * b * vertex));
  float hold = kHeld;
  while (hold * most > 60000.0) hold *= 0.5f;
  return hold;
}

// The settings that the two preparing kernels need.
void fill_plan(const srs_newton& h, NewtonPlan* plan) {
  plan->eps = h.eps;
  plan->steps = h.steps;
  plan->hold_p = hold_of_p(h);
  double bound = 0.0;
  for (float c : h.coefficients) bound += std::fabs((double)c);
  plan->growth = bound > 1.0 ? std::log2(bound) : 0.0;
}

// Fills what the two preparing kernels and the product grid share.  The sources'
// own fields are set by the caller.
void fill_source(const NewtonShape& s, char* space, int first, int64_t matrices,
                 NewtonSource* f) {
  f->m = (int)s.m;
  f->n = (int)s.n;
  f->row_units = (uint32_t)((s.n + 7) / 8);
  f->units = (uint32_t)(s.m * f->row_units);
  f->first = first;
  // Enough CTAs for several per SM; each thread gets at least 4 vectors.
  int64_t chunks = (8ll * sm_count() + matrices - 1) / matrices;
  const int64_t most = (f->units + 4 * kThreads - 1) / (4 * kThreads);
  if (chunks > most) chunks = most;
  if (chunks > kSumChunks) chunks = kSumChunks;
  f->chunks = chunks < 1 ? 1 : (int)chunks;
  f->x0 = reinterpret_cast<__half*>(space + s.x[0]);
  f->low = s.x_low / 2;
  f->ld = s.ld;
  f->x_elems = s.x_elems;
  f->factors = reinterpret_cast<float*>(space + s.factors);
}

// The map of a matrix and, for SPLIT, that of its low part behind it.
template <bool SPLIT>
int encode_parts(ProductOperand o, int64_t low, int64_t batch, CUtensorMap* maps) {
  if (int rc = encode_operand(o, 2, batch, 128, &maps[0])) return rc;
  if (!SPLIT) return SRS_OK;
  o.base = static_cast<const char*>(o.base) + low;
  return encode_operand(o, 2, batch, 128, &maps[1]);
}

template <bool SPLIT>
int fill_class(const NewtonShape& s, char* space, const NewtonResult& result,
               NewtonClass<SPLIT>* c) {
  const bool tall = s.m > s.n;
  const int64_t longer = tall ? s.m : s.n;
  c->m = (int)s.m;
  c->n = (int)s.n;
  c->small = (int)s.small;
  c->tall = tall ? 1 : 0;
  c->long_slices = (int)((longer + 63) / 64);
  c->small_slices = (int)((s.small + 63) / 64);
  c->ld = s.ld;
  c->x_elems = s.x_elems;
  c->small_ld = s.small_ld;
  c->small_elems = s.small_elems;
  c->x_low = s.x_low;
  c->small_low = s.small_low;
  c->g_at = reinterpret_cast<__half*>(space + s.g);
  c->p_at = reinterpret_cast<__half*>(space + s.p);
  c->factors = reinterpret_cast<const float*>(space + s.factors);
  c->out = static_cast<char*>(result.out);
  c->out_format = result.out_format;
  c->update = result.update ? 1 : 0;
  c->first = result.first;
  c->step = result.step;
  c->decay = result.decay;
  for (int i = 0; i < 2; ++i) {
    c->x[i] = reinterpret_cast<__half*>(space + s.x[i]);
    // G sums along the longer side, which is contiguous unless X is tall; X = P X
    // sums along the shorter one
    const ProductOperand along{c->x[i], s.small, longer, s.ld, s.x_elems, tall};
    const ProductOperand across{c->x[i], longer, s.small, s.ld, s.x_elems, !tall};
    if (int rc = encode_parts<SPLIT>(along, s.x_low, s.batch, c->along[i])) return rc;
    if (int rc = encode_parts<SPLIT>(across, s.x_low, s.batch, c->across[i])) return rc;
  }
  ProductOperand g{c->g_at, s.small, s.small, s.small_ld, s.small_elems, false};
  ProductOperand p{c->p_at, s.small, s.small, s.small_ld, s.small_elems, false};
  if (int rc = encode_parts<SPLIT>(g, s.small_low, s.batch, c->g)) return rc;
  if (int rc = encode_parts<SPLIT>(p, s.small_low, s.batch, c->p)) return rc;
  g.rows_inner = p.rows_inner = true;
  if (int rc = encode_parts<SPLIT>(g, s.small_low, s.batch, c->g_t)) return rc;
  return encode_parts<SPLIT>(p, s.small_low, s.batch, c->p_t);
}

template <int CG, bool SPLIT>
int launch_newton(NewtonWork<SPLIT>& w, const srs_muon_class* shapes, cudaStream_t stream) {
  const void* kernel = reinterpret_cast<const void*>(&newton_kernel<CG, SPLIT>);
  using S = ProductShape<kOperandF16, CG>;
  int resident = 0;
  if (int rc = prepare_kernel(kernel, CG, S::kThreads, S::kSmem, &resident)) return rc;
  w.edge = 128 * CG;
  int64_t triangles = 0, grids = 0;
  for (int i = 0; i < w.classes; ++i) {
    NewtonClass<SPLIT>& c = w.shape[i];
    const uint32_t edge = (uint32_t)((c.small + w.edge - 1) / w.edge);
    c.each_triangle = make_divider(edge * (edge + 1) / 2);
    c.grid = make_grid((uint32_t)((c.m + w.edge - 1) / w.edge),
                       (uint32_t)((c.n + w.edge - 1) / w.edge));
    c.each_grid = make_divider(c.grid.rows * c.grid.cols);
    w.triangles[i] = (uint32_t)triangles;
    w.grids[i] = (uint32_t)grids;
    triangles += shapes[i].count * c.each_triangle.d;
    grids += shapes[i].count * c.each_grid.d;
  }
  w.triangles[w.classes] = (uint32_t)triangles;
  w.grids[w.classes] = (uint32_t)grids;
  if (triangles >= (1ll << 31) || grids >= (1ll << 31))
    return fail(SRS_ERR_INVALID_ARGUMENT, "too many matrices for one call");
  const int64_t most = triangles > grids ? triangles : grids;
  return launch_groups(kernel, most < resident ? most : resident, CG, S::kThreads, S::kSmem, true,
                       &w, stream, "newton_kernel launch");
}

// Rough time of the three products of a step with tiles of 128 * cg, in cycles of
// one SM: 512 a slice for the pair, 350 for the single CTA (256 of MMA, but twice
// the loads for it), and what a tile's results take.  Measured (us, single against
// pair): 1024^2 140, 184; 2048^2 243, 265; 2500^2 423, 371; 3500^2 958, 787;
// 12 x 768^2 218, 222; 24 x 768^2 400, 359; 4 x (1024 x 4096) 414, 435; the rule is wrong
// between the two kinds by up to a ninth (3001 x 3333, single: 750, 669).
double step_cycles(const srs_muon_class* shapes, int count, bool split, int cg) {
  const int64_t groups = sm_count() / cg, edge = 128 * cg;
  const double slice = cg == 2 ? 512.0 : 350.0, rest = cg == 2 ? 5000.0 : 2000.0;
  double total = 0.0;
  for (int kind = 0; kind < 3; ++kind) {
    double work = 0.0, longest = 0.0;
    int64_t tiles = 0;
    for (int i = 0; i < count; ++i) {
      const srs_muon_class& c = shapes[i];
      const int64_t small = c.m < c.n ? c.m : c.n, t = (small + edge - 1) / edge;
      const int64_t each =
          kind < 2 ? t * (t + 1) / 2 : (c.m + edge - 1) / edge * ((c.n + edge - 1) / edge);
      const int64_t summed = kind == 0 ? c.m + c.n - small : small;
      const double cycles =
          (split ? 3.0 : 1.0) * slice * (double)((summed + 63) / 64) + rest;
      tiles += c.count * each;
      work += cycles * (double)(c.count * each);
      if (cycles > longest) longest = cycles;
    }
    // whole rounds of the grid, at the tiles' mean cost
    const double rounds = (double)((tiles + groups - 1) / groups);
    const double time = tiles > 0 ? rounds * work / (double)tiles : 0.0;
    total += time > longest ? time : longest;
  }
  return total;
}

// CTAs to a tile: 2 or 1.
int tile_group(const srs_muon_class* shapes, int count, bool split) {
  return step_cycles(shapes, count, split, 2) <= step_cycles(shapes, count, split, 1) ? 2 : 1;
}

template <bool SPLIT>
int run_newton(NewtonWork<SPLIT>& w, const srs_muon_class* shapes, const srs_newton* h,
               unsigned int* counters, cudaStream_t stream) {
  w.steps = h->steps;
  w.a = h->coefficients[0];
  w.b = h->coefficients[1];
  w.c = h->coefficients[2];
  w.hold_p = hold_of_p(*h);
  w.counters = counters;
  if (int rc = status_word(&w.status_at)) return rc;
  return tile_group(shapes, w.classes, SPLIT) == 2 ? launch_newton<2, SPLIT>(w, shapes, stream)
                                                   : launch_newton<1, SPLIT>(w, shapes, stream);
}

int check_matrices(int64_t batch, int64_t m, int64_t n) {
  if (batch < 0 || m < 0 || n < 0)
    return fail(SRS_ERR_INVALID_ARGUMENT, "negative size (%lld, %lld, %lld)", (long long)batch,
                (long long)m, (long long)n);
  if (batch > 65535 || m > (1 << 24) || n > (1 << 24) || m * n > (1ll << 32))
    return fail(SRS_ERR_INVALID_ARGUMENT,
                "matrices of %lld x %lld (batch %lld) are too large: at most 2^32 elements, 2^24 "
                "rows or columns and 65535 matrices",
                (long long)m, (long long)n, (long long)batch);
  return SRS_OK;
}

int check_newton(const srs_newton* h) {
  if (h == nullptr) return fail(SRS_ERR_INVALID_ARGUMENT, "null Newton-Schulz settings");
  if (h->steps < 1 || h->steps > SRS_NEWTON_MAX_STEPS)
    return fail(SRS_ERR_INVALID_ARGUMENT, "steps must be in [1, %d], got %d",
                SRS_NEWTON_MAX_STEPS, h->steps);
  if (!(h->eps >= 0.0f) || !std::isfinite(h->eps))
    return fail(SRS_ERR_INVALID_ARGUMENT, "eps must be finite and non-negative");
  for (float c : h->coefficients)
    if (!std::isfinite(c)) return fail(SRS_ERR_INVALID_ARGUMENT, "coefficients must be finite");
  return SRS_OK;
}

int check_space(const void* space, int64_t bytes, int64_t need) {
  if (space == nullptr || bytes < need)
    return fail(SRS_ERR_INVALID_ARGUMENT, "workspace of %lld bytes, %lld needed",
                (long long)(space == nullptr ? 0 : bytes), (long long)need);
  if (reinterpret_cast<uintptr_t>(space) % 256 != 0)
    return fail(SRS_ERR_INVALID_ARGUMENT, "workspace must be 256-byte aligned");
  return SRS_OK;
}

}  // namespace
}  // namespace srs

using namespace srs;

extern "C" int64_t srs_newton_workspace(int64_t batch, int64_t m, int64_t n, int y_format) {
  if (batch <= 0 || m <= 0 || n <= 0) return 0;
  int64_t at = 0;
  lay_out_head(batch, &at);
  lay_out(batch, m, n, y_format != SRS_FMT_BF16, &at);
  return at;
}

extern "C" int srs_orthogonalize(const void* x, int x_format, int64_t row_pitch,
                                 int64_t batch_stride, void* y, int y_format, int64_t batch,
                                 int64_t m, int64_t n, const srs_newton* h, void* workspace,
                                 int64_t workspace_bytes, void* stream) {
  clear_error();
  if (x_format < SRS_FMT_F32 || x_format > SRS_FMT_F16 || y_format < SRS_FMT_F32 ||
      y_format > SRS_FMT_F16)
    return fail(SRS_ERR_INVALID_ARGUMENT, "unsupported matrix format (%d, %d)", x_format, y_format);
  if (int rc = check_newton(h)) return rc;
  if (int rc = check_matrices(batch, m, n)) return rc;
  if (batch == 0 || m == 0 || n == 0) return SRS_OK;
  if (x == nullptr || y == nullptr)
    return fail(SRS_ERR_INVALID_ARGUMENT, "null input or output pointer");
  if (row_pitch < 0 || batch_stride < 0)
    return fail(SRS_ERR_INVALID_ARGUMENT, "negative pitch");
  const uintptr_t at = reinterpret_cast<uintptr_t>(x);
  if (at % fmt_bytes(x_format) != 0 ||
      reinterpret_cast<uintptr_t>(y) % fmt_bytes(y_format) != 0)
    return fail(SRS_ERR_INVALID_ARGUMENT, "input/output pointers are not element aligned");
  if (int rc = check_space(workspace, workspace_bytes, srs_newton_workspace(batch, m, n, y_format)))
    return rc;
  if (int rc = check_device()) return rc;
  if (int rc = check_products()) return rc;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  char* space = static_cast<char*>(workspace);
  int64_t used = 0;
  const int64_t partial = lay_out_head(batch, &used);
  const NewtonShape shape = lay_out(batch, m, n, y_format != SRS_FMT_BF16, &used);
  NewtonPlan plan{};
  plan.classes = 1;
  plan.partial = reinterpret_cast<double*>(space + partial);
  plan.counters = reinterpret_cast<unsigned int*>(space);
  fill_plan(*h, &plan);
  NewtonSource& s = plan.source[0];
  s.x = x;
  s.x_format = x_format;
  s.row_pitch = row_pitch;
  s.batch_stride = batch_stride;
  s.vec = at % 16 == 0 && row_pitch % 8 == 0 && batch_stride % 8 == 0;
  fill_source(shape, space, 0, batch, &s);
  const NewtonResult result{y, y_format, false, 0, 0.0f, 0.0f};
  const auto run = [&](auto& work) {
    work.classes = 1;
    if (int rc = fill_class(shape, space, result, &work.shape[0])) return rc;
    if (int rc = launch_prepare<kPlain>(plan, batch, s.chunks, st)) return rc;
    const srs_muon_class matrices{batch, m, n, 0.0f, 0};
    return run_newton(work, &matrices, h, plan.counters, st);
  };
  if (y_format != SRS_FMT_BF16) {
    NewtonWork<true> work{};
    return run(work);
  }
  NewtonWork<false> work{};
  return run(work);
}

static int check_classes(const srs_muon_class* classes, int n_classes, int64_t* matrices) {
  if (n_classes < 0 || n_classes > SRS_MUON_MAX_CLASSES)
    return fail(SRS_ERR_INVALID_ARGUMENT, "between 0 and %d shapes in a call, got %d",
                SRS_MUON_MAX_CLASSES, n_classes);
  if (n_classes > 0 && classes == nullptr)
    return fail(SRS_ERR_INVALID_ARGUMENT, "null shape table");
  *matrices = 0;
  for (int i = 0; i < n_classes; ++i) {
    if (int rc = check_matrices(classes[i].count, classes[i].m, classes[i].n)) return rc;
    if (classes[i].count == 0 || classes[i].m == 0 || classes[i].n == 0)
      return fail(SRS_ERR_INVALID_ARGUMENT, "shape %d is empty", i);
    *matrices += classes[i].count;
  }
  if (*matrices > kMaxMatrices)
    return fail(SRS_ERR_INVALID_ARGUMENT, "%lld matrices in one call (at most %d)",
                (long long)*matrices, kMaxMatrices);
  return SRS_OK;
}

extern "C" int srs_newton_tile(const srs_muon_class* classes, int n_classes, int y_format) {
  clear_error();
  if (n_classes < 0 || n_classes > SRS_MUON_MAX_CLASSES || (n_classes > 0 && classes == nullptr))
    return fail(SRS_ERR_INVALID_ARGUMENT, "between 0 and %d shapes in a call, got %d",
                SRS_MUON_MAX_CLASSES, n_classes);
  for (int i = 0; i < n_classes; ++i)
    if (int rc = check_matrices(classes[i].count, classes[i].m, classes[i].n)) return rc;
  return 128 * tile_group(classes, n_classes, y_format != SRS_FMT_BF16);
}

extern "C" int64_t srs_muon_workspace(const srs_muon_class* classes, int n_classes) {
  clear_error();
  int64_t matrices = 0, at = 0;
  if (check_classes(classes, n_classes, &matrices) != SRS_OK) return -1;
  if (n_classes == 0) return 0;
  lay_out_head(matrices, &at);
  for (int i = 0; i < n_classes; ++i)
    lay_out(classes[i].count, classes[i].m, classes[i].n, false, &at);
  return at;
}

extern "C" int srs_muon_multi(const srs_row* rows, const srs_muon_class* classes, int n_classes,
                              int u_format, int u_rule, const srs_muon_hparams* hp,
                              const srs_newton* h, const srs_rng* rng, void* workspace,
                              int64_t workspace_bytes, void* stream) {
  clear_error();
  if (!valid_format(u_format))
    return fail(SRS_ERR_INVALID_ARGUMENT, "unknown state format %d", u_format);
  if (!valid_rule(u_rule)) return fail(SRS_ERR_INVALID_ARGUMENT, "unknown rounding rule %d", u_rule);
  if (hp == nullptr || rng == nullptr)
    return fail(SRS_ERR_INVALID_ARGUMENT, "null hyperparameter or rng pointer");
  if (rng->key_mode != SRS_KEY_DERIVE && rng->key_mode != SRS_KEY_GIVEN)
    return fail(SRS_ERR_INVALID_ARGUMENT, "unknown key_mode %d", rng->key_mode);
  if (int rc = check_newton(h)) return rc;
  int64_t matrices = 0;
  if (int rc = check_classes(classes, n_classes, &matrices)) return rc;
  if (matrices == 0) return SRS_OK;
  if (rows == nullptr) return fail(SRS_ERR_INVALID_ARGUMENT, "null row table");
  for (int64_t i = 0; i < matrices; ++i) {
    const srs_row& r = rows[i];
    if (r.param == 0 || r.grad == 0 || r.state[0] == 0)
      return fail(SRS_ERR_INVALID_ARGUMENT, "row %lld: null address", (long long)i);
    const uint64_t p = (r.flags & SRS_ROW_PARAM_BF16) ? 2 : 4;
    const uint64_t g = (r.flags & SRS_ROW_GRAD_BF16) ? 2 : 4, u = (uint64_t)fmt_bytes(u_format);
    const bool vec = (r.flags & SRS_ROW_VECTOR_OK) != 0u;
    if (r.param % p != 0 || r.grad % (vec ? 16 : g) != 0 ||
        r.state[0] % (vec ? (u == 1 ? 8 : 16) : u) != 0)
      return fail(SRS_ERR_INVALID_ARGUMENT,
                  "row %lld: an address is not aligned as its flags promise", (long long)i);
  }
  if (int rc = check_space(workspace, workspace_bytes, srs_muon_workspace(classes, n_classes)))
    return rc;
  if (int rc = check_device()) return rc;
  if (int rc = check_products()) return rc;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  char* space = static_cast<char*>(workspace);
  int64_t used = 0;
  const int64_t partial = lay_out_head(matrices, &used);
  NewtonPlan plan{};
  plan.classes = n_classes;
  plan.partial = reinterpret_cast<double*>(space + partial);
  plan.counters = reinterpret_cast<unsigned int*>(space);
  fill_plan(*h, &plan);
  plan.rng = *rng;
  plan.momentum = hp->momentum;
  plan.nesterov = hp->nesterov;
  plan.u_rule = u_rule;
  NewtonWork<false> work{};
  work.classes = n_classes;
  int first = 0, chunks = 1;
  for (int i = 0; i < n_classes; ++i) {
    const srs_muon_class& c = classes[i];
    const NewtonShape shape = lay_out(c.count, c.m, c.n, false, &used);
    NewtonSource& s = plan.source[i];
    fill_source(shape, space, first, matrices, &s);
    if (s.chunks > chunks) chunks = s.chunks;
    const NewtonResult result{nullptr, 0, true, first, hp->decay, c.neg_step};
    if (int rc = fill_class(shape, space, result, &work.shape[i])) return rc;
    first += (int)c.count;
  }
  for (int64_t i = 0; i < matrices; ++i) {
    const srs_row& r = rows[i];
    plan.matrix[i] = {r.param, r.grad, r.state[0], r.param_index, r.offset, r.flags, 0u};
    work.param[i] = r.param;
    work.param_bf16[i] = (r.flags & SRS_ROW_PARAM_BF16) ? 1 : 0;
  }
  int rc = SRS_OK;
  switch (u_format) {
    case SRS_FMT_F32: rc = launch_prepare<SRS_FMT_F32>(plan, matrices, chunks, st); break;
    case SRS_FMT_BF16: rc = launch_prepare<SRS_FMT_BF16>(plan, matrices, chunks, st); break;
    case SRS_FMT_F16: rc = launch_prepare<SRS_FMT_F16>(plan, matrices, chunks, st); break;
    case SRS_FMT_E4M3: rc = launch_prepare<SRS_FMT_E4M3>(plan, matrices, chunks, st); break;
    default: rc = launch_prepare<SRS_FMT_E5M2>(plan, matrices, chunks, st); break;
  }
  if (rc != SRS_OK) return rc;
  return run_newton(work, classes, h, plan.counters, st);
}
