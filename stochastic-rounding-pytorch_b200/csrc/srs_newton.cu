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
// Number formats.  G, P and X are held in FP16, accumulated in FP32.  Their
// sizes are bounded (eigenvalues of a few units), so FP16's 11 significant bits are usable where
// BF16 would keep 8: the steps multiply rounding errors of small singular
// directions by up to a^5 = 485, and eight times smaller errors keep the result
// within about 1e-3 of exact arithmetic for gradient-like spectra (1e-2 with BF16).
// X_0 is held as V * 2^j with a power of two that puts |V * 2^j|_F between
// sqrt(min(m, n)) / 4 and sqrt(min(m, n)): BF16 inputs are then held exactly, and
// the remaining factor rho enters the first products in FP32.  The norm is
// summed in FP64, so no input in range overflows or vanishes in it.
//
// Reads of V: one for the norm and one for X_0.  For an optimizer step both
// passes compute V from the gradient and the momentum (8 or fewer bytes an
// element) rather than keeping V in FP32 (8 bytes more of traffic and 4 of
// memory); the second pass stores u'.
#include <cmath>

#include "srs_host.h"
#include "srs_product.cuh"

namespace srs {
namespace {

constexpr int kSumChunks = 256;  // most partial sums of a matrix
constexpr int kPlain = -1;       // source template value: a plain tensor
// G and P are held times 2^8: their small elements (1 / m and less in the first
// steps) then stay among FP16's normal numbers, and eigenvalues up to 255 fit.
constexpr float kHeld = 256.0f;

struct NewtonSource {
  const void* x;      // plain: the tensor
  int x_format;       // plain: SRS_FMT_F32, SRS_FMT_BF16 or SRS_FMT_F16
  int64_t row_pitch, batch_stride;
  int vec;            // plain: rows start on 16-byte boundaries
  const srs_row* rows;  // Muon: one row per matrix
  srs_rng rng;
  float momentum;
  int nesterov;
  int u_rule;
  int m, n;           // rows, columns
  uint32_t units;     // vectors of 8 per matrix: m * ceil(n / 8)
  uint32_t row_units;
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
__device__ __forceinline__ void source8(const NewtonSource& s, const srs_row& row, uint32_t ctr,
                                        int batch, uint32_t u, float (&v)[kVec]) {
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
    load_state8<U>(reinterpret_cast<const void*>(row.state[0]), w.at, w.count, vec, old);
    float next[kVec];
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      next[j] = __fadd_rn(__fmul_rn(old[j], s.momentum), g[j]);
      v[j] = s.nesterov ? __fadd_rn(__fmul_rn(next[j], s.momentum), g[j]) : next[j];
    }
    if constexpr (STORE)
      store_state8<U>(reinterpret_cast<void*>(row.state[0]), w.at, w.count, vec, next,
                      ctr + (uint32_t)w.at, s.u_rule);
  }
}

template <int U>
__device__ __forceinline__ void open_row(const NewtonSource& s, int batch, srs_row* row,
                                         uint32_t* ctr) {
  if constexpr (U != kPlain) {
    *row = s.rows[batch];
    const uint32_t key = (s.rng.key_mode == SRS_KEY_GIVEN) ? row->param_index
                                                           : update_key(s.rng, row->param_index);
    *ctr = row->offset + state_key(key, 0u);
  }
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

// Partial sums of squares, in an order that depends on the sizes alone.
template <int U>
__global__ void __launch_bounds__(kThreads) newton_sum_kernel(const NewtonSource s,
                                                              double* __restrict__ partial) {
  __shared__ double shared[kThreads / 32];
  const int batch = blockIdx.y;
  srs_row row{};
  uint32_t ctr = 0;
  open_row<U>(s, batch, &row, &ctr);
  double sum = 0.0;
  for (uint32_t u = blockIdx.x * kThreads + threadIdx.x; u < s.units; u += gridDim.x * kThreads) {
    float v[kVec];
    source8<U, false>(s, row, ctr, batch, u, v);
#pragma unroll
    for (int j = 0; j < kVec; ++j) sum = fma((double)v[j], (double)v[j], sum);
  }
  const double total = block_sum(sum, shared);
  if (threadIdx.x == 0) partial[(int64_t)batch * gridDim.x + blockIdx.x] = total;
}

// X_0 = V * 2^j in FP16 (row pitch `ld`, padding zero) and rho = (|V|_F + eps) * 2^j.
template <int U>
__global__ void __launch_bounds__(kThreads)
newton_scale_kernel(const NewtonSource s, const double* __restrict__ partial, int chunks,
                    double eps, int target, __half* __restrict__ x0, int64_t ld,
                    int64_t batch_stride, float* __restrict__ rho) {
  __shared__ double shared[kThreads / 32];
  const int batch = blockIdx.y;
  const double part =
      (int)threadIdx.x < chunks ? partial[(int64_t)batch * chunks + threadIdx.x] : 0.0;
  const double norm = sqrt(block_sum(part, shared)) + eps;
  int exponent = 0;
  const bool finite = norm < INFINITY;  // false for NaN
  const double fraction = finite ? frexp(norm, &exponent) : 0.0;
  const int j = target - exponent;
  // Two exact factors, as 2^j itself may not be an FP32 number.
  const float scale0 = finite ? (float)ldexp(1.0, j / 2) : __int_as_float(0x7FC00000);
  const float scale1 = (float)ldexp(1.0, j - j / 2);
  if (blockIdx.x == 0 && threadIdx.x == 0)
    rho[batch] = finite ? (float)ldexp(fraction, target) : __int_as_float(0x7FC00000);

  srs_row row{};
  uint32_t ctr = 0;
  open_row<U>(s, batch, &row, &ctr);
  __half* out = x0 + (int64_t)batch * batch_stride;
  for (uint32_t u = blockIdx.x * kThreads + threadIdx.x; u < s.units; u += gridDim.x * kThreads) {
    float v[kVec];
    source8<U, true>(s, row, ctr, batch, u, v);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < kVec; ++i) v[i] = v[i] * scale0 * scale1;
    encode8<SRS_FMT_F16>(v, 0u, SRS_RULE_NEAREST, w);
    const Unit at = unit_of(s, u, ld);
    *reinterpret_cast<uint4*>(out + at.at) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

int64_t round_up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }

// Workspace: partial sums, rho, two copies of X and G and P, each aligned to 256 bytes.
struct NewtonSpace {
  int64_t ld, small_ld, x_elems, small_elems;
  int64_t partial, rho, x[2], g, p, bytes;
};

NewtonSpace newton_space(int64_t batch, int64_t m, int64_t n) {
  NewtonSpace s{};
  const int64_t small = m < n ? m : n;
  s.ld = round_up(n, 8);
  s.small_ld = round_up(small, 8);
  s.x_elems = m * s.ld;
  s.small_elems = small * s.small_ld;
  int64_t at = 0;
  const auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += round_up(bytes, 256);
    return here;
  };
  s.partial = take(batch * kSumChunks * 8);
  s.rho = take(batch * 4);
  s.x[0] = take(batch * s.x_elems * 2);
  s.x[1] = take(batch * s.x_elems * 2);
  s.g = take(batch * s.small_elems * 2);
  s.p = take(batch * s.small_elems * 2);
  s.bytes = at;
  return s;
}

template <int U>
int prepare(const NewtonSource& source, int64_t batch, const NewtonSpace& w, char* space,
            double eps, cudaStream_t stream) {
  // Enough CTAs for a few per SM; each gets at least 4 vectors a thread.
  int64_t chunks = (4ll * sm_count() + batch - 1) / batch;
  const int64_t most = (source.units + 4 * kThreads - 1) / (4 * kThreads);
  if (chunks > most) chunks = most;
  if (chunks > kSumChunks) chunks = kSumChunks;
  if (chunks < 1) chunks = 1;
  const dim3 grid((unsigned)chunks, (unsigned)batch);
  double* partial = reinterpret_cast<double*>(space + w.partial);
  newton_sum_kernel<U><<<grid, kThreads, 0, stream>>>(source, partial);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "newton_sum_kernel launch");
  const int64_t small = source.m < source.n ? source.m : source.n;
  int target = 0;  // floor(log2(sqrt(small)))
  while ((1ll << (2 * (target + 1))) <= small) ++target;
  newton_scale_kernel<U><<<grid, kThreads, 0, stream>>>(
      source, partial, (int)chunks, eps, target, reinterpret_cast<__half*>(space + w.x[0]), w.ld,
      w.x_elems, reinterpret_cast<float*>(space + w.rho));
  e = cudaGetLastError();
  return e == cudaSuccess ? SRS_OK : cuda_fail(e, "newton_scale_kernel launch");
}

struct NewtonResult {
  int epilogue;  // kEpilogueStore or kEpilogueMuon
  void* out;
  int out_format;
  int64_t ldd, batch_stride;
  const srs_row* rows;
  float decay, step;
};

int newton_steps(int64_t batch, int64_t m, int64_t n, const srs_newton* h, const NewtonSpace& w,
                 char* space, const NewtonResult& result, cudaStream_t stream) {
  const bool tall = m > n;
  const int64_t small = tall ? n : m;
  const float* rho = reinterpret_cast<const float*>(space + w.rho);
  __half* g = reinterpret_cast<__half*>(space + w.g);
  __half* p = reinterpret_cast<__half*>(space + w.p);
  for (int i = 0; i < h->steps; ++i) {
    const void* x = space + w.x[i & 1];
    void* next = space + w.x[(i + 1) & 1];
    const bool last = i == h->steps - 1;
    const auto symmetric = [&](float alpha, float beta, float diagonal, const __half* addend,
                               __half* out, const float* scale) {
      ProductArgs args{};
      args.symmetric = 1;
      args.e.alpha = alpha;
      args.e.beta = beta;
      args.e.diagonal = diagonal;
      args.e.addend = addend;
      args.e.out = out;
      args.e.ldd = w.small_ld;
      args.e.batch_stride = w.small_elems;
      args.e.rho = scale;
      args.e.rho_power = 2;
      return args;
    };
    // G = X X^T (X^T X): both operands are X, k along the longer side
    const ProductOperand along{x, small, tall ? m : n, w.ld, w.x_elems, tall};
    if (int rc = launch_product(kOperandF16, kEpilogueSymmetric, along, along, batch, 0, 0,
                                symmetric(kHeld, 0.0f, 0.0f, nullptr, g, i == 0 ? rho : nullptr),
                                stream))
      return rc;
    // P = a I + b G + c G G
    const ProductOperand gram{g, small, small, w.small_ld, w.small_elems, false};
    if (int rc = launch_product(
            kOperandF16, kEpilogueSymmetric, gram, gram, batch, 0, 0,
            symmetric(h->coefficients[2] / kHeld, h->coefficients[1], h->coefficients[0] * kHeld,
                      g, p, nullptr),
            stream))
      return rc;
    // X = P X (X P): P is symmetric, so either of its sides serves as k
    const ProductOperand poly{p, small, small, w.small_ld, w.small_elems, false};
    const ProductOperand across{x, tall ? m : n, small, w.ld, w.x_elems, !tall};
    ProductArgs args{};
    args.e.alpha = 1.0f / kHeld;
    args.e.rho = i == 0 ? rho : nullptr;
    args.e.rho_power = 1;
    args.e.out = last ? result.out : next;
    args.e.out_format = last ? result.out_format : SRS_FMT_F16;
    args.e.ldd = last ? result.ldd : w.ld;
    args.e.batch_stride = last ? result.batch_stride : w.x_elems;
    args.e.rows = result.rows;
    args.e.decay = result.decay;
    args.e.step = result.step;
    if (int rc = launch_product(kOperandF16, last ? result.epilogue : kEpilogueStore,
                                tall ? across : poly, tall ? poly : across, batch, 0, 0, args,
                                stream))
      return rc;
  }
  return SRS_OK;
}

int check_newton(int64_t batch, int64_t m, int64_t n, const srs_newton* h) {
  if (h == nullptr) return fail(SRS_ERR_INVALID_ARGUMENT, "null Newton-Schulz settings");
  if (batch < 0 || m < 0 || n < 0)
    return fail(SRS_ERR_INVALID_ARGUMENT, "negative size (%lld, %lld, %lld)", (long long)batch,
                (long long)m, (long long)n);
  if (batch > 65535 || m > (1 << 24) || n > (1 << 24) || m * n > (1ll << 32))
    return fail(SRS_ERR_INVALID_ARGUMENT,
                "matrices of %lld x %lld (batch %lld) are too large: at most 2^32 elements, 2^24 "
                "rows or columns and 65535 matrices",
                (long long)m, (long long)n, (long long)batch);
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

extern "C" int64_t srs_newton_workspace(int64_t batch, int64_t m, int64_t n) {
  if (batch <= 0 || m <= 0 || n <= 0) return 0;
  return newton_space(batch, m, n).bytes;
}

extern "C" int srs_orthogonalize(const void* x, int x_format, int64_t row_pitch,
                                 int64_t batch_stride, void* y, int y_format, int64_t batch,
                                 int64_t m, int64_t n, const srs_newton* h, void* workspace,
                                 int64_t workspace_bytes, void* stream) {
  clear_error();
  if (x_format < SRS_FMT_F32 || x_format > SRS_FMT_F16 || y_format < SRS_FMT_F32 ||
      y_format > SRS_FMT_F16)
    return fail(SRS_ERR_INVALID_ARGUMENT, "unsupported matrix format (%d, %d)", x_format, y_format);
  if (int rc = check_newton(batch, m, n, h)) return rc;
  if (batch == 0 || m == 0 || n == 0) return SRS_OK;
  if (x == nullptr || y == nullptr)
    return fail(SRS_ERR_INVALID_ARGUMENT, "null input or output pointer");
  if (row_pitch < 0 || batch_stride < 0)
    return fail(SRS_ERR_INVALID_ARGUMENT, "negative pitch");
  const uintptr_t at = reinterpret_cast<uintptr_t>(x);
  if (at % fmt_bytes(x_format) != 0 ||
      reinterpret_cast<uintptr_t>(y) % fmt_bytes(y_format) != 0)
    return fail(SRS_ERR_INVALID_ARGUMENT, "input/output pointers are not element aligned");
  const NewtonSpace w = newton_space(batch, m, n);
  if (int rc = check_space(workspace, workspace_bytes, w.bytes)) return rc;
  if (int rc = check_device()) return rc;
  NewtonSource s{};
  s.x = x;
  s.x_format = x_format;
  s.row_pitch = row_pitch;
  s.batch_stride = batch_stride;
  s.vec = at % 16 == 0 && row_pitch % 8 == 0 && batch_stride % 8 == 0;
  s.m = (int)m;
  s.n = (int)n;
  s.row_units = (uint32_t)((n + 7) / 8);
  s.units = (uint32_t)(m * s.row_units);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  char* space = static_cast<char*>(workspace);
  if (int rc = prepare<kPlain>(s, batch, w, space, h->eps, st)) return rc;
  NewtonResult r{};
  r.epilogue = kEpilogueStore;
  r.out = y;
  r.out_format = y_format;
  r.ldd = n;
  r.batch_stride = m * n;
  return newton_steps(batch, m, n, h, w, space, r, st);
}

extern "C" int srs_muon_multi(const srs_row* rows, int64_t n_rows, int64_t m, int64_t n,
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
  if (int rc = check_newton(n_rows, m, n, h)) return rc;
  if (n_rows == 0 || m == 0 || n == 0) return SRS_OK;
  if (rows == nullptr || reinterpret_cast<uintptr_t>(rows) % 16 != 0)
    return fail(SRS_ERR_INVALID_ARGUMENT, "row table must be 16-byte aligned");
  const NewtonSpace w = newton_space(n_rows, m, n);
  if (int rc = check_space(workspace, workspace_bytes, w.bytes)) return rc;
  if (int rc = check_device()) return rc;
  NewtonSource s{};
  s.rows = rows;
  s.rng = *rng;
  s.momentum = hp->momentum;
  s.nesterov = hp->nesterov;
  s.u_rule = u_rule;
  s.m = (int)m;
  s.n = (int)n;
  s.row_units = (uint32_t)((n + 7) / 8);
  s.units = (uint32_t)(m * s.row_units);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  char* space = static_cast<char*>(workspace);
  int rc = SRS_OK;
  switch (u_format) {
    case SRS_FMT_F32: rc = prepare<SRS_FMT_F32>(s, n_rows, w, space, h->eps, st); break;
    case SRS_FMT_BF16: rc = prepare<SRS_FMT_BF16>(s, n_rows, w, space, h->eps, st); break;
    case SRS_FMT_F16: rc = prepare<SRS_FMT_F16>(s, n_rows, w, space, h->eps, st); break;
    case SRS_FMT_E4M3: rc = prepare<SRS_FMT_E4M3>(s, n_rows, w, space, h->eps, st); break;
    default: rc = prepare<SRS_FMT_E5M2>(s, n_rows, w, space, h->eps, st); break;
  }
  if (rc != SRS_OK) return rc;
  NewtonResult r{};
  r.epilogue = kEpilogueMuon;
  r.rows = rows;
  r.decay = hp->decay;
  r.step = hp->neg_step;
  return newton_steps(n_rows, m, n, h, w, space, r, st);
}
