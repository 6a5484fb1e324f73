// Rows of FP8 blocks: block exponents and rounding, as every kernel that quantises does them.
#pragma once

#include "srs_common.cuh"

namespace srs {

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

// What a product's host side checks the rest of a quantisation with: counter of element 0.
inline uint32_t block_counter(uint32_t seed, uint32_t offset, uint32_t copy) {
  uint32_t x = seed ^ copy;
  x ^= x >> 16;
  x *= 0x7FEB352Du;
  x ^= x >> 15;
  x *= 0x846CA68Bu;
  return offset + (x ^ (x >> 16));
}

}  // namespace srs
