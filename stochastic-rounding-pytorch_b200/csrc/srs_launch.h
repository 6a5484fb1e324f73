// Host side of the tensor-core products: tensor maps, the status word of bounded
// waits and launches of persistent grids (implemented in srs_product.cu).
#pragma once

#include <cstdint>
#include <cuda.h>
#include <cuda_runtime.h>

#include "srs_b200.h"

namespace srs {

// An operand in global memory: `rows` x `k` per batch entry.  k contiguous: row
// pitch `pitch` elements; rows_inner: element (i, k) at k * pitch + i.
struct ProductOperand {
  const void* base;
  int64_t rows, k, pitch, batch_stride;  // elements
  bool rows_inner;
};

// Tensor map of an operand: boxes of `box_rows` rows x `box_bytes` (32, 64, 128) of k, or of 64 rows x
// 64 k when the row index is contiguous; elements outside the operand read as zero.
int encode_operand(const ProductOperand& o, int element_bytes, int64_t batch, int box_rows,
                   CUtensorMap* map, int box_bytes = 128);

// The word of the current device in which bounded waits record where they ran out.
int status_word(unsigned int** word);

// SRS_ERR_WAIT, once, when a wait has run out since the last check: every entry point that
// launches products asks before its first launch.
int check_products();

// Opt-in shared memory of a kernel, and how many of its CTA groups (1 or 2 CTAs) can be
// resident on the current device; remembered per kernel and device.
int prepare_kernel(const void* kernel, int group, int threads, int smem, int* resident);

// Launches `kernel` with one argument on groups * group CTAs; `cooperative` when its CTAs
// wait for one another; `overlap` when it may start before the kernel ahead of it in the
// stream has finished (it then waits for that kernel itself).
int launch_groups(const void* kernel, int64_t groups, int group, int threads, int smem,
                  bool cooperative, void* argument, cudaStream_t stream, const char* what,
                  bool overlap = false);

// What is quantised to FP8 blocks, and where to (srs_quantize_blocks, _stack and _groups):
// one matrix, a stack of them (`matrices`, `x_stride` elements apart), rows of groups (`ends`;
// the transposed copy in the products' form), or rows in another order (`order`: row i of
// the copy is row order[i] of x; rows alone).  `for_product`: ahead of a product of the same call.
struct QuantizeCall {
  const void* x;
  int x_format;
  int64_t rows, cols, x_pitch;
  int out_format, rule;
  bool square;
  uint32_t seed, offset;
  srs_block_copy copy{}, turned{};
  int64_t matrices = 1, x_stride = 0;
  const int32_t* ends = nullptr;
  int groups = 0;
  const int32_t* order = nullptr;
  bool for_product = false;
  bool overlap = false;  // rows alone: may start beside the kernel ahead, which it reads nothing of
};
int quantize(const QuantizeCall& q, cudaStream_t stream);
constexpr int64_t kMaxQuantizedRows = 65535ll * 64;

int check_operand(const char* what, const srs_blocks* b, int64_t k);
int check_groups(const int32_t* ends, int groups);

// Low-rank adapters beside a product: their low part and its second matrices.
inline int thin_columns(int64_t tokens) { return tokens <= 16 ? 16 : tokens <= 32 ? 32 : 64; }

struct AdapterCall {
  const void* pairs;
  const void* up;  // rows x rank a matrix, or (rows_inner) rank x rows; `pitch`, `stride` elements
  int64_t pitch, stride;
  bool rows_inner;
  int count, rank, format;
  const int32_t* order;
  const int32_t* ends;
  // FP16: powers of two of the tokens' pairs (thin: in the batch's order, else the adapters')
  const int32_t* exponents;
};

// FP8 blocks: d = a b^T (operands checked by the caller).  Element (i, j)
// of d is stored at i * row_stride + j * col_stride; only products with a thin side
// (at most kThinRows rows) take a col_stride other than 1.  `overlap`: the kernel ahead
// writes nothing of a.
constexpr int kThinRows = 64;
int launch_block_product(const srs_blocks& a, const srs_blocks& b, int64_t k, void* d,
                         int d_format, cudaStream_t stream);
int launch_thin(const srs_blocks& a, const srs_blocks& b, int64_t k, void* d, int d_format,
                int64_t row_stride, int64_t col_stride, bool overlap, cudaStream_t stream,
                const AdapterCall* adapters = nullptr);
// The same for rows in groups: a's rows by their group's matrix of w (few rows a group).
int launch_expert_thin(const srs_blocks& a, const srs_blocks& w, int experts, const int32_t* ends,
                       int64_t k, void* d, int d_format, bool overlap, cudaStream_t stream);

// Low-rank adapters in a large product (srs_adapter_product.cu).  The low part of tokens in their
// adapters' order enters as pairs of 16-bit numbers, high and what it leaves, in items of
// `edge` rows: an item is a tile of the product and one adapter that has tokens in it, other rows
// not written.  Item of tile i and the r-th adapter with tokens: i + r (each step along the tokens
// raises one of the two, so no two items share a number).  A row has the rank's high parts, in
// whole 16s, and the others behind them in one slice of 64 for ranks up to 32; else whole
// slices of 64 of high parts and then as many of the others.  A thin product's items have one row
// a token in the batch's order (zero but for the adapter's own), one item an adapter with tokens,
// and thin_columns rows.
struct PairShape {
  int pitch, rest_at;  // elements of a row, first of the second parts
  int slices;
};
inline PairShape pair_shape(int rank) {
  if (rank <= 32) return {64, (rank + 15) / 16 * 16, 1};
  const int wide = (rank + 63) / 64 * 64;
  return {2 * wide, wide, wide / 32};
}
inline int64_t pair_items(int64_t tokens, int64_t adapters, int64_t edge) {
  return (tokens + edge - 1) / edge + (adapters < tokens ? adapters : tokens);
}

int adapter_edge(int64_t tokens, int64_t n, int64_t k);  // of the tiles: 128 or 256
int launch_adapter_product(const srs_blocks& rows, const srs_blocks& w, int64_t k,
                           const AdapterCall& a, int edge, void* d, cudaStream_t stream);

}  // namespace srs
