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

// Tensor map of an operand: boxes of `box_rows` rows x 128 bytes of k, or of 64 rows x
// 64 k when the row index is contiguous; elements outside the operand read as zero.
int encode_operand(const ProductOperand& o, int element_bytes, int64_t batch, int box_rows,
                   CUtensorMap* map);

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

// FP8 blocks: d = a b^T (operands checked by the caller).  Element (i, j)
// of d is stored at i * row_stride + j * col_stride; only products with a thin side
// (at most kThinRows rows) take a col_stride other than 1.  `overlap`: the kernel ahead
// writes nothing of a.
constexpr int kThinRows = 64;
int launch_block_product(const srs_blocks& a, const srs_blocks& b, int64_t k, void* d,
                         int d_format, cudaStream_t stream);
int launch_thin(const srs_blocks& a, const srs_blocks& b, int64_t k, void* d, int d_format,
                int64_t row_stride, int64_t col_stride, bool overlap, cudaStream_t stream);

}  // namespace srs
