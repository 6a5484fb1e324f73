// Instantiations and launches of the tensor-core products.
#include <mutex>
#include <unordered_map>

#include "srs_host.h"
#include "srs_product.cuh"
#include "srs_thin.cuh"

namespace srs {
namespace {

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                 const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                 const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

std::mutex g_lock;
EncodeTiled g_encode = nullptr;
std::unordered_map<const void*, int> g_clusters[128];  // resident CTA groups per device

int find_encode(EncodeTiled* out) {
  std::lock_guard<std::mutex> lock(g_lock);
  if (g_encode == nullptr) {
    void* symbol = nullptr;
    cudaDriverEntryPointQueryResult found{};
    const cudaError_t e =
        cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &symbol, cudaEnableDefault, &found);
    if (e != cudaSuccess) return cuda_fail(e, "cudaGetDriverEntryPoint(cuTensorMapEncodeTiled)");
    if (found != cudaDriverEntryPointSuccess || symbol == nullptr)
      return fail(SRS_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
    g_encode = reinterpret_cast<EncodeTiled>(symbol);
  }
  *out = g_encode;
  return SRS_OK;
}

// Tensor map of one operand: boxes of 128 rows x 128 bytes of k, or of 64 rows
// x 64 k when the row index is contiguous; outside elements read as zero.
int encode_operand(const ProductOperand& o, int kind, int64_t batch, CUtensorMap* map,
                   uint32_t rows = 128) {
  EncodeTiled encode = nullptr;
  if (int rc = find_encode(&encode)) return rc;
  const uint64_t size = kind == kOperandF8 ? 1 : 2;
  const cuuint64_t dims[3] = {(cuuint64_t)(o.rows_inner ? o.rows : o.k),
                              (cuuint64_t)(o.rows_inner ? o.k : o.rows), (cuuint64_t)batch};
  const uint64_t entry = batch > 1 ? (uint64_t)o.batch_stride : (uint64_t)o.pitch * dims[1];
  const cuuint64_t strides[2] = {(cuuint64_t)o.pitch * size, entry * size};
  const cuuint32_t box[3] = {(cuuint32_t)(kSliceBytes / size), o.rows_inner ? 64u : rows, 1u};
  const cuuint32_t ones[3] = {1, 1, 1};
  const CUresult r = encode(
      map, kind == kOperandF8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
      const_cast<void*>(o.base), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
      CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(SRS_ERR_CUDA,
                "cuTensorMapEncodeTiled failed (%d) for %lld x %lld, pitch %lld at %p", (int)r,
                (long long)o.rows, (long long)o.k, (long long)o.pitch, o.base);
  return SRS_OK;
}

__device__ unsigned int g_product_status;  // where a bounded wait ran out (0: nowhere)

int status_word(unsigned int** word) {
  void* p = nullptr;
  const cudaError_t e = cudaGetSymbolAddress(&p, g_product_status);
  if (e != cudaSuccess) return cuda_fail(e, "cudaGetSymbolAddress(product status)");
  *word = static_cast<unsigned int*>(p);
  return SRS_OK;
}

template <int KIND, int CG, int EPILOGUE>
int launch(const CUtensorMap& map_a, const CUtensorMap& map_b, const ProductArgs& args,
           cudaStream_t stream) {
  using S = ProductShape<KIND, CG>;
  const auto kernel = &product_kernel<KIND, CG, EPILOGUE>;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
  cudaLaunchConfig_t config{};
  cudaLaunchAttribute cluster{};
  config.blockDim = dim3(kProductThreads);
  config.dynamicSmemBytes = S::kSmem;
  config.stream = stream;
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = CG;
  cluster.val.clusterDim.y = 1;
  cluster.val.clusterDim.z = 1;
  if (CG == 2) {
    config.attrs = &cluster;
    config.numAttrs = 1;
  }
  int groups = 0;
  {
    std::lock_guard<std::mutex> lock(g_lock);
    const auto it = g_clusters[dev].find(reinterpret_cast<const void*>(kernel));
    if (it != g_clusters[dev].end()) groups = it->second;
  }
  if (groups == 0) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem);
    if (e != cudaSuccess) return cuda_fail(e, "product shared memory");
    if (CG == 2) {
      config.gridDim = dim3((unsigned)(sm_count() / CG * CG));
      e = cudaOccupancyMaxActiveClusters(&groups, kernel, &config);
      if (e != cudaSuccess) return cuda_fail(e, "cudaOccupancyMaxActiveClusters");
      if (groups < 1) return fail(SRS_ERR_CUDA, "the product kernel's CTA pairs do not fit");
      if (groups > sm_count() / CG) groups = sm_count() / CG;
    } else {
      groups = sm_count();
    }
    std::lock_guard<std::mutex> lock(g_lock);
    g_clusters[dev][reinterpret_cast<const void*>(kernel)] = groups;
  }
  const int64_t used = args.n_tiles < groups ? args.n_tiles : groups;
  config.gridDim = dim3((unsigned)(used * CG));
  e = cudaLaunchKernelEx(&config, kernel, map_a, map_b, args);
  return e == cudaSuccess ? SRS_OK : cuda_fail(e, "product launch");
}

template <int KIND, int CG>
int launch_epilogue(int epilogue, const CUtensorMap& map_a, const CUtensorMap& map_b,
                    const ProductArgs& args, cudaStream_t stream) {
  if constexpr (KIND == kOperandF16) {
    if (epilogue == kEpilogueSymmetric)
      return launch<KIND, CG, kEpilogueSymmetric>(map_a, map_b, args, stream);
    if (epilogue == kEpilogueMuon)
      return launch<KIND, CG, kEpilogueMuon>(map_a, map_b, args, stream);
  }
  return launch<KIND, CG, kEpilogueStore>(map_a, map_b, args, stream);
}

int64_t tiles_for(int64_t m, int64_t n, int64_t edge, bool symmetric) {
  const int64_t tm = (m + edge - 1) / edge, tn = (n + edge - 1) / edge;
  return symmetric ? tm * (tm + 1) / 2 : tm * tn;
}

}  // namespace

int launch_product(int kind, int epilogue, const ProductOperand& a, const ProductOperand& b,
                   int64_t batch, int a_format, int b_format, ProductArgs args,
                   cudaStream_t stream) {
  const int sms = sm_count();
  // Time in units of one 128 x 128 tile on one SM: the 256 x 256 pair does two
  // such units per SM at a time; the single-CTA form loads twice the bytes per
  // unit, which makes its units about a fifth longer.
  const bool symmetric = args.symmetric != 0;
  const int64_t small = batch * tiles_for(a.rows, b.rows, 128, symmetric);
  const int64_t large = batch * tiles_for(a.rows, b.rows, 256, symmetric);
  const int64_t pairs = sms / 2;
  const double time_small = 1.2 * (double)((small + sms - 1) / sms);
  const double time_large = 2.0 * (double)((large + pairs - 1) / pairs);
  const int cg = time_large <= time_small ? 2 : 1;
  const int edge = 128 * cg;

  CUtensorMap map_a, map_b;
  if (int rc = encode_operand(a, kind, batch, &map_a)) return rc;
  if (int rc = encode_operand(b, kind, batch, &map_b)) return rc;
  if (int rc = status_word(&args.status)) return rc;
  args.m = (int)a.rows;
  args.n = (int)b.rows;
  args.k = (int)a.k;
  args.tiles_m = (int)((a.rows + edge - 1) / edge);
  args.tiles_n = (int)((b.rows + edge - 1) / edge);
  args.tiles_per_entry = cg == 2 ? large / batch : small / batch;
  args.n_tiles = batch * args.tiles_per_entry;
  args.a_rows_inner = a.rows_inner ? 1 : 0;
  args.b_rows_inner = b.rows_inner ? 1 : 0;
  // Instruction descriptor: operand formats, operand orders, N / 8, M / 16 and,
  // for FP16, FP32 accumulation; for FP8, UE8M0 scales.
  uint32_t idesc = (uint32_t)(edge >> 3) << 17 | (uint32_t)(edge >> 4) << 24;
  if (kind == kOperandF16) {
    idesc |= 1u << 4;
    if (a.rows_inner) idesc |= 1u << 15;
    if (b.rows_inner) idesc |= 1u << 16;
  } else {
    idesc |= (a_format == SRS_FMT_E5M2 ? 1u : 0u) << 7;
    idesc |= (b_format == SRS_FMT_E5M2 ? 1u : 0u) << 10;
    idesc |= 1u << 23;
  }
  args.idesc = idesc;
  if (kind == kOperandF16)
    return cg == 2 ? launch_epilogue<kOperandF16, 2>(epilogue, map_a, map_b, args, stream)
                   : launch_epilogue<kOperandF16, 1>(epilogue, map_a, map_b, args, stream);
  return cg == 2 ? launch_epilogue<kOperandF8, 2>(epilogue, map_a, map_b, args, stream)
                 : launch_epilogue<kOperandF8, 1>(epilogue, map_a, map_b, args, stream);
}

namespace {

template <int BN>
int launch_thin_as(const CUtensorMap& map_a, const CUtensorMap& map_b, const ThinArgs& args,
                   int splits, cudaStream_t stream) {
  using S = ThinShape<BN>;
  const auto kernel = &thin_product_kernel<BN>;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
  {
    std::lock_guard<std::mutex> lock(g_lock);
    int& set = g_clusters[dev][reinterpret_cast<const void*>(kernel)];
    if (set == 0) {
      e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem);
      if (e != cudaSuccess) return cuda_fail(e, "thin product shared memory");
      set = 1;
    }
  }
  cudaLaunchConfig_t config{};
  cudaLaunchAttribute cluster{};
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = (unsigned)splits;
  cluster.val.clusterDim.y = 1;
  cluster.val.clusterDim.z = 1;
  config.gridDim = dim3((unsigned)((args.m + 127) / 128 * splits));
  config.blockDim = dim3(kProductThreads);
  config.dynamicSmemBytes = S::kSmem;
  config.stream = stream;
  config.attrs = &cluster;
  config.numAttrs = 1;
  e = cudaLaunchKernelEx(&config, kernel, map_a, map_b, args);
  return e == cudaSuccess ? SRS_OK : cuda_fail(e, "thin product launch");
}

}  // namespace

int launch_thin(const ProductOperand& a, const ProductOperand& b, int a_format, int b_format,
                const ProductArgs& scales, void* out, int out_format, int64_t row_stride,
                int64_t col_stride, cudaStream_t stream) {
  const int columns = b.rows <= 16 ? 16 : b.rows <= 32 ? 32 : 64;
  CUtensorMap map_a, map_b;
  if (int rc = encode_operand(a, kOperandF8, 1, &map_a)) return rc;
  if (int rc = encode_operand(b, kOperandF8, 1, &map_b, (uint32_t)columns)) return rc;
  ThinArgs args{};
  if (int rc = status_word(&args.status)) return rc;
  args.m = (int)a.rows;
  args.n = (int)b.rows;
  args.slices = (int)((a.k + kSliceBytes - 1) / kSliceBytes);
  args.scale_a = scales.scale_a;
  args.scale_b = scales.scale_b;
  args.scale_a_pitch = scales.scale_a_pitch;
  args.scale_b_pitch = scales.scale_b_pitch;
  args.scale_a_shift = scales.scale_a_shift;
  args.scale_b_shift = scales.scale_b_shift;
  args.idesc = (uint32_t)(columns >> 3) << 17 | (128u >> 4) << 24 |
               (a_format == SRS_FMT_E5M2 ? 1u : 0u) << 7 |
               (b_format == SRS_FMT_E5M2 ? 1u : 0u) << 10 | 1u << 23;
  args.out = out;
  args.out_format = out_format;
  args.row_stride = row_stride;
  args.col_stride = col_stride;
  // Split k while all CTAs still fit at two an SM and each keeps two slices.
  const int64_t tiles = (a.rows + 127) / 128;
  int splits = 1;
  while (splits < 8 && tiles * splits * 2 <= 2ll * sm_count() && args.slices >= 4 * splits)
    splits *= 2;
  if (columns == 16) return launch_thin_as<16>(map_a, map_b, args, splits, stream);
  if (columns == 32) return launch_thin_as<32>(map_a, map_b, args, splits, stream);
  return launch_thin_as<64>(map_a, map_b, args, splits, stream);
}

int read_product_status(unsigned int* out) {
  const cudaError_t e = cudaMemcpyFromSymbol(out, g_product_status, sizeof(*out));
  return e == cudaSuccess ? SRS_OK : cuda_fail(e, "product status");
}

}  // namespace srs

extern "C" int srs_product_status(uint32_t* status) {
  using namespace srs;
  clear_error();
  if (status == nullptr) return fail(SRS_ERR_INVALID_ARGUMENT, "null status");
  if (int rc = check_device()) return rc;
  return read_product_status(status);
}
