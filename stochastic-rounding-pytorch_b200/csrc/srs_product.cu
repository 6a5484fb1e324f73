// Launches of the tensor-core products, and the products of FP8 blocks.
#include <mutex>
#include <unordered_map>

#include "srs_host.h"
#include "srs_launch.h"
#include "srs_product.cuh"
#include "srs_thin.cuh"

namespace srs {
namespace {

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                 const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                 const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

constexpr int kMaxDevices = 128;
std::mutex g_lock;
EncodeTiled g_encode = nullptr;
std::unordered_map<const void*, int> g_resident[kMaxDevices];
unsigned int* g_status[kMaxDevices];  // host memory: where a bounded wait ran out (0: nowhere)

int device_index(int* dev) {
  const cudaError_t e = cudaGetDevice(dev);
  if (e != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
  if (*dev < 0 || *dev >= kMaxDevices) return fail(SRS_ERR_UNSUPPORTED_DEVICE, "device %d", *dev);
  return SRS_OK;
}

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

}  // namespace

int encode_operand(const ProductOperand& o, int element_bytes, int64_t batch, int box_rows,
                   CUtensorMap* map) {
  EncodeTiled encode = nullptr;
  if (int rc = find_encode(&encode)) return rc;
  const uint64_t size = (uint64_t)element_bytes;
  const cuuint64_t dims[3] = {(cuuint64_t)(o.rows_inner ? o.rows : o.k),
                              (cuuint64_t)(o.rows_inner ? o.k : o.rows), (cuuint64_t)batch};
  const uint64_t entry = batch > 1 ? (uint64_t)o.batch_stride : (uint64_t)o.pitch * dims[1];
  const cuuint64_t strides[2] = {(cuuint64_t)o.pitch * size, entry * size};
  const cuuint32_t box[3] = {(cuuint32_t)(kSliceBytes / size),
                             o.rows_inner ? 64u : (cuuint32_t)box_rows, 1u};
  const cuuint32_t ones[3] = {1, 1, 1};
  const CUresult r = encode(
      map, size == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
      const_cast<void*>(o.base), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
      CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(SRS_ERR_CUDA,
                "cuTensorMapEncodeTiled failed (%d) for %lld x %lld, pitch %lld at %p", (int)r,
                (long long)o.rows, (long long)o.k, (long long)o.pitch, o.base);
  return SRS_OK;
}

int status_word(unsigned int** word) {
  int dev = 0;
  if (int rc = device_index(&dev)) return rc;
  std::lock_guard<std::mutex> lock(g_lock);
  if (g_status[dev] == nullptr) {
    void* p = nullptr;  // one address for the host and the device (unified addressing)
    const cudaError_t e =
        cudaHostAlloc(&p, sizeof(unsigned int), cudaHostAllocMapped | cudaHostAllocPortable);
    if (e != cudaSuccess) return cuda_fail(e, "cudaHostAlloc(product status)");
    g_status[dev] = static_cast<unsigned int*>(p);
    *g_status[dev] = 0u;
  }
  *word = g_status[dev];
  return SRS_OK;
}

int check_products() {
  unsigned int* word = nullptr;
  if (int rc = status_word(&word)) return rc;
  if (__atomic_load_n(word, __ATOMIC_RELAXED) == 0u) return SRS_OK;
  const unsigned int where = __atomic_exchange_n(word, 0u, __ATOMIC_RELAXED);
  return fail(SRS_ERR_WAIT,
              "a wait inside an earlier product kernel on this device ran out (0x%x): the results "
              "of product calls since the last check are not valid",
              where);
}

int prepare_kernel(const void* kernel, int group, int threads, int smem, int* resident) {
  int dev = 0;
  if (int rc = device_index(&dev)) return rc;
  const int sms = sm_count();
  {
    std::lock_guard<std::mutex> lock(g_lock);
    const auto it = g_resident[dev].find(kernel);
    if (it != g_resident[dev].end()) {
      *resident = it->second;
      return SRS_OK;
    }
  }
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return cuda_fail(e, "kernel shared memory");
  int groups = 0;
  if (group > 1) {
    cudaLaunchConfig_t config{};
    cudaLaunchAttribute cluster{};
    cluster.id = cudaLaunchAttributeClusterDimension;
    cluster.val.clusterDim.x = (unsigned)group;
    cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
    config.gridDim = dim3((unsigned)(sms / group * group));
    config.blockDim = dim3((unsigned)threads);
    config.dynamicSmemBytes = (size_t)smem;
    config.attrs = &cluster;
    config.numAttrs = 1;
    e = cudaOccupancyMaxActiveClusters(&groups, kernel, &config);
    if (e != cudaSuccess) return cuda_fail(e, "cudaOccupancyMaxActiveClusters");
    if (groups > sms / group) groups = sms / group;
  } else {
    e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&groups, kernel, threads, (size_t)smem);
    if (e != cudaSuccess) return cuda_fail(e, "cudaOccupancyMaxActiveBlocksPerMultiprocessor");
    groups *= sms;
    if (groups > sms) groups = sms;
  }
  if (groups < 1) return fail(SRS_ERR_CUDA, "the product kernel does not fit the device");
  std::lock_guard<std::mutex> lock(g_lock);
  g_resident[dev][kernel] = groups;
  *resident = groups;
  return SRS_OK;
}

int launch_groups(const void* kernel, int64_t groups, int group, int threads, int smem,
                  bool cooperative, void* argument, cudaStream_t stream, const char* what,
                  bool overlap) {
  cudaLaunchConfig_t config{};
  cudaLaunchAttribute attributes[3]{};
  config.gridDim = dim3((unsigned)(groups * group));
  config.blockDim = dim3((unsigned)threads);
  config.dynamicSmemBytes = (size_t)smem;
  config.stream = stream;
  config.attrs = attributes;
  if (group > 1) {
    cudaLaunchAttribute& a = attributes[config.numAttrs++];
    a.id = cudaLaunchAttributeClusterDimension;
    a.val.clusterDim.x = (unsigned)group;
    a.val.clusterDim.y = a.val.clusterDim.z = 1;
  }
  if (cooperative) {
    cudaLaunchAttribute& a = attributes[config.numAttrs++];
    a.id = cudaLaunchAttributeCooperative;
    a.val.cooperative = 1;
  }
  if (overlap) {
    cudaLaunchAttribute& a = attributes[config.numAttrs++];
    a.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    a.val.programmaticStreamSerializationAllowed = 1;
  }
  void* arguments[1] = {argument};
  const cudaError_t e = cudaLaunchKernelExC(&config, kernel, arguments);
  return e == cudaSuccess ? SRS_OK : cuda_fail(e, what);
}

namespace {

// One product of FP8 blocks: a single list of tiles.
struct BlockProduct {
  CUtensorMap map_a, map_b;
  int m, n, slices;
  TileGrid grid;
  uint32_t instruction_formats;
  const uint8_t* scale_a;
  const uint8_t* scale_b;
  int64_t scale_a_pitch, scale_b_pitch;
  int scale_a_shift, scale_b_shift;  // 7 when one scale covers 128 rows
  char* out;
  int format;
  unsigned int* status_at;
  int edge;  // of a tile
};

struct BlockScales {
  const uint8_t* a;
  const uint8_t* b;
  int64_t a_pitch, b_pitch;
  int a_shift, b_shift, m, n;
  bool a_words, b_words;
};

struct BlockSource {
  const BlockProduct& w;
  __device__ int phases() const { return 1; }
  __device__ uint32_t tiles(int) const { return w.grid.rows * w.grid.cols; }
  __device__ uint32_t formats() const { return w.instruction_formats; }
  __device__ unsigned int* counter(int) const { return nullptr; }
  __device__ unsigned int* status() const { return w.status_at; }
  __device__ int longest() const { return w.slices; }
  __device__ TileLoad load(int, uint32_t t) const {
    int row, col;
    w.grid.at(t, &row, &col);
    return {&w.map_a, &w.map_b, row * w.edge, col * w.edge, 0, w.slices, false, false};
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
    return s;
  }
  __device__ BlockScales scales() const {
    return {w.scale_a,       w.scale_b,       w.scale_a_pitch, w.scale_b_pitch,
            w.scale_a_shift, w.scale_b_shift, w.m,             w.n,
            scale_words(w.scale_a, w.scale_a_pitch, 0),
            scale_words(w.scale_b, w.scale_b_pitch, 0)};
  }
};

template <int CG>
__global__ void __launch_bounds__(ProductShape<kOperandF8, CG>::kThreads, 1)
block_product_kernel(const __grid_constant__ BlockProduct w) {
  run_products<kOperandF8, CG, false, false>(BlockSource{w});
}

template <int CG>
int launch_blocks(BlockProduct& w, cudaStream_t stream) {
  const void* kernel = reinterpret_cast<const void*>(&block_product_kernel<CG>);
  using S = ProductShape<kOperandF8, CG>;
  int resident = 0;
  if (int rc = prepare_kernel(kernel, CG, S::kThreads, S::kSmem, &resident)) return rc;
  const int64_t tiles = (int64_t)w.grid.rows * w.grid.cols;
  return launch_groups(kernel, tiles < resident ? tiles : resident, CG, S::kThreads, S::kSmem,
                       false, &w, stream, "block product launch");
}

int operand_map(const srs_blocks& b, int64_t k, int box_rows, CUtensorMap* map) {
  const ProductOperand o{reinterpret_cast<const void*>(b.data), b.rows, k, b.pitch, 0, false};
  return encode_operand(o, 1, 1, box_rows, map);
}

uint32_t format_bits(const srs_blocks& a, const srs_blocks& b) {
  return (a.format == SRS_FMT_E5M2 ? 1u : 0u) << 7 | (b.format == SRS_FMT_E5M2 ? 1u : 0u) << 10;
}

}  // namespace

int launch_block_product(const srs_blocks& a, const srs_blocks& b, int64_t k, void* d,
                         int d_format, cudaStream_t stream) {
  const auto tiles = [&](int64_t edge) {
    return ((a.rows + edge - 1) / edge) * ((b.rows + edge - 1) / edge);
  };
  // Rough times in cycles: 512 a slice for a 256 x 256 pair, 350 for a 128 x 128 tile
  // (256 of MMA, but twice the loads for it), and what a tile's results take.
  const int64_t sms = sm_count(), pairs = sms / 2, slices = (k + kSliceBytes - 1) / kSliceBytes;
  const double time_small = (350.0 * slices + 2000.0) * (double)((tiles(128) + sms - 1) / sms);
  const double time_large = (512.0 * slices + 5000.0) * (double)((tiles(256) + pairs - 1) / pairs);
  const int cg = time_large <= time_small ? 2 : 1;
  if (tiles(128 * cg) >= (1ll << 31))
    return fail(SRS_ERR_INVALID_ARGUMENT, "a result of %lld x %lld is too large",
                (long long)a.rows, (long long)b.rows);
  BlockProduct w{};
  if (int rc = operand_map(a, k, 128, &w.map_a)) return rc;
  if (int rc = operand_map(b, k, 128, &w.map_b)) return rc;
  if (int rc = status_word(&w.status_at)) return rc;
  w.m = (int)a.rows;
  w.n = (int)b.rows;
  w.slices = (int)((k + kSliceBytes - 1) / kSliceBytes);
  w.edge = 128 * cg;
  w.grid = make_grid((uint32_t)((a.rows + w.edge - 1) / w.edge),
                     (uint32_t)((b.rows + w.edge - 1) / w.edge));
  w.instruction_formats = format_bits(a, b);
  w.scale_a = reinterpret_cast<const uint8_t*>(a.scale);
  w.scale_b = reinterpret_cast<const uint8_t*>(b.scale);
  w.scale_a_pitch = a.scale_pitch;
  w.scale_b_pitch = b.scale_pitch;
  w.scale_a_shift = a.square ? 7 : 0;
  w.scale_b_shift = b.square ? 7 : 0;
  w.out = static_cast<char*>(d);
  w.format = d_format;
  return cg == 2 ? launch_blocks<2>(w, stream) : launch_blocks<1>(w, stream);
}

namespace {

template <int BN>
int launch_thin_as(ThinArgs& args, int splits, bool overlap, cudaStream_t stream) {
  using S = ThinShape<BN>;
  const void* kernel = reinterpret_cast<const void*>(&thin_product_kernel<BN>);
  // As many stages as fit before a whole panel: the MMA reads 128 rows from the start of
  // the last stage's panel, past the end of that stage when its tile has fewer.
  args.panel_bytes = (args.rows + 7) / 8 * 8 * kSliceBytes;
  const int stage = args.panel_bytes + BN * kSliceBytes, slack = kPanelBytes;
  args.stages = (S::kBudget - slack) / stage;
  if (args.stages > kThinMaxStages) args.stages = kThinMaxStages;
  if (args.stages < 2) return fail(SRS_ERR_CUDA, "thin product: no room for two stages");
  int bytes = args.stages * stage + slack;
  if (bytes < S::kSums) bytes = S::kSums;
  int resident = 0;
  if (int rc = prepare_kernel(kernel, 1, kThinThreads, S::kFixed + S::kBudget, &resident))
    return rc;
  return launch_groups(kernel, (args.m + args.rows - 1) / args.rows, splits, kThinThreads,
                       S::kFixed + bytes, false, &args, stream, "thin product launch", overlap);
}

}  // namespace

int launch_thin(const srs_blocks& a, const srs_blocks& b, int64_t k, void* d, int d_format,
                int64_t row_stride, int64_t col_stride, bool overlap, cudaStream_t stream) {
  const int columns = b.rows <= 16 ? 16 : b.rows <= 32 ? 32 : 64;
  ThinArgs args{};
  args.m = (int)a.rows;
  args.slices = (int)((k + kSliceBytes - 1) / kSliceBytes);
  // Tiles of 128 rows, k split while two CTAs an SM hold all of them and each keeps two
  // slices.  With more tiles than SMs nothing is split, and the tiles take the size
  // that fills whole rounds of two CTAs an SM: 28672 x 8192 by one token 44.7 -> 42.3 us.
  // (Such sizes below that, too: 4096 x 4096 in 74 tiles of 56 rows and clusters of four
  // 8.9 us, in 32 tiles and clusters of eight 7.5.)
  const int64_t sms = sm_count(), tiles = (a.rows + 127) / 128;
  int splits = 1;
  args.rows = 128;
  if (tiles > sms) {
    const int64_t rounds = (tiles + 2 * sms - 1) / (2 * sms);
    args.rows = (int)((a.rows + 2 * sms * rounds - 1) / (2 * sms * rounds));
  } else {
    while (splits < 8 && tiles * splits <= sms && args.slices >= 4 * splits) splits *= 2;
  }
  if (int rc = operand_map(a, k, args.rows, &args.map_a)) return rc;
  if (int rc = operand_map(b, k, columns, &args.map_b)) return rc;
  if (int rc = status_word(&args.status)) return rc;
  args.n = (int)b.rows;
  args.scale_a = reinterpret_cast<const uint8_t*>(a.scale);
  args.scale_b = reinterpret_cast<const uint8_t*>(b.scale);
  args.scale_a_pitch = a.scale_pitch;
  args.scale_b_pitch = b.scale_pitch;
  args.scale_a_shift = a.square ? 7 : 0;
  args.scale_b_shift = b.square ? 7 : 0;
  args.idesc = (uint32_t)(columns >> 3) << 17 | (128u >> 4) << 24 | format_bits(a, b) | 1u << 23;
  args.out = d;
  args.out_format = d_format;
  args.row_stride = row_stride;
  args.col_stride = col_stride;
  if (columns == 16) return launch_thin_as<16>(args, splits, overlap, stream);
  if (columns == 32) return launch_thin_as<32>(args, splits, overlap, stream);
  return launch_thin_as<64>(args, splits, overlap, stream);
}

}  // namespace srs

extern "C" int srs_product_status(uint32_t* status) {
  using namespace srs;
  clear_error();
  if (status == nullptr) return fail(SRS_ERR_INVALID_ARGUMENT, "null status");
  if (int rc = check_device()) return rc;
  unsigned int* word = nullptr;
  if (int rc = status_word(&word)) return rc;
  const cudaError_t e = cudaDeviceSynchronize();
  if (e != cudaSuccess) return cuda_fail(e, "product status");
  *status = __atomic_exchange_n(word, 0u, __ATOMIC_RELAXED);
  return SRS_OK;
}

extern "C" int srs_product_status_word(uint32_t** word) {
  using namespace srs;
  clear_error();
  if (word == nullptr) return fail(SRS_ERR_INVALID_ARGUMENT, "null word");
  if (int rc = check_device()) return rc;
  return status_word(word);
}
