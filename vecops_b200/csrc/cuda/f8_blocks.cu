// C ABI of the block-scaled e4m3 operators: the quantiser and the product (include/vecops_b200/decode_cuda.h).
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "decode_shim.h"
#include "f8_generic.cuh"
#include "f8_quantize.cuh"
#include "f8_stream.cuh"
#include "f8_tiled.cuh"

using namespace vb200;

namespace {

constexpr int64_t kExtentLimit = INT64_C(1) << 31;

template <typename T>
int32_t quantize_typed(const VecopsB200QuantizeBlocks& q, int sms, VecopsError* error) {
  F8QuantizeArgs p{q.src, q.src_stride_row, q.src_stride_col, static_cast<uint8_t*>(q.dst), q.dst_stride_row,
                   q.scale, q.scale_stride_row, q.scale_stride_col, q.rows, q.cols};
  // sixteen bytes per load and eight per store where every row allows it; four elements a lane where the rows of src are only contiguous
  const bool rows_ok = q.src_stride_col == 1 || q.cols == 1;
  const bool vec = rows_ok && decode_aligned(q.src, 16) && (q.rows == 1 || q.src_stride_row * static_cast<int64_t>(sizeof(T)) % 16 == 0) &&
                   decode_aligned(q.dst, 8) && (q.rows == 1 || q.dst_stride_row % 8 == 0);
  const bool unaligned = !vec && rows_ok && decode_aligned(q.dst, 4) && (q.rows == 1 || q.dst_stride_row % 4 == 0);
  cudaStream_t stream = static_cast<cudaStream_t>(q.stream);
  const int64_t col_blocks = (q.cols + 127) / 128;
  if (q.block_rows == 1) {
    const int64_t blocks = q.rows * col_blocks, per_cta = vec ? 32 : 16, most = static_cast<int64_t>(sms) * 8;
    const int64_t want = (blocks + per_cta - 1) / per_cta;
    const unsigned grid = static_cast<unsigned>(want < most ? want : most);
    if (vec) f8_quantize_rows_kernel<T><<<grid, 256, 0, stream>>>(p);
    else if (unaligned) f8_quantize_unaligned_rows_kernel<T><<<grid, 256, 0, stream>>>(p);
    else f8_quantize_strided_kernel<T><<<grid, 256, 0, stream>>>(p);
    return decode_launched("quantize_blocks", error);
  }
  const dim3 grid(static_cast<unsigned>(col_blocks), static_cast<unsigned>((q.rows + 127) / 128));
  if (grid.y > 65535u) return set_error(error, VECOPS_STATUS_INVALID_ARGUMENT, "quantize_blocks: more than 65535 x 128 rows");
  if (vec) f8_quantize_tiles_kernel<T, true><<<grid, 256, 0, stream>>>(p);
  else if (unaligned) f8_quantize_unaligned_tiles_kernel<T><<<grid, 256, 0, stream>>>(p);
  else f8_quantize_tiles_kernel<T, false><<<grid, 256, 0, stream>>>(p);
  return decode_launched("quantize_blocks", error);
}

int32_t check_f8(const VecopsB200MatmulF8& p, VecopsError* error) {
  if (p.m < 0 || p.n < 0 || p.k < 0 || p.m >= kExtentLimit || p.n >= kExtentLimit || p.k >= kExtentLimit)
    return set_error(error, VECOPS_STATUS_INVALID_ARGUMENT, "matmul_f8: extent out of range");
  if (p.c_dtype != VECOPS_DTYPE_BF16 && p.c_dtype != VECOPS_DTYPE_F16 && p.c_dtype != VECOPS_DTYPE_F32)
    return set_error(error, VECOPS_STATUS_INVALID_ARGUMENT, "matmul_f8 stores bf16, f16 or f32, not dtype %u", p.c_dtype);
  if (p.kernel >= VECOPS_B200_F8_COUNT_) return set_error(error, VECOPS_STATUS_INVALID_ARGUMENT, "matmul_f8: unknown kernel %u", p.kernel);
  if (p.a_stride_m < 0 || p.a_stride_k < 0 || p.b_stride_n < 0 || p.b_stride_k < 0 || p.a_scale_stride_m < 0 || p.a_scale_stride_k < 0 ||
      p.b_scale_stride_n < 0 || p.b_scale_stride_k < 0 || p.c_stride_m < 0 || p.c_stride_n < 0)
    return set_error(error, VECOPS_STATUS_INVALID_ARGUMENT, "matmul_f8: negative stride");
  if ((p.m > 1 && p.c_stride_m == 0) || (p.n > 1 && p.c_stride_n == 0))
    return set_error(error, VECOPS_STATUS_INVALID_ARGUMENT, "matmul_f8: elements of c share memory");
  return VECOPS_STATUS_OK;
}

// Whether TMA can address both operands: contiguous along K, rows on 16-byte boundaries; and whether the tiles' coordinates, which
// reach past an extent by less than a tile, fit 32 bits.
bool f8_addressable(const VecopsB200MatmulF8& p) {
  constexpr int64_t kTiledLimit = kExtentLimit - 256;
  if (p.m > kTiledLimit || p.n > kTiledLimit || p.k > kTiledLimit) return false;
  auto rows = [&](const void* base, int64_t count, int64_t stride, int64_t stride_k) {
    return (stride_k == 1 || p.k == 1) && decode_aligned(base, 16) && (count == 1 || (stride % 16 == 0 && stride >= p.k));
  };
  return p.k > 0 && rows(p.a, p.m, p.a_stride_m, p.a_stride_k) && rows(p.b, p.n, p.b_stride_n, p.b_stride_k);
}

constexpr int64_t kStreamRows = 128;  // rows of A the streaming kernel holds at most

int32_t select_f8(const VecopsB200MatmulF8& p, uint32_t* kernel, VecopsError* error) {
  const bool addressable = f8_addressable(p);
  if ((p.kernel == VECOPS_B200_F8_STREAM || p.kernel == VECOPS_B200_F8_TILED) && !addressable)
    return set_error(error, VECOPS_STATUS_NOT_APPLICABLE, "matmul_f8: kernel %u needs operands contiguous along K on 16-byte aligned rows, and extents up to 2^31 - 256", p.kernel);
  if (p.kernel == VECOPS_B200_F8_STREAM && p.m > kStreamRows)
    return set_error(error, VECOPS_STATUS_NOT_APPLICABLE, "matmul_f8: the streaming kernel serves up to %lld rows, not %lld", (long long)kStreamRows, (long long)p.m);
  if (p.kernel != VECOPS_B200_F8_AUTO) *kernel = p.kernel;
  else if (!addressable) *kernel = VECOPS_B200_F8_GENERIC;
  else *kernel = p.m <= kStreamRows ? VECOPS_B200_F8_STREAM : VECOPS_B200_F8_TILED;
  return VECOPS_STATUS_OK;
}

// Lets `kernel` use `bytes` of shared memory on `device`, once per device.
int32_t raise_shared(const void* kernel, int bytes, int device, std::atomic<bool>* raised, VecopsError* error) {
  if (device >= 0 && device < 64 && raised[device].load()) return VECOPS_STATUS_OK;
  const cudaError_t status = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (status != cudaSuccess) return set_error(error, VECOPS_STATUS_EXECUTION_ERROR, "cudaFuncSetAttribute(matmul_f8): %s", cudaGetErrorString(status));
  if (device >= 0 && device < 64) raised[device].store(true);
  return VECOPS_STATUS_OK;
}

int32_t f8_operand_map(CUtensorMap* map, const void* base, int64_t rows, int64_t k, int64_t stride, uint32_t box_rows, VecopsError* error) {
  const uint64_t dims[2] = {static_cast<uint64_t>(k), static_cast<uint64_t>(rows)};
  const uint64_t strides[1] = {static_cast<uint64_t>(rows == 1 ? (k + 15) / 16 * 16 : stride)};
  const uint32_t box[2] = {128, box_rows};
  return shim_encode_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, base, dims, strides, box, error);
}

F8StreamArgs f8_args(const VecopsB200MatmulF8& q, uint32_t* status) {
  return {q.a_scale, q.a_scale_stride_m, q.a_scale_stride_k, q.b_scale, q.b_scale_stride_n, q.b_scale_stride_k, q.c, q.c_stride_m, q.c_stride_n,
          static_cast<int>(q.m), static_cast<int>(q.n), static_cast<int>(q.k), status};
}

// One launch, cluster of `cluster` CTAs along x, as a programmatic dependent: the kernel's set-up overlaps the end of the one before it.
cudaError_t launch_f8(const void* kernel, unsigned grid, int threads, int smem, int cluster, cudaStream_t stream, void** args) {
  cudaLaunchConfig_t config = {};
  cudaLaunchAttribute attributes[2] = {};
  attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attributes[0].val.programmaticStreamSerializationAllowed = 1;
  attributes[1].id = cudaLaunchAttributeClusterDimension;
  attributes[1].val.clusterDim.x = static_cast<unsigned>(cluster);
  attributes[1].val.clusterDim.y = attributes[1].val.clusterDim.z = 1;
  config.gridDim = dim3(grid);
  config.blockDim = dim3(static_cast<unsigned>(threads));
  config.dynamicSmemBytes = static_cast<size_t>(smem);
  config.stream = stream;
  config.attrs = attributes;
  config.numAttrs = 2;
  return cudaLaunchKernelExC(&config, kernel, args);
}

// How many clusters of `cluster` CTAs of the tiled kernel (all its variants take the same resources) run at once.
int resident_clusters(const void* kernel, int threads, int smem, int cluster, int device) {
  static std::atomic<int> known[64][4];  // [device][log2 of the cluster], the count plus one
  const int bits = cluster == 8 ? 3 : cluster == 4 ? 2 : 1;
  if (device >= 0 && device < 64 && known[device][bits].load() > 0) return known[device][bits].load() - 1;
  cudaLaunchConfig_t config = {};
  cudaLaunchAttribute attribute = {};
  attribute.id = cudaLaunchAttributeClusterDimension;
  attribute.val.clusterDim.x = static_cast<unsigned>(cluster);
  attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
  config.gridDim = dim3(static_cast<unsigned>(cluster));
  config.blockDim = dim3(static_cast<unsigned>(threads));
  config.dynamicSmemBytes = static_cast<size_t>(smem);
  config.attrs = &attribute;
  config.numAttrs = 1;
  int clusters = 0;
  if (cudaOccupancyMaxActiveClusters(&clusters, kernel, &config) != cudaSuccess) clusters = 0;
  (void)cudaGetLastError();
  if (device >= 0 && device < 64) known[device][bits].store(clusters + 1);
  return clusters;
}

template <int kCols, typename OutT>
int32_t run_stream_typed(const VecopsB200MatmulF8& q, const DecodeDevice& device, VecopsError* error) {
  using G = F8Stream<kCols>;
  static std::atomic<bool> raised[64];
  const void* kernel = reinterpret_cast<const void*>(f8_stream_kernel<kCols, OutT>);
  int32_t rc = raise_shared(kernel, G::kSmemBytes, device.index, raised, error);
  if (rc != VECOPS_STATUS_OK) return rc;
  CUtensorMap map_w, map_x;
  rc = f8_operand_map(&map_w, q.b, q.n, q.k, q.b_stride_n, G::kRows, error);
  if (rc != VECOPS_STATUS_OK) return rc;
  rc = f8_operand_map(&map_x, q.a, q.m, q.k, q.a_stride_m, G::kCols, error);
  if (rc != VECOPS_STATUS_OK) return rc;
  // as many slices of K as there are SMs for, each at least two blocks long
  const int64_t tiles = (q.n + G::kRows - 1) / G::kRows, blocks = (q.k + 127) / 128;
  int slice_bits = 0;
  while (slice_bits < 3 && (tiles << (slice_bits + 1)) <= device.sms && blocks >= (4 << slice_bits)) ++slice_bits;
  const int slices = 1 << slice_bits;
  if (tiles * slices > 0x7fffffff) return set_error(error, VECOPS_STATUS_INVALID_ARGUMENT, "matmul_f8: N out of range");
  F8StreamArgs p = f8_args(q, device.status);
  void* args[] = {&map_w, &map_x, &p, &slice_bits};
  const cudaError_t status = launch_f8(kernel, static_cast<unsigned>(tiles * slices), G::kThreads, G::kSmemBytes, slices, static_cast<cudaStream_t>(q.stream), args);
  if (status != cudaSuccess) return set_error(error, VECOPS_STATUS_EXECUTION_ERROR, "matmul_f8 (stream) launch: %s", cudaGetErrorString(status));
  return decode_launched("matmul_f8 (stream)", error);
}

template <typename OutT>
int32_t run_stream(const VecopsB200MatmulF8& q, const DecodeDevice& device, VecopsError* error) {
  if (q.m <= 16) return run_stream_typed<16, OutT>(q, device, error);
  if (q.m <= 32) return run_stream_typed<32, OutT>(q, device, error);
  if (q.m <= 64) return run_stream_typed<64, OutT>(q, device, error);
  return run_stream_typed<128, OutT>(q, device, error);
}

template <typename OutT>
int32_t run_tiled(const VecopsB200MatmulF8& q, const DecodeDevice& device, VecopsError* error) {
  using G = F8Tiled;
  static std::atomic<bool> raised[64];
  const void* kernel = reinterpret_cast<const void*>(f8_tiled_kernel<OutT>);
  int32_t rc = raise_shared(kernel, G::kSmemBytes, device.index, raised, error);
  if (rc != VECOPS_STATUS_OK) return rc;
  CUtensorMap map_a, map_b, map_c;
  rc = f8_operand_map(&map_a, q.a, q.m, q.k, q.a_stride_m, 128, error);
  if (rc != VECOPS_STATUS_OK) return rc;
  rc = f8_operand_map(&map_b, q.b, q.n, q.k, q.b_stride_n, 128, error);
  if (rc != VECOPS_STATUS_OK) return rc;
  constexpr int64_t kElem = sizeof(OutT);
  int tma_store = q.c_stride_n == 1 && decode_aligned(q.c, 16) && q.c_stride_m * kElem % 16 == 0 && q.c_stride_m >= q.n ? 1 : 0;
  map_c = map_a;
  if (tma_store) {
    const uint64_t dims[2] = {static_cast<uint64_t>(q.n), static_cast<uint64_t>(q.m)};
    const uint64_t strides[1] = {static_cast<uint64_t>(q.c_stride_m * kElem)};
    const uint32_t box[2] = {static_cast<uint32_t>(128 / kElem), G::kOutRows};
    const CUtensorMapDataType type = q.c_dtype == VECOPS_DTYPE_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                     : q.c_dtype == VECOPS_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    rc = shim_encode_map(&map_c, type, 2, q.c, dims, strides, box, error);
    if (rc != VECOPS_STATUS_OK) return rc;
  }
  const int64_t tiles_m = (q.m + G::kTile - 1) / G::kTile, tiles_n = (q.n + G::kTile - 1) / G::kTile;
  if (tiles_m * tiles_n > 0x7fffffff) return set_error(error, VECOPS_STATUS_INVALID_ARGUMENT, "matmul_f8: too many tiles");
  const int64_t tiles = tiles_m * tiles_n, blocks = (q.k + 127) / 128;
  int slice_bits = 0;
  while (slice_bits < 2 && blocks >= (8 << slice_bits) && tiles <= resident_clusters(kernel, G::kThreads, G::kSmemBytes, 4 << slice_bits, device.index)) ++slice_bits;
  const int64_t workers = tiles < device.sms / 2 ? tiles : device.sms / 2;
  const int64_t group = G::kGroupBytes / (static_cast<int64_t>(G::kTile) * (q.k < 1 ? 1 : q.k));
  int raster_group = static_cast<int>(group < 1 ? 1 : group < tiles_m ? group : tiles_m);
  F8StreamArgs p = f8_args(q, device.status);
  void* args[] = {&map_a, &map_b, &map_c, &p, &tma_store, &raster_group, &slice_bits};
  const cudaError_t status = launch_f8(kernel, static_cast<unsigned>(2 * workers << slice_bits), G::kThreads, G::kSmemBytes, 2 << slice_bits, static_cast<cudaStream_t>(q.stream), args);
  if (status != cudaSuccess) return set_error(error, VECOPS_STATUS_EXECUTION_ERROR, "matmul_f8 (tiled) launch: %s", cudaGetErrorString(status));
  return decode_launched("matmul_f8 (tiled)", error);
}

template <typename OutT>
int32_t run_generic(const VecopsB200MatmulF8& q, int sms, VecopsError* error) {
  const F8Args p{static_cast<const uint8_t*>(q.a), q.a_stride_m, q.a_stride_k, q.a_scale, q.a_scale_stride_m, q.a_scale_stride_k,
                 static_cast<const uint8_t*>(q.b), q.b_stride_n, q.b_stride_k, q.b_scale, q.b_scale_stride_n, q.b_scale_stride_k,
                 q.c, q.c_stride_m, q.c_stride_n, q.m, q.n, q.k};
  const int64_t tiles = ((q.m + 31) / 32) * ((q.n + 31) / 32);
  const unsigned grid = static_cast<unsigned>(tiles < static_cast<int64_t>(sms) * 64 ? tiles : static_cast<int64_t>(sms) * 64);
  cudaStream_t stream = static_cast<cudaStream_t>(q.stream);
  f8_generic_kernel<OutT><<<grid, 256, 0, stream>>>(p);
  return decode_launched("matmul_f8 (generic)", error);
}

template <typename OutT>
int32_t run_f8(uint32_t kernel, const VecopsB200MatmulF8& q, const DecodeDevice& device, VecopsError* error) {
  if (kernel == VECOPS_B200_F8_STREAM) return run_stream<OutT>(q, device, error);
  if (kernel == VECOPS_B200_F8_TILED) return run_tiled<OutT>(q, device, error);
  return run_generic<OutT>(q, device.sms, error);
}

}  // namespace

extern "C" {

int32_t vecops_b200_quantize_blocks(const VecopsB200QuantizeBlocks* quantize, VecopsError* error) {
  if (quantize == nullptr || quantize->struct_size < sizeof(VecopsB200QuantizeBlocks))
    return set_error(error, VECOPS_STATUS_ABI_MISMATCH, "quantize record is null or too small");
  const VecopsB200QuantizeBlocks& q = *quantize;
  if (q.block_rows != 1 && q.block_rows != 128)
    return set_error(error, VECOPS_STATUS_INVALID_ARGUMENT, "quantize_blocks: block_rows is 1 or 128, not %u", q.block_rows);
  if (q.src_dtype != VECOPS_DTYPE_F32 && q.src_dtype != VECOPS_DTYPE_BF16 && q.src_dtype != VECOPS_DTYPE_F16)
    return set_error(error, VECOPS_STATUS_INVALID_ARGUMENT, "quantize_blocks reads f32, bf16 or f16, not dtype %u", q.src_dtype);
  if (q.rows < 0 || q.cols < 0 || q.rows >= kExtentLimit || q.cols >= kExtentLimit)
    return set_error(error, VECOPS_STATUS_INVALID_ARGUMENT, "quantize_blocks: extent out of range");
  if (q.src_stride_row < 0 || q.src_stride_col < 0 || q.scale_stride_row < 0 || q.scale_stride_col < 0)
    return set_error(error, VECOPS_STATUS_INVALID_ARGUMENT, "quantize_blocks: negative stride");
  if (q.rows == 0 || q.cols == 0) return VECOPS_STATUS_OK;
  if (q.rows > 1 && q.dst_stride_row < q.cols)
    return set_error(error, VECOPS_STATUS_INVALID_ARGUMENT, "quantize_blocks: rows of dst overlap (pitch %lld for %lld columns)",
                     (long long)q.dst_stride_row, (long long)q.cols);
  if ((q.rows > q.block_rows && q.scale_stride_row == 0) || (q.cols > 128 && q.scale_stride_col == 0))
    return set_error(error, VECOPS_STATUS_INVALID_ARGUMENT, "quantize_blocks: scales share memory");
  if (q.src == nullptr || q.dst == nullptr || q.scale == nullptr) return set_error(error, VECOPS_STATUS_INVALID_ARGUMENT, "quantize_blocks: null pointer");
  const DeviceRestore restore;
  DecodeDevice device;
  int32_t rc = decode_enter(q.device_index, &device, error);
  if (rc != VECOPS_STATUS_OK) return rc;
  if (q.src_dtype == VECOPS_DTYPE_F32) rc = quantize_typed<float>(q, device.sms, error);
  else if (q.src_dtype == VECOPS_DTYPE_BF16) rc = quantize_typed<__nv_bfloat16>(q, device.sms, error);
  else rc = quantize_typed<__half>(q, device.sms, error);
  if (rc != VECOPS_STATUS_OK) return rc;
  return decode_finish("quantize_blocks", q.flags, q.stream, device.index, error);
}

int32_t vecops_b200_matmul_f8_select(const VecopsB200MatmulF8* problem, uint32_t* kernel, VecopsError* error) {
  if (problem == nullptr || problem->struct_size < sizeof(VecopsB200MatmulF8) || kernel == nullptr)
    return set_error(error, VECOPS_STATUS_ABI_MISMATCH, "matmul_f8 record is null or too small, or no output pointer");
  const int32_t rc = check_f8(*problem, error);
  return rc != VECOPS_STATUS_OK ? rc : select_f8(*problem, kernel, error);
}

int32_t vecops_b200_matmul_f8_run(const VecopsB200MatmulF8* problem, VecopsError* error) {
  if (problem == nullptr || problem->struct_size < sizeof(VecopsB200MatmulF8))
    return set_error(error, VECOPS_STATUS_ABI_MISMATCH, "matmul_f8 record is null or too small");
  const VecopsB200MatmulF8& p = *problem;
  int32_t rc = check_f8(p, error);
  if (rc != VECOPS_STATUS_OK) return rc;
  uint32_t kernel = 0;
  rc = select_f8(p, &kernel, error);
  if (rc != VECOPS_STATUS_OK) return rc;
  if (p.m == 0 || p.n == 0) return VECOPS_STATUS_OK;
  if (p.c == nullptr || (p.k > 0 && (p.a == nullptr || p.b == nullptr || p.a_scale == nullptr || p.b_scale == nullptr)))
    return set_error(error, VECOPS_STATUS_INVALID_ARGUMENT, "matmul_f8: null pointer");
  const DeviceRestore restore;
  DecodeDevice device;
  rc = decode_enter(p.device_index, &device, error);
  if (rc != VECOPS_STATUS_OK) return rc;
  if (p.c_dtype == VECOPS_DTYPE_BF16) rc = run_f8<__nv_bfloat16>(kernel, p, device, error);
  else if (p.c_dtype == VECOPS_DTYPE_F16) rc = run_f8<__half>(kernel, p, device, error);
  else rc = run_f8<float>(kernel, p, device, error);
  if (rc != VECOPS_STATUS_OK) return rc;
  return decode_finish("matmul_f8", p.flags, p.stream, device.index, error);
}

}  // extern "C"
