// C ABI of the block-scaled e4m3 operators: the quantiser and the product (include/vecops_b200/decode_cuda.h).
#include <cuda_runtime.h>
#include <stdint.h>

#include "decode_shim.h"
#include "f8_generic.cuh"
#include "f8_quantize.cuh"

using namespace vb200;

namespace {

constexpr int64_t kExtentLimit = INT64_C(1) << 31;

template <typename T>
int32_t quantize_typed(const VecopsB200QuantizeBlocks& q, int sms, VecopsError* error) {
  F8QuantizeArgs p{q.src, q.src_stride_row, q.src_stride_col, static_cast<uint8_t*>(q.dst), q.dst_stride_row,
                   q.scale, q.scale_stride_row, q.scale_stride_col, q.rows, q.cols};
  // sixteen bytes per load and eight per store where every row allows it
  const bool vec = (q.src_stride_col == 1 || q.cols == 1) && decode_aligned(q.src, 16) &&
                   (q.rows == 1 || q.src_stride_row * static_cast<int64_t>(sizeof(T)) % 16 == 0) && decode_aligned(q.dst, 8) &&
                   (q.rows == 1 || q.dst_stride_row % 8 == 0);
  cudaStream_t stream = static_cast<cudaStream_t>(q.stream);
  const int64_t col_blocks = (q.cols + 127) / 128;
  if (q.block_rows == 1) {
    const int64_t want = (q.rows * col_blocks + 15) / 16;
    const unsigned grid = static_cast<unsigned>(want < static_cast<int64_t>(sms) * 64 ? want : static_cast<int64_t>(sms) * 64);
    if (vec) f8_quantize_rows_kernel<T, true><<<grid, 256, 0, stream>>>(p);
    else f8_quantize_rows_kernel<T, false><<<grid, 256, 0, stream>>>(p);
    return decode_launched("quantize_blocks", error);
  }
  const dim3 grid(static_cast<unsigned>(col_blocks), static_cast<unsigned>((q.rows + 127) / 128));
  if (grid.y > 65535u) return set_error(error, VECOPS_STATUS_INVALID_ARGUMENT, "quantize_blocks: more than 65535 x 128 rows");
  if (vec) f8_quantize_tiles_kernel<T, true><<<grid, 256, 0, stream>>>(p);
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

int32_t select_f8(const VecopsB200MatmulF8& p, uint32_t* kernel, VecopsError* error) {
  if (p.kernel == VECOPS_B200_F8_STREAM || p.kernel == VECOPS_B200_F8_TILED)
    return set_error(error, VECOPS_STATUS_NOT_APPLICABLE, "matmul_f8: kernel %u cannot serve this call", p.kernel);
  *kernel = VECOPS_B200_F8_GENERIC;
  return VECOPS_STATUS_OK;
}

int32_t run_generic(const VecopsB200MatmulF8& q, int sms, VecopsError* error) {
  const F8Args p{static_cast<const uint8_t*>(q.a), q.a_stride_m, q.a_stride_k, q.a_scale, q.a_scale_stride_m, q.a_scale_stride_k,
                 static_cast<const uint8_t*>(q.b), q.b_stride_n, q.b_stride_k, q.b_scale, q.b_scale_stride_n, q.b_scale_stride_k,
                 q.c, q.c_stride_m, q.c_stride_n, q.m, q.n, q.k};
  const int64_t tiles = ((q.m + 31) / 32) * ((q.n + 31) / 32);
  const unsigned grid = static_cast<unsigned>(tiles < static_cast<int64_t>(sms) * 64 ? tiles : static_cast<int64_t>(sms) * 64);
  cudaStream_t stream = static_cast<cudaStream_t>(q.stream);
  if (q.c_dtype == VECOPS_DTYPE_BF16) f8_generic_kernel<__nv_bfloat16><<<grid, 256, 0, stream>>>(p);
  else if (q.c_dtype == VECOPS_DTYPE_F16) f8_generic_kernel<__half><<<grid, 256, 0, stream>>>(p);
  else f8_generic_kernel<float><<<grid, 256, 0, stream>>>(p);
  return decode_launched("matmul_f8 (generic)", error);
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
  rc = run_generic(p, device.sms, error);
  if (rc != VECOPS_STATUS_OK) return rc;
  return decode_finish("matmul_f8", p.flags, p.stream, device.index, error);
}

}  // extern "C"
