// Block quantiser to e4m3: the larger of 2^-110 and max |x| of a block becomes 448, everything else keeps its ratio to it.
//
//     amax = min(max(max |x|, 2^-110), largest f32)     scale = amax / 448     q = e4m3(x * (448 / amax))
//
// One division per block and one multiplication per element: x * (448 / amax) differs from x / scale by at most
// 1.5 fp32 roundings, 2^13 times finer than an e4m3 step.  Memory bound: an element is read once and one byte written.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <float.h>
#include <stdint.h>

namespace vb200 {

struct F8Quantize {
  static constexpr int kBlock = 128;
  static constexpr float kMax = 448.f;
  static constexpr float kAmaxFloor = 7.70371977754894341e-34f;  // 2^-110
};

template <typename T>
__device__ __forceinline__ float f8_source(T x);
template <>
__device__ __forceinline__ float f8_source<float>(float x) { return x; }
template <>
__device__ __forceinline__ float f8_source<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <>
__device__ __forceinline__ float f8_source<__half>(__half x) { return __half2float(x); }

// Eight consecutive elements of a row from column `col`; what lies past `cols` reads as zero.  kVec: the row starts on a
// 16-byte boundary and is contiguous, so eight elements that are all there come in 16-byte loads.
template <typename T, bool kVec>
__device__ __forceinline__ void f8_load8(const T* row, long long stride_col, long long col, long long cols, float (&x)[8]) {
  if (kVec && col + 8 <= cols) {
    uint4 raw[sizeof(T) / 2];
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) raw[i] = __ldg(reinterpret_cast<const uint4*>(row + col) + i);
    const T* values = reinterpret_cast<const T*>(raw);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = f8_source(values[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = col + e < cols ? f8_source(row[(col + e) * stride_col]) : 0.f;
  }
}

__device__ __forceinline__ float f8_block_amax(const float (&x)[8], float amax) {
#pragma unroll
  for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fabsf(x[e]));  // (fmaxf drops a NaN)
  return amax;
}

__device__ __forceinline__ float f8_bounded_amax(float amax) { return fminf(fmaxf(amax, F8Quantize::kAmaxFloor), FLT_MAX); }

template <bool kVec>
__device__ __forceinline__ void f8_store8(uint8_t* row, long long col, long long cols, const float (&x)[8], float factor) {
  uint16_t pairs[4];
#pragma unroll
  for (int e = 0; e < 4; ++e)
    pairs[e] = __nv_cvt_float2_to_fp8x2(make_float2(x[2 * e] * factor, x[2 * e + 1] * factor), __NV_SATFINITE, __NV_E4M3);
  if (kVec && col + 8 <= cols) {
    *reinterpret_cast<uint2*>(row + col) = make_uint2(pairs[0] | (static_cast<uint32_t>(pairs[1]) << 16), pairs[2] | (static_cast<uint32_t>(pairs[3]) << 16));
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (col + e < cols) row[col + e] = static_cast<uint8_t>(pairs[e >> 1] >> (8 * (e & 1)));
  }
}

struct F8QuantizeArgs {
  const void* src;
  long long src_sr, src_sc;
  uint8_t* dst;
  long long dst_sr;
  float* scale;
  long long scale_sr, scale_sc;
  long long rows, cols;
};

// 1 x 128 blocks: sixteen threads per block, eight elements each.
template <typename T, bool kVec>
__global__ void __launch_bounds__(256) f8_quantize_rows_kernel(const F8QuantizeArgs p) {
  const long long col_blocks = (p.cols + F8Quantize::kBlock - 1) / F8Quantize::kBlock;
  const long long total = p.rows * col_blocks;
  const int lane = threadIdx.x & 15;
  for (long long block = (blockIdx.x * 256ll + threadIdx.x) >> 4; block < total; block += gridDim.x * 16ll) {
    const long long row = block / col_blocks, col_block = block - row * col_blocks;
    const long long col = col_block * F8Quantize::kBlock + lane * 8;
    float x[8];
    f8_load8<T, kVec>(static_cast<const T*>(p.src) + row * p.src_sr, p.src_sc, col, p.cols, x);
    float amax = f8_block_amax(x, 0.f);
    const unsigned members = 0xffffu << (threadIdx.x & 16);  // the other half of the warp may be done
#pragma unroll
    for (int offset = 8; offset > 0; offset >>= 1) amax = fmaxf(amax, __shfl_xor_sync(members, amax, offset));
    amax = f8_bounded_amax(amax);
    f8_store8<kVec>(p.dst + row * p.dst_sr, col, p.cols, x, F8Quantize::kMax / amax);
    if (lane == 0) p.scale[row * p.scale_sr + col_block * p.scale_sc] = amax / F8Quantize::kMax;
  }
}

// 128 x 128 blocks: one CTA per block holds it in registers between the maximum and the conversion.
template <typename T, bool kVec>
__global__ void __launch_bounds__(256) f8_quantize_tiles_kernel(const F8QuantizeArgs p) {
  __shared__ float warp_amax[8];
  const long long row0 = blockIdx.y * static_cast<long long>(F8Quantize::kBlock) + (threadIdx.x >> 4);
  const long long col = blockIdx.x * static_cast<long long>(F8Quantize::kBlock) + (threadIdx.x & 15) * 8;
  float x[8][8];
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const long long row = row0 + 16 * i;
    f8_load8<T, kVec>(static_cast<const T*>(p.src) + (row < p.rows ? row : 0) * p.src_sr, p.src_sc, col, row < p.rows ? p.cols : 0, x[i]);
    amax = f8_block_amax(x[i], amax);
  }
#pragma unroll
  for (int offset = 16; offset > 0; offset >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, offset));
  if ((threadIdx.x & 31) == 0) warp_amax[threadIdx.x >> 5] = amax;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) amax = fmaxf(amax, warp_amax[w]);
  amax = f8_bounded_amax(amax);
  const float factor = F8Quantize::kMax / amax;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const long long row = row0 + 16 * i;
    if (row < p.rows) f8_store8<kVec>(p.dst + row * p.dst_sr, col, p.cols, x[i], factor);
  }
  if (threadIdx.x == 0) p.scale[blockIdx.y * p.scale_sr + blockIdx.x * p.scale_sc] = amax / F8Quantize::kMax;
}

}  // namespace vb200
