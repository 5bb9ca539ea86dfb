// Block quantiser to e4m3: the larger of 2^-110 and max |x| of a block becomes 448, everything else keeps its ratio to it.
//
//     amax = min(max(max |x|, 2^-110), largest f32)     scale = amax / 448     q = e4m3(x * (448 / amax))
//
// One division per block and one multiplication per element: x * (448 / amax) differs from x / scale by at most
// 1.5 fp32 roundings, 2^13 times finer than an e4m3 step.  Memory bound: an element is read once and one byte written.
// Measured at 4096 x 14336 bf16 (178 MB): 32 us for 1 x 128 blocks, 33.5 us for 128 x 128, 5.5 and 5.3 TB/s; fp32 (295 MB): 46 and 59
// us, 6.4 and 5.0 TB/s (a CTA of the tile kernel holds twice the registers, so fewer of them load at once).  Rows off 16-byte
// boundaries, 1322 x 12485 bf16 (50 MB): 15.3 and 17 us, 3.2 and 2.9 TB/s; by the kernel for any strides 32 us.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <float.h>
#include <stdint.h>

#include <type_traits>

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

// Eight neighbouring elements of a row of any stride from column `col` on; what lies past `cols` reads as zero.
template <typename T>
__device__ __forceinline__ void f8_load8(const T* row, long long stride_col, long long col, long long cols, float (&x)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = col + e < cols ? f8_source(row[(col + e) * stride_col]) : 0.f;
}

__device__ __forceinline__ float f8_block_amax(const float (&x)[8], float amax) {
#pragma unroll
  for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fabsf(x[e]));  // (fmaxf drops a NaN)
  return amax;
}

__device__ __forceinline__ float f8_bounded_amax(float amax) { return fminf(fmaxf(amax, F8Quantize::kAmaxFloor), FLT_MAX); }

__device__ __forceinline__ void f8_store8(uint8_t* row, long long col, long long cols, const float (&x)[8], float factor) {
  uint16_t pairs[4];
#pragma unroll
  for (int e = 0; e < 4; ++e)
    pairs[e] = __nv_cvt_float2_to_fp8x2(make_float2(x[2 * e] * factor, x[2 * e + 1] * factor), __NV_SATFINITE, __NV_E4M3);
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (col + e < cols) row[col + e] = static_cast<uint8_t>(pairs[e >> 1] >> (8 * (e & 1)));
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

// The largest of amax and eight elements that still lie as they were loaded; a NaN does not count.
template <typename T>
__device__ __forceinline__ float f8_raw_amax(const uint4& raw) {
  if constexpr (sizeof(T) == 2) {
    // two at a time: the sign bits off, packed maxima
    uint32_t top = raw.x & 0x7fff7fffu;
    const uint32_t words[3] = {raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      const uint32_t w = words[i] & 0x7fff7fffu;
      if constexpr (std::is_same<T, __half>::value) asm("max.f16x2 %0, %0, %1;" : "+r"(top) : "r"(w));
      else asm("max.bf16x2 %0, %0, %1;" : "+r"(top) : "r"(w));
    }
    const T* pair = reinterpret_cast<const T*>(&top);
    return fmaxf(f8_source(pair[0]), f8_source(pair[1]));
  } else {
    const float* x = reinterpret_cast<const float*>(&raw);
    return fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
  }
}

// The 16 bytes' worth of elements, scaled, rounded and stored; `left` of them are inside the row.
template <typename T, bool kVec>
__device__ __forceinline__ void f8_store_raw(uint8_t* dst, const uint4& raw, float factor, int left) {
  constexpr int kPerLoad = 16 / sizeof(T);
  const T* x = reinterpret_cast<const T*>(&raw);
  uint32_t words[kPerLoad / 4];
#pragma unroll
  for (int w = 0; w < kPerLoad / 4; ++w) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(f8_source(x[4 * w]) * factor, f8_source(x[4 * w + 1]) * factor), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(f8_source(x[4 * w + 2]) * factor, f8_source(x[4 * w + 3]) * factor), __NV_SATFINITE, __NV_E4M3);
    words[w] = lo | hi << 16;
  }
  if (kVec && left >= kPerLoad) {
    if constexpr (kPerLoad == 8) *reinterpret_cast<uint2*>(dst) = make_uint2(words[0], words[1]);
    else *reinterpret_cast<uint32_t*>(dst) = words[0];
  } else {
#pragma unroll
    for (int e = 0; e < kPerLoad; ++e)
      if (e < left) dst[e] = static_cast<uint8_t>(words[e >> 2] >> (8 * (e & 3)));
  }
}

// Four elements, scaled, rounded and stored in one word (dst is on a 4-byte boundary); `left` of them are inside the row.
__device__ __forceinline__ void f8_store4(uint8_t* dst, const float (&x)[4], float factor, int left) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(x[0] * factor, x[1] * factor), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(x[2] * factor, x[3] * factor), __NV_SATFINITE, __NV_E4M3);
  const uint32_t word = lo | hi << 16;
  if (left >= 4) {
    *reinterpret_cast<uint32_t*>(dst) = word;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < left) dst[e] = static_cast<uint8_t>(word >> (8 * e));
  }
}

// 1 x 128 blocks of rows that allow 16-byte loads: eight threads a block, the elements held as loaded between the maximum
// and the conversion; two blocks' loads in flight per thread.  One division a block gives both the factor (lanes 0..6) and the
// scale (lane 7).  Instructions bound it as much as memory does: 20 an element, in a first form that converted before it
// compared and divided twice, moved 3.0 TB/s.
template <typename T>
__global__ void __launch_bounds__(256) f8_quantize_rows_kernel(const F8QuantizeArgs p) {
  constexpr int kPerLoad = 16 / sizeof(T), kLoads = F8Quantize::kBlock / 8 / kPerLoad, kTogether = sizeof(T) == 4 ? 1 : 2;
  const int col_blocks = static_cast<int>((p.cols + F8Quantize::kBlock - 1) / F8Quantize::kBlock);
  const int lane = threadIdx.x & 7;
  const unsigned members = 0xffu << (threadIdx.x & 24);
  // blocks are counted along the rows; from one to this thread group's next one by adding, not by dividing
  const long long step = gridDim.x * 32ll;
  const long long step_rows = step / col_blocks;
  const int step_cols = static_cast<int>(step - step_rows * col_blocks);
  const long long start = blockIdx.x * 32ll + (threadIdx.x >> 3);
  long long row = start / col_blocks;
  int col_block = static_cast<int>(start - row * col_blocks);
  while (row < p.rows) {
    uint4 raw[kTogether][kLoads];
    long long rows[kTogether];
    int cols[kTogether];
#pragma unroll
    for (int i = 0; i < kTogether; ++i) {
      rows[i] = row, cols[i] = col_block;
      const T* src = static_cast<const T*>(p.src) + row * p.src_sr + col_block * F8Quantize::kBlock;
      const int left = static_cast<int>(min(static_cast<long long>(F8Quantize::kBlock), p.cols - col_block * static_cast<long long>(F8Quantize::kBlock)));
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        const int at = (j * 8 + lane) * kPerLoad;
        raw[i][j] = make_uint4(0, 0, 0, 0);
        if (row < p.rows) {
          if (at + kPerLoad <= left) {
            raw[i][j] = __ldg(reinterpret_cast<const uint4*>(src + at));
          } else if (at < left) {
            T* x = reinterpret_cast<T*>(&raw[i][j]);
            for (int e = 0; e < kPerLoad; ++e)
              if (at + e < left) x[e] = src[at + e];
          }
        }
      }
      row += step_rows, col_block += step_cols;
      if (col_block >= col_blocks) col_block -= col_blocks, ++row;
    }
#pragma unroll
    for (int i = 0; i < kTogether; ++i) {
      if (rows[i] >= p.rows) break;
      float amax = f8_raw_amax<T>(raw[i][0]);
#pragma unroll
      for (int j = 1; j < kLoads; ++j) amax = fmaxf(amax, f8_raw_amax<T>(raw[i][j]));
#pragma unroll
      for (int offset = 4; offset > 0; offset >>= 1) amax = fmaxf(amax, __shfl_xor_sync(members, amax, offset));
      amax = f8_bounded_amax(amax);
      const float ratio = (lane == 7 ? amax : F8Quantize::kMax) / (lane == 7 ? F8Quantize::kMax : amax);
      const float factor = __shfl_sync(members, ratio, 0, 8);
      if (lane == 7) p.scale[rows[i] * p.scale_sr + cols[i] * p.scale_sc] = ratio;
      uint8_t* dst = p.dst + rows[i] * p.dst_sr + cols[i] * static_cast<long long>(F8Quantize::kBlock);
      const int left = static_cast<int>(min(static_cast<long long>(F8Quantize::kBlock), p.cols - cols[i] * static_cast<long long>(F8Quantize::kBlock)));
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        const int at = (j * 8 + lane) * kPerLoad;
        f8_store_raw<T, true>(dst + at, raw[i][j], factor, left - at);
      }
    }
  }
}

// 1 x 128 blocks of rows that are contiguous but off 16-byte boundaries: sixteen threads a block, twice four neighbouring
// elements each, one load an element, two blocks' loads in flight together.
template <typename T>
__global__ void __launch_bounds__(256) f8_quantize_unaligned_rows_kernel(const F8QuantizeArgs p) {
  constexpr int kTogether = 2;
  const int col_blocks = static_cast<int>((p.cols + F8Quantize::kBlock - 1) / F8Quantize::kBlock);
  const int lane = threadIdx.x & 15;
  const unsigned members = 0xffffu << (threadIdx.x & 16);
  const long long step = gridDim.x * 16ll;
  const long long step_rows = step / col_blocks;
  const int step_cols = static_cast<int>(step - step_rows * col_blocks);
  const long long start = blockIdx.x * 16ll + (threadIdx.x >> 4);
  long long row = start / col_blocks;
  int col_block = static_cast<int>(start - row * col_blocks);
  while (row < p.rows) {
    T raw[kTogether][2][4];
    long long rows[kTogether];
    int cols[kTogether];
#pragma unroll
    for (int i = 0; i < kTogether; ++i) {
      rows[i] = row, cols[i] = col_block;
      const T* src = static_cast<const T*>(p.src) + row * p.src_sr + col_block * F8Quantize::kBlock + lane * 4;
      const int left = row < p.rows ? static_cast<int>(min(128ll, p.cols - col_block * static_cast<long long>(F8Quantize::kBlock))) - lane * 4 : 0;
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int e = 0; e < 4; ++e) raw[i][half][e] = half * 64 + e < left ? src[half * 64 + e] : T(0.f);
      row += step_rows, col_block += step_cols;
      if (col_block >= col_blocks) col_block -= col_blocks, ++row;
    }
#pragma unroll
    for (int i = 0; i < kTogether; ++i) {
      if (rows[i] >= p.rows) break;
      float x[2][4], amax = 0.f;
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[half][e] = f8_source(raw[i][half][e]), amax = fmaxf(amax, fabsf(x[half][e]));
#pragma unroll
      for (int offset = 8; offset > 0; offset >>= 1) amax = fmaxf(amax, __shfl_xor_sync(members, amax, offset));
      amax = f8_bounded_amax(amax);
      const float ratio = (lane == 15 ? amax : F8Quantize::kMax) / (lane == 15 ? F8Quantize::kMax : amax);
      const float factor = __shfl_sync(members, ratio, 0, 16);
      if (lane == 15) p.scale[rows[i] * p.scale_sr + cols[i] * p.scale_sc] = ratio;
      uint8_t* dst = p.dst + rows[i] * p.dst_sr + cols[i] * static_cast<long long>(F8Quantize::kBlock) + lane * 4;
      const int left = static_cast<int>(min(128ll, p.cols - cols[i] * static_cast<long long>(F8Quantize::kBlock))) - lane * 4;
#pragma unroll
      for (int half = 0; half < 2; ++half) f8_store4(dst + half * 64, x[half], factor, left - half * 64);
    }
  }
}

// 1 x 128 blocks of any strides: sixteen threads per block, eight elements each.
template <typename T>
__global__ void __launch_bounds__(256) f8_quantize_strided_kernel(const F8QuantizeArgs p) {
  const long long col_blocks = (p.cols + F8Quantize::kBlock - 1) / F8Quantize::kBlock;
  const long long total = p.rows * col_blocks;
  const int lane = threadIdx.x & 15;
  for (long long block = (blockIdx.x * 256ll + threadIdx.x) >> 4; block < total; block += gridDim.x * 16ll) {
    const long long row = block / col_blocks, col_block = block - row * col_blocks;
    const long long col = col_block * F8Quantize::kBlock + lane * 8;
    float x[8];
    f8_load8(static_cast<const T*>(p.src) + row * p.src_sr, p.src_sc, col, p.cols, x);
    float amax = f8_block_amax(x, 0.f);
    const unsigned members = 0xffffu << (threadIdx.x & 16);  // the other half of the warp may be done
#pragma unroll
    for (int offset = 8; offset > 0; offset >>= 1) amax = fmaxf(amax, __shfl_xor_sync(members, amax, offset));
    amax = f8_bounded_amax(amax);
    f8_store8(p.dst + row * p.dst_sr, col, p.cols, x, F8Quantize::kMax / amax);
    if (lane == 0) p.scale[row * p.scale_sr + col_block * p.scale_sc] = amax / F8Quantize::kMax;
  }
}

// 128 x 128 blocks of contiguous rows off 16-byte boundaries: a row a warp at a time, four neighbouring elements a lane.
template <typename T>
__global__ void __launch_bounds__(256) f8_quantize_unaligned_tiles_kernel(const F8QuantizeArgs p) {
  constexpr int kLoads = F8Quantize::kBlock / 8;
  __shared__ float warp_amax[8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long row0 = blockIdx.y * static_cast<long long>(F8Quantize::kBlock) + warp;
  const long long col = blockIdx.x * static_cast<long long>(F8Quantize::kBlock) + lane * 4;
  const int left = static_cast<int>(max(0ll, min(4ll, p.cols - col)));
  T raw[kLoads][4];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const long long row = row0 + 8 * i;
    const T* src = static_cast<const T*>(p.src) + row * p.src_sr + col;
#pragma unroll
    for (int e = 0; e < 4; ++e) raw[i][e] = row < p.rows && e < left ? src[e] : T(0.f);
  }
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < kLoads; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) amax = fmaxf(amax, fabsf(f8_source(raw[i][e])));
#pragma unroll
  for (int offset = 16; offset > 0; offset >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, offset));
  if (lane == 0) warp_amax[warp] = amax;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) amax = fmaxf(amax, warp_amax[w]);
  amax = f8_bounded_amax(amax);
  const float factor = F8Quantize::kMax / amax;
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const long long row = row0 + 8 * i;
    float x[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = f8_source(raw[i][e]);
    if (row < p.rows) f8_store4(p.dst + row * p.dst_sr + col, x, factor, left);
  }
  if (threadIdx.x == 0) p.scale[blockIdx.y * p.scale_sr + blockIdx.x * p.scale_sc] = amax / F8Quantize::kMax;
}

// 128 x 128 blocks: one CTA per block holds it, as loaded, in registers between the maximum and the conversion.
template <typename T, bool kVec>
__global__ void __launch_bounds__(256) f8_quantize_tiles_kernel(const F8QuantizeArgs p) {
  constexpr int kPerLoad = 16 / sizeof(T), kPieces = F8Quantize::kBlock / kPerLoad, kRowStep = 256 / kPieces, kLoads = F8Quantize::kBlock / kRowStep;
  __shared__ float warp_amax[8];
  const long long row0 = blockIdx.y * static_cast<long long>(F8Quantize::kBlock) + threadIdx.x / kPieces;
  const long long col = blockIdx.x * static_cast<long long>(F8Quantize::kBlock) + threadIdx.x % kPieces * kPerLoad;
  const int left = static_cast<int>(max(0ll, min(static_cast<long long>(kPerLoad), p.cols - col)));
  uint4 raw[kLoads];
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const long long row = row0 + kRowStep * i;
    raw[i] = make_uint4(0, 0, 0, 0);
    if (row < p.rows) {
      const T* src = static_cast<const T*>(p.src) + row * p.src_sr + col * p.src_sc;
      if (kVec && left == kPerLoad) {
        raw[i] = __ldg(reinterpret_cast<const uint4*>(src));
      } else {
        T* x = reinterpret_cast<T*>(&raw[i]);
#pragma unroll
        for (int e = 0; e < kPerLoad; ++e)
          if (e < left) x[e] = src[e * p.src_sc];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kLoads; ++i) amax = fmaxf(amax, f8_raw_amax<T>(raw[i]));
#pragma unroll
  for (int offset = 16; offset > 0; offset >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, offset));
  if ((threadIdx.x & 31) == 0) warp_amax[threadIdx.x >> 5] = amax;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) amax = fmaxf(amax, warp_amax[w]);
  amax = f8_bounded_amax(amax);
  const float factor = F8Quantize::kMax / amax;
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const long long row = row0 + kRowStep * i;
    if (row < p.rows) f8_store_raw<T, kVec>(p.dst + row * p.dst_sr + col, raw[i], factor, left);
  }
  if (threadIdx.x == 0) p.scale[blockIdx.y * p.scale_sr + blockIdx.x * p.scale_sc] = amax / F8Quantize::kMax;
}

}  // namespace vb200
