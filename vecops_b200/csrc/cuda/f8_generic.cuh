// Block-scaled e4m3 product on the CUDA cores, for operands the tensor-core kernels cannot address (strides along K,
// rows off 16-byte boundaries).  C[m,n] = sum_b sa[m,b] sb[n/128,b] sum_{k in b} A[m,k] B[n,k]: 32 x 32 outputs per CTA, four per
// thread, 32 k at a time through shared memory; a block's sum is kept apart until its 128 k are done.  Bound by its shared
// memory reads: 512 x 4096 x 14336 takes 5.1 ms, 12 TFLOP/s (the tensor cores: 33 us).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <stdint.h>

namespace vb200 {

struct F8Args {
  const uint8_t* a;
  long long a_sm, a_sk;
  const float* a_scale;
  long long as_sm, as_sk;
  const uint8_t* b;
  long long b_sn, b_sk;
  const float* b_scale;
  long long bs_sn, bs_sk;
  void* c;
  long long c_sm, c_sn;
  long long m, n, k;
};

template <typename OutT>
__device__ __forceinline__ OutT f8_out(float x);
template <>
__device__ __forceinline__ float f8_out<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 f8_out<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half f8_out<__half>(float x) { return __float2half_rn(x); }

__device__ __forceinline__ float f8_value(uint8_t bits) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(bits, __NV_E4M3)));
}

template <typename OutT>
__global__ void __launch_bounds__(256) f8_generic_kernel(const F8Args p) {
  __shared__ float a_tile[32][33], b_tile[32][33];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const long long tiles_m = (p.m + 31) / 32, tiles_n = (p.n + 31) / 32;
  for (long long tile = blockIdx.x; tile < tiles_m * tiles_n; tile += gridDim.x) {
    const long long m0 = tile % tiles_m * 32, n0 = tile / tiles_m * 32;
    const long long n = n0 + tx;
    float total[4] = {0.f, 0.f, 0.f, 0.f};
    for (long long k0 = 0; k0 < p.k; k0 += 128) {
      float part[4] = {0.f, 0.f, 0.f, 0.f};
      for (long long k1 = k0; k1 < k0 + 128 && k1 < p.k; k1 += 32) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = ty + 8 * i;
          const bool there = k1 + tx < p.k;
          a_tile[r][tx] = there && m0 + r < p.m ? f8_value(p.a[(m0 + r) * p.a_sm + (k1 + tx) * p.a_sk]) : 0.f;
          b_tile[r][tx] = there && n0 + r < p.n ? f8_value(p.b[(n0 + r) * p.b_sn + (k1 + tx) * p.b_sk]) : 0.f;
        }
        __syncthreads();
#pragma unroll
        for (int kk = 0; kk < 32; ++kk) {
          const float b = b_tile[tx][kk];
#pragma unroll
          for (int i = 0; i < 4; ++i) part[i] = fmaf(a_tile[ty + 8 * i][kk], b, part[i]);
        }
      }
      const long long block = k0 / 128;
      const float sb = n < p.n ? p.b_scale[n / 128 * p.bs_sn + block * p.bs_sk] : 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const long long m = m0 + ty + 8 * i;
        if (m < p.m) total[i] = fmaf(part[i], p.a_scale[m * p.as_sm + block * p.as_sk] * sb, total[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const long long m = m0 + ty + 8 * i;
      if (m < p.m && n < p.n) static_cast<OutT*>(p.c)[m * p.c_sm + n * p.c_sn] = f8_out<OutT>(total[i]);
    }
  }
}

}  // namespace vb200
