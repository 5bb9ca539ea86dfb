// Appending new tokens to a paged key/value cache, queries and keys rotated by position on the way.
//
// A pair (x1, x2) of the rotated dims becomes (x1 c - x2 s, x2 c + x1 s) in fp32 and is rounded once; everything else is
// copied bit by bit.  Memory bound: every element is read and written once.  A CTA takes a token at a time: slot, page and
// position are looked up once, and one thread moves 32 bytes - eight pairs of a rotated head, or sixteen dims of a copied
// one - in two 16-byte loads and two 16-byte stores; the cosines and sines of a token are re-read by its heads out of L1.
// Measured: 8191 tokens of 32 + 8 + 8 heads of 128, half of each rotated (203 MB): 38 us, 5.3 TB/s - what is left to the copy rate
// is the chain from a token's slot and position to its angles; the same launch with 64 tokens: 2.4 us, that chain once.  Heads of 120, by
// single pairs: 8191 tokens (191 MB) 146 us, 64 tokens 7.3 us.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace vb200 {

struct CacheAppendArgs {
  const void *q, *k, *v;
  long long q_st, q_sh, k_st, k_sh, v_st, v_sh;
  void* q_out;
  long long qo_st, qo_sh;
  void *k_cache, *v_cache;
  long long kc_sp, kc_ss, kc_sh, vc_sp, vc_ss, vc_sh;
  const long long *slots, *positions;
  const float* cos_sin;
  long long cos_sin_stride, max_positions;
  long long tokens, total_slots;
  int q_heads, kv_heads, head_dim, rotary, page_size, interleaved;
};

template <typename T>
__device__ __forceinline__ float append_up(T x);
template <>
__device__ __forceinline__ float append_up<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <>
__device__ __forceinline__ float append_up<__half>(__half x) { return __half2float(x); }
template <typename T>
__device__ __forceinline__ T append_down(float x);
template <>
__device__ __forceinline__ __nv_bfloat16 append_down<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half append_down<__half>(float x) { return __float2half_rn(x); }

// kVec: head_dim and rotary are multiples of 16, every row starts on a 16-byte boundary and the table's rows do.  Otherwise a
// unit is one pair or one copied dim.
constexpr int kAppendThreads = 384;  // at most
template <typename T, bool kVec>
__global__ void __launch_bounds__(kAppendThreads) cache_append_kernel(const CacheAppendArgs p) {
  const int half = p.rotary / 2;
  const int rotated_units = kVec ? p.rotary / 16 : half;
  const int units = kVec ? p.head_dim / 16 : half + (p.head_dim - p.rotary);  // per head
  const int per_token = (p.q_heads + 2 * p.kv_heads) * units;                 // queries, then keys, then values
  for (long long token = blockIdx.x; token < p.tokens; token += gridDim.x) {
    const long long slot = p.slots[token];
    const long long position = p.rotary > 0 ? p.positions[token] : 0;
    const bool there = slot >= 0 && slot < p.total_slots && (p.rotary == 0 || (position >= 0 && position < p.max_positions));
    const long long page = there ? slot / p.page_size : 0, offset = slot - page * p.page_size;
    for (int i = threadIdx.x; i < per_token; i += blockDim.x) {
      int head = i / units;
      const int unit = i - head * units;
      const bool query = head < p.q_heads, key = !query && head < p.q_heads + p.kv_heads;
      const bool rotate = unit < rotated_units && (query || key);
      head -= query ? 0 : key ? p.q_heads : p.q_heads + p.kv_heads;
      const T* src = query ? static_cast<const T*>(p.q) + token * p.q_st + head * p.q_sh
                     : key ? static_cast<const T*>(p.k) + token * p.k_st + head * p.k_sh : static_cast<const T*>(p.v) + token * p.v_st + head * p.v_sh;
      // where the unit's two 16-byte pieces lie: the two halves of eight pairs, or sixteen dims side by side
      const bool apart = unit < rotated_units && p.interleaved == 0;
      const int v1 = apart ? unit * 8 : unit * 16, v2 = apart ? half + unit * 8 : unit * 16 + 8;
      uint4 raw1, raw2;
      if constexpr (kVec) {  // (on their way before the slot is known: the row exists whether it is padding or not)
        raw1 = *reinterpret_cast<const uint4*>(src + v1);
        raw2 = *reinterpret_cast<const uint4*>(src + v2);
      }
      if (!query && !there) continue;
      T* dst = query ? static_cast<T*>(p.q_out) + token * p.qo_st + head * p.qo_sh
               : key ? static_cast<T*>(p.k_cache) + page * p.kc_sp + offset * p.kc_ss + head * p.kc_sh
                     : static_cast<T*>(p.v_cache) + page * p.vc_sp + offset * p.vc_ss + head * p.vc_sh;
      const float* angles = p.cos_sin + position * p.cos_sin_stride;
      if constexpr (kVec) {
        if (!there) {
          raw1 = raw2 = make_uint4(0, 0, 0, 0);
        } else {
          if (rotate) {
            float4 table[4];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              table[e] = __ldg(reinterpret_cast<const float4*>(angles + unit * 8) + e);
              table[2 + e] = __ldg(reinterpret_cast<const float4*>(angles + half + unit * 8) + e);
            }
            const float *c = reinterpret_cast<const float*>(table), *s = c + 8;
            T* x1 = reinterpret_cast<T*>(&raw1);
            T* x2 = reinterpret_cast<T*>(&raw2);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              T& first = p.interleaved ? (e < 4 ? x1[2 * e] : x2[2 * e - 8]) : x1[e];
              T& second = p.interleaved ? (e < 4 ? x1[2 * e + 1] : x2[2 * e - 7]) : x2[e];
              const float a = append_up(first), b = append_up(second);
              first = append_down<T>(a * c[e] - b * s[e]);
              second = append_down<T>(b * c[e] + a * s[e]);
            }
          }
        }
        *reinterpret_cast<uint4*>(dst + v1) = raw1;
        *reinterpret_cast<uint4*>(dst + v2) = raw2;
      } else if (unit < rotated_units) {
        const int d1 = p.interleaved ? 2 * unit : unit, d2 = p.interleaved ? 2 * unit + 1 : half + unit;
        if (!there) {
          dst[d1] = dst[d2] = append_down<T>(0.f);
        } else if (!rotate) {
          const T a = src[d1], b = src[d2];
          dst[d1] = a, dst[d2] = b;
        } else {
          const float c = angles[unit], s = angles[half + unit];
          const float a = append_up(src[d1]), b = append_up(src[d2]);
          dst[d1] = append_down<T>(a * c - b * s);
          dst[d2] = append_down<T>(b * c + a * s);
        }
      } else {
        const int d = p.rotary + unit - rotated_units;
        dst[d] = there ? src[d] : append_down<T>(0.f);
      }
    }
  }
}

}  // namespace vb200
