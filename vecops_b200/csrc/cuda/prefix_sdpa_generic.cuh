// Shared-prefix attention, one warp per query row: for head dims, strides and alignments the tensor-core kernels cannot
// address.  The keys are walked one by one with a running maximum m and sum l,
//     m' = max(m, s)   l = l e^(m - m') + e^(s - m')   O = O e^(m - m') + e^(s - m') v      out = O / l
// in fp32; a lane holds head_dim / 32 of q and O.  Bound by the latency of a key after the other: 64 sequences behind 8192 keys of
// 8 heads of 128 in pages of 24 or of 1 take 11.8 ms, of 8 heads of 256 16.4 ms (heads of 128 in pages of 16 by the tensor-core
// kernels: 40 us).
#pragma once

#include <math.h>
#include <stdint.h>

#include "cache_append.cuh"

namespace vb200 {

struct PrefixSdpaArgs {
  const void* q;
  long long q_st, q_sh;
  void* out;
  long long o_st, o_sh;
  const void* k;
  long long k_sp, k_ss, k_sh;
  const void* v;
  long long v_sp, v_ss, v_sh;
  const int *prefix_pages, *page_table, *lengths, *query_starts;
  long long table_stride;
  int table_width;
  int tokens, batch, q_heads, kv_heads, group, head_dim;
  int pages, page_size, prefix_len;
  float scale;
};

// Which sequence owns token t and how many suffix keys the token sees; false for a token without one (padding).
__device__ __forceinline__ bool prefix_token(const PrefixSdpaArgs& p, int t, int& sequence, int& sees) {
  int newer = 0;  // newer tokens of the same sequence in this call
  if (p.query_starts == nullptr) {
    sequence = t;
  } else {
    int low = 0, high = p.batch;  // the last b with query_starts[b] <= t
    if (t < p.query_starts[0] || t >= p.query_starts[p.batch]) return false;
    while (high - low > 1) {
      const int middle = (low + high) / 2;
      if (p.query_starts[middle] <= t) low = middle;
      else high = middle;
    }
    sequence = low;
    newer = min(p.tokens, p.query_starts[low + 1]) - 1 - t;
  }
  const int length = p.lengths[sequence];
  if (length < 0) return false;
  const long long most = static_cast<long long>(p.table_width) * p.page_size;
  const long long seen = length - static_cast<long long>(newer);
  sees = static_cast<int>(seen < 0 ? 0 : seen < most ? seen : most);
  return true;
}

template <typename T>
__global__ void __launch_bounds__(256) prefix_sdpa_generic_kernel(const PrefixSdpaArgs p) {
  const long long row = (blockIdx.x * 256ll + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (row >= static_cast<long long>(p.tokens) * p.q_heads) return;
  const int t = static_cast<int>(row / p.q_heads), head = static_cast<int>(row % p.q_heads), kv = head / p.group;
  const T* q = static_cast<const T*>(p.q) + t * p.q_st + head * p.q_sh;
  T* out = static_cast<T*>(p.out) + t * p.o_st + head * p.o_sh;
  const T* k = static_cast<const T*>(p.k) + kv * p.k_sh;
  const T* v = static_cast<const T*>(p.v) + kv * p.v_sh;
  constexpr int kPerLane = 8;  // head dims up to 256
  float x[kPerLane], o[kPerLane];
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) {
    const int d = lane + 32 * i;
    x[i] = d < p.head_dim ? append_up(q[d]) : 0.f;
    o[i] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  int sequence = 0, sees = 0;
  const bool real = prefix_token(p, t, sequence, sees);
  const int keys = real ? p.prefix_len + sees : 0;
  for (int j = 0; j < keys; ++j) {
    const int local = j < p.prefix_len ? j : j - p.prefix_len;
    const int slot = local / p.page_size, offset = local - slot * p.page_size;
    const int page = j < p.prefix_len ? p.prefix_pages[slot] : p.page_table[sequence * p.table_stride + slot];
    if (page < 0 || page >= p.pages) continue;
    const T* key = k + page * p.k_sp + offset * p.k_ss;
    const T* value = v + page * p.v_sp + offset * p.v_ss;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
      const int d = lane + 32 * i;
      if (d < p.head_dim) s = fmaf(x[i], append_up(key[d]), s);
    }
#pragma unroll
    for (int offset_lane = 16; offset_lane > 0; offset_lane >>= 1) s += __shfl_xor_sync(0xffffffffu, s, offset_lane);
    s *= p.scale;
    const float m_new = fmaxf(m, s);
    // while every score is -inf (or NaN, which fmaxf drops and w keeps) each key counts once: l tells that there was one
    const float keep = m_new == -INFINITY ? 1.f : __expf(m - m_new), w = m_new != -INFINITY ? __expf(s - m_new) : s == -INFINITY ? 1.f : s;
    l = fmaf(l, keep, w);
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
      const int d = lane + 32 * i;
      if (d < p.head_dim) o[i] = fmaf(o[i], keep, w * append_up(value[d]));
    }
    m = m_new;
  }
  const float reciprocal = l == 0.f ? 0.f : m == -INFINITY ? NAN : 1.f / l;  // no key: zeros; only keys whose score is -inf: 0 / 0
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) {
    const int d = lane + 32 * i;
    if (d < p.head_dim) out[d] = append_down<T>(o[i] * reciprocal);
  }
}

}  // namespace vb200
