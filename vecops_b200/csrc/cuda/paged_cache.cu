// C ABI of the paged key/value cache: appending to it and attention over it (include/vecops_b200/decode_cuda.h).
#include <cuda_runtime.h>
#include <stdint.h>

#include "cache_append.cuh"
#include "decode_shim.h"
#include "prefix_sdpa_generic.cuh"

using namespace vb200;

namespace {

bool sixteen_bit(uint32_t dtype) { return dtype == VECOPS_DTYPE_BF16 || dtype == VECOPS_DTYPE_F16; }

int32_t check_append(const VecopsB200CacheAppend& a, VecopsError* error) {
  if (!sixteen_bit(a.dtype)) return set_error(error, VECOPS_STATUS_INVALID_ARGUMENT, "cache_append serves bf16 and f16, not dtype %u", a.dtype);
  if (a.tokens < 0 || a.q_heads < 0 || a.kv_heads < 0 || a.head_dim < 0 || a.pages < 0 || a.page_size < 0 || a.tokens >= (INT64_C(1) << 31) ||
      a.q_heads + 2 * a.kv_heads > (1 << 20) || a.head_dim > (1 << 10) || a.page_size >= (INT64_C(1) << 31))
    return set_error(error, VECOPS_STATUS_INVALID_ARGUMENT, "cache_append: extent out of range");
  if (a.pages > 0 && a.page_size > INT64_MAX / a.pages) return set_error(error, VECOPS_STATUS_INVALID_ARGUMENT, "cache_append: the cache has too many slots");
  if (a.rotary < 0 || a.rotary > a.head_dim || a.rotary % 2 != 0)
    return set_error(error, VECOPS_STATUS_INVALID_ARGUMENT, "cache_append: rotary dims must be even and 0..head_dim, not %lld", (long long)a.rotary);
  if (a.interleaved > 1) return set_error(error, VECOPS_STATUS_INVALID_ARGUMENT, "cache_append: interleaved is 0 or 1");
  const int64_t strides[] = {a.q_stride_token, a.q_stride_head, a.k_stride_token, a.k_stride_head, a.v_stride_token, a.v_stride_head,
                             a.q_out_stride_token, a.q_out_stride_head, a.k_stride_page, a.k_stride_slot, a.k_cache_stride_head,
                             a.v_stride_page, a.v_stride_slot, a.v_cache_stride_head, a.cos_sin_stride, a.max_positions};
  for (int64_t s : strides)
    if (s < 0) return set_error(error, VECOPS_STATUS_INVALID_ARGUMENT, "cache_append: negative stride or table size");
  if (a.tokens == 0 || a.head_dim == 0) return VECOPS_STATUS_OK;
  if ((a.q == nullptr) != (a.q_out == nullptr) && a.q_heads > 0)
    return set_error(error, VECOPS_STATUS_INVALID_ARGUMENT, "cache_append: q and q_out come together");
  if (a.slots == nullptr || (a.kv_heads > 0 && (a.k == nullptr || a.v == nullptr)) ||
      (a.kv_heads > 0 && a.pages > 0 && a.page_size > 0 && (a.k_cache == nullptr || a.v_cache == nullptr)) ||
      (a.rotary > 0 && (a.positions == nullptr || (a.cos_sin == nullptr && a.max_positions > 0))))
    return set_error(error, VECOPS_STATUS_INVALID_ARGUMENT, "cache_append: null pointer");
  return VECOPS_STATUS_OK;
}

bool append_vectors(const VecopsB200CacheAppend& a) {
  const int64_t strides[] = {a.q_stride_token, a.q_stride_head, a.k_stride_token, a.k_stride_head, a.v_stride_token, a.v_stride_head,
                             a.q_out_stride_token, a.q_out_stride_head, a.k_stride_page, a.k_stride_slot, a.k_cache_stride_head,
                             a.v_stride_page, a.v_stride_slot, a.v_cache_stride_head};
  for (int64_t s : strides)
    if (s % 8 != 0) return false;
  for (const void* p : {a.q, a.k, a.v, static_cast<const void*>(a.q_out), static_cast<const void*>(a.k_cache), static_cast<const void*>(a.v_cache)})
    if (!decode_aligned(p, 16)) return false;
  return a.head_dim % 16 == 0 && a.rotary % 16 == 0;
}

int32_t check_prefix(const VecopsB200PrefixAttention& a, VecopsError* error) {
  if (!sixteen_bit(a.dtype)) return set_error(error, VECOPS_STATUS_INVALID_ARGUMENT, "prefix_sdpa serves bf16 and f16, not dtype %u", a.dtype);
  const int64_t limit = (INT64_C(1) << 31) - 256;
  if (a.tokens < 0 || a.batch < 0 || a.pages < 0 || a.prefix_len < 0 || a.table_width < 0 || a.tokens >= limit || a.batch >= limit || a.pages >= limit ||
      a.prefix_len >= limit || a.table_width >= limit || a.page_size < 1 || a.page_size >= limit)
    return set_error(error, VECOPS_STATUS_INVALID_ARGUMENT, "prefix_sdpa: extent out of range");
  if (a.q_heads < 1 || a.kv_heads < 1 || a.q_heads % a.kv_heads != 0 || a.q_heads > 65535)
    return set_error(error, VECOPS_STATUS_INVALID_ARGUMENT, "prefix_sdpa: %lld query heads over %lld key heads", (long long)a.q_heads, (long long)a.kv_heads);
  if (a.head_dim < 1 || a.head_dim > 256) return set_error(error, VECOPS_STATUS_INVALID_ARGUMENT, "prefix_sdpa: head_dim must be 1..256, not %lld", (long long)a.head_dim);
  if (a.table_width * a.page_size >= limit - a.prefix_len)
    return set_error(error, VECOPS_STATUS_INVALID_ARGUMENT, "prefix_sdpa: a sequence could have 2^31 keys");
  if (a.query_starts == nullptr && a.tokens != a.batch)
    return set_error(error, VECOPS_STATUS_INVALID_ARGUMENT, "prefix_sdpa: without query_starts every sequence has one token (%lld tokens, %lld sequences)",
                     (long long)a.tokens, (long long)a.batch);
  const int64_t strides[] = {a.q_stride_token, a.q_stride_head, a.out_stride_token, a.out_stride_head, a.k_stride_page, a.k_stride_slot,
                             a.k_stride_head, a.v_stride_page, a.v_stride_slot, a.v_stride_head, a.table_stride};
  for (int64_t s : strides)
    if (s < 0) return set_error(error, VECOPS_STATUS_INVALID_ARGUMENT, "prefix_sdpa: negative stride");
  if (a.tokens == 0) return VECOPS_STATUS_OK;
  if (a.q == nullptr || a.out == nullptr || (a.pages > 0 && (a.k_cache == nullptr || a.v_cache == nullptr)) || (a.batch > 0 && a.lengths == nullptr) ||
      (a.prefix_len > 0 && a.prefix_pages == nullptr) || (a.batch > 0 && a.table_width > 0 && a.page_table == nullptr))
    return set_error(error, VECOPS_STATUS_INVALID_ARGUMENT, "prefix_sdpa: null pointer");
  return VECOPS_STATUS_OK;
}

PrefixSdpaArgs prefix_args(const VecopsB200PrefixAttention& a) {
  PrefixSdpaArgs p{};
  p.q = a.q, p.q_st = a.q_stride_token, p.q_sh = a.q_stride_head;
  p.out = a.out, p.o_st = a.out_stride_token, p.o_sh = a.out_stride_head;
  p.k = a.k_cache, p.k_sp = a.k_stride_page, p.k_ss = a.k_stride_slot, p.k_sh = a.k_stride_head;
  p.v = a.v_cache, p.v_sp = a.v_stride_page, p.v_ss = a.v_stride_slot, p.v_sh = a.v_stride_head;
  p.prefix_pages = a.prefix_pages, p.page_table = a.page_table, p.lengths = a.lengths, p.query_starts = a.query_starts;
  p.table_stride = a.table_stride, p.table_width = static_cast<int>(a.table_width);
  p.tokens = static_cast<int>(a.tokens), p.batch = static_cast<int>(a.batch);
  p.q_heads = static_cast<int>(a.q_heads), p.kv_heads = static_cast<int>(a.kv_heads), p.group = static_cast<int>(a.q_heads / a.kv_heads);
  p.head_dim = static_cast<int>(a.head_dim);
  p.pages = static_cast<int>(a.pages), p.page_size = static_cast<int>(a.page_size), p.prefix_len = static_cast<int>(a.prefix_len);
  p.scale = a.scale;
  return p;
}

}  // namespace

extern "C" {

int32_t vecops_b200_cache_append(const VecopsB200CacheAppend* append, VecopsError* error) {
  if (append == nullptr || append->struct_size < sizeof(VecopsB200CacheAppend))
    return set_error(error, VECOPS_STATUS_ABI_MISMATCH, "cache_append record is null or too small");
  const VecopsB200CacheAppend& a = *append;
  int32_t rc = check_append(a, error);
  if (rc != VECOPS_STATUS_OK) return rc;
  CacheAppendArgs p{};
  p.q = a.q, p.q_st = a.q_stride_token, p.q_sh = a.q_stride_head;
  p.k = a.k, p.k_st = a.k_stride_token, p.k_sh = a.k_stride_head;
  p.v = a.v, p.v_st = a.v_stride_token, p.v_sh = a.v_stride_head;
  p.q_out = a.q_out, p.qo_st = a.q_out_stride_token, p.qo_sh = a.q_out_stride_head;
  p.k_cache = a.k_cache, p.kc_sp = a.k_stride_page, p.kc_ss = a.k_stride_slot, p.kc_sh = a.k_cache_stride_head;
  p.v_cache = a.v_cache, p.vc_sp = a.v_stride_page, p.vc_ss = a.v_stride_slot, p.vc_sh = a.v_cache_stride_head;
  p.slots = reinterpret_cast<const long long*>(a.slots), p.positions = reinterpret_cast<const long long*>(a.positions);
  p.cos_sin = a.cos_sin, p.cos_sin_stride = a.cos_sin_stride, p.max_positions = a.max_positions;
  p.tokens = a.tokens, p.total_slots = a.pages * a.page_size;
  p.q_heads = a.q == nullptr ? 0 : static_cast<int>(a.q_heads);
  p.kv_heads = static_cast<int>(a.kv_heads), p.head_dim = static_cast<int>(a.head_dim);
  p.rotary = static_cast<int>(a.rotary), p.page_size = static_cast<int>(a.page_size), p.interleaved = static_cast<int>(a.interleaved);
  const bool vec = append_vectors(a);
  const int64_t per_token = (p.q_heads + 2 * static_cast<int64_t>(p.kv_heads)) * (vec ? p.head_dim / 16 : p.head_dim - p.rotary / 2);
  if (a.tokens == 0 || per_token == 0) return VECOPS_STATUS_OK;
  const DeviceRestore restore;
  DecodeDevice device;
  rc = decode_enter(a.device_index, &device, error);
  if (rc != VECOPS_STATUS_OK) return rc;
  const int64_t want = (a.tokens * per_token + 255) / 256;
  const unsigned grid = static_cast<unsigned>(want < static_cast<int64_t>(device.sms) * 64 ? want : static_cast<int64_t>(device.sms) * 64);
  cudaStream_t stream = static_cast<cudaStream_t>(a.stream);
  if (a.dtype == VECOPS_DTYPE_BF16) {
    if (vec) cache_append_kernel<__nv_bfloat16, true><<<grid, 256, 0, stream>>>(p);
    else cache_append_kernel<__nv_bfloat16, false><<<grid, 256, 0, stream>>>(p);
  } else {
    if (vec) cache_append_kernel<__half, true><<<grid, 256, 0, stream>>>(p);
    else cache_append_kernel<__half, false><<<grid, 256, 0, stream>>>(p);
  }
  rc = decode_launched("cache_append", error);
  if (rc != VECOPS_STATUS_OK) return rc;
  return decode_finish("cache_append", a.flags, a.stream, device.index, error);
}

int32_t vecops_b200_prefix_sdpa_workspace(const VecopsB200PrefixAttention* attention, uint64_t* bytes, VecopsError* error) {
  if (attention == nullptr || attention->struct_size < sizeof(VecopsB200PrefixAttention) || bytes == nullptr)
    return set_error(error, VECOPS_STATUS_ABI_MISMATCH, "prefix attention record is null or too small, or no output pointer");
  const int32_t rc = check_prefix(*attention, error);
  if (rc == VECOPS_STATUS_OK) *bytes = 0;
  return rc;
}

int32_t vecops_b200_prefix_sdpa_run(const VecopsB200PrefixAttention* attention, VecopsError* error) {
  if (attention == nullptr || attention->struct_size < sizeof(VecopsB200PrefixAttention))
    return set_error(error, VECOPS_STATUS_ABI_MISMATCH, "prefix attention record is null or too small");
  const VecopsB200PrefixAttention& a = *attention;
  int32_t rc = check_prefix(a, error);
  if (rc != VECOPS_STATUS_OK) return rc;
  if (a.tokens == 0) return VECOPS_STATUS_OK;
  const DeviceRestore restore;
  DecodeDevice device;
  rc = decode_enter(a.device_index, &device, error);
  if (rc != VECOPS_STATUS_OK) return rc;
  const PrefixSdpaArgs p = prefix_args(a);
  const int64_t blocks = (a.tokens * a.q_heads + 7) / 8;
  if (blocks >= (INT64_C(1) << 31)) return set_error(error, VECOPS_STATUS_INVALID_ARGUMENT, "prefix_sdpa: too many query rows");
  cudaStream_t stream = static_cast<cudaStream_t>(a.stream);
  if (a.dtype == VECOPS_DTYPE_BF16) prefix_sdpa_generic_kernel<__nv_bfloat16><<<static_cast<unsigned>(blocks), 256, 0, stream>>>(p);
  else prefix_sdpa_generic_kernel<__half><<<static_cast<unsigned>(blocks), 256, 0, stream>>>(p);
  rc = decode_launched("prefix_sdpa (generic)", error);
  if (rc != VECOPS_STATUS_OK) return rc;
  return decode_finish("prefix_sdpa", a.flags, a.stream, device.index, error);
}

}  // extern "C"
