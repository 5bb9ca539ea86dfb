// C ABI of the paged key/value cache: appending to it and attention over it (include/vecops_b200/decode_cuda.h).
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "cache_append.cuh"
#include "decode_shim.h"
#include "prefix_sdpa.cuh"
#include "prefix_sdpa_generic.cuh"
#include "suffix_sdpa.cuh"

using namespace vb200;

namespace {

bool sixteen_bit(uint32_t dtype) { return dtype == VECOPS_DTYPE_BF16 || dtype == VECOPS_DTYPE_F16; }

int32_t check_append(const VecopsB200CacheAppend& a, VecopsError* error) {
  if (!sixteen_bit(a.dtype)) return set_error(error, VECOPS_STATUS_INVALID_ARGUMENT, "cache_append serves bf16 and f16, not dtype %u", a.dtype);
  if (a.tokens < 0 || a.q_heads < 0 || a.kv_heads < 0 || a.head_dim < 0 || a.pages < 0 || a.page_size < 0 || a.tokens >= (INT64_C(1) << 31) ||
      a.q_heads > (1 << 20) || a.kv_heads > (1 << 20) || a.q_heads + 2 * a.kv_heads > (1 << 20) || a.head_dim > (1 << 10) || a.page_size >= (INT64_C(1) << 31))
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
  auto shares = [&](int64_t page, int64_t slot, int64_t head) { return (a.pages > 1 && page == 0) || (a.page_size > 1 && slot == 0) || (a.kv_heads > 1 && head == 0); };
  if (shares(a.k_stride_page, a.k_stride_slot, a.k_cache_stride_head) || shares(a.v_stride_page, a.v_stride_slot, a.v_cache_stride_head) ||
      (a.q != nullptr && ((a.tokens > 1 && a.q_out_stride_token == 0) || (a.q_heads > 1 && a.q_out_stride_head == 0))))
    return set_error(error, VECOPS_STATUS_INVALID_ARGUMENT, "cache_append: rows of the cache or of q_out share memory");
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
  if (a.rotary > 0 && (!decode_aligned(a.cos_sin, 16) || a.cos_sin_stride % 4 != 0)) return false;
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
  if (a.tokens * a.q_heads > 4 * INT64_C(0x7fffffff)) return set_error(error, VECOPS_STATUS_INVALID_ARGUMENT, "prefix_sdpa: too many query rows");
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
  if ((a.tokens > 1 && a.out_stride_token == 0) || (a.q_heads > 1 && a.out_stride_head == 0))
    return set_error(error, VECOPS_STATUS_INVALID_ARGUMENT, "prefix_sdpa: rows of out share memory");
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

// ---------------------------------------------------------------- the two-kernel form: prefix on tcgen05, suffix and merge behind it

// Few sequences behind a short prefix, or one behind any: the suffix kernel reads the prefix for every item, in front of its suffix, and
// there is no prefix kernel, if what is read again comes to no more than this.  With / without the prefix kernel, 128-dim heads
// unless told otherwise: 12 sequences of 2 heads of 64 behind 644 keys (4 MB again) 10.0 / 8.1 us, 4 of 8 behind 512 (6 MB) 9.9 / 10.5
// and a launch less, 183 of 1 behind 209 (19 MB) 16.0 / 12.2, one of 8 behind 16384 (none) 23.5 / 17.6; 16 of 8 behind
// 1000 (61 MB) 15.8 / 17.3, 7 of 8 of 64 behind 4877 (60 MB) 13.2 / 18.4.
constexpr int64_t kRereadBytes = INT64_C(32) << 20;

struct PrefixPlan {
  bool fast = false;  // the two kernels can address this call; the one-warp-per-row kernel serves the rest
  int dim = 0;        // head dims a kernel is built for: 64 or 128
  int both_rows = 0, row_blocks = 0, tiles = 0, tiles_per_chunk = 0, chunks = 0, records = 0;
  int prefix_slices = 0;  // joined: no prefix kernel, every item of the suffix kernel starts with the prefix
  int tokens_per_item = 1, group_tiles = 1, item_rows = 1, workers = 0, beside = 0, beside_most = 0;
  int64_t slots = 0, fragments = 0;
  uint64_t ml_at = 0, fragment_o_at = 0, fragment_ml_at = 0, sums_at = 0, total = 0;
};

// Whether every row of the operands can be loaded and stored in sixteen bytes, and the caches' pages be addressed by TMA (whose strides are
// not 0; heads that share their rows are one head to it).
bool prefix_addressable(const VecopsB200PrefixAttention& a) {
  auto rows_ok = [](const void* base, int64_t n0, int64_t s0, int64_t n1, int64_t s1, int64_t n2, int64_t s2) {
    return decode_aligned(base, 16) && (n0 <= 1 || s0 % 8 == 0) && (n1 <= 1 || s1 % 8 == 0) && (n2 <= 1 || s2 % 8 == 0);
  };
  return rows_ok(a.q, a.tokens, a.q_stride_token, a.q_heads, a.q_stride_head, 1, 0) && rows_ok(a.out, a.tokens, a.out_stride_token, a.q_heads, a.out_stride_head, 1, 0) &&
         rows_ok(a.k_cache, a.pages, a.k_stride_page, a.page_size, a.k_stride_slot, a.kv_heads, a.k_stride_head) &&
         rows_ok(a.v_cache, a.pages, a.v_stride_page, a.page_size, a.v_stride_slot, a.kv_heads, a.v_stride_head) &&
         (a.pages <= 1 || (a.k_stride_page > 0 && a.v_stride_page > 0)) && (a.page_size <= 1 || (a.k_stride_slot > 0 && a.v_stride_slot > 0));
}

// By the extents alone (and whether there are query_starts): what the scratch is sized by must not change with an address.
PrefixPlan plan_prefix(const VecopsB200PrefixAttention& a, int sms) {
  PrefixPlan p;
  const bool pages_ok = a.page_size % 128 == 0 || (a.page_size % 8 == 0 && 128 % a.page_size == 0);  // a tile of 128 keys is whole pages or lies in one
  p.fast = a.head_dim <= 128 && a.head_dim % 8 == 0 && (a.prefix_len == 0 || pages_ok) &&
           a.tokens * (a.q_heads / a.kv_heads) <= INT64_C(256) * 65535 &&  // (row blocks are a grid's third dimension)
           a.kv_heads <= 65535 && a.batch < (1 << 24) && a.tokens < (1 << 24);
  if (!p.fast) return p;
  p.dim = a.head_dim <= 64 ? 64 : 128;
  const int64_t group = a.q_heads / a.kv_heads, rows = a.tokens * group;
  p.tokens_per_item = static_cast<int>(group <= 16 ? 16 / group : 1);
  p.group_tiles = static_cast<int>((group + 15) / 16);
  p.item_rows = static_cast<int>(group >= 16 ? 16 : (a.query_starts == nullptr ? 1 : p.tokens_per_item) * group);
  p.slots = a.query_starts == nullptr ? a.batch : a.tokens / p.tokens_per_item + a.batch + 1;
  const int64_t columns = a.kv_heads * p.group_tiles;
  const bool prefix = a.prefix_len > 0 && a.tokens > 0 && a.pages > 0;
  if (prefix && p.slots * p.group_tiles - 1 <= kRereadBytes / (a.kv_heads * a.prefix_len * p.dim * 4)) p.prefix_slices = static_cast<int>((a.prefix_len + 15) / 16);
  // warps for every slice the table could hold, up to what the SMs hold at once (slices are counted in 32 bits)
  const int64_t table_slices = (a.table_width * a.page_size + 15) / 16, slices = p.prefix_slices + table_slices;
  if (slices > 0 && p.slots * columns > ((INT64_C(1) << 31) - 1) / (slices + kItemWeight)) {
    p.fast = false;
    return p;
  }
  constexpr int64_t kSmWarps = SuffixSdpa<64>::kCtasPerSm * SuffixSdpa<64>::kWarps;
  const int64_t most = sms * kSmWarps;
  int64_t wanted = p.slots * columns;
  wanted = slices == 0 || wanted >= most ? (slices == 0 ? 1 : most) : (wanted * slices < most ? wanted * slices : most);
  p.workers = static_cast<int>((wanted + 3) / 4 * 4);
  p.fragments = p.workers + p.slots * columns;
  if (prefix && p.prefix_slices == 0) {
    p.both_rows = rows > 128 ? 1 : 0;
    p.row_blocks = static_cast<int>(p.both_rows ? (rows + 255) / 256 : 1);
    p.tiles = static_cast<int>((a.prefix_len + 127) / 128);
    // How the prefix is cut decides how many SMs it takes, and for how long; the suffixes go on the others meanwhile, or behind it.
    // In us, as measured: an item of the prefix kernel takes 2 for a key tile and for five more - Q, the first loads, the record it
    // leaves; a record of 10000 rows of 128 dims 2 to write and merge; the suffix kernel 5 to start, a warp of it 1.4 (64 dims: 1)
    // a position - a slice of 16 keys, or a part of an item's start - and all of it what the memory takes; of what is left to
    // it behind the prefix kernel, the free SMs have done one and a half times their share.  The lengths are on the device: taken to be
    // half of the table's.  Every SM for the prefix / cut as this finds best: 64 sequences of 8 heads of 128 behind 8192 keys,
    // up to 1024 of their own, 52.4 / 40.4 us; 128 behind 4096, 2048, 112 / 107; 192 behind 16384, 512, 98 / 92; 100 of one to
    // three tokens behind 3000, 200, 31.7 / 28.3; 256 behind 32768, 512, 182 / 182; and where it errs, a table for 8192 keys with
    // 100 in it, 29.3 / 34.9.
    const int64_t base = a.kv_heads * p.row_blocks;
    const double record_us = static_cast<double>(a.kv_heads) * rows * p.dim / 6.4e5;
    const double position_us = 0.5 + 0.9 * p.dim / 128, start_us = 5;
    const int64_t items = a.query_starts == nullptr || a.tokens / p.tokens_per_item < a.batch ? a.batch : a.tokens / p.tokens_per_item;
    const double positions = table_slices == 0 ? 0 : static_cast<double>(items) * columns * (table_slices * 0.5 + (a.query_starts == nullptr ? 1 : 2) * kItemWeight);
    auto suffix_us = [&](double warps) {
      const double by_warps = positions / warps * position_us, by_memory = positions * 64 * p.dim / 5.5e6;
      return start_us + (by_warps > by_memory ? by_warps : by_memory);
    };
    // each length of a chunk once, from the longest on: the fewest chunks that are shorter (the rest cut alike)
    auto each_cut = [&](auto&& cut) {
      for (int per_chunk = p.tiles, used = 1; used <= 128;) {
        const int64_t waves = (base * used + sms - 1) / sms;
        cut(per_chunk, used, 2.0 * waves * (per_chunk + 5));
        if (per_chunk == 1) break;
        used = (p.tiles + per_chunk - 2) / (per_chunk - 1);
        per_chunk = (p.tiles + used - 1) / used;
      }
    };
    double shortest = 1e30, best = 1e30;
    each_cut([&](int, int, double prefix_us) { shortest = prefix_us < shortest ? prefix_us : shortest; });
    each_cut([&](int per_chunk, int used, double prefix_us) {
      if (prefix_us > 1.8 * shortest) return;  // (not at any price for the prefix: a table may be far wider than its lengths)
      const int64_t free_sms = base * used < sms ? sms - base * used : 0;
      const int64_t beside = free_sms * kSmWarps < p.workers ? free_sms * kSmWarps : p.workers;
      const double all_us = suffix_us(p.workers), meanwhile = 1.5 * prefix_us * free_sms / sms;
      const double after = prefix_us + (all_us > meanwhile ? all_us - meanwhile : 0), along = beside == 0 ? after : suffix_us(static_cast<double>(beside));
      const double cost = record_us * used + (along < prefix_us ? prefix_us : along < after ? along : after);
      if (cost < best) {
        best = cost, p.tiles_per_chunk = per_chunk, p.chunks = used;
        // Beside the prefix kernel if that ends sooner than all warps behind it, which is decided where the lengths are; a third in its
        // favour, as CTAs that there is no room for start late.  (On all SMs / beside it: 64 sequences of 8 heads behind 512 keys
        // 18.6 / 14.6 us, 64 of 4 behind 1066 14.7 / 11.2.)
        p.beside = static_cast<int>(beside);
        const double limit = beside == p.workers ? 2147483647.0 : 1.33 * prefix_us / position_us * beside * p.workers / (p.workers - beside);
        p.beside_most = limit < 2147483647.0 ? static_cast<int>(limit) : 2147483647;
      }
    });
    p.records = p.both_rows ? p.chunks : 2 * p.chunks;
  }

  auto place = [&](uint64_t bytes) {
    const uint64_t at = p.total;
    p.total += (bytes + 255) / 256 * 256;
    return at;
  };
  const uint64_t record_rows = static_cast<uint64_t>(p.records) * a.kv_heads * rows;
  place(record_rows * p.dim * 4);
  p.ml_at = place(record_rows * 8);
  p.fragment_o_at = place(static_cast<uint64_t>(p.fragments) * p.item_rows * p.dim * 4);
  p.fragment_ml_at = place(static_cast<uint64_t>(p.fragments) * p.item_rows * 8);
  p.sums_at = place(static_cast<uint64_t>(p.slots + 1) * 4);
  return p;
}

template <typename T, int kDim>
int32_t run_prefix(const VecopsB200PrefixAttention& a, const PrefixPlan& plan, const DecodeDevice& device, VecopsError* error) {
  using G = PrefixTc<kDim>;
  const PrefixSdpaArgs args = prefix_args(a);
  cudaStream_t stream = static_cast<cudaStream_t>(a.stream);
  cudaLaunchAttribute attributes[1] = {};
  attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attributes[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config = {};
  config.stream = stream;
  config.attrs = attributes;
  static std::atomic<bool> raised[64];
  if (device.index >= 64 || !raised[device.index].load()) {
    cudaError_t status = cudaFuncSetAttribute(prefix_sdpa_kernel<T, kDim>, cudaFuncAttributeMaxDynamicSharedMemorySize, G::kSmemBytes);
    for (auto kernel : {suffix_sdpa_kernel<T, kDim, true, false>, suffix_sdpa_kernel<T, kDim, false, false>, suffix_sdpa_kernel<T, kDim, true, true>, suffix_sdpa_kernel<T, kDim, false, true>})
      if (status == cudaSuccess) status = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SuffixSdpa<kDim>::kSmemBytes);
    if (status != cudaSuccess) return set_error(error, VECOPS_STATUS_EXECUTION_ERROR, "cudaFuncSetAttribute(prefix_sdpa): %s", cudaGetErrorString(status));
    if (device.index < 64) raised[device.index].store(true);
  }
  const int rows = static_cast<int>(a.tokens * (a.q_heads / a.kv_heads));
  float* partial_o = static_cast<float*>(a.workspace);
  float2* partial_ml = reinterpret_cast<float2*>(static_cast<char*>(a.workspace) + plan.ml_at);
  if (plan.records > 0) {
    PrefixTcArgs p{};
    p.a = args;
    p.rows = rows, p.row_blocks = plan.row_blocks, p.tiles = plan.tiles, p.tiles_per_chunk = plan.tiles_per_chunk, p.both_rows = plan.both_rows;
    p.box_keys = static_cast<int>(a.page_size < 128 ? a.page_size : 128);
    p.partial_o = partial_o, p.partial_ml = partial_ml, p.status = device.status;
    CUtensorMap map_k, map_v;
    auto cache_map = [&](CUtensorMap* map, const void* base, int64_t page, int64_t slot, int64_t head, int* head_step) {
      *head_step = head > 0 ? 1 : 0;
      // (a dimension of one has no stride that matters, but the map wants a legal one)
      auto bytes = [](int64_t n, int64_t stride) { return static_cast<uint64_t>(n > 1 ? stride * 2 : 16); };
      const uint64_t dims[4] = {static_cast<uint64_t>(a.head_dim), static_cast<uint64_t>(a.page_size), static_cast<uint64_t>(head > 0 ? a.kv_heads : 1),
                                static_cast<uint64_t>(a.pages)};
      const uint64_t strides[3] = {bytes(a.page_size, slot), bytes(static_cast<int64_t>(dims[2]), head), bytes(a.pages, page)};
      const uint32_t box[4] = {64, static_cast<uint32_t>(p.box_keys), 1, 1};
      const CUtensorMapDataType type = std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
      return shim_encode_map(map, type, 4, base, dims, strides, box, error);
    };
    int32_t rc = cache_map(&map_k, a.k_cache, a.k_stride_page, a.k_stride_slot, a.k_stride_head, &p.k_head_step);
    if (rc != VECOPS_STATUS_OK) return rc;
    rc = cache_map(&map_v, a.v_cache, a.v_stride_page, a.v_stride_slot, a.v_stride_head, &p.v_head_step);
    if (rc != VECOPS_STATUS_OK) return rc;
    config.gridDim = dim3(static_cast<unsigned>(plan.chunks), static_cast<unsigned>(a.kv_heads), static_cast<unsigned>(plan.row_blocks));
    config.blockDim = dim3(G::kThreads);
    config.dynamicSmemBytes = G::kSmemBytes;
    config.numAttrs = 1;
    const cudaError_t status = cudaLaunchKernelEx(&config, prefix_sdpa_kernel<T, kDim>, map_k, map_v, p);
    if (status != cudaSuccess) return set_error(error, VECOPS_STATUS_EXECUTION_ERROR, "prefix_sdpa launch: %s", cudaGetErrorString(status));
    rc = decode_launched("prefix_sdpa", error);
    if (rc != VECOPS_STATUS_OK) return rc;
  }
  SuffixSdpaArgs s{};
  s.a = args;
  s.rows = rows;
  s.tokens_per_item = plan.tokens_per_item, s.group_tiles = plan.group_tiles, s.item_rows = plan.item_rows;
  s.slots = static_cast<int>(plan.slots), s.workers = plan.workers, s.beside = plan.beside, s.beside_most = plan.beside_most;
  s.records = plan.records, s.prefix_slices = plan.prefix_slices, s.partial_o = partial_o, s.partial_ml = partial_ml;
  char* base = static_cast<char*>(a.workspace);
  s.fragment_o = reinterpret_cast<float*>(base + plan.fragment_o_at), s.fragment_ml = reinterpret_cast<float2*>(base + plan.fragment_ml_at);
  s.sums = reinterpret_cast<int*>(base + plan.sums_at);
  config.gridDim = dim3(static_cast<unsigned>(plan.workers / SuffixSdpa<kDim>::kWarps));
  config.blockDim = dim3(SuffixSdpa<kDim>::kThreads);
  config.dynamicSmemBytes = SuffixSdpa<kDim>::kSmemBytes;
  config.numAttrs = 1;
  const bool whole_pages = a.page_size % 16 == 0, joined = plan.prefix_slices > 0;
  const auto suffix = whole_pages ? (joined ? suffix_sdpa_kernel<T, kDim, true, true> : suffix_sdpa_kernel<T, kDim, true, false>)
                                  : (joined ? suffix_sdpa_kernel<T, kDim, false, true> : suffix_sdpa_kernel<T, kDim, false, false>);
  cudaError_t status = cudaLaunchKernelEx(&config, suffix, s);
  if (status != cudaSuccess) return set_error(error, VECOPS_STATUS_EXECUTION_ERROR, "suffix_sdpa launch: %s", cudaGetErrorString(status));
  int32_t rc = decode_launched("suffix_sdpa", error);
  if (rc != VECOPS_STATUS_OK) return rc;
  // few rows: four warps share one's partial results
  const int64_t out_rows = a.tokens * a.q_heads;
  const bool shared_rows = out_rows <= static_cast<int64_t>(device.sms) * 4;
  const int64_t blocks = shared_rows ? out_rows : (out_rows + 3) / 4;
  config.gridDim = dim3(static_cast<unsigned>(blocks));
  config.blockDim = dim3(128);
  config.dynamicSmemBytes = 0;
  status = shared_rows ? cudaLaunchKernelEx(&config, sdpa_merge_rows_kernel<T, kDim, 4>, s) : cudaLaunchKernelEx(&config, sdpa_merge_rows_kernel<T, kDim, 1>, s);
  if (status != cudaSuccess) return set_error(error, VECOPS_STATUS_EXECUTION_ERROR, "sdpa_merge_rows launch: %s", cudaGetErrorString(status));
  return decode_launched("sdpa_merge_rows", error);
}

template <typename T>
int32_t run_prefix_generic(const VecopsB200PrefixAttention& a, VecopsError* error) {
  const int64_t blocks = (a.tokens * a.q_heads + 7) / 8;
  prefix_sdpa_generic_kernel<T><<<static_cast<unsigned>(blocks), 256, 0, static_cast<cudaStream_t>(a.stream)>>>(prefix_args(a));
  return decode_launched("prefix_sdpa (generic)", error);
}

template <typename T>
int32_t run_prefix_typed(const VecopsB200PrefixAttention& a, const PrefixPlan& plan, const DecodeDevice& device, VecopsError* error) {
  if (!plan.fast) return run_prefix_generic<T>(a, error);
  return plan.dim == 64 ? run_prefix<T, 64>(a, plan, device, error) : run_prefix<T, 128>(a, plan, device, error);
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
  const unsigned grid = static_cast<unsigned>(a.tokens < static_cast<int64_t>(device.sms) * 64 ? a.tokens : static_cast<int64_t>(device.sms) * 64);
  // many tokens: small CTAs, whose lookups overlap with others' copies (8191 tokens: 38 us with 128 threads, 55 with 384); few: a token's
  // copies all at once (64 tokens: 2.4 us with 384, 3.2 with 128)
  const int64_t most = a.tokens >= static_cast<int64_t>(device.sms) * 8 ? 128 : kAppendThreads;
  const unsigned threads = static_cast<unsigned>(per_token < most ? (per_token + 31) / 32 * 32 : most);
  cudaStream_t stream = static_cast<cudaStream_t>(a.stream);
  if (a.dtype == VECOPS_DTYPE_BF16) {
    if (vec) cache_append_kernel<__nv_bfloat16, true><<<grid, threads, 0, stream>>>(p);
    else cache_append_kernel<__nv_bfloat16, false><<<grid, threads, 0, stream>>>(p);
  } else {
    if (vec) cache_append_kernel<__half, true><<<grid, threads, 0, stream>>>(p);
    else cache_append_kernel<__half, false><<<grid, threads, 0, stream>>>(p);
  }
  rc = decode_launched("cache_append", error);
  if (rc != VECOPS_STATUS_OK) return rc;
  return decode_finish("cache_append", a.flags, a.stream, device.index, error);
}

int32_t vecops_b200_prefix_sdpa_workspace(const VecopsB200PrefixAttention* attention, uint64_t* bytes, VecopsError* error) {
  if (attention == nullptr || attention->struct_size < sizeof(VecopsB200PrefixAttention) || bytes == nullptr)
    return set_error(error, VECOPS_STATUS_ABI_MISMATCH, "prefix attention record is null or too small, or no output pointer");
  const int32_t rc = check_prefix(*attention, error);
  if (rc != VECOPS_STATUS_OK) return rc;
  // the SM count of the device the record names, or of a B200 when no device can be asked
  int sms = 148, device = attention->device_index;
  if (vecops_b200_device_count() > 0 && (device >= 0 || cudaGetDevice(&device) == cudaSuccess)) {
    int asked = 0;
    if (shim_device_facts(device, &asked, nullptr, nullptr, nullptr) == VECOPS_STATUS_OK && asked > 0) sms = asked;
  }
  *bytes = plan_prefix(*attention, sms).total;
  return VECOPS_STATUS_OK;
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
  const PrefixPlan plan = prefix_addressable(a) ? plan_prefix(a, device.sms) : PrefixPlan{};
  if (plan.total != 0 && (a.workspace == nullptr || !decode_aligned(a.workspace, 256) || a.workspace_size < plan.total))
    return set_error(error, VECOPS_STATUS_INVALID_ARGUMENT, "prefix_sdpa needs %llu bytes of 256-byte aligned device scratch (vecops_b200_prefix_sdpa_workspace)",
                     (unsigned long long)plan.total);
  rc = a.dtype == VECOPS_DTYPE_BF16 ? run_prefix_typed<__nv_bfloat16>(a, plan, device, error) : run_prefix_typed<__half>(a, plan, device, error);
  if (rc != VECOPS_STATUS_OK) return rc;
  return decode_finish("prefix_sdpa", a.flags, a.stream, device.index, error);
}

}  // extern "C"
