// Attention over each sequence's own suffix, and the merge with what the prefix kernel left: the second and third kernels of
// shared-prefix attention; the first and second when there is no prefix, or when few read it: every item then starts with its keys.
//
// An item is up to sixteen query rows of one sequence and one key/value head - the queries that read this head, of one
// token or of a few neighbouring ones - and the keys they see, in slices of sixteen.  The work is the keys' way from
// memory: every key and value is used by at most sixteen rows.  So all slices of all items, in order, are dealt out evenly to
// the warps of the grid whatever the lengths are - an item counts as kItemWeight slices more, for what starting on it costs; a
// warp keeps the next slice in flight by cp.async while it multiplies one with mma.sync m16n8k16, whose sixteen rows are the
// item's (tcgen05's 128 would be nearly empty).  Warps share nothing and meet at no barrier.  Each runs m' = max(m, s), l, O over its part of an item and leaves them as a fragment;
// sdpa_merge_rows_kernel, launched behind, joins a row's fragments and its prefix records,
//     M = max m_c      out = sum_c 2^(m_c - M) O_c / sum_c 2^(m_c - M) l_c           (m in units of log2(e))
// in an order that does not depend on timing.  p is rounded to the type of V for the product with it, as in the prefix kernel, and added to l as
// it is.  Keys that some of an item's rows see and others do not - at most fifteen, the
// newest tokens' own - go past the tensor core: there a zero probability times whatever a later token's value holds
// would still be NaN.
//
// Measured, 8 heads of 128: 128 sequences of 1024 keys (537 MB) 89 us, 6.0 TB/s; 64 sequences of up to 1024 keys (137 MB) 30 us,
// 4.5 TB/s, where starting and ending weigh more.  A few short sequences: 8 us with the merge, one dependent trip to memory
// after the other through the two kernels.
#pragma once

#include "prefix_sdpa.cuh"

namespace vb200 {

template <int kDim>
struct SuffixSdpa {
  static constexpr int kWarps = 4, kThreads = 32 * kWarps;
  static constexpr int kCtasPerSm = 2;
  static constexpr int kRows = 16, kKeys = 16;
  static constexpr int kStages = 2;
  static constexpr int kRowBytes = kDim * 2;
  static constexpr int kTileBytes = kKeys * kRowBytes;
  static constexpr int kWarpBytes = kStages * 2 * kTileBytes;
  static constexpr int kProbOffset = kWarps * kWarpBytes;
  static constexpr int kProbBytes = kRows * kKeys * 4;  // per warp: probabilities of the keys that only some rows see
  static constexpr int kSmemBytes = kProbOffset + kWarps * kProbBytes + kWarps * kStages * 4;
};

struct SuffixSdpaArgs {
  PrefixSdpaArgs a;
  int rows;             // tokens * group, per key/value head: the prefix records' rows
  int tokens_per_item;  // neighbouring tokens of one sequence in an item
  int group_tiles;      // items a token is cut into when its group has more than sixteen heads
  int slots;            // of items per (head, group tile), idle ones included
  int workers;          // warps of the suffix kernel
  int beside;           // ... that there is room for beside the prefix kernel's CTAs
  int beside_most;      // what may be dealt to them
  int records;          // of the prefix kernel
  int prefix_slices;    // without one: slices of the prefix that every item starts with (the joined form), or 0
  const float* partial_o;
  const float2* partial_ml;
  int item_rows;        // rows an item has at most
  float* fragment_o;    // [warp + item][item_rows][kDim]
  float2* fragment_ml;  // [warp + item][item_rows]
  int* sums;            // [slot] weight of the slots before it, written where the slot has any; then [slots] the sum of all
};

// Without query_starts slot b is sequence b's one token; with them sequence b's items are the slots from
// query_starts[b] / tokens_per_item + b on: apart from each other, and found without a sum.
constexpr int kItemWeight = 2;  // slices' worth of time that an item's lookups, queries and fragment take (measured: 2.5 us of 1 to 2 us each)

// Warps that `all` is dealt to: two positions at least to each - a slice's fragment costs the merge as much as the slice - and, if
// they would be done before the prefix kernel is, no more than there is room for beside it: CTAs that do not fit start when it ends.
__device__ __forceinline__ int suffix_workers(int workers, int beside, int beside_most, int all) {
  return min(all <= beside_most ? beside : workers, (all + 1) / 2);
}

// Suffix keys that token t sees of a sequence whose newest token is `newest`: of those the table has room for (fewer than 2^31).
__device__ __forceinline__ int suffix_sees(const PrefixSdpaArgs& a, int length, int newest, int t) {
  return max(0, min(length - (newest - t), a.table_width * a.page_size));
}

// The last sequence whose query_starts pass `before`, by a search 32 wide; the whole warp comes here.
template <typename Before>
__device__ __forceinline__ int suffix_search(int batch, const Before& before) {
  const int lane = threadIdx.x & 31;
  int low = 0, high = batch;
  while (high - low > 1) {
    const int step = (high - low + 31) / 32, probe = low + lane * step;
    const int found = 31 - __clz(__ballot_sync(0xffffffffu, probe < high && before(probe)) | 1u);
    low += found * step;
    high = min(high, low + step);
  }
  return low;
}

// Slices and weight of the item whose newest token is `last`.
__device__ __forceinline__ int suffix_slices(const PrefixSdpaArgs& a, int prefix_slices, int length, int newest, int last) {
  return length < 0 ? 0 : prefix_slices + (suffix_sees(a, length, newest, last) + 15) / 16;
}
__device__ __forceinline__ int suffix_weight(int slices) { return slices > 0 ? slices + kItemWeight : 0; }

template <typename T>
__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma_16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma_16816<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

// Sixteen bytes to shared memory, or zeros when `bytes` is 0 (nothing is read then).
__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kPending>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory");
}

template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t x);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t x) {
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&x));
}
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t x) {
  return __half22float2(*reinterpret_cast<const __half2*>(&x));
}

// kWholePages: page_size is a multiple of sixteen, so a slice lies in one page.  kJoined: there is no prefix kernel, and an item's slices
// are those of the prefix, then those of its suffix.
template <typename T, int kDim, bool kWholePages, bool kJoined>
__global__ void __launch_bounds__(SuffixSdpa<kDim>::kThreads, SuffixSdpa<kDim>::kCtasPerSm) suffix_sdpa_kernel(const SuffixSdpaArgs p) {
  using G = SuffixSdpa<kDim>;
  extern __shared__ __align__(128) uint8_t smem[];
  const uint32_t smem_base = smem_u32(smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const PrefixSdpaArgs& a = p.a;
  const int prefix_slices = kJoined ? p.prefix_slices : 0;
  volatile uint32_t* present = reinterpret_cast<volatile uint32_t*>(smem + G::kProbOffset + G::kWarps * G::kProbBytes) + warp * G::kStages;
  if (p.records == 0) grid_dependency_wait();  // (with a prefix kernel in between, the kernels before that one are done already)
  grid_launch_dependents();

  // ---------------------------------------------------------------- this warp's positions [position, end)
  // Every warp adds the weights up for itself, a lane per run of sequences: no barrier, one trip to memory for a small batch.
  struct Tokens {
    int begin, end;  // of a sequence
  };
  auto tokens_of = [&](int b) -> Tokens {
    if (a.query_starts == nullptr) return {b, b + 1};
    return {max(0, a.query_starts[b]), min(a.tokens, a.query_starts[b + 1])};
  };
  const int per_lane = (a.batch + 31) / 32;
  int sum = 0;
  for (int b = lane * per_lane; b < min(a.batch, (lane + 1) * per_lane); ++b) {
    const int length = a.lengths[b];
    const Tokens tokens = tokens_of(b);
    for (int first = tokens.begin; first < tokens.end; first += p.tokens_per_item)
      sum += suffix_weight(suffix_slices(a, prefix_slices, length, tokens.end - 1, min(tokens.end, first + p.tokens_per_item) - 1));
  }
  int before = sum;
#pragma unroll
  for (int offset = 1; offset < 32; offset <<= 1) {
    const int other = __shfl_up_sync(0xffffffffu, before, offset);
    if (lane >= offset) before += other;
  }
  const int total = __shfl_sync(0xffffffffu, before, 31);
  before -= sum;
  const int columns = a.kv_heads * p.group_tiles;  // items of a slot
  const int all = total * columns;                 // (the host has made sure that it fits)
  const int worker = static_cast<int>(blockIdx.x) * G::kWarps + warp;
  if (worker == 0 && lane == 0) p.sums[p.slots] = total;
  const int workers = suffix_workers(p.workers, p.beside, p.beside_most, all);  // (no warp is dealt nothing while another has something)
  int position = worker < workers ? static_cast<int>(static_cast<long long>(all) * worker / workers) : 0;
  const int end = worker < workers ? static_cast<int>(static_cast<long long>(all) * (worker + 1) / workers) : 0;
  // the run of sequences that the first position lies in, to be walked from its first
  const int in_run = 31 - __clz(__ballot_sync(0xffffffffu, before <= position / columns) | 1u);
  int slot_sum = __shfl_sync(0xffffffffu, before, in_run);  // weight of the slots before `slot`
  int sequence = in_run * per_lane, length = 0, slices = 0, weight = 0, slot = 0, first = 0;
  Tokens tokens{0, 0};
  if (position < end) {
    tokens = tokens_of(sequence), length = a.lengths[sequence];
    first = tokens.begin, slot = a.query_starts != nullptr ? first / p.tokens_per_item + sequence : sequence;
  }
  const uint32_t ring = smem_base + warp * G::kWarpBytes;
  float* probabilities = reinterpret_cast<float*>(smem + G::kProbOffset + warp * G::kProbBytes);
  while (position < end) {
    for (;;) {  // on to the slot that has the position
      if (first < tokens.end) {
        slices = suffix_slices(a, prefix_slices, length, tokens.end - 1, min(tokens.end, first + p.tokens_per_item) - 1);
        weight = suffix_weight(slices);
        if (position < (slot_sum + weight) * columns) break;
        slot_sum += weight;
        first += p.tokens_per_item, ++slot;
      } else {
        if (++sequence >= a.batch) break;  // (the sums agree with the walk: not reached)
        tokens = tokens_of(sequence), length = a.lengths[sequence];
        first = tokens.begin, slot = a.query_starts != nullptr ? first / p.tokens_per_item + sequence : sequence;
      }
    }
    if (sequence >= a.batch) break;
    if (lane == 0) p.sums[slot] = slot_sum;
    const int in_slot = position - slot_sum * columns;
    const int column = in_slot / weight, in_item = in_slot - column * weight;
    if (column < 0 || column >= columns) break;  // (query_starts that decrease: the sums may have wrapped)
    const int stop = min(weight, in_item + end - position);
    position += stop - in_item;
    const int first_slice = max(0, in_item - kItemWeight), mine = max(0, stop - kItemWeight) - first_slice;
    if (mine <= 0) continue;  // (only the item's extra weight was dealt to this warp)
    const int count = min(p.tokens_per_item, tokens.end - first);
    const int kv = column / p.group_tiles, group0 = column % p.group_tiles * 16;
    const int heads = min(16, a.group - group0), rows = count * heads;  // rows are [token][head in group]
    auto sees_of = [&](int t) { return suffix_sees(a, length, tokens.end - 1, t); };
    const int all_see = sees_of(first), some_see = sees_of(first + count - 1);

    const T* k_base = static_cast<const T*>(a.k) + kv * a.k_sh;
    const T* v_base = static_cast<const T*>(a.v) + kv * a.v_sh;
    const int* pages = a.page_table + sequence * a.table_stride;
    constexpr int kPieces = kDim / 8;           // 16-byte pieces of a row
    constexpr int kRowsPerStep = 32 / kPieces;  // rows a warp-wide copy covers
    const int piece = lane % kPieces, sub_row = lane / kPieces;
    // pages of the next two slices, looked up ahead: the slice's own, or - pages that end inside a slice - that of this lane's key (lanes 0..15)
    auto in_prefix = [&](int i) { return kJoined && first_slice + i < prefix_slices; };
    auto first_key = [&](int i) { return (in_prefix(i) ? first_slice + i : first_slice + i - prefix_slices) * G::kKeys; };  // of slice i, in its own sequence
    int page_slot = 0, page_offset = 0;  // where the slice to be looked up next starts
    if constexpr (kWholePages) page_slot = first_key(0) / a.page_size, page_offset = first_key(0) - page_slot * a.page_size;
    int look = 0;
    auto page_of_next = [&] {
      int page = -1;
      if constexpr (kWholePages) {
        if (kJoined && first_slice + look == prefix_slices) page_slot = page_offset = 0;
        if (look < mine && (in_prefix(look) || page_slot < a.table_width)) page = __ldg((in_prefix(look) ? a.prefix_pages : pages) + page_slot);
        page_offset += G::kKeys;
        if (page_offset >= a.page_size) page_offset = 0, ++page_slot;
      } else {
        const int key = first_key(look) + (lane & 15);
        if (look < mine && key < (in_prefix(look) ? a.prefix_len : some_see)) page = __ldg((in_prefix(look) ? a.prefix_pages : pages) + key / a.page_size);
      }
      ++look;
      return page;
    };
    int offset_next = page_offset;
    int page_next = page_of_next(), page_after = page_of_next();
    auto issue = [&](int i) {
      if (i < mine) {
        const int stage = i % G::kStages, page = page_next;
        page_next = page_after;
        page_after = page_of_next();
        const bool there = page >= 0 && page < a.pages;
        const uint32_t dst = ring + stage * 2 * G::kTileBytes + sub_row * G::kRowBytes;
        uint32_t mask;
        long long k_at = 0, v_at = 0;
        if constexpr (kWholePages) {
          const int keys = min(G::kKeys, (in_prefix(i) ? a.prefix_len : some_see) - first_key(i));
          if (kJoined && first_slice + i == prefix_slices) offset_next = 0;
          mask = there ? 0xffffu >> (16 - keys) : 0u;
          if (there) {
            k_at = page * a.k_sp + (offset_next + sub_row) * a.k_ss, v_at = page * a.v_sp + (offset_next + sub_row) * a.v_ss;
          }
          offset_next += G::kKeys;
          if (offset_next >= a.page_size) offset_next = 0;
        } else {
          mask = __ballot_sync(0xffffffffu, there) & 0xffffu;
          const long long offset = (first_key(i) + (lane & 15)) % a.page_size;
          if (there) k_at = page * a.k_sp + offset * a.k_ss, v_at = page * a.v_sp + offset * a.v_ss;
        }
        if (lane == 0) present[stage] = mask;
        const T *k_from = k_base + k_at, *v_from = v_base + v_at;
#pragma unroll
        for (int step = 0; step < G::kKeys / kRowsPerStep; ++step) {
          const int row = step * kRowsPerStep + sub_row;
          if constexpr (!kWholePages) {
            k_from = k_base + __shfl_sync(0xffffffffu, k_at, row);
            v_from = v_base + __shfl_sync(0xffffffffu, v_at, row);
          }
          // (nothing is read where the size is 0: the address may be any)
          const uint32_t bytes = (mask >> row & 1u) != 0 && piece * 8 < a.head_dim ? 16 : 0;
          const uint32_t to = dst + step * kRowsPerStep * G::kRowBytes + ((piece ^ (row & 7)) << 4);
          cp_async_16(to, bytes != 0 ? k_from + piece * 8 : k_base, bytes);
          cp_async_16(to + G::kTileBytes, bytes != 0 ? v_from + piece * 8 : v_base, bytes);
          if constexpr (kWholePages) k_from += kRowsPerStep * a.k_ss, v_from += kRowsPerStep * a.v_ss;
        }
      }
      cp_async_commit();
    };

    const int r_low = lane >> 2, r_high = r_low + 8;
    uint32_t q[kDim / 16][4];
    const int sees[2] = {r_low < rows ? sees_of(first + r_low / heads) : 0, r_high < rows ? sees_of(first + r_high / heads) : 0};
    const float scale = a.scale * 1.4426950408889634f;
    float o[kDim / 8][4];
#pragma unroll
    for (int nt = 0; nt < kDim / 8; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[nt][e] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};  // m is never NaN: a NaN score shows in l
    uint32_t keyed[2] = {0u, 0u};                             // not zero: the row has seen a key

    for (int i = 1 - G::kStages; i < mine; ++i) {
      issue(i + G::kStages - 1);
      if (i < 0) {
        // Q, by way of the second stage, which is filled with keys only after this: the A fragments of sixteen rows
        const uint32_t q_tile = ring + 2 * G::kTileBytes;
#pragma unroll
        for (int step = 0; step < G::kRows / kRowsPerStep; ++step) {
          const int row = step * kRowsPerStep + sub_row;
          const bool there = row < rows && piece * 8 < a.head_dim;
          const int t = first + (there ? row / heads : 0), head = kv * a.group + group0 + (there ? row % heads : 0);
          cp_async_16(q_tile + row * G::kRowBytes + ((piece ^ (row & 7)) << 4), static_cast<const T*>(a.q) + t * a.q_st + head * a.q_sh + (there ? piece * 8 : 0), there ? 16 : 0);
        }
        cp_async_commit();
        cp_async_wait<0>();
        __syncwarp();
#pragma unroll
        for (int ks = 0; ks < kDim / 16; ++ks) {
          const int row = lane & 15, at = ks * 2 + (lane >> 4);
          ldmatrix_x4(q[ks], q_tile + row * G::kRowBytes + ((at ^ (row & 7)) << 4));
        }
        __syncwarp();
        continue;
      }
      cp_async_wait<G::kStages - 1>();
      __syncwarp();
      const int stage = i % G::kStages, key0 = first_key(i);
      const bool of_prefix = in_prefix(i);  // (every row sees it)
      const uint32_t k_tile = ring + stage * 2 * G::kTileBytes, v_tile = k_tile + G::kTileBytes;
      float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int ks = 0; ks < kDim / 16; ++ks) {
        const int key = (lane >> 4) * 8 + (lane & 7), piece = ks * 2 + ((lane >> 3) & 1);
        uint32_t b[4];
        ldmatrix_x4(b, k_tile + key * G::kRowBytes + ((piece ^ (key & 7)) << 4));
        mma_16816<T>(s[0], q[ks], b[0], b[1]);
        mma_16816<T>(s[1], q[ks], b[2], b[3]);
      }
      const uint32_t mask = present[stage];
      uint32_t visible[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        visible[h] = of_prefix ? mask : mask & ((1u << max(0, min(G::kKeys, sees[h] - key0))) - 1u);
        keyed[h] |= visible[h];
      }
      float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int nt = 0; nt < 2; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = nt * 8 + (lane & 3) * 2 + (e & 1);
          s[nt][e] = (visible[e >> 1] >> key & 1u) != 0 ? s[nt][e] * scale : -INFINITY;
          top[e >> 1] = fmaxf(top[e >> 1], s[nt][e]);
        }
      bool moves = false;
      float m_new[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
        top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
        // the maximum is moved only when it would grow by more than 2^8: O and l carry the same one, so nothing is lost
        m_new[h] = top[h] > m[h] + 8.f ? top[h] : m[h];
        moves = moves || m_new[h] != m[h];
      }
      if (__any_sync(0xffffffffu, moves)) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float keep = m_new[h] == m[h] ? 1.f : exp2_approx(m[h] - m_new[h]);
          m[h] = m_new[h];
          l[h] *= keep;
#pragma unroll
          for (int nt = 0; nt < kDim / 8; ++nt) o[nt][2 * h] *= keep, o[nt][2 * h + 1] *= keep;
        }
      }
#pragma unroll
      for (int nt = 0; nt < 2; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float base = m[e >> 1] == -INFINITY ? 0.f : m[e >> 1];
          s[nt][e] = exp2_approx(s[nt][e] - base);
          l[e >> 1] += s[nt][e];
        }
      if (!of_prefix && key0 + G::kKeys > all_see && all_see < some_see) {
        // keys that not every row sees: added here, one by one, where a row that does not see a key does not touch its value
        __syncwarp();
#pragma unroll
        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int key = nt * 8 + (lane & 3) * 2 + (e & 1);
            probabilities[(e < 2 ? r_low : r_high) * G::kKeys + key] = s[nt][e];
            if (key0 + key >= all_see) s[nt][e] = 0.f;
          }
        __syncwarp();
#pragma unroll 1
        for (int key = max(0, all_see - key0); key < min(G::kKeys, some_see - key0); ++key) {
          const float p_low = probabilities[r_low * G::kKeys + key], p_high = probabilities[r_high * G::kKeys + key];
#pragma unroll
          for (int nt = 0; nt < kDim / 8; ++nt) {
            uint32_t raw;
            asm volatile("ld.shared.u32 %0, [%1];" : "=r"(raw) : "r"(v_tile + key * G::kRowBytes + ((nt ^ (key & 7)) << 4) + (lane & 3) * 4) : "memory");
            const float2 x = unpack2<T>(raw);
            if (p_low != 0.f) o[nt][0] = fmaf(p_low, x.x, o[nt][0]), o[nt][1] = fmaf(p_low, x.y, o[nt][1]);
            if (p_high != 0.f) o[nt][2] = fmaf(p_high, x.x, o[nt][2]), o[nt][3] = fmaf(p_high, x.y, o[nt][3]);
          }
        }
        __syncwarp();
        for (int piece = lane; piece < G::kKeys * kPieces; piece += 32) {
          const int key = piece / kPieces;
          if (key0 + key >= all_see)
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(v_tile + key * G::kRowBytes + (piece % kPieces << 4)), "r"(0) : "memory");
        }
        __syncwarp();
      }
      const uint32_t pa[4] = {prefix_pack<T>(s[0][0], s[0][1]), prefix_pack<T>(s[0][2], s[0][3]), prefix_pack<T>(s[1][0], s[1][1]),
                              prefix_pack<T>(s[1][2], s[1][3])};
#pragma unroll
      for (int nt = 0; nt < kDim / 8; nt += 2) {
        const int key = ((lane >> 3) & 1) * 8 + (lane & 7), piece = nt + (lane >> 4);
        uint32_t b[4];
        ldmatrix_x4_trans(b, v_tile + key * G::kRowBytes + ((piece ^ (key & 7)) << 4));
        mma_16816<T>(o[nt], pa, b[0], b[1]);
        mma_16816<T>(o[nt + 1], pa, b[2], b[3]);
      }
      __syncwarp();  // the slice has been read by every lane before its stage is filled again
    }
    cp_async_wait<0>();
    __syncwarp();

    // ---- the fragment leaves
    const size_t at = (static_cast<size_t>(worker) + static_cast<size_t>(slot) * columns + column) * p.item_rows;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = h == 0 ? r_low : r_high;
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
      if (m[h] == -INFINITY && keyed[h] != 0) l[h] += 1.f;  // scores of -inf alone are keys all the same (or NaN, which l keeps)
      if (r < rows) {
        if ((lane & 3) == 0) __stcg(p.fragment_ml + at + r, make_float2(m[h], l[h]));
#pragma unroll
        for (int nt = 0; nt < kDim / 8; ++nt)
          __stcg(reinterpret_cast<float2*>(p.fragment_o + (at + r) * kDim + nt * 8 + (lane & 3) * 2), make_float2(o[nt][2 * h], o[nt][2 * h + 1]));
      }
    }
  }
  // this kernel is done when the prefix kernel is, too: the merge waits for this one alone.  One CTA sees to that; the others make room
  if (blockIdx.x == 0) grid_dependency_wait();
}

// The merge: kRowWarps warps per query row, each with its share of the row's partial results.
template <typename T, int kDim, int kRowWarps>
__global__ void __launch_bounds__(128) sdpa_merge_rows_kernel(const SuffixSdpaArgs p) {
  const PrefixSdpaArgs& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int part = warp % kRowWarps;
  const long long index = static_cast<long long>(blockIdx.x) * (4 / kRowWarps) + warp / kRowWarps;  // row: token, query head
  const bool there = index < static_cast<long long>(a.tokens) * a.q_heads;
  const int t = there ? static_cast<int>(index / a.q_heads) : 0, head = there ? static_cast<int>(index - static_cast<long long>(t) * a.q_heads) : 0;
  const int kv = head / a.group, in_group = head - kv * a.group;

  // the row's sequence (the suffix kernel lets this one start only when the kernels before the attention are done: what they
  // wrote is read without waiting for it)
  int sequence = t, start = t, newest = t;
  bool owned = there;
  if (a.query_starts != nullptr) {
    owned = there && a.batch > 0 && t >= a.query_starts[0] && t < a.query_starts[a.batch];
    sequence = owned ? suffix_search(a.batch, [&](int b) { return a.query_starts[b] <= t; }) : 0;  // (the same for the warp)
    if (owned) start = max(0, a.query_starts[sequence]), newest = min(a.tokens, a.query_starts[sequence + 1]) - 1;
  }
  const int length = owned ? a.lengths[sequence] : -1;
  owned = owned && length >= 0;
  grid_dependency_wait();
  grid_launch_dependents();
  // its item and fragments
  int fragments = 0;
  size_t first_fragment = 0;  // its row in the fragments
  if (owned) {
    const int tile = (t - start) / p.tokens_per_item, first = start + tile * p.tokens_per_item;
    const int slot = a.query_starts != nullptr ? start / p.tokens_per_item + sequence + tile : sequence;
    const int last = min(newest, first + p.tokens_per_item - 1);
    const int slices = suffix_slices(a, p.prefix_slices, length, newest, last), weight = suffix_weight(slices);
    if (slices > 0) {
      const int columns = a.kv_heads * p.group_tiles, column = kv * p.group_tiles + in_group / 16;
      const int all = __ldcg(p.sums + p.slots) * columns, from = __ldcg(p.sums + slot) * columns + column * weight;
      const int workers = suffix_workers(p.workers, p.beside, p.beside_most, all);
      auto worker_of = [&](int at) { return static_cast<int>(((at + 1ll) * workers - 1) / all); };  // whose [all w / workers, all (w + 1) / workers) has it
      // (kept within the fragments whatever the sums are, should query_starts decrease)
      const int first_worker = workers <= 0 ? 0 : min(max(worker_of(from + kItemWeight), 0), workers - 1);  // (the item's extra weight lies before its slices)
      fragments = workers <= 0 ? 0 : min(worker_of(from + weight - 1), workers - 1) - first_worker + 1;
      const int heads = min(16, a.group - in_group / 16 * 16);
      first_fragment = (static_cast<size_t>(first_worker) + static_cast<size_t>(slot) * columns + column) * p.item_rows + (t - first) * heads + in_group % 16;
    }
  }
  // ---- this warp's share: eight partial results at a time, a lane per (m, l), four dims a lane, all their loads together
  const bool active = lane * 4 < kDim;
  float m = -INFINITY, l = 0.f;
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
  auto join = [&](int count, const float2* ml_at, const float* o_at, size_t step) {  // partial c: ml_at[c * step], o_at[c * step * kDim]
#pragma unroll 1
    for (int c0 = part * 8; c0 < count; c0 += kRowWarps * 8) {
      const int here = min(8, count - c0);
      const float2 ml = lane < here ? __ldcg(ml_at + (c0 + lane) * step) : make_float2(-INFINITY, 0.f);
      float4 x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e)
        x[e] = e < here && active ? __ldcg(reinterpret_cast<const float4*>(o_at + (c0 + e) * step * kDim) + lane) : make_float4(0.f, 0.f, 0.f, 0.f);
      const uint32_t keyed = __ballot_sync(0xffffffffu, ml.x != -INFINITY || ml.y != 0.f);  // the partial results that have a key
      if (keyed == 0) continue;
      float highest = ml.x;
#pragma unroll
      for (int offset = 4; offset > 0; offset >>= 1) highest = fmaxf(highest, __shfl_xor_sync(0xffffffffu, highest, offset));
      highest = __shfl_sync(0xffffffffu, highest, 0);
      // (what is the maximum itself counts once, -inf too: it still is one key or more if nothing higher comes)
      const float m_new = fmaxf(m, highest), keep = m == m_new ? 1.f : exp2_approx(m - m_new);
      m = m_new;
      const float weight = ml.x == m ? 1.f : exp2_approx(ml.x - m);
      l = l * keep + weight * ml.y;
      sum.x *= keep, sum.y *= keep, sum.z *= keep, sum.w *= keep;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float w = __shfl_sync(0xffffffffu, weight, e);
        if ((keyed >> e & 1u) != 0)  // (a partial result without a key may hold anything)
          sum.x = fmaf(w, x[e].x, sum.x), sum.y = fmaf(w, x[e].y, sum.y), sum.z = fmaf(w, x[e].z, sum.z), sum.w = fmaf(w, x[e].w, sum.w);
      }
    }
  };
  const size_t record_row = static_cast<size_t>(kv) * p.rows + static_cast<size_t>(t) * a.group + in_group;
  if (owned) {
    join(p.records, p.partial_ml + record_row, p.partial_o + record_row * kDim, static_cast<size_t>(a.kv_heads) * p.rows);
    join(fragments, p.fragment_ml + first_fragment, p.fragment_o + first_fragment * kDim, p.item_rows);
  }
#pragma unroll
  for (int offset = 4; offset > 0; offset >>= 1) l += __shfl_xor_sync(0xffffffffu, l, offset);  // (the first eight lanes')
  l = __shfl_sync(0xffffffffu, l, 0);
  if constexpr (kRowWarps > 1) {
    __shared__ float4 other_sum[kRowWarps][kDim / 4];
    __shared__ float2 other_ml[kRowWarps];
    if (active) other_sum[part][lane] = sum;
    if (lane == 0) other_ml[part] = make_float2(m, l);
    __syncthreads();
    if (part != 0) return;
    float highest = m;
#pragma unroll
    for (int w = 1; w < kRowWarps; ++w) highest = fmaxf(highest, other_ml[w].x);
    m = highest, l = 0.f, sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kRowWarps; ++w) {
      const float weight = other_ml[w].x == highest ? 1.f : exp2_approx(other_ml[w].x - highest);
      l += weight * other_ml[w].y;
      if (active) {
        const float4 x = other_sum[w][lane];
        sum.x = fmaf(weight, x.x, sum.x), sum.y = fmaf(weight, x.y, sum.y), sum.z = fmaf(weight, x.z, sum.z), sum.w = fmaf(weight, x.w, sum.w);
      }
    }
  }
  const float reciprocal = l == 0.f ? 0.f : m == -INFINITY ? NAN : 1.f / l;  // no key: zeros; only keys whose score is -inf: 0 / 0
  if (there && active && lane * 4 < a.head_dim) {
    T* out = static_cast<T*>(a.out) + t * a.o_st + head * a.o_sh + lane * 4;
    *reinterpret_cast<uint2*>(out) = make_uint2(prefix_pack<T>(sum.x * reciprocal, sum.y * reciprocal), prefix_pack<T>(sum.z * reciprocal, sum.w * reciprocal));
  }
}

}  // namespace vb200
