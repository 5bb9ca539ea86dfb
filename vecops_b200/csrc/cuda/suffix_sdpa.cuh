// Attention over each sequence's own suffix, merged with what the prefix kernel left: the second half of shared-prefix
// attention, and all of it when there is no prefix.
//
// A work item is up to sixteen query rows of one sequence and one key/value head - the queries that read this head, of one
// token or of a few neighbouring ones - against the keys they see.  Its time is the keys' way from memory: every key and
// value is used by at most sixteen rows.  So the keys go sixteen at a time to the warps of a CTA, and of a cluster of CTAs
// where there are few items; a warp keeps three such slices in flight for itself by cp.async (no barrier in the
// loop) and multiplies them with mma.sync m16n8k16, whose sixteen rows are the item's; tcgen05's 128 rows would be nearly
// empty.  Each warp runs the recurrence m' = max(m, s), l, O of its own slices; at the end the warps of the cluster and
// the prefix kernel's records meet,
//     M = max m_c      out = sum_c 2^(m_c - M) O_c / sum_c 2^(m_c - M) l_c           (m in units of log2(e))
// in an order that does not depend on timing.  Keys that some of the item's rows see and others do not - at most fifteen, the
// newest tokens' own - go past the tensor core: there a zero probability times whatever a later token's value holds
// would still be NaN.
#pragma once

#include "prefix_sdpa.cuh"

namespace vb200 {

template <int kDim>
struct SuffixSdpa {
  static constexpr int kWarps = 4, kThreads = 32 * kWarps;
  static constexpr int kRows = 16, kKeys = 16;
  static constexpr int kStages = 3;
  static constexpr int kRowBytes = kDim * 2;
  static constexpr int kTileBytes = kKeys * kRowBytes;
  static constexpr int kWarpBytes = kStages * 2 * kTileBytes;
  static constexpr int kPitch = kDim + 4;  // floats of a row of O while the warps meet, over the ring
  static constexpr int kExtraOffset = kWarps * kWarpBytes;
  static constexpr int kProbBytes = kRows * kKeys * 4;  // per warp: probabilities of the keys that only some rows see
  static constexpr int kMlOffset = kExtraOffset + kWarps * kProbBytes;  // [warp][row] (m, l)
  static constexpr int kSmemBytes = kMlOffset + kWarps * kRows * 8 + kWarps * kStages * 4;
  static constexpr int kMaxSplit = 8;  // CTAs of a cluster
  static_assert(kRows * kPitch * 4 <= kWarpBytes, "a warp's O lies over its ring");
};

struct SuffixSdpaArgs {
  PrefixSdpaArgs a;
  int rows;             // tokens * group, per key/value head: the prefix records' rows
  int tokens_per_item;  // neighbouring tokens of one sequence in an item
  int group_tiles;      // items a token is cut into when its group has more than sixteen heads
  int slots;            // items per key/value head, idle ones included
  int split_bits;
  int records;          // of the prefix kernel; 0: there is none, and nothing to wait for but the kernels before
  const float* partial_o;
  const float2* partial_ml;
};

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

template <typename T, int kDim>
__global__ void __launch_bounds__(SuffixSdpa<kDim>::kThreads, 2) suffix_sdpa_kernel(const SuffixSdpaArgs p) {
  using G = SuffixSdpa<kDim>;
  extern __shared__ __align__(128) uint8_t smem[];
  const uint32_t smem_base = smem_u32(smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = 1 << p.split_bits, part = static_cast<int>(blockIdx.x) & (split - 1);
  const int kv = static_cast<int>(blockIdx.y) / p.group_tiles, group0 = static_cast<int>(blockIdx.y) % p.group_tiles * 16;
  const int slot = static_cast<int>(blockIdx.x) >> p.split_bits;
  const PrefixSdpaArgs& a = p.a;
  if (p.records == 0) grid_dependency_wait();  // (with a prefix kernel in between, the kernels before that one are done already)

  // ---------------------------------------------------------------- which sequence, which of its tokens
  // Sequence b's items are the slots from query_starts[b] / tokens_per_item + b on: apart from each other, and found without a sum.
  int sequence = slot, first = slot, count = 1, begin_all = 0, end_all = a.tokens;
  bool idle = slot >= p.slots || slot >= a.batch;
  if (a.query_starts != nullptr) {
    idle = slot >= p.slots - 1 || a.batch == 0;
    begin_all = a.query_starts[0], end_all = a.query_starts[a.batch];
    int low = 0, high = a.batch;  // the last b whose slots start at or before this one
    while (high - low > 1) {
      const int step = (high - low + 31) / 32;
      const int probe = low + lane * step;
      const bool before = probe < high && a.query_starts[probe] / p.tokens_per_item + probe <= slot;
      const int found = 31 - __clz(__ballot_sync(0xffffffffu, before) | 1u);
      low += found * step;
      high = min(high, low + step);
    }
    if (!idle) {
      sequence = low;
      const int start = a.query_starts[low], tile = slot - (start / p.tokens_per_item + low);
      first = start + tile * p.tokens_per_item;
      count = min(p.tokens_per_item, a.query_starts[low + 1] - first);
      idle = tile < 0 || first < 0 || count <= 0 || first + count > a.tokens;
    }
  }
  if (slot == p.slots - 1 && a.query_starts != nullptr && part == 0 && group0 == 0) {
    // the spare last slot zeroes the tokens of no sequence
    for (int t = warp; t < a.tokens; t += G::kWarps) {
      if (t >= begin_all && t < end_all) continue;
      for (int i = lane; i < a.group * a.head_dim; i += 32)
        (static_cast<T*>(a.out) + t * a.o_st + (kv * a.group + i / a.head_dim) * a.o_sh)[i % a.head_dim] = append_down<T>(0.f);
    }
  }
  if (idle) return;  // (uniform over the cluster, whose CTAs share the slot)
  const int length = a.lengths[sequence];
  const int heads = min(16, a.group - group0);  // rows are [token][head in group]
  const int rows = count * heads;
  if (length < 0) {
    if (part == 0) {
      for (int i = threadIdx.x; i < rows * a.head_dim; i += G::kThreads) {
        const int r = i / a.head_dim, t = first + r / heads, head = kv * a.group + group0 + r % heads;
        (static_cast<T*>(a.out) + t * a.o_st + head * a.o_sh)[i % a.head_dim] = append_down<T>(0.f);
      }
    }
    return;
  }
  // suffix keys the item's first and last token see
  const int newest = a.query_starts != nullptr ? a.query_starts[sequence + 1] - 1 : first;
  const long long capacity = static_cast<long long>(a.table_width) * a.page_size;
  auto sees_of = [&](int t) {
    const long long seen = static_cast<long long>(length) - (newest - t);
    return static_cast<int>(seen < 0 ? 0 : seen < capacity ? seen : capacity);
  };
  const int all_see = sees_of(first), some_see = sees_of(first + count - 1);

  // ---------------------------------------------------------------- this warp's slices: worker, worker + workers, ...
  const int workers = G::kWarps << p.split_bits, worker = part * G::kWarps + warp;
  const int slices = (some_see + G::kKeys - 1) / G::kKeys;
  const int mine = slices > worker ? (slices - worker + workers - 1) / workers : 0;
  const uint32_t ring = smem_base + warp * G::kWarpBytes;
  volatile uint32_t* present = reinterpret_cast<volatile uint32_t*>(smem + G::kMlOffset + G::kWarps * G::kRows * 8) + warp * G::kStages;
  const T* k_base = static_cast<const T*>(a.k) + kv * a.k_sh;
  const T* v_base = static_cast<const T*>(a.v) + kv * a.v_sh;
  const int* table = a.page_table + sequence * a.table_stride;
  auto page_of = [&](int i) {  // page of this lane's key (lanes 0..15) in slice i, or -1
    const int key = (worker + i * workers) * G::kKeys + (lane & 15);
    return i < mine && key < some_see ? __ldg(table + key / a.page_size) : -1;
  };
  constexpr int kPieces = kDim / 8;                   // 16-byte pieces of a row
  constexpr int kRowsPerStep = 32 / kPieces;          // rows a warp-wide copy covers
  int page_next = page_of(0);
  auto issue = [&](int i) {
    const int stage = i % G::kStages;
    const int page = page_next;
    page_next = page_of(i + 1);
    if (i < mine) {
      const int key = (worker + i * workers) * G::kKeys + (lane & 15);
      const bool there = page >= 0 && page < a.pages;
      const uint32_t mask = __ballot_sync(0xffffffffu, there) & 0xffffu;
      if (lane == 0) present[stage] = mask;
      const long long offset = key % a.page_size;
      const long long k_at = there ? page * a.k_sp + offset * a.k_ss : 0, v_at = there ? page * a.v_sp + offset * a.v_ss : 0;
      const uint32_t dst = ring + stage * 2 * G::kTileBytes;
      const int piece = lane % kPieces;
#pragma unroll
      for (int step = 0; step < G::kKeys / kRowsPerStep; ++step) {
        const int row = step * kRowsPerStep + lane / kPieces;
        const long long k_row = __shfl_sync(0xffffffffu, k_at, row), v_row = __shfl_sync(0xffffffffu, v_at, row);
        const uint32_t bytes = (mask >> row & 1u) != 0 && piece * 8 < a.head_dim ? 16 : 0;
        const uint32_t to = dst + row * G::kRowBytes + ((piece ^ (row & 7)) << 4);
        cp_async_16(to, k_base + k_row + (bytes != 0 ? piece * 8 : 0), bytes);
        cp_async_16(to + G::kTileBytes, v_base + v_row + (bytes != 0 ? piece * 8 : 0), bytes);
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < G::kStages - 1; ++i) issue(i);

  // Q: the A fragments of sixteen rows
  const int r_low = lane >> 2, r_high = r_low + 8;
  uint32_t q[kDim / 16][4];
  {
    const T* q_row[2];
    bool there[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = h == 0 ? r_low : r_high;
      there[h] = r < rows;
      const int t = first + (there[h] ? r / heads : 0), head = kv * a.group + group0 + (there[h] ? r % heads : 0);
      q_row[h] = static_cast<const T*>(a.q) + t * a.q_st + head * a.q_sh;
    }
#pragma unroll
    for (int ks = 0; ks < kDim / 16; ++ks)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = ks * 16 + (lane & 3) * 2 + (e >> 1) * 8;
        q[ks][e] = there[e & 1] && d < a.head_dim ? *reinterpret_cast<const uint32_t*>(q_row[e & 1] + d) : 0u;
      }
  }
  const int sees[2] = {r_low < rows ? sees_of(first + r_low / heads) : 0, r_high < rows ? sees_of(first + r_high / heads) : 0};
  const float scale = a.scale * 1.4426950408889634f;
  float o[kDim / 8][4];
#pragma unroll
  for (int nt = 0; nt < kDim / 8; ++nt)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[nt][e] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  float* probabilities = reinterpret_cast<float*>(smem + G::kExtraOffset + warp * G::kProbBytes);

  for (int i = 0; i < mine; ++i) {
    issue(i + G::kStages - 1);
    cp_async_wait<G::kStages - 1>();
    __syncwarp();
    const int stage = i % G::kStages, key0 = (worker + i * workers) * G::kKeys;
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
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int key = nt * 8 + (lane & 3) * 2 + (e & 1);
        const bool keep = key0 + key < sees[e >> 1] && (mask >> key & 1u) != 0;
        s[nt][e] = keep ? s[nt][e] * scale : -INFINITY;
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
    if (key0 + G::kKeys > all_see && all_see < some_see) {
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

  // ---------------------------------------------------------------- the warps leave (O, m, l) in shared memory
  float* mine_o = reinterpret_cast<float*>(smem + warp * G::kWarpBytes);
  float2* mine_ml = reinterpret_cast<float2*>(smem + G::kMlOffset) + warp * G::kRows;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    if ((lane & 3) == 0) mine_ml[h == 0 ? r_low : r_high] = make_float2(m[h], l[h]);
#pragma unroll
    for (int nt = 0; nt < kDim / 8; ++nt)
      *reinterpret_cast<float2*>(mine_o + (h == 0 ? r_low : r_high) * G::kPitch + nt * 8 + (lane & 3) * 2) = make_float2(o[nt][2 * h], o[nt][2 * h + 1]);
  }
  __syncthreads();
  if (split > 1) cluster_sync_all();
  if (p.records > 0) grid_dependency_wait();  // the prefix kernel's records

  // ---------------------------------------------------------------- and meet: a warp per row, four dims a lane
  for (int r = part + (warp << p.split_bits); r < rows; r += G::kWarps << p.split_bits) {
    const int t = first + r / heads, in_group = group0 + r % heads;
    // lane c holds (m, l) of partial c: the warps of the cluster first, then the records of the prefix, 32 at a time
    const uint32_t ml_at = smem_base + G::kMlOffset + ((lane & (G::kWarps - 1)) * G::kRows + r) * 8;
    float2 ml = make_float2(-INFINITY, 0.f);
    if (lane < workers) {
      const uint32_t from = map_to_cta(ml_at, lane / G::kWarps);
      ml = make_float2(ld_shared_cluster_f32(from), ld_shared_cluster_f32(from + 4));
    }
    const size_t record_row = static_cast<size_t>(kv) * p.rows + static_cast<size_t>(t) * a.group + in_group;
    const size_t record_step = static_cast<size_t>(a.kv_heads) * p.rows;
    float highest = ml.x;
    for (int c = lane; c < p.records; c += 32) highest = fmaxf(highest, __ldcg(p.partial_ml + c * record_step + record_row).x);
#pragma unroll
    for (int offset = 16; offset > 0; offset >>= 1) highest = fmaxf(highest, __shfl_xor_sync(0xffffffffu, highest, offset));
    float weight = ml.x == -INFINITY ? 0.f : exp2_approx(ml.x - highest);
    float total = weight * ml.y;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    const bool active = lane * 4 < kDim;
    for (int c = 0; c < workers; ++c) {
      const float w = __shfl_sync(0xffffffffu, weight, c);
      if (w == 0.f || !active) continue;
      const float4 x = ld_shared_cluster_v4(map_to_cta(smem_base + (c & (G::kWarps - 1)) * G::kWarpBytes + (r * G::kPitch + lane * 4) * 4, c / G::kWarps));
      sum.x = fmaf(w, x.x, sum.x), sum.y = fmaf(w, x.y, sum.y), sum.z = fmaf(w, x.z, sum.z), sum.w = fmaf(w, x.w, sum.w);
    }
    for (int c0 = 0; c0 < p.records; c0 += 32) {
      float2 record = make_float2(-INFINITY, 0.f);
      if (c0 + lane < p.records) record = __ldcg(p.partial_ml + (c0 + lane) * record_step + record_row);
      weight = record.x == -INFINITY ? 0.f : exp2_approx(record.x - highest);
      total += weight * record.y;
      const int here = min(32, p.records - c0);
      for (int c = 0; c < here; c += 8) {
        float4 x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float w = __shfl_sync(0xffffffffu, weight, (c + e) & 31);
          x[e] = c + e < here && w != 0.f && active ? __ldcg(reinterpret_cast<const float4*>(p.partial_o + ((c0 + c + e) * record_step + record_row) * kDim) + lane)
                                                    : make_float4(0.f, 0.f, 0.f, 0.f);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float w = c + e < here ? __shfl_sync(0xffffffffu, weight, (c + e) & 31) : 0.f;
          if (w != 0.f) sum.x = fmaf(w, x[e].x, sum.x), sum.y = fmaf(w, x[e].y, sum.y), sum.z = fmaf(w, x[e].z, sum.z), sum.w = fmaf(w, x[e].w, sum.w);
        }
      }
    }
#pragma unroll
    for (int offset = 16; offset > 0; offset >>= 1) total += __shfl_xor_sync(0xffffffffu, total, offset);
    const float reciprocal = total == 0.f ? 0.f : 1.f / total;  // no key: zeros
    if (active && lane * 4 < a.head_dim) {
      T* out = static_cast<T*>(a.out) + t * a.o_st + (kv * a.group + in_group) * a.o_sh + lane * 4;
      *reinterpret_cast<uint2*>(out) = make_uint2(prefix_pack<T>(sum.x * reciprocal, sum.y * reciprocal), prefix_pack<T>(sum.z * reciprocal, sum.w * reciprocal));
    }
  }
  if (split > 1) {  // no CTA leaves while another still reads its partials
    __syncwarp();
    cluster_sync_all();
  }
}

}  // namespace vb200
