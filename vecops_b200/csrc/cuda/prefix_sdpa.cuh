// Attention over a prefix that all sequences share: the queries of the whole batch against the prefix's keys, once.
//
// For one key/value head the rows are every query of every token that reads it, row = token * group + head in group, so
// the prefix is one dense attention of tokens * group rows and its keys are read once per row block instead of once per
// sequence.  Per tile of 128 keys and block of 128 rows, in units of log2(e):
//     s = q.k * scale      m' = max(m, max_j s)      p = 2^(s - m')      l = l 2^(m - m') + sum p      O = O 2^(m - m') + p.V
// What bounds it: the tensor cores (two products of 128 x 128 x head_dim a tile) and, as close behind, 128 x 128
// exponentials at 16 a clock.  So two softmax groups of four warps (a thread per row) take turns with the tensor cores: while one
// computes its probabilities, the MMAs of the other run.  With more than 128 rows the groups hold two row blocks and
// share every key tile; with fewer they take the key tiles in turn and leave two partial results.  P goes back to tensor
// memory, over the scores it came from, and is the A operand of the second product there: it costs no shared memory
// bandwidth.  The maximum is only moved when it would grow by more than 2^8: O is rescaled (a round trip through
// registers) a few times at the start and then hardly ever; l and O carry the same maximum, so nothing is lost.
//   warp 0      page numbers and TMA: K and V tiles, page by page, through one ring; V is used as it lies, [key][dim]
//   warp 1      issues the MMAs
//   warps 4-11  two softmax groups; they also bring Q to shared memory
// A work item is (row block, head, chunk of key tiles); each group leaves (O, m, l) of its rows in scratch, and the suffix
// kernel, launched behind, merges them.  Every wait is bounded.
#pragma once

#include <math.h>

#include "gemm_tcgen05.cuh"  // status codes, report_status, pack_out16x2
#include "prefix_sdpa_generic.cuh"

namespace vb200 {

template <int kDim>
struct PrefixTc {
  static constexpr int kRows = 128, kKeys = 128;
  static constexpr int kAtoms = kDim / 64;               // 64 head dims (128 bytes) per swizzle atom
  static constexpr int kAtomBytes = 128 * 128;
  static constexpr int kTileBytes = kAtoms * kAtomBytes;  // Q, K or V: 128 rows
  static constexpr int kSlots = kDim == 128 ? 5 : 8;
  static constexpr int kQOffset = 0;
  static constexpr int kRingOffset = 2 * kTileBytes;
  static constexpr int kMaskOffset = kRingOffset + kSlots * kTileBytes;
  static constexpr int kMaskSlots = 16;                  // per key tile: which sixteenths lie in pages outside the cache
  static constexpr int kBarrierOffset = kMaskOffset + kMaskSlots * 4;
  static constexpr int kBarriers = 2 * kSlots + 5;
  static constexpr int kSmemBytes = kBarrierOffset + kBarriers * 8 + 16 + 1024;
  static constexpr int kThreads = 384;
  static constexpr int kTmemColumns = 512;               // group g: scores (and probabilities over them) at 256 g, O at 256 g + 128
};
static_assert(PrefixTc<128>::kSmemBytes <= 227 * 1024 && PrefixTc<64>::kSmemBytes <= 227 * 1024, "shared memory budget");

struct PrefixTcArgs {
  PrefixSdpaArgs a;
  int rows;            // tokens * group, per key/value head
  int row_blocks;      // work items' blocks: 256 rows, or 128 when there is one group's worth
  int tiles, tiles_per_chunk;
  int both_rows;       // 1: the groups hold two blocks of 128 rows; 0: one block, the groups take the key tiles in turn
  int box_keys;        // keys per TMA box: min(page_size, 128)
  float* partial_o;    // [record][kv head][row][kDim]
  float2* partial_ml;  // [record][kv head][row] (m, l)
  uint32_t* status;
};

template <typename T>
__device__ __forceinline__ uint32_t prefix_pack(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t prefix_pack<__nv_bfloat16>(float lo, float hi) { return pack_out16x2<__nv_bfloat16>(lo, hi); }
template <>
__device__ __forceinline__ uint32_t prefix_pack<__half>(float lo, float hi) { return pack_out16x2<__half>(lo, hi); }

template <typename T, int kDim>
__global__ void __launch_bounds__(PrefixTc<kDim>::kThreads, 1)
prefix_sdpa_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const PrefixTcArgs p) {
  using G = PrefixTc<kDim>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
  const uint32_t full_bar = smem_base + G::kBarrierOffset;  // [slots] a K or V tile landed        (TMA -> MMA)
  const uint32_t empty_bar = full_bar + 8 * G::kSlots;      // [slots] the MMAs that read it done  (MMA -> TMA)
  const uint32_t q_bar = empty_bar + 8 * G::kSlots;         //     Q in shared memory              (softmax -> MMA)
  const uint32_t s_bar = q_bar + 8;                         // [2] scores ready, O up to date      (MMA -> softmax)
  const uint32_t p_bar = s_bar + 16;                        // [2] probabilities ready             (softmax -> MMA)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem_gen + G::kBarrierOffset + 8 * G::kBarriers);
  volatile uint32_t* abort_flag = tmem_slot + 1;
  volatile uint32_t* absent = reinterpret_cast<volatile uint32_t*>(smem_gen + G::kMaskOffset);

  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const int kv = blockIdx.y, row_block = blockIdx.z, chunk = blockIdx.x;
  const int first_tile = chunk * p.tiles_per_chunk;
  const int n = min(p.tiles_per_chunk, p.tiles - first_tile);  // >= 1
  const int row0 = row_block * (p.both_rows ? 2 * G::kRows : G::kRows);
  // what the MMA warp reads of the next tile while it still owes a product: K runs `lead` tiles ahead of V
  const int lead = p.both_rows ? 1 : 2;

  if (threadIdx.x == 0) {
    for (int s = 0; s < G::kSlots; ++s) {
      mbar_init(full_bar + 8 * s, 1);
      mbar_init(empty_bar + 8 * s, 1);
    }
    mbar_init(q_bar, 8);
    for (int g = 0; g < 2; ++g) {
      mbar_init(s_bar + 8 * g, 1);
      mbar_init(p_bar + 8 * g, 4);
    }
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_descriptor(&map_k);
    tma_prefetch_descriptor(&map_v);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), G::kTmemColumns);
    tmem_relinquish();
  }
  tcgen05_fence_before_sync();
  __syncthreads();
  tcgen05_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  // The suffix kernel may start only when the kernels before this one are done: it reads what they wrote without waiting.
  grid_dependency_wait();
  grid_launch_dependents();

  auto give_up = [&](uint32_t code) {
    report_status(p.status, code);
    *abort_flag = 1;
  };

  if (warp < 4) {
    if (warp == 0) {
      // ---------------------------------------------------------------- pages and TMA: a lane per page of the tile
      const int boxes = G::kKeys / p.box_keys;
      auto page_of = [&](int tile) {  // page number of this lane's box, or one that is outside any cache
        const int key = (first_tile + tile) * G::kKeys + lane * p.box_keys;
        return lane < boxes && tile < n && key < p.a.prefix_len ? __ldg(p.a.prefix_pages + key / p.a.page_size) : -1;
      };
      int slot = 0;
      uint32_t phase = 1;
      bool ok = true;
      auto load = [&](const CUtensorMap* map, int tile, int page) {
        if (!mbar_wait(empty_bar + 8 * slot, phase, abort_flag)) {
          if (lane == 0) give_up(kStatusProducerWait);
          ok = false;
          return;
        }
        const int key = (first_tile + tile) * G::kKeys + lane * p.box_keys;
        const bool mine = lane < boxes && key < p.a.prefix_len;
        const uint32_t loads = __popc(__ballot_sync(0xffffffffu, mine));
        if (lane == 0) mbar_arrive_expect_tx(full_bar + 8 * slot, loads * p.box_keys * 128 * G::kAtoms);
        __syncwarp();
        if (mine) {
          const uint32_t dst = smem_base + G::kRingOffset + slot * G::kTileBytes + lane * p.box_keys * 128;
#pragma unroll
          for (int atom = 0; atom < G::kAtoms; ++atom)  // a page outside the cache reads as zeros
            tma_load_4d(dst + atom * G::kAtomBytes, map, full_bar + 8 * slot, atom * 64, key % p.a.page_size, kv, page);
        }
        if (++slot == G::kSlots) slot = 0, phase ^= 1u;
      };
      // K tiles [0, lead), then V tile j and K tile j + lead in turn; a tile's pages are looked up ahead of both
      int k_pages[2] = {page_of(0), page_of(1)};  // of the next two K tiles
      int v_pages[2] = {0, 0};                    // of the `lead` K tiles loaded last, oldest first
      auto load_k = [&](int tile) {
        const int page = k_pages[0];
        k_pages[0] = k_pages[1];
        k_pages[1] = page_of(tile + 2);
        const int key = (first_tile + tile) * G::kKeys + lane * p.box_keys;
        const bool gone = lane < boxes && key < p.a.prefix_len && (page < 0 || page >= p.a.pages);
        uint32_t mask = __ballot_sync(0xffffffffu, gone);
        if (lane == 0) absent[tile % G::kMaskSlots] = mask;
        load(&map_k, tile, page);
        if (lead == 1) v_pages[0] = page;
        else v_pages[0] = v_pages[1], v_pages[1] = page;
      };
      for (int tile = 0; ok && tile < lead && tile < n; ++tile) load_k(tile);
      if (lead == 2 && n == 1) v_pages[0] = v_pages[1];
      for (int tile = 0; ok && tile < n; ++tile) {
        load(&map_v, tile, v_pages[0]);
        if (!ok) break;
        if (tile + lead < n) load_k(tile + lead);
        else v_pages[0] = v_pages[1];
      }
    } else if (warp == 1) {
      // ---------------------------------------------------------------- MMAs
      const uint32_t type = std::is_same<T, __nv_bfloat16>::value ? kUmmaBF16 : kUmmaF16;
      const uint32_t idesc_s = umma_instr_desc(kUmmaAccF32, type, type, 128, 128);
      const uint32_t idesc_o = umma_instr_desc(kUmmaAccF32, type, type, 128, kDim, true);  // B = V, N-major
      const int q_steps = (p.a.head_dim + 15) / 16;  // what lies past head_dim is zero in both operands
      const bool leader = elect_one();
      bool ok = true;
      int slot = 0;
      uint32_t phase = 0;
      auto wait = [&](uint32_t bar, uint32_t parity) {
        if (ok && !mbar_wait(bar, parity, abort_flag)) {
          if (leader) give_up(kStatusMmaWaitFull);
          ok = false;
        }
      };
      auto next_slot = [&] {
        if (++slot == G::kSlots) slot = 0, phase ^= 1u;
      };
      auto scores = [&](int g, int at) {  // S_g = Q_g . K^T
        const uint32_t q = smem_base + G::kQOffset + (p.both_rows ? g * G::kTileBytes : 0), k = smem_base + G::kRingOffset + at * G::kTileBytes;
        if (leader) {
          for (int ks = 0; ks < q_steps; ++ks)
            umma_f16(tmem_base + g * 256, umma_smem_desc_sw128(q + (ks >> 2) * G::kAtomBytes) + 2 * (ks & 3),
                     umma_smem_desc_sw128(k + (ks >> 2) * G::kAtomBytes) + 2 * (ks & 3), idesc_s, ks > 0 ? 1u : 0u);
        }
        __syncwarp();
      };
      auto commit = [&](uint32_t bar) {
        if (leader) umma_commit(bar);
        __syncwarp();
      };
      wait(q_bar, 0);
      for (int tile = 0; ok && tile < lead && tile < n; ++tile) {
        wait(full_bar + 8 * slot, phase);
        if (!ok) break;
        tcgen05_fence_after_sync();
        for (int g = p.both_rows ? 0 : tile; g < (p.both_rows ? 2 : tile + 1); ++g) {
          scores(g, slot);
          commit(s_bar + 8 * g);
        }
        commit(empty_bar + 8 * slot);
        next_slot();
      }
      for (int tile = 0; ok && tile < n; ++tile) {
        const int v_slot = slot;
        const uint32_t v_phase = phase;
        next_slot();
        const int k_slot = slot;
        const uint32_t k_phase = phase;
        const bool more = tile + lead < n;
        const uint32_t v = smem_base + G::kRingOffset + v_slot * G::kTileBytes;
        wait(full_bar + 8 * v_slot, v_phase);
        if (!ok) break;
        const int last = p.a.prefix_len - (first_tile + tile) * G::kKeys;
        if (last < G::kKeys) {
          // the prefix ends inside the tile: whatever lies behind it, NaN included, must not meet the zero probabilities there
          for (int i = lane; i < (G::kKeys - last) * 8 * G::kAtoms; i += 32) {
            const int row = last + i / (8 * G::kAtoms), piece = i % (8 * G::kAtoms);
            const uint32_t dst = v + (piece >> 3) * G::kAtomBytes + row * 128 + ((piece & 7) << 4);
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(dst), "r"(0) : "memory");
          }
          fence_proxy_async_smem();
          __syncwarp();
        }
        for (int g = p.both_rows ? 0 : tile & 1; ok && g < (p.both_rows ? 2 : (tile & 1) + 1); ++g) {
          const int turn = p.both_rows ? tile : tile >> 1;  // how many tiles this group had before
          wait(p_bar + 8 * g, static_cast<uint32_t>(turn) & 1u);
          if (!ok) break;
          tcgen05_fence_after_sync();
          if (leader) {
#pragma unroll
            for (int ks = 0; ks < G::kKeys / 16; ++ks)  // 16 keys: 8 columns of P, 16 rows of V
              umma_f16_from_tmem(tmem_base + g * 256 + 128, tmem_base + g * 256 + ks * 8, umma_smem_desc_sw128_mn(v + ks * 16 * 128, G::kAtomBytes, 1024), idesc_o,
                                 turn > 0 || ks > 0 ? 1u : 0u);
          }
          __syncwarp();
          if (more) {
            wait(full_bar + 8 * k_slot, k_phase);
            if (!ok) break;
            tcgen05_fence_after_sync();
            scores(g, k_slot);  // (over P_g: the tensor core works in order)
          }
          commit(s_bar + 8 * g);
        }
        if (!ok) break;
        commit(empty_bar + 8 * v_slot);
        if (more) {
          commit(empty_bar + 8 * k_slot);
          next_slot();
        }
      }
    }
  } else {
    // ---------------------------------------------------------------- softmax: a thread per row
    const int g = (warp - 4) >> 2, quarter = warp & 3;
    const int thread = static_cast<int>(threadIdx.x) - 128;
    {
      // Q: rows of 16-byte pieces under the 128-byte swizzle; rows past the last and dims past head_dim are zero
      // (eight rows' loads in flight together)
      constexpr int kPieces = kDim / 8, kRowStep = 256 / kPieces, kTogether = 8;
      const int piece = thread % kPieces;
      const bool in_head = piece * 8 < p.a.head_dim;
#pragma unroll 1
      for (int first = thread / kPieces; first < (p.both_rows ? 2 * G::kRows : G::kRows); first += kRowStep * kTogether) {
        uint4 x[kTogether];
#pragma unroll
        for (int i = 0; i < kTogether; ++i) {
          const int r = row0 + first + i * kRowStep;
          x[i] = make_uint4(0, 0, 0, 0);
          if (r < p.rows && in_head) {
            const int t = r / p.a.group, head = kv * p.a.group + r - t * p.a.group;
            x[i] = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(p.a.q) + t * p.a.q_st + head * p.a.q_sh + piece * 8));
          }
        }
#pragma unroll
        for (int i = 0; i < kTogether; ++i) {
          const int row = first + i * kRowStep;
          const uint32_t dst = smem_base + G::kQOffset + (row >> 7) * G::kTileBytes + (piece >> 3) * G::kAtomBytes + (row & 127) * 128 + (((piece & 7) ^ (row & 7)) << 4);
          if (row < (p.both_rows ? 2 * G::kRows : G::kRows))
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(x[i].x), "r"(x[i].y), "r"(x[i].z), "r"(x[i].w) : "memory");
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_bar);
    }
    const int row = row0 + (p.both_rows ? g * G::kRows : 0) + quarter * 32 + lane;
    const uint32_t my_tmem = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + g * 256;
    const float signed_scale = p.a.scale * 1.4426950408889634f;  // scores in units of log2(e)
    const float scale = signed_scale == 0.f ? 1.f : fabsf(signed_scale);
    const int box_shift = 31 - __clz(p.box_keys);
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    int turn = 0;
    auto wait_scores = [&] {
      if (!__all_sync(0xffffffffu, mbar_wait(s_bar + 8 * g, static_cast<uint32_t>(turn) & 1u, abort_flag))) {
        if (lane == 0) give_up(kStatusEpilogueWait);
        ok = false;
      }
      tcgen05_fence_after_sync();
    };
    for (int tile = p.both_rows ? 0 : g; ok && tile < n; tile += p.both_rows ? 1 : 2, ++turn) {
      wait_scores();
      if (!ok) break;
      // Two passes over the scores where they lie, 32 columns at a time: the maximum, then the probabilities, which go over
      // columns already read.  (128 scores held in registers instead spilled, and the code, unrolled, took longer to fetch
      // than a short item takes to run.)
      const int last = p.a.prefix_len - (first_tile + tile) * G::kKeys;
      const uint32_t gone = absent[tile % G::kMaskSlots];
      const bool cut = last < G::kKeys || gone != 0;  // (the same for the whole item)
      auto load_scores = [&](int col, float (&t)[32]) {
        tmem_load_32x32(my_tmem + col, reinterpret_cast<uint32_t(&)[32]>(t));
        tmem_load_wait();
        if (signed_scale <= 0.f) {  // (so that the factor below is positive: the maximum, and a masked -inf, keep their meaning)
          const float sign = signed_scale < 0.f ? -1.f : 0.f;
#pragma unroll
          for (int j = 0; j < 32; ++j) t[j] *= sign;
        }
        if (cut) {
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (col + j >= last || (gone >> ((col + j) >> box_shift) & 1u) != 0) t[j] = -INFINITY;
        }
      };
      float highest = -INFINITY;
#pragma unroll 1
      for (int col = 0; col < 128; col += 32) {
        float t[32];
        load_scores(col, t);
        float top[4] = {t[0], t[1], t[2], t[3]};
#pragma unroll
        for (int j = 4; j < 32; ++j) top[j & 3] = fmaxf(top[j & 3], t[j]);
        highest = fmaxf(highest, fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])));
      }
      const float tile_max = highest * scale;
      const bool moves = turn == 0 || tile_max > m + 8.f;
      if (turn == 0) {
        m = tile_max;
      } else if (__any_sync(0xffffffffu, moves)) {
        const float m_new = moves ? tile_max : m;
        const float keep = moves ? exp2_approx(m - m_new) : 1.f;
        l *= keep;
        m = m_new;
#pragma unroll 1
        for (int col = 0; col < kDim; col += 32) {
          uint32_t o[32];
          tmem_load_32x32(my_tmem + 128 + col, o);
          tmem_load_wait();
#pragma unroll
          for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * keep);
          tmem_store_32x32(my_tmem + 128 + col, o);
        }
      }
      const float m_use = m == -INFINITY ? 0.f : m;  // nothing kept so far: every p is 0
      float sums[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
      for (int col = 0; col < 128; col += 32) {
        float t[32];
        load_scores(col, t);
        uint32_t packed[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const float p0 = exp2_approx(fmaf(t[2 * j], scale, -m_use)), p1 = exp2_approx(fmaf(t[2 * j + 1], scale, -m_use));
          sums[(2 * j) & 3] += p0;
          sums[(2 * j + 1) & 3] += p1;
          packed[j] = prefix_pack<T>(p0, p1);
        }
        tmem_store_32x16(my_tmem + col / 2, packed);
      }
      l += (sums[0] + sums[1]) + (sums[2] + sums[3]);
      tmem_store_wait();
      tcgen05_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_bar + 8 * g);
    }
    // ---- this group's rows of the chunk leave: O, m, l
    const int record = p.both_rows ? chunk : 2 * chunk + g;
    const size_t at = (static_cast<size_t>(record) * p.a.kv_heads + kv) * p.rows + row;
    if (turn > 0 && ok) wait_scores();  // the last product is in O
    if (ok && turn > 0) {
#pragma unroll 1
      for (int col = 0; col < kDim; col += 32) {
        uint32_t o[32];
        tmem_load_32x32(my_tmem + 128 + col, o);
        tmem_load_wait();
        if (row < p.rows) {
          float4* to = reinterpret_cast<float4*>(p.partial_o + at * kDim + col);
#pragma unroll
          for (int j = 0; j < 8; ++j)
            __stcg(to + j, make_float4(__uint_as_float(o[4 * j]), __uint_as_float(o[4 * j + 1]), __uint_as_float(o[4 * j + 2]), __uint_as_float(o[4 * j + 3])));
        }
      }
    }
    if (row < p.rows) __stcg(p.partial_ml + at, make_float2(turn > 0 && ok ? m : -INFINITY, turn > 0 && ok ? l : 0.f));
  }

  // ---------------------------------------------------------------- teardown
  __syncthreads();
  if (*abort_flag != 0) {
    for (int i = 0; i < 1000; ++i) __nanosleep(1000);
    __syncthreads();
  }
  if (warp == 1) {
    tcgen05_fence_after_sync();
    tmem_dealloc(tmem_base, G::kTmemColumns);
  }
}

}  // namespace vb200
