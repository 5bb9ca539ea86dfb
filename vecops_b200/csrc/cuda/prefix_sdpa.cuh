// Attention over a prefix that all sequences share: the queries of the whole batch against the prefix's keys, once.
//
// For one key/value head the rows are every query of every token that reads it, row = token * group + head in group, so
// the prefix is one dense attention of tokens * group rows and its keys are read once per row block instead of once per
// sequence.  Per tile of 128 keys and block of 128 rows, in units of log2(e):
//     s = q.k * scale      m' = max(m, max_j s)      p = 2^(s - m')      l = l 2^(m - m') + sum p      O = O 2^(m - m') + p.V
// What bounds it: the tensor cores (two products of 128 x 128 x head_dim a tile) and, as close behind, 128 x 128
// exponentials at 16 a clock.  So two softmax groups take turns with the tensor cores: while one computes its
// probabilities, the MMAs of the other run.  With more than 128 rows the groups hold two row blocks and share every key
// tile; with fewer they take the key tiles in turn and leave two partial results.  A group's step is a chain - scores,
// maximum, probabilities, product, next scores - of which only one link at a time is its own, so eight warps, two threads a
// row, make the softmax link short, and a few of the exponentials are computed on the multiply-add units.  P goes back to
// tensor memory, over the scores it came from, and is the A operand of the second product there: it costs no shared
// memory bandwidth.  The maximum is only moved when it would grow by more than 2^8: O is rescaled (a round trip through
// registers) a few times at the start and then hardly ever; l and O carry the same maximum, so nothing is lost.  P is rounded to the
// type of V, as one MMA's operands are of one type, and O = P.V alone takes it so: l adds the fp32 values.  Against 64 bits the result is
// off by 1.3 to 1.4 times what a form with fp32 P is (bf16: 0.0021 to 0.0023 of the result's norm and 0.0017, the rounding of the result
// itself); P in tf32 would need V widened to 32 bits, at half the rate.
//   warp 0      page numbers and TMA, page by page: a ring of steps, V tile t with the K tile that is multiplied after it; V is
//               used as it lies, [key][dim]
//   warp 1      issues the MMAs (two issuing warps, one per group, measured 17 % slower: their MMAs alternate between
//               accumulators); what it waits for is kept to one barrier per step and one per group, as a wait costs it
//               some 150 cycles even when there is nothing to wait for
//   warps 4-19  two softmax groups; they also bring Q to shared memory
// A work item is (row block, head, chunk of key tiles); each group leaves (O, m, l) of its rows in scratch, and the merge
// kernel joins them.  Every wait is bounded.
//
// Measured: 256 sequences of 32 query heads behind 32768 keys of 8 heads of 128 (137 GFLOP): 138 us with the merge, 990 TFLOP/s,
// 0.59 of the measured bf16 rate, at 1.64 GHz under the power limit; the tensor pipe is busy 57 % of the time, the
// special-function pipe 43 %, and a step of both groups takes some 3500 cycles for 2048 of MMAs - each group's chain of
// products and softmax, of which only half lies under the other group's.  Few rows are bound by what a call begins and ends
// with: some 4500 cycles to the first scores, 1500 to 3500 for the record.
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
  static constexpr int kFirstSoftmaxWarp = 4, kGroupWarps = 8;
  // Q's place, which O leaves through at the end: 2 KB a softmax warp.  The ring begins behind all of it, as one group's O leaves while
  // the last V tile of the other is still to be multiplied.
  static constexpr int kStageBytes = 2048;
  __host__ __device__ static constexpr int q_bytes(bool both_rows) {
    const int q = (both_rows ? 2 : 1) * kTileBytes, staged = 2 * kGroupWarps * kStageBytes;
    return q > staged ? q : staged;
  }
  // what is left beside Q: steps of a V and a K tile.  One row block needs less for Q and has room for more of them.
  static constexpr int kSpace = 224 * 1024;
  static constexpr int kMostSteps = 6;
  __host__ __device__ static constexpr int steps(bool both_rows) {
    const int fit = (kSpace - q_bytes(both_rows)) / (2 * kTileBytes);
    return fit < kMostSteps ? fit : kMostSteps;
  }
  static constexpr int kMaskOffset = kSpace;
  static constexpr int kMaskSlots = 16;                  // per key tile: which of its pages lie outside the cache
  static constexpr int kExchangeOffset = kMaskOffset + kMaskSlots * 4;
  static constexpr int kExchangeBytes = 2 * 2 * 128 * 4;  // [group][half of the row][row] fp32
  static constexpr int kBarrierOffset = kExchangeOffset + kExchangeBytes;
  static constexpr int kBarriers = 2 * kMostSteps + 5;
  static constexpr int kAlign = 256;                     // of dynamic shared memory; the tiles' swizzle wants 1024
  static constexpr int kSmemBytes = kBarrierOffset + kBarriers * 8 + 8 + 1024 - kAlign;
  static constexpr int kThreads = 32 * (kFirstSoftmaxWarp + 2 * kGroupWarps);
  static constexpr int kPolynomialPairs = 4;             // of 16 pairs of exponentials, those computed beside the special-function units
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
  int k_head_step, v_head_step;  // from head to head in the maps: 1, or 0 when all heads have the same rows
  float* partial_o;    // [record][kv head][row][kDim]
  float2* partial_ml;  // [record][kv head][row] (m, l); (-inf, 0) for no key, (-inf, > 0) for keys whose scores are all -inf
  uint32_t* status;
};

template <typename T>
__device__ __forceinline__ uint32_t prefix_pack(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t prefix_pack<__nv_bfloat16>(float lo, float hi) { return pack_out16x2<__nv_bfloat16>(lo, hi); }
template <>
__device__ __forceinline__ uint32_t prefix_pack<__half>(float lo, float hi) { return pack_out16x2<__half>(lo, hi); }

// Two fp32 values in one 64-bit register, and arithmetic on both at once.
__device__ __forceinline__ unsigned long long f2_pack(float x, float y) {
  unsigned long long v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(x), "f"(y));
  return v;
}
__device__ __forceinline__ float2 f2_unpack(unsigned long long v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ unsigned long long f2_add(unsigned long long a, unsigned long long b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ unsigned long long f2_mul(unsigned long long a, unsigned long long b) {
  unsigned long long r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ unsigned long long f2_fma(unsigned long long a, unsigned long long b, unsigned long long c) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ unsigned long long f2_same(float x) { return f2_pack(x, x); }

// 2^x for two x <= 127 on the multiply-add units, where ex2 is what everything waits for: x = n + f with n the nearest integer,
// 2^f by a polynomial of degree 5 fitted to the smallest relative error on [-1/2, 1/2] (2.2e-7 with its fp32 roundings, what
// ex2.approx has), 2^n from its bits.  Below -127 the result is 0; NaN stays NaN.
__device__ __forceinline__ unsigned long long f2_exp2(unsigned long long x) {
  float2 v = f2_unpack(x);
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(v.x) : "f"(-127.f));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(v.y) : "f"(-127.f));
  x = f2_pack(v.x, v.y);
  constexpr float kShift = 12582912.f + 127.f;  // 1.5 * 2^23: the sum's last bits are n + 127
  const unsigned long long shifted = f2_add(x, f2_same(kShift));
  const unsigned long long f = f2_add(x, f2_mul(f2_add(shifted, f2_same(-kShift)), f2_same(-1.f)));
  unsigned long long r = f2_fma(f, f2_same(0x1.5c08e6p-10f), f2_same(0x1.3d0c52p-7f));
  r = f2_fma(r, f, f2_same(0x1.c6b6e4p-5f));
  r = f2_fma(r, f, f2_same(0x1.ebf918p-3f));
  r = f2_fma(r, f, f2_same(0x1.62e428p-1f));
  r = f2_fma(r, f, f2_same(0x1.000002p+0f));
  const float2 n = f2_unpack(shifted);
  return f2_mul(r, f2_pack(__int_as_float(__float_as_int(n.x) << 23), __int_as_float(__float_as_int(n.y) << 23)));
}

template <typename T, int kDim>
__global__ void __launch_bounds__(PrefixTc<kDim>::kThreads, 1)
prefix_sdpa_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const PrefixTcArgs p) {
  using G = PrefixTc<kDim>;
  extern __shared__ __align__(PrefixTc<128>::kAlign) uint8_t smem_raw[];
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
  const uint32_t full_bar = smem_base + G::kBarrierOffset;  // [steps] a step's tiles landed       (TMA -> MMA)
  const uint32_t empty_bar = full_bar + 8 * G::kMostSteps;  // [steps] the MMAs that read it done  (MMA -> TMA)
  const uint32_t q_bar = empty_bar + 8 * G::kMostSteps;     //     Q in shared memory              (softmax -> MMA)
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
  // K runs `lead` tiles ahead of V: steps [0, lead) bring a K tile each, step lead + t brings V tile t and K tile t + lead
  const int lead = min(p.both_rows ? 1 : 2, n), steps = G::steps(p.both_rows != 0);
  const uint32_t ring = smem_base + G::q_bytes(p.both_rows != 0);  // Q lies before it

  if (threadIdx.x == 0) {
    for (int s = 0; s < G::kMostSteps; ++s) {
      mbar_init(full_bar + 8 * s, 1);
      mbar_init(empty_bar + 8 * s, 1);
    }
    mbar_init(q_bar, 2 * G::kGroupWarps);
    for (int g = 0; g < 2; ++g) {
      mbar_init(s_bar + 8 * g, 1);
      mbar_init(p_bar + 8 * g, G::kGroupWarps);
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

  if (warp == 0) {
    // ---------------------------------------------------------------- pages and TMA: a lane per page of the tile
    const int boxes = G::kKeys / p.box_keys;
    auto key_of = [&](int tile) { return (first_tile + tile) * G::kKeys + lane * p.box_keys; };  // first key of this lane's box
    auto mine = [&](int tile) { return lane < boxes && tile < n && key_of(tile) < p.a.prefix_len; };
    auto page_of = [&](int tile) { return mine(tile) ? __ldg(p.a.prefix_pages + key_of(tile) / p.a.page_size) : -1; };
    auto bytes_of = [&](int tile) { return __popc(__ballot_sync(0xffffffffu, mine(tile))) * p.box_keys * 128 * G::kAtoms; };
    auto load = [&](const CUtensorMap* map, int tile, int head, int page, uint32_t to, uint32_t bar) {
      if (mine(tile)) {
#pragma unroll
        for (int atom = 0; atom < G::kAtoms; ++atom)  // a page outside the cache reads as zeros
          tma_load_4d(to + atom * G::kAtomBytes + lane * p.box_keys * 128, map, bar, atom * 64, key_of(tile) % p.a.page_size, head, page);
      }
    };
    int ahead[2] = {page_of(0), page_of(1)};  // of the next K tiles, looked up before they are needed
    int before[2] = {-1, -1};                 // of the last two, whose V tiles follow
    int slot = 0;
    uint32_t phase = 1;
    for (int step = 0; step < lead + n; ++step) {
      const int k_tile = step, v_tile = step - lead;  // either may not exist
      const int k_page = ahead[0], v_page = lead == 1 ? before[0] : before[1];
      ahead[0] = ahead[1], ahead[1] = page_of(step + 2);
      before[1] = before[0], before[0] = k_page;
      if (!mbar_wait(empty_bar + 8 * slot, phase, abort_flag)) {
        if (lane == 0) give_up(kStatusProducerWait);
        break;
      }
      const uint32_t bar = full_bar + 8 * slot, to = ring + slot * 2 * G::kTileBytes;
      const int bytes = (k_tile < n ? bytes_of(k_tile) : 0) + (v_tile >= 0 ? bytes_of(v_tile) : 0);
      const uint32_t gone = __ballot_sync(0xffffffffu, mine(k_tile) && (k_page < 0 || k_page >= p.a.pages));
      if (lane == 0) {
        if (k_tile < n) absent[k_tile % G::kMaskSlots] = gone;
        mbar_arrive_expect_tx(bar, bytes);
      }
      __syncwarp();
      if (v_tile >= 0) load(&map_v, v_tile, kv * p.v_head_step, v_page, to, bar);
      if (k_tile < n) load(&map_k, k_tile, kv * p.k_head_step, k_page, to + G::kTileBytes, bar);
      if (++slot == steps) slot = 0, phase ^= 1u;
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMAs
    const uint32_t type = std::is_same<T, __nv_bfloat16>::value ? kUmmaBF16 : kUmmaF16;
    const uint32_t idesc_s = umma_instr_desc(kUmmaAccF32, type, type, 128, 128);
    const uint32_t idesc_o = umma_instr_desc(kUmmaAccF32, type, type, 128, kDim, true);  // B = V, N-major
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
    auto scores = [&](int g, uint32_t k) {  // S_g = Q_g . K^T
      const uint32_t q = smem_base + (p.both_rows ? g * G::kTileBytes : 0);
      if (leader) {
#pragma unroll
        for (int ks = 0; ks < kDim / 16; ++ks)  // (what lies past head_dim is zero in both operands)
          umma_f16(tmem_base + g * 256, umma_smem_desc_sw128(q + (ks >> 2) * G::kAtomBytes) + 2 * (ks & 3),
                   umma_smem_desc_sw128(k + (ks >> 2) * G::kAtomBytes) + 2 * (ks & 3), idesc_s, ks > 0 ? 1u : 0u);
      }
    };
    wait(q_bar, 0);
    for (int step = 0; ok && step < lead + n; ++step) {
      wait(full_bar + 8 * slot, phase);
      if (!ok) break;
      const int tile = step - lead;  // whose probabilities are multiplied with V
      const uint32_t v = ring + slot * 2 * G::kTileBytes, k = v + G::kTileBytes;
      const int last = p.a.prefix_len - (first_tile + tile) * G::kKeys;
      if (tile >= 0 && last < G::kKeys) {
        // the prefix ends inside the tile: whatever lies behind it, NaN included, must not meet the zero probabilities there
        for (int i = lane; i < (G::kKeys - last) * 8 * G::kAtoms; i += 32) {
          const int row = last + i / (8 * G::kAtoms), piece = i % (8 * G::kAtoms);
          const uint32_t dst = v + (piece >> 3) * G::kAtomBytes + row * 128 + ((piece & 7) << 4);
          asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(dst), "r"(0) : "memory");
        }
        fence_proxy_async_smem();
        __syncwarp();
      }
      const int turn = p.both_rows ? tile : tile >> 1;  // how many tiles a group had before
      for (int g = p.both_rows ? 0 : step & 1; g < (p.both_rows ? 2 : (step & 1) + 1); ++g) {
        // in turn, one row block: K tile `step` and V tile `step - 2` are of the same group (a single tile has lead 1)
        const int who = p.both_rows || lead == 2 ? g : 0;
        if (tile >= 0) {
          wait(p_bar + 8 * who, static_cast<uint32_t>(turn) & 1u);
          if (!ok) break;
          tcgen05_fence_after_sync();
          if (leader) {
#pragma unroll
            for (int ks = 0; ks < G::kKeys / 16; ++ks)  // 16 keys: 8 columns of P (64 keys' lie over those keys' scores), 16 rows of V
              umma_f16_from_tmem(tmem_base + who * 256 + 128, tmem_base + who * 256 + (ks >> 2) * 64 + (ks & 3) * 8, umma_smem_desc_sw128_mn(v + ks * 16 * 128, G::kAtomBytes, 1024), idesc_o,
                                 turn > 0 || ks > 0 ? 1u : 0u);
          }
        } else {
          tcgen05_fence_after_sync();
        }
        if (step < n) scores(who, k);  // (over P: the tensor core works in order)
        if (leader) umma_commit(s_bar + 8 * who);
      }
      if (!ok) break;
      if (leader) umma_commit(empty_bar + 8 * slot);
      __syncwarp();
      if (++slot == steps) slot = 0, phase ^= 1u;
    }
  } else if (warp >= G::kFirstSoftmaxWarp) {
    // ---------------------------------------------------------------- softmax: two threads a row
    const int group_warp = (warp - G::kFirstSoftmaxWarp) % G::kGroupWarps;
    const int g = (warp - G::kFirstSoftmaxWarp) / G::kGroupWarps, quarter = warp & 3, half = group_warp >> 2;
    {
      // Q: rows of 16-byte pieces under the 128-byte swizzle; rows past the last and dims past head_dim are zero
      // (all of a thread's rows in flight together: one trip to memory)
      constexpr int kLoaders = 64 * G::kGroupWarps;
      constexpr int kPieces = kDim / 8, kRowStep = kLoaders / kPieces, kMine = 2 * G::kRows / kRowStep;
      const int thread = static_cast<int>(threadIdx.x) - 32 * G::kFirstSoftmaxWarp;
      const int piece = thread % kPieces, first = thread / kPieces;
      const int q_rows = min(p.both_rows ? 2 * G::kRows : G::kRows, p.rows - row0);
      const bool in_head = piece * 8 < p.a.head_dim;
      int t = (row0 + first) / p.a.group, in_group = row0 + first - t * p.a.group;
      const int t_step = kRowStep / p.a.group, in_group_step = kRowStep - t_step * p.a.group;
      const T* base = static_cast<const T*>(p.a.q) + static_cast<long long>(kv) * p.a.group * p.a.q_sh + piece * 8;
      uint4 x[kMine];
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        x[i] = make_uint4(0, 0, 0, 0);
        if (first + i * kRowStep < q_rows && in_head) x[i] = __ldg(reinterpret_cast<const uint4*>(base + t * p.a.q_st + in_group * p.a.q_sh));
        t += t_step, in_group += in_group_step;
        if (in_group >= p.a.group) ++t, in_group -= p.a.group;
      }
      const uint32_t to = smem_base + (piece >> 3) * G::kAtomBytes;
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        const int row = first + i * kRowStep;
        const uint32_t dst = to + (row >> 7) * G::kTileBytes + (row & 127) * 128 + (((piece & 7) ^ (row & 7)) << 4);
        if (i < kMine / 2 || p.both_rows)
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(x[i].x), "r"(x[i].y), "r"(x[i].z), "r"(x[i].w) : "memory");
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_bar);
    }
    const int row_local = quarter * 32 + lane;
    const int row = row0 + (p.both_rows ? g * G::kRows : 0) + row_local;
    const uint32_t my_tmem = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + g * 256;
    const uint32_t my_scores = my_tmem + half * 64, my_o = my_tmem + 128 + half * (kDim / 2);
    volatile float* exchange = reinterpret_cast<volatile float*>(smem_gen + G::kExchangeOffset) + g * 256 + row_local;  // [half][row]
    auto meet = [&] { asm volatile("bar.sync %0, 64;" ::"r"(1 + g * 4 + quarter) : "memory"); };         // the two warps of a quarter's rows
    const float signed_scale = p.a.scale * 1.4426950408889634f;  // scores in units of log2(e)
    const float scale = signed_scale == 0.f ? 1.f : fabsf(signed_scale);
    const unsigned long long scale2 = f2_same(scale);
    const int box_shift = 31 - __clz(p.box_keys);
    float m = -INFINITY, l = 0.f;  // m is never NaN: a NaN score shows in l
    bool ok = true, keyed = false;  // keyed: a page of the group's tiles is in the cache
    int turn = 0;
    auto wait_scores = [&] {
      if (ok && !__all_sync(0xffffffffu, mbar_wait(s_bar + 8 * g, static_cast<uint32_t>(turn) & 1u, abort_flag))) {
        if (lane == 0) give_up(kStatusEpilogueWait);
        ok = false;
      }
      tcgen05_fence_after_sync();
    };
    // (a warp whose wait ran out keeps walking the tiles without touching anything: its partner meets it at every barrier)
    for (int tile = p.both_rows ? 0 : g; tile < n; tile += p.both_rows ? 1 : 2, ++turn) {
      wait_scores();
      // Two passes over the scores where they lie, 32 columns at a time: the maximum, then the probabilities, which go over
      // columns already read.  (Held in registers between the two they spilled.)
      const int last = p.a.prefix_len - (first_tile + tile) * G::kKeys - half * 64;
      const uint32_t gone = absent[tile % G::kMaskSlots];
      keyed = keyed || __popc(gone) * p.box_keys < min(G::kKeys, last + half * 64);
      auto load_scores = [&](int col, float (&t)[32]) {
        tmem_load_32x32(my_scores + col, reinterpret_cast<uint32_t(&)[32]>(t));
        tmem_load_wait();
        if (signed_scale <= 0.f) {  // (so that the factor below is positive: the maximum, and a masked -inf, keep their meaning)
          const float sign = signed_scale < 0.f ? -1.f : 0.f;
#pragma unroll
          for (int j = 0; j < 32; ++j) t[j] *= sign;
        }
        if (last < 64 || gone != 0) {
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (col + j >= last || (gone >> ((half * 64 + col + j) >> box_shift) & 1u) != 0) t[j] = -INFINITY;
        }
      };
      float highest = -INFINITY;
      if (ok) {
#pragma unroll 1
        for (int col = 0; col < 64; col += 32) {
          float t[32];
          load_scores(col, t);
          float top[2] = {highest, t[0]};
#pragma unroll
          for (int j = 0; j < 32; j += 2) asm("max.f32 %0, %0, %1, %2;" : "+f"(top[(j >> 1) & 1]) : "f"(t[j]), "f"(t[j + 1]));
          highest = fmaxf(top[0], top[1]);
        }
      }
      // The two halves agree on the row's maximum.  (In 32 bits: rounded to 16, one of thousands is off by tens, and p past what fp16 holds.)
      exchange[half * 128] = highest;
      meet();
      const float tile_max = fmaxf(highest, exchange[(half ^ 1) * 128]) * scale;
      const bool moves = turn == 0 || tile_max > m + 8.f;
      if (turn == 0) {
        m = tile_max;
      } else if (__any_sync(0xffffffffu, moves)) {
        const float m_new = moves ? tile_max : m;
        const float keep = moves ? exp2_approx(m - m_new) : 1.f;
        l *= keep;
        m = m_new;
        if (ok) {
          uint32_t o[32];
#pragma unroll 1
          for (int col = 0; col < kDim / 2; col += 32) {
            tmem_load_32x32(my_o + col, o);
            tmem_load_wait();
#pragma unroll
            for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * keep);
            tmem_store_32x32(my_o + col, o);
          }
        }
      }
      if (ok) {
        const unsigned long long minus_m2 = f2_same(m == -INFINITY ? 0.f : -m);  // nothing kept so far: every p is 0
        unsigned long long sums[2] = {0ull, 0ull};
#pragma unroll 1
        for (int col = 0; col < 64; col += 32) {
          float t[32];
          load_scores(col, t);
          uint32_t packed[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            unsigned long long e = f2_fma(f2_pack(t[2 * j], t[2 * j + 1]), scale2, minus_m2);
            if (j * G::kPolynomialPairs % 16 < G::kPolynomialPairs) {
              e = f2_exp2(e);
            } else {
              const float2 x = f2_unpack(e);
              e = f2_pack(exp2_approx(x.x), exp2_approx(x.y));
            }
            sums[j & 1] = f2_add(sums[j & 1], e);
            const float2 probability = f2_unpack(e);
            packed[j] = prefix_pack<T>(probability.x, probability.y);
          }
          tmem_store_32x16(my_scores + col / 2, packed);
        }
        const float2 sum = f2_unpack(f2_add(sums[0], sums[1]));
        l += sum.x + sum.y;
        tmem_store_wait();
        tcgen05_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_bar + 8 * g);
      }
      // (the exchange is written again only after the next scores, which wait for both warps' probabilities)
    }
    // ---- this group's rows of the chunk leave: O, m, l
    const int record = p.both_rows ? chunk : 2 * chunk + g;
    const size_t at = (static_cast<size_t>(record) * p.a.kv_heads + kv) * p.rows + row;
    if (turn > 0) wait_scores();  // the last product is in O
    if (ok && turn > 0) {
      // through shared memory - Q's place: every product of scores is done, the other group's last one with V may not be - so that
      // whole 64-byte pieces of a row leave together (a thread storing its own row, 16 bytes at a time, took 6 us)
      const uint32_t stage = smem_base + (warp - G::kFirstSoftmaxWarp) * G::kStageBytes;
      const int first_row = row - lane;
#pragma unroll 1
      for (int col = 0; col < kDim / 2; col += 16) {
        uint32_t o[16];
        tmem_load_32x16(my_o + col, o);
        tmem_load_wait();
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 4; ++j)
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(stage + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4)), "r"(o[4 * j]), "r"(o[4 * j + 1]),
                       "r"(o[4 * j + 2]), "r"(o[4 * j + 3]) : "memory");
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = i * 8 + (lane >> 2), piece = lane & 3;
          float4 x;
          asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w) : "r"(stage + r * 64 + ((piece ^ ((r >> 1) & 3)) << 4)) : "memory");
          if (first_row + r < p.rows) __stcg(reinterpret_cast<float4*>(p.partial_o + (at - lane + r) * kDim + half * (kDim / 2) + col) + piece, x);
        }
      }
    }
    // the row's sum: the second half's goes to the first through the place of its own maxima, which the first has read: its
    // probabilities of the last tile have arrived
    if (half == 1) exchange[128] = l;
    meet();
    if (half == 0) l += exchange[128];
    if (m == -INFINITY && keyed) l += 1.f;  // scores of -inf alone are keys all the same (or NaN, which l keeps)
    if (half == 0 && row < p.rows) __stcg(p.partial_ml + at, make_float2(turn > 0 && ok ? m : -INFINITY, turn > 0 && ok ? l : 0.f));
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
