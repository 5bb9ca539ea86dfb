// Block-scaled e4m3 product at tensor-core rate: CTA pairs on 256 x 256 tiles of C.
//
//     C[m,n] = sum_b (sa[m,b] sb[n/128,b]) sum_{k in b} A[m,k] B[n,k]
//
// A block's scales apply to its sum over 128 k, so every 128-k step of the main loop is an accumulation of its own, which
// eight warps read back from tensor memory and add, scaled, to totals in registers while the tensor cores work on the next.
// Four MMAs of 256 columns take 512 cycles; a step of the totals' loop takes some 750: the wait for its sums, 340 for reading
// them back while the MMAs of the other accumulator work on the same tensor memory, 256 of multiply-adds.  That loop is what
// bounds the kernel: without its multiply-adds it reached 2.7 PFLOP/s, with them 4096 x 14336 x 4096 takes 209 us, 2.3
// PFLOP/s.  (Tensor memory holds two accumulators of 256 columns.  Four of 128 hide the round trip better, but an MMA of 128
// columns takes 80 cycles, not 64, and measured 12 % slower; sixteen warps of totals, wider reads, reads across steps and
// scales fetched a step ahead measured slower or the same.)  512 x 4096 x 14336, cut into slices of K: 33 us.  Roles, per CTA:
//   warp 0      TMA: its 128 rows of A and its 128 of the tile's 256 rows of B per step, a ring of kStages
//   warp 1      (leader CTA) issues tcgen05.mma.cta_group::2, M = 256, N = 256, four of 32 k per accumulator
//   warps 2-3   fetch the scales into a ring in shared memory, up to 32 steps ahead (fetched by the totals' own threads, 32
//               rows a warp and each in a line of its own, they took as long as the product itself)
//   warps 4-11  totals - a thread owns one row and 128 columns of C, all of one weight block: one factor sa * sb per step
//               and one fused multiply-add per element, two per instruction - then the store of the tile by TMA
// Persistent: pairs walk the tiles `worker, worker + workers, ...`.  With fewer tiles than pairs, K is cut into 2 or 4 slices:
// the pairs of a tile's slices form a cluster, and each of its CTAs sums a share of the rows through the others' shared memory.
#pragma once

#include "f8_stream.cuh"

namespace vb200 {

struct F8Tiled {
  static constexpr int kTile = 256;
  static constexpr int kOperandBytes = 128 * 128;  // 128 rows x 128 bytes of A, and as much of B
  static constexpr int kStageBytes = 2 * kOperandBytes;
  static constexpr int kStages = 5;
  static constexpr int kAccumulators = 2;
  static constexpr int kTotalWarps = 8;
  static constexpr int kFirstTotalWarp = 4;  // register shares are per warpgroup
  static constexpr int kThreads = 32 * (kFirstTotalWarp + kTotalWarps);
  // 384 threads x 168 registers at launch; the totals take what the other warpgroup gives up: (56 + 2 x 224) x 128 = 168 x 384
  static constexpr int kFewRegisters = 56, kManyRegisters = 224;
  static constexpr int kOutRows = 16;                        // rows of C a warp stages at a time, 128 bytes of each
  // ... and how many such pieces may be on their way (one, with the room in a sixth stage, took 2 % longer)
  static constexpr int kOutBuffers = 3;
  static constexpr int kOutOffset = kStages * kStageBytes;
  static constexpr int kOutBytes = kTotalWarps * kOutBuffers * kOutRows * 128;
  static constexpr int kScaleSteps = 4, kScaleSlots = 8;     // a slot holds four steps' scales of the tile's 128 rows and two weight blocks
  static constexpr int kScaleOffset = kOutOffset + kOutBytes;
  static constexpr int kSlotFloats = kScaleSteps * (128 + 2);
  static constexpr int kBarrierOffset = kScaleOffset + kScaleSlots * kSlotFloats * 4;
  static constexpr int kBarriers = 2 * kStages + kAccumulators + 2 * kScaleSlots;
  static constexpr int kSmemBytes = kBarrierOffset + kBarriers * 8 + 8 + 1024;
  static constexpr int kTmemColumns = 512;
  static constexpr int kMaxSlices = 4;  // pairs of one cluster, 8 CTAs
  static constexpr long long kGroupBytes = 32ll << 20;  // raster: row tiles holding this much of A share each sweep over N
};
static_assert((F8Tiled::kFewRegisters + 2 * F8Tiled::kManyRegisters) * 128 <= 168 * F8Tiled::kThreads, "register split");
static_assert(128 * 1024 <= F8Tiled::kStages * F8Tiled::kStageBytes, "the totals of a slice are left over the ring");
static_assert(F8Tiled::kSmemBytes <= 227 * 1024, "shared memory budget");
static_assert(F8Tiled::kBarrierOffset % 8 == 0, "barriers are 8-byte words");

// acc += v * s on two floats at once
__device__ __forceinline__ void f8_fma2(float2& acc, uint32_t v0, uint32_t v1, float s) {
  unsigned long long a, v, f;
  asm("mov.b64 %0, {%1, %2};" : "=l"(a) : "f"(acc.x), "f"(acc.y));
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "r"(v0), "r"(v1));
  asm("mov.b64 %0, {%1, %1};" : "=l"(f) : "f"(s));
  asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(a) : "l"(v), "l"(f));
  asm("mov.b64 {%0, %1}, %2;" : "=f"(acc.x), "=f"(acc.y) : "l"(a));
}

template <typename OutT>
__global__ void __launch_bounds__(F8Tiled::kThreads, 1)
f8_tiled_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_c,
                const F8StreamArgs p, int tma_store, int raster_group, int slice_bits) {
  using G = F8Tiled;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
  const uint32_t full_bar = smem_base + G::kBarrierOffset;        // [stages] both CTAs' tiles landed          (TMA -> MMA; the leader's)
  const uint32_t done_bar = full_bar + 8 * G::kStages;            // [stages] a step is multiplied: its sums are ready, its stage is free
                                                                  //           (MMA -> totals and TMA of both)
  const uint32_t read_bar = done_bar + 8 * G::kStages;            // [accumulators] read back (totals of both -> MMA; the leader's)
  const uint32_t scale_full_bar = read_bar + 8 * G::kAccumulators;  // [slots]
  const uint32_t scale_empty_bar = scale_full_bar + 8 * G::kScaleSlots;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem_gen + G::kBarrierOffset + 8 * G::kBarriers);
  volatile uint32_t* abort_flag = tmem_slot + 1;
  float* scale_ring = reinterpret_cast<float*>(smem_gen + G::kScaleOffset);  // [slot][step][128 rows of A, 2 blocks of B]

  // (through a shuffle, so that the compiler knows it to be the same for the whole warp: the roles' loops then run on uniform registers)
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const uint32_t cluster_rank = cluster_cta_rank(), rank = cluster_rank & 1u, leader_rank = cluster_rank & ~1u;
  const uint16_t both = static_cast<uint16_t>(3u << leader_rank);
  const int slice = static_cast<int>(cluster_rank >> 1);
  const int worker = static_cast<int>(blockIdx.x >> (1 + slice_bits)), workers = static_cast<int>(gridDim.x >> (1 + slice_bits));
  const int tiles_m = (p.m + G::kTile - 1) / G::kTile, tiles_n = (p.n + G::kTile - 1) / G::kTile;
  const int num_tiles = tiles_m * tiles_n;
  const int all_kb = (p.k + 127) / 128;
  const int kb_begin = static_cast<int>(static_cast<long long>(all_kb) * slice >> slice_bits);
  const int num_kb = static_cast<int>(static_cast<long long>(all_kb) * (slice + 1) >> slice_bits) - kb_begin;

  if (threadIdx.x == 0) {
    for (int s = 0; s < G::kStages; ++s) {
      mbar_init(full_bar + 8 * s, 1);
      mbar_init(done_bar + 8 * s, 1);
    }
    for (int a = 0; a < G::kAccumulators; ++a) mbar_init(read_bar + 8 * a, 2 * G::kTotalWarps);
    for (int s = 0; s < G::kScaleSlots; ++s) {
      mbar_init(scale_full_bar + 8 * s, 2);
      mbar_init(scale_empty_bar + 8 * s, G::kTotalWarps);
    }
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_descriptor(&map_a);
    tma_prefetch_descriptor(&map_b);
    if (tma_store) tma_prefetch_descriptor(&map_c);
  }
  if (warp == 1) {
    tmem_alloc_pair(smem_u32(tmem_slot), G::kTmemColumns);
    tmem_relinquish_pair();
  }
  tcgen05_fence_before_sync();
  __syncthreads();
  cluster_sync_all();  // the peer's barriers exist before anything signals them
  tcgen05_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  grid_launch_dependents();
  grid_dependency_wait();

  auto give_up = [&](uint32_t code) {
    report_status(p.status, code);
    *abort_flag = 1;
  };

  if (warp < G::kFirstTotalWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(G::kFewRegisters));
    if (warp == 0 && lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = worker; ok && tile < num_tiles; tile += workers) {
        int tm, tn;
        tile_coords(tile, tiles_m, tiles_n, raster_group, tm, tn);
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mbar_wait(done_bar + 8 * stage, phase ^ 1u, abort_flag)) {
            give_up(kStatusProducerWait);
            ok = false;
            break;
          }
          const uint32_t a_dst = smem_base + stage * G::kStageBytes;
          const uint32_t leader_full = map_to_cta(full_bar + 8 * stage, leader_rank);
          if (rank == 0) mbar_arrive_expect_tx(full_bar + 8 * stage, 2 * G::kStageBytes);
          tma_load_2d_pair(a_dst, &map_a, leader_full, (kb_begin + kb) * 128, tm * G::kTile + static_cast<int>(rank) * 128);
          tma_load_2d_pair(a_dst + G::kOperandBytes, &map_b, leader_full, (kb_begin + kb) * 128, tn * G::kTile + static_cast<int>(rank) * 128);
          if (++stage == G::kStages) stage = 0, phase ^= 1u;
        }
      }
    } else if (warp == 1 && rank == 0) {
      // the whole warp walks the loop, one elected lane issues: what the instructions take stays in uniform registers
      constexpr uint32_t idesc = umma_instr_desc(kUmmaAccF32, kUmmaE4M3, kUmmaE4M3, 256, 256);
      const bool leader = elect_one();
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      for (int tile = worker; ok && tile < num_tiles; tile += workers) {
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mbar_wait(full_bar + 8 * stage, phase, abort_flag)) {
            if (leader) give_up(kStatusMmaWaitFull);
            ok = false;
            break;
          }
          if (!mbar_wait(read_bar + 8 * acc, acc_phase ^ 1u, abort_flag)) {
            if (leader) give_up(kStatusMmaWaitTmem);
            ok = false;
            break;
          }
          tcgen05_fence_after_sync();
          const uint64_t a_desc = umma_smem_desc_sw128(smem_base + stage * G::kStageBytes);
          const uint64_t b_desc = umma_smem_desc_sw128(smem_base + stage * G::kStageBytes + G::kOperandBytes);
          if (leader) {
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) umma_f8_pair(tmem_base + acc * G::kTile, a_desc + 2 * kk, b_desc + 2 * kk, idesc, kk != 0 ? 1u : 0u);
            umma_commit_pair_of(done_bar + 8 * stage, both);
          }
          __syncwarp();
          if (++stage == G::kStages) stage = 0, phase ^= 1u;
          acc ^= 1;
          if (acc == 0) acc_phase ^= 1u;
        }
      }
    } else if (warp >= 2) {
      const int row_in_tile = (warp - 2) * 64 + 2 * lane;  // two rows a thread
      int slot = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = worker; ok && tile < num_tiles; tile += workers) {
        int tm, tn;
        tile_coords(tile, tiles_m, tiles_n, raster_group, tm, tn);
        const int row = tm * G::kTile + static_cast<int>(rank) * 128 + row_in_tile;
        const int block = 2 * tn + (warp - 2);  // weight block fetched by lanes 0..3 of the warp, one step each
        const float* a_scale = p.a_scale + static_cast<long long>(row) * p.as_sm + kb_begin * p.as_sk;
        const float* b_scale = p.b_scale + static_cast<long long>(block) * p.bs_sn + kb_begin * p.bs_sk;
        for (int kb = 0; kb < num_kb; kb += G::kScaleSteps) {
          float a[G::kScaleSteps][2], b = 0.f;
#pragma unroll
          for (int g = 0; g < G::kScaleSteps; ++g) {  // (what lies past the matrix is never stored: its factor is 0)
            a[g][0] = kb + g < num_kb && row < p.m ? __ldg(a_scale + (kb + g) * p.as_sk) : 0.f;
            a[g][1] = kb + g < num_kb && row + 1 < p.m ? __ldg(a_scale + p.as_sm + (kb + g) * p.as_sk) : 0.f;
          }
          if (lane < G::kScaleSteps && kb + lane < num_kb && block * 128 < p.n) b = __ldg(b_scale + (kb + lane) * p.bs_sk);
          if (!__all_sync(0xffffffffu, mbar_wait(scale_empty_bar + 8 * slot, phase ^ 1u, abort_flag))) {
            if (lane == 0) give_up(kStatusProducerWait);
            ok = false;
            break;
          }
          float* to = scale_ring + slot * G::kSlotFloats;
#pragma unroll
          for (int g = 0; g < G::kScaleSteps; ++g) *reinterpret_cast<float2*>(to + g * 130 + row_in_tile) = make_float2(a[g][0], a[g][1]);
          if (lane < G::kScaleSteps) to[lane * 130 + 128 + (warp - 2)] = b;
          __syncwarp();
          if (lane == 0) mbar_arrive(scale_full_bar + 8 * slot);
          if (++slot == G::kScaleSlots) slot = 0, phase ^= 1u;
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(G::kManyRegisters));
    const int quarter = warp & 3, half = (warp - G::kFirstTotalWarp) >> 2;
    const uint32_t out_ring = smem_base + G::kOutOffset + (warp - G::kFirstTotalWarp) * (G::kOutBuffers * G::kOutRows * 128);
    int out_at = 0;
    const uint32_t my_tmem = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + half * 128;
    int stage = 0, acc = 0, slot = 0;
    uint32_t phase = 0, slot_phase = 0;
    bool ok = true;
    for (int tile = worker; ok && tile < num_tiles; tile += workers) {
      int tm, tn;
      tile_coords(tile, tiles_m, tiles_n, raster_group, tm, tn);
      const int row0 = tm * G::kTile + static_cast<int>(rank) * 128 + quarter * 32;
      const int col0 = tn * G::kTile + half * 128;
      bool early = false;  // the next step's sums are ready: asked under this step's last multiplications (asked when needed, it took some 180 cycles)
      float2 total[64];
#pragma unroll
      for (int j = 0; j < 64; ++j) total[j] = make_float2(0.f, 0.f);
      float factor[G::kScaleSteps] = {0.f, 0.f, 0.f, 0.f};
      for (int kb = 0; kb < num_kb; ++kb) {
        if ((kb & (G::kScaleSteps - 1)) == 0) {
          if (!__all_sync(0xffffffffu, mbar_wait(scale_full_bar + 8 * slot, slot_phase, abort_flag))) {
            if (lane == 0) give_up(kStatusEpilogueWait);
            ok = false;
            break;
          }
          const float* from = scale_ring + slot * G::kSlotFloats;
#pragma unroll
          for (int g = 0; g < G::kScaleSteps; ++g) factor[g] = from[g * 130 + quarter * 32 + lane] * from[g * 130 + 128 + half];
          __syncwarp();
          if (lane == 0) mbar_arrive(scale_empty_bar + 8 * slot);
          if (++slot == G::kScaleSlots) slot = 0, slot_phase ^= 1u;
        }
        const float s = factor[0];
#pragma unroll
        for (int g = 0; g + 1 < G::kScaleSteps; ++g) factor[g] = factor[g + 1];
        if (!__all_sync(0xffffffffu, early) && !__all_sync(0xffffffffu, mbar_wait(done_bar + 8 * stage, phase, abort_flag))) {
          if (lane == 0) give_up(kStatusEpilogueWait);
          ok = false;
          break;
        }
        tcgen05_fence_after_sync();
        const uint32_t taddr = my_tmem + acc * G::kTile;
        uint32_t v[2][16];
        tmem_load_32x16(taddr, v[0]);
#pragma unroll
        for (int chunk = 0; chunk < 8; ++chunk) {
          tmem_load_wait();
          if (chunk == 7) early = mbar_test_wait(done_bar + 8 * (stage + 1 == G::kStages ? 0 : stage + 1), stage + 1 == G::kStages ? phase ^ 1u : phase);
          if (chunk + 1 < 8) {
            tmem_load_32x16(taddr + 16 * (chunk + 1), v[(chunk + 1) & 1]);
          } else {
            tcgen05_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster_relaxed(map_to_cta(read_bar + 8 * acc, leader_rank));
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) f8_fma2(total[8 * chunk + j], v[chunk & 1][2 * j], v[chunk & 1][2 * j + 1], s);
        }
        if (++stage == G::kStages) stage = 0, phase ^= 1u;
        acc ^= 1;
      }
      if (!ok) break;
      if (slice_bits > 0) {
        // every MMA of this CTA is done and has read what TMA brought: the totals go over the ring as rows of 256 floats, their
        // 16-byte pieces swizzled by the row so that neither these stores nor the reads below meet in a bank
        const int row = quarter * 32 + lane;
#pragma unroll
        for (int piece = 0; piece < 32; ++piece) {
          const uint32_t dst = smem_base + row * 1024 + (((half * 32 + piece) ^ (row & 7)) << 4);
          const float2 x = total[2 * piece], y = total[2 * piece + 1];
          asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "f"(x.x), "f"(x.y), "f"(y.x), "f"(y.y) : "memory");
        }
        break;  // (one tile per cluster)
      }
      // ---- the tile leaves: 128 bytes of sixteen rows at a time
      constexpr int kSlabCols = 128 / static_cast<int>(sizeof(OutT));
#pragma unroll
      for (int slab = 0; slab < 128 / kSlabCols; ++slab) {
        if (col0 + slab * kSlabCols >= p.n || row0 >= p.m) continue;  // (uniform over the warp)
        // (TMA clips rows of C to whole 16 bytes, not to elements: a row that ends in between ends by the other way)
        const bool by_tma = tma_store && (p.n % (16 / static_cast<int>(sizeof(OutT))) == 0 || col0 + (slab + 1) * kSlabCols <= p.n);
        uint32_t w[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          if constexpr (sizeof(OutT) == 2) {
            const float2 f = total[slab * 32 + e];
            w[e] = pack_out16x2<OutT>(f.x, f.y);
          } else {
            const float2 f = total[slab * 16 + e / 2];
            w[e] = __float_as_uint(e & 1 ? f.y : f.x);
          }
        }
#pragma unroll 1
        for (int part = 0; part < 32 / G::kOutRows; ++part) {
          if (tma_store && lane == 0) tma_store_wait_read<G::kOutBuffers - 1>();  // what was in this buffer has left it
          __syncwarp();
          const uint32_t out_buf = out_ring + out_at * (G::kOutRows * 128);
          if (++out_at == G::kOutBuffers) out_at = 0;
          if (lane / G::kOutRows == part) {
#pragma unroll
            for (int piece = 0; piece < 8; ++piece) {
              const uint32_t dst = out_buf + (lane % G::kOutRows) * 128 + ((piece ^ (lane & 7)) << 4);
              asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(w[4 * piece]), "r"(w[4 * piece + 1]), "r"(w[4 * piece + 2]),
                           "r"(w[4 * piece + 3]) : "memory");
            }
          }
          if (by_tma) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              // rows and columns past C are clipped (a store that starts past it would be empty)
              if (row0 + part * G::kOutRows < p.m) tma_store_2d(&map_c, out_buf, col0 + slab * kSlabCols, row0 + part * G::kOutRows);
              tma_store_commit();
            }
          } else {
            // Rows of C that TMA cannot address - off 16-byte boundaries, or strided - leave element by element, neighbouring lanes with
            // neighbouring columns.  (A thread storing the row it owns made 4096 x 14335 x 4096 three times as slow as 14336 columns.)
            __syncwarp();
            if (tma_store && lane == 0) tma_store_commit();  // (an empty one: the buffers are counted by their groups)
            constexpr int kPer16 = 16 / static_cast<int>(sizeof(OutT));
            const OutT* staged = reinterpret_cast<const OutT*>(smem_gen + (out_buf - smem_base));
            const int first = row0 + part * G::kOutRows, rows = min(G::kOutRows, p.m - first);
            const int col = col0 + slab * kSlabCols + lane;
            OutT* c = static_cast<OutT*>(p.c) + first * p.c_sm + col * p.c_sn;
#pragma unroll 1
            for (int r0 = 0; r0 < rows; r0 += 4, c += 4 * p.c_sm) {
              OutT x[4][kSlabCols / 32];  // (all on their way before the first is stored)
#pragma unroll
              for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int j = 0; j < kSlabCols / 32; ++j)
                  x[r][j] = staged[(r0 + r) * kSlabCols + (((32 * j + lane) / kPer16) ^ ((r0 + r) & 7)) * kPer16 + lane % kPer16];
#pragma unroll
              for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int j = 0; j < kSlabCols / 32; ++j)
                  if (r0 + r < rows && col + 32 * j < p.n) c[r * p.c_sm + 32 * j * p.c_sn] = x[r][j];
            }
          }
        }
      }
    }
    if (lane == 0) tma_store_wait_all<0>();
  }

  __syncthreads();
  if (slice_bits > 0) {
    // ---- the slices of the tile meet: this CTA sums every 2^slice_bits-th of its 128 rows, in slice order
    cluster_sync_all();
    if (*abort_flag == 0) {
      int tm, tn;
      tile_coords(worker, tiles_m, tiles_n, raster_group, tm, tn);
      const bool wide = f8_wide_store(p);
      const int first_row = tm * G::kTile + static_cast<int>(rank) * 128;
      for (int item = warp; item < 256 >> slice_bits; item += G::kThreads / 32) {  // half a row each
        const int row = slice + (item >> 1 << slice_bits), piece = (item & 1) * 32 + lane;
        if (first_row + row >= p.m) break;
        const float4 sum = f8_sum_slices<G::kMaxSlices>(smem_base + row * 1024 + ((piece ^ (row & 7)) << 4), 1 << slice_bits, static_cast<int>(rank), 2);
        f8_store4<OutT>(p, first_row + row, tn * G::kTile + 4 * piece, sum, wide);
      }
    }
  }

  // ---------------------------------------------------------------- teardown
  __syncthreads();
  if (*abort_flag != 0) {
    for (int i = 0; i < 1000; ++i) __nanosleep(1000);
    __syncthreads();
  }
  cluster_sync_all();  // neither CTA's barriers or tensor memory go away while the other may still signal or multiply
  if (warp == 1) {
    tcgen05_fence_after_sync();
    tmem_dealloc_pair(tmem_base, G::kTmemColumns);
  }
}

}  // namespace vb200
