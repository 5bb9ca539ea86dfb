// Block-scaled e4m3 product at tensor-core rate: CTA pairs on 256 x 256 tiles of C.
//
//     C[m,n] = sum_b (sa[m,b] sb[n/128,b]) sum_{k in b} A[m,k] B[n,k]
//
// A block's scales apply to its sum over 128 k, so each 128-k step of the main loop is an accumulation of its own: four
// tcgen05.mma.cta_group::2 of 32 k into one of two 256-column fp32 accumulators in tensor memory, which eight warps then
// read back and add, scaled, to totals in registers - 128 a thread - while the tensor cores fill the other one.  A thread
// owns one row of C and 128 columns of it, all of one weight block: one factor sa * sb per step, one fused multiply-add
// per element (two per instruction, fma.rn.f32x2).  Roles, per CTA:
//   warp 0      TMA: its 128 rows of A and its 128 of the tile's 256 rows of B per step, a ring of kStages
//   warp 1      (leader CTA) issues the MMAs of the pair
//   warps 2-9   totals, then the store of the tile through shared memory by TMA (or directly where C cannot take that)
// Persistent: pairs walk the tiles `worker, worker + workers, ...`; the MMAs of the next tile start while this one is stored.
#pragma once

#include "f8_stream.cuh"

namespace vb200 {

struct F8Tiled {
  static constexpr int kTile = 256;
  static constexpr int kOperandBytes = 128 * 128;  // 128 rows x 128 bytes of A, and as much of B
  static constexpr int kStageBytes = 2 * kOperandBytes;
  static constexpr int kStages = 6;
  static constexpr int kTotalWarps = 8;
  static constexpr int kThreads = 32 * (2 + kTotalWarps);
  static constexpr int kStageOutBytes = 32 * 128;  // 32 rows x 128 bytes of C, per warp
  static constexpr int kOutOffset = kStages * kStageBytes;
  static constexpr int kBarrierOffset = kOutOffset + kTotalWarps * kStageOutBytes;
  static constexpr int kSmemBytes = kBarrierOffset + 256 + 1024;
  static constexpr int kTmemColumns = 512;
  static constexpr long long kGroupBytes = 32ll << 20;  // raster: row tiles holding this much of A share each sweep over N
};
static_assert(F8Tiled::kSmemBytes <= 227 * 1024, "shared memory budget");

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
                const F8StreamArgs p, int tma_store, int raster_group) {
  using G = F8Tiled;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
  const uint32_t full_bar = smem_base + G::kBarrierOffset;      // [stages] both CTAs' tiles landed   (TMA -> MMA; the leader's)
  const uint32_t empty_bar = full_bar + 8 * G::kStages;         // [stages] tiles multiplied          (MMA -> TMA of both)
  const uint32_t tmem_full_bar = empty_bar + 8 * G::kStages;    // [2] a step's sums are ready        (MMA -> totals of both)
  const uint32_t tmem_empty_bar = tmem_full_bar + 16;           // [2] ... and have been read         (totals of both -> MMA; the leader's)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem_gen + G::kBarrierOffset + 16 * G::kStages + 32);
  volatile uint32_t* abort_flag = tmem_slot + 1;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_cta_rank();
  const int worker = static_cast<int>(blockIdx.x >> 1), workers = static_cast<int>(gridDim.x >> 1);
  const int tiles_m = (p.m + G::kTile - 1) / G::kTile, tiles_n = (p.n + G::kTile - 1) / G::kTile;
  const int num_tiles = tiles_m * tiles_n;
  const int num_kb = (p.k + 127) / 128;

  if (threadIdx.x == 0) {
    for (int s = 0; s < G::kStages; ++s) {
      mbar_init(full_bar + 8 * s, 1);
      mbar_init(empty_bar + 8 * s, 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(tmem_full_bar + 8 * a, 1);
      mbar_init(tmem_empty_bar + 8 * a, 2 * G::kTotalWarps);
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

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = worker; ok && tile < num_tiles; tile += workers) {
        int tm, tn;
        tile_coords(tile, tiles_m, tiles_n, raster_group, tm, tn);
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mbar_wait(empty_bar + 8 * stage, phase ^ 1u, abort_flag)) {
            give_up(kStatusProducerWait);
            ok = false;
            break;
          }
          const uint32_t a_dst = smem_base + stage * G::kStageBytes;
          const uint32_t leader_full = map_to_cta(full_bar + 8 * stage, 0);
          if (rank == 0) mbar_arrive_expect_tx(full_bar + 8 * stage, 2 * G::kStageBytes);
          tma_load_2d_pair(a_dst, &map_a, leader_full, kb * 128, tm * G::kTile + static_cast<int>(rank) * 128);
          tma_load_2d_pair(a_dst + G::kOperandBytes, &map_b, leader_full, kb * 128, tn * G::kTile + static_cast<int>(rank) * 128);
          if (++stage == G::kStages) stage = 0, phase ^= 1u;
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      constexpr uint32_t idesc = umma_instr_desc(kUmmaAccF32, kUmmaE4M3, kUmmaE4M3, 256, 256);
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      for (int tile = worker; ok && tile < num_tiles; tile += workers) {
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mbar_wait_cluster(tmem_empty_bar + 8 * acc, acc_phase ^ 1u, abort_flag)) {
            give_up(kStatusMmaWaitTmem);
            ok = false;
            break;
          }
          if (!mbar_wait(full_bar + 8 * stage, phase, abort_flag)) {
            give_up(kStatusMmaWaitFull);
            ok = false;
            break;
          }
          tcgen05_fence_after_sync();
          const uint64_t a_desc = umma_smem_desc_sw128(smem_base + stage * G::kStageBytes);
          const uint64_t b_desc = umma_smem_desc_sw128(smem_base + stage * G::kStageBytes + G::kOperandBytes);
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) umma_f8_pair(tmem_base + acc * G::kTile, a_desc + 2 * kk, b_desc + 2 * kk, idesc, kk != 0 ? 1u : 0u);
          umma_commit_pair(empty_bar + 8 * stage);
          umma_commit_pair(tmem_full_bar + 8 * acc);
          if (++stage == G::kStages) stage = 0, phase ^= 1u;
          acc ^= 1;
          if (acc == 0) acc_phase ^= 1u;
        }
      }
    }
  } else {
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    const uint32_t out_buf = smem_base + G::kOutOffset + (warp - 2) * G::kStageOutBytes;
    int acc = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    for (int tile = worker; ok && tile < num_tiles; tile += workers) {
      int tm, tn;
      tile_coords(tile, tiles_m, tiles_n, raster_group, tm, tn);
      const int row0 = tm * G::kTile + static_cast<int>(rank) * 128 + quarter * 32;
      const int row = row0 + lane, col0 = tn * G::kTile + half * 128;
      const bool live = row < p.m && col0 < p.n;  // (what lies past the matrix is multiplied by zero and never stored)
      const float* a_scale = p.a_scale + (live ? row * p.as_sm : 0);
      const float* b_scale = p.b_scale + (live ? col0 / 128 * p.bs_sn : 0);
      float2 total[64];
#pragma unroll
      for (int j = 0; j < 64; ++j) total[j] = make_float2(0.f, 0.f);
      float next_a = live ? __ldg(a_scale) : 0.f, next_b = live ? __ldg(b_scale) : 0.f;
      for (int kb = 0; kb < num_kb; ++kb) {
        const float s = next_a * next_b;
        if (live && kb + 1 < num_kb) {  // the next step's scales arrive during this one
          next_a = __ldg(a_scale + (kb + 1) * p.as_sk);
          next_b = __ldg(b_scale + (kb + 1) * p.bs_sk);
        }
        if (!__all_sync(0xffffffffu, mbar_wait_cluster(tmem_full_bar + 8 * acc, acc_phase, abort_flag))) {
          if (lane == 0) give_up(kStatusEpilogueWait);
          ok = false;
          break;
        }
        tcgen05_fence_after_sync();
        const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + acc * G::kTile + half * 128;
        uint32_t v[2][16];
        tmem_load_32x16(taddr, v[0]);
#pragma unroll
        for (int chunk = 0; chunk < 8; ++chunk) {
          tmem_load_wait();
          if (chunk + 1 < 8) {
            tmem_load_32x16(taddr + 16 * (chunk + 1), v[(chunk + 1) & 1]);
          } else {
            tcgen05_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(map_to_cta(tmem_empty_bar + 8 * acc, 0));
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) f8_fma2(total[8 * chunk + j], v[chunk & 1][2 * j], v[chunk & 1][2 * j + 1], s);
        }
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1u;
      }
      if (!ok) break;
      // ---- the tile leaves: 128 bytes of every row at a time
      constexpr int kSlabCols = 128 / static_cast<int>(sizeof(OutT));
#pragma unroll
      for (int slab = 0; slab < 128 / kSlabCols; ++slab) {
        if (col0 + slab * kSlabCols >= p.n || row0 >= p.m) continue;  // (uniform over the warp)
        if (tma_store) {
          if (lane == 0) tma_store_wait_read<0>();  // the slab before this one has left the buffer
          __syncwarp();
#pragma unroll
          for (int piece = 0; piece < 8; ++piece) {
            uint32_t w[4];
            if constexpr (sizeof(OutT) == 2) {
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float2 f = total[slab * 32 + piece * 4 + e];
                w[e] = pack_out16x2<OutT>(f.x, f.y);
              }
            } else {
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const float2 f = total[slab * 16 + piece * 2 + e];
                w[2 * e] = __float_as_uint(f.x), w[2 * e + 1] = __float_as_uint(f.y);
              }
            }
            const uint32_t dst = out_buf + lane * 128 + ((piece ^ (lane & 7)) << 4);
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&map_c, out_buf, col0 + slab * kSlabCols, row0);  // rows and columns past C are clipped
            tma_store_commit();
          }
        } else if (row < p.m) {
          OutT* c = static_cast<OutT*>(p.c) + row * p.c_sm;
#pragma unroll
          for (int j = 0; j < kSlabCols; ++j) {
            const int col = col0 + slab * kSlabCols + j;
            const float2 f = total[(slab * kSlabCols + j) / 2];
            if (col < p.n) c[col * p.c_sn] = f8_out<OutT>(j & 1 ? f.y : f.x);
          }
        }
      }
    }
    if (lane == 0) tma_store_wait_all<0>();
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
