// Block-scaled e4m3 product for few rows of A (M <= 256): every byte of the weights B crosses the memory bus once and the
// kernel's time is that stream.
//
//     C[m,n] = sum_b (sa[m,b] sb[n/128,b]) sum_{k in b} A[m,k] B[n,k]
//
// The weights are the MMA's 128-row operand (D^T = B . A^T), so a CTA's 128 output columns share one weight scale per
// block and A is the narrow operand, padded to kCols rows.  A CTA owns 128 columns of C and one of S slices of K:
//   warp 0    TMA: a 128-row x 128-byte tile of B and a kCols x 128-byte tile of A per stage
//   warp 1    four tcgen05.mma of 32 k per stage into one of two fp32 accumulators - one accumulator per 128-k block, because
//             the block's scales apply to its sum
//   the rest  read the accumulator of each block back (thread = column of C) and add it, scaled, to the running totals
//             in registers; sa * sb come from shared memory, 32 blocks of them fetched at a time
// The S slices of a tile form a cluster and meet in shared memory: CTA r sums rows m = r (mod S) of all slices, in slice
// order, so results do not depend on timing.
#pragma once

#include "f8_generic.cuh"
#include "gemm_tcgen05.cuh"  // status codes, report_status
#include "ptx.cuh"

namespace vb200 {

template <int kColsT>
struct F8Stream {
  static constexpr int kCols = kColsT;  // rows of A, padded: the MMA's N
  static constexpr int kRows = 128;     // columns of C per CTA: the MMA's M
  static constexpr int kWBytes = kRows * 128;
  static constexpr int kXBytes = kCols * 128;
  static constexpr int kStageBytes = kWBytes + kXBytes;
  // up to 64 rows two CTAs share an SM: while one waits for its first tile or stores, the other streams
  static constexpr int kCtasPerSm = kCols <= 64 ? 2 : 1;
  static constexpr int kStages = kCols == 16 ? 5 : kCols <= 64 ? 4 : kCols == 128 ? 6 : 4;
  static constexpr int kRingBytes = kStages * kStageBytes;
  static constexpr int kScaleBlocks = 32;
  static constexpr int kScaleOffset = kRingBytes;
  static constexpr int kScaleBytes = kScaleBlocks * kCols * 4;
  // the slices' meeting place: [slice][row of A / S][column of C].  Apart from the ring where there is room (no barrier is
  // needed before a slice writes into another CTA then), over the drained ring otherwise.
  static constexpr bool kExchangeApart = kCols <= 32;
  static constexpr int kExchangeBytes = kCols * kRows * 4;
  static constexpr int kExchangeOffset = kExchangeApart ? kScaleOffset + kScaleBytes : 0;
  static constexpr int kBarrierOffset = kScaleOffset + kScaleBytes + (kExchangeApart ? kExchangeBytes : 0);
  static constexpr int kSmemBytes = kBarrierOffset + 256 + 1024;  // + alignment slack
  static constexpr int kPromoteWarps = kCols == 256 ? 8 : 4;
  static constexpr int kThreads = 32 * (2 + kPromoteWarps);
  static constexpr int kThreadCols = kCols / (kPromoteWarps / 4);  // totals per thread
  static constexpr int kTmemColumns = kCols == 16 ? 32 : 2 * kCols;
  static_assert(kExchangeApart || kExchangeBytes <= kRingBytes, "the exchange lies over the ring");
  static_assert(kCtasPerSm * (kSmemBytes + 1024) <= 228 * 1024, "shared memory budget");
};

struct F8StreamArgs {
  const float* a_scale;
  long long as_sm, as_sk;
  const float* b_scale;
  long long bs_sn, bs_sk;
  void* c;
  long long c_sm, c_sn;
  int m, n, k;
  uint32_t* status;
};

// A scale, fetched where the source says: an ordinary load may be moved down to its first use, behind the waits it is meant to overlap.
__device__ __forceinline__ float f8_load_scale(const float* p) {
  float x;
  asm volatile("ld.global.nc.f32 %0, [%1];" : "=f"(x) : "l"(p));
  return x;
}

template <int kColsT, typename OutT>
__global__ void __launch_bounds__(F8Stream<kColsT>::kThreads, F8Stream<kColsT>::kCtasPerSm)
f8_stream_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const F8StreamArgs p, int slices) {
  using G = F8Stream<kColsT>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
  const uint32_t full_bar = smem_base + G::kBarrierOffset;      // [stages] tiles landed              (TMA -> MMA)
  const uint32_t empty_bar = full_bar + 8 * G::kStages;         // [stages] tiles multiplied          (MMA -> TMA)
  const uint32_t tmem_full_bar = empty_bar + 8 * G::kStages;    // [2] a block's sums are ready       (MMA -> totals)
  const uint32_t tmem_empty_bar = tmem_full_bar + 16;           // [2] ... and have been read         (totals -> MMA)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem_gen + G::kBarrierOffset + 16 * G::kStages + 32);
  volatile uint32_t* abort_flag = tmem_slot + 1;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int slice = static_cast<int>(blockIdx.x) % slices;  // = rank in the cluster
  const int n0 = static_cast<int>(blockIdx.x) / slices * G::kRows;
  const int num_kb = (p.k + 127) / 128;
  const int kb_begin = static_cast<int>(static_cast<long long>(num_kb) * slice / slices);
  const int kb_end = static_cast<int>(static_cast<long long>(num_kb) * (slice + 1) / slices);

  if (threadIdx.x == 0) {
    for (int s = 0; s < G::kStages; ++s) {
      mbar_init(full_bar + 8 * s, 1);
      mbar_init(empty_bar + 8 * s, 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(tmem_full_bar + 8 * a, 1);
      mbar_init(tmem_empty_bar + 8 * a, G::kPromoteWarps);
    }
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_descriptor(&map_w);
    tma_prefetch_descriptor(&map_x);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), G::kTmemColumns);
    tmem_relinquish();
  }
  tcgen05_fence_before_sync();
  __syncthreads();
  if (G::kExchangeApart && slices > 1) cluster_arrive();  // this CTA runs: the others may write into its exchange
  tcgen05_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  grid_launch_dependents();
  grid_dependency_wait();

  auto give_up = [&](uint32_t code) {
    report_status(p.status, code);
    *abort_flag = 1;
  };
  float total[G::kThreadCols];
  const int quarter = warp & 3;
  const int col_part = warp < 2 ? 0 : (warp - 2) >> 2;  // which kThreadCols rows of A this thread totals
  const int row_local = quarter * 32 + lane;            // column of C inside the tile

  if (warp == 0) {
    if (lane == 0) {
      for (int kb = kb_begin; kb < kb_end; ++kb) {
        const int i = kb - kb_begin, s = i % G::kStages;
        if (!mbar_wait(empty_bar + 8 * s, (static_cast<uint32_t>(i / G::kStages) & 1u) ^ 1u, abort_flag)) {
          give_up(kStatusProducerWait);
          break;
        }
        mbar_arrive_expect_tx(full_bar + 8 * s, G::kStageBytes);
        tma_load_2d(smem_base + s * G::kStageBytes, &map_w, full_bar + 8 * s, kb * 128, n0);
        tma_load_2d(smem_base + s * G::kStageBytes + G::kWBytes, &map_x, full_bar + 8 * s, kb * 128, 0);  // rows past M: zeros
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = umma_instr_desc(kUmmaAccF32, kUmmaE4M3, kUmmaE4M3, G::kRows, G::kCols);
      for (int kb = kb_begin; kb < kb_end; ++kb) {
        const int i = kb - kb_begin, s = i % G::kStages, acc = i & 1;
        if (!mbar_wait(tmem_empty_bar + 8 * acc, (static_cast<uint32_t>(i >> 1) & 1u) ^ 1u, abort_flag)) {
          give_up(kStatusMmaWaitTmem);
          break;
        }
        if (!mbar_wait(full_bar + 8 * s, static_cast<uint32_t>(i / G::kStages) & 1u, abort_flag)) {
          give_up(kStatusMmaWaitFull);
          break;
        }
        tcgen05_fence_after_sync();
        const uint64_t w_desc = umma_smem_desc_sw128(smem_base + s * G::kStageBytes);
        const uint64_t x_desc = umma_smem_desc_sw128(smem_base + s * G::kStageBytes + G::kWBytes);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) umma_f8(tmem_base + acc * G::kCols, w_desc + 2 * kk, x_desc + 2 * kk, idesc, kk != 0 ? 1u : 0u);
        umma_commit(empty_bar + 8 * s);
        umma_commit(tmem_full_bar + 8 * acc);
      }
    }
  } else {
    const int thread = static_cast<int>(threadIdx.x) - 64;
    float* scales = reinterpret_cast<float*>(smem_gen + G::kScaleOffset);  // [block][row of A]
    const float* b_scale = p.b_scale + static_cast<long long>(n0 / 128) * p.bs_sn;
#pragma unroll
    for (int j = 0; j < G::kThreadCols; ++j) total[j] = 0.f;
    bool ok = true;
    for (int kb = kb_begin; kb < kb_end; ++kb) {
      const int i = kb - kb_begin, acc = i & 1;
      if (i % G::kScaleBlocks == 0) {
        if (i != 0) asm volatile("bar.sync 1, %0;" ::"n"(G::kPromoteWarps * 32) : "memory");  // the previous scales have been used
        // a thread's scales belong to one block: one weight scale, and the loads of all its rows in flight together
        constexpr int kRowStep = G::kPromoteWarps * 32 / G::kScaleBlocks, kRows = G::kCols / kRowStep;
        const int block = thread % G::kScaleBlocks, first_row = thread / G::kScaleBlocks;
        const bool there = kb + block < kb_end;
        const float bs = there ? f8_load_scale(b_scale + (kb + block) * p.bs_sk) : 0.f;
        constexpr int kTogether = kRows < 16 ? kRows : 16;
#pragma unroll 1
        for (int r0 = 0; r0 < kRows && r0 * kRowStep < p.m; r0 += kTogether) {
          float s[kTogether];
#pragma unroll
          for (int r = 0; r < kTogether; ++r) {
            const int row = first_row + (r0 + r) * kRowStep;
            s[r] = there && row < p.m ? f8_load_scale(p.a_scale + row * p.as_sm + (kb + block) * p.as_sk) : 0.f;
          }
#pragma unroll
          for (int r = 0; r < kTogether; ++r) scales[block * G::kCols + first_row + (r0 + r) * kRowStep] = s[r] * bs;
        }
        asm volatile("bar.sync 1, %0;" ::"n"(G::kPromoteWarps * 32) : "memory");
      }
      // (a warp whose wait ran out keeps meeting the others at the barriers above)
      if (ok && !__all_sync(0xffffffffu, mbar_wait(tmem_full_bar + 8 * acc, static_cast<uint32_t>(i >> 1) & 1u, abort_flag))) {
        if (lane == 0) give_up(kStatusEpilogueWait);
        ok = false;
      }
      if (!ok) continue;
      tcgen05_fence_after_sync();
      const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + acc * G::kCols + col_part * G::kThreadCols;
      const float* s = scales + i % G::kScaleBlocks * G::kCols + col_part * G::kThreadCols;
      // sixteen columns per read, the next sixteen on their way while these are added
      uint32_t v[2][16];
      tmem_load_32x16(taddr, v[0]);
#pragma unroll
      for (int chunk = 0; chunk < G::kThreadCols / 16; ++chunk) {
        tmem_load_wait();
        if (chunk + 1 < G::kThreadCols / 16) {
          tmem_load_32x16(taddr + 16 * (chunk + 1), v[(chunk + 1) & 1]);
        } else {
          tcgen05_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(tmem_empty_bar + 8 * acc);
        }
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
          const float4 f = *reinterpret_cast<const float4*>(s + 16 * chunk + j);
          total[16 * chunk + j] = fmaf(__uint_as_float(v[chunk & 1][j]), f.x, total[16 * chunk + j]);
          total[16 * chunk + j + 1] = fmaf(__uint_as_float(v[chunk & 1][j + 1]), f.y, total[16 * chunk + j + 1]);
          total[16 * chunk + j + 2] = fmaf(__uint_as_float(v[chunk & 1][j + 2]), f.z, total[16 * chunk + j + 2]);
          total[16 * chunk + j + 3] = fmaf(__uint_as_float(v[chunk & 1][j + 3]), f.w, total[16 * chunk + j + 3]);
        }
      }
    }
  }

  // ---------------------------------------------------------------- the slices meet; every thread of the cluster comes here
  __syncthreads();
  const int n = n0 + row_local;
  OutT* c = static_cast<OutT*>(p.c) + static_cast<long long>(n) * p.c_sn;
  if (slices == 1) {
    if (warp >= 2 && *abort_flag == 0 && n < p.n) {
#pragma unroll
      for (int j = 0; j < G::kThreadCols; ++j) {
        const int row = col_part * G::kThreadCols + j;
        if (row < p.m) c[row * p.c_sm] = f8_out<OutT>(total[j]);
      }
    }
  } else {
    // another CTA's shared memory may be written once that CTA runs - and, where the exchange lies over its ring, once
    // its ring is idle
    if constexpr (!G::kExchangeApart) cluster_arrive();
    cluster_wait();
    if (warp >= 2) {
      const uint32_t mine = smem_base + G::kExchangeOffset + (static_cast<uint32_t>(slice) * (G::kCols / slices) * G::kRows + row_local) * 4;
#pragma unroll
      for (int j = 0; j < G::kThreadCols; ++j) {
        const int row = col_part * G::kThreadCols + j;
        if (row < p.m) st_shared_cluster_f32(map_to_cta(mine + static_cast<uint32_t>(row / slices) * (G::kRows * 4), row % slices), total[j]);
      }
    }
    cluster_sync_all();
    if (warp >= 2 && *abort_flag == 0 && n < p.n) {
      const float* sums = reinterpret_cast<const float*>(smem_gen + G::kExchangeOffset) + row_local;
      const int stride = G::kCols / slices * G::kRows;
      for (int j = col_part; j * slices + slice < p.m; j += G::kPromoteWarps / 4) {
        float sum = 0.f;
        for (int other = 0; other < slices; ++other) sum += sums[other * stride + j * G::kRows];
        c[(j * slices + slice) * p.c_sm] = f8_out<OutT>(sum);
      }
    }
  }
  __syncthreads();
  if (*abort_flag != 0) {
    // a wait ran out: give copies and MMAs still in flight time to land before shared and tensor memory go back
    for (int i = 0; i < 1000; ++i) __nanosleep(1000);
    __syncthreads();
  }
  if (warp == 1) {
    tcgen05_fence_after_sync();
    tmem_dealloc(tmem_base, G::kTmemColumns);
  }
}

}  // namespace vb200
