// Block-scaled e4m3 product for few rows of A (M <= 128): every byte of the weights B crosses the memory bus once and the
// kernel's time is that stream.
//
//     C[m,n] = sum_b (sa[m,b] sb[n/128,b]) sum_{k in b} A[m,k] B[n,k]
//
// The weights are the MMA's 128-row operand (D^T = B . A^T), so a CTA's 128 output columns share one weight scale per
// block and A is the narrow operand, padded to kCols rows.  A CTA owns 128 columns of C and one of S slices of K:
//   warp 0    TMA: a 128-row x 128-byte tile of B and a kCols x 128-byte tile of A per stage
//   warp 1    four tcgen05.mma of 32 k per stage into one of kAccs fp32 accumulators - one accumulator per 128-k block, because
//             the block's scales apply to its sum
//   the rest  read the accumulator of each block back (thread = column of C) and add it, scaled, to the running totals
//             in registers; sa * sb come from shared memory, 32 blocks of them fetched at a time
// The S slices of a tile form a cluster: each leaves its totals in its own shared memory, over the drained ring, and CTA r
// sums rows m = r (mod S) of all slices, in slice order, so results do not depend on timing.  The store is a loop over
// shared memory, not code unrolled over the registers: instructions that run once are fetched at about 100 cycles a
// line, and 64 rows of unrolled stores took 5 us.
//
// Measured: 1 x 14336 x 4096 (58.7 MB of weights) 12.5 us in a graph, 4.7 TB/s: the stream itself runs at 7.3 TB/s, above what a
// copy reaches, and starting, the slices' meeting and the store are the other 3.7 us.  61 x 4100 x 4176: 8.2 us.  What is in
// flight decides: with the rings half as deep the two took 13.8 and 15.6 us.
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
  // accumulators in flight: the round trip MMA -> totals -> MMA of one is several times what its MMAs take
  static constexpr int kAccs = kCols <= 32 ? 8 : 4;
  // as many stages as fit: what streams from memory is what is in flight, about 2.2 us of it at full rate
  static constexpr int kStages = kCols == 16 ? 12 : kCols == 32 ? 11 : kCols == 64 ? 9 : 6;
  static constexpr int kRingBytes = kStages * kStageBytes;
  static constexpr int kMaxSlices = 8;  // the portable cluster size
  static constexpr int kScaleBlocks = 32;
  static constexpr int kScaleOffset = kRingBytes;
  static constexpr int kScaleBytes = kScaleBlocks * kCols * 4;
  static constexpr int kBarrierOffset = kScaleOffset + kScaleBytes;
  static constexpr int kSmemBytes = kBarrierOffset + 16 * (kStages + kAccs) + 8 + 1024;  // + alignment slack
  static constexpr int kPromoteWarps = kCols == 16 ? 4 : 8;
  static constexpr int kThreads = 32 * (2 + kPromoteWarps);
  static constexpr int kThreadCols = kCols / (kPromoteWarps / 4);  // totals per thread
  static constexpr int kTmemColumns = kAccs * kCols;
  static_assert(kTmemColumns <= 512, "tensor memory of one SM");
  static_assert(kCols * kRows * 4 <= kRingBytes, "the totals are left over the ring");
  static_assert(kSmemBytes <= 227 * 1024, "shared memory budget");
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

// Four neighbouring values of a row of C from column `n` on.
template <typename OutT>
__device__ __forceinline__ void f8_store4(const F8StreamArgs& p, int row, int n, const float4& sum, bool wide) {
  OutT* c = static_cast<OutT*>(p.c) + row * p.c_sm + n * p.c_sn;
  if (wide && n + 4 <= p.n) {
    if constexpr (sizeof(OutT) == 2) *reinterpret_cast<uint2*>(c) = make_uint2(pack_out16x2<OutT>(sum.x, sum.y), pack_out16x2<OutT>(sum.z, sum.w));
    else *reinterpret_cast<float4*>(c) = sum;
  } else {
    if (n < p.n) c[0] = f8_out<OutT>(sum.x);
    if (n + 1 < p.n) c[p.c_sn] = f8_out<OutT>(sum.y);
    if (n + 2 < p.n) c[2 * p.c_sn] = f8_out<OutT>(sum.z);
    if (n + 3 < p.n) c[3 * p.c_sn] = f8_out<OutT>(sum.w);
  }
}

// ... in one store where every row of C allows it.
__device__ __forceinline__ bool f8_wide_store(const F8StreamArgs& p) {
  return p.c_sn == 1 && (reinterpret_cast<uintptr_t>(p.c) & 15) == 0 && p.c_sm % 4 == 0;
}

// The sum over the slices, in their order, of sixteen bytes that each left at `at` in its shared memory; slice s is CTA first + step * s.
template <int kMaxSlices>
__device__ __forceinline__ float4 f8_sum_slices(uint32_t at, int slices, int first, int step) {
  float4 part[kMaxSlices];  // all slices' reads in flight together
#pragma unroll
  for (int other = 0; other < kMaxSlices; ++other)
    if (other < slices) part[other] = ld_shared_cluster_v4(map_to_cta(at, first + step * other));
  float4 sum = part[0];
#pragma unroll
  for (int other = 1; other < kMaxSlices; ++other)
    if (other < slices) sum.x += part[other].x, sum.y += part[other].y, sum.z += part[other].z, sum.w += part[other].w;
  return sum;
}

template <int kColsT, typename OutT>
__global__ void __launch_bounds__(F8Stream<kColsT>::kThreads, 1)
f8_stream_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const F8StreamArgs p, int slice_bits) {
  using G = F8Stream<kColsT>;
  const int slices = 1 << slice_bits;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
  const uint32_t full_bar = smem_base + G::kBarrierOffset;      // [stages] tiles landed              (TMA -> MMA)
  const uint32_t empty_bar = full_bar + 8 * G::kStages;         // [stages] tiles multiplied          (MMA -> TMA)
  const uint32_t tmem_full_bar = empty_bar + 8 * G::kStages;    // [accs] a block's sums are ready    (MMA -> totals)
  const uint32_t tmem_empty_bar = tmem_full_bar + 8 * G::kAccs;  // [accs] ... and have been read         (totals -> MMA)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem_gen + G::kBarrierOffset + 16 * (G::kStages + G::kAccs));
  volatile uint32_t* abort_flag = tmem_slot + 1;

  // (through a shuffle, so that the compiler knows it to be the same for the whole warp: the roles' loops then run on uniform registers)
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const int slice = static_cast<int>(blockIdx.x) & (slices - 1);  // = rank in the cluster
  const int n0 = (static_cast<int>(blockIdx.x) >> slice_bits) * G::kRows;
  const int num_kb = (p.k + 127) / 128;
  const int kb_begin = static_cast<int>(static_cast<long long>(num_kb) * slice >> slice_bits);
  const int kb_end = static_cast<int>(static_cast<long long>(num_kb) * (slice + 1) >> slice_bits);

  if (threadIdx.x == 0) {
    for (int s = 0; s < G::kStages; ++s) {
      mbar_init(full_bar + 8 * s, 1);
      mbar_init(empty_bar + 8 * s, 1);
    }
    for (int a = 0; a < G::kAccs; ++a) {
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
  tcgen05_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  grid_launch_dependents();
  grid_dependency_wait();

  auto give_up = [&](uint32_t code) {
    report_status(p.status, code);
    *abort_flag = 1;
  };
  if (warp == 0) {
    const bool leader = elect_one();
    for (int kb = kb_begin, s = 0, phase = 1; kb < kb_end; ++kb) {
      if (!mbar_wait(empty_bar + 8 * s, static_cast<uint32_t>(phase), abort_flag)) {
        if (leader) give_up(kStatusProducerWait);
        break;
      }
      if (leader) {
        mbar_arrive_expect_tx(full_bar + 8 * s, G::kStageBytes);
        tma_load_2d(smem_base + s * G::kStageBytes, &map_w, full_bar + 8 * s, kb * 128, n0);
        tma_load_2d(smem_base + s * G::kStageBytes + G::kWBytes, &map_x, full_bar + 8 * s, kb * 128, 0);  // rows past M: zeros
      }
      __syncwarp();
      if (++s == G::kStages) s = 0, phase ^= 1;
    }
  } else if (warp == 1) {
    // the whole warp walks the loop, one elected lane issues: what the instructions take stays in uniform registers
    constexpr uint32_t idesc = umma_instr_desc(kUmmaAccF32, kUmmaE4M3, kUmmaE4M3, G::kRows, G::kCols);
    const bool leader = elect_one();
    int acc = 0, acc_phase = 1;
    for (int kb = kb_begin, s = 0, phase = 0; kb < kb_end; ++kb) {
      if (!mbar_wait(full_bar + 8 * s, static_cast<uint32_t>(phase), abort_flag)) {
        if (leader) give_up(kStatusMmaWaitFull);
        break;
      }
      if (!mbar_wait(tmem_empty_bar + 8 * acc, static_cast<uint32_t>(acc_phase), abort_flag)) {
        if (leader) give_up(kStatusMmaWaitTmem);
        break;
      }
      tcgen05_fence_after_sync();
      const uint64_t w_desc = umma_smem_desc_sw128(smem_base + s * G::kStageBytes);
      const uint64_t x_desc = umma_smem_desc_sw128(smem_base + s * G::kStageBytes + G::kWBytes);
      if (leader) {
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) umma_f8(tmem_base + acc * G::kCols, w_desc + 2 * kk, x_desc + 2 * kk, idesc, kk != 0 ? 1u : 0u);
        umma_commit(empty_bar + 8 * s);
        umma_commit(tmem_full_bar + 8 * acc);
      }
      __syncwarp();
      if (++s == G::kStages) s = 0, phase ^= 1;
      if (++acc == G::kAccs) acc = 0, acc_phase ^= 1;
    }
  } else {
    const int thread = static_cast<int>(threadIdx.x) - 64;
    float* scales = reinterpret_cast<float*>(smem_gen + G::kScaleOffset);  // [block][row of A]
    const float* b_scale = p.b_scale + static_cast<long long>(n0 / 128) * p.bs_sn;
    const int quarter = warp & 3, col_part = (warp - 2) >> 2;  // a thread totals column quarter * 32 + lane of C for kThreadCols rows of A
    float total[G::kThreadCols];
#pragma unroll
    for (int j = 0; j < G::kThreadCols; ++j) total[j] = 0.f;
    bool ok = true;
    for (int kb = kb_begin; kb < kb_end; ++kb) {
      const int i = kb - kb_begin, acc = i % G::kAccs;
      if (i % G::kScaleBlocks == 0) {
        if (i != 0) asm volatile("bar.sync 1, %0;" ::"n"(G::kPromoteWarps * 32) : "memory");  // the previous scales have been used
        // a thread's scales belong to one block: one weight scale, and the loads of all its rows in flight together
        constexpr int kRowStep = G::kPromoteWarps * 32 / G::kScaleBlocks, kRows = G::kCols / kRowStep;
        const int block = thread % G::kScaleBlocks, first_row = thread / G::kScaleBlocks;
        const bool there = kb + block < kb_end;
        const float bs = there ? f8_load_scale(b_scale + (kb + block) * p.bs_sk) : 0.f;
        constexpr int kTogether = kRows < 8 ? kRows : 8;
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
      // the block's factors come into registers ahead of its sums, sixteen at a time
      const float* s = scales + i % G::kScaleBlocks * G::kCols + col_part * G::kThreadCols;
      float4 f[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) f[j] = reinterpret_cast<const float4*>(s)[j];
      // (a warp whose wait ran out keeps meeting the others at the barriers above)
      if (ok && !__all_sync(0xffffffffu, mbar_wait(tmem_full_bar + 8 * acc, static_cast<uint32_t>(i / G::kAccs) & 1u, abort_flag))) {
        if (lane == 0) give_up(kStatusEpilogueWait);
        ok = false;
      }
      if (!ok) continue;
      tcgen05_fence_after_sync();
      const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + acc * G::kCols + col_part * G::kThreadCols;
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
        float* sum = total + 16 * chunk;
        const uint32_t* x = v[chunk & 1];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          sum[4 * j] = fmaf(__uint_as_float(x[4 * j]), f[j].x, sum[4 * j]);
          sum[4 * j + 1] = fmaf(__uint_as_float(x[4 * j + 1]), f[j].y, sum[4 * j + 1]);
          sum[4 * j + 2] = fmaf(__uint_as_float(x[4 * j + 2]), f[j].z, sum[4 * j + 2]);
          sum[4 * j + 3] = fmaf(__uint_as_float(x[4 * j + 3]), f[j].w, sum[4 * j + 3]);
          if (chunk + 1 < G::kThreadCols / 16) f[j] = reinterpret_cast<const float4*>(s)[4 * (chunk + 1) + j];
        }
      }
    }
    // every MMA of this CTA is done and has read what TMA brought: the totals go over the ring, [row of A][column of C]
    if (ok) {
      float* mine = reinterpret_cast<float*>(smem_gen) + col_part * G::kThreadCols * G::kRows + quarter * 32 + lane;
#pragma unroll
      for (int j = 0; j < G::kThreadCols; ++j) mine[j * G::kRows] = total[j];
    }
  }

  // ---------------------------------------------------------------- the slices meet; every thread of the cluster comes here
  __syncthreads();
  if (slices > 1) cluster_sync_all();
  if (*abort_flag == 0) {
    // a warp per row: four columns a lane
    constexpr int kWarps = G::kThreads / 32;
    const int n = n0 + 4 * lane;
    const uint32_t totals = smem_base + 16 * lane;
    const bool wide = f8_wide_store(p);
    for (int row = slice + (warp << slice_bits); row < p.m; row += kWarps << slice_bits)
      f8_store4<OutT>(p, row, n, f8_sum_slices<G::kMaxSlices>(totals + row * (G::kRows * 4), slices, 0, 1), wide);
  }
  if (slices > 1) {  // no CTA leaves while another still reads its totals
    __syncwarp();
    cluster_sync_all();
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
