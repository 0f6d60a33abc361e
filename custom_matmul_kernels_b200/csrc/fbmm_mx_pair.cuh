// The 4-bit product on CTA pairs (cta_group::2), for products with many tiles: a 256 x 256 tile, each
// CTA supplying 128 rows of A and 128 of B, so that 256 elements of k cost a CTA 35 KB of copies for 512
// cycles of MMA (the 128 x 128 tile of fbmm_mx_gemm.cuh: 34 KB for 128). Every CTA multiplies its own
// rows of A with all 256 of B, so its tensor memory holds the scales of its rows of A and of all rows of B.
//
// The scales come by tensor map (their copies are counted on the issuing CTA's barrier, which only
// tensor copies with cta_group::2 can reach from the other CTA); groups that do not exist are filled with
// zero, which with the zero codes behind k adds nothing.
//
// One accumulator stage: 256 columns of sums and 5 x 24 of scales leave no room for a second. Eight
// epilogue warps take the whole tile into registers (128 columns a thread) and release it before they
// store, so that the next tile's MMAs wait for the loads only.
#pragma once
#include "fbmm_x16_gemm.cuh"

namespace fbmm {

constexpr int kMxPairPart = 128 * kMxRowBytes;                          // 16 KB
constexpr int kMxPairStage = 2 * kMxPairPart + 3 * kMxScaleStage;      // A, B, scales of A, of B (two groups)
constexpr int kMxPairStages = 5;
constexpr int kMxPairSfCols = 24;
constexpr int kMxPairEpiBytes = 8 * 4096;
constexpr int kMxPairSmem = 1024 + kMxPairStages * kMxPairStage + kMxPairEpiBytes + 256;
constexpr int kMxPairThreads = 320;
static_assert(kMxPairSmem <= static_cast<int>(kMxSmemLimit), "shared memory");

struct MxPairArgs {
  void* C;
  long long ldc, stride_c;
  int l, m, n, k;
  int a_shared, b_shared, as_shared, bs_shared;  // one matrix of codes / scales for every batch
  int out_type;
  int m_tiles, n_tiles;
  int align;
};

__device__ __forceinline__ void mx_umma_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t sfa,
                                             uint32_t sfb, uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %6, 0;\n"
      "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n"
      "}\n"
      ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
      : "memory");
}
// The same shared-memory offset of each CTA to the same columns of its own tensor memory.
__device__ __forceinline__ void mx_copy_scales_pair(uint32_t tmem, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
}

struct MxPairBarriers {
  uint64_t full[kMxPairStages], empty[kMxPairStages], acc_full, acc_empty;
  uint32_t tmem_base, abort_flag;
};
static_assert(sizeof(MxPairBarriers) <= 256, "barrier block");

__global__ void __launch_bounds__(kMxPairThreads, 1)
mx_gemm_pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                    const __grid_constant__ CUtensorMap map_sa, const __grid_constant__ CUtensorMap map_sb,
                    const MxPairArgs a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* epi = smem + kMxPairStages * kMxPairStage;
  MxPairBarriers* bars = reinterpret_cast<MxPairBarriers*>(epi + kMxPairEpiBytes);
  volatile uint32_t* abort_flag = &bars->abort_flag;
  const uint32_t warp = warp_index(), lane = lane_id();
  const uint32_t rank = cluster_cta_rank();
  if (threadIdx.x == 0) {
    bars->abort_flag = 0;
    for (int s = 0; s < kMxPairStages; ++s) { mbar_init(&bars->full[s], 1); mbar_init(&bars->empty[s], 1); }
    mbar_init(&bars->acc_full, 1);
    mbar_init(&bars->acc_empty, 16);
    fence_barrier_init();
    tma_prefetch_desc(&map_a);
    tma_prefetch_desc(&map_b);
    tma_prefetch_desc(&map_sa);
    tma_prefetch_desc(&map_sb);
  }
  if (warp == 1) {
    tmem_alloc_pair(&bars->tmem_base, 512);
    tmem_relinquish_alloc_permit_pair();
  }
  tcgen05_fence_before_sync();
  cluster_sync_all();
  tcgen05_fence_after_sync();
  const uint32_t tmem = bars->tmem_base;
  const uint32_t bars0 = map_to_cta(smem_u32(bars), 0), bars1 = map_to_cta(smem_u32(bars), 1);
  auto off = [&](const uint64_t* b) -> uint32_t { return smem_u32(b) - smem_u32(bars); };
  auto commit = [&](uint64_t* bar) {
    umma_commit_pair(bars0 + off(bar));
    umma_commit_pair(bars1 + off(bar));
  };
  const int kblocks = (a.k + kMxStageK - 1) / kMxStageK;
  const long long units = static_cast<long long>(a.m_tiles) * a.n_tiles * a.l;
  const long long u0 = blockIdx.x >> 1, du = gridDim.x >> 1;

  if (warp == 0) {
    {
      uint32_t stage = 0, phase = 0;
      bool ok = true;
      mx_wait_for_previous();
      for (long long u = u0; u < units && ok; u += du) {
        int b, mt, nt;
        x16_decode(u, a.m_tiles, a.n_tiles, b, mt, nt);
        const int mr = mt * 256 + static_cast<int>(rank) * 128, nr = nt * 256 + static_cast<int>(rank) * 128;
        for (int kb = 0; kb < kblocks; ++kb) {
          ok = __all_sync(0xffffffffu, mbar_wait_cluster(&bars->empty[stage], phase ^ 1u, abort_flag));
          if (!ok) break;
          uint8_t* st = smem + stage * kMxPairStage;
          uint8_t* sf = st + 2 * kMxPairPart;
          const uint32_t full = bars0 + off(&bars->full[stage]);
          if (elect_one()) {
            if (rank == 0) mbar_arrive_expect_tx(&bars->full[stage], 2 * kMxPairStage);
            tma_load_3d_pair(st, &map_a, full, kb * kMxRowBytes, mr, a.a_shared ? 0 : b, kL2EvictLast);
            tma_load_3d_pair(st + kMxPairPart, &map_b, full, kb * kMxRowBytes, nr, a.b_shared ? 0 : b, kL2EvictLast);
            tma_load_3d_pair(sf, &map_sa, full, kb * (kMxScaleStage / 4), mr / 128, a.as_shared ? 0 : b, kL2EvictLast);
            tma_load_3d_pair(sf + kMxScaleStage, &map_sb, full, kb * (kMxScaleStage / 4), nt * 2, a.bs_shared ? 0 : b, kL2EvictLast);
          }
          __syncwarp();
          if (++stage == kMxPairStages) { stage = 0; phase ^= 1u; }
        }
      }
      if (!ok) {  // copies in flight land before the CTA leaves
        const long long t0 = clock64();
        while (clock64() - t0 < 2000000LL) {}
      }
    }
  } else if (warp == 1) {
    if (rank == 0) {
      uint32_t stage = 0, phase = 0, acc_phase = 0;
      bool ok = true;
      for (long long u = u0; u < units && ok; u += du) {
        ok = __all_sync(0xffffffffu, mbar_wait_cluster(&bars->acc_empty, acc_phase ^ 1u, abort_flag));
        if (!ok) break;
        for (int kb = 0; kb < kblocks; ++kb) {
          ok = __all_sync(0xffffffffu, mbar_wait_cluster(&bars->full[stage], phase, abort_flag));
          if (!ok) break;
          tcgen05_fence_after_sync();
          const uint32_t st = smem_u32(smem + stage * kMxPairStage);
          const uint32_t sf = st + 2 * kMxPairPart;
          const uint32_t t_sf = tmem + 256 + stage * kMxPairSfCols;  // per group of k: 4 columns of A, 8 of B
          const uint64_t ad = mx_desc_codes(st), bd = mx_desc_codes(st + kMxPairPart);
          if (elect_one()) {
#pragma unroll
            for (int g = 0; g < 2; ++g) {
              mx_copy_scales_pair(t_sf + g * 12, mx_desc_scales(sf + g * kMxGroupBytes));
              mx_copy_scales_pair(t_sf + g * 12 + 4, mx_desc_scales(sf + kMxScaleStage + g * kMxGroupBytes));
              mx_copy_scales_pair(t_sf + g * 12 + 8, mx_desc_scales(sf + 2 * kMxScaleStage + g * kMxGroupBytes));
            }
#pragma unroll
            for (int q = 0; q < 4; ++q)
              mx_umma_pair(tmem, ad + q * 2, bd + q * 2, mx_idesc(256, 256, (q & 1) * 2), t_sf + (q >> 1) * 12,
                           t_sf + (q >> 1) * 12 + 4, (kb | q) != 0 ? 1u : 0u);
            commit(&bars->empty[stage]);
            if (kb == kblocks - 1) commit(&bars->acc_full);
          }
          __syncwarp();
          if (++stage == kMxPairStages) { stage = 0; phase ^= 1u; }
        }
        acc_phase ^= 1u;
      }
    }
  } else {
    const uint32_t quarter = warp & 3u;
    const int half = static_cast<int>((warp - 2) >> 2);
    uint8_t* stage_mem = epi + (warp - 2) * 4096;
    uint32_t acc_phase = 0;
    bool ok = true;
    for (long long u = u0; u < units && ok; u += du) {
      int b, mt, nt;
      x16_decode(u, a.m_tiles, a.n_tiles, b, mt, nt);
      ok = mbar_wait_cluster(&bars->acc_full, acc_phase, abort_flag);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tcgen05_fence_after_sync();
      const uint32_t t = tmem + ((quarter * 32u) << 16) + half * 128;
      uint32_t v[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld_32x32b_x32(t + c * 32, v[c]);
      tmem_ld_wait();
      tcgen05_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive_values(bars0 + off(&bars->acc_empty));
      acc_phase ^= 1u;
      const int m0 = mt * 256 + static_cast<int>(rank) * 128 + static_cast<int>(quarter) * 32;
#pragma unroll
      for (int c = 0; c < 4; c += 2) {
        const int n0 = nt * 256 + half * 128 + c * 32;
        if (n0 < a.n && m0 < a.m)
          mx_store_rows(stage_mem, v[c], v[c + 1], a.C, b * a.stride_c + static_cast<long long>(m0) * a.ldc + n0, a.ldc,
                        a.out_type, a.m - m0, a.n - n0, a.align);
      }
    }
  }
  tcgen05_fence_before_sync();
  cluster_sync_all();
  if (threadIdx.x == 0 && *abort_flag != 0) atomicOr(&g_mx_status[0], 1u);
  if (warp == 1) {
    tcgen05_fence_after_sync();
    tmem_dealloc_pair(tmem, 512);
  }
}

}  // namespace fbmm
