// The 4-bit product for few rows of A (a decoding step): C[m][n] for m <= NT rows, and for tiles of 128 rows
// where whole tiles are too few for the SMs. The weights fill the 128-row side of the MMA and are streamed once,
// which is what bounds the product (17/32 byte per weight). A comes as codes (T = uint8_t), copied beside the
// weights, or as fp32 / fp16 / bf16, which every CTA quantises for its own range of k (fbmm_mx_quant.cuh's rules,
// straight into the swizzled tiles and scale groups that the MMA reads) while the first weights are on their
// way: no separate pass, no workspace, one launch, as long as there is little to quantise (few_rows_fused
// in fbmm_mx_api.cu).
//
// Few tiles of n leave SMs idle, so k is split over a cluster of S CTAs; the partial sums meet in
// shared memory and every CTA of the cluster adds up its share of the rows over the cluster in rank
// order: the result does not depend on timing. One token at 4096 x 4096: 5.8 us over three weights in
// turn, 6.1 us over thirty (9.2 us as a quantising pass and an unsplit product); 16 rows of codes at n = 16384, k = 8192:
// 11.0 us with weights partly in L2, 15.7 us from memory (17.6 us with the quantiser ahead of it), where
// longer weights stream at 6.5 TB/s behind 5 us of launch, set-up, first bytes and joining.
//
// Roles: warp 0 copies, warp 1 issues MMAs, the others quantise, then warps 2-5 read the sums.
#pragma once
#include <type_traits>

#include "fbmm_mx_gemm.cuh"

namespace fbmm {

constexpr int kMxRowsWeights = kMxM * kMxRowBytes + kMxScaleStage;  // weights and their scales per stage: 17 KB
constexpr int kMxRowsMaxStages = 8;

struct MxRowsArgs {
  const void* x;            // A [l][m][k], k contiguous
  long long ldx, stride_x;  // elements
  void* C;
  long long ldc, stride_c;
  int l, m, n, k;
  int w_shared, sw_shared, a_shared, sa_shared;
  int out_type;
  int align;                // bytes that C's rows are aligned to
  int n_tiles, m_tiles, splits, blocks_per_split;  // blocks of 256 k
  int stages;
};

struct MxRowsBarriers {
  uint64_t full[kMxRowsMaxStages], empty[kMxRowsMaxStages], a_ready, acc_full;
  uint32_t tmem_base, abort_flag;
};
static_assert(sizeof(MxRowsBarriers) <= 256, "barrier block");

template <int NT, typename T>
struct MxRowsShape {
  static constexpr bool kCodes = std::is_same<T, uint8_t>::value;
  static constexpr int kABlock = NT * kMxRowBytes + kMxScaleStage;  // per 256 k: codes of A, scales
  static constexpr int kStage = kMxRowsWeights + (kCodes ? kABlock : 0);
  static constexpr int kSums = NT * 128 * 4;
  static constexpr int kSfBase = NT > 64 ? NT : 64;  // tensor-memory column of the scales, 16 per stage
  static constexpr int kMaxStages = (256 - kSfBase) / 16 < kMxRowsMaxStages ? (256 - kSfBase) / 16 : kMxRowsMaxStages;
  static constexpr int kThreads = kCodes ? 192 : 320;
  static constexpr int kQuantWarps = kThreads / 32 - 2;
  __host__ __device__ static constexpr int ring(int stages) {
    return ((stages * kStage > kSums ? stages * kStage : kSums) + 1023) / 1024 * 1024;
  }
  static constexpr int smem(int stages, int blocks) { return 1024 + ring(stages) + (kCodes ? 0 : blocks * kABlock) + 256; }
};

// Without an eviction priority: a decoding step's weights may or may not fit L2 until the next one.
__device__ __forceinline__ void tma_load_3d_normal(void* smem_dst, const void* tmap, uint64_t* bar, int32_t c0, int32_t c1,
                                                   int32_t c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(smem_u32(smem_dst)), "l"(reinterpret_cast<uint64_t>(tmap)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}

template <int NT, typename T>
__global__ void __launch_bounds__(MxRowsShape<NT, T>::kThreads, 2)
mx_rows_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_sw,
               const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_sa, const MxRowsArgs a) {
  using S = MxRowsShape<NT, T>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* a_codes = smem + S::ring(a.stages);  // unless they come in the ring
  uint8_t* a_scales = a_codes + a.blocks_per_split * (NT * kMxRowBytes);
  MxRowsBarriers* bars = reinterpret_cast<MxRowsBarriers*>(
      smem + S::ring(a.stages) + (S::kCodes ? 0 : a.blocks_per_split * S::kABlock));
  volatile uint32_t* abort_flag = &bars->abort_flag;
  const uint32_t warp = warp_index(), lane = lane_id();
  const uint32_t split = cluster_cta_rank();
  const int unit = static_cast<int>(blockIdx.x / static_cast<uint32_t>(a.splits));
  const int mt = unit % a.m_tiles, column = unit / a.m_tiles;
  const int b = column / a.n_tiles, n0 = (column - b * a.n_tiles) * kMxM;
  const int m0 = mt * NT, rows = min(NT, a.m - m0);  // more than one tile of rows only at NT = 128
  const int kblocks = (a.k + kMxStageK - 1) / kMxStageK;
  const int first = static_cast<int>(split) * a.blocks_per_split;
  const int count = max(0, min(a.blocks_per_split, kblocks - first));  // this CTA's blocks of 256 k
  auto load_weights = [&](int stage, int i) {  // block i of this CTA's range
    uint8_t* st = smem + stage * S::kStage;
    mbar_arrive_expect_tx(&bars->full[stage], S::kStage);
    tma_load_3d_normal(st, &map_w, &bars->full[stage], (first + i) * kMxRowBytes, n0, a.w_shared ? 0 : b);
    tma_load_3d_normal(st + kMxM * kMxRowBytes, &map_sw, &bars->full[stage], (first + i) * (kMxScaleStage / 4), n0 / kMxM,
                       a.sw_shared ? 0 : b);
  };
  auto load_a = [&](int stage, int i) {
    uint8_t* st = smem + stage * S::kStage + kMxRowsWeights;
    tma_load_3d(st, &map_a, &bars->full[stage], (first + i) * kMxRowBytes, m0, a.a_shared ? 0 : b, kL2EvictLast);
    tma_load_3d(st + NT * kMxRowBytes, &map_sa, &bars->full[stage], (first + i) * (kMxScaleStage / 4), m0 / 128,
                a.sa_shared ? 0 : b, kL2EvictLast);
  };
  const int early = min(count, a.stages);
  if (warp == 0) {
    // the first copies of the ring leave before anything else, those of A once what may be quantising it is done
    if (elect_one()) {
      bars->abort_flag = 0;
      for (int s = 0; s < a.stages; ++s) { mbar_init(&bars->full[s], 1); mbar_init(&bars->empty[s], 1); }
      mbar_init(&bars->a_ready, S::kQuantWarps);
      mbar_init(&bars->acc_full, 1);
      fence_barrier_init();
      for (int i = 0; i < early; ++i) load_weights(i, i);
      if (S::kCodes) {
        mx_wait_for_previous();
        for (int i = 0; i < early; ++i) load_a(i, i);
      }
    }
    __syncwarp();
  }
  if (warp == 1) {
    tmem_alloc(&bars->tmem_base, 256);
    tmem_relinquish_alloc_permit();
  }
  tcgen05_fence_before_sync();
  __syncthreads();
  tcgen05_fence_after_sync();
  const uint32_t tmem = bars->tmem_base;  // sums, then scales
  bool ok = true;

  if (warp == 0) {
    int stage = early == a.stages ? 0 : early;
    uint32_t phase = 1;  // a stage is used again once its first use is done
    for (int i = early; i < count; ++i) {
      ok = __all_sync(0xffffffffu, mbar_wait(&bars->empty[stage], phase ^ 1u, abort_flag));
      if (!ok) break;
      if (elect_one()) {
        load_weights(stage, i);
        if (S::kCodes) load_a(stage, i);
      }
      __syncwarp();
      if (++stage == a.stages) { stage = 0; phase ^= 1u; }
    }
    if (!ok) {  // copies in flight land before the CTA leaves
      const long long t0 = clock64();
      while (clock64() - t0 < 2000000LL) {}
    }
  } else if (warp == 1) {
    int stage = 0;
    uint32_t phase = 0;
    if (!S::kCodes && count > 0) ok = __all_sync(0xffffffffu, mbar_wait(&bars->a_ready, 0, abort_flag));
    for (int i = 0; i < count && ok; ++i) {
      ok = __all_sync(0xffffffffu, mbar_wait(&bars->full[stage], phase, abort_flag));
      if (!ok) break;
      tcgen05_fence_after_sync();
      const uint32_t st = smem_u32(smem + stage * S::kStage);
      const uint32_t qa = S::kCodes ? st + kMxRowsWeights : smem_u32(a_codes + i * (NT * kMxRowBytes));
      const uint32_t qs = S::kCodes ? qa + NT * kMxRowBytes : smem_u32(a_scales + i * kMxScaleStage);
      const uint32_t t_sf = tmem + S::kSfBase + stage * 16;
      const uint64_t pd = mx_desc_codes(st), qd = mx_desc_codes(qa);
      if (elect_one()) {
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          mx_copy_scales(t_sf + g * 8, mx_desc_scales(st + kMxM * kMxRowBytes + g * kMxGroupBytes));
          mx_copy_scales(t_sf + g * 8 + 4, mx_desc_scales(qs + g * kMxGroupBytes));
        }
#pragma unroll
        for (int q = 0; q < 4; ++q)
          mx_umma(tmem, pd + q * 2, qd + q * 2, mx_idesc(kMxM, NT, (q & 1) * 2), t_sf + (q >> 1) * 8, t_sf + (q >> 1) * 8 + 4,
                  (i | q) != 0 ? 1u : 0u);
        umma_commit(&bars->empty[stage]);
        if (i == count - 1) umma_commit(&bars->acc_full);
      }
      __syncwarp();
      if (++stage == a.stages) { stage = 0; phase ^= 1u; }
    }
  } else if constexpr (!S::kCodes) {
    // A's rows, blocks of 32 elements: neighbouring threads take neighbouring blocks of a row. Rows from m to NT
    // keep whatever is there (their sums are not read); blocks behind k get a scale of 2^-127, as their weights have.
    const T* X = static_cast<const T*>(a.x) + b * a.stride_x;
    const int align = mx_row_alignment<T>(a.x, a.ldx, a.stride_x);
    const int per_row = count * (kMxStageK / kMxBlock);
    const int total = per_row * a.m;
    constexpr int kThreads = S::kQuantWarps * 32;
    constexpr int kBatch = sizeof(T) == 4 ? 1 : 2;  // blocks per thread whose loads are in flight together
    for (int i0 = static_cast<int>(threadIdx.x) - 64; i0 < total; i0 += kThreads * kBatch) {
      MxRaw<T> x[kBatch];
      int row[kBatch], blk[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const int i = i0 + j * kThreads;
        row[j] = i < total ? i / per_row : 0;
        blk[j] = i < total ? i - row[j] * per_row : 0;
        const int k0 = first * kMxStageK + blk[j] * kMxBlock;
        x[j].load(X + row[j] * a.ldx + k0, i < total ? min(max(a.k - k0, 0), kMxBlock) : 0, align);
      }
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        if (i0 + j * kThreads >= total) break;
        const bool real = first * kMxStageK + blk[j] * kMxBlock < a.k;
        const uint32_t E = real ? mx_scale_byte<4, T>(x[j].amax_bits()) : 0u;
        uint32_t c[4];
        mx_encode<4, T>(x[j], E, c);
        const int tile = blk[j] >> 3, piece = blk[j] & 7, r = row[j];
        *reinterpret_cast<uint4*>(a_codes + tile * (NT * kMxRowBytes) + r * kMxRowBytes + ((piece ^ (r & 7)) << 4)) =
            make_uint4(c[0], c[1], c[2], c[3]);
        a_scales[tile * kMxScaleStage + (piece >> 2) * kMxGroupBytes + mx_scale_at(r, piece & 3)] = static_cast<uint8_t>(E);
      }
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(&bars->a_ready);
  }

  // partial sums [NT][128] to shared memory, over the ring: every copy has landed and every MMA is done
  float* sums = reinterpret_cast<float*>(smem);
  if (warp >= 2 && warp < 6) {
    const uint32_t quarter = warp & 3u;
    const int col = static_cast<int>(quarter * 32 + lane);
    if (count > 0) ok = __all_sync(0xffffffffu, mbar_wait(&bars->acc_full, 0, abort_flag));
    if (ok) {
      tcgen05_fence_after_sync();
#pragma unroll 1
      for (int c = 0; c < NT && c < rows; c += 32) {
        uint32_t v[32];
        if (count > 0) {
          tmem_ld_32x32b_x32(tmem + ((quarter * 32u) << 16) + c, v);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = 0;
        }
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (c + j < NT) sums[(c + j) * 128 + col] = __uint_as_float(v[j]);
      }
    }
  }
  // Tensor memory goes back before anything waits for another CTA: several CTAs fit an SM, and one that
  // held columns here while its peer waited for columns elsewhere could close a circle.
  tcgen05_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tcgen05_fence_after_sync();
    tmem_dealloc(tmem, 256);
  }
  cluster_sync_all();
  const int failed = *abort_flag != 0;
  if (!failed) {
    // a warp per row of this CTA's share, four columns a lane (four rows at once measured slower by a microsecond:
    // more instructions to fetch outweigh the loads in flight)
    constexpr int kWarps = S::kThreads / 32;
    const int col = n0 + static_cast<int>(lane) * 4;
    const uint32_t at = smem_u32(sums) + lane * 16;
    const int size = a.out_type == 0 ? 4 : 2;
    const bool vec = a.align >= (a.out_type == 0 ? 16 : 8) && col + 4 <= a.n;
    for (int r = static_cast<int>(split) + a.splits * static_cast<int>(warp); r < rows; r += kWarps * a.splits) {
      float s[4] = {0.f, 0.f, 0.f, 0.f};
      for (int q0 = 0; q0 < a.splits; q0 += 4) {
        float4 v[4];
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (q0 + q < a.splits) v[q] = ld_cluster_f32x4(map_to_cta(at + r * 512, static_cast<uint32_t>(q0 + q)));
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (q0 + q < a.splits) { s[0] += v[q].x; s[1] += v[q].y; s[2] += v[q].z; s[3] += v[q].w; }
      }
      const long long to = b * a.stride_c + static_cast<long long>(m0 + r) * a.ldc + col;
      if (vec) {
        uint8_t* p = static_cast<uint8_t*>(a.C) + to * size;
        if (size == 4) *reinterpret_cast<float4*>(p) = make_float4(s[0], s[1], s[2], s[3]);
        else *reinterpret_cast<uint2*>(p) = make_uint2(mx_pack_out(a.out_type, s[0], s[1]), mx_pack_out(a.out_type, s[2], s[3]));
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) if (col + j < a.n) mx_store_one(a.C, a.out_type, to + j, s[j]);
      }
    }
  }
  cluster_leave();
  if (threadIdx.x == 0 && failed) atomicOr(&g_mx_status[0], 1u);
}

}  // namespace fbmm
