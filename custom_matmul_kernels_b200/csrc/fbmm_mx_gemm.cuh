// Product of two 4-bit microscaled operands on the block-scaled tensor cores:
//   C[b][m][n] = sum_k 2^(Ea + Eb - 254) a[m][k] b[n][k],  scales per 32 elements of k.
//
// tcgen05.mma.kind::mxf4.block_scale multiplies the 4-bit elements and applies both scales itself;
// products and scales are exact, the sum is kept in fp32 in tensor memory. A k-block of a stage is
// 256 elements: 128 bytes of codes per row (one 128-byte swizzle row, four MMAs of 64 elements) and
// two 512-byte groups of scales per 128 rows, which tcgen05.cp moves from shared to tensor memory
// in the order they are stored in (fbmm_mx_quant.cuh). The tensor-memory columns of the scales
// belong to the ring stage, so they are rewritten only after the commit that frees the stage.
// Elements behind k and groups of scales that do not exist are zero by the tensor maps' fill: they add
// nothing (a zero scale byte is 2^-127).
//
// Roles of a CTA: warp 0 issues the copies, warp 1 the scale copies and MMAs, warps 2-5 move
// accumulators to global memory. Two accumulator stages, persistent, one CTA per SM.
#pragma once
#include "fbmm_mx_quant.cuh"
#include "sm100_primitives.cuh"

namespace fbmm {

__device__ unsigned int g_mx_status[1];  // bit 0: a bounded wait ran out

constexpr int kMxM = 128;              // rows of the MMA's first operand per tile
constexpr int kMxStageK = 256;         // elements of k per ring stage
constexpr int kMxRowBytes = 128;       // their codes
constexpr int kMxScaleStage = 1024;    // scale bytes of 128 rows per stage (two groups)
constexpr uint32_t kMxSmemLimit = 227 * 1024;
constexpr int kMxMaxStages = 8;
constexpr int kMxThreads = 192;
constexpr int kMxEpiBytes = 4 * 4096;  // staging, 4 KB per epilogue warp

// p supplies the 128-row operand of the MMA, q the other one.
struct MxGemmArgs {
  void* C;
  long long ldc, stride_c;  // elements
  int l, k, p_rows, q_rows;
  int p_shared, q_shared, sp_shared, sq_shared;  // one matrix of codes / scales for every batch
  int out_type;  // 0 fp32, 1 fp16, 2 bf16
  int p_tiles, q_tiles;
  int align;     // bytes that C's rows are aligned to: 16, 8, 4 or 2
};

struct MxShape {
  static constexpr int BN = 128;
  static constexpr int kPBytes = kMxM * kMxRowBytes, kQBytes = BN * kMxRowBytes;
  static constexpr int kSfCols = 16;  // tensor-memory columns of a stage's scales
  static constexpr int kStageBytes = kPBytes + kQBytes + 2 * kMxScaleStage;
  static constexpr int kSfBase = 2 * BN;
  static constexpr int kFit = static_cast<int>((kMxSmemLimit - 1024 - 256 - kMxEpiBytes) / kStageBytes);
  static constexpr int kStages = kFit < kMxMaxStages ? kFit : kMxMaxStages;
  static constexpr int kSmem = 1024 + kStages * kStageBytes + kMxEpiBytes + 256;
  static_assert(kSfBase + kStages * kSfCols <= 512, "tensor memory");
};

struct MxBarriers {
  uint64_t full[kMxMaxStages], empty[kMxMaxStages], acc_full[2], acc_empty[2];
  uint32_t tmem_base, abort_flag;
};
static_assert(sizeof(MxBarriers) <= 256, "barrier block");

// Instruction descriptor of kind::mxf4 with one UE8M0 scale per 32 elements: A and B e2m1 (1 at bits
// 7 and 10), N >> 3 at 17, scale type UE8M0 at 23, M >> 4 at 24; bits 4 and 29 pick the pair of
// bytes (0 or 2) of the scale words that belongs to an MMA.
__host__ __device__ constexpr uint32_t mx_idesc(uint32_t m, uint32_t n, uint32_t sf) {
  return (sf << 4) | (1u << 7) | (1u << 10) | ((n >> 3) << 17) | (1u << 23) | ((m >> 4) << 24) | (sf << 29);
}
// K-major codes, 128-byte swizzle, 8-row groups 1024 bytes apart.
__device__ __forceinline__ uint64_t mx_desc_codes(uint32_t smem_addr) {
  return static_cast<uint64_t>((smem_addr >> 4) & 0x3fffu) | (static_cast<uint64_t>(1024 >> 4) << 32) |
         (static_cast<uint64_t>(1) << 46) | (static_cast<uint64_t>(2) << 61);
}
// A 512-byte group of scales, no swizzle: 32 rows of 16 bytes, 8-row groups 128 bytes apart.
__device__ __forceinline__ uint64_t mx_desc_scales(uint32_t smem_addr) {
  return static_cast<uint64_t>((smem_addr >> 4) & 0x3fffu) | (static_cast<uint64_t>(16 >> 4) << 16) |
         (static_cast<uint64_t>(128 >> 4) << 32) | (static_cast<uint64_t>(1) << 46);
}
__device__ __forceinline__ void mx_umma(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t sfa,
                                        uint32_t sfb, uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %6, 0;\n"
      "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n"
      "}\n"
      ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
      : "memory");
}
// 512 bytes of scales -> 4 columns of tensor memory, in all four lane quarters.
__device__ __forceinline__ void mx_copy_scales(uint32_t tmem, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
}
// One lane of the (converged) warp, always the same one. The loops that issue copies and MMAs run on the whole warp
// and only the issuing instructions are under this predicate: with the loop itself on one lane every tcgen05
// instruction took about 100 cycles to issue, which bound all three kernels (4-bit 8192^3 236 us, on the whole warp 183 us).
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n"
      ".reg .pred P;\n"
      "elect.sync _|P, 0xffffffff;\n"
      "selp.u32 %0, 1, 0, P;\n"
      "}\n"
      : "=r"(p));
  return p != 0;
}
__device__ __forceinline__ uint32_t warp_index() { return __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0); }

__device__ __forceinline__ uint32_t mx_pack_out(int out_type, float a, float b) {
  if (out_type == 2) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ void mx_store_one(void* C, int out_type, long long at, float v) {
  if (out_type == 0) static_cast<float*>(C)[at] = v;
  else if (out_type == 1) static_cast<__half*>(C)[at] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(C)[at] = __float2bfloat16_rn(v);
}

// Four neighbouring partial sums in the shared memory of a CTA of the cluster.
__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
// The last barrier of a cluster whose CTAs have read one another's shared memory: none goes while it is being read. Its
// release is one of shared memory only, since one that covers the results just stored would wait for them to land
// (about a microsecond).
__device__ __forceinline__ void cluster_leave() {
  asm volatile(
      "fence.release.sync_restrict::shared::cta.cluster;\n"
      "barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// 32 rows of a warp's accumulators (lane = row) -> row-major C, 128 bytes of every row at a time: 64 columns
// (v0, v1) of a 16-bit type, or 32 columns of fp32 in two calls. The lanes' 16-byte pieces cross the
// warp's staging area (piece index xor row, free of bank conflicts) so that every store instruction covers
// four whole 128-byte lines (16-bit results of 8192 x 8192 with k = 256: 68 us with 64-byte pieces of rows, 44 us
// with lines; a plain fill writes 3.9 TB/s). The staging area is read ahead of the stores, which the compiler must take
// for writes to it and would wait on (4-bit operands of that size: bf16 results 45 -> 35 us, fp32 results 73 -> 47 us;
// 16-bit operands 44 -> 41 us).
// Rows on 8-byte boundaries leave in pieces of that size (bf16 8192 x 4092, k = 1024: 62 -> 49 us), others by element (8192 x 4091: 54 us).
// `c0`: element (row 0, column 0) of the block.
template <typename Word>
__device__ __forceinline__ void mx_store_lines(uint8_t* stage, Word word, void* C, long long c0, long long ldc, int size,
                                               int rows, int cols, int align) {
  const int lane = static_cast<int>(lane_id());
  uint4* st = reinterpret_cast<uint4*>(stage);
  cols = min(cols, 128 / size);
  __syncwarp();
#pragma unroll
  for (int c = 0; c < 8; ++c) st[lane * 8 + (c ^ (lane & 7))] = word(c);
  __syncwarp();
  if (align == 16) {
    const int c = lane & 7, r0 = lane >> 3, left = cols * size - c * 16;  // left: bytes of the row from this piece on
    const int end = left > 0 ? min(rows, 32) : 0;
    uint8_t* at = static_cast<uint8_t*>(C) + (c0 + r0 * ldc) * size + c * 16;
    uint4 x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = r0 + 4 * i;
      x[i] = st[r * 8 + (c ^ (r & 7))];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i, at += 4 * ldc * size) {
      if (r0 + 4 * i >= end) break;
      if (left >= 16) {
        *reinterpret_cast<uint4*>(at) = x[i];
      } else {
        const uint32_t e[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
        for (int j = 0; j < 16 / size; ++j) {
          if (j * size >= left) break;
          if (size == 4) reinterpret_cast<uint32_t*>(at)[j] = e[j];
          else reinterpret_cast<uint16_t*>(at)[j] = static_cast<uint16_t>(e[j >> 1] >> (16 * (j & 1)));
        }
      }
    }
  } else if (align == 8) {  // two rows at a time in 8-byte pieces
    const int c = lane & 15, left = cols * size - c * 8;  // bytes of the row from this piece on
    const int end = left > 0 ? min(rows, 32) : 0;
    uint8_t* at = static_cast<uint8_t*>(C) + (c0 + (lane >> 4) * ldc) * size + c * 8;
#pragma unroll 1
    for (int r0 = lane >> 4; r0 < end; r0 += 8) {
      uint2 x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = r0 + 2 * i;
        x[i] = reinterpret_cast<const uint2*>(st + r * 8 + ((c >> 1) ^ (r & 7)))[c & 1];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i, at += 2 * ldc * size) {
        if (r0 + 2 * i >= end) break;
        if (left >= 8) {
          *reinterpret_cast<uint2*>(at) = x[i];
        } else {
          if (left >= 4) reinterpret_cast<uint32_t*>(at)[0] = x[i].x;
          if (size == 2 && (left & 2)) reinterpret_cast<uint16_t*>(at)[left >> 1 & 2] = static_cast<uint16_t>(left & 4 ? x[i].y : x[i].x);
        }
      }
    }
  } else {  // rows at any alignment: neighbouring lanes store neighbouring elements of one row (pairs of 16-bit
            // elements, where rows are 4-byte aligned, measured the same)
    const int end = min(rows, 32);
    uint8_t* row = static_cast<uint8_t*>(C) + (c0 + lane) * size;
#pragma unroll 1
    for (int r0 = 0; r0 < end; r0 += 8) {
      uint32_t x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = r0 + i;
        if (size == 4) {
          x[i] = reinterpret_cast<const uint32_t*>(st + r * 8 + ((lane >> 2) ^ (r & 7)))[lane & 3];
        } else {  // elements `lane` and 32 + lane
          const int p = lane >> 3, e = lane & 7;
          x[i] = reinterpret_cast<const uint16_t*>(st + r * 8 + (p ^ (r & 7)))[e] |
                 static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(st + r * 8 + ((4 + p) ^ (r & 7)))[e]) << 16;
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i, row += ldc * size) {
        if (r0 + i >= end) break;
        if (size == 4) {
          if (lane < cols) *reinterpret_cast<uint32_t*>(row) = x[i];
        } else {
          if (lane < cols) *reinterpret_cast<uint16_t*>(row) = static_cast<uint16_t>(x[i]);
          if (lane + 32 < cols) reinterpret_cast<uint16_t*>(row)[32] = static_cast<uint16_t>(x[i] >> 16);
        }
      }
    }
  }
}
__device__ __forceinline__ void mx_store_rows(uint8_t* stage, const uint32_t (&v0)[32], const uint32_t (&v1)[32], void* C,
                                              long long c0, long long ldc, int out_type, int rows, int cols, int align) {
  if (out_type == 0) {
    mx_store_lines(stage, [&](int c) { return make_uint4(v0[4 * c], v0[4 * c + 1], v0[4 * c + 2], v0[4 * c + 3]); }, C, c0,
                   ldc, 4, rows, cols, align);
    mx_store_lines(stage, [&](int c) { return make_uint4(v1[4 * c], v1[4 * c + 1], v1[4 * c + 2], v1[4 * c + 3]); }, C,
                   c0 + 32, ldc, 4, rows, cols - 32, align);
  } else {
    mx_store_lines(stage, [&](int c) {
      const uint32_t (&v)[32] = c < 4 ? v0 : v1;
      uint32_t p[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        p[j] = mx_pack_out(out_type, __uint_as_float(v[8 * (c & 3) + 2 * j]), __uint_as_float(v[8 * (c & 3) + 2 * j + 1]));
      return make_uint4(p[0], p[1], p[2], p[3]);
    }, C, c0, ldc, 2, rows, cols, align);
  }
}

// p = A, q = B; a 128 x 128 tile.
__global__ void __launch_bounds__(kMxThreads, 1)
mx_gemm_kernel(const __grid_constant__ CUtensorMap map_p, const __grid_constant__ CUtensorMap map_q,
               const __grid_constant__ CUtensorMap map_sp, const __grid_constant__ CUtensorMap map_sq, const MxGemmArgs a) {
  using S = MxShape;
  constexpr int BN = S::BN;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* epi = smem + S::kStages * S::kStageBytes;
  MxBarriers* bars = reinterpret_cast<MxBarriers*>(epi + kMxEpiBytes);
  volatile uint32_t* abort_flag = &bars->abort_flag;
  const uint32_t warp = warp_index(), lane = lane_id();
  if (threadIdx.x == 0) {
    bars->abort_flag = 0;
    for (int s = 0; s < S::kStages; ++s) { mbar_init(&bars->full[s], 1); mbar_init(&bars->empty[s], 1); }
    for (int s = 0; s < 2; ++s) { mbar_init(&bars->acc_full[s], 1); mbar_init(&bars->acc_empty[s], 4); }
    fence_barrier_init();
    tma_prefetch_desc(&map_p);
    tma_prefetch_desc(&map_q);
    tma_prefetch_desc(&map_sp);
    tma_prefetch_desc(&map_sq);
  }
  if (warp == 1) {
    tmem_alloc(&bars->tmem_base, 512);
    tmem_relinquish_alloc_permit();
  }
  tcgen05_fence_before_sync();
  __syncthreads();
  tcgen05_fence_after_sync();
  const uint32_t tmem = bars->tmem_base;

  const int kblocks = (a.k + kMxStageK - 1) / kMxStageK;
  const long long per_batch = static_cast<long long>(a.p_tiles) * a.q_tiles;
  const long long units = per_batch * a.l;
  auto decode = [&](long long u, int& b, int& pt, int& qt) {
    b = static_cast<int>(u / per_batch);
    const int r = static_cast<int>(u - b * per_batch);
    pt = r % a.p_tiles;
    qt = r / a.p_tiles;
  };

  if (warp == 0) {
    uint32_t stage = 0, phase = 0;
    bool ok = true;
    mx_wait_for_previous();
    for (long long u = blockIdx.x; u < units && ok; u += gridDim.x) {
      int b, pt, qt;
      decode(u, b, pt, qt);
      for (int kb = 0; kb < kblocks; ++kb) {
        ok = __all_sync(0xffffffffu, mbar_wait(&bars->empty[stage], phase ^ 1u, abort_flag));
        if (!ok) break;
        uint8_t* st = smem + stage * S::kStageBytes;
        uint8_t* sf = st + S::kPBytes + S::kQBytes;
        uint64_t* full = &bars->full[stage];
        if (elect_one()) {
          mbar_arrive_expect_tx(full, S::kStageBytes);
          tma_load_3d(st, &map_p, full, kb * kMxRowBytes, pt * kMxM, a.p_shared ? 0 : b, kL2EvictLast);
          tma_load_3d(st + S::kPBytes, &map_q, full, kb * kMxRowBytes, qt * BN, a.q_shared ? 0 : b, kL2EvictLast);
          tma_load_3d(sf, &map_sp, full, kb * (kMxScaleStage / 4), pt, a.sp_shared ? 0 : b, kL2EvictLast);
          tma_load_3d(sf + kMxScaleStage, &map_sq, full, kb * (kMxScaleStage / 4), qt * BN / 128, a.sq_shared ? 0 : b,
                      kL2EvictLast);
        }
        __syncwarp();
        if (++stage == S::kStages) { stage = 0; phase ^= 1u; }
      }
    }
    if (!ok) {  // copies in flight land before the CTA leaves
      const long long t0 = clock64();
      while (clock64() - t0 < 2000000LL) {}
    }
  } else if (warp == 1) {
    uint32_t stage = 0, phase = 0, acc = 0, acc_phase = 0;
    bool ok = true;
    for (long long u = blockIdx.x; u < units && ok; u += gridDim.x) {
      ok = __all_sync(0xffffffffu, mbar_wait(&bars->acc_empty[acc], acc_phase ^ 1u, abort_flag));
      if (!ok) break;
      const uint32_t d = tmem + acc * BN;
      for (int kb = 0; kb < kblocks; ++kb) {
        ok = __all_sync(0xffffffffu, mbar_wait(&bars->full[stage], phase, abort_flag));
        if (!ok) break;
        tcgen05_fence_after_sync();
        const uint32_t st = smem_u32(smem + stage * S::kStageBytes);
        const uint32_t sf = st + S::kPBytes + S::kQBytes;
        const uint32_t t_sf = tmem + S::kSfBase + stage * S::kSfCols;  // per group of k: 4 columns of p, then q's
        const uint64_t pd = mx_desc_codes(st), qd = mx_desc_codes(st + S::kPBytes);
        if (elect_one()) {
#pragma unroll
          for (int g = 0; g < 2; ++g)
            mx_copy_scales(t_sf + g * 8, mx_desc_scales(sf + g * kMxGroupBytes)),
            mx_copy_scales(t_sf + g * 8 + 4, mx_desc_scales(sf + kMxScaleStage + g * kMxGroupBytes));
#pragma unroll
          for (int q = 0; q < 4; ++q)
            mx_umma(d, pd + q * 2, qd + q * 2, mx_idesc(kMxM, BN, (q & 1) * 2), t_sf + (q >> 1) * 8, t_sf + (q >> 1) * 8 + 4,
                    (kb | q) != 0 ? 1u : 0u);
          umma_commit(&bars->empty[stage]);
          if (kb == kblocks - 1) umma_commit(&bars->acc_full[acc]);
        }
        __syncwarp();
        if (++stage == S::kStages) { stage = 0; phase ^= 1u; }
      }
      if (++acc == 2) { acc = 0; acc_phase ^= 1u; }
    }
  } else {
    const uint32_t quarter = warp & 3u;
    uint8_t* stage_mem = epi + (warp - 2) * 4096;
    uint32_t acc = 0, acc_phase = 0;
    bool ok = true;
    for (long long u = blockIdx.x; u < units && ok; u += gridDim.x) {
      int b, pt, qt;
      decode(u, b, pt, qt);
      ok = mbar_wait(&bars->acc_full[acc], acc_phase, abort_flag);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tcgen05_fence_after_sync();
      const uint32_t t = tmem + acc * BN + ((quarter * 32u) << 16);
      const int p0 = pt * kMxM + static_cast<int>(quarter) * 32;
      bool held = true;  // released with the last load, before the stores behind it
      auto release = [&]() {
        tcgen05_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->acc_empty[acc]);
        held = false;
      };
#pragma unroll 1
      for (int c = 0; c < BN; c += 64) {
        const int q0 = qt * BN + c;
        if (q0 >= a.q_rows || p0 >= a.p_rows) break;  // warp-uniform
        uint32_t v0[32], v1[32];
        tmem_ld_32x32b_x32(t + c, v0);
        tmem_ld_32x32b_x32(t + c + 32, v1);
        tmem_ld_wait();
        if (c + 64 >= BN || q0 + 64 >= a.q_rows) release();
        mx_store_rows(stage_mem, v0, v1, a.C, b * a.stride_c + static_cast<long long>(p0) * a.ldc + q0, a.ldc, a.out_type,
                      a.p_rows - p0, a.q_rows - q0, a.align);
      }
      if (held) release();
      if (++acc == 2) { acc = 0; acc_phase ^= 1u; }
    }
  }
  tcgen05_fence_before_sync();
  __syncthreads();
  if (threadIdx.x == 0 && *abort_flag != 0) atomicOr(&g_mx_status[0], 1u);
  if (warp == 1) {
    tcgen05_fence_after_sync();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace fbmm
