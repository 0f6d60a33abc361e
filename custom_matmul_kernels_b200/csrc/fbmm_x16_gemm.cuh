// 16-bit products for training: D[b][x][y] = sum_j X[b][x][j] * Y[b][y][j] with fp32 sums, each
// operand fp16 / bf16 in either storage order, or one of them microscaled (fbmm_mx_quant.cuh) with
// its blocks along its own output axis. The forward pass, the gradient of the activations
// and the gradient of the weights from 8-bit activations are this one product in three layouts:
//   C  = A B        X = A [m][k]        j contiguous     Y = B [k][n]   y contiguous (or B^T stored: j)
//   dA = dC B^T     X = dC [m][n]       j contiguous     Y = B [k][n]   j contiguous
//   dB = A8^T dC    X = A8 [m][k]       microscaled      Y = dC [m][n]  y contiguous
//   dA = dC W4      X = dC              j contiguous     Y = W4 [n][k]  microscaled
//
// tcgen05.mma.kind::f16 takes both K-major and MN-major tiles, so no operand is transposed in memory.
// Microscaled codes arrive raw by TMA (8 KB or 4 KB per stage, half or a quarter of what the
// 16-bit values would take out of L2) with their 512-byte group of scales; four warps turn them into
// 16-bit values (code * 2^(E-127), rounded to the type: exact for bf16) in the MN-major
// swizzled tile that the MMA reads. A dequantised copy of the operand never exists in memory.
//
// PAIR: two CTAs (cta_group::2) share a 256 x 256 tile, each supplying 128 rows of X and 128 of Y
// from its own shared memory, so per 64 elements of j a CTA fetches 32 KB for 512 cycles of MMA;
// without it a CTA does a 128 x 128 tile (the same 32 KB for 256 cycles), for products with few tiles.
//
// SPLIT (single CTAs): few tiles and a long j, as where one side of a weight is narrow. A cluster of CTAs shares a
// tile's j; the partial sums meet in shared memory and every CTA adds up and stores its share of the rows, in
// rank order. 8-bit dB of 4096 x 64 over 8192: 18 us on 128 CTAs against 46 on 32.
//
// Roles of a CTA: warp 0 copies, warp 1 (the even CTA's) MMAs, four warps for codes where an operand
// is microscaled, four warps for the epilogue. Two accumulator stages, persistent.
#pragma once
#include "fbmm_mx_gemm.cuh"

namespace fbmm {

enum X16Kind { kX16K = 0, kX16MN = 1, kX16Mx4 = 2, kX16Mx8 = 3 };

constexpr int kX16J = 64;                   // j per stage: 128 bytes of a K-major row
constexpr int kX16Part = 128 * kX16J * 2;   // 16 KB: 128 rows of one operand
constexpr int kX16Stages = 5;
constexpr int kX16Expanders = 3;            // groups of four warps that expand codes, in turn
static_assert(kX16Expanders <= kX16Stages, "a group's stages must not be further apart than the ring");
constexpr int kX16Chunk = 64 * kX16J * 2;   // MN-major: 64 rows x 64 j

struct X16Operand {
  const uint8_t* scales;   // microscaled: groups [j / 128][rows / 128][512]
  long long scale_stride;  // bytes, 0 = shared
  int rows;
  int shared;              // one matrix of elements or codes for every batch; the scales have a stride of their own
};

struct X16Args {
  X16Operand x, y;
  void* C;
  long long ldc, stride_c;
  int l, J;
  int dtype;     // 1 fp16, 2 bf16
  int x_tiles, y_tiles;
  int align;  // as MxGemmArgs
  int splits, blocks_per_split;  // SPLIT: CTAs per tile, stages of j each
};

template <int XK, int YK>
struct X16Shape {
  static constexpr bool kMx = XK >= kX16Mx4 || YK >= kX16Mx4;
  static constexpr int kBits = (XK == kX16Mx4 || YK == kX16Mx4) ? 4 : 8;
  static constexpr int kRaw = kMx ? kX16J * 128 * kBits / 8 + kMxGroupBytes : 0;
  static constexpr int kStageBytes = 2 * kX16Part + (kMx ? (kRaw + 1023) / 1024 * 1024 : 0);
  static constexpr int kSmem = 1024 + kX16Stages * kStageBytes + kMxEpiBytes + 256;
  static_assert(kSmem <= static_cast<int>(kMxSmemLimit), "shared memory");
  static constexpr int kEpiWarp = kMx ? 2 + 4 * kX16Expanders : 2;
  static constexpr int kThreads = (kEpiWarp + 4) * 32;
};

struct X16Barriers {
  uint64_t full[kX16Stages], raw[kX16Stages], empty[kX16Stages], acc_full[2], acc_empty[2];
  uint32_t tmem_base, abort_flag;
};
static_assert(sizeof(X16Barriers) <= 256, "barrier block");

__device__ __forceinline__ void umma_f16_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                              uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n"
      "}\n"
      ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Untiled copy of `bytes` (a multiple of 16, both addresses 16-byte aligned) into shared memory.
__device__ __forceinline__ void mx_bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// Shared-memory descriptor of a 128-row part with the 128-byte swizzle. K-major: 8-row groups 1024
// bytes apart, an MMA step (16 j) is 32 bytes. MN-major: chunks of 64 rows kX16Chunk apart, 8-j groups 1024 bytes
// apart, an MMA step is 2048 bytes.
__device__ __forceinline__ uint64_t x16_desc(uint32_t smem_addr, bool mn_major) {
  const uint64_t lbo = mn_major ? kX16Chunk : 16;
  return static_cast<uint64_t>((smem_addr >> 4) & 0x3fffu) | ((lbo >> 4) << 16) | (static_cast<uint64_t>(1024 >> 4) << 32) |
         (static_cast<uint64_t>(1) << 46) | (static_cast<uint64_t>(2) << 61);
}

// Reports to the pair's issuing CTA, by cluster-window address, that this warp's values lie in its own CTA's shared
// memory (behind their proxy fence), or that the warp has read its accumulators. A release at cluster scope, as two CTAs
// are ordered by nothing less, but of shared memory only: one that covers global memory too took each warp about
// 1400 cycles beside 16 writing warps, twice the expansion (8-bit gradient of weights at 4096^3: 145 us against
// 110 us). Passing the reports on through one warp of the CTA measured the same as this.
__device__ __forceinline__ void mbar_arrive_values(uint32_t cluster_addr) {
  asm volatile(
      "fence.release.sync_restrict::shared::cta.cluster;\n"
      "mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];"
      ::"r"(cluster_addr)
      : "memory");
}

// A stage's raw codes -> 16-bit values in MN-major order; 128 threads, 16 codes of a row of 128 at a time.
// Eight neighbouring lanes take 64 codes of rows j and j ^ 5: with the 128-byte swizzle on the raw
// 8-bit rows (4-bit rows are 64 bytes and need none) and on the values, neither their reads nor
// their writes share a bank. Rows behind the last j are zero codes whose scale bytes may be anything.
template <int BITS, bool BF16>
__device__ __forceinline__ void x16_expand(const uint8_t* raw, uint8_t* dst, int j0, int j_end, int tid) {
  const uint8_t* sc = raw + kX16J * 128 * BITS / 8;
  const int half = (tid >> 3) & 1;             // which 64 of the row
  const int u = half * 4 + (tid & 3);          // 16-code piece of the row
  const int base = (tid >> 4) & 3, flip = (tid & 4) ? 5 : 0;
  uint32_t c[4][BITS / 2], E[4];
  bool in_range = true;
  uint32_t nan = 0;
#pragma unroll
  for (int it = 0; it < 4; ++it) {
    const int j = (((tid >> 6) * 4 + it) << 3) | (base ^ flip);
    if (BITS == 8) {
      const uint4 v = *reinterpret_cast<const uint4*>(raw + j * 128 + ((u ^ (j & 7)) << 4));
      c[it][0] = v.x; c[it][1] = v.y; c[it][BITS / 2 - 2] = v.z; c[it][BITS / 2 - 1] = v.w;
    } else {
      const uint2 v = *reinterpret_cast<const uint2*>(raw + j * 64 + u * 8);
      c[it][0] = v.x; c[it][1] = v.y;
    }
    E[it] = sc[mx_scale_at((j0 + j) & 127, u >> 1)];
    if (j0 + j >= j_end) E[it] = 127;
    in_range = in_range && MxFast<BITS, BF16>::in_range(E[it]);
    nan |= mx_nan_codes<BITS>(c[it]);
  }
  const bool fast = __all_sync(0xffffffffu, in_range && nan == 0);
  auto expand = [&](bool quick) {
#pragma unroll
    for (int it = 0; it < 4; ++it) {
      const int j = (((tid >> 6) * 4 + it) << 3) | (base ^ flip);
      uint32_t w[8];
      mx_values16<BITS, BF16>(c[it], E[it], quick, w);
      uint8_t* row = dst + half * kX16Chunk + j * 128;
      const int unit = ((u & 3) * 2) ^ (j & 7);
      *reinterpret_cast<uint4*>(row + unit * 16) = make_uint4(w[0], w[1], w[2], w[3]);
      *reinterpret_cast<uint4*>(row + (unit ^ 1) * 16) = make_uint4(w[4], w[5], w[6], w[7]);
    }
  };
  if (fast) expand(true); else expand(false);
}

// Tiles in bands of 8 along x, so that the tiles in flight share few rows of either operand (bands of 4 and
// 16 and a sixth stage measured the same at 8192 x 4096 x 4096, where the power cap sets the clock).
__device__ __forceinline__ void x16_decode(long long u, int x_tiles, int y_tiles, int& b, int& xt, int& yt) {
  const long long per_batch = static_cast<long long>(x_tiles) * y_tiles;
  b = static_cast<int>(u / per_batch);
  const int r = static_cast<int>(u - b * per_batch);
  const int band = r / (8 * y_tiles);
  const int in = r - band * 8 * y_tiles;
  const int height = min(8, x_tiles - band * 8);
  yt = in / height;
  xt = band * 8 + in - yt * height;
}

template <int XK, int YK, bool PAIR, bool SPLIT>
__global__ void __launch_bounds__(X16Shape<XK, YK>::kThreads, 1)
x16_gemm_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_y, const X16Args a) {
  static_assert(!(PAIR && SPLIT), "a split tile belongs to single CTAs");
  using S = X16Shape<XK, YK>;
  constexpr int kCtas = PAIR ? 2 : 1;
  constexpr int kTile = 128 * kCtas;
  constexpr uint32_t kDense = (XK < kX16Mx4 ? kX16Part : 0) + (YK < kX16Mx4 ? kX16Part : 0);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* epi = smem + kX16Stages * S::kStageBytes;
  X16Barriers* bars = reinterpret_cast<X16Barriers*>(epi + kMxEpiBytes);
  volatile uint32_t* abort_flag = &bars->abort_flag;
  const uint32_t warp = warp_index(), lane = lane_id();
  const uint32_t rank = PAIR ? cluster_cta_rank() : 0u;
  if (threadIdx.x == 0) {
    bars->abort_flag = 0;
    for (int s = 0; s < kX16Stages; ++s) {
      mbar_init(&bars->full[s], 1 + (S::kMx ? 4 * kCtas : 0));  // the copies, and the expanders' warps
      mbar_init(&bars->raw[s], 1);
      mbar_init(&bars->empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) { mbar_init(&bars->acc_full[s], 1); mbar_init(&bars->acc_empty[s], 4 * kCtas); }
    fence_barrier_init();
    tma_prefetch_desc(&map_x);
    tma_prefetch_desc(&map_y);
  }
  if (warp == 1) {
    if (PAIR) { tmem_alloc_pair(&bars->tmem_base, 512); tmem_relinquish_alloc_permit_pair(); }
    else { tmem_alloc(&bars->tmem_base, 512); tmem_relinquish_alloc_permit(); }
  }
  tcgen05_fence_before_sync();
  if (PAIR) cluster_sync_all(); else __syncthreads();
  tcgen05_fence_after_sync();
  const uint32_t tmem = bars->tmem_base;
  const uint32_t bars0 = PAIR ? map_to_cta(smem_u32(bars), 0) : smem_u32(bars);
  const uint32_t bars1 = PAIR ? map_to_cta(smem_u32(bars), 1) : smem_u32(bars);
  auto off = [&](const uint64_t* b) -> uint32_t { return smem_u32(b) - smem_u32(bars); };
  auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
    return PAIR ? mbar_wait_cluster(bar, parity, abort_flag) : mbar_wait(bar, parity, abort_flag);
  };
  auto commit = [&](uint64_t* bar) {
    if (PAIR) { umma_commit_pair(bars0 + off(bar)); umma_commit_pair(bars1 + off(bar)); }
    else umma_commit(bar);
  };

  const long long units = static_cast<long long>(a.x_tiles) * a.y_tiles * a.l;
  const uint32_t split = SPLIT ? cluster_cta_rank() : 0u;
  const long long u0 = PAIR ? blockIdx.x >> 1 : SPLIT ? blockIdx.x / static_cast<uint32_t>(a.splits) : blockIdx.x;
  const long long du = PAIR ? gridDim.x >> 1 : SPLIT ? units : gridDim.x;
  // stages of j that this CTA sums: all, or its range (which may be empty)
  const int all_blocks = (a.J + kX16J - 1) / kX16J;
  const int jb0 = SPLIT ? min(all_blocks, static_cast<int>(split) * a.blocks_per_split) : 0;
  const int jb1 = SPLIT ? min(all_blocks, jb0 + a.blocks_per_split) : all_blocks;

  if (warp == 0) {
    {
      uint32_t stage = 0, phase = 0;
      bool ok = true;
      mx_wait_for_previous();
      // 128 rows of one operand, from row r0: to the part's place, or its raw codes
      auto load = [&](const CUtensorMap* map, int kind, uint8_t* part, uint8_t* raw, int j0, int r0, int b,
                      const X16Operand& op) {
        const int mb = op.shared ? 0 : b;  // of the elements or codes
        uint64_t* full = &bars->full[stage];
        if (kind == kX16K) {
          if (PAIR) tma_load_3d_pair(part, map, bars0 + off(full), j0, r0, mb, kL2EvictLast);
          else tma_load_3d(part, map, full, j0, r0, mb, kL2EvictLast);
        } else if (kind == kX16MN) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            if (PAIR) tma_load_3d_pair(part + c * kX16Chunk, map, bars0 + off(full), r0 + c * 64, j0, mb, kL2EvictLast);
            else tma_load_3d(part + c * kX16Chunk, map, full, r0 + c * 64, j0, mb, kL2EvictLast);
          }
        } else {
          const int bytes = kX16J * 128 * S::kBits / 8;
          const int groups = (op.rows + 127) / 128;
          const bool exists = r0 < op.rows;
          mbar_arrive_expect_tx(&bars->raw[stage], bytes + (exists ? kMxGroupBytes : 0));
          tma_load_3d(raw, map, &bars->raw[stage], r0 / (8 / S::kBits), j0, mb, kL2EvictLast);
          if (exists)
            mx_bulk_load(raw + bytes,
                         op.scales + b * op.scale_stride +
                             (static_cast<long long>(j0 / 128) * groups + r0 / 128) * kMxGroupBytes,
                         kMxGroupBytes, &bars->raw[stage]);
        }
      };
      for (long long u = u0; u < units && ok; u += du) {
        int b, xt, yt;
        x16_decode(u, a.x_tiles, a.y_tiles, b, xt, yt);
        const int xr = xt * kTile + static_cast<int>(rank) * 128, yr = yt * kTile + static_cast<int>(rank) * 128;
        for (int jb = jb0; jb < jb1; ++jb) {
          ok = __all_sync(0xffffffffu, wait(&bars->empty[stage], phase ^ 1u));
          if (!ok) break;
          uint8_t* st = smem + stage * S::kStageBytes;
          if (elect_one()) {
            if (rank == 0) mbar_arrive_expect_tx(&bars->full[stage], kDense * kCtas);
            load(&map_x, XK, st, st + 2 * kX16Part, jb * kX16J, xr, b, a.x);
            load(&map_y, YK, st + kX16Part, st + 2 * kX16Part, jb * kX16J, yr, b, a.y);
          }
          __syncwarp();
          if (++stage == kX16Stages) { stage = 0; phase ^= 1u; }
        }
      }
      if (!ok) {  // copies in flight land before the CTA leaves
        const long long t0 = clock64();
        while (clock64() - t0 < 2000000LL) {}
      }
    }
  } else if (warp == 1) {
    if (rank == 0) {
      uint32_t stage = 0, phase = 0, acc = 0, acc_phase = 0;
      bool ok = true;
      constexpr bool kXmn = XK != kX16K, kYmn = YK != kX16K;
      const uint32_t idesc = make_idesc_f16(kTile, kTile, a.dtype == 2) | (kXmn ? 1u << 15 : 0u) | (kYmn ? 1u << 16 : 0u);
      for (long long u = u0; u < units && ok; u += du) {
        ok = __all_sync(0xffffffffu, wait(&bars->acc_empty[acc], acc_phase ^ 1u));
        if (!ok) break;
        const uint32_t d = tmem + acc * 256;
        for (int jb = jb0; jb < jb1; ++jb) {
          ok = __all_sync(0xffffffffu, wait(&bars->full[stage], phase));
          if (!ok) break;
          tcgen05_fence_after_sync();
          const uint32_t st = smem_u32(smem + stage * S::kStageBytes);
          const uint64_t xd = x16_desc(st, kXmn), yd = x16_desc(st + kX16Part, kYmn);
          if (elect_one()) {
#pragma unroll
            for (int q = 0; q < kX16J / 16; ++q) {
              const uint64_t xs = xd + q * ((kXmn ? 2048 : 32) >> 4), ys = yd + q * ((kYmn ? 2048 : 32) >> 4);
              if (PAIR) umma_f16_pair(d, xs, ys, idesc, (jb != jb0 || q != 0) ? 1u : 0u);
              else umma_f16(d, xs, ys, idesc, (jb != jb0 || q != 0) ? 1u : 0u);
            }
            commit(&bars->empty[stage]);
            if (jb == jb1 - 1) commit(&bars->acc_full[acc]);
          }
          __syncwarp();
          if (++stage == kX16Stages) { stage = 0; phase ^= 1u; }
        }
        if (++acc == 2) { acc = 0; acc_phase ^= 1u; }
      }
    }
  } else if (S::kMx && warp < S::kEpiWarp) {
    uint32_t stage = 0, phase = 0;
    bool ok = true;
    const int tid = static_cast<int>(threadIdx.x - 64) & 127;
    int turn = static_cast<int>(warp - 2) >> 2;  // stages until this group's next one
    for (long long u = u0; u < units && ok; u += du)
      for (int jb = jb0; jb < jb1; ++jb) {
        if (turn != 0) {
          --turn;
          if (++stage == kX16Stages) { stage = 0; phase ^= 1u; }
          continue;
        }
        turn = kX16Expanders - 1;
        // First the stage's release by its last use, as the copies wait for it. Copies land out of order, and the last
        // use was another group's: with the codes' barrier alone a group could come a round early and take
        // the phase before the unfinished one for the one it wants. (The release itself is never a round behind: this
        // group's last stage was loaded, so the MMAs eight stages back, and all before them, are done.)
        ok = wait(&bars->empty[stage], phase ^ 1u) && mbar_wait(&bars->raw[stage], phase, abort_flag);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        uint8_t* st = smem + stage * S::kStageBytes;
        uint8_t* dst = st + (XK >= kX16Mx4 ? 0 : kX16Part);
        if (a.dtype == 2) x16_expand<S::kBits, true>(st + 2 * kX16Part, dst, jb * kX16J, a.J, tid);
        else x16_expand<S::kBits, false>(st + 2 * kX16Part, dst, jb * kX16J, a.J, tid);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive_values(bars0 + off(&bars->full[stage]));
        if (++stage == kX16Stages) { stage = 0; phase ^= 1u; }
      }
  } else {
    const uint32_t quarter = warp & 3u;
    uint8_t* stage_mem = epi + (warp - S::kEpiWarp) * 4096;
    uint32_t acc = 0, acc_phase = 0;
    bool ok = true;
    for (long long u = u0; u < units && ok; u += du) {
      int b, xt, yt;
      x16_decode(u, a.x_tiles, a.y_tiles, b, xt, yt);
      if (!SPLIT || jb1 > jb0) ok = __all_sync(0xffffffffu, wait(&bars->acc_full[acc], acc_phase));
      if (!ok) break;
      tcgen05_fence_after_sync();
      const uint32_t t = tmem + acc * 256 + ((quarter * 32u) << 16);
      if (SPLIT) {
        // partial sums [row][column] over the ring (every copy has landed and every MMA is done), 16-byte
        // pieces of a row xor its number: lanes write and read them on different banks
        const int r = static_cast<int>(quarter * 32 + lane);
        float4* sums = reinterpret_cast<float4*>(smem) + r * 32;
#pragma unroll 1
        for (int c = 0; c < 128; c += 32) {
          uint32_t v[32];
          if (jb1 > jb0) {
            tmem_ld_32x32b_x32(t + c, v);
            tmem_ld_wait();
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = 0;
          }
#pragma unroll
          for (int j = 0; j < 8; ++j)
            sums[(c / 4 + j) ^ (r & 31)] = make_float4(__uint_as_float(v[4 * j]), __uint_as_float(v[4 * j + 1]),
                                                       __uint_as_float(v[4 * j + 2]), __uint_as_float(v[4 * j + 3]));
        }
        break;
      }
      const int x0 = xt * kTile + static_cast<int>(rank) * 128 + static_cast<int>(quarter) * 32;
      bool held = true;  // released with the last load, before the stores behind it
      auto release = [&]() {
        tcgen05_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive_values(bars0 + off(&bars->acc_empty[acc]));
        held = false;
      };
#pragma unroll 1
      for (int c = 0; c < kTile; c += 64) {
        const int y0 = yt * kTile + c;
        if (y0 >= a.y.rows || x0 >= a.x.rows) break;  // warp-uniform
        uint32_t v0[32], v1[32];
        tmem_ld_32x32b_x32(t + c, v0);
        tmem_ld_32x32b_x32(t + c + 32, v1);
        tmem_ld_wait();
        if (c + 64 >= kTile || y0 + 64 >= a.y.rows) release();
        mx_store_lines(stage_mem, [&](int i) {
          const uint32_t (&v)[32] = i < 4 ? v0 : v1;
          uint32_t p[4];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            p[j] = mx_pack_out(a.dtype, __uint_as_float(v[8 * (i & 3) + 2 * j]), __uint_as_float(v[8 * (i & 3) + 2 * j + 1]));
          return make_uint4(p[0], p[1], p[2], p[3]);
        }, a.C, b * a.stride_c + static_cast<long long>(x0) * a.ldc + y0, a.ldc, 2, a.x.rows - x0, a.y.rows - y0,
                       a.align);
      }
      if (held) release();
      if (++acc == 2) { acc = 0; acc_phase ^= 1u; }
    }
  }
  tcgen05_fence_before_sync();
  if (PAIR) cluster_sync_all(); else __syncthreads();
  const bool failed = *abort_flag != 0;
  if (threadIdx.x == 0 && failed) atomicOr(&g_mx_status[0], 1u);
  if (warp == 1) {
    tcgen05_fence_after_sync();
    if (PAIR) tmem_dealloc_pair(tmem, 512); else tmem_dealloc(tmem, 512);
  }
  if (SPLIT) {
    cluster_sync_all();
    if (!failed) {
      int b, xt, yt;
      x16_decode(u0, a.x_tiles, a.y_tiles, b, xt, yt);
      const int rows = min(128, a.x.rows - xt * 128), col = yt * 128 + static_cast<int>(lane) * 4;
      const bool vec = a.align >= 8 && col + 4 <= a.y.rows;
      const uint32_t base = smem_u32(smem);
      for (int r = static_cast<int>(split) + a.splits * static_cast<int>(warp); r < rows; r += (S::kThreads / 32) * a.splits) {
        const uint32_t at = base + static_cast<uint32_t>(r) * 512 + ((lane ^ (static_cast<uint32_t>(r) & 31u)) << 4);
        float s[4] = {0.f, 0.f, 0.f, 0.f};
        for (int q0 = 0; q0 < a.splits; q0 += 4) {
          float4 v[4];
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (q0 + q < a.splits) v[q] = ld_cluster_f32x4(map_to_cta(at, static_cast<uint32_t>(q0 + q)));
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (q0 + q < a.splits) { s[0] += v[q].x; s[1] += v[q].y; s[2] += v[q].z; s[3] += v[q].w; }
        }
        const long long to = b * a.stride_c + static_cast<long long>(xt * 128 + r) * a.ldc + col;
        if (vec) {
          *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.C) + to) =
              make_uint2(mx_pack_out(a.dtype, s[0], s[1]), mx_pack_out(a.dtype, s[2], s[3]));
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) if (col + j < a.y.rows) mx_store_one(a.C, a.dtype, to + j, s[j]);
        }
      }
    }
    cluster_leave();
  }
}

// Rows of `cols` 16-bit elements at any alignment -> rows padded to `pitch` (a multiple of 8) elements, zeros in the
// padding: what the tensor maps of operands with odd pitches or bases are made over. Eight elements a thread, by the
// widest loads (`align` bytes, 2 to 16) that every row allows. One launch serves both operands of a product: the
// first `blocks` blocks take p, the others q.
struct X16Repack {
  const uint16_t* src;
  long long ld, stride;
  uint16_t* dst;
  int rows, cols, pitch, align;
  long long pieces;
};

__global__ void __launch_bounds__(256) x16_repack_kernel(const X16Repack p, const X16Repack q, const unsigned blocks) {
  mx_let_next_start();
  mx_wait_for_previous();
  const bool first = blockIdx.x < blocks;
  const X16Repack s = first ? p : q;
  const int per_row = s.pitch / 8;
  const long long step = static_cast<long long>(first ? blocks : gridDim.x - blocks) * 256;
  for (long long i = static_cast<long long>(first ? blockIdx.x : blockIdx.x - blocks) * 256 + threadIdx.x; i < s.pieces; i += step) {
    // over all batches; in 32 bits where they suffice
    const long long row = s.pieces <= 0x7fffffff ? static_cast<unsigned>(i) / static_cast<unsigned>(per_row) : i / per_row;
    const int c = static_cast<int>(i - row * per_row) * 8;
    const long long b = s.pieces <= 0x7fffffff ? static_cast<unsigned>(row) / static_cast<unsigned>(s.rows) : row / s.rows;
    const uint16_t* from = s.src + b * s.stride + (row - b * s.rows) * s.ld + c;
    uint32_t w[4];
    if (s.align >= 8 && c + 8 <= s.cols) {
      const uint2 lo = __ldg(reinterpret_cast<const uint2*>(from)), hi = __ldg(reinterpret_cast<const uint2*>(from) + 1);
      w[0] = lo.x; w[1] = lo.y; w[2] = hi.x; w[3] = hi.y;
    } else if (s.align >= 4 && c + 8 <= s.cols) {
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = __ldg(reinterpret_cast<const uint32_t*>(from) + j);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t lo = c + 2 * j < s.cols ? __ldg(from + 2 * j) : 0u, hi = c + 2 * j + 1 < s.cols ? __ldg(from + 2 * j + 1) : 0u;
        w[j] = lo | (hi << 16);
      }
    }
    *reinterpret_cast<uint4*>(s.dst + i * 8) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

}  // namespace fbmm
