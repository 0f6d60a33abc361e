// Host side of the microscaled entry points: quantisation, its inverse and the 4-bit product.
#include <algorithm>
#include <atomic>
#include <cstdint>

#include "../../include/fbmm.h"
#include "fbmm_host.h"
#include "fbmm_mx_gemm.cuh"
#include "fbmm_mx_quant.cuh"
#include "fbmm_mx_rows.cuh"
#include "fbmm_mx_pair.cuh"
#include "fbmm_x16_gemm.cuh"

namespace {

using namespace fbmm;
using fbmm_host::fail;

int check_shape(int l, int rows, int k) {
  if (l <= 0 || rows <= 0 || k <= 0) return fail(FBMM_ERR_INVALID, "l, rows, k must be positive, got %d %d %d", l, rows, k);
  // extents that tile arithmetic can round up, and scale groups that a grid can count
  if (k > (1 << 29) || rows > 0x7fffff00) return fail(FBMM_ERR_INVALID, "matrix of %d x %d is too large", rows, k);
  const long long groups = static_cast<long long>((rows + 127) / 128) * ((k + 127) / 128);
  if (groups > 0x7fffffffLL / l) return fail(FBMM_ERR_INVALID, "matrix of %d x %d x %d is too large", l, rows, k);
  return FBMM_OK;
}

int check_bits(int bits) {
  if (bits != 4 && bits != 8) return fail(FBMM_ERR_INVALID, "bits must be 4 or 8, got %d", bits);
  return FBMM_OK;
}

int check_type(int dtype) {
  if (dtype != FBMM_F32 && dtype != FBMM_F16 && dtype != FBMM_BF16)
    return fail(FBMM_ERR_INVALID, "dtype must be FBMM_F32 (0), FBMM_F16 (1) or FBMM_BF16 (2), got %d", dtype);
  return FBMM_OK;
}

// 'n' or 't' in either case; 0 for anything else.
int layout_letter(int letter) {
  if (letter == 'n' || letter == 'N') return 'n';
  return letter == 't' || letter == 'T' ? 't' : 0;
}

int elem_size(int dtype) { return dtype == FBMM_F32 ? 4 : 2; }

// A microscaled operand as the entry points take it.
int check_mx(const char* name, const unsigned char* codes, long long stride_codes, const unsigned char* scales,
             long long stride_scales, int l) {
  if (codes == nullptr || scales == nullptr) return fail(FBMM_ERR_INVALID, "%s codes or scales are null", name);
  if (((reinterpret_cast<uintptr_t>(codes) | reinterpret_cast<uintptr_t>(scales)) & 15u) != 0)
    return fail(FBMM_ERR_ALIGN, "%s codes or scales are not 16-byte aligned", name);
  if (l > 1 && (stride_codes < 0 || stride_scales < 0 || (stride_codes & 15) != 0 || (stride_scales & 15) != 0))
    return fail(FBMM_ERR_ALIGN, "%s batch strides %lld and %lld are not non-negative multiples of 16 bytes", name,
                stride_codes, stride_scales);
  return FBMM_OK;
}

int check_quantize_source(const void* X, int dtype, int layout, long long ldx, long long stride_x, int l, int rows, int k) {
  int rc;
  if ((rc = check_shape(l, rows, k)) != FBMM_OK) return rc;
  if ((rc = check_type(dtype)) != FBMM_OK) return rc;
  if (layout_letter(layout) == 0) return fail(FBMM_ERR_INVALID, "layout must be 'n' or 't', got %d", layout);
  if (X == nullptr) return fail(FBMM_ERR_INVALID, "the source is null");
  if ((reinterpret_cast<uintptr_t>(X) & static_cast<uintptr_t>(elem_size(dtype) - 1)) != 0)
    return fail(FBMM_ERR_ALIGN, "the source is not aligned to its element type");
  if (ldx < (layout_letter(layout) == 'n' ? k : rows)) return fail(FBMM_ERR_INVALID, "source pitch %lld smaller than its row length", ldx);
  if (l > 1 && stride_x < 0) return fail(FBMM_ERR_INVALID, "source batch stride is negative");
  return FBMM_OK;
}

int check_result(const void* C, int dtype, long long ldc, long long stride_c, int l, int m, int n) {
  int rc;
  if ((rc = check_type(dtype)) != FBMM_OK) return rc;
  if (C == nullptr) return fail(FBMM_ERR_INVALID, "C is null");
  if ((reinterpret_cast<uintptr_t>(C) & static_cast<uintptr_t>(elem_size(dtype) - 1)) != 0)
    return fail(FBMM_ERR_ALIGN, "C is not aligned to its element type");
  if (ldc < n) return fail(FBMM_ERR_INVALID, "ldc %lld smaller than a row of C (%d)", ldc, n);
  if (l > 1 && stride_c < static_cast<long long>(m - 1) * ldc + n)
    return fail(FBMM_ERR_INVALID, "batches of C overlap (stride %lld)", stride_c);
  if (static_cast<long long>((m + 127) / 128) * ((n + 127) / 128) > 0x3fffffffLL)
    return fail(FBMM_ERR_INVALID, "product of %d x %d is too large", m, n);
  return FBMM_OK;
}

unsigned group_count(int l, int rows, int k) {
  return static_cast<unsigned>(static_cast<long long>(l) * ((rows + 127) / 128) * ((k + 127) / 128));
}

template <int BITS, typename T>
int launch_quantize(cudaStream_t stream, const MxQuantArgs& a, bool transposed) {
  const unsigned grid = group_count(a.l, a.rows, a.k);
  if (transposed) mx_quantize_t_kernel<BITS, T><<<grid, 256, 0, stream>>>(a);
  else mx_quantize_kernel<BITS, T><<<grid, 256, 0, stream>>>(a);
  FBMM_HOST_CUDA(cudaGetLastError());
  return FBMM_OK;
}

template <int BITS, typename T>
int launch_dequantize(cudaStream_t stream, const MxDequantArgs& a) {
  mx_dequantize_kernel<BITS, T><<<group_count(a.l, a.rows, a.k), 256, 0, stream>>>(a);
  FBMM_HOST_CUDA(cudaGetLastError());
  return FBMM_OK;
}

// Tensor map over the codes of [l][rows][k] 4-bit elements: boxes of 128 bytes x box_rows rows.
int codes_map(CUtensorMap* map, const unsigned char* codes, long long stride, int l, int rows, int k, int box_rows) {
  const cuuint64_t pitch = static_cast<cuuint64_t>(mx_pitch(k, 4));
  const bool one = l == 1 || stride == 0;
  const cuuint64_t dims[3] = {pitch, static_cast<cuuint64_t>(rows), one ? 1u : static_cast<cuuint64_t>(l)};
  const cuuint64_t strides[2] = {pitch, one ? pitch * static_cast<cuuint64_t>(rows) : static_cast<cuuint64_t>(stride)};
  const cuuint32_t box[3] = {kMxRowBytes, static_cast<cuuint32_t>(box_rows), 1};
  return fbmm_host::tensor_map_3d(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, codes, dims, strides, box, true);
}

// Bytes that every row of a matrix is aligned to: 16, 8, 4 or 2; pitch and batch stride in bytes.
int row_align(const void* base, long long pitch, long long stride) {
  const uint64_t low = reinterpret_cast<uintptr_t>(base) | static_cast<uint64_t>(pitch) | static_cast<uint64_t>(stride);
  return (low & 15) == 0 ? 16 : (low & 7) == 0 ? 8 : (low & 3) == 0 ? 4 : 2;
}

constexpr int kMxMaxSplits = 8;  // CTAs that share a tile's sum: the portable cluster size

// The kernel's shared-memory limit is set once per device.
template <auto kKernel>
int prepare(int* dev) {
  static std::atomic<unsigned long long> ready{0};
  FBMM_HOST_CUDA(cudaGetDevice(dev));
  const unsigned long long bit = 1ull << (*dev & 63);
  if ((ready.load(std::memory_order_relaxed) & bit) == 0) {
    FBMM_HOST_CUDA(cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kMxSmemLimit)));
    ready.fetch_or(bit, std::memory_order_relaxed);
  }
  return FBMM_OK;
}

// How many clusters of this size run at once: fewer than the SMs divided by it, since a cluster stays within a group
// of SMs (15 clusters of eight on 148 SMs). Asked once per device and size.
template <auto kKernel>
int clusters_at_once(int threads, int smem, int cluster, int* count) {
  static std::atomic<int> known[64][kMxMaxSplits + 1];  // count + 1
  int rc, dev = 0;
  if ((rc = prepare<kKernel>(&dev)) != FBMM_OK) return rc;
  std::atomic<int>& slot = known[dev & 63][cluster];
  *count = slot.load(std::memory_order_relaxed) - 1;
  if (*count >= 0) return FBMM_OK;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(cluster));
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = static_cast<unsigned>(cluster);
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  FBMM_HOST_CUDA(cudaOccupancyMaxActiveClusters(count, kKernel, &cfg));
  slot.store(*count + 1, std::memory_order_relaxed);
  return FBMM_OK;
}

// A launch with a cluster and the right to start (set up barriers and tensor memory) before the kernel ahead of it
// in the stream has ended. Kernels whose copies all wait for that kernel always have it; the few-row kernel,
// which asks for weights before it waits, only behind a quantiser, which cannot be writing them.
template <auto kKernel, typename... Args>
int launch(cudaStream_t stream, long long grid, int threads, int smem, int cluster, bool overlap, const Args&... args) {
  int rc, dev = 0;
  if ((rc = prepare<kKernel>(&dev)) != FBMM_OK) return rc;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2] = {};
  if (cluster > 1) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = static_cast<unsigned>(cluster);
    attr[cfg.numAttrs].val.clusterDim.y = 1;
    attr[cfg.numAttrs].val.clusterDim.z = 1;
    ++cfg.numAttrs;
  }
  if (overlap) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
    ++cfg.numAttrs;
  }
  cfg.attrs = attr;
  FBMM_HOST_CUDA(cudaLaunchKernelEx(&cfg, kKernel, args...));
  return FBMM_OK;
}

// A 4-bit operand [l][rows][k]; strides in bytes.
struct MxSide {
  const unsigned char* codes;
  long long stride;
  const unsigned char* scales;
  long long scale_stride;
  int rows;
};

// Tensor map over scales [l][row groups][k groups][512]: boxes of two k groups x row_groups.
int scales_map(CUtensorMap* map, const unsigned char* scales, long long stride, int l, int rows, int k, int row_groups) {
  const cuuint64_t pitch = static_cast<cuuint64_t>((k + kMxGroupK - 1) / kMxGroupK) * kMxGroupBytes;
  const cuuint64_t groups = static_cast<cuuint64_t>((rows + kMxGroupRows - 1) / kMxGroupRows);
  const bool one = l == 1 || stride == 0;
  const cuuint64_t dims[3] = {pitch / 4, groups, one ? 1u : static_cast<cuuint64_t>(l)};
  const cuuint64_t strides[2] = {pitch, one ? pitch * groups : static_cast<cuuint64_t>(stride)};
  const cuuint32_t box[3] = {kMxScaleStage / 4, static_cast<cuuint32_t>(row_groups), 1};
  return fbmm_host::tensor_map_3d(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, scales, dims, strides, box, false);
}

int launch_mx_gemm(cudaStream_t stream, int sms, const MxSide& p, const MxSide& q, MxGemmArgs a) {
  CUtensorMap mp, mq, msp, msq;
  int rc;
  if ((rc = codes_map(&mp, p.codes, p.stride, a.l, p.rows, a.k, kMxM)) != FBMM_OK) return rc;
  if ((rc = codes_map(&mq, q.codes, q.stride, a.l, q.rows, a.k, MxShape::BN)) != FBMM_OK) return rc;
  if ((rc = scales_map(&msp, p.scales, p.scale_stride, a.l, p.rows, a.k, 1)) != FBMM_OK) return rc;
  if ((rc = scales_map(&msq, q.scales, q.scale_stride, a.l, q.rows, a.k, 1)) != FBMM_OK) return rc;
  a.p_rows = p.rows; a.q_rows = q.rows;
  a.p_shared = p.stride == 0; a.q_shared = q.stride == 0;
  a.sp_shared = p.scale_stride == 0; a.sq_shared = q.scale_stride == 0;
  a.p_tiles = (p.rows + kMxM - 1) / kMxM;
  a.q_tiles = (q.rows + MxShape::BN - 1) / MxShape::BN;
  const long long units = static_cast<long long>(a.p_tiles) * a.q_tiles * a.l;
  return launch<mx_gemm_kernel>(stream, std::min<long long>(units, sms), kMxThreads, MxShape::kSmem, 1, true, mp, mq, msp, msq, a);
}

int launch_mx_pair(cudaStream_t stream, int sms, const MxSide& A, const MxSide& B, const MxGemmArgs& g) {
  CUtensorMap ma, mb, msa, msb;
  int rc;
  if ((rc = codes_map(&ma, A.codes, A.stride, g.l, A.rows, g.k, 128)) != FBMM_OK) return rc;
  if ((rc = codes_map(&mb, B.codes, B.stride, g.l, B.rows, g.k, 128)) != FBMM_OK) return rc;
  if ((rc = scales_map(&msa, A.scales, A.scale_stride, g.l, A.rows, g.k, 1)) != FBMM_OK) return rc;
  if ((rc = scales_map(&msb, B.scales, B.scale_stride, g.l, B.rows, g.k, 2)) != FBMM_OK) return rc;
  MxPairArgs a{};
  a.C = g.C; a.ldc = g.ldc; a.stride_c = g.stride_c;
  a.l = g.l; a.m = A.rows; a.n = B.rows; a.k = g.k;
  a.a_shared = A.stride == 0; a.b_shared = B.stride == 0;
  a.as_shared = A.scale_stride == 0; a.bs_shared = B.scale_stride == 0;
  a.out_type = g.out_type; a.align = g.align;
  a.m_tiles = (a.m + 255) / 256;
  a.n_tiles = (a.n + 255) / 256;
  const long long units = static_cast<long long>(a.m_tiles) * a.n_tiles * a.l;
  return launch<mx_gemm_pair_kernel>(stream, 2 * std::min<long long>(units, sms / 2), kMxPairThreads, kMxPairSmem, 2, true, ma, mb,
                                     msa, msb, a);
}

constexpr int kMxFewRows = 64;  // rows of A up to which the weights take the 128-row side of the MMA

// How many CTAs share the k of a tile in the few-row kernel. A CTA takes about 0.25 us per 256 k (one
// stage's latency over the depth of the ring; 0.35 us with 128 rows), joining the sums 0.7 us (4), and a second CTA
// on an SM starts 0.7 us late; two fit an SM. The least sum of these decides (measured: n = 16384,
// k = 8192 11.0 us on 256 CTAs against 12.4 on 128; n = 1024, k = 8192 4.9 us on 64 against 11.2 on 8).
// Tiles of 128 rows share k only while all their CTAs run at once, one to an SM: beyond, whole tiles or pairs of them
// reuse more of what they copy (512 rows, n = 5120, k = 8192: 15.3 us on 40 pairs, 30.0 us on 640 CTAs; 128 rows at
// 4096 x 4096 8.1 us on 128 against 9.0 on 32, 256 rows 10.8 on 128 against 9.3 on 64).
void rows_splits(int sms, int l, int m, int n, int k, int* splits, int* blocks) {
  const int kblocks = (k + kMxStageK - 1) / kMxStageK;
  const bool tall = m > kMxFewRows;
  const long long base = static_cast<long long>((n + kMxM - 1) / kMxM) * l * (tall ? (m + 127) / 128 : 1);
  long long best = 0;
  for (int s = 1; s <= kMxMaxSplits && (s == 1 || s <= kblocks); s *= 2) {
    // a cluster stays within a group of SMs: of four and eight 33 and 15 run at once on 148 SMs, with two
    // CTAs to an SM 71 and 33 (128 rows, n = 2048, k = 8192: 9.3 us in fours against 14.8 in eights, two waves)
    const int permille = s <= 2 ? 1000 : tall ? (s == 4 ? 900 : 813) : (s == 4 ? 960 : 900);
    const long long ctas = base * s, per = (kblocks + s - 1) / s, slots = (tall ? 1ll : 2ll) * sms * permille / 1000;
    if (tall && s > 1 && ctas > slots) break;
    const long long cost = (s > 1 ? (tall ? 4000 : 700) : 0) + (tall ? 350 : 250) * per * ((ctas + slots - 1) / slots) +
                           700 * ((ctas - 1) / sms);
    if (s == 1 || cost < best) {
      best = cost;
      *splits = s;
      *blocks = static_cast<int>(per);
    }
  }
}

// Whether the kernel quantises A itself. Every CTA quantises its range of k of all rows: up to 1024 blocks
// of 32 (four a thread) that hides behind the first weights; beyond, a pass of its own is faster
// (16 rows: 6.2 against 6.9 us at 4096 x 4096, 512 blocks; 15.6 against 12.5 us at n = 16384, k = 8192, 2048 blocks).
// The quantised rows also have to fit beside the ring.
bool few_rows_fused(int sms, int l, int m, int n, int k, int layout) {
  if (m > kMxFewRows || layout_letter(layout) != 'n') return false;
  int splits, blocks;
  rows_splits(sms, l, m, n, k, &splits, &blocks);
  const int stages = std::min(4, blocks);
  const int smem = m <= 16 ? MxRowsShape<16, float>::smem(stages, blocks) : MxRowsShape<64, float>::smem(stages, blocks);
  return static_cast<long long>(m) * blocks * (kMxStageK / kMxBlock) <= 1024 && smem <= static_cast<int>(kMxSmemLimit);
}

template <int NT, typename T>
int launch_mx_rows(cudaStream_t stream, int sms, bool overlap, const MxSide& W, const MxSide* A, MxRowsArgs a) {
  using S = MxRowsShape<NT, T>;
  CUtensorMap mw, msw, ma, msa;
  int rc;
  if ((rc = codes_map(&mw, W.codes, W.stride, a.l, W.rows, a.k, kMxM)) != FBMM_OK) return rc;
  if ((rc = scales_map(&msw, W.scales, W.scale_stride, a.l, W.rows, a.k, 1)) != FBMM_OK) return rc;
  a.w_shared = W.stride == 0; a.sw_shared = W.scale_stride == 0;
  if (S::kCodes) {
    if ((rc = codes_map(&ma, A->codes, A->stride, a.l, A->rows, a.k, NT)) != FBMM_OK) return rc;
    if ((rc = scales_map(&msa, A->scales, A->scale_stride, a.l, A->rows, a.k, 1)) != FBMM_OK) return rc;
    a.a_shared = A->stride == 0; a.sa_shared = A->scale_stride == 0;
  } else {
    ma = mw; msa = msw;
  }
  a.n_tiles = (a.n + kMxM - 1) / kMxM;
  a.m_tiles = NT == 128 ? (a.m + NT - 1) / NT : 1;
  rows_splits(sms, a.l, a.m, a.n, a.k, &a.splits, &a.blocks_per_split);
  const long long grid = static_cast<long long>(a.n_tiles) * a.m_tiles * a.l * a.splits;
  if (grid > 0x7fffffffLL) return fail(FBMM_ERR_INVALID, "product of %d x %d x %d is too large", a.l, a.m, a.n);
  const int limit = static_cast<int>(kMxSmemLimit);
  const int budget = grid > sms && S::smem(3, a.blocks_per_split) <= limit / 2 ? limit / 2 : limit;
  a.stages = std::min(S::kMaxStages, a.blocks_per_split);
  while (a.stages > 1 && S::smem(a.stages, a.blocks_per_split) > budget) --a.stages;
  const int smem = S::smem(a.stages, a.blocks_per_split);
  if (smem > limit) return fail(FBMM_ERR_INVALID, "internal: few-row kernel wants %d bytes of shared memory", smem);
  return launch<mx_rows_kernel<NT, T>>(stream, grid, S::kThreads, smem, a.splits, overlap, mw, msw, ma, msa, a);
}

template <int NT>
int launch_mx_rows_fused(cudaStream_t stream, int sms, int dtype, const MxSide& W, const MxRowsArgs& a) {
  if (dtype == FBMM_F32) return launch_mx_rows<NT, float>(stream, sms, false, W, nullptr, a);
  if (dtype == FBMM_F16) return launch_mx_rows<NT, __half>(stream, sms, false, W, nullptr, a);
  return launch_mx_rows<NT, __nv_bfloat16>(stream, sms, false, W, nullptr, a);
}

// C = A @ B^T of two 4-bit operands; `overlap`: the kernel ahead in the stream is the quantiser that writes A.
int mx4_product(cudaStream_t stream, bool overlap, const unsigned char* a_codes, long long stride_a,
                const unsigned char* a_scales, long long stride_as, const unsigned char* b_codes, long long stride_b,
                const unsigned char* b_scales, long long stride_bs, void* C, int dtype, long long ldc, long long stride_c, int l,
                int m, int n, int k) {
  int rc, sms;
  if ((rc = check_shape(l, m, k)) != FBMM_OK) return rc;
  if ((rc = check_shape(l, n, k)) != FBMM_OK) return rc;
  if ((rc = check_mx("A", a_codes, stride_a, a_scales, stride_as, l)) != FBMM_OK) return rc;
  if ((rc = check_mx("B", b_codes, stride_b, b_scales, stride_bs, l)) != FBMM_OK) return rc;
  if ((rc = check_result(C, dtype, ldc, stride_c, l, m, n)) != FBMM_OK) return rc;
  if ((rc = fbmm_host::device_sms(&sms)) != FBMM_OK) return rc;
  MxGemmArgs a{};
  a.C = C; a.ldc = ldc; a.stride_c = l > 1 ? stride_c : 0;
  a.l = l; a.k = k; a.out_type = dtype;
  const long long size = elem_size(dtype);
  a.align = row_align(C, ldc * size, a.stride_c * size);
  const MxSide A{a_codes, stride_a, a_scales, stride_as, m}, B{b_codes, stride_b, b_scales, stride_bs, n};
  int splits, blocks;
  rows_splits(sms, l, m, n, k, &splits, &blocks);
  if (m <= kMxFewRows || splits > 1) {
    MxRowsArgs r{};
    r.C = C; r.ldc = ldc; r.stride_c = a.stride_c;
    r.l = l; r.m = m; r.n = n; r.k = k;
    r.out_type = dtype; r.align = a.align;
    if (m > kMxFewRows) return launch_mx_rows<128, uint8_t>(stream, sms, overlap, B, &A, r);
    return m <= 16 ? launch_mx_rows<16, uint8_t>(stream, sms, overlap, B, &A, r) : launch_mx_rows<64, uint8_t>(stream, sms, overlap, B, &A, r);
  }
  const long long pairs = static_cast<long long>((m + 255) / 256) * ((n + 255) / 256) * l;
  const long long singles = static_cast<long long>((m + 127) / 128) * ((n + 127) / 128) * l;
  const long long pair_waves = (pairs + sms / 2 - 1) / (sms / 2), single_waves = (singles + sms - 1) / sms;
  if (5 * pair_waves <= 4 * single_waves) return launch_mx_pair(stream, sms, A, B, a);
  return launch_mx_gemm(stream, sms, A, B, a);
}

// One operand of a 16-bit product: a dense matrix of `rows` x J (J contiguous, or the rows), or a
// microscaled one stored [J][rows] with its blocks along the rows.
struct X16Side {
  int kind;
  const void* ptr;              // elements or codes
  long long ld, stride;         // elements (dense); stride in bytes for codes
  const unsigned char* scales;
  long long scale_stride;
  int rows;
};

int check_x16_side(const char* name, const X16Side& s, int J, int l) {
  if (s.kind >= kX16Mx4) {  // [J][rows], its blocks along the rows
    const int rc = check_shape(l, J, s.rows);
    return rc != FBMM_OK ? rc : check_mx(name, static_cast<const unsigned char*>(s.ptr), s.stride, s.scales, s.scale_stride, l);
  }
  if (s.ptr == nullptr) return fail(FBMM_ERR_INVALID, "%s is null", name);
  const int inner = s.kind == kX16K ? J : s.rows;
  if (s.ld < inner) return fail(FBMM_ERR_INVALID, "%s pitch %lld smaller than its row length %d", name, s.ld, inner);
  if ((reinterpret_cast<uintptr_t>(s.ptr) & 1u) != 0) return fail(FBMM_ERR_ALIGN, "%s is not 2-byte aligned", name);
  if (l > 1 && s.stride < 0) return fail(FBMM_ERR_INVALID, "%s batch stride is negative", name);
  return FBMM_OK;
}

// Scratch for a dense operand that tensor maps cannot describe (base, pitch or batch stride not a multiple of 16
// bytes); 0 for one that they can.
size_t repack_bytes(const void* ptr, long long ld, long long stride, int l, int outer, int inner) {
  const bool batched = l > 1 && stride != 0;
  if (((reinterpret_cast<uintptr_t>(ptr) | static_cast<uint64_t>(ld * 2) | (batched ? static_cast<uint64_t>(stride * 2) : 0)) & 15) == 0)
    return 0;
  const size_t pitch = (static_cast<size_t>(inner) + 7) / 8 * 8;
  return ((batched ? static_cast<size_t>(l) : 1) * outer * pitch * 2 + 255) / 256 * 256;
}

// The repacking of such an operand into the workspace; makes the side describe the copy.
X16Repack repack_side(X16Side* s, int J, int l, unsigned char* ws) {
  const int outer = s->kind == kX16K ? s->rows : J, inner = s->kind == kX16K ? J : s->rows;
  const bool batched = l > 1 && s->stride != 0;
  X16Repack r{};
  r.src = static_cast<const uint16_t*>(s->ptr);
  r.ld = s->ld;
  r.stride = batched ? s->stride : 0;
  r.dst = reinterpret_cast<uint16_t*>(ws);
  r.rows = outer;
  r.cols = inner;
  r.pitch = (inner + 7) / 8 * 8;
  r.pieces = static_cast<long long>(batched ? l : 1) * outer * (r.pitch / 8);
  r.align = row_align(s->ptr, s->ld * 2, r.stride * 2);
  s->ptr = ws;
  s->ld = r.pitch;
  s->stride = batched ? static_cast<long long>(outer) * r.pitch : 0;
  return r;
}

int x16_map(CUtensorMap* map, const X16Side& s, int J, int l, int dtype) {
  const bool one = l == 1 || s.stride == 0;
  const cuuint64_t batches = one ? 1u : static_cast<cuuint64_t>(l);
  if (s.kind >= kX16Mx4) {
    const int bits = s.kind == kX16Mx4 ? 4 : 8;
    const cuuint64_t pitch = static_cast<cuuint64_t>(mx_pitch(s.rows, bits));
    const cuuint64_t dims[3] = {pitch, static_cast<cuuint64_t>(J), batches};
    const cuuint64_t strides[2] = {pitch, one ? pitch * dims[1] : static_cast<cuuint64_t>(s.stride)};
    const cuuint32_t box[3] = {static_cast<cuuint32_t>(128 * bits / 8), kX16J, 1};
    return fbmm_host::tensor_map_3d(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, s.ptr, dims, strides, box, bits == 8);
  }
  const bool kmajor = s.kind == kX16K;
  const cuuint64_t pitch = static_cast<cuuint64_t>(s.ld) * 2u;
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(kmajor ? J : s.rows), static_cast<cuuint64_t>(kmajor ? s.rows : J), batches};
  const cuuint64_t strides[2] = {pitch, one ? pitch * dims[1] : static_cast<cuuint64_t>(s.stride) * 2u};
  const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(kmajor ? 128 : kX16J), 1};
  return fbmm_host::tensor_map_3d(map, dtype == FBMM_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                                  s.ptr, dims, strides, box, true);
}

template <int XK, int YK, bool PAIR, bool SPLIT = false>
int launch_x16(cudaStream_t stream, int sms, const CUtensorMap& mx, const CUtensorMap& my, X16Args a) {
  using S = X16Shape<XK, YK>;
  constexpr int kTile = PAIR ? 256 : 128;
  a.x_tiles = (a.x.rows + kTile - 1) / kTile;
  a.y_tiles = (a.y.rows + kTile - 1) / kTile;
  const long long units = static_cast<long long>(a.x_tiles) * a.y_tiles * a.l;
  const long long grid = SPLIT ? units * a.splits : PAIR ? 2 * std::min<long long>(units, sms / 2) : std::min<long long>(units, sms);
  return launch<x16_gemm_kernel<XK, YK, PAIR, SPLIT>>(stream, grid, S::kThreads, S::kSmem, PAIR ? 2 : SPLIT ? a.splits : 1, true, mx,
                                                      my, a);
}

template <int XK, int YK>
int launch_x16_any(cudaStream_t stream, int sms, const CUtensorMap& mx, const CUtensorMap& my, X16Args a) {
  // 256 x 256 tiles on pairs unless they leave SMs idle: a wave of pair tiles is twice the work of a
  // wave of 128 x 128 tiles and takes 1.25 times as long (1570 against 980 TFLOP/s at 4096^3)
  auto tiles = [&](int tile) {
    return static_cast<long long>((a.x.rows + tile - 1) / tile) * ((a.y.rows + tile - 1) / tile) * a.l;
  };
  auto waves = [&](int tile, long long workers) { return (tiles(tile) + workers - 1) / workers; };
  if (5 * waves(256, sms / 2) <= 4 * waves(128, sms)) return launch_x16<XK, YK, true>(stream, sms, mx, my, a);
  // Fewer tiles than SMs: j over a cluster of up to eight CTAs per tile, while all clusters run at once, where it pays.
  // In ns: a stage takes about 250, an expanded one 340; joining the sums 4500 (8-bit dB of 4096 x 64 over 8192:
  // 46.1 us whole, 18.0 in fours; 512 x 512 over 4096: 25.6 and 11.5; dense 4096 x 64 over 4096: 19.2 and 11.1).
  using S = X16Shape<XK, YK>;
  constexpr long long kStageNs = XK >= kX16Mx4 || YK >= kX16Mx4 ? 340 : 250, kJoinNs = 4500;
  const int blocks = (a.J + kX16J - 1) / kX16J;
  long long best = kStageNs * blocks;
  a.splits = 1;
  for (int s = 2; s <= kMxMaxSplits && tiles(128) * s <= sms && kJoinNs < best; ++s) {
    const int each = (blocks + s - 1) / s;
    if (kJoinNs + kStageNs * each >= best) continue;
    int rc, at_once;
    if ((rc = clusters_at_once<x16_gemm_kernel<XK, YK, false, true>>(S::kThreads, S::kSmem, s, &at_once)) != FBMM_OK) return rc;
    if (tiles(128) > at_once) continue;
    best = kJoinNs + kStageNs * each;
    a.splits = s;
    a.blocks_per_split = each;
  }
  if (a.splits > 1) return launch_x16<XK, YK, false, true>(stream, sms, mx, my, a);
  return launch_x16<XK, YK, false>(stream, sms, mx, my, a);
}

int x16_product(cudaStream_t stream, X16Side x, X16Side y, int dtype, void* C, long long ldc, long long stride_c, int l, int J,
                void* workspace, size_t workspace_bytes) {
  int rc, sms;
  if (l <= 0 || x.rows <= 0 || y.rows <= 0 || J <= 0)
    return fail(FBMM_ERR_INVALID, "l, m, n, k must be positive, got %d %d %d %d", l, x.rows, y.rows, J);
  if (x.rows > 0x7fffff00 || y.rows > 0x7fffff00 || J > 0x7fffff00)
    return fail(FBMM_ERR_INVALID, "product of %d x %d x %d is too large", x.rows, y.rows, J);
  if (dtype != FBMM_F16 && dtype != FBMM_BF16)
    return fail(FBMM_ERR_INVALID, "dtype must be FBMM_F16 (1) or FBMM_BF16 (2), got %d", dtype);
  if ((rc = check_x16_side("A", x, J, l)) != FBMM_OK) return rc;
  if ((rc = check_x16_side("B", y, J, l)) != FBMM_OK) return rc;
  if ((rc = check_result(C, dtype, ldc, stride_c, l, x.rows, y.rows)) != FBMM_OK) return rc;
  if ((reinterpret_cast<uintptr_t>(workspace) & 15u) != 0) return fail(FBMM_ERR_ALIGN, "workspace is not 16-byte aligned");
  // refused before a device is asked for
  unsigned char* const ws = static_cast<unsigned char*>(workspace);
  const size_t need_x = x.kind >= kX16Mx4 ? 0 : repack_bytes(x.ptr, x.ld, x.stride, l, x.kind == kX16K ? x.rows : J, x.kind == kX16K ? J : x.rows);
  const size_t need_y = y.kind >= kX16Mx4 ? 0 : repack_bytes(y.ptr, y.ld, y.stride, l, y.kind == kX16K ? y.rows : J, y.kind == kX16K ? J : y.rows);
  if (need_x + need_y > 0 && ws == nullptr)
    return fail(FBMM_ERR_ALIGN, "%s is not addressable (16-byte base, pitch and batch stride) and there is no workspace to repack it in",
                need_x ? "A" : "B");
  if (need_x + need_y > 0 && workspace_bytes < need_x + need_y)
    return fail(FBMM_ERR_WORKSPACE, "repacking needs %zu workspace bytes, got %zu", need_x + need_y, workspace_bytes);
  if ((rc = fbmm_host::device_sms(&sms)) != FBMM_OK) return rc;
  if (need_x + need_y > 0) {
    X16Repack p{}, q{};
    if (need_x) p = repack_side(&x, J, l, ws);
    if (need_y) q = repack_side(&y, J, l, ws + need_x);
    auto blocks = [](const X16Repack& r) { return std::min<long long>((r.pieces + 255) / 256, 1 << 20); };
    if ((rc = launch<x16_repack_kernel>(stream, blocks(p) + blocks(q), 256, 0, 1, true, p, q, static_cast<unsigned>(blocks(p)))) != FBMM_OK)
      return rc;
  }
  CUtensorMap mx, my;
  if ((rc = x16_map(&mx, x, J, l, dtype)) != FBMM_OK) return rc;
  if ((rc = x16_map(&my, y, J, l, dtype)) != FBMM_OK) return rc;
  X16Args a{};
  a.x = X16Operand{x.scales, l > 1 ? x.scale_stride : 0, x.rows, l > 1 && x.stride == 0};
  a.y = X16Operand{y.scales, l > 1 ? y.scale_stride : 0, y.rows, l > 1 && y.stride == 0};
  a.C = C; a.ldc = ldc; a.stride_c = l > 1 ? stride_c : 0;
  a.l = l; a.J = J; a.dtype = dtype;
  a.align = row_align(C, ldc * 2, a.stride_c * 2);
#define FBMM_X16(XK, YK) \
  if (x.kind == XK && y.kind == YK) return launch_x16_any<XK, YK>(stream, sms, mx, my, a)
  FBMM_X16(kX16K, kX16K);
  FBMM_X16(kX16K, kX16MN);
  FBMM_X16(kX16MN, kX16K);
  FBMM_X16(kX16MN, kX16MN);
  FBMM_X16(kX16K, kX16Mx4);
  FBMM_X16(kX16MN, kX16Mx4);
  FBMM_X16(kX16K, kX16Mx8);
  FBMM_X16(kX16MN, kX16Mx8);
  FBMM_X16(kX16Mx4, kX16MN);
  FBMM_X16(kX16Mx8, kX16MN);
#undef FBMM_X16
  return fail(FBMM_ERR_INVALID, "internal: no kernel for kinds %d and %d", x.kind, y.kind);
}

int layout_kind(const char* name, int letter, int k_major_letter, int* kind) {
  if (layout_letter(letter) == 0) return fail(FBMM_ERR_INVALID, "%s layout must be 'n' or 't', got %d", name, letter);
  *kind = layout_letter(letter) == k_major_letter ? kX16K : kX16MN;
  return FBMM_OK;
}

}  // namespace

namespace fbmm_host {
int mx_status(unsigned int* bits) {
  const unsigned int zero = 0;
  FBMM_HOST_CUDA(cudaMemcpyFromSymbol(bits, fbmm::g_mx_status, sizeof(*bits)));
  if (*bits != 0) FBMM_HOST_CUDA(cudaMemcpyToSymbol(fbmm::g_mx_status, &zero, sizeof(zero)));
  return FBMM_OK;
}
}  // namespace fbmm_host

extern "C" {

size_t fbmm_mx_codes_bytes(int l, int rows, int k, int bits) {
  if (l <= 0 || rows <= 0 || k <= 0 || k > (1 << 29) || (bits != 4 && bits != 8)) return 0;
  return static_cast<size_t>(l) * rows * static_cast<size_t>(mx_pitch(k, bits));
}

size_t fbmm_mx_scales_bytes(int l, int rows, int k) {
  if (l <= 0 || rows <= 0 || rows > 0x7fffff00 || k <= 0 || k > (1 << 29)) return 0;
  return static_cast<size_t>(l) * static_cast<size_t>(mx_scale_bytes(rows, k));
}

int fbmm_mx_quantize(void* stream_, const void* X, int dtype, int layout, long long ldx, long long stride_x, int bits,
                     unsigned char* codes, unsigned char* scales, int l, int rows, int k) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  int rc, sms;
  if ((rc = check_quantize_source(X, dtype, layout, ldx, stride_x, l, rows, k)) != FBMM_OK) return rc;
  if ((rc = check_bits(bits)) != FBMM_OK) return rc;
  if ((rc = check_mx("output", codes, 0, scales, 0, 1)) != FBMM_OK) return rc;
  if ((rc = fbmm_host::device_sms(&sms)) != FBMM_OK) return rc;
  const MxQuantArgs a{X, ldx, l > 1 ? stride_x : 0, codes, scales, rows, k, l};
  const bool t = layout_letter(layout) == 't';
  if (bits == 4) {
    if (dtype == FBMM_F32) return launch_quantize<4, float>(stream, a, t);
    if (dtype == FBMM_F16) return launch_quantize<4, __half>(stream, a, t);
    return launch_quantize<4, __nv_bfloat16>(stream, a, t);
  }
  if (dtype == FBMM_F32) return launch_quantize<8, float>(stream, a, t);
  if (dtype == FBMM_F16) return launch_quantize<8, __half>(stream, a, t);
  return launch_quantize<8, __nv_bfloat16>(stream, a, t);
}

int fbmm_mx_dequantize(void* stream_, const unsigned char* codes, long long stride_codes, const unsigned char* scales,
                       long long stride_scales, int bits, void* out, int dtype, long long ldo, long long stride_o, int l,
                       int rows, int k) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  int rc, sms;
  if ((rc = check_shape(l, rows, k)) != FBMM_OK) return rc;
  if ((rc = check_bits(bits)) != FBMM_OK) return rc;
  if ((rc = check_type(dtype)) != FBMM_OK) return rc;
  if ((rc = check_mx("input", codes, stride_codes, scales, stride_scales, l)) != FBMM_OK) return rc;
  if (out == nullptr) return fail(FBMM_ERR_INVALID, "out is null");
  if ((reinterpret_cast<uintptr_t>(out) & static_cast<uintptr_t>(elem_size(dtype) - 1)) != 0)
    return fail(FBMM_ERR_ALIGN, "out is not aligned to its element type");
  if (ldo < k) return fail(FBMM_ERR_INVALID, "out pitch %lld smaller than k = %d", ldo, k);
  if (l > 1 && stride_o < static_cast<long long>(rows - 1) * ldo + k)
    return fail(FBMM_ERR_INVALID, "out batches overlap (stride %lld)", stride_o);
  if ((rc = fbmm_host::device_sms(&sms)) != FBMM_OK) return rc;
  const MxDequantArgs a{codes, scales, l > 1 ? stride_codes : 0, l > 1 ? stride_scales : 0, out, ldo,
                        l > 1 ? stride_o : 0, rows, k, l};
  if (bits == 4) {
    if (dtype == FBMM_F32) return launch_dequantize<4, float>(stream, a);
    if (dtype == FBMM_F16) return launch_dequantize<4, __half>(stream, a);
    return launch_dequantize<4, __nv_bfloat16>(stream, a);
  }
  if (dtype == FBMM_F32) return launch_dequantize<8, float>(stream, a);
  if (dtype == FBMM_F16) return launch_dequantize<8, __half>(stream, a);
  return launch_dequantize<8, __nv_bfloat16>(stream, a);
}

int fbmm_mx4_bmm(void* stream, const unsigned char* a_codes, long long stride_a, const unsigned char* a_scales,
                 long long stride_as, const unsigned char* b_codes, long long stride_b, const unsigned char* b_scales,
                 long long stride_bs, void* C, int dtype, long long ldc, long long stride_c, int l, int m, int n, int k) {
  return mx4_product(static_cast<cudaStream_t>(stream), false, a_codes, stride_a, a_scales, stride_as, b_codes, stride_b, b_scales,
                     stride_bs, C, dtype, ldc, stride_c, l, m, n, k);
}

size_t fbmm_mx4_bmm_tensor_workspace_bytes(int l, int m, int n, int k, int a_layout) {
  if (l <= 0 || m <= 0 || n <= 0 || k <= 0 || n > 0x7fffff00 || m > 0x7fffff00 || k > (1 << 29)) return 0;
  if (few_rows_fused(fbmm_host::sms_or_default(), l, m, n, k, a_layout)) return 0;
  return (fbmm_mx_codes_bytes(l, m, k, 4) + 255) / 256 * 256 + fbmm_mx_scales_bytes(l, m, k);
}

int fbmm_mx4_bmm_tensor(void* stream, const void* A, int a_dtype, int a_layout, long long lda, long long stride_a,
                        const unsigned char* b_codes, long long stride_b, const unsigned char* b_scales,
                        long long stride_bs, void* C, int dtype, long long ldc, long long stride_c, int l, int m, int n,
                        int k, void* workspace, size_t workspace_bytes) {
  int rc, sms;
  if ((rc = check_quantize_source(A, a_dtype, a_layout, lda, stride_a, l, m, k)) != FBMM_OK) return rc;
  if ((rc = check_shape(l, n, k)) != FBMM_OK) return rc;
  if (few_rows_fused(fbmm_host::sms_or_default(), l, m, n, k, a_layout)) {
    if ((rc = check_mx("B", b_codes, stride_b, b_scales, stride_bs, l)) != FBMM_OK) return rc;
    if ((rc = check_result(C, dtype, ldc, stride_c, l, m, n)) != FBMM_OK) return rc;
    if ((rc = fbmm_host::device_sms(&sms)) != FBMM_OK) return rc;
    MxRowsArgs a{};
    a.x = A; a.ldx = lda; a.stride_x = l > 1 ? stride_a : 0;
    a.C = C; a.ldc = ldc; a.stride_c = l > 1 ? stride_c : 0;
    a.l = l; a.m = m; a.n = n; a.k = k;
    a.out_type = dtype;
    const long long size = elem_size(dtype);
    a.align = row_align(C, ldc * size, a.stride_c * size);
    const MxSide W{b_codes, stride_b, b_scales, stride_bs, n};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return m <= 16 ? launch_mx_rows_fused<16>(s, sms, a_dtype, W, a) : launch_mx_rows_fused<64>(s, sms, a_dtype, W, a);
  }
  const size_t need = fbmm_mx4_bmm_tensor_workspace_bytes(l, m, n, k, a_layout);
  if (workspace == nullptr || workspace_bytes < need)
    return fail(FBMM_ERR_WORKSPACE, "fbmm_mx4_bmm_tensor needs %zu workspace bytes, got %zu", need,
                workspace == nullptr ? static_cast<size_t>(0) : workspace_bytes);
  unsigned char* codes = static_cast<unsigned char*>(workspace);
  unsigned char* scales = codes + (need - fbmm_mx_scales_bytes(l, m, k));
  if ((rc = fbmm_mx_quantize(stream, A, a_dtype, a_layout, lda, stride_a, 4, codes, scales, l, m, k)) != FBMM_OK) return rc;
  return mx4_product(static_cast<cudaStream_t>(stream), true, codes, static_cast<long long>(m) * mx_pitch(k, 4), scales,
                     mx_scale_bytes(m, k), b_codes, stride_b, b_scales, stride_bs, C, dtype, ldc, stride_c, l, m, n, k);
}

size_t fbmm_x16_repack_bytes(const void* X, long long ld, long long stride, int l, int outer, int inner) {
  if (l <= 0 || outer <= 0 || inner <= 0) return 0;
  return repack_bytes(X, ld, stride, l, outer, inner);
}

int fbmm_dense_bmm_x16(void* stream, const void* A, int a_layout, long long lda, long long stride_a, const void* B,
                       int b_layout, long long ldb, long long stride_b, int dtype, void* C, long long ldc,
                       long long stride_c, int l, int m, int n, int k, void* workspace,
                       size_t workspace_bytes) {
  X16Side x{0, A, lda, stride_a, nullptr, 0, m}, y{0, B, ldb, stride_b, nullptr, 0, n};
  int rc;
  if ((rc = layout_kind("A", a_layout, 'n', &x.kind)) != FBMM_OK) return rc;
  if ((rc = layout_kind("B", b_layout, 't', &y.kind)) != FBMM_OK) return rc;
  return x16_product(static_cast<cudaStream_t>(stream), x, y, dtype, C, ldc, stride_c, l, k, workspace, workspace_bytes);
}

int fbmm_dense_mx_bmm_x16(void* stream, const void* A, int a_layout, long long lda, long long stride_a, int dtype,
                          const unsigned char* b_codes, long long stride_b, const unsigned char* b_scales,
                          long long stride_bs, int bits, void* C, long long ldc, long long stride_c, int l, int m, int n,
                          int k, void* workspace,
                       size_t workspace_bytes) {
  int rc;
  if ((rc = check_bits(bits)) != FBMM_OK) return rc;
  X16Side x{0, A, lda, stride_a, nullptr, 0, m};
  const X16Side y{bits == 4 ? kX16Mx4 : kX16Mx8, b_codes, 0, stride_b, b_scales, stride_bs, n};
  if ((rc = layout_kind("A", a_layout, 'n', &x.kind)) != FBMM_OK) return rc;
  return x16_product(static_cast<cudaStream_t>(stream), x, y, dtype, C, ldc, stride_c, l, k, workspace, workspace_bytes);
}

int fbmm_mx_dense_bmm_x16(void* stream, const unsigned char* a_codes, long long stride_a, const unsigned char* a_scales,
                          long long stride_as, int bits, const void* B, long long ldb, long long stride_b, int dtype,
                          void* C, long long ldc, long long stride_c, int l, int m, int n, int k, void* workspace,
                       size_t workspace_bytes) {
  int rc;
  if ((rc = check_bits(bits)) != FBMM_OK) return rc;
  const X16Side x{bits == 4 ? kX16Mx4 : kX16Mx8, a_codes, 0, stride_a, a_scales, stride_as, m};
  const X16Side y{kX16MN, B, ldb, stride_b, nullptr, 0, n};
  return x16_product(static_cast<cudaStream_t>(stream), x, y, dtype, C, ldc, stride_c, l, k, workspace, workspace_bytes);
}

}  // extern "C"
