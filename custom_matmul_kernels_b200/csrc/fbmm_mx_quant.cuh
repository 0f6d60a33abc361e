// Microscaled storage: elements of 4 bits (e2m1: 0 0.5 1 1.5 2 3 4 6) or 8 bits (e4m3, largest
// 448) with one power-of-two scale per block of 32 along k. Quantisation and its inverse.
//
// Storage of a [rows, k] matrix: codes [rows][ceil(k/32)*32*bits/8] bytes (two 4-bit elements per
// byte, the lower k in the low half; zeros behind k), scales in groups of 128 rows x 4 blocks of
// 512 bytes, [ceil(rows/128)][ceil(k/128)][512], row r and block b of a group at byte
// (r % 32) * 16 + (r / 32) * 4 + b. That is the order in which the tensor cores' scale factors go
// to tensor memory, so a group is one contiguous 512-byte copy for the product kernel. A scale
// byte E stands for 2^(E - 127); 255 marks a block that holds an infinity or a NaN (every element
// reads back as NaN).
//
// The block's scale, from the exponent field f and the mantissa of its largest magnitude:
//   4 bits  E = f - 2, i.e. 2^(floor(log2 amax) - 2): values in (6, 8) * 2^e saturate at 6.
//   8 bits  the least E that keeps amax <= 448 * 2^e: f - 8, or f - 7 where the mantissa is above
//           1.75. Not below `low` (a finer step than the source type's own would not survive the
//           way back into it), and where amax could round up past the type's largest value the
//           elements stop at 240.
// Both rules were compared on normal, Laplace and Student-t(4) values: relative rms error at 4 bits
// 0.115 / 0.126 / 0.131 with saturation against 0.116 / 0.132 / 0.139 without; at 8 bits 0.030 /
// 0.031 / 0.032 against 0.0265 for all three. Multiplying by 2^-e is exact, so the only rounding is
// the one to the element type (to nearest, ties to even).
#pragma once
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

namespace fbmm {

constexpr int kMxBlock = 32;       // elements per scale
constexpr int kMxGroupRows = 128;  // rows of a 512-byte group of scales
constexpr int kMxGroupK = 128;     // elements along k of a group
constexpr int kMxGroupBytes = 512;

__host__ __device__ inline long long mx_pitch(int k, int bits) { return static_cast<long long>((k + 31) / 32) * (4 * bits); }
__host__ __device__ inline long long mx_scale_bytes(int rows, int k) {
  return static_cast<long long>((rows + 127) / 128) * ((k + 127) / 128) * kMxGroupBytes;
}
__device__ __forceinline__ int mx_scale_at(int row_in_group, int block_in_group) {
  return (row_in_group & 31) * 16 + (row_in_group >> 5) * 4 + block_in_group;
}

// Element types of the sources: the least scale byte at 8 bits, and the one whose codes stop at 240.
template <typename T> struct MxSource;
template <> struct MxSource<float> { static constexpr int kLow8 = 0, kTop8 = 247; };
template <> struct MxSource<__nv_bfloat16> { static constexpr int kLow8 = 3, kTop8 = 247; };
template <> struct MxSource<__half> { static constexpr int kLow8 = 112, kTop8 = 135; };

__device__ __forceinline__ float mx_to_float(float v) { return v; }
__device__ __forceinline__ float mx_to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float mx_to_float(__half v) { return __half2float(v); }

// Scale byte of a block from the bits of its largest magnitude as fp32.
template <int BITS, typename T>
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t amax_bits) {
  const int f = static_cast<int>(amax_bits >> 23);
  if (f == 255) return 255u;
  if (BITS == 4) return static_cast<uint32_t>(max(f - 2, 0));
  const int e = f - 8 + ((amax_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return static_cast<uint32_t>(max(e, MxSource<T>::kLow8));
}
// 2^(127 - E), what the elements of a block with scale byte E are multiplied by (E <= 252)
__device__ __forceinline__ float mx_inverse_scale(uint32_t E) { return __uint_as_float((254u - E) << 23); }
// 2^(E - 127)
__device__ __forceinline__ float mx_scale_value(uint32_t E) {
  return E == 255u ? __uint_as_float(0x7fc00000u) : __uint_as_float(E == 0 ? 0x00400000u : E << 23);
}

// Eight scaled values -> eight 4-bit codes (to nearest even, saturating).
__device__ __forceinline__ uint32_t mx_pack4(const float (&y)[8]) {
  uint32_t r;
  asm("{\n"
      ".reg .b8 b0, b1, b2, b3;\n"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n"
      "mov.b32 %0, {b0, b1, b2, b3};\n"
      "}\n"
      : "=r"(r)
      : "f"(y[0]), "f"(y[1]), "f"(y[2]), "f"(y[3]), "f"(y[4]), "f"(y[5]), "f"(y[6]), "f"(y[7]));
  return r;
}
// Four scaled values -> four 8-bit codes.
__device__ __forceinline__ uint32_t mx_pack8(float a, float b, float c, float d) {
  uint32_t r;
  asm("{\n"
      ".reg .b16 lo, hi;\n"
      "cvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n"
      "cvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n"
      "mov.b32 %0, {lo, hi};\n"
      "}\n"
      : "=r"(r)
      : "f"(a), "f"(b), "f"(c), "f"(d));
  return r;
}
// Eight 4-bit codes -> eight halves (exact), in pairs.
__device__ __forceinline__ void mx_unpack4(uint32_t c, uint32_t (&h)[4]) {
  asm("{\n"
      ".reg .b8 b0, b1, b2, b3;\n"
      "mov.b32 {b0, b1, b2, b3}, %4;\n"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n"
      "}\n"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(c));
}
// Four 8-bit codes -> four halves (exact), in pairs.
__device__ __forceinline__ void mx_unpack8(uint32_t c, uint32_t& h0, uint32_t& h1) {
  asm("{\n"
      ".reg .b16 lo, hi;\n"
      "mov.b32 {lo, hi}, %2;\n"
      "cvt.rn.f16x2.e4m3x2 %0, lo;\n"
      "cvt.rn.f16x2.e4m3x2 %1, hi;\n"
      "}\n"
      : "=r"(h0), "=r"(h1)
      : "r"(c));
}
__device__ __forceinline__ float2 mx_half2_floats(uint32_t h) {
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// Eight elements from global memory as fp32; `n` of them exist (0..8), the rest read as zero.
// `wide`: p is aligned for vector loads.
template <typename T>
__device__ __forceinline__ void mx_load8(const T* p, int n, bool wide, float (&x)[8]) {
  if (wide && n == 8) {
    if (sizeof(T) == 4) {
      const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
      x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    } else {
      const uint4 a = __ldg(reinterpret_cast<const uint4*>(p));
      const T* v = reinterpret_cast<const T*>(&a);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = mx_to_float(v[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = i < n ? mx_to_float(p[i]) : 0.f;
  }
}

// Scales, rounds and packs eight elements: one word of 4-bit codes, or two words of 8-bit codes.
template <int BITS, typename T>
__device__ __forceinline__ void mx_encode8(const float (&x)[8], uint32_t E, uint32_t (&w)[BITS / 4]) {
  const float inv = E == 255u ? 0.f : mx_inverse_scale(E);
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = x[i] * inv;
  if (BITS == 4) {
    w[0] = mx_pack4(y);
  } else {
    if (E == MxSource<T>::kTop8) {
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = fminf(fmaxf(y[i], -240.f), 240.f);
    }
    w[0] = mx_pack8(y[0], y[1], y[2], y[3]);
    w[BITS / 4 - 1] = mx_pack8(y[4], y[5], y[6], y[7]);
  }
}

struct MxQuantArgs {
  const void* x;
  long long ldx, stride_x;  // elements
  uint8_t* codes;           // [l][rows][pitch]
  uint8_t* scales;          // [l][row groups][k groups][512]
  int rows, k, l;
};

// Blocks of the three kernels below count groups along k first, then along the rows, then batches.
__device__ __forceinline__ void mx_group_of_block(int rows, int k, int& kg, int& rg, long long& b) {
  const uint32_t kgs = static_cast<uint32_t>((k + kMxGroupK - 1) / kMxGroupK);
  const uint32_t rgs = static_cast<uint32_t>((rows + kMxGroupRows - 1) / kMxGroupRows);
  const uint32_t rest = blockIdx.x / kgs;
  kg = static_cast<int>(blockIdx.x - rest * kgs);
  b = rest / rgs;
  rg = static_cast<int>(rest - static_cast<uint32_t>(b) * rgs);
}

// Source [l][rows][k], k contiguous. One CTA of 256 threads per scale group (128 rows x 128 k): a
// thread takes eight elements of a row at a time, four lanes make a block (its largest magnitude by
// two shuffles on the fp32 bits, whose order is that of the magnitudes, NaN above all), 16 lanes a
// row of the group, so loads are 256 contiguous bytes per row of a 16-bit source. The group's 512
// scale bytes are gathered in shared memory and leave as one contiguous piece.
template <int BITS, typename T>
__global__ void __launch_bounds__(256) mx_quantize_kernel(const MxQuantArgs a) {
  __shared__ __align__(16) uint8_t sc[kMxGroupBytes];
  int kg, rg;
  long long b;
  mx_group_of_block(a.rows, a.k, kg, rg, b);
  const int lane16 = threadIdx.x & 15, sub = threadIdx.x >> 4;
  const int k0 = kg * kMxGroupK + lane16 * 8;
  const long long pitch = mx_pitch(a.k, BITS);
  const T* X = static_cast<const T*>(a.x) + b * a.stride_x;
  uint8_t* codes = a.codes + b * a.rows * pitch;
  const bool wide = ((reinterpret_cast<uintptr_t>(a.x) | (a.ldx * sizeof(T)) | (a.stride_x * sizeof(T))) & 15) == 0;
  const int n = min(max(a.k - k0, 0), 8);
  const int rows_here = min(a.rows - rg * kMxGroupRows, kMxGroupRows);
  const bool stored = k0 < static_cast<int>(pitch * 8 / BITS);  // the padding of the last block is stored too
  if (rows_here < kMxGroupRows || kg * kMxGroupK + kMxGroupK > a.k) {
    if (threadIdx.x < 32) reinterpret_cast<uint4*>(sc)[threadIdx.x] = make_uint4(0, 0, 0, 0);
    __syncthreads();
  }
  constexpr int kBatch = 4;  // rows per thread whose loads are in flight together
#pragma unroll
  for (int r0 = 0; r0 < kMxGroupRows / 16; r0 += kBatch) {
    if (r0 * 16 >= rows_here) break;
    float x[kBatch][8];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int r = (r0 + j) * 16 + sub;
      const long long row = static_cast<long long>(rg) * kMxGroupRows + r;
      mx_load8<T>(X + row * a.ldx + k0, r < rows_here ? n : 0, wide, x[j]);
    }
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int r = (r0 + j) * 16 + sub;
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(x[j][i]) & 0x7fffffffu);
      m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
      m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
      const uint32_t E = mx_scale_byte<BITS, T>(m);
      uint32_t w[BITS / 4];
      mx_encode8<BITS, T>(x[j], E, w);
      if (r < rows_here && stored) {
        uint8_t* at = codes + (static_cast<long long>(rg) * kMxGroupRows + r) * pitch + static_cast<long long>(k0) * BITS / 8;
        if (BITS == 4) *reinterpret_cast<uint32_t*>(at) = w[0];
        else *reinterpret_cast<uint2*>(at) = make_uint2(w[0], w[BITS / 4 - 1]);
        if ((lane16 & 3) == 0) sc[mx_scale_at(r, lane16 >> 2)] = static_cast<uint8_t>(E);
      }
    }
  }
  __syncthreads();
  uint8_t* out = a.scales + b * mx_scale_bytes(a.rows, a.k) +
                 (static_cast<long long>(rg) * ((a.k + kMxGroupK - 1) / kMxGroupK) + kg) * kMxGroupBytes;
  if (threadIdx.x < 32) reinterpret_cast<uint4*>(out)[threadIdx.x] = reinterpret_cast<const uint4*>(sc)[threadIdx.x];
}

// Source [l][k][rows], rows contiguous (a matrix quantised along its first dimension). Same group
// per CTA; a thread owns one row of the group and half of its blocks: loads run along the rows (32 lanes on
// consecutive rows), the block's largest magnitude needs no other lane, and the codes cross shared
// memory so that they leave as whole row pieces.
template <int BITS, typename T>
__global__ void __launch_bounds__(256) mx_quantize_t_kernel(const MxQuantArgs a) {
  constexpr int kRowBytes = kMxGroupK * BITS / 8;  // 64 or 128 bytes of codes per row of a group
  constexpr int kPad = 16;
  __shared__ __align__(16) uint8_t sc[kMxGroupBytes];
  __shared__ __align__(16) uint8_t st[kMxGroupRows * (kRowBytes + kPad)];
  int kg, rg;
  long long b;
  mx_group_of_block(a.rows, a.k, kg, rg, b);
  const int r = threadIdx.x & 127, half = threadIdx.x >> 7;
  const int row = rg * kMxGroupRows + r;
  const bool row_ok = row < a.rows;
  const T* X = static_cast<const T*>(a.x) + b * a.stride_x + row;
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int blk = half * 2 + q;
    const int k0 = kg * kMxGroupK + blk * kMxBlock;
    float x[32];
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      x[i] = (row_ok && k0 + i < a.k) ? mx_to_float(X[static_cast<long long>(k0 + i) * a.ldx]) : 0.f;
      m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
    }
    const bool real = row_ok && k0 < a.k;
    const uint32_t E = real ? mx_scale_byte<BITS, T>(m) : 0u;
    sc[mx_scale_at(r, blk)] = static_cast<uint8_t>(E);
    uint32_t w[4][BITS / 4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      float y[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = x[c * 8 + i];
      mx_encode8<BITS, T>(y, E, w[c]);
    }
    uint4* at = reinterpret_cast<uint4*>(st + r * (kRowBytes + kPad) + blk * (kMxBlock * BITS / 8));
    if (BITS == 4) {
      at[0] = make_uint4(w[0][0], w[1][0], w[2][0], w[3][0]);
    } else {
      constexpr int h = BITS / 4 - 1;
      at[0] = make_uint4(w[0][0], w[0][h], w[1][0], w[1][h]);
      at[1] = make_uint4(w[2][0], w[2][h], w[3][0], w[3][h]);
    }
  }
  __syncthreads();
  const long long pitch = mx_pitch(a.k, BITS);
  uint8_t* codes = a.codes + b * a.rows * pitch;
  constexpr int kChunks = kRowBytes / 16;
  for (int i = threadIdx.x; i < kMxGroupRows * kChunks; i += 256) {
    const int rr = i / kChunks, c = i % kChunks;
    const long long off = static_cast<long long>(kg) * kRowBytes + c * 16;
    if (rg * kMxGroupRows + rr < a.rows && off < pitch)
      *reinterpret_cast<uint4*>(codes + (static_cast<long long>(rg) * kMxGroupRows + rr) * pitch + off) =
          *reinterpret_cast<const uint4*>(st + rr * (kRowBytes + kPad) + c * 16);
  }
  uint8_t* out = a.scales + b * mx_scale_bytes(a.rows, a.k) +
                 (static_cast<long long>(rg) * ((a.k + kMxGroupK - 1) / kMxGroupK) + kg) * kMxGroupBytes;
  if (threadIdx.x < 32) reinterpret_cast<uint4*>(out)[threadIdx.x] = reinterpret_cast<const uint4*>(sc)[threadIdx.x];
}

__device__ __forceinline__ void mx_store(float* p, float v) { *p = v; }
__device__ __forceinline__ void mx_store(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void mx_store(__half* p, float v) { *p = __float2half_rn(v); }

struct MxDequantArgs {
  const uint8_t* codes;
  const uint8_t* scales;
  long long stride_codes, stride_scales;  // bytes, 0 = the same matrix for every batch
  void* out;
  long long ldo, stride_o;  // elements
  int rows, k, l;
};

// The inverse: element * 2^(E - 127), exact in fp32, rounded once to the output type. The same
// groups and lanes as mx_quantize_kernel.
template <int BITS, typename T>
__global__ void __launch_bounds__(256) mx_dequantize_kernel(const MxDequantArgs a) {
  __shared__ __align__(16) uint8_t sc[kMxGroupBytes];
  int kg, rg;
  long long b;
  mx_group_of_block(a.rows, a.k, kg, rg, b);
  const uint8_t* src = a.scales + b * a.stride_scales +
                       (static_cast<long long>(rg) * ((a.k + kMxGroupK - 1) / kMxGroupK) + kg) * kMxGroupBytes;
  const int lane16 = threadIdx.x & 15, sub = threadIdx.x >> 4;
  const int k0 = kg * kMxGroupK + lane16 * 8;
  const long long pitch = mx_pitch(a.k, BITS);
  const uint8_t* codes = a.codes + b * a.stride_codes;
  T* out = static_cast<T*>(a.out) + b * a.stride_o;
  const bool wide = ((reinterpret_cast<uintptr_t>(a.out) | (a.ldo * sizeof(T)) | (a.stride_o * sizeof(T))) & 15) == 0;
  const int n = min(max(a.k - k0, 0), 8);
  const int rows_here = min(a.rows - rg * kMxGroupRows, kMxGroupRows);
  uint32_t w[8][BITS / 4];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int r = j * 16 + sub;
#pragma unroll
    for (int q = 0; q < BITS / 4; ++q) w[j][q] = 0;
    if (r < rows_here && n > 0) {
      const uint8_t* at = codes + (static_cast<long long>(rg) * kMxGroupRows + r) * pitch + static_cast<long long>(k0) * BITS / 8;
      if (BITS == 4) {
        w[j][0] = __ldg(reinterpret_cast<const uint32_t*>(at));
      } else {
        const uint2 v = __ldg(reinterpret_cast<const uint2*>(at));
        w[j][0] = v.x; w[j][BITS / 4 - 1] = v.y;
      }
    }
  }
  if (threadIdx.x < 32) reinterpret_cast<uint4*>(sc)[threadIdx.x] = __ldg(reinterpret_cast<const uint4*>(src) + threadIdx.x);
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int r = j * 16 + sub;
    if (r >= rows_here || n == 0) continue;
    const float s = mx_scale_value(sc[mx_scale_at(r, lane16 >> 2)]);
    uint32_t h[4];
    if (BITS == 4) {
      mx_unpack4(w[j][0], h);
    } else {
      mx_unpack8(w[j][0], h[0], h[1]);
      mx_unpack8(w[j][BITS / 4 - 1], h[2], h[3]);
    }
    float x[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = mx_half2_floats(h[i]);
      x[2 * i] = f.x * s; x[2 * i + 1] = f.y * s;
    }
    T* at = out + (static_cast<long long>(rg) * kMxGroupRows + r) * a.ldo + k0;
    if (wide && n == 8) {
      if (sizeof(T) == 4) {
        reinterpret_cast<float4*>(at)[0] = make_float4(x[0], x[1], x[2], x[3]);
        reinterpret_cast<float4*>(at)[1] = make_float4(x[4], x[5], x[6], x[7]);
      } else {
        uint4 v;
        T* t = reinterpret_cast<T*>(&v);
#pragma unroll
        for (int i = 0; i < 8; ++i) mx_store(t + i, x[i]);
        *reinterpret_cast<uint4*>(at) = v;
      }
    } else {
      for (int i = 0; i < n; ++i) mx_store(at + i, x[i]);
    }
  }
}

}  // namespace fbmm
