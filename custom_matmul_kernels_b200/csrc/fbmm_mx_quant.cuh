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
#include <type_traits>

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

__device__ __forceinline__ void mx_load_v8(const void* p, uint32_t* r) {  // 32 bytes, 32-byte aligned
  asm("ld.global.nc.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
      : "l"(p));
}
__device__ __forceinline__ void mx_store_v8(void* p, const uint32_t* r) {
  asm volatile("st.global.v8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
               "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "l"(p)
               : "memory");
}

// A block of 32 elements as raw words, packed two to a word for the 16-bit types.
template <typename T>
struct MxRaw {
  static constexpr int kWords = 32 * static_cast<int>(sizeof(T)) / 4;
  uint32_t w[kWords];

  // From contiguous storage; `n` (0..32) of the elements exist, the others are zero. `align`: bytes (32,
  // 16 or less) that every row of the matrix is aligned to.
  __device__ __forceinline__ void load(const T* p, int n, int align) {
    if (n == 32 && align >= 32) {
#pragma unroll
      for (int i = 0; i < kWords; i += 8) mx_load_v8(reinterpret_cast<const uint32_t*>(p) + i, w + i);
    } else if (n == 32 && align >= 16) {
#pragma unroll
      for (int i = 0; i < kWords; i += 4) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(p) + i / 4);
        w[i] = v.x; w[i + 1] = v.y; w[i + 2] = v.z; w[i + 3] = v.w;
      }
    } else {
      const bool whole = n == 32;
#pragma unroll
      for (int i = 0; i < kWords; ++i) {
        if (sizeof(T) == 4) {
          w[i] = whole || i < n ? __ldg(reinterpret_cast<const uint32_t*>(p) + i) : 0u;
        } else {
          const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
          const uint32_t lo = whole || 2 * i < n ? __ldg(h + 2 * i) : 0u;
          const uint32_t hi = whole || 2 * i + 1 < n ? __ldg(h + 2 * i + 1) : 0u;
          w[i] = lo | (hi << 16);
        }
      }
    }
  }

  // fp32 bits of the largest magnitude; infinity and NaN come out on top. The 16-bit types are compared as
  // packed pairs (one instruction per two elements).
  __device__ __forceinline__ uint32_t amax_bits() const;
  // Elements 8c .. 8c+7 times 2^(127 - E), as fp32: exact (what falls below the normal numbers rounds to zero
  // either way).
  __device__ __forceinline__ void scaled(int c, uint32_t E, float (&y)[8]) const;
};
template <>
__device__ __forceinline__ uint32_t MxRaw<float>::amax_bits() const {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 32; ++i) m = max(m, w[i] & 0x7fffffffu);
  return m;
}
template <>
__device__ __forceinline__ uint32_t MxRaw<__nv_bfloat16>::amax_bits() const {
  const __nv_bfloat162* v = reinterpret_cast<const __nv_bfloat162*>(w);
  __nv_bfloat162 m = __habs2(v[0]);
#pragma unroll
  for (int i = 1; i < 16; ++i) m = __hmax2_nan(m, __habs2(v[i]));
  const uint32_t b = *reinterpret_cast<const uint32_t*>(&m) & 0x7fff7fffu;
  return max(b << 16, b & 0xffff0000u);
}
template <>
__device__ __forceinline__ uint32_t MxRaw<__half>::amax_bits() const {
  const __half2* v = reinterpret_cast<const __half2*>(w);
  __half2 m = __habs2(v[0]);
#pragma unroll
  for (int i = 1; i < 16; ++i) m = __hmax2_nan(m, __habs2(v[i]));
  const float2 f = __half22float2(m);
  return max(__float_as_uint(f.x) & 0x7fffffffu, __float_as_uint(f.y) & 0x7fffffffu);
}
template <>
__device__ __forceinline__ void MxRaw<float>::scaled(int c, uint32_t E, float (&y)[8]) const {
  const float inv = mx_inverse_scale(E);
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = __uint_as_float(w[c * 8 + i]) * inv;
}
template <>
__device__ __forceinline__ void MxRaw<__nv_bfloat16>::scaled(int c, uint32_t E, float (&y)[8]) const {
  const float inv = mx_inverse_scale(E);  // its upper half is the same power of two as bf16
  const uint32_t h = __byte_perm(__float_as_uint(inv), 0, 0x3232);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 v = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&w[c * 4 + i]),
                                     *reinterpret_cast<const __nv_bfloat162*>(&h));
    const uint32_t b = *reinterpret_cast<const uint32_t*>(&v);
    y[2 * i] = __uint_as_float(b << 16);
    y[2 * i + 1] = __uint_as_float(b & 0xffff0000u);
  }
}
template <>
__device__ __forceinline__ void MxRaw<__half>::scaled(int c, uint32_t E, float (&y)[8]) const {
  const float inv = mx_inverse_scale(E);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = mx_half2_floats(w[c * 4 + i]);
    y[2 * i] = f.x * inv;
    y[2 * i + 1] = f.y * inv;
  }
}

// The codes of a block with scale byte E: 4 words of 4-bit or 8 words of 8-bit codes.
template <int BITS, typename T>
__device__ __forceinline__ void mx_encode(const MxRaw<T>& x, uint32_t E, uint32_t (&out)[BITS]) {
  const bool top = BITS == 8 && E == MxSource<T>::kTop8;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    float y[8];
    x.scaled(c, min(E, 254u), y);
    if (BITS == 4) {
      out[c] = mx_pack4(y);
    } else {
      if (top) {
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = fminf(fmaxf(y[i], -240.f), 240.f);
      }
      out[2 * c] = mx_pack8(y[0], y[1], y[2], y[3]);
      out[(2 * c + 1) & (BITS - 1)] = mx_pack8(y[4], y[5], y[6], y[7]);
    }
  }
}

struct MxQuantArgs {
  const void* x;
  long long ldx, stride_x;  // elements
  uint8_t* codes;           // [l][rows][pitch]
  uint8_t* scales;          // [l][row groups][k groups][512]
  int rows, k, l;
};

// Programmatic dependent launch: the products may start while the kernel ahead of them in the stream still
// runs (the quantisers let them at once), and none of their copies of what it may have written leaves before it
// is complete and visible. Without such a launch both do nothing.
__device__ __forceinline__ void mx_let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void mx_wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Blocks of the three kernels below count groups along k first, then along the rows, then batches.
__device__ __forceinline__ void mx_group_of_block(int rows, int k, int& kg, int& rg, long long& b) {
  const uint32_t kgs = static_cast<uint32_t>((k + kMxGroupK - 1) / kMxGroupK);
  const uint32_t rgs = static_cast<uint32_t>((rows + kMxGroupRows - 1) / kMxGroupRows);
  const uint32_t rest = blockIdx.x / kgs;
  kg = static_cast<int>(blockIdx.x - rest * kgs);
  b = rest / rgs;
  rg = static_cast<int>(rest - static_cast<uint32_t>(b) * rgs);
}

// Bytes (32, 16, or the element size) that every row of a matrix is aligned to.
template <typename T>
__device__ __forceinline__ int mx_row_alignment(const void* p, long long ld, long long stride) {
  const uint64_t bits = reinterpret_cast<uintptr_t>(p) | static_cast<uint64_t>(ld * sizeof(T)) |
                        static_cast<uint64_t>(stride * sizeof(T));
  return (bits & 31) == 0 ? 32 : (bits & 15) == 0 ? 16 : static_cast<int>(sizeof(T));
}

// Source [l][rows][k], k contiguous. One CTA of 256 threads per scale group (128 rows x 128 k), a thread
// per block, two in turn: 64 to 128 contiguous bytes of the source in 32-byte loads, no exchange between
// threads. Four neighbouring lanes cover a row of the group (its codes are 64 or 128 contiguous bytes), and
// the 32 scale bytes of a warp are 8 whole words of one 128-byte line of the group. Bound by the memory
// traffic: 8192 x 8192 bf16 to 4 bits 26.1 us, 6.5 TB/s (eight elements a thread with shuffles for the
// block's largest magnitude: 54 us).
template <int BITS, typename T>
__global__ void __launch_bounds__(256) mx_quantize_kernel(const MxQuantArgs a) {
  mx_let_next_start();
  int kg, rg;
  long long b;
  mx_group_of_block(a.rows, a.k, kg, rg, b);
  const int blk = threadIdx.x & 3, sub = threadIdx.x >> 2;
  const int k0 = kg * kMxGroupK + blk * kMxBlock;
  const long long pitch = mx_pitch(a.k, BITS);
  const T* X = static_cast<const T*>(a.x) + b * a.stride_x;
  uint8_t* codes = a.codes + b * a.rows * pitch;
  uint8_t* group = a.scales + b * mx_scale_bytes(a.rows, a.k) +
                   (static_cast<long long>(rg) * ((a.k + kMxGroupK - 1) / kMxGroupK) + kg) * kMxGroupBytes;
  const int align = mx_row_alignment<T>(a.x, a.ldx, a.stride_x);
  const int n = min(max(a.k - k0, 0), kMxBlock);
  MxRaw<T> x[2];
  if (align >= 16) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const long long row = static_cast<long long>(rg) * kMxGroupRows + j * 64 + sub;
      x[j].load(X + row * a.ldx + k0, row < a.rows ? n : 0, align);
    }
  } else {
    // rows at any alignment: single-element loads run along the rows (a warp on 8 rows, 32 neighbouring elements
    // a load) and cross shared memory (fp16 3 x 1003 x 1111 to 8 bits: 7.0 us with a block's elements loaded by
    // its thread, 5.4 us this way)
    using Word = typename std::conditional<sizeof(T) == 4, uint32_t, uint16_t>::type;
    constexpr int kPitch = kMxGroupK * static_cast<int>(sizeof(T)) + 16;
    __shared__ __align__(16) uint8_t tile[64 * kPitch];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int cols = min(a.k - kg * kMxGroupK, kMxGroupK);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      Word e[8][4];
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const long long row = static_cast<long long>(rg) * kMxGroupRows + j * 64 + warp * 8 + q;
        const Word* p = reinterpret_cast<const Word*>(X + row * a.ldx + kg * kMxGroupK) + lane;
#pragma unroll
        for (int i = 0; i < 4; ++i) e[q][i] = row < a.rows && i * 32 + lane < cols ? __ldg(p + i * 32) : Word(0);
      }
      __syncthreads();
#pragma unroll
      for (int q = 0; q < 8; ++q)
#pragma unroll
        for (int i = 0; i < 4; ++i) reinterpret_cast<Word*>(tile + (warp * 8 + q) * kPitch)[i * 32 + lane] = e[q][i];
      __syncthreads();
      const uint4* from = reinterpret_cast<const uint4*>(tile + sub * kPitch + blk * (kMxBlock * static_cast<int>(sizeof(T))));
#pragma unroll
      for (int i = 0; i < MxRaw<T>::kWords; i += 4) {
        const uint4 v = from[i / 4];
        x[j].w[i] = v.x; x[j].w[i + 1] = v.y; x[j].w[i + 2] = v.z; x[j].w[i + 3] = v.w;
      }
    }
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int r = j * 64 + sub;
    const long long row = static_cast<long long>(rg) * kMxGroupRows + r;
    const bool real = row < a.rows && n > 0;
    const uint32_t E = real ? mx_scale_byte<BITS, T>(x[j].amax_bits()) : 0u;
    group[mx_scale_at(r, blk)] = static_cast<uint8_t>(E);
    if (real) {
      uint32_t c[BITS];
      mx_encode<BITS, T>(x[j], E, c);
      uint4* at = reinterpret_cast<uint4*>(codes + row * pitch + static_cast<long long>(k0) * BITS / 8);
      at[0] = make_uint4(c[0], c[1], c[2], c[3]);
      if (BITS == 8) at[1] = make_uint4(c[BITS - 4], c[BITS - 3], c[BITS - 2], c[BITS - 1]);
    }
  }
}

// Source [l][k][rows], rows contiguous (a matrix quantised along its first dimension). Same group
// per CTA. A thread owns a block of a row (two neighbouring rows where the source is 16-bit and
// aligned for pairs), so loads run along the rows, 128 bytes per warp, 32 of them in flight, and the block's
// largest magnitude needs no other thread. The codes cross shared memory so that they leave as whole row
// pieces. 8192 x 8192 bf16 to 4 bits 27.7 us, 6.1 TB/s (41 us while every load carried its own bounds
// check: instruction issue was the limit).
template <int BITS, typename T>
__global__ void __launch_bounds__(256, 4) mx_quantize_t_kernel(const MxQuantArgs a) {
  mx_let_next_start();
  constexpr int kRowBytes = kMxGroupK * BITS / 8;  // 64 or 128 bytes of codes per row of a group
  constexpr int kPad = 16;
  __shared__ __align__(16) uint8_t sc[kMxGroupBytes];
  __shared__ __align__(16) uint8_t st[kMxGroupRows * (kRowBytes + kPad)];
  // groups along the rows first: neighbouring CTAs read neighbouring pieces of the same source rows
  const uint32_t kgs = static_cast<uint32_t>((a.k + kMxGroupK - 1) / kMxGroupK);
  const uint32_t rgs = static_cast<uint32_t>((a.rows + kMxGroupRows - 1) / kMxGroupRows);
  const uint32_t rest = blockIdx.x / rgs;
  const int rg = static_cast<int>(blockIdx.x - rest * rgs);
  const long long b = rest / kgs;
  const int kg = static_cast<int>(rest - static_cast<uint32_t>(b) * kgs);
  const T* X = static_cast<const T*>(a.x) + b * a.stride_x;
  const bool pairs = sizeof(T) == 2 && ((reinterpret_cast<uintptr_t>(a.x) | static_cast<uint64_t>(a.ldx * 2) |
                                         static_cast<uint64_t>(a.stride_x * 2)) & 3) == 0;
  // a row's place in the staging area: lanes that hold every other row still write to different banks
  auto slot = [&](int r) -> int { return pairs ? (r >> 1) + (r & 1) * 64 : r; };
  auto put = [&](int r, int blk, const MxRaw<T>& x, bool real) {
    const uint32_t E = real ? mx_scale_byte<BITS, T>(x.amax_bits()) : 0u;
    sc[mx_scale_at(r, blk)] = static_cast<uint8_t>(E);
    uint32_t c[BITS];
    mx_encode<BITS, T>(x, E, c);
    uint4* at = reinterpret_cast<uint4*>(st + slot(r) * (kRowBytes + kPad) + blk * (kMxBlock * BITS / 8));
    at[0] = make_uint4(c[0], c[1], c[2], c[3]);
    if (BITS == 8) at[1] = make_uint4(c[BITS - 4], c[BITS - 3], c[BITS - 2], c[BITS - 1]);
  };
  const int row0 = rg * kMxGroupRows;
  const bool whole = row0 + kMxGroupRows <= a.rows && kg * kMxGroupK + kMxGroupK <= a.k;
  if (pairs) {
    const int r = (threadIdx.x & 63) * 2, blk = threadIdx.x >> 6;
    const int k0 = kg * kMxGroupK + blk * kMxBlock;
    const int have = min(max(a.rows - (row0 + r), 0), 2);  // rows of this pair
    uint32_t v[32];
    const T* p = X + static_cast<long long>(k0) * a.ldx + row0 + r;
    if (whole) {
#pragma unroll
      for (int i = 0; i < 32; ++i, p += a.ldx) v[i] = __ldg(reinterpret_cast<const uint32_t*>(p));
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i, p += a.ldx) {
        v[i] = 0;
        if (k0 + i < a.k) {
          if (have == 2) v[i] = __ldg(reinterpret_cast<const uint32_t*>(p));
          else if (have == 1) v[i] = __ldg(reinterpret_cast<const uint16_t*>(p));
        }
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      MxRaw<T> x;
#pragma unroll
      for (int i = 0; i < MxRaw<T>::kWords; ++i)
        x.w[i] = __byte_perm(v[(2 * i) & 31], v[(2 * i + 1) & 31], h ? 0x7632 : 0x5410);
      put(r + h, blk, x, h < have && k0 < a.k);
    }
  } else {
    const int r = threadIdx.x & 127;
    const bool row_ok = row0 + r < a.rows;
#pragma unroll 1
    for (int q = 0; q < 2; ++q) {
      const int blk = (threadIdx.x >> 7) * 2 + q;
      const int k0 = kg * kMxGroupK + blk * kMxBlock;
      MxRaw<T> x;
      const T* p = X + static_cast<long long>(k0) * a.ldx + row0 + r;
      uint32_t e[32];
      auto word = [](const T* at) -> uint32_t {
        return sizeof(T) == 4 ? __ldg(reinterpret_cast<const uint32_t*>(at)) : __ldg(reinterpret_cast<const uint16_t*>(at));
      };
      if (whole) {
#pragma unroll
        for (int i = 0; i < 32; ++i, p += a.ldx) e[i] = word(p);
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i, p += a.ldx) e[i] = row_ok && k0 + i < a.k ? word(p) : 0u;
      }
#pragma unroll
      for (int i = 0; i < MxRaw<T>::kWords; ++i)
        x.w[i] = sizeof(T) == 4 ? e[i & 31] : e[(2 * i) & 31] | (e[(2 * i + 1) & 31] << 16);
      put(r, blk, x, row_ok && k0 < a.k);
    }
  }
  __syncthreads();
  const long long pitch = mx_pitch(a.k, BITS);
  uint8_t* codes = a.codes + b * a.rows * pitch;
  constexpr int kChunks = kRowBytes / 16;
  for (int i = threadIdx.x; i < kMxGroupRows * kChunks; i += 256) {
    const int rr = i / kChunks, c = i % kChunks;
    const long long off = static_cast<long long>(kg) * kRowBytes + c * 16;
    if (row0 + rr < a.rows && off < pitch)
      *reinterpret_cast<uint4*>(codes + static_cast<long long>(row0 + rr) * pitch + off) =
          *reinterpret_cast<const uint4*>(st + slot(rr) * (kRowBytes + kPad) + c * 16);
  }
  uint8_t* out = a.scales + b * mx_scale_bytes(a.rows, a.k) +
                 (static_cast<long long>(rg) * ((a.k + kMxGroupK - 1) / kMxGroupK) + kg) * kMxGroupBytes;
  if (threadIdx.x < 32) reinterpret_cast<uint4*>(out)[threadIdx.x] = reinterpret_cast<const uint4*>(sc)[threadIdx.x];
}

struct MxDequantArgs {
  const uint8_t* codes;
  const uint8_t* scales;
  long long stride_codes, stride_scales;  // bytes, 0 = the same matrix for every batch
  void* out;
  long long ldo, stride_o;  // elements
  int rows, k, l;
};

// 16 codes as eight packed pairs of 16-bit values, scaled by 2^(E - 127).
//
// The fast form moves the code's fields to where the 16-bit type has them (sign to bit 15, exponent
// and mantissa as one piece, zero and subnormal codes included), which gives the value times a
// power of two (bf16: 2^-120 for e4m3 and 2^-126 for e2m1; fp16: 2^-8 and 2^-14), and multiplies
// packed pairs by the power of two that is left: four or five integer instructions and one
// multiplication per pair, where converting through fp16 and fp32 takes one slow conversion and five
// more instructions. It rounds once, in that multiplication. Scales whose remaining power the
// type cannot hold as a normal number, the NaN scale, and 8-bit NaN codes (mx_nan_codes) take the general form.
template <int BITS, bool BF16>
struct MxFast {
  static constexpr int kBias = BF16 ? (BITS == 8 ? 120 : 126) : (BITS == 8 ? -104 : -98);  // E + kBias = exponent field
  static constexpr int kTop = BF16 ? 254 : 30;
  __device__ static __forceinline__ bool in_range(uint32_t E) {
    const int f = static_cast<int>(E) + kBias;
    return f >= 1 && f <= kTop;
  }
  __device__ static __forceinline__ uint32_t scale(uint32_t E) {  // both halves
    return ((E + static_cast<uint32_t>(kBias)) << (BF16 ? 7 : 10)) * 0x10001u;
  }
};
// Non-zero where one of 8-bit codes is 0x7f or 0xff: adding one to every byte carries into bit 7 where the lower seven
// bits are all set. A carry that leaves a byte comes from 0xff, so what it does to the next changes no answer.
// Two instructions per four codes: 8-bit gradient of weights 8192 x 4096 x 4096 212 -> 220 us (with three-input maxima of the
// shifted codes 223 us).
template <int BITS>
__device__ __forceinline__ uint32_t mx_nan_codes(const uint32_t (&c)[BITS / 2]) {
  uint32_t any = 0;
  if (BITS == 8) {
#pragma unroll
    for (int q = 0; q < BITS / 2; ++q) any |= (c[q] + 0x01010101u) ^ c[q];
  }
  return any & 0x80808080u;
}
template <bool BF16>
__device__ __forceinline__ uint32_t mx_mul2(uint32_t a, uint32_t b) {
  uint32_t r;
  if (BF16) asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <bool BF16>
__device__ __forceinline__ uint32_t mx_pack16(float a, float b) {
  if (BF16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <int BITS>
__device__ __forceinline__ void mx_unpack16(const uint32_t (&c)[BITS / 2], uint32_t (&h)[8]) {  // halves, unscaled
  if (BITS == 8) {
#pragma unroll
    for (int q = 0; q < 4; ++q) mx_unpack8(c[q & (BITS / 2 - 1)], h[2 * q], h[2 * q + 1]);
  } else {
    uint32_t a[4], b[4];
    mx_unpack4(c[0], a);
    mx_unpack4(c[1], b);
#pragma unroll
    for (int q = 0; q < 4; ++q) { h[q] = a[q]; h[q + 4] = b[q]; }
  }
}
template <int BITS, bool BF16>
__device__ __forceinline__ void mx_values16(const uint32_t (&c)[BITS / 2], uint32_t E, bool fast, uint32_t (&w)[8]) {
  if (fast) {
    const uint32_t s = MxFast<BITS, BF16>::scale(E);
    if (BITS == 8) {
      constexpr int kShift = BF16 ? 4 : 1;
      constexpr uint32_t kMag = BF16 ? 0x07f007f0u : 0x3f803f80u;
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const uint32_t t = __byte_perm(c[q >> 1], 0, (q & 1) ? 0x3424 : 0x1404);  // two codes, each in a high byte
        w[q] = mx_mul2<BF16>(((t >> kShift) & kMag) | (t & 0x80008000u), s);
      }
    } else {
      constexpr int kShift = BF16 ? 6 : 9;
      constexpr uint32_t kMag = 7u * 0x10001u << kShift;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t y[4];  // elements i and i + 4 of the word
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t m = 4 * i <= kShift ? c[h] << (kShift - 4 * i) : c[h] >> (4 * i - kShift);
          y[i] = mx_mul2<BF16>((m & kMag) | ((c[h] << (12 - 4 * i)) & 0x80008000u), s);
        }
        w[h * 4 + 0] = __byte_perm(y[0], y[1], 0x5410);
        w[h * 4 + 1] = __byte_perm(y[2], y[3], 0x5410);
        w[h * 4 + 2] = __byte_perm(y[0], y[1], 0x7632);
        w[h * 4 + 3] = __byte_perm(y[2], y[3], 0x7632);
      }
    }
  } else {
    const float s = mx_scale_value(E);
    uint32_t h[8];
    mx_unpack16<BITS>(c, h);
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const float2 f = mx_half2_floats(h[q]);
      w[q] = mx_pack16<BF16>(f.x * s, f.y * s);
    }
  }
}

// The inverse: element * 2^(E - 127), exact in fp32, rounded once to the output type. The groups of
// mx_quantize_kernel, 16 elements a thread and step: eight neighbouring lanes write a row of the group (256 or 512
// contiguous bytes) in 32-byte stores. 8192 x 8192 from 4 bits to
// bf16 28.9 us, 5.9 TB/s.
template <int BITS, typename T>
__global__ void __launch_bounds__(256) mx_dequantize_kernel(const MxDequantArgs a) {
  int kg, rg;
  long long b;
  mx_group_of_block(a.rows, a.k, kg, rg, b);
  const uint8_t* group = a.scales + b * a.stride_scales +
                         (static_cast<long long>(rg) * ((a.k + kMxGroupK - 1) / kMxGroupK) + kg) * kMxGroupBytes;
  const int u = threadIdx.x & 7, sub = threadIdx.x >> 3;
  const int k0 = kg * kMxGroupK + u * 16;
  const int n = min(max(a.k - k0, 0), 16);
  const long long pitch = mx_pitch(a.k, BITS);
  const uint8_t* codes = a.codes + b * a.stride_codes + static_cast<long long>(k0) * BITS / 8;
  T* out = static_cast<T*>(a.out) + b * a.stride_o + k0;
  const int align = mx_row_alignment<T>(a.out, a.ldo, a.stride_o);
  __shared__ uint32_t lines[8][4 * 128 * sizeof(T) / 4];  // per warp, four rows of the group
  uint32_t c[4][BITS / 2], E[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int r = j * 32 + sub;
    const long long row = static_cast<long long>(rg) * kMxGroupRows + r;
#pragma unroll
    for (int q = 0; q < BITS / 2; ++q) c[j][q] = 0;
    E[j] = 127;
    if (row < a.rows && n > 0) {
      if (BITS == 4) {
        const uint2 v = __ldg(reinterpret_cast<const uint2*>(codes + row * pitch));
        c[j][0] = v.x; c[j][1] = v.y;
      } else {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(codes + row * pitch));
        c[j][0] = v.x; c[j][1] = v.y; c[j][BITS / 2 - 2] = v.z; c[j][BITS / 2 - 1] = v.w;
      }
      E[j] = __ldg(group + mx_scale_at(r, u >> 1));
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const long long row = static_cast<long long>(rg) * kMxGroupRows + j * 32 + sub;
    T* at = out + row * a.ldo;
    constexpr int kWords = 16 * static_cast<int>(sizeof(T)) / 4;
    uint32_t w[kWords];
    if (sizeof(T) == 2) {
      constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
      uint32_t v[8];
      mx_values16<BITS, kBf16>(c[j], E[j], MxFast<BITS, kBf16>::in_range(E[j]) && mx_nan_codes<BITS>(c[j]) == 0, v);
#pragma unroll
      for (int q = 0; q < 8; ++q) w[q] = v[q];
    } else {
      const float s = mx_scale_value(E[j]);
      uint32_t h[8];
      mx_unpack16<BITS>(c[j], h);
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const float2 f = mx_half2_floats(h[q]);
        w[(2 * q) % kWords] = __float_as_uint(f.x * s);
        w[(2 * q + 1) % kWords] = __float_as_uint(f.y * s);
      }
    }
    if (align >= 16) {
      if (row >= a.rows) continue;
      if (n == 16) {
        if (align >= 32) {
#pragma unroll
          for (int i = 0; i < kWords; i += 8) mx_store_v8(reinterpret_cast<uint32_t*>(at) + i, w + i);
        } else {
#pragma unroll
          for (int i = 0; i < kWords; i += 4)
            reinterpret_cast<uint4*>(at)[i / 4] = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (i < n) {
            if (sizeof(T) == 4) reinterpret_cast<uint32_t*>(at)[i] = w[i % kWords];
            else reinterpret_cast<uint16_t*>(at)[i] = static_cast<uint16_t>(w[i / 2] >> (16 * (i & 1)));
          }
      }
    } else {
      // rows at any alignment: the warp's four rows through shared memory, so that single-element stores
      // are at least neighbours (28 -> 4.5 us for 3 x 1003 x 1111 elements)
      uint32_t* mine = lines[threadIdx.x >> 5];
      __syncwarp();
#pragma unroll
      for (int i = 0; i < kWords; ++i) mine[(sub & 3) * (8 * kWords) + u * kWords + i] = w[i];
      __syncwarp();
      const T* from = reinterpret_cast<const T*>(mine);
      const int lane = threadIdx.x & 31;
      const int cols = min(a.k - kg * kMxGroupK, kMxGroupK);
      for (int rr = 0; rr < 4; ++rr) {
        const long long to = row - (sub & 3) + rr;
        if (to >= a.rows) break;
        T* line = static_cast<T*>(a.out) + b * a.stride_o + to * a.ldo + kg * kMxGroupK;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (i * 32 + lane < cols) line[i * 32 + lane] = from[rr * 128 + i * 32 + lane];
      }
    }
  }
}

}  // namespace fbmm
