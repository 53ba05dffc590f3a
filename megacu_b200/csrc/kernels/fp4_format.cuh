// 4-bit block formats: e2m1 elements (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign),
// two per byte, the lower nibble first, and one scale byte per block of a row.
//
//   MX  blocks of 32, scale 2^e (ue8m0), e = floor(log2 amax) - 2
//   NV  blocks of 16, scale e4m3 (unsigned), rne(min(amax / 6, 448))
//   z = g * x with g a power of two; value = element * scale / g
//
// Scale bytes lie in tiles of 128 rows x 4 blocks (512 bytes), the order the
// tensor core's scale operands take: row r, block b of a tile at byte
// (r % 32) * 16 + (r / 32) * 4 + b. Tiles of a row tile are contiguous along k.
#pragma once

#include <cuda_fp16.h>

#include <cstdint>

#if defined(__CUDACC__)
#define MEGACU_FP4_HD __host__ __device__
#else
#define MEGACU_FP4_HD
#endif

namespace megacu_b200 {

inline constexpr int kScaleTileRows = 128;
inline constexpr int kScaleTileBytes = 512;

MEGACU_FP4_HD constexpr int fp4_block(bool nv) { return nv ? 16 : 32; }
// Elements of a row that one scale tile covers.
MEGACU_FP4_HD constexpr int fp4_tile_cols(bool nv) { return 4 * fp4_block(nv); }
MEGACU_FP4_HD constexpr int scale_byte(int row, int block) {
  return (row % 32) * 16 + (row % 128) / 32 * 4 + block % 4;
}

#if defined(__CUDACC__)

// Eight floats to eight e2m1 (round to nearest even, saturating), f[0] in the
// lowest nibble.
__device__ __forceinline__ std::uint32_t e2m1x8(float const (&f)[8]) {
  std::uint32_t r;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(r)
      : "f"(f[0]), "f"(f[1]), "f"(f[2]), "f"(f[3]), "f"(f[4]), "f"(f[5]), "f"(f[6]), "f"(f[7]));
  return r;
}

// Eight e2m1 to four pairs.
__device__ __forceinline__ void from_e2m1x8(std::uint32_t w, __half2 (&h)[4]) {
  std::uint32_t r[4];
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
      : "r"(w));
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = *reinterpret_cast<__half2 *>(&r[i]);
}

// e4m3 of a non-negative float (round to nearest even, at most 448).
__device__ __forceinline__ std::uint32_t to_e4m3(float v) {
  std::uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.0f), "f"(v));
  return r & 0xffu;
}

__device__ __forceinline__ float from_e4m3(std::uint32_t byte) {
  std::uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(static_cast<std::uint16_t>(byte)));
  return __half2float(__ushort_as_half(static_cast<std::uint16_t>(r & 0xffffu)));
}

__device__ __forceinline__ float pow2(int e) {  // -126 <= e <= 127
  return __int_as_float((e + 127) << 23);
}

#endif  // __CUDACC__

}  // namespace megacu_b200
