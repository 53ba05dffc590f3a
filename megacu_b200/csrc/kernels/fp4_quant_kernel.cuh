// Quantisation of matrices to the 4-bit block formats, and the values back.
//
// Bound by memory: 2 (or 4) bytes read and 0.53-0.56 written per element, so
// the arithmetic has about 14 lane operations per 16-bit element. Every
// decision (scale and element) is the exact value's:
//  * MX divides by a power of two, which is exact.
//  * NV with 16-bit inputs: z / s is a multiple of 2^-2 (a tie) or at least
//    2^-14 away from every tie (11-bit over 4-bit mantissas), so rounding
//    z * (1 / s), which is within 2^-20, to multiples of 2^-16 restores every
//    tie and crosses none. One FMA with 1.5 * 2^7 and one subtraction do it.
//  * NV with 32-bit inputs compares |z| with the seven borders times s, each
//    exact in 32 bits; the scale divides with a sticky bit (round to odd).
#pragma once

#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "fp4_format.cuh"
#include "vec.cuh"

namespace megacu_b200 {

struct fp4_matrix_params {
  std::int64_t rows;     // rows of the quantised matrix
  std::int32_t cols;     // multiple of 32
  std::int64_t stride;   // elements between the rows of x (of x as stored)
  std::int32_t log2_scale;
  std::int32_t tiles;    // scale tiles per row tile
  std::uint32_t col_tiles;  // CTAs per row tile, each kQuantCols columns
  std::int32_t topk;     // > 0: row r is x's row slot_of_row[r] / topk
  std::int64_t x_rows;   // topk > 0: rows of x; an entry past them has no row
  std::int32_t const *slot_of_row;  // nullptr: every row; < 0: the row is left as it was
  std::uint8_t *data;    // [rows, cols / 2]
  std::uint8_t *scales;
};

// Scale byte and multiplier of one block. `bits` is the largest |x| as its
// 32-bit float pattern (so that NaN sorts above infinity above numbers).
struct fp4_block_scale {
  std::uint32_t byte;
  float mul;    // MX: z / scale = x * mul * mul2. NV: 16-bit x: x * mul; 32-bit x: see encode
  float mul2;
};

template <bool kNv, bool kWide>
__device__ __forceinline__ fp4_block_scale block_scale(std::uint32_t bits, int log2_scale) {
  fp4_block_scale b;
  b.mul2 = 1.0f;
  if (bits >= 0x7f800000u) {  // infinity or NaN: the whole block is NaN
    b.byte = kNv ? 0x7fu : 0xffu;
    b.mul = 0.0f;
    return b;
  }
  float const amax = __uint_as_float(bits);
  if constexpr (!kNv) {
    int const fl = bits >= 0x00800000u ? static_cast<int>(bits >> 23) - 127
                                       : 31 - __clz(static_cast<int>(bits)) - 149;
    int e = fl + log2_scale - 2;
    e = bits == 0 ? -127 : min(max(e, -127), 127);
    int const f = log2_scale - e;
    b.byte = static_cast<std::uint32_t>(e + 127);
    b.mul = pow2(min(max(f, -126), 126));
    if (f > 126) b.mul2 = pow2(f - 126);  // tiny blocks: exact in two steps
  } else {
    float const g = pow2(log2_scale);
    float const a = fminf(amax * g, 4096.0f);  // past 6 * 448 the scale stays 448
    float v;
    if constexpr (kWide) {
      v = __fdiv_rz(a, 6.0f);
      if (fmaf(-6.0f, v, a) != 0.0f) v = __uint_as_float(__float_as_uint(v) | 1u);
    } else {
      v = __fdiv_rn(a, 6.0f);
    }
    b.byte = to_e4m3(v);
    float const s = from_e4m3(b.byte);
    b.mul = s == 0.0f ? 0.0f : kWide ? s : __fdiv_rn(g, s);
    b.mul2 = g;
  }
  return b;
}

// z / scale ready for the conversion's rounding.
template <bool kNv, bool kWide>
__device__ __forceinline__ float scaled(float x, fp4_block_scale const &b) {
  if constexpr (!kNv) {
    return x * b.mul;
  } else if constexpr (!kWide) {
    return fmaf(x, b.mul, 192.0f) - 192.0f;
  } else {
    // The element's magnitude by exact comparisons; ties go to the even code.
    float const z = fabsf(x * b.mul2), s = b.mul;
    float q = z > 0.25f * s ? 0.5f : 0.0f;
    q = z >= 0.75f * s ? 1.0f : q;
    q = z > 1.25f * s ? 1.5f : q;
    q = z >= 1.75f * s ? 2.0f : q;
    q = z > 2.5f * s ? 3.0f : q;
    q = z >= 3.5f * s ? 4.0f : q;
    q = z > 5.0f * s ? 6.0f : q;
    return copysignf(s == 0.0f ? 0.0f : q, x);
  }
}

// Eight elements to one 32-bit word.
template <bool kNv, bool kWide>
__device__ __forceinline__ std::uint32_t encode8(float const *x, fp4_block_scale const &b) {
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float v = x[i];
    if constexpr (!kNv) {
      if (b.mul2 != 1.0f) v *= b.mul2;
    }
    y[i] = scaled<kNv, kWide>(v, b);
  }
  std::uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) w |= e2m1x2(y[2 * i], y[2 * i + 1]) << (8 * i);
  // A NaN block holds zeros; so does an NV block whose scale rounds to zero.
  bool const empty = kNv ? b.mul == 0.0f : b.byte == 0xffu;
  return empty ? 0u : w;
}

template <class T>
__device__ __forceinline__ std::uint32_t abs_bits(T v) {
  return __float_as_uint(to_f32(v)) & 0x7fffffffu;
}

// 16 consecutive elements, by 16-byte loads when the rows allow it.
template <class T, bool kVec>
__device__ __forceinline__ void load16(T const *p, T (&v)[16]) {
  if constexpr (kVec) {
    constexpr int kN = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < 16 / kN; ++i) {
      *reinterpret_cast<vec<T, kN> *>(&v[i * kN]) = load_vec<T, kN>(p + i * kN);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = p[i];
  }
}

inline constexpr int kQuantThreads = 256;
inline constexpr int kQuantCols = 256;  // columns of a CTA's tile of 128 rows

// A CTA quantises 128 rows x 256 columns: 16 lanes per row with 16 elements
// each (512 bytes of a 16-bit row, 128 bytes of elements out), so that it
// owns whole scale tiles and writes them as 16-byte vectors.
template <class T, bool kNv, bool kVec>
__global__ void __launch_bounds__(kQuantThreads) fp4_quantize_kernel(fp4_matrix_params p,
                                                                    T const *x) {
  constexpr bool kWide = std::is_same_v<T, float>;
  constexpr int kTileCols = fp4_tile_cols(kNv);
  constexpr int kTiles = kQuantCols / kTileCols;
  __shared__ alignas(16) std::uint8_t smem[kTiles * kScaleTileBytes];
  std::int64_t const row_tile = blockIdx.x / p.col_tiles;
  std::int64_t const row0 = row_tile * kScaleTileRows;
  int const col0 = static_cast<int>(blockIdx.x % p.col_tiles) * kQuantCols;
  int const lane16 = threadIdx.x % 16, sub = threadIdx.x / 16;
  int const col = col0 + lane16 * 16;
  for (int i = threadIdx.x; i < kTiles * kScaleTileBytes / 4; i += kQuantThreads) {
    reinterpret_cast<std::uint32_t *>(smem)[i] = 0;
  }
  __syncthreads();
  std::uint32_t done = 0;  // passes that wrote this thread's row
#pragma unroll 2
  for (int pass = 0; pass < kScaleTileRows / 16; ++pass) {
    int const r = pass * 16 + sub;
    std::int64_t const row = row0 + r;
    std::int64_t src = row;
    bool in = row < p.rows;
    if (in && p.slot_of_row != nullptr) {
      std::int32_t const slot = p.slot_of_row[row];
      in = slot >= 0;
      if (p.topk > 0) {
        src = slot / p.topk;
        in = in && src < p.x_rows;
      }
    }
    if (in) done |= 1u << pass;
    // Both lanes of an MX block are in or out together (cols % 32 == 0).
    if (!in || col >= p.cols) continue;
    T v[16];
    load16<T, kVec>(x + src * p.stride + col, v);
    std::uint32_t bits = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) bits = max(bits, abs_bits(v[i]));
    if constexpr (!kNv) {
      bits = max(bits, __shfl_xor_sync(3u << (threadIdx.x % 32 & ~1u), bits, 1));
    }
    fp4_block_scale const b = block_scale<kNv, kWide>(bits, p.log2_scale);
    float f[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) f[i] = to_f32(v[i]);
    uint2 out;
    out.x = encode8<kNv, kWide>(f, b);
    out.y = encode8<kNv, kWide>(f + 8, b);
    *reinterpret_cast<uint2 *>(p.data + row * (p.cols / 2) + col / 2) = out;
    if (kNv || lane16 % 2 == 0) {
      int const blk = lane16 * 16 / fp4_block(kNv);
      smem[blk / 4 * kScaleTileBytes + scale_byte(r, blk)] = static_cast<std::uint8_t>(b.byte);
    }
  }
  __syncthreads();
  int const tile0 = col0 / kTileCols;
  int const tiles = min(kTiles, p.tiles - tile0);
  std::uint8_t *const dst = p.scales + (row_tile * p.tiles + tile0) * kScaleTileBytes;
  if (p.slot_of_row == nullptr) {
    for (int i = threadIdx.x; i < tiles * kScaleTileBytes / 16; i += kQuantThreads) {
      reinterpret_cast<uint4 *>(dst)[i] = reinterpret_cast<uint4 const *>(smem)[i];
    }
  } else if (lane16 < tiles) {
    // Only the rows written above: their four bytes of each tile.
#pragma unroll
    for (int pass = 0; pass < kScaleTileRows / 16; ++pass) {
      if ((done >> pass & 1u) == 0) continue;
      int const at = lane16 * kScaleTileBytes + scale_byte(pass * 16 + sub, 0);
      *reinterpret_cast<std::uint32_t *>(dst + at) =
          *reinterpret_cast<std::uint32_t const *>(smem + at);
    }
  }
}

inline constexpr int kQuantTThreads = 512;

// The transpose: x is [cols, rows] as stored and its columns become the rows
// of the quantised matrix. A thread reads 32 elements down two neighbouring
// columns (a warp reads 64 neighbouring columns of each row, 128 bytes of a
// 16-bit type); the CTA's 128 x 256 tile of elements is turned in shared
// memory so that each row leaves as 128 contiguous bytes.
template <class T, bool kNv, bool kPair>
__global__ void __launch_bounds__(kQuantTThreads) fp4_quantize_t_kernel(fp4_matrix_params p,
                                                                       T const *x) {
  constexpr bool kWide = std::is_same_v<T, float>;
  constexpr int kTileCols = fp4_tile_cols(kNv);
  constexpr int kTiles = kQuantCols / kTileCols;
  __shared__ alignas(16) std::uint8_t scales[kTiles * kScaleTileBytes];
  __shared__ uint4 turned[kScaleTileRows][8];
  std::int64_t const row_tile = blockIdx.x / p.col_tiles;
  std::int64_t const row0 = row_tile * kScaleTileRows;
  int const col0 = static_cast<int>(blockIdx.x % p.col_tiles) * kQuantCols;
  for (int i = threadIdx.x; i < kTiles * kScaleTileBytes / 4; i += kQuantTThreads) {
    reinterpret_cast<std::uint32_t *>(scales)[i] = 0;
  }
  __syncthreads();
  int const r = threadIdx.x % 64 * 2, chunk = threadIdx.x / 64;
  std::int64_t const row = row0 + r;
  int const col = col0 + chunk * 32;
  if (col < p.cols && row < p.rows) {
    bool const two = row + 1 < p.rows;
    T v[2][32];
    T const *src = x + col * p.stride + row;
#pragma unroll
    for (int i = 0; i < 32; ++i, src += p.stride) {
      if constexpr (kPair) {
        vec<T, 2> const pair = *reinterpret_cast<vec<T, 2> const *>(src);
        v[0][i] = pair.v[0];
        v[1][i] = pair.v[1];
      } else {
        v[0][i] = src[0];
        v[1][i] = two ? src[1] : from_f32<T>(0.0f);
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (h == 1 && !two) break;
      std::uint32_t out[4];
      constexpr int kBlock = fp4_block(kNv);
#pragma unroll
      for (int k = 0; k < 32 / kBlock; ++k) {
        std::uint32_t bits = 0;
#pragma unroll
        for (int i = 0; i < kBlock; ++i) bits = max(bits, abs_bits(v[h][k * kBlock + i]));
        fp4_block_scale const b = block_scale<kNv, kWide>(bits, p.log2_scale);
#pragma unroll
        for (int i = 0; i < kBlock / 8; ++i) {
          float f[8];
#pragma unroll
          for (int c = 0; c < 8; ++c) f[c] = to_f32(v[h][k * kBlock + i * 8 + c]);
          out[k * (kBlock / 8) + i] = encode8<kNv, kWide>(f, b);
        }
        int const blk = chunk * (32 / kBlock) + k;
        scales[blk / 4 * kScaleTileBytes + scale_byte(r + h, blk)] =
            static_cast<std::uint8_t>(b.byte);
      }
      turned[r + h][chunk ^ (r / 2 % 8)] = make_uint4(out[0], out[1], out[2], out[3]);
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < kScaleTileRows * 8; i += kQuantTThreads) {
    int const rr = i / 8, c = i % 8;
    if (row0 + rr < p.rows && col0 + c * 32 < p.cols) {
      *reinterpret_cast<uint4 *>(p.data + (row0 + rr) * (p.cols / 2) + col0 / 2 + c * 16) =
          turned[rr][c ^ (rr / 2 % 8)];
    }
  }
  int const tile0 = col0 / kTileCols;
  int const tiles = min(kTiles, p.tiles - tile0);
  std::uint8_t *const dst = p.scales + (row_tile * p.tiles + tile0) * kScaleTileBytes;
  for (int i = threadIdx.x; i < tiles * kScaleTileBytes / 16; i += kQuantTThreads) {
    reinterpret_cast<uint4 *>(dst)[i] = reinterpret_cast<uint4 const *>(scales)[i];
  }
}

// The values: element * scale / g, exact in 32 bits and rounded once. A
// thread decodes 16 elements.
template <class T, bool kNv, bool kVec>
__global__ void __launch_bounds__(kQuantThreads) fp4_dequantize_kernel(fp4_matrix_params p, T *y) {
  int const per_row = p.cols / 16;
  std::int64_t const total = p.rows * per_row;
  std::int64_t const step = static_cast<std::int64_t>(gridDim.x) * kQuantThreads;
  for (std::int64_t i = static_cast<std::int64_t>(blockIdx.x) * kQuantThreads + threadIdx.x;
       i < total; i += step) {
    std::int64_t const row = i / per_row;
    int const col = static_cast<int>(i - row * per_row) * 16;
    uint2 const d = *reinterpret_cast<uint2 const *>(p.data + row * (p.cols / 2) + col / 2);
    int const blk = col / fp4_block(kNv);
    std::uint32_t const byte =
        p.scales[((row / kScaleTileRows) * p.tiles + blk / 4) * kScaleTileBytes +
                 scale_byte(static_cast<int>(row % kScaleTileRows), blk)];
    // scale / g as two factors, each a normal power of two (or e4m3 / 2^k).
    float s1, s2;
    if constexpr (kNv) {
      s1 = from_e4m3(byte);
      s2 = pow2(-p.log2_scale);
    } else {
      int const e = static_cast<int>(byte) - 127 - p.log2_scale;
      s1 = byte == 0xffu ? __int_as_float(0x7fffffff) : pow2(e / 2);
      s2 = pow2(e - e / 2);
    }
    T out[16];
#pragma unroll
    for (int b = 0; b < 8; ++b) {
      std::uint32_t const w = b < 4 ? d.x : d.y;
      float2 const f = __half22float2(from_e2m1x2(w >> (8 * (b % 4)) & 0xffu));
      out[2 * b] = from_f32<T>(f.x * s1 * s2);
      out[2 * b + 1] = from_f32<T>(f.y * s1 * s2);
    }
    T *const dst = y + row * p.stride + col;
    if constexpr (kVec) {
      constexpr int kN = 16 / sizeof(T);
#pragma unroll
      for (int c = 0; c < 16 / kN; ++c) {
        store_vec<T, kN>(dst + c * kN, *reinterpret_cast<vec<T, kN> const *>(&out[c * kN]));
      }
    } else {
#pragma unroll
      for (int c = 0; c < 16; ++c) dst[c] = out[c];
    }
  }
}

}  // namespace megacu_b200
