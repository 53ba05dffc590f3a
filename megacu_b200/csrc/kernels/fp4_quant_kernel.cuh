// Quantisation of matrices to the 4-bit block formats, and the values back.
//
// Bound by memory as long as an element costs few instructions: 2 (or 4) bytes
// read and 0.53-0.56 written per element leave about 14 per 16-bit element at
// full issue rate. Every decision (scale and element) is the exact value's:
//  * MX divides by a power of two, which is exact.
//  * NV with 16-bit inputs: amax / 6 is a tie between two scales or at least
//    2^-11 of itself away from every tie (11-bit against 7-bit integers), so
//    amax * (1 / 6), within 2^-22, rounded to 13 significant bits restores
//    every tie and crosses none. Likewise z / s is a multiple of 2^-2 (a tie)
//    or at least 2^-14 away from one: z * (1 / s), within 2^-20, is rounded to
//    multiples of 2^-16 by one FMA with 1.5 * 2^7 and one subtraction.
//  * NV with 32-bit inputs compares |z| with the seven borders times s, each
//    exact in 32 bits; the scale divides with a sticky bit (round to odd).
#pragma once

#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "chained.cuh"
#include "fp4_format.cuh"
#include "vec.cuh"

namespace megacu_b200 {

struct fp4_matrix_params {
  std::int64_t rows;     // rows of the quantised matrix
  std::int32_t cols;     // multiple of 32
  std::int64_t stride;   // elements between the rows of x (of x as stored)
  std::int32_t log2_scale;
  std::int32_t tiles;    // scale tiles per row tile
  std::uint32_t col_tiles;  // CTAs that share their rows, each kQuantCols columns
  std::int32_t topk;     // > 0: row r is x's row slot_of_row[r] / topk
  std::int64_t x_rows;   // topk > 0: rows of x; an entry past them has no row
  std::int32_t const *slot_of_row;  // nullptr: every row; < 0: the row is left as it was
  std::uint8_t *data;    // [rows, cols / 2]
  std::uint8_t *scales;
};

// Scale byte and multipliers of one block.
struct fp4_block_scale {
  std::uint32_t byte;
  float mul;   // MX: z / scale = x * mul * mul2. NV: 16-bit x: x * mul; 32-bit x: see scaled()
  float mul2;  // MX: 1 in an ordinary block
  bool empty;  // a NaN block or an NV scale of zero: the elements are zeros
};

// MX blocks whose scale is E + log2 g - 2 and whose multiplier is 2^(129 - E)
// for amax = 1.f * 2^(E - 127): all but zero, subnormal, infinite and NaN ones
// and scales at the ends of the range.
__device__ __forceinline__ bool ordinary_mx(std::uint32_t bits, int log2_scale) {
  int const exponent = static_cast<int>(bits >> 23);
  int const byte = exponent + log2_scale - 2;
  return exponent >= 2 && exponent < 255 && byte >= 0 && byte <= 254;
}

// `bits` is the largest |x| as its 32-bit float pattern (NaN sorts above
// infinity above numbers).
template <bool kNv, bool kWide>
__device__ __forceinline__ fp4_block_scale block_scale(std::uint32_t bits, int log2_scale) {
  fp4_block_scale b;
  b.mul2 = 1.0f;
  if constexpr (!kNv) {  // ordinary blocks
    int const exponent = static_cast<int>(bits >> 23);
    b.byte = static_cast<std::uint32_t>(exponent + log2_scale - 2);
    b.mul = __int_as_float((256 - exponent) << 23);
    b.empty = false;
  } else {
    float const g = pow2(log2_scale);
    float const a = fminf(__uint_as_float(bits) * g, 4096.0f);  // past 6 * 448 it stays 448
    float v;
    if constexpr (kWide) {
      v = __fdiv_rz(a, 6.0f);
      if (fmaf(-6.0f, v, a) != 0.0f) v = __uint_as_float(__float_as_uint(v) | 1u);
    } else {
      v = __uint_as_float((__float_as_uint(a * (1.0f / 6.0f)) + 0x400u) & ~0x7ffu);
    }
    b.byte = to_e4m3(v);
    float const s = from_e4m3(b.byte);
    float inverse;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inverse) : "f"(s));
    b.mul = kWide ? s : g * inverse;
    b.mul2 = g;
    b.empty = b.byte == 0;
    if (bits >= 0x7f800000u) {
      b.byte = 0x7fu;
      b.empty = true;
    }
  }
  return b;
}

// Every other MX block.
__device__ __forceinline__ fp4_block_scale rare_mx(std::uint32_t bits, int log2_scale) {
  int const exponent = static_cast<int>(bits >> 23);
  int const fl = exponent > 0 ? exponent - 127 : 31 - __clz(static_cast<int>(bits)) - 149;
  int const e = bits == 0 ? -127 : min(max(fl + log2_scale - 2, -127), 127);
  int const f = log2_scale - e;
  fp4_block_scale b;
  b.empty = exponent == 255;
  b.byte = b.empty ? 0xffu : static_cast<std::uint32_t>(e + 127);
  b.mul = pow2(min(max(f, -126), 126));
  b.mul2 = f > 126 ? pow2(f - 126) : 1.0f;  // exact in two steps
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
    return copysignf(q, x);
  }
}

// Eight elements to one 32-bit word.
template <bool kNv, bool kWide>
__device__ __forceinline__ std::uint32_t encode8(float (&x)[8], fp4_block_scale const &b) {
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = scaled<kNv, kWide>(x[i], b);
  return kNv && b.empty ? 0u : e2m1x8(x);
}

// The largest |v[i]| of 16-bit pairs or 32-bit words as a 32-bit float pattern.
// Magnitudes of one type order as their bit patterns do, NaN above infinity.
template <class T, int kWords>
__device__ __forceinline__ std::uint32_t max_abs(std::uint32_t const *w) {
  if constexpr (sizeof(T) == 4) {
    std::uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < kWords; ++i) m = max(m, w[i] & 0x7fffffffu);
    return m;
  } else {
    std::uint32_t m = w[0] & 0x7fff7fffu;
#pragma unroll
    for (int i = 1; i + 1 < kWords; i += 2) {
      m = __vimax3_u16x2(m, w[i] & 0x7fff7fffu, w[i + 1] & 0x7fff7fffu);
    }
    if constexpr (kWords % 2 == 0) m = __vmaxu2(m, w[kWords - 1] & 0x7fff7fffu);
    m = max(m & 0xffffu, m >> 16);
    if constexpr (std::is_same_v<T, __nv_bfloat16>) {
      return m << 16;
    } else {
      return __float_as_uint(__half2float(__ushort_as_half(static_cast<std::uint16_t>(m))));
    }
  }
}

template <class T>
__device__ __forceinline__ float element(std::uint32_t const *w, int i) {
  if constexpr (sizeof(T) == 4) {
    return __uint_as_float(w[i]);
  } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
    return __uint_as_float(i % 2 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
  } else {
    return __half2float(__ushort_as_half(static_cast<std::uint16_t>(w[i / 2] >> (16 * (i % 2)))));
  }
}

// Eight elements from element `first` of `w` to one 32-bit word.
template <class T, bool kNv>
__device__ __forceinline__ std::uint32_t encode_words(std::uint32_t const *w, int first,
                                                      fp4_block_scale const &b) {
  float f[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = element<T>(w, first + i);
  return encode8<kNv, std::is_same_v<T, float>>(f, b);
}

// The elements of a block, or of half of one, plain and coded.
template <class T, int kElements>
struct fp4_words {
  std::uint32_t w[kElements * sizeof(T) / 4];
};
template <int kElements>
struct fp4_coded {
  std::uint32_t w[kElements / 8];
  std::uint32_t byte;
};

// A call, not inlined: predicated into the ordinary path, these instructions
// cost every block.
template <class T, int kElements>
__device__ __noinline__ fp4_coded<kElements> encode_rare_mx(fp4_words<T, kElements> v,
                                                            std::uint32_t bits, int log2_scale) {
  fp4_block_scale const b = rare_mx(bits, log2_scale);
  fp4_coded<kElements> out;
#pragma unroll
  for (int k = 0; k < kElements / 8; ++k) {
    float f[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = element<T>(v.w, k * 8 + i) * b.mul2;
    out.w[k] = b.empty ? 0u : encode8<false, std::is_same_v<T, float>>(f, b);
  }
  out.byte = b.byte;
  return out;
}

template <class T, bool kNv, int kElements>
__device__ __forceinline__ fp4_coded<kElements> encode_block(fp4_words<T, kElements> const &v,
                                                             std::uint32_t bits, int log2_scale) {
  if (!kNv && !ordinary_mx(bits, log2_scale)) {
    return encode_rare_mx<T, kElements>(v, bits, log2_scale);
  }
  fp4_block_scale const b = block_scale<kNv, std::is_same_v<T, float>>(bits, log2_scale);
  fp4_coded<kElements> out;
#pragma unroll
  for (int k = 0; k < kElements / 8; ++k) out.w[k] = encode_words<T, kNv>(v.w, k * 8, b);
  out.byte = b.byte;
  return out;
}

// 16 consecutive elements as words, by 32-byte loads when the rows allow it.
template <class T, bool kVec>
__device__ __forceinline__ void load16(T const *p, fp4_words<T, 16> &words) {
  std::uint32_t *const w = words.w;
  if constexpr (kVec) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) {
      bytes32 const v = load32_once(reinterpret_cast<char const *>(p) + 32 * i);
#pragma unroll
      for (int j = 0; j < 8; ++j) w[8 * i + j] = v.w[j];
    }
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 16; ++i) w[i] = reinterpret_cast<std::uint32_t const *>(p)[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      std::uint16_t const *const q = reinterpret_cast<std::uint16_t const *>(p) + 2 * i;
      w[i] = q[0] | static_cast<std::uint32_t>(q[1]) << 16;
    }
  }
}

inline constexpr int kQuantThreads = 256;
inline constexpr int kQuantCols = 256;  // columns of a CTA
inline constexpr int kQuantRows = 64;   // rows of a CTA: 16 of each 32 rows of a scale tile

// Column tiles that a CTA of a masked matrix takes one after another: its rows
// are looked up once, and the few rows of a routed batch make one wave of CTAs
// (256 x 8 rows over 64 experts x 4096 f16 NV: 10.5 us, 12.9 with one each).
inline constexpr int kMaskedSpan = 4;

// A CTA quantises 64 rows x 256 columns (neighbouring CTAs neighbouring
// columns, so that rows stream through DRAM in order): 16 lanes per row with 16
// elements each (512 bytes of a 16-bit row, 128 bytes of elements out). Its
// rows are rows [16 s, 16 s + 16) of each quarter of a 128-row scale tile,
// so that the scale bytes it owns are 256 contiguous bytes of each of its scale
// tiles. kMasked (slot_of_row): 64 consecutive rows instead, since an expert's
// rows fill the front of its tiles, so that CTAs without any end at once. Four
// passes per CTA, all four rows' loads in flight: with two, what a thread does
// once (addresses, barriers) was a third of its instructions.
template <class T, bool kNv, bool kVec, bool kMasked>
__global__ void __launch_bounds__(kQuantThreads) fp4_quantize_kernel(fp4_matrix_params p,
                                                                    T const *x) {
  constexpr int kTileCols = fp4_tile_cols(kNv);
  constexpr int kTiles = kQuantCols / kTileCols;
  constexpr int kPasses = kQuantRows / 16;
  constexpr int kSlices = kScaleTileRows / kQuantRows;
  constexpr int kPer = kQuantRows / 4;  // rows of each quarter
  // [tile][row] of four scale bytes: whole matrices in the scale tile's order
  __shared__ alignas(16) std::uint32_t bytes[kTiles][kQuantRows];
  grid_start_next();
  grid_wait();
  std::uint32_t const rows_cta = blockIdx.x / p.col_tiles;
  std::int64_t const row_tile = rows_cta / kSlices;
  int const slice = static_cast<int>(rows_cta % kSlices);
  int const lane16 = threadIdx.x % 16;
  // Where row l of the CTA lies in its row tile, and in `bytes`.
  auto tile_row = [&](int l) {
    return kMasked ? slice * kQuantRows + l : l / kPer * 32 + slice * kPer + l % kPer;
  };
  auto byte_row = [&](int l) { return kMasked ? l : l % kPer * 4 + l / kPer; };

  std::uint32_t have = 0;  // passes whose row is written
  std::int64_t src[kPasses];
#pragma unroll
  for (int pass = 0; pass < kPasses; ++pass) {
    std::int64_t const row =
        row_tile * kScaleTileRows + tile_row(pass * 16 + static_cast<int>(threadIdx.x) / 16);
    src[pass] = row;
    bool in = row < p.rows;
    if constexpr (kMasked) {
      std::int32_t const slot = in ? p.slot_of_row[row] : -1;
      in = slot >= 0;
      if (p.topk > 0) {
        src[pass] = slot / p.topk;
        in = in && src[pass] < p.x_rows;
      }
    }
    if (in) have |= 1u << pass;
  }
  if (kMasked && __syncthreads_or(have != 0) == 0) return;

  constexpr int kSpan = kMasked ? kMaskedSpan : 1;
  int col0 = static_cast<int>(blockIdx.x - rows_cta * p.col_tiles) * (kSpan * kQuantCols);
  for (int span = 0; span < kSpan && col0 < p.cols; ++span, col0 += kQuantCols) {
    int const col = col0 + lane16 * 16;
    fp4_words<T, 16> w[kPasses];
#pragma unroll
    for (int pass = 0; pass < kPasses; ++pass) {
      if ((have >> pass & 1u) && col < p.cols) {
        load16<T, kVec>(x + src[pass] * p.stride + col, w[pass]);
      }
    }
    if (span > 0) __syncthreads();  // `bytes` of the columns before are stored
#pragma unroll
    for (int pass = 0; pass < kPasses; ++pass) {
      int const l = pass * 16 + threadIdx.x / 16;
      std::uint32_t byte = 0;
      // Both lanes of an MX block are in or out together (cols % 32 == 0).
      if ((have >> pass & 1u) && col < p.cols) {
        std::uint32_t bits = max_abs<T, 4 * sizeof(T)>(w[pass].w);
        if constexpr (!kNv) {
          bits = max(bits, __shfl_xor_sync(3u << (threadIdx.x % 32 & ~1u), bits, 1));
        }
        fp4_coded<16> const coded = encode_block<T, kNv, 16>(w[pass], bits, p.log2_scale);
        byte = coded.byte;
        std::int64_t const row = row_tile * kScaleTileRows + tile_row(l);
        *reinterpret_cast<uint2 *>(p.data + row * (p.cols / 2) + col / 2) =
            make_uint2(coded.w[0], coded.w[1]);
      }
      if (kNv || lane16 % 2 == 0) {
        int const blk = lane16 * 16 / fp4_block(kNv);
        reinterpret_cast<std::uint8_t *>(&bytes[blk / 4][byte_row(l)])[blk % 4] =
            static_cast<std::uint8_t>(byte);
      }
    }
    __syncthreads();
    int const tile0 = col0 / kTileCols;
    int const tiles = min(kTiles, p.tiles - tile0);
    std::uint8_t *const dst = p.scales + (row_tile * p.tiles + tile0) * kScaleTileBytes;
    if constexpr (!kMasked) {
      if (static_cast<int>(threadIdx.x) < tiles * kPer) {
        int const tile = threadIdx.x / kPer, r = threadIdx.x % kPer;
        *reinterpret_cast<uint4 *>(dst + tile * kScaleTileBytes + (slice * kPer + r) * 16) =
            *reinterpret_cast<uint4 const *>(&bytes[tile][r * 4]);
      }
    } else if (lane16 < tiles) {
      // Only the rows written above: their four bytes of each tile.
#pragma unroll
      for (int pass = 0; pass < kPasses; ++pass) {
        int const l = pass * 16 + threadIdx.x / 16;
        if ((have >> pass & 1u) == 0) continue;
        *reinterpret_cast<std::uint32_t *>(dst + lane16 * kScaleTileBytes +
                                           scale_byte(tile_row(l), 0)) = bytes[lane16][l];
      }
    }
  }
}

inline constexpr int kScatterRows = 32;  // rows of x per CTA

// The gathered form the other way round: each row of x is quantised once and
// written to the rows of its `topk` choices (row_of_slot, `p.slot_of_row`
// here). Same bits; the gather quantises a row once per choice, which takes
// longer than the writes (8192 tokens x 8 choices x 4096 MX: 111 us
// against 43).
template <class T, bool kNv, bool kVec>
__global__ void __launch_bounds__(kQuantThreads) fp4_quantize_scatter_kernel(fp4_matrix_params p,
                                                                            T const *x) {
  constexpr int kPasses = kScatterRows / 16;
  constexpr int kLanes = fp4_tile_cols(kNv) / 16;  // lanes that share four scale bytes
  grid_start_next();
  grid_wait();
  std::uint32_t const rows_cta = blockIdx.x / p.col_tiles;
  int const lane16 = threadIdx.x % 16;
  int const col =
      static_cast<int>(blockIdx.x - rows_cta * p.col_tiles) * kQuantCols + lane16 * 16;
  std::int64_t const row0 =
      static_cast<std::int64_t>(rows_cta) * kScatterRows + threadIdx.x / 16;
  fp4_words<T, 16> w[kPasses];
#pragma unroll
  for (int pass = 0; pass < kPasses; ++pass) {
    std::int64_t const row = row0 + pass * 16;
    if (row < p.x_rows && col < p.cols) load16<T, kVec>(x + row * p.stride + col, w[pass]);
  }
#pragma unroll
  for (int pass = 0; pass < kPasses; ++pass) {
    std::int64_t const row = row0 + pass * 16;
    bool const in = row < p.x_rows && col < p.cols;
    std::uint32_t bits = in ? max_abs<T, 4 * sizeof(T)>(w[pass].w) : 0;
    if constexpr (!kNv) bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, 1));
    fp4_coded<16> coded{};
    if (in) coded = encode_block<T, kNv, 16>(w[pass], bits, p.log2_scale);
    // Four blocks' bytes to the first of their lanes; past the columns zeros.
    int const blk = col / fp4_block(kNv);
    std::uint32_t bytes = (coded.byte & 0xffu) << (8 * (blk % 4));
#pragma unroll
    for (int d = 1; d < kLanes; d *= 2) bytes |= __shfl_xor_sync(0xffffffffu, bytes, d);
    if (!in) continue;
    std::int32_t const *const at = p.slot_of_row + row * p.topk;
    for (int j = 0; j < p.topk; ++j) {
      std::int64_t const r = at[j];
      if (r < 0 || r >= p.rows) continue;
      *reinterpret_cast<uint2 *>(p.data + r * (p.cols / 2) + col / 2) =
          make_uint2(coded.w[0], coded.w[1]);
      if (lane16 % kLanes == 0) {
        *reinterpret_cast<std::uint32_t *>(
            p.scales + ((r / kScaleTileRows) * p.tiles + blk / 4) * kScaleTileBytes +
            scale_byte(static_cast<int>(r % kScaleTileRows), 0)) = bytes;
      }
    }
  }
}

inline constexpr int kQuantTRows = 64;  // rows of the quantised matrix per CTA

// The transpose: x is [cols, rows] as stored and its columns become the rows
// of the quantised matrix. A thread reads 32 elements down two neighbouring
// columns (a warp reads 64 neighbouring columns of each row, 128 bytes of a
// 16-bit type); the CTA's 64 x 256 tile of elements is turned in shared
// memory so that each row leaves as 128 contiguous bytes.
template <class T, bool kNv, bool kPair>
__global__ void __launch_bounds__(kQuantThreads, 2) fp4_quantize_t_kernel(fp4_matrix_params p,
                                                                         T const *x) {
  constexpr int kTileCols = fp4_tile_cols(kNv);
  constexpr int kTiles = kQuantCols / kTileCols;
  constexpr int kBlock = fp4_block(kNv);
  constexpr int kWordBlock = kBlock * sizeof(T) / 4;
  grid_start_next();
  grid_wait();
  // [tile][row % 32][row / 32] of four scale bytes
  __shared__ alignas(8) std::uint32_t bytes[kTiles][32][2];
  __shared__ uint4 turned[kQuantTRows][8];
  std::uint32_t const rows_cta = blockIdx.x / p.col_tiles;
  std::int64_t const row_tile = rows_cta / 2;
  int const part = static_cast<int>(rows_cta % 2);
  std::int64_t const row0 = row_tile * kScaleTileRows + part * kQuantTRows;
  int const col0 = static_cast<int>(blockIdx.x - rows_cta * p.col_tiles) * kQuantCols;
  int const r = threadIdx.x % 32 * 2, chunk = threadIdx.x / 32;
  std::int64_t const row = row0 + r;
  int const col = col0 + chunk * 32;
  bool const in = col < p.cols && row < p.rows;
  bool const two = row + 1 < p.rows;
  std::uint32_t w[2][8 * sizeof(T)];
  if (in) {
    T const *src = x + col * p.stride + row;
#pragma unroll
    for (int i = 0; i < 32; ++i, src += p.stride) {
      if constexpr (sizeof(T) == 4) {
        if constexpr (kPair) {
          uint2 const v = *reinterpret_cast<uint2 const *>(src);
          w[0][i] = v.x;
          w[1][i] = v.y;
        } else {
          w[0][i] = __float_as_uint(src[0]);
          w[1][i] = two ? __float_as_uint(src[1]) : 0;
        }
      } else {
        std::uint32_t v;
        if constexpr (kPair) {
          v = *reinterpret_cast<std::uint32_t const *>(src);
        } else {
          auto const *const q = reinterpret_cast<std::uint16_t const *>(src);
          v = q[0] | (two ? static_cast<std::uint32_t>(q[1]) << 16 : 0u);
        }
        // One word holds a column pair of one row; pack rows 2k, 2k + 1 of
        // each column into a word below.
        w[i % 2][i / 2] = v;
      }
    }
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        std::uint32_t const even = w[0][i], odd = w[1][i];
        w[0][i] = __byte_perm(even, odd, 0x5410);
        w[1][i] = __byte_perm(even, odd, 0x7632);
      }
    }
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    std::uint32_t out[4];
#pragma unroll
    for (int k = 0; k < 32 / kBlock; ++k) {
      std::uint32_t byte = 0;
      if (in && (h == 0 || two)) {
        fp4_words<T, kBlock> v;
#pragma unroll
        for (int i = 0; i < kWordBlock; ++i) v.w[i] = w[h][k * kWordBlock + i];
        fp4_coded<kBlock> const coded = encode_block<T, kNv, kBlock>(
            v, max_abs<T, kWordBlock>(v.w), p.log2_scale);
#pragma unroll
        for (int i = 0; i < kBlock / 8; ++i) out[k * (kBlock / 8) + i] = coded.w[i];
        byte = coded.byte;
      }
      int const blk = chunk * (32 / kBlock) + k;
      reinterpret_cast<std::uint8_t *>(&bytes[blk / 4][(r + h) % 32][(r + h) / 32])[blk % 4] =
          static_cast<std::uint8_t>(byte);
    }
    if (in && (h == 0 || two)) {
      turned[r + h][chunk ^ (r / 2 % 8)] = make_uint4(out[0], out[1], out[2], out[3]);
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = threadIdx.x; i < kQuantTRows * 8; i += kQuantThreads) {
    int const rr = i / 8, c = i % 8;
    if (row0 + rr < p.rows && col0 + c * 32 < p.cols) {
      *reinterpret_cast<uint4 *>(p.data + (row0 + rr) * (p.cols / 2) + col0 / 2 + c * 16) =
          turned[rr][c ^ (rr / 2 % 8)];
    }
  }
  int const tile0 = col0 / kTileCols;
  int const tiles = min(kTiles, p.tiles - tile0);
  std::uint8_t *const dst = p.scales + (row_tile * p.tiles + tile0) * kScaleTileBytes + part * 8;
  if (static_cast<int>(threadIdx.x) < tiles * 32) {
    int const tile = threadIdx.x / 32, rr = threadIdx.x % 32;
    *reinterpret_cast<uint2 *>(dst + tile * kScaleTileBytes + rr * 16) =
        *reinterpret_cast<uint2 const *>(bytes[tile][rr]);
  }
}

// 16 elements of the type.
template <class T>
struct alignas(32) fp4_plain {
  T v[16];
};

// Elements times s1 and, for kTwo, s2: the first product is exact then, the
// second rounds once.
template <class T, bool kTwo>
__device__ __forceinline__ fp4_plain<T> decode16(uint2 d, float s1, float s2) {
  fp4_plain<T> out;
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    __half2 h[4];
    from_e2m1x8(b == 0 ? d.x : d.y, h);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float2 f = __half22float2(h[i]);
      f.x *= s1;
      f.y *= s1;
      if constexpr (kTwo) {
        f.x *= s2;
        f.y *= s2;
      }
      out.v[8 * b + 2 * i] = from_f32<T>(f.x);
      out.v[8 * b + 2 * i + 1] = from_f32<T>(f.y);
    }
  }
  return out;
}

// MX scales that with 1 / g are no normal power of two, and NaN. A call, so
// that ordinary blocks do not pay for it.
template <class T>
__device__ __noinline__ fp4_plain<T> decode_rare_mx(uint2 d, int e, bool nan) {
  float const s1 = nan ? __int_as_float(0x7fffffff) : pow2(e < 0 ? -100 : 100);
  return decode16<T, true>(d, s1, nan ? 1.0f : pow2(e < 0 ? e + 100 : e - 100));
}

// The values: element * scale / g, rounded once. A thread decodes 16 elements
// of each of four rows, whose loads are all in flight.
template <class T, bool kNv, bool kVec>
__global__ void __launch_bounds__(kQuantThreads) fp4_dequantize_kernel(fp4_matrix_params p, T *y) {
  constexpr int kPasses = kQuantRows / 16;
  grid_start_next();
  grid_wait();
  std::uint32_t const per_row = static_cast<std::uint32_t>(p.cols) / 16;
  std::uint32_t const rows_cta = blockIdx.x / p.col_tiles;
  std::uint32_t const i = (blockIdx.x - rows_cta * p.col_tiles) * 16 + threadIdx.x % 16;
  if (i >= per_row) return;
  int const col = static_cast<int>(i) * 16;
  int const blk = col / fp4_block(kNv);
  std::int64_t const row0 =
      static_cast<std::int64_t>(rows_cta) * kQuantRows + threadIdx.x / 16;
  uint2 d[kPasses];
  std::uint32_t byte[kPasses];
#pragma unroll
  for (int pass = 0; pass < kPasses; ++pass) {
    std::int64_t const row = row0 + pass * 16;
    if (row < p.rows) {
      d[pass] = *reinterpret_cast<uint2 const *>(p.data + row * (p.cols / 2) + col / 2);
      byte[pass] = p.scales[((row / kScaleTileRows) * p.tiles + blk / 4) * kScaleTileBytes +
                            scale_byte(static_cast<int>(row % kScaleTileRows), blk)];
    }
  }
#pragma unroll
  for (int pass = 0; pass < kPasses; ++pass) {
    std::int64_t const row = row0 + pass * 16;
    if (row >= p.rows) break;
    fp4_plain<T> out;
    if constexpr (kNv) {
      out = decode16<T, false>(d[pass], from_e4m3(byte[pass]) * pow2(-p.log2_scale), 1.0f);
    } else {
      int const e = static_cast<int>(byte[pass]) - 127 - p.log2_scale;
      bool const nan = byte[pass] == 0xffu;
      if (e >= -126 && e <= 127 && !nan) {
        out = decode16<T, false>(d[pass], pow2(e), 1.0f);
      } else {
        out = decode_rare_mx<T>(d[pass], e, nan);
      }
    }
    T *const dst = y + row * p.stride + col;
    if constexpr (kVec) {
#pragma unroll
      for (int c = 0; c < static_cast<int>(sizeof(T)) / 2; ++c) {
        store32(reinterpret_cast<char *>(dst) + 32 * c,
                reinterpret_cast<bytes32 const *>(out.v)[c]);
      }
    } else {
#pragma unroll
      for (int c = 0; c < 16; ++c) dst[c] = out.v[c];
    }
  }
}

}  // namespace megacu_b200
