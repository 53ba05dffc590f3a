// Product of two 4-bit block-scaled matrices on the tensor cores:
//   out[i, j] = alpha * sum_k A[i, k] B[j, k]
// and its gated form act = silu(alpha G) * (alpha U) with two B operands, both
// also by expert (each 128-row tile of A against its expert's B).
//
// tcgen05.mma block-scaled kinds: mxf4 (blocks of 32, ue8m0) and mxf4nvf4
// (blocks of 16, e4m3), K = 64 per instruction, fp32 accumulators in TMEM. One
// MMA covers 128 rows of A and BN rows of B.
//
//   warp 0     TMA producer: 128 rows x 256 elements of A, BN rows of B
//              (128-byte swizzle) and their scale tiles per stage
//   warp 1     TMEM allocation, scale copies shared -> TMEM, MMA issue
//   warps 2-5  epilogue: accumulators -> alpha / SwiGLU -> out type -> memory
//
// TMEM holds two accumulators and the scales of a stage. With BN = 256 the two
// accumulators share 64 columns (0..255 and 192..447, scales from 448): the
// epilogue drains the shared columns first and then lets the next tile's MMAs
// start, so a tile's epilogue overlaps the next tile's MMAs.
//
// A few rows (decode): bound by the weights' stream, so the tile's K is split
// over the CTAs of a cluster (params.split) to occupy every SM; each CTA then
// sums one slice of the tile's columns over the cluster, in rank order,
// through distributed shared memory (the drained stage ring).
//
// Every wait is bounded; one that gives up sets the error word in `events`.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "fp4_format.cuh"
#include "layout.h"
#include "sm100_ptx.cuh"
#include "vec.cuh"

namespace megacu_b200 {

inline constexpr int kFp4Threads = 192;
inline constexpr int kFp4BlockM = 128;
inline constexpr int kFp4BlockK = 256;  // elements per stage: one 128-byte swizzled row
inline constexpr int kFp4SmallRows = 32;  // rows of the smaller A box
inline constexpr int kFp4MaxSplit = 8;

struct fp4_gemm_params {
  std::int32_t n, k;
  std::int32_t m_tiles;      // 128-row tiles of A (by expert: of its capacity)
  std::int32_t n_tiles;      // tiles of BN columns (SwiGLU: of BN / 2)
  std::int32_t n_row_tiles;  // scale row tiles of one B matrix, ceil(n / 128)
  std::int32_t rows;         // rows of A
  std::int32_t group_m;      // raster band height in tile rows
  std::int32_t experts;      // 0: one B for all rows
  std::int32_t split;        // CTAs of a cluster that share a tile's K
  std::int32_t scale_tiles;  // scale tiles per row tile
  std::int32_t out_dtype;    // MEGACU_DTYPE_*
  std::int32_t vec_store;    // out rows allow 16-byte stores
  std::int64_t out_stride;
  float alpha;
  float const *alphas;            // per expert, or nullptr
  std::int32_t const *offsets;    // [experts + 1], multiples of 128
  std::int32_t const *counts;     // [experts]
  std::uint8_t const *a_scales;
  std::uint8_t const *b_scales;
  std::uint8_t const *b2_scales;  // SwiGLU: up
  void *out;
  std::uint32_t *events;
  unsigned long long timeout_ns;
};

template <bool kNv, int BN>
struct fp4_config {
  static constexpr int scale_tiles = kFp4BlockK / fp4_tile_cols(kNv);  // per row tile and stage
  static constexpr int a_bytes = kFp4BlockM * 128;
  static constexpr int b_bytes = BN * 128;
  static constexpr int sfa_bytes = scale_tiles * kScaleTileBytes;
  static constexpr int sfb_bytes = BN / 128 * sfa_bytes;
  static constexpr int stage_bytes = a_bytes + b_bytes + sfa_bytes + sfb_bytes;
  static constexpr int stages = BN == 256 ? 4 : 6;
  static constexpr int ring_bytes = stages * stage_bytes;
  static constexpr int staging_bytes = 4 * 2048;  // 2 KB per epilogue warp
  static constexpr int smem_bytes = 1024 + ring_bytes + staging_bytes + 256;
  static constexpr int acc1 = BN == 256 ? 192 : BN;  // columns of the second accumulator
  static constexpr int sf_column = acc1 + BN;
  static constexpr int tmem_columns = 512;
  static_assert(smem_bytes <= 232448, "dynamic shared memory per CTA");
  static_assert(sf_column + scale_tiles * 4 * (1 + BN / 128) <= tmem_columns, "TMEM");
  static_assert(BN * 128 * 4 <= ring_bytes, "the split's exchange fits the ring");
};

namespace ptx {

// D (+)= A * B with block scales from TMEM.
template <bool kNv>
__device__ __forceinline__ void umma_fp4(std::uint32_t d, std::uint64_t a, std::uint64_t b,
                                         std::uint32_t idesc, std::uint32_t sfa,
                                         std::uint32_t sfb, std::uint32_t accumulate) {
  if constexpr (kNv) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X "
        "[%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        :: "r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
  } else {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X "
        "[%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        :: "r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
  }
}

// One scale tile (32 rows of 16 bytes in shared memory) into four TMEM
// columns, repeated for the four groups of 32 lanes.
__device__ __forceinline__ void copy_scale_tile(std::uint32_t tmem, std::uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" :: "r"(tmem), "l"(desc)
               : "memory");
}

// Contiguous copy global -> shared; addresses and size multiples of 16.
__device__ __forceinline__ void bulk_load(void *dst, void const *src, std::uint32_t bytes,
                                          std::uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
      :: "r"(smem_addr(dst)), "l"(src), "r"(bytes), "r"(smem_addr(bar))
      : "memory");
}

// Descriptor of a scale tile: no swizzle, 8-row groups 128 bytes apart.
__device__ __forceinline__ std::uint64_t scale_desc(std::uint32_t start) {
  return static_cast<std::uint64_t>((start >> 4) & 0x3fffu) |
         (static_cast<std::uint64_t>(128 >> 4) << 32) | (static_cast<std::uint64_t>(1) << 46);
}

}  // namespace ptx

// Instruction descriptor of the block-scaled kinds: e2m1 A and B, both
// K-major; scale_id picks the byte (pair) of the scale columns.
template <bool kNv>
__host__ __device__ constexpr std::uint32_t fp4_idesc(std::uint32_t m, std::uint32_t n,
                                                      std::uint32_t scale_id) {
  return (scale_id << 4)            // B scale id
         | (1u << 7) | (1u << 10)   // A, B: e2m1
         | ((n >> 3) << 17)
         | ((kNv ? 0u : 1u) << 23)  // scales: e4m3 or ue8m0
         | ((m >> 7) << 27)
         | (scale_id << 29);        // A scale id
}

// Tile t of the raster: bands of group_m tile rows walked column by column.
struct fp4_tile {
  std::int32_t row, col;
};

__host__ __device__ inline fp4_tile fp4_locate(std::int32_t t, std::int32_t m_tiles,
                                               std::int32_t n_tiles, std::int32_t group_m) {
  std::int32_t const band = t / (group_m * n_tiles);
  std::int32_t const first = band * group_m;
  std::int32_t const height = m_tiles - first < group_m ? m_tiles - first : group_m;
  std::int32_t const in = t - first * n_tiles;
  return {first + in % height, in / height};
}

namespace detail {

// The expert whose rows hold `row` (whole warp; offsets ascend, the row is
// below offsets[experts]): how many e have offsets[e + 1] <= row, by two
// 32-wide counts.
__device__ __forceinline__ std::int32_t find_expert(std::int32_t const *offsets,
                                                    std::int32_t experts, std::int32_t row) {
  std::int32_t const lane = static_cast<std::int32_t>(ptx::lane_id());
  std::int32_t const step = (experts + 31) / 32;
  std::int32_t const last = (lane + 1) * step;
  bool const below = last <= experts && offsets[last] <= row;
  std::int32_t const base = __popc(__ballot_sync(0xffffffffu, below)) * step;
  std::int32_t const at = base + lane + 1;
  bool const in = lane < step && at <= experts && offsets[at] <= row;
  return min(base + __popc(__ballot_sync(0xffffffffu, in)), experts - 1);
}

// What one tile row needs besides its raster place (whole warp).
struct fp4_rows {
  std::int32_t expert, valid;  // rows of the tile that exist
  float alpha;
};

__device__ __forceinline__ fp4_rows locate_rows(fp4_gemm_params const &p, std::int32_t row) {
  fp4_rows r{0, p.rows - row, p.alpha};
  if (p.experts > 0) {
    r.expert = find_expert(p.offsets, p.experts, row);
    r.valid = min(r.valid, p.counts[r.expert] - (row - p.offsets[r.expert]));
    if (p.alphas != nullptr) r.alpha *= p.alphas[r.expert];
  }
  return r;
}

__device__ __forceinline__ void fp4_error(std::uint32_t *events, std::uint32_t tile,
                                          std::uint32_t site) {
  auto *const ctrl = reinterpret_cast<control_block *>(events);
  if (atomicCAS(&ctrl->error_code, 0u, static_cast<std::uint32_t>(err_local_timeout)) == 0u) {
    ctrl->error_info[0] = tile;
    ctrl->error_info[1] = 0;
    ctrl->error_info[2] = site;
  }
}

__device__ __forceinline__ std::uint32_t pack16(std::int32_t dtype, float lo, float hi) {
  if (dtype == 1) {
    __half2 const v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<std::uint32_t const *>(&v);
  }
  return ptx::pack_bf16x2(lo, hi);
}

// Stores NC (16 or 32) consecutive columns from `col` of a warp's 32 rows:
// lane = row on entry; through `stage` (2 KB) so that each row leaves as 16-byte
// vectors of neighbouring lanes. `rows` rows exist.
template <int NC>
__device__ __forceinline__ void store_columns(fp4_gemm_params const &p, std::uint8_t *stage,
                                              float const (&v)[NC], std::int64_t row0,
                                              std::int32_t rows, std::int32_t col) {
  std::uint32_t const lane = ptx::lane_id();
  bool const wide = p.out_dtype == 3;
  std::uint32_t const size = wide ? 4 : 2;
  std::uint32_t const passes = wide && NC == 32 ? 2 : 1;
  std::uint32_t const chunks = wide ? 4 : NC / 8;    // 16-byte vectors per row and pass
  std::uint32_t const per_pass = chunks * 16 / size;  // columns per pass
#pragma unroll
  for (std::uint32_t pass = 0; pass < 2; ++pass) {
    if (pass >= passes) break;
#pragma unroll
    for (std::uint32_t c = 0; c < 4; ++c) {
      if (c >= chunks) break;
      uint4 q;
      if (wide) {
        std::uint32_t const i = (pass * 16 + c * 4) % NC;
        q = make_uint4(__float_as_uint(v[i]), __float_as_uint(v[i + 1]),
                       __float_as_uint(v[i + 2]), __float_as_uint(v[i + 3]));
      } else {
        std::uint32_t const i = c * 8 % NC;
        q = make_uint4(pack16(p.out_dtype, v[i], v[i + 1]), pack16(p.out_dtype, v[i + 2], v[i + 3]),
                       pack16(p.out_dtype, v[i + 4], v[i + 5]),
                       pack16(p.out_dtype, v[i + 6], v[i + 7]));
      }
      *reinterpret_cast<uint4 *>(stage + lane * 64 + ((c ^ (lane >> 1)) & 3) * 16) = q;
    }
    __syncwarp();
    for (std::uint32_t i = lane; i < 32 * chunks; i += 32) {
      std::uint32_t const r = i / chunks, c = i % chunks;
      std::int32_t const first = col + static_cast<std::int32_t>(pass * per_pass + c * 16 / size);
      if (static_cast<std::int32_t>(r) < rows && first < p.n) {
        uint4 const q = *reinterpret_cast<uint4 const *>(stage + r * 64 + ((c ^ (r >> 1)) & 3) * 16);
        std::uint8_t *const dst = static_cast<std::uint8_t *>(p.out) +
                                  ((row0 + r) * p.out_stride + first) * size;
        std::int32_t const left = p.n - first;
        if (p.vec_store && left >= static_cast<std::int32_t>(16 / size)) {
          *reinterpret_cast<uint4 *>(dst) = q;
        } else {
          std::uint32_t const w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
          for (std::int32_t e = 0; e < 8; ++e) {
            if (wide) {
              if (e < 4 && e < left) reinterpret_cast<std::uint32_t *>(dst)[e] = w[e % 4];
            } else if (e < left) {
              reinterpret_cast<std::uint16_t *>(dst)[e] =
                  static_cast<std::uint16_t>(w[e / 2] >> (16 * (e % 2)));
            }
          }
        }
      }
    }
    __syncwarp();
  }
}

__device__ __forceinline__ float swiglu(float g, float u) {
  return g / (1.0f + __expf(-g)) * u;
}

}  // namespace detail

template <bool kNv, bool kSwiglu, int BN>
__global__ void __launch_bounds__(kFp4Threads, 1)
    fp4_gemm_kernel(__grid_constant__ CUtensorMap const map_a,
                    __grid_constant__ CUtensorMap const map_a_small,
                    __grid_constant__ CUtensorMap const map_b,
                    __grid_constant__ CUtensorMap const map_b2,
                    __grid_constant__ fp4_gemm_params const p) {
  using cfg = fp4_config<kNv, BN>;
  static_assert(!kSwiglu || BN == 256, "128 gate and 128 up columns");
  constexpr int kStages = cfg::stages;
  constexpr int kActCols = kSwiglu ? BN / 2 : BN;
  extern __shared__ std::uint8_t raw_smem[];
  std::uint8_t *const smem = reinterpret_cast<std::uint8_t *>(
      (reinterpret_cast<std::uintptr_t>(raw_smem) + 1023) & ~static_cast<std::uintptr_t>(1023));
  // [A | B] of every stage (1024-byte aligned), then the scales, the epilogue
  // staging and the barriers.
  std::uint8_t *const scales = smem + kStages * (cfg::a_bytes + cfg::b_bytes);
  std::uint8_t *const staging = smem + cfg::ring_bytes;
  auto *const full = reinterpret_cast<std::uint64_t *>(staging + cfg::staging_bytes);
  std::uint64_t *const empty = full + kStages;
  std::uint64_t *const acc_full = empty + kStages;
  std::uint64_t *const acc_free = acc_full + 1;
  auto *const tmem_slot = reinterpret_cast<std::uint32_t *>(acc_free + 1);
  std::uint32_t *const abort_word = &reinterpret_cast<control_block *>(p.events)->error_code;

  std::int32_t const warp = static_cast<std::int32_t>(threadIdx.x) / 32;
  std::uint32_t const lane = ptx::lane_id();
  std::int32_t const split = p.split;
  std::int32_t const rank = split > 1 ? static_cast<std::int32_t>(ptx::cluster_ctarank()) : 0;
  std::int32_t const unit0 = static_cast<std::int32_t>(blockIdx.x) / split;
  std::int32_t const units = static_cast<std::int32_t>(gridDim.x) / split;
  std::int32_t const k_blocks = (p.k + kFp4BlockK - 1) / kFp4BlockK;
  std::int32_t const kb0 = rank * k_blocks / split;
  std::int32_t const kb1 = (rank + 1) * k_blocks / split;
  std::int32_t const m_tiles =
      p.experts > 0 ? min(p.offsets[p.experts] / kFp4BlockM, p.m_tiles) : p.m_tiles;
  std::int32_t const tiles = m_tiles * p.n_tiles;

  if (threadIdx.x == 0) {
    ptx::prefetch_tensor_map(&map_a);
    ptx::prefetch_tensor_map(&map_a_small);
    ptx::prefetch_tensor_map(&map_b);
    if constexpr (kSwiglu) ptx::prefetch_tensor_map(&map_b2);
    for (int s = 0; s < kStages; ++s) {
      ptx::mbar_init(&full[s], 1);
      ptx::mbar_init(&empty[s], 1);
    }
    ptx::mbar_init(acc_full, 1);
    ptx::mbar_init(acc_free, 4);
    ptx::fence_barrier_init();
    ptx::fence_proxy_async_shared();
  }
  if (warp == 1) {
    ptx::tmem_alloc(tmem_slot, cfg::tmem_columns);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before_sync();
  __syncthreads();
  ptx::tc_fence_after_sync();
  std::uint32_t const tmem = *tmem_slot;

  if (warp == 0) {
    // ---------------- TMA producer ----------------
    std::uint32_t stage = 0, phase = 0, issued = 0;
    bool ok = true;
    for (std::int32_t t = unit0; ok && t < tiles; t += units) {
      fp4_tile const c = fp4_locate(t, m_tiles, p.n_tiles, p.group_m);
      std::int32_t const row = c.row * kFp4BlockM;
      detail::fp4_rows const rows = detail::locate_rows(p, row);
      std::int32_t const boxes =
          min(max((rows.valid + kFp4SmallRows - 1) / kFp4SmallRows, 1), 4);
      std::int32_t const b_row = rows.expert * p.n + c.col * kActCols;
      std::int32_t const b_tile = c.col * (kActCols / 128);
      std::int32_t const b_tiles = kSwiglu ? 1 : min(BN / 128, p.n_row_tiles - b_tile);
      std::int64_t const a_scale = static_cast<std::int64_t>(c.row) * p.scale_tiles;
      std::int64_t const b_scale =
          (static_cast<std::int64_t>(rows.expert) * p.n_row_tiles + b_tile) * p.scale_tiles;
      for (std::int32_t kb = kb0; kb < kb1; ++kb) {
        if (!ptx::mbar_wait(&empty[stage], phase ^ 1u, abort_word, p.timeout_ns)) {
          if (lane == 0) detail::fp4_error(p.events, static_cast<std::uint32_t>(t), 51);
          ok = false;
          break;
        }
        if (lane == 0) {
          std::int32_t const st0 = kb * cfg::scale_tiles;
          std::uint32_t const sf_bytes = static_cast<std::uint32_t>(
              min(cfg::scale_tiles, p.scale_tiles - st0) * kScaleTileBytes);
          std::uint8_t *const sa = smem + stage * (cfg::a_bytes + cfg::b_bytes);
          std::uint8_t *const sb = sa + cfg::a_bytes;
          std::uint8_t *const sfa = scales + stage * (cfg::sfa_bytes + cfg::sfb_bytes);
          std::uint8_t *const sfb = sfa + cfg::sfa_bytes;
          ptx::mbar_arrive_expect_tx(
              &full[stage], static_cast<std::uint32_t>(boxes) * kFp4SmallRows * 128 +
                                cfg::b_bytes + sf_bytes * (1 + (kSwiglu ? 2 : b_tiles)));
          std::int32_t const x = kb * 128;
          if (boxes == 4) {
            ptx::tma_load_2d(&map_a, &full[stage], sa, x, row);
          } else {
            for (std::int32_t i = 0; i < boxes; ++i) {
              ptx::tma_load_2d(&map_a_small, &full[stage], sa + i * kFp4SmallRows * 128, x,
                               row + i * kFp4SmallRows);
            }
          }
          ptx::tma_load_2d(&map_b, &full[stage], sb, x, b_row);
          if constexpr (kSwiglu) {
            ptx::tma_load_2d(&map_b2, &full[stage], sb + cfg::b_bytes / 2, x, b_row);
          }
          ptx::bulk_load(sfa, p.a_scales + (a_scale + st0) * kScaleTileBytes, sf_bytes,
                         &full[stage]);
          ptx::bulk_load(sfb, p.b_scales + (b_scale + st0) * kScaleTileBytes, sf_bytes,
                         &full[stage]);
          if constexpr (kSwiglu) {
            ptx::bulk_load(sfb + cfg::sfa_bytes, p.b2_scales + (b_scale + st0) * kScaleTileBytes,
                           sf_bytes, &full[stage]);
          } else if constexpr (BN == 256) {
            if (b_tiles == 2) {
              ptx::bulk_load(sfb + cfg::sfa_bytes,
                             p.b_scales + (b_scale + p.scale_tiles + st0) * kScaleTileBytes,
                             sf_bytes, &full[stage]);
            }
          }
        }
        __syncwarp();
        ++issued;
        if (++stage == kStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
    if (!ok) {
      // Copies still in flight land before the CTA may exit.
      std::uint32_t const pending = issued < kStages ? issued : kStages;
      for (std::uint32_t i = 0; i < pending; ++i) {
        if (stage == 0) phase ^= 1u;
        stage = stage == 0 ? kStages - 1 : stage - 1;
        ptx::mbar_wait(&full[stage], phase, nullptr, p.timeout_ns);
      }
    }
  } else if (warp == 1) {
    // ---------------- scale copies and MMA issue ----------------
    if (lane == 0) {
      std::uint32_t stage = 0, phase = 0, tile_index = 0;
      std::uint32_t const sf = tmem + cfg::sf_column;
      bool ok = true;
      for (std::int32_t t = unit0; ok && t < tiles; t += units, ++tile_index) {
        if (tile_index > 0 &&
            !ptx::mbar_wait(acc_free, (tile_index - 1) & 1u, abort_word, p.timeout_ns)) {
          detail::fp4_error(p.events, static_cast<std::uint32_t>(t), 52);
          break;
        }
        ptx::tc_fence_after_sync();
        std::uint32_t const acc = tmem + (tile_index & 1u) * cfg::acc1;
        for (std::int32_t kb = kb0; kb < kb1; ++kb) {
          if (!ptx::mbar_wait(&full[stage], phase, abort_word, p.timeout_ns)) {
            detail::fp4_error(p.events, static_cast<std::uint32_t>(t), 53);
            ok = false;
            break;
          }
          ptx::tc_fence_after_sync();
          std::uint32_t const sa = ptx::smem_addr(smem + stage * (cfg::a_bytes + cfg::b_bytes));
          std::uint32_t const sb = sa + cfg::a_bytes;
          std::uint32_t const sfa =
              ptx::smem_addr(scales + stage * (cfg::sfa_bytes + cfg::sfb_bytes));
          std::uint32_t const sfb = sfa + cfg::sfa_bytes;
          std::int32_t const steps = min(4, (p.k - kb * kFp4BlockK + 63) / 64);
#pragma unroll
          for (std::int32_t j = 0; j < 4; ++j) {
            if (j >= steps) break;
            // NV: one scale tile per 64 of K; MX: one per 128, a byte pair each.
            std::int32_t const st = kNv ? j : j / 2;
            std::uint32_t const ta = sf + st * 4 * (1 + BN / 128);
            std::uint32_t const tb = ta + 4;
            if (kNv || j % 2 == 0) {
              ptx::copy_scale_tile(ta, ptx::scale_desc(sfa + st * kScaleTileBytes));
#pragma unroll
              for (int h = 0; h < BN / 128; ++h) {
                ptx::copy_scale_tile(tb + 4 * h, ptx::scale_desc(sfb + h * cfg::sfa_bytes +
                                                                 st * kScaleTileBytes));
              }
            }
            ptx::umma_fp4<kNv>(acc, ptx::smem_desc_sw128(sa + j * 32, 16, 1024),
                               ptx::smem_desc_sw128(sb + j * 32, 16, 1024),
                               fp4_idesc<kNv>(kFp4BlockM, BN, kNv ? 0 : j % 2 * 2), ta, tb,
                               kb > kb0 || j > 0);
          }
          ptx::umma_commit(&empty[stage]);
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        ptx::umma_commit(acc_full);
        // MMAs in flight end before the CTA may free its TMEM.
        if (!ok) ptx::mbar_wait(acc_full, tile_index & 1u, nullptr, p.timeout_ns);
      }
    }
    __syncwarp();
  } else {
    // ---------------- epilogue ----------------
    std::int32_t const quarter = warp & 3;  // TMEM lanes [32 quarter, +32)
    std::uint8_t *const stage = staging + quarter * 2048;
    std::uint32_t const lanes = static_cast<std::uint32_t>(quarter * 32) << 16;
    std::uint32_t tile_index = 0;
    for (std::int32_t t = unit0; t < tiles; t += units, ++tile_index) {
      fp4_tile const c = fp4_locate(t, m_tiles, p.n_tiles, p.group_m);
      std::int32_t const row = c.row * kFp4BlockM;
      detail::fp4_rows const rows = detail::locate_rows(p, row);
      std::int32_t const valid = rows.valid - quarter * 32;
      float const alpha = rows.alpha;
      if (!ptx::mbar_wait(acc_full, tile_index & 1u, abort_word, p.timeout_ns)) {
        if (lane == 0) detail::fp4_error(p.events, static_cast<std::uint32_t>(t), 54);
        break;
      }
      ptx::tc_fence_after_sync();
      std::uint32_t const acc = tmem + lanes + (tile_index & 1u) * cfg::acc1;
      if (split > 1) {
        // The columns of every slice to its CTA, once every ring is drained
        // (after the cluster barrier below); kept out of this loop.
        break;
      }
      if (BN < 256 && lane == 0) ptx::mbar_arrive(acc_free);  // the other accumulator is drained
      // Chunks of 32 output columns, the shared TMEM columns (192..255) first:
      // in the first accumulator the last ones, in the second the first ones.
      constexpr int kChunks = kActCols / 32;
      int const first = BN == 256 && (tile_index & 1u) == 0 ? kChunks - 2 : 0;
#pragma unroll 1
      for (int i = 0; i < kChunks; ++i) {
        int const chunk = i + first < kChunks ? i + first : i + first - kChunks;
        float v[32];
        std::uint32_t raw[32];
        ptx::tmem_load_32x32b_x32(acc + chunk * 32, raw);
        if constexpr (kSwiglu) {
          std::uint32_t up[32];
          ptx::tmem_load_32x32b_x32(acc + kActCols + chunk * 32, up);
          ptx::tmem_wait_load();
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            v[e] = detail::swiglu(alpha * __uint_as_float(raw[e]), alpha * __uint_as_float(up[e]));
          }
        } else {
          ptx::tmem_wait_load();
#pragma unroll
          for (int e = 0; e < 32; ++e) v[e] = alpha * __uint_as_float(raw[e]);
        }
        if (BN == 256 && i == 1) {
          ptx::tc_fence_before_sync();
          if (lane == 0) ptx::mbar_arrive(acc_free);
        }
        std::int32_t const col = c.col * kActCols + chunk * 32;
        if (valid > 0 && col < p.n) {
          detail::store_columns<32>(p, stage, v, row + quarter * 32, valid, col);
        }
      }
      ptx::tc_fence_before_sync();
    }
  }

  if (split > 1) {
    // One tile per cluster: each CTA holds the partial sums of its K range.
    // Every CTA's ring is drained past the first barrier (its epilogue has
    // seen its last commit); slices are [rank][part][4 columns][128 rows].
    __syncwarp();
    ptx::cluster_sync();
    bool const have = unit0 < tiles;
    fp4_tile const c = have ? fp4_locate(unit0, m_tiles, p.n_tiles, p.group_m) : fp4_tile{0, 0};
    std::int32_t const row = c.row * kFp4BlockM;
    std::int32_t const slice = kActCols / split;  // output columns per CTA
    constexpr int kParts = kSwiglu ? 2 : 1;
    std::int32_t valid = 0;
    float alpha = p.alpha;
    std::int32_t const quarter = warp & 3;
    if (have && warp >= 2) {
      detail::fp4_rows const rows = detail::locate_rows(p, row);
      valid = rows.valid - quarter * 32;
      alpha = rows.alpha;
      if (valid > 0) {
        ptx::tc_fence_after_sync();
        std::uint32_t const acc = tmem + (static_cast<std::uint32_t>(quarter * 32) << 16);
#pragma unroll 1
        for (int chunk = 0; chunk < BN / 32; ++chunk) {
          std::uint32_t raw[32];
          ptx::tmem_load_32x32b_x32(acc + chunk * 32, raw);
          ptx::tmem_wait_load();
          if (static_cast<std::int32_t>(lane) < valid) {
#pragma unroll
            for (int q = 0; q < 8; ++q) {
              std::int32_t const col = chunk * 32 + q * 4;
              std::int32_t const part = kSwiglu ? col / kActCols : 0;
              std::int32_t const in = col - part * kActCols;
              std::int32_t const to = in / slice;
              std::uint32_t const at = static_cast<std::uint32_t>(
                  ((rank * kParts + part) * (slice / 4) + (in - to * slice) / 4) * 2048 +
                  (quarter * 32 + static_cast<std::int32_t>(lane)) * 16);
              ptx::st_shared_remote_v4(ptx::map_to_rank(smem + at, static_cast<std::uint32_t>(to)),
                                       raw[q * 4], raw[q * 4 + 1], raw[q * 4 + 2], raw[q * 4 + 3]);
            }
          }
        }
      }
    }
    __syncwarp();
    ptx::cluster_sync();
    if (valid > 0) {
      std::uint8_t *const stage = staging + quarter * 2048;
      std::uint32_t const mine = (static_cast<std::uint32_t>(quarter * 32) + lane) * 16;
      for (std::int32_t c0 = 0; c0 < slice; c0 += 16) {
        std::int32_t const col = c.col * kActCols + rank * slice + c0;
        if (col >= p.n) break;
        float sum[kParts][16] = {};
        for (std::int32_t src = 0; src < split; ++src) {
#pragma unroll
          for (int part = 0; part < kParts; ++part) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              float4 const f = *reinterpret_cast<float4 const *>(
                  smem + ((src * kParts + part) * (slice / 4) + c0 / 4 + q) * 2048 + mine);
              sum[part][q * 4] += f.x;
              sum[part][q * 4 + 1] += f.y;
              sum[part][q * 4 + 2] += f.z;
              sum[part][q * 4 + 3] += f.w;
            }
          }
        }
        float v[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          v[e] = kSwiglu ? detail::swiglu(alpha * sum[0][e], alpha * sum[kParts - 1][e])
                         : alpha * sum[0][e];
        }
        detail::store_columns<16>(p, stage, v, row + quarter * 32, valid, col);
      }
    }
  }

  ptx::tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    ptx::tc_fence_after_sync();
    ptx::tmem_dealloc(tmem, cfg::tmem_columns);
  }
}

}  // namespace megacu_b200
