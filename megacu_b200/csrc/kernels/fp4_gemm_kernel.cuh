// Product of two 4-bit block-scaled matrices on the tensor cores:
//   out[i, j] = alpha * sum_k A[i, k] B[j, k]
// and its gated form act = silu(alpha G) * (alpha U) with two B operands, both
// also by expert (each 128-row tile of A against its expert's B).
//
// tcgen05.mma block-scaled kinds: mxf4 (blocks of 32, ue8m0) and mxf4nvf4
// (blocks of 16, e4m3), K = 64 per instruction, fp32 accumulators in TMEM.
//
//   warp 0     TMA producer: 128 rows x 256 elements of A, the tile's rows of B
//              (128-byte swizzle) and their scale tiles per stage; the first
//              tile's first stages are issued before the CTA's set-up ends
//   warp 1     TMEM allocation, scale copies shared -> TMEM, MMA issue
//   warps 2-9  epilogue: accumulators -> alpha / SwiGLU -> out type -> memory;
//              two warps per 32 rows take alternate chunks of 32 columns
//
// TMEM holds two accumulators and the scales of a stage. With BN = 256 the two
// accumulators share 64 columns (0..255 and 192..447, scales from 448): the
// epilogue drains the shared columns first and then lets the next tile's MMAs
// start, so a tile's epilogue overlaps the next tile's MMAs.
//
// kPair: a 2-CTA cluster computes 256 x 256 tiles with cta_group::2 MMAs. Each
// CTA stages its own 128 rows of A and half of B (SwiGLU: gate and up), so an
// SM moves 35 KB per 256 of K instead of 51, and holds its rows' accumulators
// and every B row's scales. One CTA alone is bound by shared memory: its loads
// and its MMAs' operand reads together exceed what the SM moves in the time of
// the MMAs.
//
// A few rows (decode): bound by the weights' stream, so the tile's K is split
// over the CTAs of a cluster (params.split) to occupy every SM; each CTA then
// sums one slice of the tile's columns over the cluster, in rank order,
// through distributed shared memory (the drained stage ring).
//
// Every wait is bounded; one that gives up sets the error word in `events`. A
// CTA leaves only when its loads have landed and its MMAs have ended, whichever
// wait gave up (stage_ring.h); on the normal path they have long since.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>
#include <type_traits>

#include "chained.cuh"
#include "fp4_format.cuh"
#include "layout.h"
#include "sm100_ptx.cuh"
#include "stage_ring.h"
#include "vec.cuh"

namespace megacu_b200 {

inline constexpr int kFp4EpilogueWarps = 8;
inline constexpr int kFp4Threads = 64 + 32 * kFp4EpilogueWarps;
inline constexpr int kFp4BlockM = 128;
inline constexpr int kFp4BlockK = 256;  // elements per stage: one 128-byte swizzled row
inline constexpr int kFp4SmallRows = 32;  // rows of the smaller A box
// Experts whose places are kept in shared memory: each tile's place is looked up
// before its loads, and four dependent global loads took 1.7 us, as long as the
// stage ring lasts.
inline constexpr int kFp4TableExperts = 256;
// Bound of the waits that only let copies and MMAs in flight end: they take
// microseconds, and nothing that an earlier error stopped is among them.
inline constexpr unsigned long long kFp4DrainNs = 1000000000ull;
// Bound of a follower's wait for a commit that may have been issued or not.
inline constexpr unsigned long long kFp4CommitNs = 10000000ull;

// b2, b2_scales: SwiGLU's up; a_small: A in boxes of kFp4SmallRows rows.
struct fp4_maps {
  CUtensorMap a, a_small, b, b2, a_scales, b_scales, b2_scales;
};

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
  std::int32_t row_bytes;    // 32, 16 or 0: what out's start and rows are multiples of
  std::int64_t out_stride;
  float alpha;
  float const *alphas;            // per expert, or nullptr
  std::int32_t const *offsets;    // [experts + 1], multiples of 128
  std::int32_t const *counts;     // [experts]
  void *out;
  std::uint32_t *events;
  unsigned long long timeout_ns;
};

// Where each expert's rows are, for at most kFp4TableExperts of them.
struct fp4_expert_table {
  std::int32_t end[kFp4TableExperts];            // offsets[e] + counts[e]
  std::uint16_t first_tile[kFp4TableExperts + 4];  // offsets[e] / 128, experts + 1 entries
};

// kRows: rows of A that a stage holds, 128, or 32 for products of at most 32
// rows; the MMA still reads 128, whatever follows, into accumulators that are
// never stored.
template <bool kNv, int BN, bool kPair, int kRows>
struct fp4_config {
  static constexpr int scale_tiles = kFp4BlockK / fp4_tile_cols(kNv);  // per row tile and stage
  static constexpr int b_tiles = BN > 128 ? BN / 128 : 1;  // row tiles of B whose scales it holds
  static constexpr int a_bytes = kRows * 128;
  static constexpr int b_bytes = BN * 128 / (kPair ? 2 : 1);
  static constexpr int sfa_bytes = scale_tiles * kScaleTileBytes;
  static constexpr int sfb_bytes = b_tiles * sfa_bytes;
  static constexpr int stage_bytes = a_bytes + b_bytes + sfa_bytes + sfb_bytes;
  // Bytes of a row that an epilogue warp stores at a time. 64 leave faster
  // than 32 (a 2048 x 1792 SwiGLU's last tile 2.7 against 3.2 us) but their
  // staging must not cost the fourth stage.
  static constexpr int barrier_bytes = (2 * 15 + 2) * 8 + 16;  // of at most 15 stages
  static constexpr int fixed_bytes = 1024 + barrier_bytes + sizeof(fp4_expert_table);
  static constexpr int segment =
      BN == 256 && (232448 - fixed_bytes - kFp4EpilogueWarps * 2048) / stage_bytes >= 4 ? 64 : 32;
  static constexpr int staging_bytes = kFp4EpilogueWarps * 32 * segment;
  static constexpr int overhead = fixed_bytes + staging_bytes;
  static constexpr int stages = (232448 - overhead) / stage_bytes;
  static constexpr int ring_bytes = stages * stage_bytes;
  static constexpr int smem_bytes = overhead + ring_bytes;
  static constexpr int acc1 = BN == 256 ? 192 : BN;  // columns of the second accumulator
  static constexpr int sf_column = acc1 + BN;
  static constexpr int tmem_columns = 512;
  static_assert(stages >= 4 && stages <= 15, "stage ring and its barriers");
  static_assert(sf_column + scale_tiles * 4 * (1 + b_tiles) <= tmem_columns, "TMEM");
  static_assert(BN * 128 * 4 <= ring_bytes, "the split's exchange fits the ring");
  static_assert(kFp4BlockM * 128 <= a_bytes + b_bytes + stages * (sfa_bytes + sfb_bytes),
                "the last stage's 128 rows end inside the ring");
};

namespace ptx {

// One lane of a converged warp. The tensor core's instructions take uniform
// registers; in a branch on this predicate the compiler knows that one lane
// runs and keeps the operands there. In a branch on `lane == 0` it moves each
// into place first: 170 cycles per MMA and 62 per scale copy at issue, against
// MMAs of 128 cycles (measured; 4096 x 8192 x 8192 MX: 156 -> 105 us). The same
// holds for TMA loads.
__device__ __forceinline__ bool elect_one() {
  std::uint32_t elected;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\t"
               "selp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(elected));
  return elected != 0;
}

// D (+)= A * B with block scales from TMEM.
template <bool kNv, bool kPair>
__device__ __forceinline__ void umma_fp4(std::uint32_t d, std::uint64_t a, std::uint64_t b,
                                         std::uint32_t idesc, std::uint32_t sfa,
                                         std::uint32_t sfb, std::uint32_t accumulate) {
#define MEGACU_FP4_MMA(group, kind)                                              \
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"                  \
               "tcgen05.mma.cta_group::" group ".kind::" kind                    \
               " [%0], %1, %2, %3, [%4], [%5], p;\n\t}"                          \
               :: "r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate) \
               : "memory")
  if constexpr (kNv && kPair) {
    MEGACU_FP4_MMA("2", "mxf4nvf4.block_scale.scale_vec::4X");
  } else if constexpr (kNv) {
    MEGACU_FP4_MMA("1", "mxf4nvf4.block_scale.scale_vec::4X");
  } else if constexpr (kPair) {
    MEGACU_FP4_MMA("2", "mxf4.block_scale.scale_vec::2X");
  } else {
    MEGACU_FP4_MMA("1", "mxf4.block_scale.scale_vec::2X");
  }
#undef MEGACU_FP4_MMA
}

// One scale tile (32 rows of 16 bytes in shared memory) into four TMEM
// columns, repeated for the four groups of 32 lanes; with kPair in both CTAs,
// each from its own shared memory.
template <bool kPair>
__device__ __forceinline__ void copy_scale_tile(std::uint32_t tmem, std::uint64_t desc) {
  if constexpr (kPair) {
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" :: "r"(tmem), "l"(desc)
                 : "memory");
  } else {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" :: "r"(tmem), "l"(desc)
                 : "memory");
  }
}

// Arrives on `bar` (with kPair: on both CTAs' barrier at that place) when
// every earlier copy and MMA of this thread has completed.
template <bool kPair>
__device__ __forceinline__ void commit_fp4(std::uint64_t *bar) {
  if constexpr (kPair) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64"
        " [%0], %1;"
        :: "r"(smem_addr(bar)), "h"(static_cast<std::uint16_t>(3))
        : "memory");
  } else {
    umma_commit(bar);
  }
}

// Shared memory by its own address space (the generic one costs more and
// keeps the compiler from ordering these freely against global stores).
__device__ __forceinline__ void st_shared_v4(std::uint32_t at, std::uint32_t a, std::uint32_t b,
                                             std::uint32_t c, std::uint32_t d) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};"
               :: "r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// map_to_rank of a shared::cta address.
__device__ __forceinline__ std::uint32_t map_to_rank(std::uint32_t local, std::uint32_t rank) {
  std::uint32_t out;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(out) : "r"(local), "r"(rank));
  return out;
}

__device__ __forceinline__ void st_shared_u32(std::uint32_t at, std::uint32_t v) {
  asm volatile("st.shared.u32 [%0], %1;" :: "r"(at), "r"(v) : "memory");
}

__device__ __forceinline__ uint4 ld_shared_v4(std::uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}

__device__ __forceinline__ std::uint32_t ld_shared_u32(std::uint32_t at) {
  std::uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
  return v;
}

__device__ __forceinline__ std::uint32_t ld_shared_u16(std::uint32_t at) {
  std::uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(at) : "memory");
  return v;
}

// Warps 0 and 1 wait for one another.
__device__ __forceinline__ void two_warps_sync() {
  __syncwarp();
  asm volatile("bar.sync 1, 64;" ::: "memory");
}

// Counts `bytes` of a barrier's announced ones as arrived.
__device__ __forceinline__ void mbar_complete_tx(std::uint64_t *bar, std::uint32_t bytes) {
  asm volatile("mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], %1;"
               :: "r"(smem_addr(bar)), "r"(bytes) : "memory");
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

// The expert whose rows hold tile row `tile` (whole warp; the experts' first
// tiles ascend, the row is below the last): how many e have first_tile(e + 1)
// <= tile, by two 32-wide counts.
template <class F>
__device__ __forceinline__ std::int32_t find_expert(F const &first_tile, std::int32_t experts,
                                                    std::int32_t tile) {
  std::int32_t const lane = static_cast<std::int32_t>(ptx::lane_id());
  std::int32_t const step = (experts + 31) / 32;
  std::int32_t const last = (lane + 1) * step;
  bool const below = last <= experts && first_tile(last) <= tile;
  std::int32_t const base = __popc(__ballot_sync(0xffffffffu, below)) * step;
  std::int32_t const at = base + lane + 1;
  bool const in = lane < step && at <= experts && first_tile(at) <= tile;
  return min(base + __popc(__ballot_sync(0xffffffffu, in)), experts - 1);
}

// What one tile row needs besides its raster place (whole warp).
struct fp4_rows {
  std::int32_t expert, valid;  // rows of the tile that exist
};

__device__ __forceinline__ fp4_rows locate_rows(fp4_gemm_params const &p,
                                                fp4_expert_table const &table, std::int32_t tile) {
  std::int32_t const row = tile * kFp4BlockM;
  fp4_rows r{0, p.rows - row};
  if (p.experts > kFp4TableExperts) {
    r.expert = find_expert([&](std::int32_t e) { return p.offsets[e] / kFp4BlockM; }, p.experts,
                           tile);
    r.valid = min(r.valid, p.counts[r.expert] - (row - p.offsets[r.expert]));
  } else if (p.experts > 0) {
    r.expert = find_expert(
        [&](std::int32_t e) { return static_cast<std::int32_t>(table.first_tile[e]); }, p.experts,
        tile);
    r.valid = min(r.valid, table.end[r.expert] - row);
  }
  return r;
}

// ptx::mbar_wait_cluster for a whole converged warp, with one answer: what
// follows are warp-wide instructions, and lanes that decided for themselves
// could give up apart.
__device__ __forceinline__ bool warp_wait(std::uint64_t *bar, std::uint32_t parity,
                                          std::uint32_t const *abort_word,
                                          unsigned long long timeout_ns) {
  std::uint32_t const a = ptx::smem_addr(bar);
  if (__all_sync(0xffffffffu, ptx::mbar_test_cluster(a, parity))) return true;
  std::uint64_t const start = ptx::now_ns();
  for (std::uint32_t spin = 1;; ++spin) {
    if (__all_sync(0xffffffffu, ptx::mbar_test_cluster(a, parity))) return true;
    if ((spin & 127u) == 0) {
      bool const over =
          ptx::ld_relaxed_gpu(abort_word) != 0 || ptx::now_ns() - start > timeout_ns;
      if (__any_sync(0xffffffffu, over)) return false;
    }
  }
}

// The waits of stage_ring.h on the `full` barriers.
struct fp4_drain {
  std::uint64_t *full;
  std::uint32_t follower_bytes;  // of one stage
  __device__ __forceinline__ void wait(std::uint32_t stage, std::uint32_t parity) const {
    ptx::mbar_wait(&full[stage], parity, nullptr, kFp4DrainNs);
  }
  __device__ __forceinline__ void announce(std::uint32_t stage) const {
    ptx::mbar_arrive_expect_tx(&full[stage], follower_bytes);
  }
  __device__ __forceinline__ void complete(std::uint32_t stage) const {
    ptx::mbar_complete_tx(&full[stage], follower_bytes);
  }
};

// A follower's epilogue warp gave up: the commit that it waited for may yet
// arrive here (the leader's MMA warp waits for its own arrival of the last). A
// call, since inlined it slows the epilogue.
__device__ __noinline__ void wait_commit(std::uint64_t *acc_full, std::uint32_t parity) {
  ptx::mbar_wait_cluster(acc_full, parity, nullptr, kFp4CommitNs);
}

// One thread of a pair's leader waits for both CTAs' loads after the MMA warp
// gave up.
template <class cfg>
__device__ __forceinline__ void drain_pair(std::uint32_t at, std::uint32_t loads,
                                           unsigned long long timeout_ns) {
  auto const volatile *const follower_loads =
      static_cast<std::uint32_t const volatile *>(__cvta_shared_to_generic(at + 4));
  auto *const full = static_cast<std::uint64_t *>(
      __cvta_shared_to_generic(at - 4 - (2 * cfg::stages + 2) * 8));
  // The follower's producer ends as soon as its wait does.
  std::uint64_t const start = ptx::now_ns();
  std::uint32_t theirs = 0;
  while ((theirs = *follower_loads) == 0) {
    std::uint64_t const waited = ptx::now_ns() - start;
    if (waited > timeout_ns && waited - timeout_ns > kFp4DrainNs) return;
  }
  drain_pair_ring(loads, theirs - 1, cfg::stages,
                  fp4_drain{full, kFp4BlockM * 128 + cfg::b_bytes + cfg::sfa_bytes +
                                      cfg::sfb_bytes});
}

// The end of a pair's producers (whole warps). Both CTAs' loads count on the
// leader's barriers, and an MMA warp that did not give up has seen them all
// land; else the leader's producer waits for them, knowing how many there are.
// `at`: the pair's two words.
template <class cfg>
__device__ __forceinline__ void end_pair_producer(std::uint32_t at, std::uint32_t loads,
                                                  bool leader, unsigned long long timeout_ns) {
  if (!leader) {
    if (ptx::lane_id() == 0) {
      ptx::st_shared_remote(ptx::map_to_rank(at + 4, 0), static_cast<std::int32_t>(loads + 1));
    }
    return;
  }
  ptx::two_warps_sync();  // the MMA warp has ended
  if (ptx::lane_id() == 0 && ptx::ld_shared_u32(at) != 0) drain_pair<cfg>(at, loads, timeout_ns);
}

__device__ __forceinline__ float locate_alpha(fp4_gemm_params const &p, std::int32_t expert) {
  return p.alphas != nullptr && p.experts > 0 ? p.alpha * p.alphas[expert] : p.alpha;
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

// Word i of a row's elements in the output type.
template <class Out, int kCount>
__device__ __forceinline__ std::uint32_t out_word(float const (&v)[kCount], int i) {
  if constexpr (std::is_same_v<Out, float>) {
    return __float_as_uint(v[i]);
  } else if constexpr (std::is_same_v<Out, __half>) {
    __half2 const h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
    return *reinterpret_cast<std::uint32_t const *>(&h);
  } else {
    return ptx::pack_bf16x2(v[2 * i], v[2 * i + 1]);
  }
}

// Where a warp's 32 rows of a tile go.
struct fp4_rows_out {
  std::uint8_t *base;        // row 0, column 0
  std::int64_t stride;       // bytes between rows
  std::int32_t rows;         // rows that exist
};

// Stores kCount consecutive columns from `col` of a warp's 32 rows (lane =
// row). Rows of 32-byte pieces go straight from the registers, a whole sector
// per lane (p.row_bytes = 32). Else kSegment bytes of each row at a time are
// turned through `stage` (no bank conflicts), so that neighbouring lanes write
// a row's segment in 16-byte pieces (p.row_bytes = 16) or its elements. The
// turn alone takes as long as the MMAs of 512 of K, since shared memory is
// busy with those (8192 x 4096 x 1024: 38 us with it, 28 without).
template <class Out, int kSegment, int kCount>
__device__ __forceinline__ void store_columns(fp4_gemm_params const &p, std::uint32_t stage,
                                              float const (&v)[kCount], fp4_rows_out const &out,
                                              std::int32_t col) {
  constexpr int kSize = sizeof(Out);
  std::uint32_t const lane = ptx::lane_id();
  if (p.row_bytes == 32 && col + kCount <= p.n) {
    if (static_cast<std::int32_t>(lane) < out.rows) {
      std::uint8_t *const dst =
          out.base + lane * out.stride + static_cast<std::int64_t>(col) * kSize;
#pragma unroll
      for (int i = 0; i < kCount * kSize / 32; ++i) {
        bytes32 q;
#pragma unroll
        for (int j = 0; j < 8; ++j) q.w[j] = out_word<Out>(v, i * 8 + j);
        store32(dst + i * 32, q);
      }
    }
    return;
  }
  constexpr int kBytes = kCount * kSize < kSegment ? kCount * kSize : kSegment;
  constexpr int kCols = kBytes / kSize;
  constexpr std::uint32_t kPieces = kBytes / 16;
  auto slot = [stage](std::uint32_t r, std::uint32_t c) {
    return stage + r * kBytes + ((c ^ (r * kPieces >> 3)) % kPieces) * 16;
  };
#pragma unroll
  for (int u = 0; u < kCount / kCols; ++u) {
    std::int32_t const first = col + u * kCols;
    if (first >= p.n) break;
#pragma unroll
    for (std::uint32_t c = 0; c < kPieces; ++c) {
      std::uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        w[i] = out_word<Out>(v, (u * kBytes + static_cast<int>(c) * 16) / 4 + i);
      }
      ptx::st_shared_v4(slot(lane, c), w[0], w[1], w[2], w[3]);
    }
    __syncwarp();
    std::uint8_t *const dst = out.base + static_cast<std::int64_t>(first) * kSize;
    if (p.row_bytes >= 16 && first + kCols <= p.n) {
      uint4 q[kPieces];
#pragma unroll
      for (std::uint32_t h = 0; h < kPieces; ++h) {
        q[h] = ptx::ld_shared_v4(slot(lane / kPieces + h * (32 / kPieces), lane % kPieces));
      }
#pragma unroll
      for (std::uint32_t h = 0; h < kPieces; ++h) {
        std::uint32_t const r = lane / kPieces + h * (32 / kPieces);
        if (static_cast<std::int32_t>(r) < out.rows) {
          *reinterpret_cast<uint4 *>(dst + r * out.stride + lane % kPieces * 16) = q[h];
        }
      }
    } else {
      // kCols lanes per row, an element each.
      std::uint32_t const e = lane % kCols, step = 32 / kCols;
      if (first + static_cast<std::int32_t>(e) < p.n) {
#pragma unroll 4
        for (std::uint32_t r = lane / kCols; r < 32; r += step) {
          if (static_cast<std::int32_t>(r) >= out.rows) break;
          std::uint32_t const at = slot(r, e * kSize / 16) + e * kSize % 16;
          if constexpr (kSize == 4) {
            *reinterpret_cast<std::uint32_t *>(dst + r * out.stride + e * 4) =
                ptx::ld_shared_u32(at);
          } else {
            *reinterpret_cast<std::uint16_t *>(dst + r * out.stride + e * 2) =
                static_cast<std::uint16_t>(ptx::ld_shared_u16(at));
          }
        }
      }
    }
    __syncwarp();
  }
}

template <int kSegment, int kCount>
__device__ __forceinline__ void store_columns(fp4_gemm_params const &p, std::uint32_t stage,
                                              float const (&v)[kCount], fp4_rows_out const &out,
                                              std::int32_t col) {
  if (p.out_dtype == 3) {
    store_columns<float, kSegment, kCount>(p, stage, v, out, col);
  } else if (p.out_dtype == 1) {
    store_columns<__half, kSegment, kCount>(p, stage, v, out, col);
  } else {
    store_columns<__nv_bfloat16, kSegment, kCount>(p, stage, v, out, col);
  }
}

__device__ __forceinline__ fp4_rows_out rows_out(fp4_gemm_params const &p, std::int64_t row,
                                                 std::int32_t rows) {
  std::int64_t const stride = p.out_stride * (p.out_dtype == 3 ? 4 : 2);
  return {static_cast<std::uint8_t *>(p.out) + row * stride, stride, rows};
}

// silu(g) * u with exp(-|g|), which neither overflows nor drives the fast
// division out of its range: g / (1 + e) for g >= 0, g e / (1 + e) below.
__device__ __forceinline__ float swiglu(float g, float u) {
  float const e = __expf(-fabsf(g));
  return __fdividef(g < 0.0f ? g * e : g, 1.0f + e) * u;
}

}  // namespace detail

template <bool kNv, bool kSwiglu, int BN, bool kPair, int kRows>
__global__ void __launch_bounds__(kFp4Threads, 1)
    fp4_gemm_kernel(__grid_constant__ fp4_maps const maps,
                    __grid_constant__ fp4_gemm_params const p) {
  using cfg = fp4_config<kNv, BN, kPair, kRows>;
  static_assert(!kSwiglu || BN == 256, "128 gate and 128 up columns");
  static_assert(!kPair || BN == 256, "pairs compute 256 x 256 tiles");
  constexpr std::uint32_t kStages = cfg::stages;
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
  // Two words of a pair's leader: whether its MMA warp gave up, and 1 + the
  // follower's loads once its producer has ended. Their address is computed
  // anew at each use, so that the epilogue holds no register for it.
  auto pair_words = [] {
    std::uint32_t raw;
    asm volatile("mov.u32 %0, %1;" : "=r"(raw) : "r"(ptx::smem_addr(raw_smem)));
    return ((raw + 1023u) & ~1023u) + cfg::ring_bytes + cfg::staging_bytes +
           (2 * kStages + 2) * 8 + 4;
  };
  auto &table = *reinterpret_cast<fp4_expert_table *>(staging + cfg::staging_bytes + cfg::barrier_bytes);
  std::uint32_t *const abort_word = &reinterpret_cast<control_block *>(p.events)->error_code;

  std::int32_t const warp =
      __shfl_sync(0xffffffffu, static_cast<std::int32_t>(threadIdx.x) / 32, 0);
  std::uint32_t const lane = ptx::lane_id();
  // A cluster is a pair, or the CTAs that share a tile's K, or one CTA.
  std::int32_t const split = kPair ? 1 : p.split;
  std::int32_t const cluster = kPair ? 2 : split;
  std::int32_t const rank =
      cluster > 1 ? static_cast<std::int32_t>(ptx::cluster_ctarank()) : 0;
  std::int32_t const unit0 = static_cast<std::int32_t>(blockIdx.x) / cluster;
  std::int32_t const units = static_cast<std::int32_t>(gridDim.x) / cluster;
  std::int32_t const k_blocks = (p.k + kFp4BlockK - 1) / kFp4BlockK;
  std::int32_t const kb0 = kPair ? 0 : rank * k_blocks / split;
  std::int32_t const kb1 = kPair ? k_blocks : (rank + 1) * k_blocks / split;
  bool const leader = !kPair || rank == 0;

  // Set-up that reads nothing of earlier kernels.
  grid_start_next();
  if (warp == 0) {
    // Lane s sets up stage s (kStages <= 15).
    if (lane < kStages) {
      ptx::mbar_init(&full[lane], 1);
      ptx::mbar_init(&empty[lane], 1);
    } else if (lane == 16) {
      ptx::mbar_init(acc_full, 1);
      ptx::mbar_init(acc_free, kFp4EpilogueWarps * (kPair ? 2 : 1));
      if constexpr (kPair) {
        ptx::st_shared_u32(pair_words(), 0);
        ptx::st_shared_u32(pair_words() + 4, 0);
      }
    }
    ptx::fence_barrier_init();
    ptx::fence_proxy_async_shared();
    __syncwarp();
  } else if (warp == 1) {
    if constexpr (kPair) {
      ptx::tmem_alloc_pair(tmem_slot, cfg::tmem_columns);
      ptx::tmem_relinquish_pair();
    } else {
      ptx::tmem_alloc(tmem_slot, cfg::tmem_columns);
      ptx::tmem_relinquish();
    }
  } else if (warp == 2 && ptx::elect_one()) {
    ptx::prefetch_tensor_map(&maps.a);
    ptx::prefetch_tensor_map(&maps.a_small);
    ptx::prefetch_tensor_map(&maps.b);
    ptx::prefetch_tensor_map(&maps.a_scales);
    ptx::prefetch_tensor_map(&maps.b_scales);
    if constexpr (kSwiglu) {
      ptx::prefetch_tensor_map(&maps.b2);
      ptx::prefetch_tensor_map(&maps.b2_scales);
    }
  }
  grid_wait();

  std::int32_t const m_tiles =
      p.experts > 0 ? min(p.offsets[p.experts] / kFp4BlockM, p.m_tiles) : p.m_tiles;
  // Rows of tiles as the raster counts them: pairs of 128-row tiles, or tiles.
  std::int32_t const unit_rows = kPair ? (m_tiles + 1) / 2 : m_tiles;
  std::int32_t const tiles = unit_rows * p.n_tiles;
  // The 128-row tile of this CTA and the column tile of unit t.
  auto locate = [&](std::int32_t t) {
    fp4_tile c = fp4_locate(t, unit_rows, p.n_tiles, p.group_m);
    if constexpr (kPair) c.row = 2 * c.row + rank;
    return c;
  };

  // Loads of the k-block `kb` of a tile into `stage` (one lane).
  struct load_place {
    std::int32_t row, a_tile, b_row, b_tile, boxes;
  };
  auto place = [&](std::int32_t t) {  // whole warp
    fp4_tile const c = locate(t);
    load_place l;
    l.row = c.row * kFp4BlockM;
    detail::fp4_rows const rows = detail::locate_rows(p, table, c.row);
    l.boxes = min(max((rows.valid + kFp4SmallRows - 1) / kFp4SmallRows, 1), kRows / kFp4SmallRows);
    if constexpr (kPair) l.boxes = 4;  // both CTAs' bytes are counted by the leader
    l.a_tile = min(c.row, m_tiles - 1) * p.scale_tiles;  // a pair's second tile may not exist
    l.b_row = rows.expert * p.n + c.col * kActCols;
    l.b_tile = (rows.expert * p.n_row_tiles + c.col * kActCols / 128) * p.scale_tiles;
    return l;
  };
  auto load = [&](load_place const &l, std::int32_t kb, std::uint32_t stage) {
    std::int32_t const st = kb * cfg::scale_tiles;
    std::uint8_t *const sa = smem + stage * (cfg::a_bytes + cfg::b_bytes);
    std::uint8_t *const sb = sa + cfg::a_bytes;
    std::uint8_t *const sfa = scales + stage * (cfg::sfa_bytes + cfg::sfb_bytes);
    std::uint8_t *const sfb = sfa + cfg::sfa_bytes;
    std::uint32_t const bar = kPair ? ptx::map_to_rank(&full[stage], 0) : 0;
    auto tma = [&](CUtensorMap const &map, void *dst, std::int32_t x, std::int32_t y) {
      if constexpr (kPair) {
        ptx::tma_load_2d_pair(&map, bar, dst, x, y);
      } else {
        ptx::tma_load_2d(&map, &full[stage], dst, x, y);
      }
    };
    if (leader) {
      std::uint32_t const mine = static_cast<std::uint32_t>(l.boxes) * kFp4SmallRows * 128 +
                                 cfg::b_bytes + cfg::sfa_bytes + cfg::sfb_bytes;
      ptx::mbar_arrive_expect_tx(&full[stage], mine * (kPair ? 2 : 1));
    }
    std::int32_t const x = kb * 128;
    if (l.boxes == 4) {
      tma(maps.a, sa, x, l.row);
    } else {
      for (std::int32_t i = 0; i < l.boxes; ++i) {
        tma(maps.a_small, sa + i * kFp4SmallRows * 128, x, l.row + i * kFp4SmallRows);
      }
    }
    if constexpr (kSwiglu) {
      if constexpr (kPair) {  // the leader stages gate, the other CTA up
        tma(leader ? maps.b : maps.b2, sb, x, l.b_row);
      } else {
        tma(maps.b, sb, x, l.b_row);
        tma(maps.b2, sb + cfg::b_bytes / 2, x, l.b_row);
      }
    } else {
      tma(maps.b, sb, x, l.b_row + (kPair ? rank * (BN / 2) : 0));
    }
    // Scale tiles: a box of a stage's tiles; past a row tile's last one it
    // holds other tiles or zeros, which no MMA reads.
    tma(maps.a_scales, sfa, 0, l.a_tile + st);
    tma(maps.b_scales, sfb, 0, l.b_tile + st);
    if constexpr (kSwiglu) {
      tma(maps.b2_scales, sfb + cfg::sfa_bytes, 0, l.b_tile + st);
    } else if constexpr (BN == 256) {
      tma(maps.b_scales, sfb + cfg::sfa_bytes, 0, l.b_tile + p.scale_tiles + st);
    }
  };

  std::uint32_t issued = 0;  // by the producer, in all
  if (!kPair && p.experts > 0) {
    if (p.experts <= kFp4TableExperts) {
      for (std::int32_t e = static_cast<std::int32_t>(threadIdx.x); e <= p.experts;
           e += kFp4Threads) {
        std::int32_t const offset = p.offsets[e];
        table.first_tile[e] = static_cast<std::uint16_t>(offset / kFp4BlockM);
        if (e < p.experts) table.end[e] = offset + p.counts[e];
      }
    }
    __syncthreads();
  }
  if (!kPair && warp == 0 && unit0 < tiles) {
    load_place const l = place(unit0);
    issued = static_cast<std::uint32_t>(min(kb1 - kb0, static_cast<std::int32_t>(kStages)));
    if (ptx::elect_one()) {
      for (std::uint32_t s = 0; s < issued; ++s) load(l, kb0 + static_cast<std::int32_t>(s), s);
    }
    __syncwarp();
  }
  ptx::tc_fence_before_sync();
  __syncthreads();
  if constexpr (kPair) ptx::cluster_sync();  // both CTAs' barriers exist
  ptx::tc_fence_after_sync();
  std::uint32_t const tmem = *tmem_slot;

  if (warp == 0) {
    // ---------------- TMA producer ----------------
    std::uint32_t stage = issued % kStages, phase = issued / kStages & 1u;
    std::int32_t skip = static_cast<std::int32_t>(issued);  // loaded during the set-up
    bool ok = true;
    for (std::int32_t t = unit0; ok && t < tiles; t += units) {
      load_place const l = place(t);
      for (std::int32_t kb = kb0 + skip; kb < kb1; ++kb) {
        if (!detail::warp_wait(&empty[stage], phase ^ 1u, abort_word, p.timeout_ns)) {
          if (lane == 0) detail::fp4_error(p.events, static_cast<std::uint32_t>(t), 51);
          ok = false;
          break;
        }
        __syncwarp();
        if (ptx::elect_one()) load(l, kb, stage);
        __syncwarp();
        ++issued;
        if (++stage == kStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      skip = 0;
    }
    if constexpr (kPair) {
      detail::end_pair_producer<cfg>(pair_words(), issued, leader, p.timeout_ns);
      __syncwarp();
    } else {
      drain_ring(issued, kStages, detail::fp4_drain{full, 0});
    }
  } else if (warp == 1 && leader) {
    // ---------------- scale copies and MMA issue ----------------
    std::uint32_t stage = 0, phase = 0, tile_index = 0, committed = 0;
    std::uint32_t const sf = tmem + cfg::sf_column;
    // Descriptors of stage 0; a stage is a multiple of 16 bytes further.
    std::uint64_t const a_desc0 = ptx::smem_desc_sw128(ptx::smem_addr(smem), 16, 1024);
    std::uint64_t const b_desc0 = a_desc0 + (cfg::a_bytes >> 4);
    std::uint64_t const sf_desc0 = ptx::scale_desc(ptx::smem_addr(scales));
    bool ok = true;
    for (std::int32_t t = unit0; ok && t < tiles; t += units, ++tile_index) {
      if (tile_index > 0 &&
          !detail::warp_wait(acc_free, (tile_index - 1) & 1u, abort_word, p.timeout_ns)) {
        if (lane == 0) detail::fp4_error(p.events, static_cast<std::uint32_t>(t), 52);
        ok = false;
        break;
      }
      ptx::tc_fence_after_sync();
      std::uint32_t const acc = tmem + (tile_index & 1u) * cfg::acc1;
      // A tile of 64 columns uses half of a scale tile's four TMEM columns.
      std::uint32_t const b_half = BN == 64 ? (locate(t).col & 1) * 2u : 0u;
      for (std::int32_t kb = kb0; kb < kb1; ++kb) {
        if (!detail::warp_wait(&full[stage], phase, abort_word, p.timeout_ns)) {
          if (lane == 0) detail::fp4_error(p.events, static_cast<std::uint32_t>(t), 53);
          ok = false;
          break;
        }
        __syncwarp();
        ptx::tc_fence_after_sync();
        std::uint32_t const at = stage * ((cfg::a_bytes + cfg::b_bytes) >> 4);
        std::uint32_t const sf_at = stage * ((cfg::sfa_bytes + cfg::sfb_bytes) >> 4);
        std::int32_t const steps = min(4, (p.k - kb * kFp4BlockK + 63) / 64);
        if (ptx::elect_one()) {
          // All of the stage's scale tiles, then its MMAs.
          std::int32_t const scale_steps = kNv ? steps : (steps + 1) / 2;
#pragma unroll
          for (std::int32_t st = 0; st < cfg::scale_tiles; ++st) {
            if (st >= scale_steps) break;
            std::uint32_t const ta = sf + st * 4 * (1 + cfg::b_tiles);
#pragma unroll
            for (int h = 0; h < 1 + cfg::b_tiles; ++h) {  // A's, then B's row tiles
              ptx::copy_scale_tile<kPair>(
                  ta + 4 * h, sf_desc0 + sf_at + ((h * cfg::sfa_bytes + st * kScaleTileBytes) >> 4));
            }
          }
#pragma unroll
          for (std::int32_t j = 0; j < 4; ++j) {
            if (j >= steps) break;
            // NV: one scale tile per 64 of K; MX: one per 128, a byte pair each.
            std::uint32_t const ta = sf + (kNv ? j : j / 2) * 4 * (1 + cfg::b_tiles);
            ptx::umma_fp4<kNv, kPair>(
                acc, a_desc0 + at + j * 2, b_desc0 + at + j * 2,
                fp4_idesc<kNv>(kFp4BlockM * (kPair ? 2 : 1), BN, kNv ? 0 : j % 2 * 2), ta, ta + 4 + b_half,
                kb > kb0 || j > 0);
          }
          ptx::commit_fp4<kPair>(&empty[stage]);
        }
        __syncwarp();
        if (++stage == kStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (ptx::elect_one()) ptx::commit_fp4<kPair>(acc_full);
      ++committed;
      __syncwarp();
    }
    // MMAs in flight end before the CTA may free its TMEM. (A tile starts when
    // the commit of the one before has arrived: one phase is open at most.)
    if (committed > 0) {
      ptx::mbar_wait_cluster(acc_full, (committed - 1) & 1u, nullptr, kFp4DrainNs);
    }
    if constexpr (kPair) {
      if (!ok && lane == 0) ptx::st_shared_u32(pair_words(), 1);
      ptx::two_warps_sync();  // with the producer's end
    }
    __syncwarp();
  } else if (warp >= 2) {
    // ---------------- epilogue ----------------
    std::int32_t const quarter = warp & 3;       // TMEM lanes [32 quarter, +32)
    std::int32_t const half = (warp - 2) / 4;    // chunks half, half + 2, ...
    std::uint32_t const stage = ptx::smem_addr(staging + (warp - 2) * 32 * cfg::segment);
    std::uint32_t const lanes = static_cast<std::uint32_t>(quarter * 32) << 16;
    std::uint32_t const free_bar = kPair ? ptx::map_to_rank(acc_free, 0) : 0;
    std::uint32_t tile_index = 0;
    for (std::int32_t t = unit0; t < tiles; t += units, ++tile_index) {
      fp4_tile const c = locate(t);
      std::int32_t const row = c.row * kFp4BlockM;
      detail::fp4_rows const rows = detail::locate_rows(p, table, c.row);
      float const alpha = detail::locate_alpha(p, rows.expert);
      detail::fp4_rows_out const out =
          detail::rows_out(p, row + quarter * 32, rows.valid - quarter * 32);
      if (!detail::warp_wait(acc_full, tile_index & 1u, abort_word, p.timeout_ns)) {
        if (lane == 0) detail::fp4_error(p.events, static_cast<std::uint32_t>(t), 54);
        if constexpr (kPair) {
          if (!leader) detail::wait_commit(acc_full, tile_index & 1u);
        }
        break;
      }
      __syncwarp();
      ptx::tc_fence_after_sync();
      if (split > 1) break;  // the cluster's exchange below
      std::uint32_t const acc = tmem + lanes + (tile_index & 1u) * cfg::acc1;
      // The next tile's MMAs may start: with BN = 256 once the shared columns
      // are drained, else at once, since the other accumulator is.
      auto release = [&] {
        ptx::tc_fence_before_sync();
        if (lane == 0) {
          if constexpr (kPair) {
            // Relaxed: nothing of this thread's memory is published, the TMEM
            // loads have completed, and a release would wait for the last
            // tile's stores (1400 cycles of every tile).
            ptx::mbar_arrive_remote_relaxed(free_bar);
          } else {
            ptx::mbar_arrive(acc_free);
          }
        }
      };
      if (BN < 256) release();
      // Chunks of 32 output columns, the shared TMEM columns (192..255) first:
      // in the first accumulator the last two, in the second the first two.
      constexpr int kChunks = kActCols / 32;
      int const first = half + (BN == 256 && (tile_index & 1u) == 0 ? kChunks - 2 : 0);
      std::uint32_t raw[32], up[kSwiglu ? 32 : 1];
      auto fetch = [&](int chunk) {
        ptx::tmem_load_32x32b_x32(acc + chunk * 32, raw);
        if constexpr (kSwiglu) ptx::tmem_load_32x32b_x32(acc + kActCols + chunk * 32, up);
      };
      fetch(first);
#pragma unroll 1
      for (int i = 0; i < kChunks / 2; ++i) {
        int const chunk = (first + 2 * i) % kChunks;
        float v[32];
        ptx::tmem_wait_load();
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          asm volatile("" : "+r"(raw[e]));  // not used before the wait
          if constexpr (kSwiglu) asm volatile("" : "+r"(up[e]));
          if constexpr (kSwiglu) {
            v[e] = detail::swiglu(alpha * __uint_as_float(raw[e]), alpha * __uint_as_float(up[e]));
          } else {
            v[e] = alpha * __uint_as_float(raw[e]);
          }
        }
        if (BN == 256 && i == 0) release();
        if (i + 1 < kChunks / 2) fetch((chunk + 2) % kChunks);  // in flight during the stores
        std::int32_t const col = c.col * kActCols + chunk * 32;
        if (out.rows > 0 && col < p.n) detail::store_columns<cfg::segment>(p, stage, v, out, col);
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
    std::int32_t const slice = kActCols / split;  // output columns per CTA
    constexpr int kParts = kSwiglu ? 2 : 1;
    std::int32_t const quarter = warp & 3, half = (warp - 2) / 4;
    fp4_tile c{0, 0};
    detail::fp4_rows_out out{nullptr, 0, 0};
    float alpha = 1.0f;
    if (warp >= 2 && unit0 < tiles) {
      c = locate(unit0);
      detail::fp4_rows const rows = detail::locate_rows(p, table, c.row);
      out = detail::rows_out(p, c.row * kFp4BlockM + quarter * 32, rows.valid - quarter * 32);
      alpha = detail::locate_alpha(p, rows.expert);
    }
    if (out.rows > 0) {
      ptx::tc_fence_after_sync();
      std::uint32_t const acc = tmem + (static_cast<std::uint32_t>(quarter * 32) << 16);
#pragma unroll 1
      for (int chunk = half; chunk < BN / 32; chunk += 2) {
        std::uint32_t raw[32];
        ptx::tmem_load_32x32b_x32(acc + chunk * 32, raw);
        ptx::tmem_wait_load();
        if (static_cast<std::int32_t>(lane) < out.rows) {
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
    __syncwarp();
    ptx::cluster_sync();
    if (out.rows > 0) {
      std::uint32_t const stage = ptx::smem_addr(staging + (warp - 2) * 32 * cfg::segment);
      std::uint32_t const mine = (static_cast<std::uint32_t>(quarter * 32) + lane) * 16;
      for (std::int32_t c0 = half * 16; c0 < slice; c0 += 32) {
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
        detail::store_columns<cfg::segment>(p, stage, v, out, col);
      }
    }
  }

  ptx::tc_fence_before_sync();
  __syncthreads();
  if constexpr (kPair) ptx::cluster_sync();  // no more accesses to the other CTA
  if (warp == 1) {
    ptx::tc_fence_after_sync();
    if constexpr (kPair) {
      ptx::tmem_dealloc_pair(tmem, cfg::tmem_columns);
    } else {
      ptx::tmem_dealloc(tmem, cfg::tmem_columns);
    }
  }
}

}  // namespace megacu_b200
