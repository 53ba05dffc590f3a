// 4-bit block formats (no counterpart in megacu): quantisation, the values
// back, and the products of quantised matrices, dense or by expert.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdint>

#include <megacu_b200.h>

#include "kernels/fp4_gemm_kernel.cuh"
#include "kernels/fp4_quant_kernel.cuh"
#include "status.h"
#include "tma_map.h"

namespace {

using namespace megacu_b200;

constexpr int kMaxDevices = 64;
constexpr std::int64_t kMaxDim = 1ll << 30;
constexpr std::int32_t kMaxExperts = 1024;
constexpr int kMaxLog2Scale = 60;

bool known_format(std::int32_t f) { return f == MEGACU_FP4_MX || f == MEGACU_FP4_NV; }
bool known_dtype(std::int32_t t) {
  return t == MEGACU_DTYPE_F16 || t == MEGACU_DTYPE_BF16 || t == MEGACU_DTYPE_F32;
}
int element_size(std::int32_t dtype) { return dtype == MEGACU_DTYPE_F32 ? 4 : 2; }

std::int64_t ceil_div(std::int64_t a, std::int64_t b) { return (a + b - 1) / b; }

std::int64_t scale_tiles(std::int64_t cols, bool nv) { return ceil_div(cols, fp4_tile_cols(nv)); }

megacu_status check_matrix(megacu_fp4_matrix const *m, int &log2_scale) {
  if (m == nullptr) return fail(MEGACU_INVALID_ARGUMENT, 2, "missing matrix");
  if (m->rows < 0 || m->cols < 1 || m->stride < 0 || m->topk < 0 || m->x_rows < 0) {
    return fail(MEGACU_INVALID_ARGUMENT, 1, "invalid matrix");
  }
  if (!known_format(m->format)) return fail(MEGACU_INVALID_ARGUMENT, 1, "unknown format");
  if (!known_dtype(m->dtype)) return fail(MEGACU_UNSUPPORTED, 20, "dtype must be f16, bf16 or f32");
  if (m->cols % 32 != 0) {
    return fail(MEGACU_INVALID_ARGUMENT, 21, "cols must be a multiple of 32 (16-byte rows)");
  }
  if (m->rows > kMaxDim || m->cols > kMaxDim || m->x_rows > kMaxDim ||
      2 * ceil_div(m->rows, kScaleTileRows) * ceil_div(m->cols, kQuantCols) > 0x7fffffffll) {
    return fail(MEGACU_UNSUPPORTED, 22, "dimension too large");
  }
  int e = 0;
  if (!(std::frexp(m->scale, &e) == 0.5f) || e - 1 > kMaxLog2Scale || e - 1 < -kMaxLog2Scale) {
    return fail(MEGACU_INVALID_ARGUMENT, 1, "scale must be a power of two, 2^-60 to 2^60");
  }
  log2_scale = e - 1;
  return ok_status();
}

fp4_matrix_params matrix_params(megacu_fp4_matrix const &m, int log2_scale, void *data,
                                void *scales, bool transpose) {
  fp4_matrix_params p{};
  p.rows = m.rows;
  p.cols = static_cast<std::int32_t>(m.cols);
  p.stride = m.stride != 0 ? m.stride : transpose ? m.rows : m.cols;
  p.log2_scale = log2_scale;
  p.tiles = static_cast<std::int32_t>(scale_tiles(m.cols, m.format == MEGACU_FP4_NV));
  p.col_tiles = static_cast<std::uint32_t>(ceil_div(m.cols, kQuantCols));
  p.topk = m.topk;
  p.x_rows = m.x_rows;
  p.data = static_cast<std::uint8_t *>(data);
  p.scales = static_cast<std::uint8_t *>(scales);
  return p;
}

// Calls f with the element type (a value of it) and the format as constants.
template <class F>
void by_type(std::int32_t dtype, std::int32_t format, F f) {
  auto with = [&](auto value) {
    if (format == MEGACU_FP4_NV) {
      f(value, std::true_type{});
    } else {
      f(value, std::false_type{});
    }
  };
  if (dtype == MEGACU_DTYPE_F16) {
    with(__half{});
  } else if (dtype == MEGACU_DTYPE_BF16) {
    with(__nv_bfloat16{});
  } else {
    with(float{});
  }
}

// ---- product ---------------------------------------------------------------------

// Bytes [rows, k / 2] in boxes of box_rows x 128 bytes, 128-byte swizzle.
bool encode_fp4_map(CUtensorMap *map, void const *base, std::int64_t rows, std::int64_t k,
                    std::uint32_t box_rows) {
  auto const encode = tensor_map_encoder();
  if (encode == nullptr) return false;
  cuuint64_t const dims[2] = {static_cast<cuuint64_t>(k / 2), static_cast<cuuint64_t>(rows)};
  cuuint64_t const strides[1] = {static_cast<cuuint64_t>(k / 2)};
  cuuint32_t const box[2] = {128, box_rows};
  cuuint32_t const elem[2] = {1, 1};
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(base), dims, strides,
                box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Scale tiles, 512 bytes each, in boxes of `box` consecutive ones.
bool encode_scale_map(CUtensorMap *map, void const *base, std::int64_t tiles, std::uint32_t box) {
  auto const encode = tensor_map_encoder();
  if (encode == nullptr) return false;
  cuuint64_t const dims[2] = {kScaleTileBytes / 4, static_cast<cuuint64_t>(tiles)};
  cuuint64_t const strides[1] = {kScaleTileBytes};
  cuuint32_t const boxes[2] = {kScaleTileBytes / 4, box};
  cuuint32_t const elem[2] = {1, 1};
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, const_cast<void *>(base), dims, strides,
                boxes, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct fp4_plan {
  int tile_n = 256;  // accumulator columns of a tile
  int split = 1;
  bool pair = false;
  std::int64_t m_tiles = 0, n_tiles = 0;
};

// The plan is made for a B200's SMs, whatever the device: it decides what is
// refused too, also by calls without a stream. The grid goes by the device.
constexpr int kPlanSms = 148;

// Clusters of `split` CTAs, one CTA per SM, that run at once: an SM's cluster
// stays within its GPC, and a B200's GPCs hold 33 clusters of 4 and 15 of 8
// (the occupancy query's answer; 16 x 2048 x 4096 split in eight, 16 clusters,
// took 11.6 us against 6.7 for 15).
std::int64_t clusters_at_once(int split) {
  return split == 8 ? 15 : split == 4 ? 33 : kPlanSms / split;
}

// Tile width and K split with the least time on the busiest SM, in us, fitted
// to measured calls on a B200 (16 to 128 rows, N 8192, K 256 / 3584 / 14336):
// a call's start-up and end, a k-block of 256 at each width (what an SM can
// load in a time that its MMAs do not exceed), a further tile on the same SM,
// and the exchange of a split, which grows with the tile's accumulators.
// 16 x 8192 x 3584: tile_n 64 takes 6.4 us, 128 6.5, 256 8.7, 128 split in two
// 8.0, 256 split in four 9.2.
// The costs are a single CTA's; whether tiles run as pairs is decided after the
// choice. It holds past the fit all the same: with 129 to 2000 rows the choice
// was within 1 % of the best of 256, 128 and 64 columns, whole or split, at
// N x K 8192 x 3584, 4096 x 4096 and 1792 x 8192 (1000 rows 15.5, 11.0 and
// 11.4 us), and at 14336 x 1024 but for 129 to 256 rows (7.0 us, 128 columns
// 6.0).
megacu_status make_plan(megacu_fp4_gemm_problem const &p, bool swiglu, fp4_plan &out) {
  std::int64_t const k_blocks = ceil_div(p.k, kFp4BlockK);
  double best = -1.0;
  for (int tile_n : {256, 128, 64}) {
    if ((swiglu && tile_n != 256) || (p.tile_n != 0 && p.tile_n != tile_n)) continue;
    double const start = tile_n == 256 ? 4.6 : tile_n == 128 ? 3.8 : 3.6;
    double const per_block = tile_n == 256 ? 0.40 : tile_n == 128 ? 0.25 : 0.21;
    for (int split : {1, 2, 4, 8}) {
      if (split > k_blocks || 16 * split > tile_n || (p.split != 0 && p.split != split)) continue;
      std::int64_t const m_tiles = ceil_div(p.m, kFp4BlockM);
      std::int64_t const n_tiles = ceil_div(p.n, swiglu ? tile_n / 2 : tile_n);
      std::int64_t const waves =
          std::max<std::int64_t>(ceil_div(m_tiles * n_tiles, clusters_at_once(split)), 1);
      double const rows = static_cast<double>(std::min<std::int64_t>(p.m, kFp4BlockM));
      double const exchange = split > 1 ? 1.5 + 0.035 * rows * tile_n / 256 : 0.0;
      double const cost = start + 0.6 * static_cast<double>(waves - 1) +
                          static_cast<double>(waves) *
                              (per_block * static_cast<double>(ceil_div(k_blocks, split)) + exchange);
      if (best < 0.0 || cost < best) {
        best = cost;
        out = {tile_n, split, false, m_tiles, n_tiles};
      }
    }
  }
  if (best < 0.0) return fail(MEGACU_UNSUPPORTED, 22, "tile_n or split not possible");
  out.pair = p.experts == 0 && out.tile_n == 256 && out.split == 1 && out.m_tiles > 1;
  if (out.m_tiles * out.n_tiles * out.split > (1 << 28)) {
    return fail(MEGACU_UNSUPPORTED, 22, "too many tiles");
  }
  return ok_status();
}

struct fp4_operands {
  void const *a, *a_scales, *b, *b_scales, *b2, *b2_scales;
};

template <bool kNv, bool kSwiglu, int BN, bool kPair = false, int kRows = kFp4BlockM>
cudaError_t launch_gemm(int device, int grid, cudaStream_t stream, fp4_maps const &maps,
                        fp4_gemm_params const &prm) {
  constexpr auto kKernel = &fp4_gemm_kernel<kNv, kSwiglu, BN, kPair, kRows>;
  constexpr int kSmem = fp4_config<kNv, BN, kPair, kRows>::smem_bytes;
  static std::atomic<bool> configured[kMaxDevices] = {};
  bool const known = device >= 0 && device < kMaxDevices;
  if (!known || !configured[device].load(std::memory_order_acquire)) {
    cudaError_t const e =
        cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e != cudaSuccess) return e;
    if (known) configured[device].store(true, std::memory_order_release);
  }
  if constexpr (kPair) {
    // As many clusters as the device holds at once, each for several tiles.
    static std::atomic<int> max_pairs[kMaxDevices] = {};
    int pairs = known ? max_pairs[device].load(std::memory_order_acquire) : 0;
    if (pairs == 0) {
      cudaLaunchConfig_t cfg{};
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = 2;
      attr[0].val.clusterDim.y = 1;
      attr[0].val.clusterDim.z = 1;
      cfg.gridDim = dim3(2);
      cfg.blockDim = dim3(kFp4Threads);
      cfg.dynamicSmemBytes = kSmem;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      cudaError_t const e = cudaOccupancyMaxActiveClusters(&pairs, kKernel, &cfg);
      if (e != cudaSuccess) return e;
      if (pairs < 1) return cudaErrorInvalidConfiguration;
      if (known) max_pairs[device].store(pairs, std::memory_order_release);
    }
    grid = std::min(grid, 2 * pairs);
  }
  return launch_chained(kKernel, static_cast<unsigned>(grid), kFp4Threads, kSmem, stream,
                        static_cast<unsigned>(kPair ? 2 : prm.split), maps, prm);
}

template <bool kNv>
cudaError_t launch_plan(fp4_plan const &plan, bool swiglu, int device, int grid,
                        cudaStream_t stream, fp4_maps const &maps, fp4_gemm_params const &prm) {
  if (swiglu) {
    return plan.pair ? launch_gemm<kNv, true, 256, true>(device, grid, stream, maps, prm)
                     : launch_gemm<kNv, true, 256>(device, grid, stream, maps, prm);
  }
  if (plan.tile_n == 256) {
    return plan.pair ? launch_gemm<kNv, false, 256, true>(device, grid, stream, maps, prm)
                     : launch_gemm<kNv, false, 256>(device, grid, stream, maps, prm);
  }
  if (plan.tile_n == 128) return launch_gemm<kNv, false, 128>(device, grid, stream, maps, prm);
  // At most 32 rows: stages without the missing rows, so more of them (13 to
  // 15 against 7 or 8, the weights of most K's whole tile in flight).
  if (prm.experts == 0 && prm.rows <= kFp4SmallRows) {
    return launch_gemm<kNv, false, 64, false, kFp4SmallRows>(device, grid, stream, maps, prm);
  }
  return launch_gemm<kNv, false, 64>(device, grid, stream, maps, prm);
}

megacu_status run_product(megacu_driver_view const &driver, fp4_operands const &op,
                          void const *offsets, void const *counts, void const *alphas, void *out,
                          void *events, megacu_fp4_gemm_problem const *problem, bool swiglu) {
  if (problem == nullptr) return fail(MEGACU_INVALID_ARGUMENT, 2, "missing problem");
  megacu_fp4_gemm_problem const &p = *problem;
  if (p.m < 0 || p.n < 1 || p.k < 1 || p.experts < 0 || p.out_stride < 0) {
    return fail(MEGACU_INVALID_ARGUMENT, 1, "invalid problem");
  }
  if (!known_format(p.format)) return fail(MEGACU_INVALID_ARGUMENT, 1, "unknown format");
  if (!known_dtype(p.out_dtype)) {
    return fail(MEGACU_UNSUPPORTED, 20, "out_dtype must be f16, bf16 or f32");
  }
  if (p.k % 32 != 0) {
    return fail(MEGACU_INVALID_ARGUMENT, 21, "k must be a multiple of 32 (16-byte rows)");
  }
  if (p.out_stride != 0 && p.out_stride < p.n) {
    return fail(MEGACU_INVALID_ARGUMENT, 1, "out_stride is smaller than n");
  }
  if (p.m > kMaxDim || p.n > kMaxDim || p.k > kMaxDim || p.experts > kMaxExperts ||
      std::max(p.experts, 1) * p.n > kMaxDim) {
    return fail(MEGACU_UNSUPPORTED, 22, "dimension or number of experts too large");
  }
  if (p.experts > 0 && p.m / kFp4BlockM > 0xffff) {
    return fail(MEGACU_UNSUPPORTED, 22, "at most 65535 tiles of 128 rows by expert");
  }
  if (p.experts > 0 && p.m % kFp4BlockM != 0) {
    return fail(MEGACU_UNSUPPORTED, 22, "rows by expert come in tiles of 128");
  }
  fp4_plan plan;
  megacu_status const st = make_plan(p, swiglu, plan);
  if (st.code != MEGACU_OK) return st;
  bool const nv = p.format == MEGACU_FP4_NV;
  std::int64_t const tiles_k = scale_tiles(p.k, nv);
  std::int64_t const a_tiles = plan.m_tiles * tiles_k;
  std::int64_t const b_tiles =
      std::max(p.experts, 1) * ceil_div(p.n, kScaleTileRows) * tiles_k;
  if (a_tiles > 0x7fffffffll || b_tiles > 0x7fffffffll) {
    return fail(MEGACU_UNSUPPORTED, 22, "operand too large");
  }
  if (p.m == 0) return ok_status();
  void const *const needed[] = {op.a, op.a_scales, op.b, op.b_scales, out, events};
  for (void const *ptr : needed) {
    if (ptr == nullptr) return fail(MEGACU_INVALID_ARGUMENT, 2, "missing storage");
  }
  if ((swiglu && (op.b2 == nullptr || op.b2_scales == nullptr)) ||
      (p.experts > 0 && (offsets == nullptr || counts == nullptr))) {
    return fail(MEGACU_INVALID_ARGUMENT, 2, "missing storage");
  }
  void const *const operands[] = {op.a, op.a_scales, op.b, op.b_scales, op.b2, op.b2_scales, events};
  for (void const *ptr : operands) {
    if (!aligned_to(ptr, 16)) {
      return fail(MEGACU_INVALID_ARGUMENT, 21, "operands and events must be 16-byte aligned");
    }
  }
  if (!aligned_to(out, element_size(p.out_dtype)) || !aligned_to(offsets, 4) ||
      !aligned_to(counts, 4) || !aligned_to(alphas, 4)) {
    return fail(MEGACU_INVALID_ARGUMENT, 21, "out and indices must be aligned to their element");
  }
  if (driver.launch.stream == nullptr) return ok_status();
  int const device = driver.launch.device_ordinal;
  device_guard const guard(device);
  if (guard.status() != cudaSuccess) return cuda_fail(guard.status(), 10);
  int sms = 0;
  cudaError_t e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
  if (e != cudaSuccess) return cuda_fail(e, 10);

  std::int64_t const b_rows = std::max(p.experts, 1) * p.n;
  std::uint32_t const b_box = swiglu || plan.pair ? 128 : static_cast<std::uint32_t>(plan.tile_n);
  std::uint32_t const scale_box = kFp4BlockK / fp4_tile_cols(nv);
  fp4_maps maps;
  if (!encode_fp4_map(&maps.a, op.a, p.m, p.k, kFp4BlockM) ||
      !encode_fp4_map(&maps.a_small, op.a, p.m, p.k, kFp4SmallRows) ||
      !encode_fp4_map(&maps.b, op.b, b_rows, p.k, b_box) ||
      !encode_fp4_map(&maps.b2, swiglu ? op.b2 : op.b, b_rows, p.k, b_box) ||
      !encode_scale_map(&maps.a_scales, op.a_scales, a_tiles, scale_box) ||
      !encode_scale_map(&maps.b_scales, op.b_scales, b_tiles, scale_box) ||
      !encode_scale_map(&maps.b2_scales, swiglu ? op.b2_scales : op.b_scales, b_tiles,
                        scale_box)) {
    return fail(MEGACU_BACKEND_ERROR, 30, "cuTensorMapEncodeTiled failed");
  }
  fp4_gemm_params prm{};
  prm.n = static_cast<std::int32_t>(p.n);
  prm.k = static_cast<std::int32_t>(p.k);
  prm.m_tiles = static_cast<std::int32_t>(plan.m_tiles);
  prm.n_tiles = static_cast<std::int32_t>(plan.n_tiles);
  prm.n_row_tiles = static_cast<std::int32_t>(ceil_div(p.n, kScaleTileRows));
  prm.rows = static_cast<std::int32_t>(p.m);
  prm.group_m = 16;
  prm.experts = p.experts;
  prm.split = plan.split;
  prm.scale_tiles = static_cast<std::int32_t>(scale_tiles(p.k, nv));
  prm.out_dtype = p.out_dtype;
  prm.out_stride = p.out_stride != 0 ? p.out_stride : p.n;
  std::int64_t const row_bytes = prm.out_stride * element_size(p.out_dtype);
  prm.row_bytes = aligned_to(out, 32) && row_bytes % 32 == 0   ? 32
                  : aligned_to(out, 16) && row_bytes % 16 == 0 ? 16
                                                               : 0;
  prm.alpha = p.alpha;
  prm.alphas = static_cast<float const *>(alphas);
  prm.offsets = static_cast<std::int32_t const *>(offsets);
  prm.counts = static_cast<std::int32_t const *>(counts);
  prm.out = out;
  prm.events = static_cast<std::uint32_t *>(events);
  prm.timeout_ns = p.timeout_ns != 0 ? p.timeout_ns : 4000000000ull;
  // Persistent, one CTA per SM; a split's cluster computes one tile.
  std::int64_t const tiles = plan.m_tiles * plan.n_tiles;
  std::int64_t const pairs = (plan.m_tiles + 1) / 2 * plan.n_tiles;
  std::int64_t const grid = plan.pair        ? 2 * std::min<std::int64_t>(pairs, sms / 2)
                            : plan.split > 1 ? tiles * plan.split
                                             : std::min<std::int64_t>(tiles, sms);
  auto const stream = static_cast<cudaStream_t>(driver.launch.stream);
  e = nv ? launch_plan<true>(plan, swiglu, device, static_cast<int>(grid), stream, maps, prm)
         : launch_plan<false>(plan, swiglu, device, static_cast<int>(grid), stream, maps, prm);
  return e == cudaSuccess ? ok_status() : cuda_fail(e, 14);
}

}  // namespace

extern "C" megacu_status megacu_b200_fp4_sizes(megacu_fp4_matrix const *matrix,
                                               std::int64_t sizes[2]) {
  int log2_scale = 0;
  megacu_status const st = check_matrix(matrix, log2_scale);
  if (st.code != MEGACU_OK) return st;
  if (sizes == nullptr) return fail(MEGACU_INVALID_ARGUMENT, 2, "missing output");
  sizes[0] = matrix->rows * (matrix->cols / 2);
  sizes[1] = ceil_div(matrix->rows, kScaleTileRows) *
             scale_tiles(matrix->cols, matrix->format == MEGACU_FP4_NV) * kScaleTileBytes;
  return ok_status();
}

extern "C" megacu_status megacu_b200_fp4_events_bytes(std::int64_t *bytes) {
  if (bytes == nullptr) return fail(MEGACU_INVALID_ARGUMENT, 2, "missing output");
  *bytes = kControlBytes;
  return ok_status();
}

extern "C" megacu_status megacu_cuda_fp4_quantize(megacu_driver_view driver, void const *x,
                                                  void const *slot_of_row, void *data,
                                                  void *scales,
                                                  megacu_fp4_matrix const *matrix) {
  int log2_scale = 0;
  megacu_status const st = check_matrix(matrix, log2_scale);
  if (st.code != MEGACU_OK) return st;
  megacu_fp4_matrix const &m = *matrix;
  bool const transpose = m.transpose != 0;
  if (m.stride != 0 && m.stride < (transpose ? m.rows : m.cols)) {
    return fail(MEGACU_INVALID_ARGUMENT, 1, "stride is smaller than a row");
  }
  if (transpose && (slot_of_row != nullptr || m.topk > 0)) {
    return fail(MEGACU_UNSUPPORTED, 22, "a transposed matrix is quantised whole");
  }
  if (m.scatter != 0 && m.topk == 0) {
    return fail(MEGACU_INVALID_ARGUMENT, 1, "scattered rows need topk");
  }
  if (m.topk > 0 && slot_of_row == nullptr) {
    return fail(MEGACU_INVALID_ARGUMENT, 2, "gathered rows need slot_of_row");
  }
  if (m.topk > 0 && m.rows > 0 && m.x_rows == 0) {
    return fail(MEGACU_INVALID_ARGUMENT, 1, "gathered rows need x_rows");
  }
  if (m.rows == 0) return ok_status();
  if (x == nullptr || data == nullptr || scales == nullptr) {
    return fail(MEGACU_INVALID_ARGUMENT, 2, "missing storage");
  }
  int const size = element_size(m.dtype);
  if (!aligned_to(data, 16) || !aligned_to(scales, 16) || !aligned_to(x, size) ||
      !aligned_to(slot_of_row, 4)) {
    return fail(MEGACU_INVALID_ARGUMENT, 21,
                "data and scales must be 16-byte aligned, x to its element");
  }
  fp4_matrix_params prm = matrix_params(m, log2_scale, data, scales, transpose);
  prm.slot_of_row = static_cast<std::int32_t const *>(slot_of_row);
  static_assert(kScaleTileRows == 2 * kQuantRows && kQuantRows == kQuantTRows, "two CTAs deep");
  bool const masked = slot_of_row != nullptr && m.scatter == 0;
  if (masked) prm.col_tiles = (prm.col_tiles + kMaskedSpan - 1) / kMaskedSpan;
  std::int64_t const row_ctas = m.scatter != 0 ? ceil_div(m.x_rows, kScatterRows)
                                               : 2 * ceil_div(m.rows, kScaleTileRows);
  if (row_ctas * prm.col_tiles > 0x7fffffffll) {
    return fail(MEGACU_UNSUPPORTED, 22, "dimension too large");
  }
  if (driver.launch.stream == nullptr) return ok_status();
  device_guard const guard(driver.launch.device_ordinal);
  if (guard.status() != cudaSuccess) return cuda_fail(guard.status(), 10);
  auto const grid = static_cast<unsigned>(row_ctas * prm.col_tiles);
  auto const stream = static_cast<cudaStream_t>(driver.launch.stream);
  cudaError_t e = cudaSuccess;
  auto launch = [&](auto kernel, auto const *src) {
    e = launch_chained(kernel, grid, kQuantThreads, 0, stream, 1, prm, src);
  };
  by_type(m.dtype, m.format, [&](auto value, auto nv) {
    using T = decltype(value);
    auto const *src = static_cast<T const *>(x);
    constexpr bool kNv = decltype(nv)::value;
    if (transpose) {
      // Pairs of columns are read together when every row starts on a pair.
      if (m.rows % 2 == 0 && prm.stride % 2 == 0 && aligned_to(x, 2 * size)) {
        launch(fp4_quantize_t_kernel<T, kNv, true>, src);
      } else {
        launch(fp4_quantize_t_kernel<T, kNv, false>, src);
      }
    } else if (m.scatter != 0) {
      prm.stride * size % 32 == 0 && aligned_to(x, 32)
          ? launch(fp4_quantize_scatter_kernel<T, kNv, true>, src)
          : launch(fp4_quantize_scatter_kernel<T, kNv, false>, src);
    } else if (prm.stride * size % 32 == 0 && aligned_to(x, 32)) {
      masked ? launch(fp4_quantize_kernel<T, kNv, true, true>, src)
             : launch(fp4_quantize_kernel<T, kNv, true, false>, src);
    } else {
      masked ? launch(fp4_quantize_kernel<T, kNv, false, true>, src)
             : launch(fp4_quantize_kernel<T, kNv, false, false>, src);
    }
  });
  return e == cudaSuccess ? ok_status() : cuda_fail(e, 14);
}

extern "C" megacu_status megacu_cuda_fp4_dequantize(megacu_driver_view driver, void const *data,
                                                    void const *scales, void *out,
                                                    megacu_fp4_matrix const *matrix) {
  int log2_scale = 0;
  megacu_status const st = check_matrix(matrix, log2_scale);
  if (st.code != MEGACU_OK) return st;
  megacu_fp4_matrix const &m = *matrix;
  if (m.transpose != 0 || m.topk != 0 || m.scatter != 0) {
    return fail(MEGACU_UNSUPPORTED, 22, "values come back row by row as quantised");
  }
  if (m.stride != 0 && m.stride < m.cols) {
    return fail(MEGACU_INVALID_ARGUMENT, 1, "stride is smaller than a row");
  }
  if (m.rows == 0) return ok_status();
  if (data == nullptr || scales == nullptr || out == nullptr) {
    return fail(MEGACU_INVALID_ARGUMENT, 2, "missing storage");
  }
  int const size = element_size(m.dtype);
  if (!aligned_to(data, 16) || !aligned_to(scales, 16) || !aligned_to(out, size)) {
    return fail(MEGACU_INVALID_ARGUMENT, 21,
                "data and scales must be 16-byte aligned, out to its element");
  }
  if (driver.launch.stream == nullptr) return ok_status();
  device_guard const guard(driver.launch.device_ordinal);
  if (guard.status() != cudaSuccess) return cuda_fail(guard.status(), 10);
  fp4_matrix_params const prm =
      matrix_params(m, log2_scale, const_cast<void *>(data), const_cast<void *>(scales), false);
  auto const grid = static_cast<unsigned>(ceil_div(m.rows, kQuantRows) * prm.col_tiles);
  auto const stream = static_cast<cudaStream_t>(driver.launch.stream);
  bool const vec = prm.stride * size % 32 == 0 && aligned_to(out, 32);
  cudaError_t e = cudaSuccess;
  by_type(m.dtype, m.format, [&](auto value, auto nv) {
    using T = decltype(value);
    constexpr bool kNv = decltype(nv)::value;
    auto *const dst = static_cast<T *>(out);
    e = vec ? launch_chained(fp4_dequantize_kernel<T, kNv, true>, grid, kQuantThreads, 0, stream,
                             1, prm, dst)
            : launch_chained(fp4_dequantize_kernel<T, kNv, false>, grid, kQuantThreads, 0, stream,
                             1, prm, dst);
  });
  return e == cudaSuccess ? ok_status() : cuda_fail(e, 14);
}

extern "C" megacu_status megacu_cuda_fp4_gemm(megacu_driver_view driver, void const *a,
                                              void const *a_scales, void const *b,
                                              void const *b_scales, void const *offsets,
                                              void const *counts, void const *alphas, void *out,
                                              void *events,
                                              megacu_fp4_gemm_problem const *problem) {
  return run_product(driver, {a, a_scales, b, b_scales, nullptr, nullptr}, offsets, counts, alphas,
                     out, events, problem, false);
}

extern "C" megacu_status megacu_cuda_fp4_gemm_swiglu(
    megacu_driver_view driver, void const *a, void const *a_scales, void const *gate,
    void const *gate_scales, void const *up, void const *up_scales, void const *offsets,
    void const *counts, void const *alphas, void *act, void *events,
    megacu_fp4_gemm_problem const *problem) {
  return run_product(driver, {a, a_scales, gate, gate_scales, up, up_scales}, offsets, counts,
                     alphas, act, events, problem, true);
}
