// Routing of tokens to experts and back (mixture of experts; no counterpart
// in megacu): entry points of the kernels in kernels/moe_kernels.cuh.
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstdint>

#include <megacu_b200.h>

#include "kernels/moe_kernels.cuh"
#include "status.h"

namespace {

using namespace megacu_b200;

constexpr std::int64_t kMaxSlots = 1ll << 30;
// Of the sort, whose second launch reads every chunk's histogram in each CTA.
// With 256 experts 2^24 slots take 0.55 ms and 2^26 6.8, with 1024 experts 2.1
// and 31; 2^30 would hold the GPU for seconds.
constexpr std::int64_t kMaxSortSlots = 1ll << 26;
constexpr std::int32_t kMaxAlign = 1024;
constexpr int kMaxDevices = 64;

// One CTA sorts up to this many slots in one launch; more are sorted in
// chunks, counted by one launch and placed by a second.
constexpr std::int64_t kSingleCtaSlots = 8192;
constexpr std::int64_t kMinChunk = 4096;
constexpr std::int64_t kChunks = 64;  // CTAs wanted; each reads every chunk's histogram
static_assert(kSingleCtaSlots <= kMoeMaxChunk, "a chunk's local experts are kept on chip");

std::int32_t chunk_of(std::int64_t slots) {
  if (slots <= kSingleCtaSlots) return static_cast<std::int32_t>(std::max<std::int64_t>(slots, 1));
  std::int64_t const even = (slots + kChunks - 1) / kChunks;
  std::int64_t const chunk = std::clamp<std::int64_t>(even, kMinChunk, kMoeMaxChunk);
  return static_cast<std::int32_t>((chunk + kMoeSortThreads - 1) / kMoeSortThreads *
                                   kMoeSortThreads);
}

std::int64_t chunks_of(std::int64_t slots) {
  std::int64_t const chunk = chunk_of(slots);
  return std::max<std::int64_t>((slots + chunk - 1) / chunk, 1);
}

std::int64_t capacity(megacu_moe_problem const &p) {
  std::int64_t const slots = p.tokens * p.topk;
  std::int64_t const most = slots + std::min<std::int64_t>(p.experts, slots) * (p.align - 1);
  return most / p.align * p.align;
}

megacu_status check_problem(megacu_moe_problem const *p) {
  if (p == nullptr) return fail(MEGACU_INVALID_ARGUMENT, 2, "missing problem");
  if (p->tokens < 0 || p->topk < 1 || p->experts < 1 || p->align < 1 || p->hidden < 0) {
    return fail(MEGACU_INVALID_ARGUMENT, 1, "invalid problem");
  }
  if (p->topk > kMoeMaxTopk || p->experts > kMoeMaxExperts || p->align > kMaxAlign ||
      p->tokens > kMaxSlots || p->tokens * p->topk > kMaxSlots) {
    return fail(MEGACU_UNSUPPORTED, 22,
                "at most 32 choices, 1024 experts, an alignment of 1024 and 2^30 slots");
  }
  static_assert(kMaxSlots + static_cast<std::int64_t>(kMoeMaxExperts) * kMaxAlign < 1ll << 31,
                "rows are 32-bit");
  return ok_status();
}

int element_size(std::int32_t dtype) {
  return dtype == MEGACU_DTYPE_F32 ? 4 : dtype == MEGACU_DTYPE_F16 || dtype == MEGACU_DTYPE_BF16 ? 2 : 0;
}

// Problem and buffers of the calls that move rows.
megacu_status check_rows(megacu_moe_problem const *p, void const *const *buffers, int n) {
  megacu_status st = check_problem(p);
  if (st.code != MEGACU_OK) return st;
  int const size = element_size(p->dtype);
  if (size == 0) return fail(MEGACU_UNSUPPORTED, 20, "rows are f16, bf16 or f32");
  if (p->hidden < 1 || p->hidden > (1 << 30)) {
    return fail(MEGACU_INVALID_ARGUMENT, 1, "hidden must be 1..2^30");
  }
  if ((p->token_stride != 0 && p->token_stride < p->hidden) ||
      (p->row_stride != 0 && p->row_stride < p->hidden)) {
    return fail(MEGACU_INVALID_ARGUMENT, 1, "a stride is smaller than hidden");
  }
  if (p->tokens == 0) return ok_status();
  for (int i = 0; i < n; ++i) {
    if (buffers[i] == nullptr) return fail(MEGACU_INVALID_ARGUMENT, 2, "missing storage");
    if (!aligned_to(buffers[i], size)) {
      return fail(MEGACU_INVALID_ARGUMENT, 21, "rows must be aligned to their element");
    }
  }
  return ok_status();
}

template <class Id>
cudaError_t launch_sort(moe_sort_params const &prm, std::int64_t chunks, int device,
                        cudaStream_t stream) {
  static std::atomic<bool> configured[kMaxDevices] = {};
  bool const known = device >= 0 && device < kMaxDevices;
  // A thread per slot and per expert, as far as they go.
  std::int64_t const wanted = std::max<std::int64_t>(prm.chunk, prm.experts);
  int const threads =
      static_cast<int>(std::min<std::int64_t>((wanted + 31) / 32 * 32, kMoeSortThreads));
  if (!known || !configured[device].load(std::memory_order_acquire)) {
    cudaError_t const e =
        cudaFuncSetAttribute(moe_place_kernel<Id>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             moe_place_smem(kMoeSortThreads / 32, kMoeMaxExperts, kMoeMaxChunk));
    if (e != cudaSuccess) return e;
    if (known) configured[device].store(true, std::memory_order_release);
  }
  auto const grid = static_cast<unsigned>(chunks);
  if (chunks > 1) {
    cudaError_t const e = launch_chained(moe_count_kernel<Id>, grid, threads,
                                         static_cast<std::size_t>(prm.experts) * 4, stream, 1, prm);
    if (e != cudaSuccess) return e;
  }
  return launch_chained(moe_place_kernel<Id>, grid, threads,
                        static_cast<std::size_t>(
                            moe_place_smem(threads / 32, prm.experts, prm.chunk)),
                        stream, 1, prm);
}

enum class rows_op { dispatch, combine, grad };

struct rows_buffers {
  void const *in = nullptr;    // x (dispatch), rows (combine), dy (grad)
  void const *rows = nullptr;  // grad: the forward's rows
  float const *weights = nullptr;
  void *out = nullptr;         // rows, y, drows
  float *dweights = nullptr;
};

template <class T, int N>
cudaError_t launch_rows(rows_op op, moe_rows_params const &prm, rows_buffers const &b,
                 cudaStream_t stream) {
  auto const grid = static_cast<unsigned>(prm.tokens);
  int const most = op == rows_op::dispatch  ? kDispatchThreads
                   : op == rows_op::combine ? kCombineThreads
                                            : kGradThreads;
  int const threads = std::min(most, ((prm.hidden + N - 1) / N + 31) / 32 * 32);
  auto const *const in = static_cast<T const *>(b.in);
  auto *const out = static_cast<T *>(b.out);
  switch (op) {
    case rows_op::dispatch:
      return launch_chained(moe_dispatch_kernel<T, N>, grid, threads, 0, stream, 1, prm, in, out);
    case rows_op::combine:
      return launch_chained(moe_combine_kernel<T, N>, grid, threads, 0, stream, 1, prm, in,
                            b.weights, out);
    default:
      return launch_chained(moe_combine_grad_kernel<T, N>, grid, threads, 0, stream, 1, prm, in,
                            static_cast<T const *>(b.rows), b.weights, out, b.dweights);
  }
}

// The widest access, up to 32 bytes for the dispatch and 16 for the calls
// that hold several rows, that every row's start and length allow.
template <class T>
cudaError_t launch_rows_typed(rows_op op, moe_rows_params const &prm, rows_buffers const &b, int bytes,
                       cudaStream_t stream) {
  if (bytes == 32 && op == rows_op::dispatch) {
    int const vectors = static_cast<int>(prm.hidden * sizeof(T) / 32);
    return launch_chained(moe_dispatch_kernel<T, 32 / sizeof(T)>,
                          static_cast<unsigned>(prm.tokens),
                          std::min(kDispatchThreads, (vectors + 31) / 32 * 32), 0, stream, 1, prm,
                          static_cast<T const *>(b.in), static_cast<T *>(b.out));
  }
  if (bytes >= 16) return launch_rows<T, 16 / sizeof(T)>(op, prm, b, stream);
  return launch_rows<T, 1>(op, prm, b, stream);
}

megacu_status run_rows(rows_op op, megacu_driver_view const &driver, rows_buffers const &b,
                       std::int32_t const *row_of_slot, megacu_moe_problem const *p) {
  void const *const buffers[] = {b.in, b.out, op == rows_op::grad ? b.rows : b.in};
  megacu_status const st = check_rows(p, buffers, 3);
  if (st.code != MEGACU_OK) return st;
  if (p->tokens > 0) {
    if (row_of_slot == nullptr ||
        (op == rows_op::grad && (b.weights == nullptr || b.dweights == nullptr))) {
      return fail(MEGACU_INVALID_ARGUMENT, 2, "missing storage");
    }
    if (!aligned_to(row_of_slot, 4) || !aligned_to(b.weights, 4) || !aligned_to(b.dweights, 4)) {
      return fail(MEGACU_INVALID_ARGUMENT, 21, "indices and weights must be 4-byte aligned");
    }
  }
  if (driver.launch.stream == nullptr || p->tokens == 0) return ok_status();
  device_guard const guard(driver.launch.device_ordinal);
  if (guard.status() != cudaSuccess) return cuda_fail(guard.status(), 10);
  moe_rows_params prm{};
  prm.tokens = p->tokens;
  prm.hidden = static_cast<std::int32_t>(p->hidden);
  prm.topk = p->topk;
  prm.token_stride = p->token_stride != 0 ? p->token_stride : p->hidden;
  prm.row_stride = p->row_stride != 0 ? p->row_stride : p->hidden;
  prm.row_of_slot = row_of_slot;
  prm.rows = static_cast<std::uint32_t>(capacity(*p));
  int const size = element_size(p->dtype);
  auto fits = [&](int n) {
    return p->hidden * size % n == 0 && prm.token_stride * size % n == 0 &&
           prm.row_stride * size % n == 0 && aligned_to(buffers[0], n) &&
           aligned_to(buffers[1], n) && aligned_to(buffers[2], n);
  };
  int const vec = fits(32) ? 32 : fits(16) ? 16 : 0;
  auto const stream = static_cast<cudaStream_t>(driver.launch.stream);
  cudaError_t const e =
      p->dtype == MEGACU_DTYPE_F16    ? launch_rows_typed<__half>(op, prm, b, vec, stream)
      : p->dtype == MEGACU_DTYPE_BF16 ? launch_rows_typed<__nv_bfloat16>(op, prm, b, vec, stream)
                                      : launch_rows_typed<float>(op, prm, b, vec, stream);
  return e == cudaSuccess ? ok_status() : cuda_fail(e, 14);
}

}  // namespace

extern "C" megacu_status megacu_b200_moe_sizes(megacu_moe_problem const *problem,
                                               std::int64_t sizes[2]) {
  megacu_status const st = check_problem(problem);
  if (st.code != MEGACU_OK) return st;
  if (sizes == nullptr) return fail(MEGACU_INVALID_ARGUMENT, 2, "missing output");
  std::int64_t const chunks = chunks_of(problem->tokens * problem->topk);
  sizes[0] = capacity(*problem);
  sizes[1] = chunks > 1 ? (chunks + 7) / 8 * 16 * problem->experts : 0;
  return ok_status();
}

extern "C" megacu_status megacu_cuda_moe_sort(megacu_driver_view driver, void const *expert_ids,
                                              void *counts, void *offsets, void *row_of_slot,
                                              void *slot_of_row, void *workspace,
                                              megacu_moe_problem const *problem) {
  megacu_status const st = check_problem(problem);
  if (st.code != MEGACU_OK) return st;
  megacu_moe_problem const &p = *problem;
  if (p.id_bytes != 0 && p.id_bytes != 4 && p.id_bytes != 8) {
    return fail(MEGACU_UNSUPPORTED, 20, "expert ids are 32 or 64 bits");
  }
  std::int64_t const slots = p.tokens * p.topk;
  if (slots > kMaxSortSlots) return fail(MEGACU_UNSUPPORTED, 22, "a sort of at most 2^26 slots");
  std::int64_t const chunks = chunks_of(slots);
  if (counts == nullptr || offsets == nullptr ||
      (slots > 0 && (expert_ids == nullptr || row_of_slot == nullptr || slot_of_row == nullptr)) ||
      (chunks > 1 && workspace == nullptr)) {
    return fail(MEGACU_INVALID_ARGUMENT, 2, "missing storage");
  }
  if (!aligned_to(expert_ids, p.id_bytes == 8 ? 8 : 4) || !aligned_to(counts, 4) ||
      !aligned_to(offsets, 4) || !aligned_to(row_of_slot, 4) || !aligned_to(slot_of_row, 4) ||
      !aligned_to(workspace, 16)) {
    return fail(MEGACU_INVALID_ARGUMENT, 21, "indices must be aligned to their element, the workspace to 16 bytes");
  }
  if (driver.launch.stream == nullptr) return ok_status();
  int const device = driver.launch.device_ordinal;
  device_guard const guard(device);
  if (guard.status() != cudaSuccess) return cuda_fail(guard.status(), 10);
  moe_sort_params prm{};
  prm.ids = expert_ids;
  prm.slots = slots;
  prm.rows = capacity(p);
  prm.chunk = chunk_of(slots);
  prm.experts = p.experts;
  prm.first = p.first_expert;
  prm.align = p.align;
  prm.histogram = static_cast<std::uint16_t *>(workspace);
  prm.chunks_pad = static_cast<std::int32_t>((chunks + 7) / 8 * 8);
  prm.counts = static_cast<std::int32_t *>(counts);
  prm.offsets = static_cast<std::int32_t *>(offsets);
  prm.row_of_slot = static_cast<std::int32_t *>(row_of_slot);
  prm.slot_of_row = static_cast<std::int32_t *>(slot_of_row);
  auto const stream = static_cast<cudaStream_t>(driver.launch.stream);
  cudaError_t const e = p.id_bytes == 8 ? launch_sort<std::int64_t>(prm, chunks, device, stream)
                                        : launch_sort<std::int32_t>(prm, chunks, device, stream);
  return e == cudaSuccess ? ok_status() : cuda_fail(e, 14);
}

extern "C" megacu_status megacu_cuda_moe_dispatch(megacu_driver_view driver, void const *x,
                                                  void const *row_of_slot, void *rows,
                                                  megacu_moe_problem const *problem) {
  rows_buffers b;
  b.in = x;
  b.out = rows;
  return run_rows(rows_op::dispatch, driver, b, static_cast<std::int32_t const *>(row_of_slot),
                  problem);
}

extern "C" megacu_status megacu_cuda_moe_combine(megacu_driver_view driver, void const *rows,
                                                 void const *weights, void const *row_of_slot,
                                                 void *y, megacu_moe_problem const *problem) {
  rows_buffers b;
  b.in = rows;
  b.weights = static_cast<float const *>(weights);
  b.out = y;
  return run_rows(rows_op::combine, driver, b, static_cast<std::int32_t const *>(row_of_slot),
                  problem);
}

extern "C" megacu_status megacu_cuda_moe_combine_grad(megacu_driver_view driver, void const *dy,
                                                      void const *rows, void const *weights,
                                                      void const *row_of_slot, void *drows,
                                                      void *dweights,
                                                      megacu_moe_problem const *problem) {
  rows_buffers b;
  b.in = dy;
  b.rows = rows;
  b.weights = static_cast<float const *>(weights);
  b.out = drows;
  b.dweights = static_cast<float *>(dweights);
  return run_rows(rows_op::grad, driver, b, static_cast<std::int32_t const *>(row_of_slot),
                  problem);
}
