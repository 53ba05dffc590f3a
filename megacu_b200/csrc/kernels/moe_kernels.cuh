// Routing of tokens to experts: a stable counting sort of the (token, choice)
// slots by expert, and the rows' way to the experts and back.
//
//   sort      row_of_slot[s] = offsets[e(s)] + #{s' < s : e(s') = e(s)}
//   dispatch  rows[row_of_slot[t, j]] = x[t]
//   combine   y[t] = sum_j w[t, j] rows[row_of_slot[t, j]]
//   gradient  drows[row_of_slot[t, j]] = w[t, j] dy[t],
//             dw[t, j] = <dy[t], rows[row_of_slot[t, j]]>
// The gradient of dispatch is combine without weights.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "chained.cuh"
#include "vec.cuh"

namespace megacu_b200 {

inline constexpr int kMoeMaxExperts = 1024;
inline constexpr int kMoeMaxTopk = 32;
inline constexpr int kMoeSortThreads = 1024;  // at most; fewer for few slots
inline constexpr int kMoeMaxChunk = 8192;     // slots per CTA

struct moe_sort_params {
  void const *ids;
  std::int64_t slots;
  std::int64_t rows;       // capacity of slot_of_row
  std::int32_t chunk;      // slots per CTA
  std::int32_t experts;
  std::int32_t first;
  std::int32_t align;
  std::uint16_t *histogram;  // [experts][chunks_pad], unused with one CTA
  std::int32_t chunks_pad;   // CTAs rounded up to 8 (16 bytes of counts)
  std::int32_t *counts;
  std::int32_t *offsets;
  std::int32_t *row_of_slot;
  std::int32_t *slot_of_row;
};

// The slot's expert here, or -1.
template <class Id>
__device__ __forceinline__ std::int32_t local_expert(moe_sort_params const &p, std::int64_t slot) {
  std::int64_t const e = static_cast<std::int64_t>(static_cast<Id const *>(p.ids)[slot]) - p.first;
  return e >= 0 && e < p.experts ? static_cast<std::int32_t>(e) : -1;
}

// Every entry of slot_of_row to -1; the slots overwrite theirs later.
__device__ __forceinline__ void clear_rows(moe_sort_params const &p) {
  for (std::int64_t r = static_cast<std::int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
       r < p.rows; r += static_cast<std::int64_t>(gridDim.x) * blockDim.x) {
    p.slot_of_row[r] = -1;
  }
}

// Histogram of one chunk of slots per CTA. Counts are at most a chunk's 8192
// slots and lie expert by expert, so that the second launch reads an expert's
// counts of eight chunks at a time.
template <class Id>
__global__ void __launch_bounds__(kMoeSortThreads) moe_count_kernel(moe_sort_params p) {
  extern __shared__ std::int32_t moe_smem[];
  for (int e = threadIdx.x; e < p.experts; e += blockDim.x) moe_smem[e] = 0;
  grid_wait();
  grid_start_next();
  __syncthreads();
  std::int64_t const begin = static_cast<std::int64_t>(blockIdx.x) * p.chunk;
  std::int64_t const end = min(begin + p.chunk, p.slots);
  for (std::int64_t s = begin + threadIdx.x; s < end; s += blockDim.x) {
    std::int32_t const e = local_expert<Id>(p, s);
    if (e >= 0) atomicAdd(&moe_smem[e], 1);
  }
  clear_rows(p);
  __syncthreads();
  for (int e = threadIdx.x; e < p.experts; e += blockDim.x) {
    p.histogram[static_cast<std::int64_t>(e) * p.chunks_pad + blockIdx.x] =
        static_cast<std::uint16_t>(moe_smem[e]);
  }
}

// Lanes of a warp with the same key of `bits` bits (a ballot per bit; a warp
// match took 0.7 to 1.3 us here against 0.1).
__device__ __forceinline__ std::uint32_t same_key(std::int32_t key, int bits) {
  std::uint32_t same = 0xffffffffu;
  for (int b = 0; b < bits; ++b) {
    std::uint32_t const set = __ballot_sync(0xffffffffu, key >> b & 1);
    same &= key >> b & 1 ? set : ~set;
  }
  return same;
}

// Places one chunk of slots per CTA. Every warp owns a contiguous part of the
// chunk, so that the order within an expert is the slots' order: the warp's
// first row of each expert is the expert's start, plus what earlier chunks
// and earlier warps hold of it; within 32 slots, lanes of one expert rank
// themselves by ballots. No counter is kept between calls and nothing depends
// on the order of atomics (they add whole numbers). Bound by the latency of a
// handful of dependent steps, so the ids are read once and kept as 16-bit
// local experts.
//
// Shared memory: cursor [warps][experts], total [experts], start [experts],
// then the chunk's local experts (int16).
__host__ __device__ inline int moe_place_smem(int warps, int experts, int chunk) {
  return (warps + 2) * experts * 4 + chunk * 2;
}

template <class Id>
__global__ void __launch_bounds__(kMoeSortThreads) moe_place_kernel(moe_sort_params p) {
  extern __shared__ std::int32_t moe_smem[];
  __shared__ std::int32_t warp_sums[32];
  int const experts = p.experts, threads = blockDim.x, warps = threads / 32;
  std::int32_t *const cursor = moe_smem;
  std::int32_t *const total = moe_smem + warps * experts;
  std::int32_t *const start = total + experts;
  auto *const local = reinterpret_cast<std::int16_t *>(start + experts);
  int const tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  bool const chunked = gridDim.x > 1;

  std::int64_t const begin = static_cast<std::int64_t>(blockIdx.x) * p.chunk;
  std::int32_t const here = static_cast<std::int32_t>(min(p.chunk + begin, p.slots) - begin);
  std::int32_t const part = (p.chunk + threads - 1) / threads * 32;
  std::int32_t const w0 = min(warp * part, here), w1 = min(w0 + part, here);
  std::int32_t *const mine = cursor + warp * experts;
  for (int e = lane; e < experts; e += 32) mine[e] = 0;
  if (chunked) {
    for (int e = tid; e < 2 * experts; e += threads) total[e] = 0;
  }
  // Also for the ids, which the first launch has read: that it has started
  // this one does not make them visible here, its end does.
  grid_wait();
  if (!chunked) clear_rows(p);  // the first launch did it for several chunks
  __syncwarp();
  for (std::int32_t s = w0 + lane; s < w1; s += 32) {
    std::int32_t const e = local_expert<Id>(p, begin + s);
    local[s] = static_cast<std::int16_t>(e);
    if (e >= 0) atomicAdd(&mine[e], 1);
  }
  // Not earlier: a product two launches on would start its CTAs while this one
  // still holds its SM, and its last CTA would wait for it (a routed block of 64
  // tokens 97 -> 102 us).
  grid_start_next();
  __syncthreads();

  // total[e] = slots of e anywhere, start[e] = slots of e in earlier chunks.
  if (chunked) {
    int const groups = p.chunks_pad / 8, last = static_cast<int>(gridDim.x);
    int const lanes = threads / experts;  // threads that share an expert's counts
    if (tid < lanes * experts) {
      int const e = tid / lanes;
      auto const *const counts =
          reinterpret_cast<uint4 const *>(p.histogram + static_cast<std::int64_t>(e) * p.chunks_pad);
      std::int32_t all = 0, before = 0;
#pragma unroll 4
      for (int g = tid % lanes; g < groups; g += lanes) {
        uint4 const v = counts[g];
        std::uint32_t const w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          int const c = g * 8 + i;
          std::int32_t const n = static_cast<std::int32_t>(w[i / 2] >> (16 * (i % 2)) & 0xffffu);
          all += c < last ? n : 0;  // past the last chunk nothing was written
          before += c < static_cast<int>(blockIdx.x) ? n : 0;
        }
      }
      if (all) atomicAdd(&total[e], all);
      if (before) atomicAdd(&start[e], before);
    }
    __syncthreads();
  }

  // One thread per expert: its rows of each warp, and an exclusive scan of the
  // padded counts.
  std::int32_t count = 0, before = 0;
  if (tid < experts) {
    std::int32_t sum = 0;
#pragma unroll 16
    for (int w = 0; w < warps; ++w) {
      std::int32_t const n = cursor[w * experts + tid];
      cursor[w * experts + tid] = sum;
      sum += n;
    }
    count = chunked ? total[tid] : sum;
    before = chunked ? start[tid] : 0;
  }
  std::int32_t const padded = (count + p.align - 1) / p.align * p.align;
  std::int32_t sum = padded;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    std::int32_t const up = __shfl_up_sync(0xffffffffu, sum, d);
    if (lane >= d) sum += up;
  }
  if (lane == 31) warp_sums[warp] = sum;
  __syncthreads();
  // Every warp scans the warps' sums (no second barrier).
  std::int32_t all_sums = lane < warps ? warp_sums[lane] : 0;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    std::int32_t const up = __shfl_up_sync(0xffffffffu, all_sums, d);
    if (lane >= d) all_sums += up;
  }
  std::int32_t const used = __shfl_sync(0xffffffffu, all_sums, 31);
  std::int32_t const earlier = __shfl_sync(0xffffffffu, all_sums, warp > 0 ? warp - 1 : 0);
  std::int32_t const offset = sum - padded + (warp > 0 ? earlier : 0);
  if (tid < experts) {
    start[tid] = offset + before;  // first row of this chunk's slots
    if (blockIdx.x == 0) {
      p.counts[tid] = count;
      p.offsets[tid] = offset;
      if (tid == experts - 1) p.offsets[experts] = used;
    }
  }
  __syncthreads();
  int const bits = 32 - __clz(experts);  // of e + 1, 0 = not here
  for (std::int32_t s0 = w0; s0 < w1; s0 += 32) {
    std::int32_t const s = s0 + lane;
    std::int32_t const e = s < w1 ? local[s] : -1;
    std::uint32_t const same = same_key(e + 1, bits);
    std::int32_t row = -1;
    if (e >= 0) row = start[e] + mine[e] + __popc(same & ((1u << lane) - 1u));
    __syncwarp();
    if (e >= 0 && lane == __ffs(same) - 1) mine[e] += __popc(same);
    __syncwarp();
    if (s < w1) p.row_of_slot[begin + s] = row;
    if (row >= 0) p.slot_of_row[row] = static_cast<std::int32_t>(begin + s);
  }
}

struct moe_rows_params {
  std::int64_t tokens;
  std::int32_t hidden;
  std::int32_t topk;
  std::int64_t token_stride;  // elements between rows of x, y and dy
  std::int64_t row_stride;    // elements between rows of rows and drows
  std::int32_t const *row_of_slot;
  std::uint32_t rows;  // capacity of the sorted order: an entry at or past it has no row
};

// The entry's row, or -1.
__device__ __forceinline__ std::int32_t row_at(moe_rows_params const &p, std::int32_t entry) {
  return static_cast<std::uint32_t>(entry) < p.rows ? entry : -1;
}

// Choices whose rows are in flight together in a thread, measured at 8192 tokens
// x 8 choices x 4096 bf16 with 256 threads: the combine takes 99 us with 2, 95
// with 4 and 119 with 8 (fewer CTAs fit an SM). The gradient, which also
// stores, takes 180 us with 8 and 128 threads, 188 with 4 and 256, 191 with 8
// and 256.
inline constexpr int kCombineGroup = 4, kCombineThreads = 256;
inline constexpr int kGradGroup = 8, kGradThreads = 128;
inline constexpr int kDispatchThreads = 256;

// One CTA per token reads its row once and writes it once per choice, 32 bytes
// per lane (94 us at the sizes above, 6.4 TB/s; 99 with 16).
template <class T, int N>
__global__ void moe_dispatch_kernel(moe_rows_params p, T const *x, T *rows) {
  grid_start_next();
  grid_wait();
  std::int64_t const t = blockIdx.x;
  std::int32_t const *const at = p.row_of_slot + t * p.topk;
  T const *const src = x + t * p.token_stride;
  for (int c = threadIdx.x * N; c < p.hidden; c += blockDim.x * N) {
    vec<T, N> const v = load_vec<T, N>(src + c);
    for (int j = 0; j < p.topk; ++j) {
      std::int32_t const r = row_at(p, at[j]);
      if (r >= 0) store_vec<T, N>(rows + r * p.row_stride + c, v);
    }
  }
}

// One CTA per token; sums in 32 bits in the order of the choices, one
// rounding. 95 us at the sizes above, 6.3 TB/s.
template <class T, int N>
__global__ void moe_combine_kernel(moe_rows_params p, T const *rows, float const *weights, T *y) {
  grid_start_next();
  grid_wait();
  std::int64_t const t = blockIdx.x;
  std::int32_t const *const at = p.row_of_slot + t * p.topk;
  float const *const w = weights == nullptr ? nullptr : weights + t * p.topk;
  for (int c = threadIdx.x * N; c < p.hidden; c += blockDim.x * N) {
    float acc[N] = {};
    for (int j0 = 0; j0 < p.topk; j0 += kCombineGroup) {
      vec<T, N> v[kCombineGroup];
      std::int32_t r[kCombineGroup];
#pragma unroll
      for (int j = 0; j < kCombineGroup; ++j) {
        r[j] = j0 + j < p.topk ? row_at(p, at[j0 + j]) : -1;
        if (r[j] >= 0) v[j] = load_vec<T, N>(rows + r[j] * p.row_stride + c);
      }
#pragma unroll
      for (int j = 0; j < kCombineGroup; ++j) {
        if (r[j] < 0) continue;
        float const f = w == nullptr ? 1.0f : w[j0 + j];
#pragma unroll
        for (int i = 0; i < N; ++i) acc[i] = fmaf(f, v[j].f32(i), acc[i]);
      }
    }
    vec<T, N> out;
#pragma unroll
    for (int i = 0; i < N; ++i) out.v[i] = from_f32<T>(acc[i]);
    store_vec<T, N>(y + t * p.token_stride + c, out);
  }
}

// One CTA per token: dy is read once per kGradGroup choices, each choice's row
// once; the dot products are summed in 32 bits per thread, then over the warp,
// then over the warps in order. 180 us at the sizes above, 6.3 TB/s.
template <class T, int N>
__global__ void moe_combine_grad_kernel(moe_rows_params p, T const *dy, T const *rows,
                                        float const *weights, T *drows, float *dweights) {
  __shared__ float partial[kGradThreads / 32][kGradGroup];
  grid_start_next();
  grid_wait();
  std::int64_t const t = blockIdx.x;
  std::int32_t const *const at = p.row_of_slot + t * p.topk;
  float const *const w = weights + t * p.topk;
  T const *const g = dy + t * p.token_stride;
  int const warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  for (int j0 = 0; j0 < p.topk; j0 += kGradGroup) {
    std::int32_t r[kGradGroup];
    float f[kGradGroup], dot[kGradGroup];
#pragma unroll
    for (int j = 0; j < kGradGroup; ++j) {
      r[j] = j0 + j < p.topk ? row_at(p, at[j0 + j]) : -1;
      f[j] = r[j] >= 0 ? w[j0 + j] : 0.0f;
      dot[j] = 0.0f;
    }
    for (int c = threadIdx.x * N; c < p.hidden; c += blockDim.x * N) {
      vec<T, N> const d = load_vec<T, N>(g + c);
      vec<T, N> v[kGradGroup];
#pragma unroll
      for (int j = 0; j < kGradGroup; ++j) {
        if (r[j] >= 0) v[j] = load_vec<T, N>(rows + r[j] * p.row_stride + c);
      }
#pragma unroll
      for (int j = 0; j < kGradGroup; ++j) {
        if (r[j] < 0) continue;
        vec<T, N> out;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          dot[j] = fmaf(d.f32(i), v[j].f32(i), dot[j]);
          out.v[i] = from_f32<T>(f[j] * d.f32(i));
        }
        store_vec<T, N>(drows + r[j] * p.row_stride + c, out);
      }
    }
#pragma unroll
    for (int j = 0; j < kGradGroup; ++j) {
#pragma unroll
      for (int m = 16; m > 0; m /= 2) dot[j] += __shfl_xor_sync(0xffffffffu, dot[j], m);
      if (lane == 0) partial[warp][j] = dot[j];
    }
    __syncthreads();
    if (threadIdx.x < kGradGroup && j0 + static_cast<int>(threadIdx.x) < p.topk) {
      float sum = 0.0f;
      for (int i = 0; i < static_cast<int>(blockDim.x) / 32; ++i) sum += partial[i][threadIdx.x];
      dweights[t * p.topk + j0 + threadIdx.x] = sum;
    }
    __syncthreads();
  }
}

}  // namespace megacu_b200
