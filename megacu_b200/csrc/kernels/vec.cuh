// Groups of N elements of a row as 32-bit floats: one access of 32 or 16 bytes
// when the rows allow it, single elements otherwise (N = 1).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

namespace megacu_b200 {

template <class T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32(float v) { return __float2bfloat16_rn(v); }

// 16 bytes that this kernel reads once: kept out of L1. The memory clobber
// keeps it before later stores, which may go to the same address.
__device__ __forceinline__ uint4 load_once(void const *p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p)
               : "memory");
  return v;
}

// 32 bytes at a time (addresses multiples of 32): a lane's whole sector in one
// access, so that neighbouring lanes do not each touch half of one twice.
struct alignas(32) bytes32 {
  std::uint32_t w[8];
};

__device__ __forceinline__ bytes32 load32_once(void const *p) {
  bytes32 v;
  asm volatile("ld.global.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(v.w[0]), "=r"(v.w[1]), "=r"(v.w[2]), "=r"(v.w[3]), "=r"(v.w[4]),
                 "=r"(v.w[5]), "=r"(v.w[6]), "=r"(v.w[7])
               : "l"(p)
               : "memory");
  return v;
}

__device__ __forceinline__ void store32(void *p, bytes32 const &v) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
               :: "l"(p), "r"(v.w[0]), "r"(v.w[1]), "r"(v.w[2]), "r"(v.w[3]), "r"(v.w[4]),
                  "r"(v.w[5]), "r"(v.w[6]), "r"(v.w[7])
               : "memory");
}

template <class T, int N>
struct alignas(sizeof(T) * N) vec {
  T v[N];
  __device__ __forceinline__ float f32(int i) const { return to_f32(v[i]); }
};

template <class T, int N>
__device__ __forceinline__ vec<T, N> load_vec(T const *p) {
  if constexpr (sizeof(T) * N == 32) {
    bytes32 const raw = load32_once(p);
    return *reinterpret_cast<vec<T, N> const *>(&raw);
  } else if constexpr (sizeof(T) * N == 16) {
    uint4 const raw = load_once(p);
    return *reinterpret_cast<vec<T, N> const *>(&raw);
  } else {
    return *reinterpret_cast<vec<T, N> const *>(p);
  }
}

template <class T, int N>
__device__ __forceinline__ void store_vec(T *p, vec<T, N> const &v) {
  if constexpr (sizeof(T) * N == 32) {
    store32(p, *reinterpret_cast<bytes32 const *>(&v));
  } else {
    *reinterpret_cast<vec<T, N> *>(p) = v;
  }
}

}  // namespace megacu_b200
