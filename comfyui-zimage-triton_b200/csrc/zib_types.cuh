// Element types and small host helpers shared by the rotary, group-norm and block-scaled 8-bit kernels.
#pragma once

#include "zib_common.cuh"

#include <atomic>
#include <cuda_fp16.h>

namespace zib {

// --- element types of the C ABI (zib_dtype) ----------------------------------

__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(float v) { return v; }

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }

// VEC consecutive elements, moved as one access of VEC * sizeof(T) bytes (at most 16)
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
  T v[VEC];
};

// element i of an array whose zib_dtype is known at run time only (weights and biases: read a
// few times per thread)
__device__ __forceinline__ float load_as_f32(const void* p, int dtype, int64_t i) {
  if (dtype == ZIB_BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
  if (dtype == ZIB_F16) return __half2float(reinterpret_cast<const __half*>(p)[i]);
  return reinterpret_cast<const float*>(p)[i];
}
__device__ __forceinline__ void store_as(void* p, int dtype, int64_t i, float v) {
  if (dtype == ZIB_BF16) reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else if (dtype == ZIB_F16) reinterpret_cast<__half*>(p)[i] = __float2half_rn(v);
  else reinterpret_cast<float*>(p)[i] = v;
}

// --- host ------------------------------------------------------------------------

inline bool known_dtype(int d) { return d == ZIB_BF16 || d == ZIB_F16 || d == ZIB_F32; }
inline int dtype_bytes(int d) { return d == ZIB_F32 ? 4 : 2; }

// multiprocessors of the current device (looked up once per device)
inline int sm_count() {
  static std::atomic<int> cached[64];  // 0: not yet; threads that look it up at once find the same
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  int n = cached[dev].load(std::memory_order_relaxed);
  if (!n) {
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    if (n <= 0) n = 148;
    cached[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

}  // namespace zib
