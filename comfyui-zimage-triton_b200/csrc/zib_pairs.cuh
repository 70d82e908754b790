// Vectors of 16- or 32-bit elements as packed fp32 pairs (f32x2).
#pragma once

#include "rot_pack.cuh"
#include "zib_types.cuh"

namespace zib {

using px::f2;

__device__ __forceinline__ f2 dup(float v) { return px::mk(v, v); }

template <int VEC>
constexpr int kPairs = VEC < 2 ? 1 : VEC / 2;

// VEC elements as fp32 pairs (a single one with 0 beside it)
__device__ __forceinline__ f2 pair_of(const __nv_bfloat16* v) {
  const uint32_t w = *reinterpret_cast<const uint32_t*>(v);
  return px::mk(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
__device__ __forceinline__ f2 pair_of(const __half* v) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(v));
  return px::mk(f.x, f.y);
}
__device__ __forceinline__ f2 pair_of(const float* v) { return px::mk(v[0], v[1]); }

template <typename T, int VEC>
__device__ __forceinline__ void unpack(const Pack<T, VEC>& t, f2 (&o)[kPairs<VEC>]) {
  if constexpr (VEC == 1) o[0] = px::mk(to_f32(t.v[0]), 0.0f);
  else
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) o[i] = pair_of(t.v + 2 * i);
}

template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> pack(const f2 (&o)[kPairs<VEC>]) {
  Pack<T, VEC> t;
#pragma unroll
  for (int i = 0; i < kPairs<VEC>; ++i) {
    float lo, hi;
    px::split(o[i], lo, hi);
    t.v[2 * i] = from_f32<T>(lo);
    if constexpr (VEC > 1) t.v[2 * i + 1] = from_f32<T>(hi);
  }
  return t;
}

}  // namespace zib
