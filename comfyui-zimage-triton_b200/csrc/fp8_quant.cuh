// e4m3 blocks of 128 with a power-of-two scale: the arithmetic that the quantising kernels share.
//
// Quantiser: a block of values (1 x 128 of an activation row, 128 x 128 of a weight) with largest
// magnitude a is held as e4m3 values q = x / s, s = 2^e with the least e >= -120 such that
// a <= 448 s.  A power of two makes the division exact, so q is the one rounding of x to e4m3's
// 4-bit mantissa (ties to even) and any implementation gives the same bits; as the format floats,
// scales between the powers would gain no precision but at the bottom of its range.  A block with
// an infinity or a NaN gets NaN for its scale and its values.
#pragma once

#include "zib_async.cuh"
#include "zib_types.cuh"

#include <cuda_fp8.h>

namespace zib {
namespace fp8 {

constexpr int kBlock = 128;

// e with s = 2^e for a block's largest magnitude (given as its fp32 bits: NaN > infinity > finite)
__device__ __forceinline__ float block_scale(uint32_t amax_bits) {
  if (amax_bits >= 0x7F800000u) return __uint_as_float(0x7FC00000u);
  // a = m 2^k with m in [1, 2); 448 = 1.75 * 2^8
  int e = (int)(amax_bits >> 23) - 127 - 8 + ((amax_bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  if (e < -120) e = -120;
  return __uint_as_float((uint32_t)(e + 127) << 23);
}
// 1 / s, exact for a power of two
__device__ __forceinline__ float inverse_scale(float s) {
  const uint32_t b = __float_as_uint(s);
  return b >= 0x7F800000u ? s : __uint_as_float((254u << 23) - b);
}
// 8 consecutive values from column k of a row of K (16-byte accesses where VEC), 0 past the end
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* __restrict__ row, int64_t k, int64_t K, float (&v)[8]) {
  if constexpr (VEC) {  // K % 8 == 0: all eight or none
    constexpr int E = 16 / sizeof(T);
#pragma unroll
    for (int h = 0; h < 8 / E; ++h) {
      Pack<T, E> t{};
      if (k < K) t = *reinterpret_cast<const Pack<T, E>*>(row + k + h * E);
#pragma unroll
      for (int j = 0; j < E; ++j) v[h * E + j] = to_f32(t.v[j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = k + j < K ? to_f32(row[k + j]) : 0.0f;
  }
}

// The largest magnitude of 8 values, as its bits.
__device__ __forceinline__ uint32_t amax8(const float (&v)[8]) {
  uint32_t a = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) a = max(a, __float_as_uint(v[j]) & 0x7FFFFFFFu);
  return a;
}

// 8-byte stores where VEC; WHOLE: K % 8 == 0
template <bool VEC, bool WHOLE = true>
__device__ __forceinline__ void store8(uint8_t* __restrict__ row, int64_t k, int64_t K, const float (&v)[8],
                                       float inv) {
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(v[4 * h] * inv, v[4 * h + 1] * inv), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(v[4 * h + 2] * inv, v[4 * h + 3] * inv), __NV_SATFINITE, __NV_E4M3);
    w[h] = lo | (hi << 16);
  }
  if constexpr (VEC && WHOLE) {
    if (k < K) *reinterpret_cast<uint2*>(row + k) = make_uint2(w[0], w[1]);
  } else if (VEC && k + 8 <= K) {
    *reinterpret_cast<uint2*>(row + k) = make_uint2(w[0], w[1]);
  } else {  // also a ragged row's end: what lies behind it stays
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (k + j < K) row[k + j] = (uint8_t)(w[j >> 2] >> (8 * (j & 3)));
  }
}

}  // namespace fp8

// fp8_block.cu: rows of x [M, K] as e4m3 q and scales s.  part (may be null): the sums of x's columns
// over slabs of rows, fp8_sum_rows(M) rows of K floats, which fp8_sum_finish adds up.
int fp8_quant_rows(const void* x, int64_t ldx, int dtype, void* q, int64_t ldq, float* s, int64_t s_m, int64_t s_k,
                   float* part, int64_t M, int64_t K, cudaStream_t st, const char* what);
int64_t fp8_sum_rows(int64_t M);
void fp8_sum_finish(const float* part, void* sum, int dtype, int64_t M, int64_t K, cudaStream_t st);
// the product on tensor cores (fp8_gemm.cu); exponents: sx are powers of two (no subnormals) or NaN, as the
// quantiser makes them; dependent: q and sx come from the launch before
int fp8_gemm(const void* q, int64_t ldq, const float* sx, int64_t sx_m, int64_t sx_k, const void* w, int64_t ldw,
             const float* sw, int64_t sw_n, int64_t sw_k, const void* bias, void* y, int64_t ldy, int dtype, int64_t M,
             int64_t N, int64_t K, bool exponents, bool dependent, cudaStream_t st, const char* what);

}  // namespace zib
