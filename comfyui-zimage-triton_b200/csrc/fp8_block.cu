// Operands of matrix products in 8-bit floating point (e4m3) with one scale for each block of 128:
// quantisers, transposed weights, and the column sums of a bias gradient.
#include "fp8_quant.cuh"

#include <type_traits>

namespace zib {
namespace fp8 {

// 8 values as they lie in memory: whole 16-byte pieces where VEC (K % 8 == 0: all eight or none)
template <typename T>
struct Raw {
  Pack<T, 16 / sizeof(T)> v[sizeof(T) / 2];
};

template <typename T, bool VEC>
__device__ __forceinline__ Raw<T> load_raw(const T* __restrict__ row, int64_t k, int64_t K) {
  constexpr int E = 16 / sizeof(T);
  Raw<T> r{};
#pragma unroll
  for (int h = 0; h < 8 / E; ++h) {
    if constexpr (VEC) {
      if (k < K) r.v[h] = *reinterpret_cast<const Pack<T, E>*>(row + k + h * E);
    } else if (k + (h + 1) * E <= K) {
#pragma unroll
      for (int j = 0; j < E; ++j) r.v[h].v[j] = row[k + h * E + j];
    } else {
#pragma unroll
      for (int j = 0; j < E; ++j)
        if (k + h * E + j < K) r.v[h].v[j] = row[k + h * E + j];
    }
  }
  return r;
}

template <typename T>
__device__ __forceinline__ void widen(const Raw<T>& r, float (&v)[8]) {
  constexpr int E = 16 / sizeof(T);
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = to_f32(r.v[j / E].v[j % E]);
}

// Largest magnitudes.  They order as their bits, so the 16-bit types are compared two at a time without
// unpacking (first in either half of the result), fp32 as they are.
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
  uint32_t m;
  asm("max.u16x2 %0, %1, %2;" : "=r"(m) : "r"(a), "r"(b));
  return m;
}
template <typename T>
__device__ __forceinline__ uint32_t join(uint32_t a, uint32_t b) {
  return sizeof(T) == 2 ? max2(a, b) : max(a, b);
}
template <typename T>
__device__ __forceinline__ uint32_t largest(const Raw<T>& r) {
  if constexpr (sizeof(T) == 2) {
    const uint4 u = *reinterpret_cast<const uint4*>(&r);
    return max2(max2(u.x & 0x7FFF7FFFu, u.y & 0x7FFF7FFFu), max2(u.z & 0x7FFF7FFFu, u.w & 0x7FFF7FFFu));
  } else {
    float f[8];
    widen(r, f);
    return amax8(f);
  }
}
// as fp32 bits
template <typename T>
__device__ __forceinline__ uint32_t largest_f32(uint32_t m) {
  if constexpr (sizeof(T) == 2) {
    const uint16_t a = (uint16_t)max(m >> 16, m & 0xFFFFu);
    return __float_as_uint(to_f32(*reinterpret_cast<const T*>(&a)));
  } else {
    return m;
  }
}
// of 8 lanes' 16 values each
template <typename T>
__device__ __forceinline__ uint32_t block_amax(const Raw<T>& lo, const Raw<T>& hi) {
  uint32_t m = join<T>(largest(lo), largest(hi));
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) m = join<T>(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
  return largest_f32<T>(m);
}

// Activation rows.  Bound by memory (3 bytes per 16-bit element).  A CTA takes 8 * wrows rows of four blocks
// (512 columns), a warp wrows of them, two rows in flight; 8 lanes x 16 values to a block (8 of
// either half of it, so that accesses stay side by side): what is done once per block and lane, its
// maximum over lanes and its scale, counts half as much as with 16 lanes.  18432 x 3840 bf16: 41 us
// (5.2 TB/s, 71% of the issue slots); 16 lanes to a block, 8 rows in flight 72 us.
// SUM: the CTA leaves the sums of its columns in part[.][K] (a bias gradient: the rows need not be read
// again for it).
constexpr int kRows = 64;
constexpr int kQuad = 4 * kBlock;

// VEC: 16-byte loads (x has aligned rows of whole eights); VST: 8-byte stores (q has aligned rows, of
// any length).  Rows of odd lengths come with unaligned x and, from a linear, aligned q: 14951 x 2129 bf16
// in 35 us.
template <typename T, bool VEC, bool VST, bool SUM>
__global__ void __launch_bounds__(256, sizeof(T) == 2 && !SUM ? 4 : 3) quant_rows_kernel(
    const T* __restrict__ x, int64_t ldx, uint8_t* __restrict__ q, int64_t ldq, float* __restrict__ s, int64_t s_m,
    int64_t s_k, float* __restrict__ part, int64_t M, int64_t K, int quads, int wrows) {
  constexpr int U = 2;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t group = blockIdx.x / quads;
  const int64_t b = 4 * (int64_t)(blockIdx.x - group * quads) + (lane >> 3);
  const int64_t k = b * kBlock + (lane & 7) * 8;
  const int64_t m0 = (group * 8 + warp) * wrows;
  const int rows = M - m0 < wrows ? (int)(M - m0) : wrows;
  const T* xr = x + m0 * ldx;
  uint8_t* qr = q + m0 * ldq;
  float* sr = s + m0 * s_m + b * s_k;
  float sum[16];
#pragma unroll
  for (int j = 0; j < 16; ++j) sum[j] = 0.0f;
#pragma unroll 1
  for (int m = 0; m < rows; m += U) {
    Raw<T> lo[U], hi[U];
#pragma unroll
    for (int r = 0; r < U; ++r) {
      const int64_t Kr = m + r < rows ? K : 0;
      lo[r] = load_raw<T, VEC>(xr + r * ldx, k, Kr);
      hi[r] = load_raw<T, VEC>(xr + r * ldx, k + 64, Kr);
    }
#pragma unroll
    for (int r = 0; r < U; ++r) {
      const float sc = block_scale(block_amax(lo[r], hi[r])), inv = inverse_scale(sc);
      const int64_t Kr = m + r < rows ? K : 0;
      float f[8];
      widen(lo[r], f);
      if constexpr (SUM)
#pragma unroll
        for (int j = 0; j < 8; ++j) sum[j] += f[j];
      store8<VST, VEC>(qr + r * ldq, k, Kr, f, inv);
      widen(hi[r], f);
      if constexpr (SUM)
#pragma unroll
        for (int j = 0; j < 8; ++j) sum[8 + j] += f[j];
      store8<VST, VEC>(qr + r * ldq, k + 64, Kr, f, inv);
      if ((lane & 7) == 0 && b * kBlock < Kr) sr[r * s_m] = sc;
    }
    xr += U * ldx;
    qr += U * ldq;
    sr += U * s_m;
  }
  if constexpr (SUM) {
    __shared__ float red[8][kQuad];
    const int c = (lane >> 3) * kBlock + (lane & 7) * 8;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      red[warp][c + j] = sum[j];
      red[warp][c + 64 + j] = sum[8 + j];
    }
    __syncthreads();
    const int64_t k0 = 4 * (int64_t)(blockIdx.x - group * quads) * kBlock;
    for (int i = threadIdx.x; i < kQuad && k0 + i < K; i += 256) {
      float v = red[0][i];
#pragma unroll
      for (int w = 1; w < 8; ++w) v += red[w][i];
      part[group * K + k0 + i] = v;
    }
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // a product may start and wait
}

// Weights: one CTA per block of 128 x 128, held in registers (as loaded) between its maximum and its
// values.  11520 x 3840 bf16 33 us (4.0 TB/s; 37 with a fourth CTA on an SM, whose registers spill, 40 with
// the values widened first), fp32 37 us (6.0 TB/s).
template <typename T, bool VEC, bool VST>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? (VEC ? 3 : 2) : 1) quant_blocks_kernel(
    const T* __restrict__ w, int64_t ldw, uint8_t* __restrict__ q, int64_t ldq, float* __restrict__ s, int64_t s_n,
    int64_t s_k, int64_t N, int64_t K) {
  __shared__ uint32_t red[8];
  const int64_t n0 = (int64_t)blockIdx.y * kBlock + (threadIdx.x >> 4);
  const int64_t k = (int64_t)blockIdx.x * kBlock + (threadIdx.x & 15) * 8;
  Raw<T> v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = load_raw<T, VEC>(w + (n0 + 16 * i) * ldw, k, n0 + 16 * i < N ? K : 0);
  uint32_t a = largest(v[0]);
#pragma unroll
  for (int i = 1; i < 8; ++i) a = join<T>(a, largest(v[i]));
  a = __reduce_max_sync(0xFFFFFFFFu, largest_f32<T>(a));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = a;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) a = max(a, red[i]);
  const float sc = block_scale(a), inv = inverse_scale(sc);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float f[8];
    widen(v[i], f);
    store8<VST, VEC>(q + (n0 + 16 * i) * ldq, k, n0 + 16 * i < N ? K : 0, f, inv);
  }
  if (threadIdx.x == 0) s[blockIdx.y * s_n + blockIdx.x * s_k] = sc;
}

// wt[k, n] = w[n, k], 64 x 64 bytes per CTA
__global__ void __launch_bounds__(256) transpose_kernel(const uint8_t* __restrict__ w, int64_t ldw,
                                                        uint8_t* __restrict__ wt, int64_t ldt, int64_t N, int64_t K) {
  __shared__ uint8_t t[64][68];
  const int64_t n0 = (int64_t)blockIdx.y * 64, k0 = (int64_t)blockIdx.x * 64;
  for (int i = threadIdx.x; i < 4096; i += 256) {
    const int r = i >> 6, c = i & 63;
    if (n0 + r < N && k0 + c < K) t[r][c] = w[(n0 + r) * ldw + k0 + c];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 4096; i += 256) {
    const int r = i >> 6, c = i & 63;
    if (k0 + r < K && n0 + c < N) wt[(k0 + r) * ldt + n0 + c] = t[c][r];
  }
}

// column sums of x [M, N] (a bias gradient): fp32 sums of slabs of rows ...
template <typename T>
__global__ void __launch_bounds__(256) col_sum_part_kernel(const T* __restrict__ x, int64_t ldx,
                                                           float* __restrict__ part, int64_t M, int64_t N,
                                                           int64_t slab) {
  const int64_t n = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (n >= N) return;
  const int64_t m0 = (int64_t)blockIdx.y * slab, m1 = m0 + slab < M ? m0 + slab : M;
  float s = 0.0f;
#pragma unroll 8
  for (int64_t m = m0; m < m1; ++m) s += to_f32(x[m * ldx + n]);
  part[blockIdx.y * N + n] = s;
}
// ... and their sums: 32 columns per CTA, 8 threads to a column
template <typename T>
__global__ void __launch_bounds__(256) col_sum_kernel(const float* __restrict__ part, T* __restrict__ y, int64_t N,
                                                      int64_t slabs) {
  __shared__ double red[8][32];
  const int c = threadIdx.x & 31, r = threadIdx.x >> 5;
  const int64_t n = (int64_t)blockIdx.x * 32 + c;
  double s = 0.0;
  if (n < N)
    for (int64_t i = r; i < slabs; i += 8) s += part[i * N + n];
  red[r][c] = s;
  __syncthreads();
  if (r == 0 && n < N) {
#pragma unroll
    for (int i = 1; i < 8; ++i) s += red[i][c];
    y[n] = from_f32<T>((float)s);
  }
}

constexpr int kMaxSlabs = 64;

static void col_sum(const float* part, void* y, int dtype, int64_t N, int64_t slabs, cudaStream_t st) {
  const unsigned g = (unsigned)ceil_div(N, 32);
  if (dtype == ZIB_BF16) col_sum_kernel<<<g, 256, 0, st>>>(part, (__nv_bfloat16*)y, N, slabs);
  else if (dtype == ZIB_F16) col_sum_kernel<<<g, 256, 0, st>>>(part, (__half*)y, N, slabs);
  else col_sum_kernel<<<g, 256, 0, st>>>(part, (float*)y, N, slabs);
}

// eight values per access: of rows x, of rows q
static bool vector_loads(const void* x, int64_t ldx, int size, int64_t rows, int64_t K) {
  return K % 8 == 0 && (uintptr_t)x % 16 == 0 && (ldx * size % 16 == 0 || rows == 1);
}
static bool vector_stores(const void* q, int64_t ldq, int64_t rows) {
  return (uintptr_t)q % 8 == 0 && (ldq % 8 == 0 || rows == 1);
}

// Rows of bytes copied to 16-byte aligned rows, a thread to 16 bytes; the bytes behind a row's end are
// left as they are.  Weights of an odd K come so in every call: a linear of 1576 x 7907 -> 750 takes
// 52 us, with single-byte copies here and single-byte stores in the quantiser 78 us.
__global__ void __launch_bounds__(256) align_rows_kernel(const uint8_t* __restrict__ w, int64_t ldw,
                                                         uint8_t* __restrict__ out, int64_t ldo, int64_t N, int64_t K) {
  const int64_t pieces = (K + 15) / 16, id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t n = id / pieces, k = (id - n * pieces) * 16;
  if (n >= N) return;
  const uint8_t* from = w + n * ldw + k;
  uint8_t* to = out + n * ldo + k;
  if (k + 16 <= K) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      u[i] = from[4 * i] | (uint32_t)from[4 * i + 1] << 8 | (uint32_t)from[4 * i + 2] << 16 |
             (uint32_t)from[4 * i + 3] << 24;
    *reinterpret_cast<uint4*>(to) = make_uint4(u[0], u[1], u[2], u[3]);
  } else {
    for (int i = 0; i < (int)(K - k); ++i) to[i] = from[i];
  }
}

}  // namespace fp8
}  // namespace zib

using namespace zib;

int64_t zib::fp8_sum_rows(int64_t M) { return ceil_div(M, fp8::kRows); }

int zib::fp8_quant_rows(const void* x, int64_t ldx, int dtype, void* q, int64_t ldq, float* s, int64_t s_m, int64_t s_k,
                        float* part, int64_t M, int64_t K, cudaStream_t st, const char* what) {
  const bool vec = fp8::vector_loads(x, ldx, dtype_bytes(dtype), M, K), vst = fp8::vector_stores(q, ldq, M);
  const int64_t quads = ceil_div(K, fp8::kQuad);
  // Rows to a warp.  Two are in flight anyway: eight make a chain of loads, which few rows wait for and
  // scalar loads lengthen (2 / 8 rows, bf16: 8 x 3840 1.9 / 3.3 us, 1024 x 3840 4.4 / 6.3, 14951 x 2129
  // 35 / 41); two are more CTAs to start (18432 x 3840 44 / 41).  Column sums want long slabs.
  const bool many = vec && ceil_div(M, fp8::kRows) * quads >= 3 * sm_count();
  const int wrows = part || many ? fp8::kRows / 8 : 2;
  const int64_t grid = ceil_div(M, 8 * wrows) * quads;
  ZIB_HOST_CHECK(grid <= 0x7FFFFFFF, ZIB_ERR_TOO_LARGE, "%s: M=%lld K=%lld", what, (long long)M, (long long)K);
  auto go = [&](auto* xt) {
    using T = std::remove_cv_t<std::remove_pointer_t<decltype(xt)>>;
    using namespace fp8;
    auto* kernel = part ? (!vst  ? quant_rows_kernel<T, false, false, true>
                           : vec ? quant_rows_kernel<T, true, true, true>
                                 : quant_rows_kernel<T, false, true, true>)
                        : (!vst  ? quant_rows_kernel<T, false, false, false>
                           : vec ? quant_rows_kernel<T, true, true, false>
                                 : quant_rows_kernel<T, false, true, false>);
    kernel<<<(unsigned)grid, 256, 0, st>>>(xt, ldx, (uint8_t*)q, ldq, s, s_m, s_k, part, M, K, (int)quads, wrows);
  };
  if (dtype == ZIB_BF16) go((const __nv_bfloat16*)x);
  else if (dtype == ZIB_F16) go((const __half*)x);
  else go((const float*)x);
  return zib_check_launch(what);
}

void zib::fp8_sum_finish(const float* part, void* sum, int dtype, int64_t M, int64_t K, cudaStream_t st) {
  fp8::col_sum(part, sum, dtype, K, fp8_sum_rows(M), st);
}

extern "C" int zib_fp8_quant_rows(const void* x, int64_t ldx, int dtype, void* q, int64_t ldq, float* s, int64_t s_m,
                                  int64_t s_k, int64_t M, int64_t K, void* stream) {
  const char* what = "zib_fp8_quant_rows";
  ZIB_HOST_CHECK(known_dtype(dtype), ZIB_ERR_INVALID_ARG, "%s: unknown dtype %d", what, dtype);
  ZIB_HOST_CHECK(M >= 0 && K >= 1 && ldx >= K && ldq >= K, ZIB_ERR_INVALID_ARG, "%s: bad shape M=%lld K=%lld", what,
                 (long long)M, (long long)K);
  if (M == 0) return ZIB_OK;
  ZIB_HOST_CHECK(x && q && s, ZIB_ERR_INVALID_ARG, "%s: null operand", what);
  return fp8_quant_rows(x, ldx, dtype, q, ldq, s, s_m, s_k, nullptr, M, K, (cudaStream_t)stream, what);
}

extern "C" int zib_fp8_quant_blocks(const void* w, int64_t ldw, int dtype, void* q, int64_t ldq, float* s, int64_t s_n,
                                    int64_t s_k, int64_t N, int64_t K, void* stream) {
  const char* what = "zib_fp8_quant_blocks";
  ZIB_HOST_CHECK(known_dtype(dtype), ZIB_ERR_INVALID_ARG, "%s: unknown dtype %d", what, dtype);
  ZIB_HOST_CHECK(N >= 1 && K >= 1 && ldw >= K && ldq >= K, ZIB_ERR_INVALID_ARG, "%s: bad shape N=%lld K=%lld", what,
                 (long long)N, (long long)K);
  ZIB_HOST_CHECK(w && q && s, ZIB_ERR_INVALID_ARG, "%s: null operand", what);
  const int64_t nb = ceil_div(N, fp8::kBlock), kb = ceil_div(K, fp8::kBlock);
  ZIB_HOST_CHECK(nb <= 65535, ZIB_ERR_TOO_LARGE, "%s: N=%lld", what, (long long)N);
  cudaStream_t st = (cudaStream_t)stream;
  const dim3 g((unsigned)kb, (unsigned)nb);
  const bool vec = fp8::vector_loads(w, ldw, dtype_bytes(dtype), N, K), vst = fp8::vector_stores(q, ldq, N);
  auto go = [&](auto* wt) {
    using T = std::remove_cv_t<std::remove_pointer_t<decltype(wt)>>;
    using namespace fp8;
    auto* kernel = !vst  ? quant_blocks_kernel<T, false, false>
                   : vec ? quant_blocks_kernel<T, true, true>
                         : quant_blocks_kernel<T, false, true>;
    kernel<<<g, 256, 0, st>>>(wt, ldw, (uint8_t*)q, ldq, s, s_n, s_k, N, K);
  };
  if (dtype == ZIB_BF16) go((const __nv_bfloat16*)w);
  else if (dtype == ZIB_F16) go((const __half*)w);
  else go((const float*)w);
  return zib_check_launch(what);
}

extern "C" int zib_fp8_align_rows(const void* w, int64_t ldw, void* out, int64_t ldo, int64_t N, int64_t K,
                                  void* stream) {
  const char* what = "zib_fp8_align_rows";
  ZIB_HOST_CHECK(N >= 0 && K >= 1 && ldw >= 0 && ldo >= K, ZIB_ERR_INVALID_ARG, "%s: bad shape N=%lld K=%lld", what,
                 (long long)N, (long long)K);
  if (N == 0) return ZIB_OK;
  ZIB_HOST_CHECK(w && out, ZIB_ERR_INVALID_ARG, "%s: null operand", what);
  ZIB_HOST_CHECK((uintptr_t)out % 16 == 0 && ldo % 16 == 0, ZIB_ERR_ALIGNMENT, "%s: out needs 16-byte aligned rows", what);
  const int64_t grid = ceil_div(N * ceil_div(K, 16), 256);
  ZIB_HOST_CHECK(grid <= 0x7FFFFFFF, ZIB_ERR_TOO_LARGE, "%s: N=%lld K=%lld", what, (long long)N, (long long)K);
  fp8::align_rows_kernel<<<(unsigned)grid, 256, 0, (cudaStream_t)stream>>>((const uint8_t*)w, ldw, (uint8_t*)out, ldo, N,
                                                                           K);
  return zib_check_launch(what);
}

extern "C" int zib_fp8_transpose(const void* w, int64_t ldw, void* wt, int64_t ldt, int64_t N, int64_t K,
                                 void* stream) {
  const char* what = "zib_fp8_transpose";
  ZIB_HOST_CHECK(N >= 1 && K >= 1 && ldw >= K && ldt >= N, ZIB_ERR_INVALID_ARG, "%s: bad shape N=%lld K=%lld", what,
                 (long long)N, (long long)K);
  ZIB_HOST_CHECK(w && wt, ZIB_ERR_INVALID_ARG, "%s: null operand", what);
  ZIB_HOST_CHECK(ceil_div(N, 64) <= 65535, ZIB_ERR_TOO_LARGE, "%s: N=%lld", what, (long long)N);
  fp8::transpose_kernel<<<dim3((unsigned)ceil_div(K, 64), (unsigned)ceil_div(N, 64)), 256, 0, (cudaStream_t)stream>>>(
      (const uint8_t*)w, ldw, (uint8_t*)wt, ldt, N, K);
  return zib_check_launch(what);
}

extern "C" int zib_col_sum(const void* x, int64_t ldx, int dtype, void* y, float* workspace, int64_t workspace_bytes,
                           int64_t M, int64_t N, void* stream) {
  const char* what = "zib_col_sum";
  ZIB_HOST_CHECK(known_dtype(dtype), ZIB_ERR_INVALID_ARG, "%s: unknown dtype %d", what, dtype);
  ZIB_HOST_CHECK(M >= 0 && N >= 1 && ldx >= N, ZIB_ERR_INVALID_ARG, "%s: bad shape M=%lld N=%lld", what, (long long)M,
                 (long long)N);
  ZIB_HOST_CHECK((x || M == 0) && y && workspace, ZIB_ERR_INVALID_ARG, "%s: null operand", what);
  ZIB_HOST_CHECK(workspace_bytes >= fp8::kMaxSlabs * N * (int64_t)sizeof(float), ZIB_ERR_INVALID_ARG,
                 "%s: workspace of %lld bytes needed", what, (long long)(fp8::kMaxSlabs * N * sizeof(float)));
  const int64_t slab = ceil_div(M > 0 ? M : 1, fp8::kMaxSlabs);
  const int slabs = (int)ceil_div(M, slab);
  const dim3 g((unsigned)ceil_div(N, 256), (unsigned)slabs);
  cudaStream_t st = (cudaStream_t)stream;
  if (slabs > 0) {
    if (dtype == ZIB_BF16) fp8::col_sum_part_kernel<<<g, 256, 0, st>>>((const __nv_bfloat16*)x, ldx, workspace, M, N, slab);
    else if (dtype == ZIB_F16) fp8::col_sum_part_kernel<<<g, 256, 0, st>>>((const __half*)x, ldx, workspace, M, N, slab);
    else fp8::col_sum_part_kernel<<<g, 256, 0, st>>>((const float*)x, ldx, workspace, M, N, slab);
  }
  fp8::col_sum(workspace, y, dtype, N, slabs, st);
  return zib_check_launch(what);
}
