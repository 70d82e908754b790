// Operands of matrix products in 8-bit floating point (e4m3) with one scale for each block of 128:
// quantisers, transposed weights, and the column sums of a bias gradient.
#include "fp8_quant.cuh"

namespace zib {
namespace fp8 {

// Activation rows.  Bound by memory (3 bytes per 16-bit element): a warp takes 8 rows of two blocks,
// 16 lanes x 8 values to a block, with all its loads in flight before the first is used; the 8 rows
// give each block one whole 32-byte sector of the scales, which lie row after row.
constexpr int kRowsPerWarp = 8;

template <typename T, bool VEC>
__global__ void __launch_bounds__(256) quant_rows_kernel(const T* __restrict__ x, int64_t ldx, uint8_t* __restrict__ q,
                                                         int64_t ldq, float* __restrict__ s, int64_t s_m, int64_t s_k,
                                                         int64_t M, int64_t K) {
  const int lane = threadIdx.x & 31;
  const int64_t pairs = (K + 2 * kBlock - 1) / (2 * kBlock);
  const int64_t id = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int64_t m0 = id / pairs * kRowsPerWarp;
  if (m0 >= M) return;
  const int64_t b = 2 * (id % pairs) + (lane >> 4), k = b * kBlock + (lane & 15) * 8;
  float v[kRowsPerWarp][8];
#pragma unroll
  for (int r = 0; r < kRowsPerWarp; ++r) load8<T, VEC>(x + (m0 + r) * ldx, k, m0 + r < M ? K : 0, v[r]);
  float mine = 0.0f;  // lane r of each half warp keeps the scale of row r
#pragma unroll
  for (int r = 0; r < kRowsPerWarp; ++r) {
    uint32_t a = amax8(v[r]);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) a = max(a, __shfl_xor_sync(0xFFFFFFFFu, a, o));
    const float sc = block_scale(a);
    if ((lane & 15) == r) mine = sc;
    store8<VEC>(q + (m0 + r) * ldq, k, m0 + r < M ? K : 0, v[r], inverse_scale(sc));
  }
  const int r = lane & 15;
  if (r < kRowsPerWarp && m0 + r < M && b * kBlock < K) s[(m0 + r) * s_m + b * s_k] = mine;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // a product may start and wait
}

// Weights: one CTA per block of 128 x 128, held in registers between its maximum and its values.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) quant_blocks_kernel(const T* __restrict__ w, int64_t ldw,
                                                           uint8_t* __restrict__ q, int64_t ldq, float* __restrict__ s,
                                                           int64_t s_n, int64_t s_k, int64_t N, int64_t K) {
  __shared__ uint32_t red[8];
  const int64_t n0 = (int64_t)blockIdx.y * kBlock + (threadIdx.x >> 4);
  const int64_t k = (int64_t)blockIdx.x * kBlock + (threadIdx.x & 15) * 8;
  float v[8][8];
  uint32_t a = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) load8<T, VEC>(w + (n0 + 16 * i) * ldw, k, n0 + 16 * i < N ? K : 0, v[i]);
#pragma unroll
  for (int i = 0; i < 8; ++i) a = max(a, amax8(v[i]));
  a = __reduce_max_sync(0xFFFFFFFFu, a);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = a;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) a = max(a, red[i]);
  const float sc = block_scale(a), inv = inverse_scale(sc);
#pragma unroll
  for (int i = 0; i < 8; ++i) store8<VEC>(q + (n0 + 16 * i) * ldq, k, n0 + 16 * i < N ? K : 0, v[i], inv);
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

// column sums of x [M, N] in fp32 (a bias gradient): partial sums of row slabs, then their sums
template <typename T>
__global__ void __launch_bounds__(256) col_sum_part_kernel(const T* __restrict__ x, int64_t ldx,
                                                           float* __restrict__ part, int64_t M, int64_t N,
                                                           int64_t slab) {
  const int64_t n = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (n >= N) return;
  const int64_t m1 = ((int64_t)blockIdx.y + 1) * slab < M ? ((int64_t)blockIdx.y + 1) * slab : M;
  float s = 0.0f;
  for (int64_t m = (int64_t)blockIdx.y * slab; m < m1; ++m) s += to_f32(x[m * ldx + n]);
  part[blockIdx.y * N + n] = s;
}
template <typename T>
__global__ void __launch_bounds__(256) col_sum_kernel(const float* __restrict__ part, T* __restrict__ y, int64_t N,
                                                      int slabs) {
  const int64_t n = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (n >= N) return;
  double s = 0.0;
  for (int i = 0; i < slabs; ++i) s += part[i * N + n];
  y[n] = from_f32<T>((float)s);
}

constexpr int kMaxSlabs = 64;

// eight values per access: columns, strides and addresses of input and output allow it
static bool whole_vectors(const void* x, int64_t ldx, int size, const void* q, int64_t ldq, int64_t rows, int64_t K) {
  return K % 8 == 0 && (uintptr_t)x % 16 == 0 && (ldx * size % 16 == 0 || rows == 1) && (uintptr_t)q % 8 == 0 &&
         (ldq % 8 == 0 || rows == 1);
}

}  // namespace fp8
}  // namespace zib

using namespace zib;

int zib::fp8_quant_rows(const void* x, int64_t ldx, int dtype, void* q, int64_t ldq, float* s, int64_t s_m, int64_t s_k,
                        int64_t M, int64_t K, cudaStream_t st, const char* what) {
  const int64_t grid = ceil_div(ceil_div(M, fp8::kRowsPerWarp) * ceil_div(K, 2 * fp8::kBlock), 8);
  ZIB_HOST_CHECK(grid <= 0x7FFFFFFF, ZIB_ERR_TOO_LARGE, "%s: M=%lld K=%lld", what, (long long)M, (long long)K);
  const bool vec = fp8::whole_vectors(x, ldx, dtype_bytes(dtype), q, ldq, M, K);
  auto go = [&](auto kernel, auto* xt) {
    kernel<<<(unsigned)grid, 256, 0, st>>>(xt, ldx, (uint8_t*)q, ldq, s, s_m, s_k, M, K);
  };
  using B = __nv_bfloat16;
  using H = __half;
  if (dtype == ZIB_BF16) go(vec ? fp8::quant_rows_kernel<B, true> : fp8::quant_rows_kernel<B, false>, (const B*)x);
  else if (dtype == ZIB_F16) go(vec ? fp8::quant_rows_kernel<H, true> : fp8::quant_rows_kernel<H, false>, (const H*)x);
  else go(vec ? fp8::quant_rows_kernel<float, true> : fp8::quant_rows_kernel<float, false>, (const float*)x);
  return zib_check_launch(what);
}

extern "C" int zib_fp8_quant_rows(const void* x, int64_t ldx, int dtype, void* q, int64_t ldq, float* s, int64_t s_m,
                                  int64_t s_k, int64_t M, int64_t K, void* stream) {
  const char* what = "zib_fp8_quant_rows";
  ZIB_HOST_CHECK(known_dtype(dtype), ZIB_ERR_INVALID_ARG, "%s: unknown dtype %d", what, dtype);
  ZIB_HOST_CHECK(M >= 0 && K >= 1 && ldx >= K && ldq >= K, ZIB_ERR_INVALID_ARG, "%s: bad shape M=%lld K=%lld", what,
                 (long long)M, (long long)K);
  if (M == 0) return ZIB_OK;
  ZIB_HOST_CHECK(x && q && s, ZIB_ERR_INVALID_ARG, "%s: null operand", what);
  return fp8_quant_rows(x, ldx, dtype, q, ldq, s, s_m, s_k, M, K, (cudaStream_t)stream, what);
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
  const bool vec = fp8::whole_vectors(w, ldw, dtype_bytes(dtype), q, ldq, N, K);
  auto go = [&](auto kernel, auto* wt) {
    kernel<<<g, 256, 0, st>>>(wt, ldw, (uint8_t*)q, ldq, s, s_n, s_k, N, K);
  };
  using B = __nv_bfloat16;
  using H = __half;
  if (dtype == ZIB_BF16) go(vec ? fp8::quant_blocks_kernel<B, true> : fp8::quant_blocks_kernel<B, false>, (const B*)w);
  else if (dtype == ZIB_F16) go(vec ? fp8::quant_blocks_kernel<H, true> : fp8::quant_blocks_kernel<H, false>, (const H*)w);
  else go(vec ? fp8::quant_blocks_kernel<float, true> : fp8::quant_blocks_kernel<float, false>, (const float*)w);
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
  const dim3 g((unsigned)ceil_div(N, 256), (unsigned)(slabs > 0 ? slabs : 1));
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == ZIB_BF16) {
    if (slabs) fp8::col_sum_part_kernel<<<g, 256, 0, st>>>((const __nv_bfloat16*)x, ldx, workspace, M, N, slab);
    fp8::col_sum_kernel<<<g.x, 256, 0, st>>>(workspace, (__nv_bfloat16*)y, N, slabs);
  } else if (dtype == ZIB_F16) {
    if (slabs) fp8::col_sum_part_kernel<<<g, 256, 0, st>>>((const __half*)x, ldx, workspace, M, N, slab);
    fp8::col_sum_kernel<<<g.x, 256, 0, st>>>(workspace, (__half*)y, N, slabs);
  } else {
    if (slabs) fp8::col_sum_part_kernel<<<g, 256, 0, st>>>((const float*)x, ldx, workspace, M, N, slab);
    fp8::col_sum_kernel<<<g.x, 256, 0, st>>>(workspace, (float*)y, N, slabs);
  }
  return zib_check_launch(what);
}
