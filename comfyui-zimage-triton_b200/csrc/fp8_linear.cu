// Linear through a block-scaled 8-bit weight: x is quantised in the call.
//
//   y[m, n] = sum_b sx[m, b] sw[n / 128, b] sum_{k in block b} q[m, k] w[n, k]  (+ bias[n]),  q, sx from x
//
// For few tokens the product is a stream over the weight, bound by memory.  A CTA takes 16 weight
// rows, its eight warps every eighth block of 128 columns; a warp keeps four blocks (8 KB) in flight,
// so an SM has 128 KB on the way.  Within a block the products run on mma.sync (m16n8k32, weight rows
// as its rows, tokens as its columns), whose fresh fp32 sums are scaled into registers block by block;
// the warps' sums meet in shared memory.  The order of k inside a product does not matter, so a
// thread's fragments are whole 16-byte loads straight from the weight: bytes 16t .. 16t + 15 of 64
// serve two MMAs.  One or two tokens are quantised by every CTA itself while its first loads are in
// flight (one launch); more are quantised once by a launch before, which this one overlaps up to its
// first use of the result.
//
// 3840 x 11520 (44 MB, 6.8 us at HBM's rate; a plain reduction over as many bytes takes 11 us): one
// token 13.0 us, eight 13.9 us behind a quantiser of 1.9 us.  Staging the weight in shared memory, one
// persistent CTA per SM, measured 18 us by one bulk copy per 1024 bytes of a row and 15 us by TMA boxes
// of 16 x 1024 bytes.
//
// More than 8 tokens run in groups of 8 through the same kernel while the weight is so small, or its rows so
// long, that the tcgen05 product's few tiles would take longer; else the rows are quantised to
// memory and that product reads them there.
#include "fp8_quant.cuh"

namespace zib {
namespace fp8 {

constexpr int kTileN = 16;
constexpr int kWarps = 8;
constexpr int kRing = 4;         // blocks in flight per warp
constexpr int kMaxTokens = 8;
constexpr int kFusedTokens = 2;  // tokens that every CTA quantises itself
constexpr int kFusedSmem = 96 * 1024;  // for them; leaves two CTAs to an SM

struct SmallParams {
  const void* x;  // FUSED: the tokens; else e4m3 rows, 16-byte aligned
  int64_t ldx;
  const float* sx;  // not FUSED: scales [kb][M]
  const uint8_t* w;
  int64_t ldw;
  const float* sw;
  int64_t sw_n, sw_k;
  const void* bias;
  void* y;
  int64_t ldy;
  int M, N, K, kb;
  int vec;  // FUSED: x's rows allow 16-byte accesses
};

// bytes of a quantised token in shared memory: whole blocks, and 64 more so that the rows of two tokens
// fall on different banks
__host__ __device__ __forceinline__ int row_bytes(int kb) { return kb * kBlock + 64; }

__device__ __forceinline__ void mma_e4m3(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, "
      "%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 16 bytes of a row from p on, 0 where !ok; nothing looks at them here, so the load stays in flight
__device__ __forceinline__ uint4 load16(const uint8_t* p, bool ok) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if (ok) v = __ldg(reinterpret_cast<const uint4*>(p));
  return v;
}

// the first `left` bytes of v, 0 behind them (what lies behind a row's end is not part of it)
__device__ __forceinline__ uint4 first_bytes(uint4 v, int left) {
  uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int l = left - 4 * i;
    if (l <= 0) u[i] = 0;
    else if (l < 4) u[i] &= (1u << (8 * l)) - 1u;
  }
  return make_uint4(u[0], u[1], u[2], u[3]);
}

// FUSED: the tokens are quantised here
template <typename T, bool FUSED>
__global__ void __launch_bounds__(kWarps * 32, 2) linear_small_kernel(const SmallParams p) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float red[kWarps][kTileN][kMaxTokens];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int n0 = blockIdx.x * kTileN;
  const int m0 = FUSED ? 0 : blockIdx.y * kMaxTokens, M = min(p.M - m0, kMaxTokens);  // this CTA's tokens

  // rows g and g + 8 of the tile
  const bool ok0 = n0 + g < p.N, ok1 = n0 + g + 8 < p.N;
  const uint8_t* r0 = p.w + (int64_t)(n0 + g) * p.ldw + 16 * t;
  const uint8_t* r1 = r0 + 8 * p.ldw;
  uint4 w[kRing][4];
  auto fetch = [&](int b, uint4 (&v)[4]) {
    const int k = b * kBlock;
    const bool lo = k + 16 * t < p.K, hi = k + 64 + 16 * t < p.K;
    v[0] = load16(r0 + k, ok0 && lo);
    v[1] = load16(r1 + k, ok1 && lo);
    v[2] = load16(r0 + k + 64, ok0 && hi);
    v[3] = load16(r1 + k + 64, ok1 && hi);
  };
#pragma unroll
  for (int i = 0; i < kRing; ++i) fetch(warp + i * kWarps, w[i]);

  const int rb = row_bytes(p.kb);
  float* ssx = reinterpret_cast<float*>(smem + (size_t)kFusedTokens * rb);  // [kb][kFusedTokens]
  if constexpr (FUSED) {
    for (int i = threadIdx.x >> 4; i < p.M * p.kb; i += kWarps * 2) {  // half a warp to a block
      const int m = i / p.kb, b = i - m * p.kb, k = b * kBlock + (lane & 15) * 8;
      float v[8];
      const T* row = reinterpret_cast<const T*>(p.x) + m * p.ldx;
      if (p.vec) load8<T, true>(row, k, p.K, v);
      else load8<T, false>(row, k, p.K, v);
      uint32_t a = amax8(v);
      const uint32_t mask = 0xFFFFu << (lane & 16);
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) a = max(a, __shfl_xor_sync(mask, a, o));
      const float sc = block_scale(a);
      store8<true>(smem + m * rb, k, p.kb * kBlock, v, inverse_scale(sc));
      if ((lane & 15) == 0) ssx[b * kFusedTokens + m] = sc;
    }
    __syncthreads();
  } else {
    asm volatile("griddepcontrol.wait;" ::: "memory");  // the quantised tokens
  }

  float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  const float* sw = p.sw + (n0 / kBlock) * p.sw_n;
  const float* sx = FUSED ? nullptr : p.sx + m0 + 2 * t;
  const bool c0 = 2 * t < M, c1 = 2 * t + 1 < M;  // columns behind the last token stay unused
  for (int b0 = warp; b0 < p.kb; b0 += kRing * kWarps) {
#pragma unroll
    for (int i = 0; i < kRing; ++i) {
      const int b = b0 + i * kWarps;
      if (b >= p.kb) break;
      const float s = __ldg(sw + b * p.sw_k);
      uint4 x0, x1;
      float sc0, sc1;
      if constexpr (FUSED) {
        const uint8_t* xr = smem + (g < p.M ? g : 0) * rb + b * kBlock + 16 * t;
        x0 = *reinterpret_cast<const uint4*>(xr);
        x1 = *reinterpret_cast<const uint4*>(xr + 64);
        sc0 = c0 ? ssx[b * kFusedTokens + 2 * t] : 0.0f;
        sc1 = c1 ? ssx[b * kFusedTokens + 2 * t + 1] : 0.0f;
      } else {
        const int k = b * kBlock + 16 * t;
        const uint8_t* xr = reinterpret_cast<const uint8_t*>(p.x) + (m0 + g) * p.ldx + k;
        x0 = load16(xr, g < M && k < p.K);
        x1 = load16(xr + 64, g < M && k + 64 < p.K);
        sc0 = c0 ? __ldg(sx + (int64_t)b * p.M) : 0.0f;
        sc1 = c1 ? __ldg(sx + (int64_t)b * p.M + 1) : 0.0f;
      }
      uint4 (&v)[4] = w[i];
      const int left = p.K - b * kBlock - 16 * t;  // bytes of a row from this thread's first one on
      if (left < 80 && p.K % 16) {  // the row ends inside one of this thread's pieces
        v[0] = first_bytes(v[0], left);
        v[1] = first_bytes(v[1], left);
        v[2] = first_bytes(v[2], left - 64);
        v[3] = first_bytes(v[3], left - 64);
        x0 = first_bytes(x0, left);
        x1 = first_bytes(x1, left - 64);
      }
      float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      mma_e4m3(d, v[0].x, v[1].x, v[0].y, v[1].y, x0.x, x0.y);
      mma_e4m3(d, v[0].z, v[1].z, v[0].w, v[1].w, x0.z, x0.w);
      mma_e4m3(d, v[2].x, v[3].x, v[2].y, v[3].y, x1.x, x1.y);
      mma_e4m3(d, v[2].z, v[3].z, v[2].w, v[3].w, x1.z, x1.w);
      acc[0] = fmaf(d[0], sc0 * s, acc[0]);
      acc[1] = fmaf(d[1], sc1 * s, acc[1]);
      acc[2] = fmaf(d[2], sc0 * s, acc[2]);
      acc[3] = fmaf(d[3], sc1 * s, acc[3]);
      if (b + kRing * kWarps < p.kb) fetch(b + kRing * kWarps, v);
    }
  }
  *reinterpret_cast<float2*>(&red[warp][g][2 * t]) = make_float2(acc[0], acc[1]);
  *reinterpret_cast<float2*>(&red[warp][g + 8][2 * t]) = make_float2(acc[2], acc[3]);
  __syncthreads();
  for (int i = threadIdx.x; i < kTileN * M; i += kWarps * 32) {
    const int m = i / kTileN, n = i % kTileN;  // a token's 16 outputs side by side
    float v = 0.0f;
#pragma unroll
    for (int k = 0; k < kWarps; ++k) v += red[k][n][m];
    if (n0 + n < p.N) {
      if (p.bias) v += to_f32(reinterpret_cast<const T*>(p.bias)[n0 + n]);
      reinterpret_cast<T*>(p.y)[(m0 + m) * p.ldy + n0 + n] = from_f32<T>(v);
    }
  }
}

static size_t fused_smem(int64_t kb) { return (size_t)kFusedTokens * (row_bytes((int)kb) + kb * sizeof(float)); }

template <typename T, bool FUSED>
static int launch_small(const SmallParams& p, cudaStream_t st, const char* what) {
  auto* kernel = linear_small_kernel<T, FUSED>;
  const size_t smem = FUSED ? fused_smem(p.kb) : 0;
  if (smem > 32 * 1024) {  // the largest size at once: another thread may launch with another one
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kFusedSmem);
    ZIB_HOST_CHECK(e == cudaSuccess, ZIB_ERR_LAUNCH, "%s: cudaFuncSetAttribute failed: %s", what,
                   cudaGetErrorString(e));
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)ceil_div(p.N, kTileN), (unsigned)ceil_div(p.M, kMaxTokens));
  cfg.blockDim = dim3(kWarps * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = FUSED ? 0 : 1;  // it waits for the quantiser itself
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
  if (e != cudaSuccess) {
    cudaGetLastError();
    zib_set_error("%s: launch failed: %s", what, cudaGetErrorString(e));
    return ZIB_ERR_LAUNCH;
  }
  return ZIB_OK;
}

template <typename T>
static int small(const SmallParams& p, bool fused, cudaStream_t st, const char* what) {
  return fused ? launch_small<T, true>(p, st, what) : launch_small<T, false>(p, st, what);
}

// This kernel or the tcgen05 product.  One group of tokens is a stream over the weight: always here.  With
// more groups a call takes about 8 us and 1 us per 2400 blocks (16 weight rows x 128 columns x 8
// tokens; a CTA costs as much as 8 of them) here, and 11 us and 1 us per 3 blocks of K there, as long as
// its tiles fill one wave.  Quantiser included, here / there: 640 x 4096, 128 tokens 17.3 / 21.2 us, 256
// tokens 25.1 / 21.5; 128 x 16384, 256 tokens 20.6 / 52.2; 11520 x 3840, 9 tokens 27.1 / 23.6; 768 x
// 256, 64 tokens 9.7 / 11.5.
static bool is_small(int64_t M, int64_t N, int64_t kb) {
  const int64_t ctas = ceil_div(M, kMaxTokens) * ceil_div(N, kTileN);
  return M <= kMaxTokens || ctas * (kb > 8 ? kb : 8) < 7200 + 800 * kb;
}

static bool is_fused(int64_t M, int64_t kb) { return M <= kFusedTokens && fused_smem(kb) <= kFusedSmem; }

}  // namespace fp8
}  // namespace zib

using namespace zib;

// scratch: quantised rows, their scales, and where the column sums are wanted their parts
struct Scratch {
  int64_t scales, part, bytes;
};

static Scratch scratch_of(int64_t M, int64_t K, bool sum) {
  const int64_t kb = ceil_div(K, fp8::kBlock);
  Scratch s{};
  if (!sum && fp8::is_fused(M, kb)) return s;
  s.scales = ceil_div(M * ceil_div(K, 16) * 16, 128) * 128;
  s.part = s.scales + ceil_div(kb * M * 4, 128) * 128;
  s.bytes = s.part + (sum ? fp8_sum_rows(M) * K * 4 : 0);
  return s;
}

extern "C" int64_t zib_fp8_block_linear_scratch(int64_t M, int64_t K, int with_sum) {
  return M < 1 || K < 1 || K >= (1ll << 31) ? 0 : scratch_of(M, K, with_sum != 0).bytes;
}

extern "C" int zib_fp8_block_linear(const void* x, int64_t ldx, int dtype, const void* w, int64_t ldw, const float* sw,
                                    int64_t sw_n, int64_t sw_k, const void* bias, void* y, int64_t ldy, void* sum,
                                    void* scratch, int64_t nscratch, int64_t M, int64_t N, int64_t K, void* stream) {
  const char* what = "zib_fp8_block_linear";
  ZIB_HOST_CHECK(known_dtype(dtype), ZIB_ERR_INVALID_ARG, "%s: unknown dtype %d", what, dtype);
  ZIB_HOST_CHECK(M >= 0 && N >= 1 && K >= 1 && ldx >= K && ldw >= K && ldy >= N, ZIB_ERR_INVALID_ARG,
                 "%s: bad shape M=%lld N=%lld K=%lld", what, (long long)M, (long long)N, (long long)K);
  ZIB_HOST_CHECK(M < (1ll << 31) - 512 && N < (1ll << 31) - 512 && K < (1ll << 31) - 512, ZIB_ERR_TOO_LARGE,
                 "%s: M=%lld N=%lld K=%lld", what, (long long)M, (long long)N, (long long)K);
  ZIB_HOST_CHECK(ldw % 16 == 0 && (uintptr_t)w % 16 == 0, ZIB_ERR_ALIGNMENT, "%s: w needs 16-byte aligned rows", what);
  cudaStream_t st = (cudaStream_t)stream;
  if (M == 0) {
    if (sum) fp8_sum_finish(nullptr, sum, dtype, 0, K, st);
    return sum ? zib_check_launch(what) : ZIB_OK;
  }
  ZIB_HOST_CHECK(x && w && sw && y, ZIB_ERR_INVALID_ARG, "%s: null operand", what);
  const int64_t kb = ceil_div(K, fp8::kBlock), ldq = ceil_div(K, 16) * 16;
  const Scratch sc = scratch_of(M, K, sum != nullptr);
  float* s = nullptr;
  if (sc.bytes) {
    ZIB_HOST_CHECK(scratch && nscratch >= sc.bytes && (uintptr_t)scratch % 128 == 0, ZIB_ERR_INVALID_ARG,
                   "%s: scratch of %lld bytes, 128-byte aligned, needed", what, (long long)sc.bytes);
    s = (float*)((uint8_t*)scratch + sc.scales);
    float* part = sum ? (float*)((uint8_t*)scratch + sc.part) : nullptr;
    const int rc = fp8_quant_rows(x, ldx, dtype, scratch, ldq, s, 1, M, part, M, K, st, what);
    if (rc) return rc;
    if (sum) fp8_sum_finish(part, sum, dtype, M, K, st);
  }
  if (!fp8::is_small(M, N, kb))
    return fp8_gemm(scratch, ldq, s, 1, M, w, ldw, sw, sw_n, sw_k, bias, y, ldy, dtype, M, N, K, true, true, st,
                    what);
  const bool fused = sc.bytes == 0;
  const int size = dtype_bytes(dtype);
  fp8::SmallParams p{};
  p.x = fused ? x : scratch; p.ldx = fused ? ldx : ldq; p.sx = s;
  p.w = (const uint8_t*)w; p.ldw = ldw; p.sw = sw; p.sw_n = sw_n; p.sw_k = sw_k;
  p.bias = bias; p.y = y; p.ldy = ldy;
  p.M = (int)M; p.N = (int)N; p.K = (int)K; p.kb = (int)kb;
  p.vec = K % 8 == 0 && (uintptr_t)x % 16 == 0 && (ldx * size % 16 == 0 || M == 1);
  if (dtype == ZIB_BF16) return fp8::small<__nv_bfloat16>(p, fused, st, what);
  if (dtype == ZIB_F16) return fp8::small<__half>(p, fused, st, what);
  return fp8::small<float>(p, fused, st, what);
}
