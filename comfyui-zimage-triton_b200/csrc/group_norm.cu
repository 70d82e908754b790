// Group normalisation with an activation over channels-last tensors, forward and backward.
//
// x [B, P, C], C channels in G groups of D = C / G; statistics over the n = P D values of a batch
// entry's group:
//   mu = sum x / n,  v = sum (x - mu)^2 / n,  r = 1 / sqrt(v + eps),  h = (x - mu) r
//   z = h w_c + b_c,  y = act(z)
// and, with g = dy act'(z), A_c = sum_p g, E_c = sum_p g h:
//   db = sum_b A_c,  dw = sum_b E_c,
//   dx = r (w_c g - c1 - h c2),  c1 = sum_c w_c A_c / n,  c2 = sum_c w_c E_c / n over the group.
//
// Bound by memory: the floor is x in and y out (forward), x and dy in and dx out (backward); the
// statistics need every value before the first output.
//
// Sums.  Runs of a few values of one group are reduced in fp32 to their sum S and their squared
// deviations from their own mean M; runs meet in fp64 as (sum S, sum M + S^2 / n_run), so a mean
// that is large against the spread costs no precision.  All sums have a fixed order (no atomics).
#include "zib_async.cuh"
#include "zib_types.cuh"

namespace zib {
namespace gn {

constexpr int kThreads = 256;
constexpr int kMaxChannels = 8192;  // one pixel's partial sums fit shared memory

struct Params {
  const void* x;
  int64_t xsb, xsp;  // element strides of batch entry and pixel
  const void* dy;
  int64_t dsb, dsp;
  void* out;  // y or dx, contiguous
  const void* w;
  const void* b;
  int wdtype;
  void* dw;
  void* db;
  float* mean;  // [B, G]
  float* rstd;
  double2* part;    // forward: [B, chunks, G] (sum x, sum x^2); backward: [B, chunks, C] (A, E) as float2
  float2* coef;     // backward: [B, G] (c1, c2)
  int64_t B, P;
  int C, G, cpg;
  int V;            // columns of VEC channels
  int vlanes, rows; // threads: vlanes columns x rows pixels
  int chunks;
  int64_t chunk;    // pixels per chunk
  int act;
  float eps;
};

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_down_sync(0xFFFFFFFFu, v, o);
  return v;
}

// --- statistics of the forward pass ----------------------------------------------

// GV consecutive channels of a thread share a group (GV divides VEC); RUN pixels per run.
template <typename T, int VEC, int GV, int RUN>
__global__ void __launch_bounds__(kThreads) stats_kernel(const Params p) {
  constexpr int NA = VEC / GV;
  using V = Pack<T, VEC>;
  extern __shared__ double2 sm[];  // [rows][V * NA]
  const int64_t b = blockIdx.y;
  const int vl = threadIdx.x % p.vlanes, r = threadIdx.x / p.vlanes;
  const int64_t p0 = (int64_t)blockIdx.x * p.chunk;
  const int64_t p1 = p0 + p.chunk < p.P ? p0 + p.chunk : p.P;
  const T* x = reinterpret_cast<const T*>(p.x) + b * p.xsb;
  if (r < p.rows) {
    for (int v = vl; v < p.V; v += p.vlanes) {
      double s[NA], q[NA];
#pragma unroll
      for (int a = 0; a < NA; ++a) s[a] = q[a] = 0.0;
      int64_t i = p0 + r;
      for (; i + (int64_t)(RUN - 1) * p.rows < p1; i += (int64_t)RUN * p.rows) {
        V t[RUN];
#pragma unroll
        for (int k = 0; k < RUN; ++k)
          t[k] = *reinterpret_cast<const V*>(x + (i + (int64_t)k * p.rows) * p.xsp + (int64_t)v * VEC);
#pragma unroll
        for (int a = 0; a < NA; ++a) {
          float sum = 0.0f;
#pragma unroll
          for (int k = 0; k < RUN; ++k)
#pragma unroll
            for (int j = 0; j < GV; ++j) sum += to_f32(t[k].v[a * GV + j]);
          const float m = sum * (1.0f / (RUN * GV));
          float dev = 0.0f;
#pragma unroll
          for (int k = 0; k < RUN; ++k)
#pragma unroll
            for (int j = 0; j < GV; ++j) {
              const float d = to_f32(t[k].v[a * GV + j]) - m;
              dev = fmaf(d, d, dev);
            }
          // sum (x - m)^2 + 2 m sum - n m^2 for the rounded m, exact in fp64 but for its last bits
          const double dm = m, ds = sum;
          s[a] += ds;
          q[a] += (double)dev + dm * (2.0 * ds - dm * (double)(RUN * GV));
        }
      }
      for (; i < p1; i += p.rows) {
        const V t = *reinterpret_cast<const V*>(x + i * p.xsp + (int64_t)v * VEC);
#pragma unroll
        for (int a = 0; a < NA; ++a)
#pragma unroll
          for (int j = 0; j < GV; ++j) {
            const double d = to_f32(t.v[a * GV + j]);
            s[a] += d;
            q[a] = fma(d, d, q[a]);
          }
      }
#pragma unroll
      for (int a = 0; a < NA; ++a) sm[(int64_t)r * p.V * NA + v * NA + a] = make_double2(s[a], q[a]);
    }
  }
  __syncthreads();
  // a warp per group: its columns of every thread row, in a fixed order
  const int cols = p.cpg / GV;  // accumulators per group and row
  for (int g = threadIdx.x >> 5; g < p.G; g += kThreads / 32) {
    double s = 0.0, q = 0.0;
    for (int k = threadIdx.x & 31; k < cols * p.rows; k += 32) {
      const double2 d = sm[(int64_t)(k / cols) * p.V * NA + g * cols + k % cols];
      s += d.x;
      q += d.y;
    }
    s = warp_sum(s);
    q = warp_sum(q);
    if ((threadIdx.x & 31) == 0) p.part[(b * p.chunks + blockIdx.x) * p.G + g] = make_double2(s, q);
  }
}

// one warp per (batch entry, group): partial sums to mean and 1 / sqrt(var + eps)
__global__ void __launch_bounds__(kThreads) finish_stats_kernel(const Params p) {
  const int64_t id = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  if (id >= p.B * p.G) return;
  const int64_t b = id / p.G, g = id - b * p.G;
  double s = 0.0, q = 0.0;
  for (int k = threadIdx.x & 31; k < p.chunks; k += 32) {
    const double2 d = p.part[(b * p.chunks + k) * p.G + g];
    s += d.x;
    q += d.y;
  }
  s = warp_sum(s);
  q = warp_sum(q);
  if ((threadIdx.x & 31) == 0) {
    const double n = (double)p.P * (double)p.cpg;
    const double m = s / n;
    double var = q / n - m * m;
    if (var < 0.0) var = 0.0;
    p.mean[id] = (float)m;
    p.rstd[id] = (float)(1.0 / sqrt(var + (double)p.eps));
  }
}

// --- activation ------------------------------------------------------------------

// 1 / (1 + e^-z): the fast exponential and division where the result is rounded to 16 bits, the
// accurate ones where it is kept in 32
template <typename T>
__device__ __forceinline__ float sigmoid(float z) {
  if constexpr (sizeof(T) == 2) return __fdividef(1.0f, 1.0f + __expf(-z));
  else return 1.0f / (1.0f + expf(-z));
}

template <typename T>
__device__ __forceinline__ float activate(float z, int act) {
  return act == ZIB_ACT_SILU ? z * sigmoid<T>(z) : z;
}

// act'(z)
template <typename T>
__device__ __forceinline__ float slope(float z, int act) {
  if (act != ZIB_ACT_SILU) return 1.0f;
  const float s = sigmoid<T>(z);
  return s * fmaf(z, 1.0f - s, 1.0f);
}

// per-thread constants of VEC channels from channel c0 of batch entry b
template <int VEC>
struct Affine {
  float mu[VEC], r[VEC], w[VEC], b[VEC];
  __device__ __forceinline__ void load(const Params& p, int64_t bi, int c0) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const int c = c0 + j;
      const int64_t g = bi * p.G + c / p.cpg;
      mu[j] = p.mean[g];
      r[j] = p.rstd[g];
      w[j] = p.w ? load_as_f32(p.w, p.wdtype, c) : 1.0f;
      b[j] = p.b ? load_as_f32(p.b, p.wdtype, c) : 0.0f;
    }
  }
};

template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads) apply_kernel(const Params p) {
  using V = Pack<T, VEC>;
  const int64_t b = blockIdx.y;
  const int vl = threadIdx.x % p.vlanes, r = threadIdx.x / p.vlanes;
  if (r >= p.rows) return;
  // last pixels first: the statistics pass read them last, so they are the ones still in L2
  const int64_t p0 = (int64_t)(gridDim.x - 1 - blockIdx.x) * p.chunk;
  const int64_t p1 = p0 + p.chunk < p.P ? p0 + p.chunk : p.P;
  const T* x = reinterpret_cast<const T*>(p.x) + b * p.xsb;
  T* y = reinterpret_cast<T*>(p.out) + b * p.P * p.C;
  for (int v = vl; v < p.V; v += p.vlanes) {
    Affine<VEC> f;
    f.load(p, b, v * VEC);
#pragma unroll 4
    for (int64_t i = p0 + r; i < p1; i += p.rows) {
      const V t = *reinterpret_cast<const V*>(x + i * p.xsp + (int64_t)v * VEC);
      V o;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float h = (to_f32(t.v[j]) - f.mu[j]) * f.r[j];
        o.v[j] = from_f32<T>(activate<T>(fmaf(h, f.w[j], f.b[j]), p.act));
      }
      *reinterpret_cast<V*>(y + i * p.C + (int64_t)v * VEC) = o;
    }
  }
}

// --- backward --------------------------------------------------------------------

// A_c and E_c of one chunk of pixels
template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads) grad_stats_kernel(const Params p) {
  using V = Pack<T, VEC>;
  extern __shared__ double2 sm[];
  float2* sf = reinterpret_cast<float2*>(sm);  // [rows][vlanes * VEC]
  const int64_t b = blockIdx.y;
  const int vl = threadIdx.x % p.vlanes, r = threadIdx.x / p.vlanes;
  const int64_t p0 = (int64_t)blockIdx.x * p.chunk;
  const int64_t p1 = p0 + p.chunk < p.P ? p0 + p.chunk : p.P;
  const T* x = reinterpret_cast<const T*>(p.x) + b * p.xsb;
  const T* dy = reinterpret_cast<const T*>(p.dy) + b * p.dsb;
  float2* part = reinterpret_cast<float2*>(p.part) + (b * p.chunks + blockIdx.x) * p.C;
  const int width = p.vlanes * VEC;
  for (int v0 = 0; v0 < p.V; v0 += p.vlanes) {
    const int v = v0 + vl;
    if (r < p.rows && v < p.V) {
      Affine<VEC> f;
      f.load(p, b, v * VEC);
      float A[VEC], E[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) A[j] = E[j] = 0.0f;
#pragma unroll 2
      for (int64_t i = p0 + r; i < p1; i += p.rows) {
        const V t = *reinterpret_cast<const V*>(x + i * p.xsp + (int64_t)v * VEC);
        const V d = *reinterpret_cast<const V*>(dy + i * p.dsp + (int64_t)v * VEC);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float h = (to_f32(t.v[j]) - f.mu[j]) * f.r[j];
          const float g = to_f32(d.v[j]) * slope<T>(fmaf(h, f.w[j], f.b[j]), p.act);
          A[j] += g;
          E[j] = fmaf(g, h, E[j]);
        }
      }
#pragma unroll
      for (int j = 0; j < VEC; ++j) sf[r * width + vl * VEC + j] = make_float2(A[j], E[j]);
    }
    __syncthreads();
    for (int c = threadIdx.x; c < width && v0 * VEC + c < p.C; c += kThreads) {
      double A = 0.0, E = 0.0;
      for (int k = 0; k < p.rows; ++k) {
        const float2 s = sf[k * width + c];
        A += s.x;
        E += s.y;
      }
      part[v0 * VEC + c] = make_float2((float)A, (float)E);
    }
    __syncthreads();
  }
}

// one CTA per group: its channels' sums over chunks, c1 and c2 per batch entry, dw and db
__global__ void __launch_bounds__(kThreads) finish_grad_kernel(const Params p) {
  __shared__ double red[2][kThreads / 32];
  const int g = blockIdx.x;
  const float2* part = reinterpret_cast<const float2*>(p.part);
  const double n = (double)p.P * (double)p.cpg;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // c1, c2
  if (p.coef) {
    for (int64_t b = 0; b < p.B; ++b) {
      double s1 = 0.0, s2 = 0.0;
      for (int64_t k = threadIdx.x; k < (int64_t)p.chunks * p.cpg; k += kThreads) {
        const int c = g * p.cpg + (int)(k % p.cpg);
        const float2 a = part[(b * p.chunks + k / p.cpg) * p.C + c];
        const double w = p.w ? (double)load_as_f32(p.w, p.wdtype, c) : 1.0;
        s1 += w * a.x;
        s2 += w * a.y;
      }
      s1 = warp_sum(s1);
      s2 = warp_sum(s2);
      if (lane == 0) { red[0][warp] = s1; red[1][warp] = s2; }
      __syncthreads();
      if (threadIdx.x == 0) {
        double t1 = 0.0, t2 = 0.0;
        for (int k = 0; k < kThreads / 32; ++k) { t1 += red[0][k]; t2 += red[1][k]; }
        p.coef[b * p.G + g] = make_float2((float)(t1 / n), (float)(t2 / n));
      }
      __syncthreads();
    }
  }
  if (!p.dw && !p.db) return;
  for (int c = g * p.cpg + warp; c < (g + 1) * p.cpg; c += kThreads / 32) {
    double A = 0.0, E = 0.0;
    for (int64_t k = lane; k < p.B * p.chunks; k += 32) {
      const float2 a = part[k * p.C + c];
      A += a.x;
      E += a.y;
    }
    A = warp_sum(A);
    E = warp_sum(E);
    if (lane == 0) {
      if (p.db) store_as(p.db, p.wdtype, c, (float)A);
      if (p.dw) store_as(p.dw, p.wdtype, c, (float)E);
    }
  }
}

template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads) grad_apply_kernel(const Params p) {
  using V = Pack<T, VEC>;
  const int64_t b = blockIdx.y;
  const int vl = threadIdx.x % p.vlanes, r = threadIdx.x / p.vlanes;
  if (r >= p.rows) return;
  const int64_t p0 = (int64_t)(gridDim.x - 1 - blockIdx.x) * p.chunk;
  const int64_t p1 = p0 + p.chunk < p.P ? p0 + p.chunk : p.P;
  const T* x = reinterpret_cast<const T*>(p.x) + b * p.xsb;
  const T* dy = reinterpret_cast<const T*>(p.dy) + b * p.dsb;
  T* dx = reinterpret_cast<T*>(p.out) + b * p.P * p.C;
  for (int v = vl; v < p.V; v += p.vlanes) {
    Affine<VEC> f;
    f.load(p, b, v * VEC);
    float c1[VEC], c2[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const float2 c = p.coef[b * p.G + (v * VEC + j) / p.cpg];
      c1[j] = c.x;
      c2[j] = c.y;
    }
#pragma unroll 2
    for (int64_t i = p0 + r; i < p1; i += p.rows) {
      const V t = *reinterpret_cast<const V*>(x + i * p.xsp + (int64_t)v * VEC);
      const V d = *reinterpret_cast<const V*>(dy + i * p.dsp + (int64_t)v * VEC);
      V o;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float h = (to_f32(t.v[j]) - f.mu[j]) * f.r[j];
        const float g = to_f32(d.v[j]) * slope<T>(fmaf(h, f.w[j], f.b[j]), p.act);
        o.v[j] = from_f32<T>(f.r[j] * (fmaf(f.w[j], g, -c1[j]) - h * c2[j]));
      }
      *reinterpret_cast<V*>(dx + i * p.C + (int64_t)v * VEC) = o;
    }
  }
}

// --- host ------------------------------------------------------------------------

static int gcd(int a, int b) {
  while (b) { const int t = a % b; a = b; b = t; }
  return a;
}

// Splits P pixels into chunks: about four CTAs per SM over the batch, at least 8 pixels per thread.
static void plan(Params& p, int vec) {
  p.V = p.C / vec;
  p.vlanes = p.V < kThreads ? p.V : kThreads;
  p.rows = kThreads / p.vlanes;
  int64_t chunks = ceil_div((int64_t)sm_count() * 4, p.B);
  const int64_t most = ceil_div(p.P, (int64_t)p.rows * 8);
  if (chunks > most) chunks = most;
  if (chunks < 1) chunks = 1;
  p.chunk = ceil_div(p.P, chunks);
  p.chunks = (int)ceil_div(p.P, p.chunk);
}

template <typename T, int VEC, int GV>
static int launch_stats(const Params& p, cudaStream_t st) {
  constexpr int RUN = sizeof(T) == 2 ? 4 : 4;
  const size_t smem = (size_t)p.rows * p.V * (VEC / GV) * sizeof(double2);
  static bool set[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (smem > 48 * 1024 && dev >= 0 && dev < 64 && !set[dev]) {
    if (cudaFuncSetAttribute(stats_kernel<T, VEC, GV, RUN>, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024) !=
        cudaSuccess)
      return zib_check_launch("zib_group_norm");
    set[dev] = true;
  }
  stats_kernel<T, VEC, GV, RUN><<<dim3(p.chunks, (unsigned)p.B), kThreads, smem, st>>>(p);
  return ZIB_OK;
}

template <typename T, int VEC>
static int forward_v(const Params& p, cudaStream_t st) {
  int rc = ZIB_OK;
  const int gv = gcd(p.cpg, VEC);
  if (gv == 8) { if constexpr (VEC == 8) rc = launch_stats<T, VEC, 8>(p, st); }
  else if (gv == 4) { if constexpr (VEC >= 4) rc = launch_stats<T, VEC, 4>(p, st); }
  else if (gv == 2) { if constexpr (VEC >= 2) rc = launch_stats<T, VEC, 2>(p, st); }
  else rc = launch_stats<T, VEC, 1>(p, st);
  if (rc) return rc;
  finish_stats_kernel<<<(unsigned)ceil_div(p.B * p.G, kThreads / 32), kThreads, 0, st>>>(p);
  apply_kernel<T, VEC><<<dim3(p.chunks, (unsigned)p.B), kThreads, 0, st>>>(p);
  return zib_check_launch("zib_group_norm");
}

template <typename T, int VEC>
static int backward_v(const Params& p, cudaStream_t st) {
  const size_t smem = (size_t)p.rows * p.vlanes * VEC * sizeof(float2);
  grad_stats_kernel<T, VEC><<<dim3(p.chunks, (unsigned)p.B), kThreads, smem, st>>>(p);
  finish_grad_kernel<<<(unsigned)p.G, kThreads, 0, st>>>(p);
  if (p.out) grad_apply_kernel<T, VEC><<<dim3(p.chunks, (unsigned)p.B), kThreads, 0, st>>>(p);
  return zib_check_launch("zib_group_norm_backward");
}

static int check(const Params& p, int64_t C, int64_t G, int dtype, const char* what) {
  ZIB_HOST_CHECK(known_dtype(dtype) && known_dtype(p.wdtype), ZIB_ERR_INVALID_ARG, "%s: unknown dtype", what);
  ZIB_HOST_CHECK(p.B >= 0 && p.P >= 0 && C >= 1 && G >= 1 && C % G == 0, ZIB_ERR_INVALID_ARG,
                 "%s: %lld channels in %lld groups", what, (long long)C, (long long)G);
  ZIB_HOST_CHECK(C <= kMaxChannels && p.B <= 65535, ZIB_ERR_TOO_LARGE,
                 "%s: at most %d channels and 65535 batch entries", what, kMaxChannels);
  ZIB_HOST_CHECK(p.act == ZIB_ACT_NONE || p.act == ZIB_ACT_SILU, ZIB_ERR_INVALID_ARG, "%s: unknown activation %d",
                 what, p.act);
  ZIB_HOST_CHECK(p.eps >= 0.0f, ZIB_ERR_INVALID_ARG, "%s: eps must not be negative", what);
  return ZIB_OK;
}

// whole 16-byte accesses where channels, strides and addresses allow them, else single elements
static bool vector_ok(const Params& p, int size) {
  const int v = 16 / size;
  auto ok = [&](const void* x, int64_t sb, int64_t sp) {
    return !x || ((uintptr_t)x % 16 == 0 && (sb % v == 0 || p.B == 1) && (sp % v == 0 || p.P == 1));
  };
  return p.C % v == 0 && ok(p.x, p.xsb, p.xsp) && ok(p.dy, p.dsb, p.dsp) && ok(p.out, 0, 0);
}

}  // namespace gn
}  // namespace zib

using namespace zib;

// chunks a launch may use at most, whatever vector width it takes
static int64_t most_chunks(int64_t B, int64_t P) {
  if (B < 1 || P < 1) return 1;
  const int64_t c = ceil_div((int64_t)sm_count() * 4, B), m = ceil_div(P, 8);
  return c < m ? c : m;
}

extern "C" int64_t zib_group_norm_workspace(int64_t B, int64_t P, int64_t C, int64_t G, int backward) {
  if (B < 0 || P < 0 || C < 1 || G < 1) return 0;
  const int64_t n = B * most_chunks(B, P);
  return backward ? n * C * (int64_t)sizeof(float2) + B * G * (int64_t)sizeof(float2)
                  : n * G * (int64_t)sizeof(double2);
}

extern "C" int zib_group_norm(const void* x, int64_t xsb, int64_t xsp, void* y, const void* w, const void* b,
                              int wdtype, float* mean, float* rstd, void* workspace, int64_t workspace_bytes,
                              int64_t B, int64_t P, int64_t C, int64_t G, int dtype, float eps, int act,
                              void* stream) {
  const char* what = "zib_group_norm";
  gn::Params p{};
  p.x = x; p.xsb = xsb; p.xsp = xsp; p.out = y; p.w = w; p.b = b; p.wdtype = wdtype;
  p.mean = mean; p.rstd = rstd; p.part = (double2*)workspace;
  p.B = B; p.P = P; p.act = act; p.eps = eps;
  int rc = gn::check(p, C, G, dtype, what);
  if (rc) return rc;
  if (B == 0 || P == 0) return ZIB_OK;
  ZIB_HOST_CHECK(x && y && mean && rstd && workspace, ZIB_ERR_INVALID_ARG, "%s: null operand", what);
  ZIB_HOST_CHECK(workspace_bytes >= zib_group_norm_workspace(B, P, C, G, 0) && (uintptr_t)workspace % 16 == 0,
                 ZIB_ERR_INVALID_ARG, "%s: workspace of %lld bytes, 16-byte aligned, needed", what,
                 (long long)zib_group_norm_workspace(B, P, C, G, 0));
  p.C = (int)C; p.G = (int)G; p.cpg = (int)(C / G);
  cudaStream_t st = (cudaStream_t)stream;
  const bool vec = gn::vector_ok(p, dtype_bytes(dtype));
  gn::plan(p, vec ? 16 / dtype_bytes(dtype) : 1);
  if (dtype == ZIB_BF16)
    return vec ? gn::forward_v<__nv_bfloat16, 8>(p, st) : gn::forward_v<__nv_bfloat16, 1>(p, st);
  if (dtype == ZIB_F16) return vec ? gn::forward_v<__half, 8>(p, st) : gn::forward_v<__half, 1>(p, st);
  return vec ? gn::forward_v<float, 4>(p, st) : gn::forward_v<float, 1>(p, st);
}

extern "C" int zib_group_norm_backward(const void* x, int64_t xsb, int64_t xsp, const void* dy, int64_t dsb,
                                       int64_t dsp, void* dx, const void* w, const void* b, int wdtype, void* dw,
                                       void* db, const float* mean, const float* rstd, void* workspace,
                                       int64_t workspace_bytes, int64_t B, int64_t P, int64_t C, int64_t G, int dtype,
                                       int act, void* stream) {
  const char* what = "zib_group_norm_backward";
  gn::Params p{};
  p.x = x; p.xsb = xsb; p.xsp = xsp; p.dy = dy; p.dsb = dsb; p.dsp = dsp; p.out = dx;
  p.w = w; p.b = b; p.wdtype = wdtype; p.dw = dw; p.db = db;
  p.mean = const_cast<float*>(mean); p.rstd = const_cast<float*>(rstd);
  p.B = B; p.P = P; p.act = act;
  int rc = gn::check(p, C, G, dtype, what);
  if (rc) return rc;
  ZIB_HOST_CHECK(B > 0 && P > 0, ZIB_ERR_INVALID_ARG, "%s: empty input", what);
  ZIB_HOST_CHECK(x && dy && mean && rstd && workspace, ZIB_ERR_INVALID_ARG, "%s: null operand", what);
  ZIB_HOST_CHECK(workspace_bytes >= zib_group_norm_workspace(B, P, C, G, 1) && (uintptr_t)workspace % 16 == 0,
                 ZIB_ERR_INVALID_ARG, "%s: workspace of %lld bytes, 16-byte aligned, needed", what,
                 (long long)zib_group_norm_workspace(B, P, C, G, 1));
  p.C = (int)C; p.G = (int)G; p.cpg = (int)(C / G);
  p.part = (double2*)workspace;
  p.coef = dx ? (float2*)((char*)workspace + B * most_chunks(B, P) * C * sizeof(float2)) : nullptr;
  cudaStream_t st = (cudaStream_t)stream;
  const bool vec = gn::vector_ok(p, dtype_bytes(dtype));
  gn::plan(p, vec ? 16 / dtype_bytes(dtype) : 1);
  if (dtype == ZIB_BF16)
    return vec ? gn::backward_v<__nv_bfloat16, 8>(p, st) : gn::backward_v<__nv_bfloat16, 1>(p, st);
  if (dtype == ZIB_F16) return vec ? gn::backward_v<__half, 8>(p, st) : gn::backward_v<__half, 1>(p, st);
  return vec ? gn::backward_v<float, 4>(p, st) : gn::backward_v<float, 1>(p, st);
}
