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
// statistics need every value before the first output, so what does not stay in L2 between the two
// passes is read twice.  The second pass walks each CTA's pixels backwards: the ones read last are
// the ones still in L2.  [1, 1048576, 128] bf16 with SiLU: 60 us for the statistics (4.5 TB/s) and 102 us
// for the outputs (5.3 TB/s; torch's copy of as many bytes takes 98 us).
//
// Launches.  Clusters of 8 CTAs sum their pixels and join the sums through distributed shared memory.
// Where one cluster holds a batch entry (a small tensor, where launches are what costs) it goes on to
// the outputs: one launch.  Elsewhere the sums of the clusters go through memory and the second
// launch adds them up in its first instructions (up to kDirectGroups groups; beyond, a small kernel
// between the two does that once).  Dependent launches start early and wait for the one before them.
//
// Sums.  A thread subtracts a value of its own group first (the mean of its first pixel's channels),
// adds the differences and their squares in fp32 over 16 pixels at most and joins them in fp64, so a mean that
// is large against the spread costs no precision.  A thread adds the backward sums A and E in fp32 over
// kGradRun pixels at most (more CTAs where there are more pixels) and joins them in fp64; a CTA's sum and
// the sum of a cluster's eight are rounded to fp32 on their way to the next fp64 sum.  All sums have a fixed
// order (no atomics).
//
// Arithmetic is on packed pairs (f32x2): at 12 elements per clock and SM, the rate of HBM, single
// operations left the SMs short of issue slots (79 us instead of 58 for the statistics of
// [1, 1048576, 128]).
#include "zib_pairs.cuh"
#include "zib_tcgen05.cuh"

namespace zib {
namespace gn {

constexpr int kThreads = 256;
constexpr int kCluster = 8;
constexpr int kMaxChannels = 8192;  // one pixel's partial sums fit shared memory
constexpr int kDirectGroups = 64;   // groups whose partial sums every CTA of the second pass adds itself
constexpr int kMaxSmem = 232448;
// Pixels whose gradient terms a thread adds in fp32: terms of one sign err by 2^-15 of their sum at worst.
// fp64 sums beside them, every 64 pixels, spilled registers: [2, 16384, 512] backward 58 -> 66 us.
constexpr int kGradRun = 512;

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
  double2* gpart;  // [B, clusters, G]: (sum x, sum x^2) or (sum w A, sum w E)
  float2* cpart;   // backward: [B, clusters, C]: (A, E)
  float2* coef;    // backward: [B, G]: (c1, c2)
  int64_t B, P;
  int64_t b0;  // first batch entry of the launch
  int C, G, cpg;
  int V;             // columns of VEC channels
  int vlanes, rows;  // threads: vlanes columns x rows pixels
  int clusters;      // per batch entry
  int chunks;        // CTAs per batch entry (kCluster * clusters in the first pass)
  int64_t chunk;     // pixels per CTA
  int act;
  int direct;        // the second pass adds the clusters' sums itself
  float eps;
};

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}

// all threads of the cluster (whose warps need not have converged)
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}

__device__ __forceinline__ double2 ld_cluster(const double2* p, uint32_t rank) {
  const uint32_t a = tc::mapa_rank(smem_u32(p), rank);
  double2 v;
  asm volatile("ld.shared::cluster.v2.f64 {%0, %1}, [%2];" : "=d"(v.x), "=d"(v.y) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ float2 ld_cluster(const float2* p, uint32_t rank) {
  const uint32_t a = tc::mapa_rank(smem_u32(p), rank);
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(a) : "memory");
  return v;
}

// a dependent launch may start (it still waits for this grid's memory), and that wait
__device__ __forceinline__ void allow_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_primary() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

using px::f2;

// --- activation ------------------------------------------------------------------

// 1 / (1 + e^-z): the accurate functions where x, and so the outputs, have 32 bits; where they have 16, the fast
// power of two and reciprocal, off by about 2^-22 + 2^-23 + |z| 2^-24 of the value (two functions, the rounded
// exponent) at worst and 0 below 2^-126.  That is 2^-13 of a 16-bit step, and what the gradients of 32-bit parameters, sums
// over such terms, then carry.
template <typename T>
__device__ __forceinline__ f2 sigmoid(f2 z) {
  float a, b;
  if constexpr (sizeof(T) == 2) {
    px::split(px::mul(z, dup(-1.4426950408889634f)), a, b);
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(a));
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(b));
    px::split(px::add(px::mk(a, b), dup(1.0f)), a, b);
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(a));
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(b));
  } else {
    px::split(z, a, b);
    a = 1.0f / (1.0f + expf(-a));
    b = 1.0f / (1.0f + expf(-b));
  }
  return px::mk(a, b);
}

template <typename T>
__device__ __forceinline__ f2 activate(f2 z, int act) {
  return act == ZIB_ACT_SILU ? px::mul(z, sigmoid<T>(z)) : z;
}

// act'(z) = s (1 + z (1 - s))
template <typename T>
__device__ __forceinline__ f2 slope(f2 z, int act) {
  if (act != ZIB_ACT_SILU) return dup(1.0f);
  const f2 s = sigmoid<T>(z);
  return px::mul(s, px::fma(z, px::sub(dup(1.0f), s), dup(1.0f)));
}

// --- a thread's share of a CTA's pixels -------------------------------------------

struct Slab {
  int64_t b, p0, p1;  // batch entry, pixels [p0, p1)
  int vl, r;          // column lane, pixel row
  __device__ __forceinline__ Slab(const Params& p, int chunk) {
    b = p.b0 + blockIdx.y;
    vl = threadIdx.x % p.vlanes;
    r = threadIdx.x / p.vlanes;
    p0 = chunk * p.chunk;
    p1 = p0 + p.chunk < p.P ? p0 + p.chunk : p.P;
    if (p0 > p1) p0 = p1;
  }
};

// --- forward statistics --------------------------------------------------------------

// Sums by group, several threads to a group (as many as the CTA has, a power of two up to 32):
// part(g, first, step) is a thread's share, done(g, sum) gets the sum in one thread of the group.
// part is also called for g >= G, where it returns 0.
template <typename Part, typename Done>
__device__ __forceinline__ void by_group(int G, Part part, Done done) {
  int n = 32;
  while (n > 1 && n * G > (int)blockDim.x) n >>= 1;
  const int per_pass = (int)blockDim.x / n, lane = (int)threadIdx.x % n;
  for (int g0 = 0; g0 < G; g0 += per_pass) {
    const int g = g0 + (int)threadIdx.x / n;
    double2 d = part(g, lane, n);
    for (int o = n >> 1; o > 0; o >>= 1) {
      d.x += __shfl_xor_sync(0xFFFFFFFFu, d.x, o);
      d.y += __shfl_xor_sync(0xFFFFFFFFu, d.y, o);
    }
    if (lane == 0 && g < G) done(g, d);
  }
}

// The sums of this CTA's pixels by group into sm[0 .. G) (sum x, sum x^2); scratch behind them.  GV
// consecutive channels of a thread share a group; RUN pixels are in flight at a time.
template <typename T, int VEC, int GV>
__device__ __forceinline__ void slab_stats(const Params& p, const Slab& s, double2* sm) {
  constexpr int NA = VEC / GV, NP = kPairs<VEC>, RUN = NA > 2 ? 8 : 16;
  using V = Pack<T, VEC>;
  const int cols = p.cpg / GV;  // sums per group and thread row
  // [rows][V * NA]; with one sum per group it is the result
  double2* scratch = cols * p.rows == 1 ? sm : sm + p.G;
  const T* x = reinterpret_cast<const T*>(p.x) + s.b * p.xsb;
  if (s.r < p.rows) {
    for (int v = s.vl; v < p.V; v += p.vlanes) {
      double sum[NA], sq[NA];
      float piv[NA];
#pragma unroll
      for (int a = 0; a < NA; ++a) {
        sum[a] = sq[a] = 0.0;
        piv[a] = 0.0f;
      }
      const T* xv = x + (int64_t)v * VEC;
      const int64_t p0 = s.p0 + s.r, step = p.rows * p.xsp;
      f2 pv[NP];
      const int n = s.p1 > p0 ? (int)((s.p1 - p0 + p.rows - 1) / p.rows) : 0;  // this thread's pixels
      const T* at = xv + p0 * p.xsp;
      for (int i = 0; i < n; i += RUN, at += RUN * step) {
        V t[RUN];
#pragma unroll
        for (int k = 0; k < RUN; ++k)
          if (i + k < n) t[k] = *reinterpret_cast<const V*>(at + k * step);
        if (i == 0) {
#pragma unroll
          for (int a = 0; a < NA; ++a) {
#pragma unroll
            for (int j = 0; j < GV; ++j) piv[a] += to_f32(t[0].v[a * GV + j]);
            piv[a] *= 1.0f / GV;
          }
#pragma unroll
          for (int j = 0; j < NP; ++j)
            pv[j] = VEC == 1 ? px::mk(piv[0], 0.0f) : px::mk(piv[2 * j / GV], piv[(2 * j + 1) / GV % NA]);
        }
        f2 u[NP], w[NP];
#pragma unroll
        for (int j = 0; j < NP; ++j) u[j] = w[j] = 0ull;
#pragma unroll
        for (int k = 0; k < RUN; ++k) {
          if (i + k >= n) break;
          f2 d[NP];
          unpack<T, VEC>(t[k], d);
#pragma unroll
          for (int j = 0; j < NP; ++j) {
            d[j] = px::sub(d[j], pv[j]);
            u[j] = px::add(u[j], d[j]);
            w[j] = px::fma(d[j], d[j], w[j]);
          }
        }
        float us[2 * NP], ws[2 * NP];
#pragma unroll
        for (int j = 0; j < NP; ++j) {
          px::split(u[j], us[2 * j], us[2 * j + 1]);
          px::split(w[j], ws[2 * j], ws[2 * j + 1]);
        }
#pragma unroll
        for (int a = 0; a < NA; ++a) {
#pragma unroll
          for (int j = 1; j < GV; ++j) {
            us[a * GV] += us[a * GV + j];
            ws[a * GV] += ws[a * GV + j];
          }
          sum[a] += (double)us[a * GV];
          sq[a] += (double)ws[a * GV];
        }
      }
      // back from the differences: sum x = sum d + n m, sum x^2 = sum d^2 + 2 m sum d + n m^2
#pragma unroll
      for (int a = 0; a < NA; ++a) {
        const double m = piv[a], nm = (double)n * GV * m;
        scratch[s.r * p.V * NA + v * NA + a] = make_double2(sum[a] + nm, sq[a] + m * (2.0 * sum[a] + nm));
      }
    }
  }
  if (scratch == sm) return;
  __syncthreads();
  // the group's columns of every thread row, in a fixed order
  by_group(p.G, [&](int g, int first, int step) {
    double a = 0.0, q = 0.0;
    if (g < p.G)
      for (int k = first; k < cols * p.rows; k += step) {
        const double2 d = scratch[(k / cols) * p.V * NA + g * cols + k % cols];
        a += d.x;
        q += d.y;
      }
    return make_double2(a, q);
  }, [&](int g, double2 d) { sm[g] = d; });
}

// the cluster's sum of element g of an array that each of its CTAs holds
template <typename D>
__device__ __forceinline__ D cluster_sum(const D* sm, int g) {
  D v[kCluster];
#pragma unroll
  for (int k = 0; k < kCluster; ++k) v[k] = ld_cluster(sm + g, k);
#pragma unroll
  for (int k = 1; k < kCluster; ++k) {
    v[0].x += v[k].x;
    v[0].y += v[k].y;
  }
  return v[0];
}

__device__ __forceinline__ void finish(const Params& p, double s, double q, float& mean, float& rstd) {
  const double n = (double)p.P * (double)p.cpg;
  const double m = s / n;
  double var = q / n - m * m;
  if (var < 0.0) var = 0.0;
  mean = (float)m;
  rstd = (float)(1.0 / sqrt(var + (double)p.eps));
}

// a thread's share of the clusters' sums of group g of batch entry b
__device__ __forceinline__ double2 cluster_share(const Params& p, int64_t b, int g, int first, int step) {
  double s = 0.0, q = 0.0;
  if (g < p.G) {
    const double2* at = p.gpart + b * p.clusters * p.G + g;
#pragma unroll 8
    for (int k = first; k < p.clusters; k += step) {
      const double2 d = __ldcg(at + (int64_t)k * p.G);
      s += d.x;
      q += d.y;
    }
  }
  return make_double2(s, q);
}

// the same by a whole warp
__device__ __forceinline__ double2 sum_clusters(const Params& p, int64_t b, int g) {
  const double2 d = cluster_share(p, b, g, threadIdx.x & 31, 32);
  return make_double2(warp_sum(d.x), warp_sum(d.y));
}

// --- outputs -----------------------------------------------------------------------

// N consecutive parameters from element c on, `missing` where there are none.  One branch on the type
// for all of them, so that the loads go out together (a branch per element, 16 loads one after the
// other, cost 5 us a launch).
template <int N, typename T>
__device__ __forceinline__ void load_typed(const T* p, float (&v)[N]) {
#pragma unroll
  for (int j = 0; j < N; ++j) v[j] = to_f32(p[j]);
}
template <int N>
__device__ __forceinline__ void load_params(const void* p, int dtype, int c, float missing, float (&v)[N]) {
  if (!p) {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = missing;
  } else if (dtype == ZIB_F32) {
    load_typed<N>(reinterpret_cast<const float*>(p) + c, v);
  } else if (dtype == ZIB_BF16) {
    load_typed<N>(reinterpret_cast<const __nv_bfloat16*>(p) + c, v);
  } else {
    load_typed<N>(reinterpret_cast<const __half*>(p) + c, v);
  }
}

// the group of each of VEC channels from c0 on
template <int VEC>
__device__ __forceinline__ void groups_of(const Params& p, int c0, int (&g)[VEC]) {
  g[0] = c0 / p.cpg;
  int left = p.cpg - (c0 - g[0] * p.cpg);  // channels of that group from c0 on
#pragma unroll
  for (int j = 1; j < VEC; ++j) {
    const bool next = --left == 0;
    g[j] = g[j - 1] + (next ? 1 : 0);
    if (next) left = p.cpg;
  }
}

// mean, 1 / sqrt(var + eps), weight and bias of VEC channels from channel c0; mean and rstd by group
template <int VEC>
struct Affine {
  f2 mu[kPairs<VEC>], r[kPairs<VEC>], w[kPairs<VEC>], b[kPairs<VEC>];
  __device__ __forceinline__ void load_params_of(const Params& p, int c0) {
    float wv[VEC], bv[VEC];
    load_params<VEC>(p.w, p.wdtype, c0, 1.0f, wv);
    load_params<VEC>(p.b, p.wdtype, c0, 0.0f, bv);
#pragma unroll
    for (int i = 0; i < kPairs<VEC>; ++i) {
      w[i] = px::mk(wv[2 * i], VEC == 1 ? 0.0f : wv[(2 * i + 1) % VEC]);
      b[i] = px::mk(bv[2 * i], VEC == 1 ? 0.0f : bv[(2 * i + 1) % VEC]);
    }
  }
  __device__ __forceinline__ void load_stats_of(const Params& p, const float* mean, const float* rstd, int c0) {
    int g[VEC];
    groups_of<VEC>(p, c0, g);
#pragma unroll
    for (int i = 0; i < kPairs<VEC>; ++i) {
      const int h = VEC == 1 ? g[0] : g[(2 * i + 1) % VEC];
      mu[i] = px::mk(mean[g[2 * i]], VEC == 1 ? 0.0f : mean[h]);
      r[i] = px::mk(rstd[g[2 * i]], VEC == 1 ? 0.0f : rstd[h]);
    }
  }
  __device__ __forceinline__ void load(const Params& p, const float* mean, const float* rstd, int c0) {
    load_params_of(p, c0);
    load_stats_of(p, mean, rstd, c0);
  }
};

// y of a CTA's pixels, last ones first; U loads in flight before the first store
template <typename T, int VEC>
__device__ __forceinline__ void slab_apply(const Params& p, const Slab& s, const float* mean, const float* rstd) {
  using V = Pack<T, VEC>;
  constexpr int U = 4, NP = kPairs<VEC>;
  if (s.r >= p.rows) return;
  const int64_t p0 = s.p0 + s.r;
  const int n = s.p1 > p0 ? (int)((s.p1 - p0 + p.rows - 1) / p.rows) : 0;
  const int64_t xstep = p.rows * p.xsp, ystep = (int64_t)p.rows * p.C;
  for (int v = s.vl; v < p.V; v += p.vlanes) {
    Affine<VEC> f;
    f.load(p, mean, rstd, v * VEC);
#pragma unroll
    for (int j = 0; j < NP; ++j) f.r[j] = px::mul(f.r[j], f.w[j]);
    const T* xv = reinterpret_cast<const T*>(p.x) + s.b * p.xsb + (p0 + (int64_t)(n - 1) * p.rows) * p.xsp + (int64_t)v * VEC;
    T* yv = reinterpret_cast<T*>(p.out) + (s.b * p.P + p0 + (int64_t)(n - 1) * p.rows) * p.C + (int64_t)v * VEC;
    for (int i = 0; i < n; i += U, xv -= U * xstep, yv -= U * ystep) {
      V t[U];
#pragma unroll
      for (int k = 0; k < U; ++k)
        if (i + k < n) t[k] = *reinterpret_cast<const V*>(xv - k * xstep);
#pragma unroll
      for (int k = 0; k < U; ++k) {
        if (i + k >= n) break;
        f2 d[NP];
        unpack<T, VEC>(t[k], d);
#pragma unroll
        for (int j = 0; j < NP; ++j) d[j] = activate<T>(px::fma(px::sub(d[j], f.mu[j]), f.r[j], f.b[j]), p.act);
        *reinterpret_cast<V*>(yv - k * ystep) = pack<T, VEC>(d);
      }
    }
  }
}

// FUSED: one cluster per batch entry, outputs included; else the clusters' sums to memory
template <typename T, int VEC, int GV, bool FUSED>
__global__ void __launch_bounds__(kThreads, 2) stats_kernel(const Params p) {
  extern __shared__ double2 sm[];  // [G], then scratch
  const Slab s(p, blockIdx.x);
  slab_stats<T, VEC, GV>(p, s, sm);
  cluster_barrier();
  if constexpr (FUSED) {
    float* mean = reinterpret_cast<float*>(sm + p.G);  // the scratch is free again
    float* rstd = mean + p.G;
    const bool first = tc::cluster_rank() == 0;
    for (int g = threadIdx.x; g < p.G; g += blockDim.x) {
      const double2 d = cluster_sum(sm, g);
      float m, r;
      finish(p, d.x, d.y, m, r);
      mean[g] = m;
      rstd[g] = r;
      if (first) {
        p.mean[s.b * p.G + g] = m;
        p.rstd[s.b * p.G + g] = r;
      }
    }
    __syncthreads();
    slab_apply<T, VEC>(p, s, mean, rstd);
  } else {
    const int rank = (int)tc::cluster_rank();
    for (int g = rank + kCluster * (int)threadIdx.x; g < p.G; g += kCluster * (int)blockDim.x)
      p.gpart[(s.b * p.clusters + blockIdx.x / kCluster) * p.G + g] = cluster_sum(sm, g);
    allow_dependents();
  }
  cluster_barrier();  // nobody leaves while its sums are read
}

// one warp per (batch entry, group)
__global__ void __launch_bounds__(256) finish_stats_kernel(const Params p) {
  const int64_t id = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  wait_for_primary();
  if (id < p.B * p.G) {
    const int64_t b = id / p.G;
    const double2 d = sum_clusters(p, b, (int)(id - b * p.G));
    float m, r;
    finish(p, d.x, d.y, m, r);
    if ((threadIdx.x & 31) == 0) {
      p.mean[id] = m;
      p.rstd[id] = r;
    }
  }
  allow_dependents();
}

// half of a chunk of the first pass: the CTAs that start first take the second halves, read last
// ([1, 1048576, 128]: 168 us forward, with whole chunks 197)
__device__ __forceinline__ Slab second_pass_slab(const Params& p) {
  const bool tail = (int)blockIdx.x < p.chunks;
  Slab s(p, tail ? blockIdx.x : blockIdx.x - p.chunks);
  const int64_t mid = s.p0 + (s.p1 - s.p0) / 2;
  if (tail) s.p0 = mid;
  else s.p1 = mid;
  return s;
}

template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads, 4) apply_kernel(const Params p) {
  __shared__ float mean[kDirectGroups], rstd[kDirectGroups];
  const Slab s = second_pass_slab(p);
  wait_for_primary();
  if (!p.direct) {
    slab_apply<T, VEC>(p, s, p.mean + s.b * p.G, p.rstd + s.b * p.G);
    return;
  }
  by_group(p.G, [&](int g, int first, int step) { return cluster_share(p, s.b, g, first, step); },
           [&](int g, double2 d) {
             finish(p, d.x, d.y, mean[g], rstd[g]);
             if (blockIdx.x == 0) {
               p.mean[s.b * p.G + g] = mean[g];
               p.rstd[s.b * p.G + g] = rstd[g];
             }
           });
  __syncthreads();
  slab_apply<T, VEC>(p, s, mean, rstd);
}

// --- backward --------------------------------------------------------------------

// A_c and E_c of a CTA's pixels into sm[0 .. C)
template <typename T, int VEC>
__device__ __forceinline__ void slab_grad_stats(const Params& p, const Slab& s, float2* sm) {
  using V = Pack<T, VEC>;
  constexpr int U = sizeof(T) == 2 ? 4 : 2, NP = kPairs<VEC>;
  float2* scratch = sm + p.C;  // [rows][vlanes * VEC]
  const int width = p.vlanes * VEC;
  const int64_t p0 = s.p0 + s.r, xstep = p.rows * p.xsp, dstep = p.rows * p.dsp;
  const int n = s.p1 > p0 ? (int)((s.p1 - p0 + p.rows - 1) / p.rows) : 0;
  for (int v0 = 0; v0 < p.V; v0 += p.vlanes) {
    const int v = v0 + s.vl;
    if (s.r < p.rows && v < p.V) {
      Affine<VEC> f;
      f.load(p, p.mean + s.b * p.G, p.rstd + s.b * p.G, v * VEC);
      const T* xv = reinterpret_cast<const T*>(p.x) + s.b * p.xsb + p0 * p.xsp + (int64_t)v * VEC;
      const T* dv = reinterpret_cast<const T*>(p.dy) + s.b * p.dsb + p0 * p.dsp + (int64_t)v * VEC;
      f2 A[NP], E[NP];
#pragma unroll
      for (int j = 0; j < NP; ++j) A[j] = E[j] = 0ull;
      for (int i = 0; i < n; i += U, xv += U * xstep, dv += U * dstep) {
        V t[U], d[U];
#pragma unroll
        for (int k = 0; k < U; ++k)
          if (i + k < n) {
            t[k] = *reinterpret_cast<const V*>(xv + k * xstep);
            d[k] = *reinterpret_cast<const V*>(dv + k * dstep);
          }
#pragma unroll
        for (int k = 0; k < U; ++k) {
          if (i + k >= n) break;
          f2 h[NP], g[NP];
          unpack<T, VEC>(t[k], h);
          unpack<T, VEC>(d[k], g);
#pragma unroll
          for (int j = 0; j < NP; ++j) {
            h[j] = px::mul(px::sub(h[j], f.mu[j]), f.r[j]);
            g[j] = px::mul(g[j], slope<T>(px::fma(h[j], f.w[j], f.b[j]), p.act));
            A[j] = px::add(A[j], g[j]);
            E[j] = px::fma(g[j], h[j], E[j]);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < NP; ++j) {
        float a0, a1, e0, e1;
        px::split(A[j], a0, a1);
        px::split(E[j], e0, e1);
        float2* at = scratch + s.r * width + s.vl * VEC + 2 * j;
        at[0] = make_float2(a0, e0);
        if constexpr (VEC > 1) at[1] = make_float2(a1, e1);
      }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < width && v0 * VEC + c < p.C; c += blockDim.x) {
      double A = 0.0, E = 0.0;
      for (int k = 0; k < p.rows; ++k) {
        const float2 t = scratch[k * width + c];
        A += t.x;
        E += t.y;
      }
      sm[v0 * VEC + c] = make_float2((float)A, (float)E);
    }
    __syncthreads();
  }
}

// dx of a CTA's pixels, last ones first
template <typename T, int VEC>
__device__ __forceinline__ void slab_grad_apply(const Params& p, const Slab& s, const float2* coef) {
  using V = Pack<T, VEC>;
  constexpr int U = sizeof(T) == 2 ? 4 : 2, NP = kPairs<VEC>;
  if (s.r >= p.rows) return;
  const int64_t p0 = s.p0 + s.r;
  const int n = s.p1 > p0 ? (int)((s.p1 - p0 + p.rows - 1) / p.rows) : 0;
  const int64_t last = p0 + (int64_t)(n - 1) * p.rows;
  const int64_t xstep = p.rows * p.xsp, dstep = p.rows * p.dsp, ostep = (int64_t)p.rows * p.C;
  for (int v = s.vl; v < p.V; v += p.vlanes) {
    Affine<VEC> f;
    f.load(p, p.mean + s.b * p.G, p.rstd + s.b * p.G, v * VEC);
    f2 c1[NP], c2[NP];
    int g[VEC];
    groups_of<VEC>(p, v * VEC, g);
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      const float2 a = coef[g[2 * j]], b = coef[VEC == 1 ? g[0] : g[(2 * j + 1) % VEC]];
      c1[j] = px::mk(-a.x, -b.x);
      c2[j] = px::mk(-a.y, -b.y);
    }
    const T* xv = reinterpret_cast<const T*>(p.x) + s.b * p.xsb + last * p.xsp + (int64_t)v * VEC;
    const T* dv = reinterpret_cast<const T*>(p.dy) + s.b * p.dsb + last * p.dsp + (int64_t)v * VEC;
    T* ov = reinterpret_cast<T*>(p.out) + (s.b * p.P + last) * p.C + (int64_t)v * VEC;
    for (int i = 0; i < n; i += U, xv -= U * xstep, dv -= U * dstep, ov -= U * ostep) {
      V t[U], d[U];
#pragma unroll
      for (int k = 0; k < U; ++k)
        if (i + k < n) {
          t[k] = *reinterpret_cast<const V*>(xv - k * xstep);
          d[k] = *reinterpret_cast<const V*>(dv - k * dstep);
        }
#pragma unroll
      for (int k = 0; k < U; ++k) {
        if (i + k >= n) break;
        f2 h[NP], g[NP];
        unpack<T, VEC>(t[k], h);
        unpack<T, VEC>(d[k], g);
#pragma unroll
        for (int j = 0; j < NP; ++j) {
          h[j] = px::mul(px::sub(h[j], f.mu[j]), f.r[j]);
          g[j] = px::mul(g[j], slope<T>(px::fma(h[j], f.w[j], f.b[j]), p.act));
          g[j] = px::mul(f.r[j], px::fma(h[j], c2[j], px::fma(f.w[j], g[j], c1[j])));
        }
        *reinterpret_cast<V*>(ov - k * ostep) = pack<T, VEC>(g);
      }
    }
  }
}

// (sum w A, sum w E) of group g over channel sums ae[0 .. C), by a warp
__device__ __forceinline__ double2 group_sums(const Params& p, const float2* ae, int g) {
  double a = 0.0, e = 0.0;
  for (int k = threadIdx.x & 31; k < p.cpg; k += 32) {
    const int c = g * p.cpg + k;
    const double w = p.w ? (double)load_as_f32(p.w, p.wdtype, c) : 1.0;
    a += w * ae[c].x;
    e += w * ae[c].y;
  }
  return make_double2(warp_sum(a), warp_sum(e));
}

template <typename T, int VEC, bool FUSED>
__global__ void __launch_bounds__(kThreads, 3) grad_stats_kernel(const Params p) {
  extern __shared__ double2 sm[];
  float2* ae = reinterpret_cast<float2*>(sm);  // [C] of this CTA, [C] scratch or the cluster's sums
  const Slab s(p, blockIdx.x);
  const int rank = (int)tc::cluster_rank();
  const int64_t cl = s.b * p.clusters + blockIdx.x / kCluster;
  slab_grad_stats<T, VEC>(p, s, ae);
  cluster_barrier();
  float2* all = ae + p.C;
  for (int c = threadIdx.x; c < p.C; c += blockDim.x) {
    const float2 t = cluster_sum(ae, c);
    all[c] = t;
    if (c % kCluster == rank) p.cpart[cl * p.C + c] = t;
  }
  __syncthreads();
  const double n = (double)p.P * (double)p.cpg;
  float2* coef = all + p.C;
  if (p.out) {
    for (int g = threadIdx.x >> 5; g < p.G; g += blockDim.x >> 5) {
      if (!FUSED && g % kCluster != rank) continue;
      const double2 t = group_sums(p, all, g);
      if ((threadIdx.x & 31) == 0) {
        if constexpr (FUSED) coef[g] = make_float2((float)(t.x / n), (float)(t.y / n));
        else p.gpart[cl * p.G + g] = t;
      }
    }
  }
  allow_dependents();
  if constexpr (FUSED) {
    __syncthreads();
    if (p.out) slab_grad_apply<T, VEC>(p, s, coef);
  }
  cluster_barrier();  // nobody leaves while its sums are read
}

// one warp per (batch entry, group): c1, c2
__global__ void __launch_bounds__(256) finish_grad_kernel(const Params p) {
  const int64_t id = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  wait_for_primary();
  if (id < p.B * p.G) {
    const int64_t b = id / p.G;
    const double n = (double)p.P * (double)p.cpg;
    const double2 t = sum_clusters(p, b, (int)(id - b * p.G));
    if ((threadIdx.x & 31) == 0) p.coef[id] = make_float2((float)(t.x / n), (float)(t.y / n));
  }
  allow_dependents();
}

// dw and db of channels from c0 on, a warp to a channel: sums over batch entries and clusters
__device__ __forceinline__ void param_grads(const Params& p, int c0, int step) {
  const int lane = threadIdx.x & 31;
  for (int c = c0 + (int)(threadIdx.x >> 5); c < p.C; c += step) {
    double A = 0.0, E = 0.0;
    for (int64_t k = lane; k < p.B * p.clusters; k += 32) {
      const float2 t = __ldcg(p.cpart + k * p.C + c);
      A += t.x;
      E += t.y;
    }
    A = warp_sum(A);
    E = warp_sum(E);
    if (lane == 0) {
      if (p.db) store_as(p.db, p.wdtype, c, (float)A);
      if (p.dw) store_as(p.dw, p.wdtype, c, (float)E);
    }
  }
}

// dw and db alone
__global__ void __launch_bounds__(256) param_grad_kernel(const Params p) {
  wait_for_primary();
  param_grads(p, (int)blockIdx.x * 8, (int)gridDim.x * 8);
}

// dx; the CTAs behind the last chunk of batch entry 0 form dw and db
// A CTA takes a whole chunk here: its first instructions (parameters, statistics, the clusters' sums)
// cost more than halves win ([2, 16384, 512]: 66.9 -> 65.3 us for both passes, [1, 16384, 320] 40.0 -> 37.2).
template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads, 3) grad_apply_kernel(const Params p) {
  __shared__ float2 coef[kDirectGroups];
  wait_for_primary();
  if ((int)blockIdx.x >= p.chunks) {
    if (p.b0 + blockIdx.y == 0) {
      const int warps = (int)blockDim.x >> 5;
      param_grads(p, ((int)blockIdx.x - p.chunks) * warps, ((int)gridDim.x - p.chunks) * warps);
    }
    return;
  }
  const Slab s(p, blockIdx.x);
  if (!p.direct) {
    slab_grad_apply<T, VEC>(p, s, p.coef + s.b * p.G);
    return;
  }
  const double n = (double)p.P * (double)p.cpg;
  by_group(p.G, [&](int g, int first, int step) { return cluster_share(p, s.b, g, first, step); },
           [&](int g, double2 d) { coef[g] = make_float2((float)(d.x / n), (float)(d.y / n)); });
  __syncthreads();
  slab_grad_apply<T, VEC>(p, s, coef);
}

// --- host ------------------------------------------------------------------------

static int gcd(int a, int b) {
  while (b) { const int t = a % b; a = b; b = t; }
  return a;
}

// clusters per batch entry, at most: four CTAs per SM in all, one cluster per 8 pixels and CTA
static int64_t most_clusters(int64_t B, int64_t P) {
  if (B < 1 || P < 1) return 1;
  int64_t c = (int64_t)sm_count() * 4 / (kCluster * B);
  const int64_t m = ceil_div(P, kCluster * 8);
  if (c > m) c = m;
  return c < 1 ? 1 : c;
}

// the same of the backward pass, whose threads' runs are bounded (a thread row to a CTA at least)
static int64_t most_grad_clusters(int64_t B, int64_t P) {
  return most_clusters(B, P) + (P > kCluster * kGradRun ? ceil_div(P, kCluster * kGradRun) : 0);
}

// One cluster per batch entry is enough up to this many bytes of x: 8 CTAs read 32 KB each in about
// the time of the second launch that they save.
constexpr int64_t kFusedBytes = 256 * 1024;

struct Plan {
  bool fused;
  unsigned threads;
};

// clusters of `kernel` that run at once on the current device (asked for once per device)
static int resident_clusters(void (*kernel)(Params), unsigned threads, size_t smem,
                             std::atomic<int> (&known)[64]) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return sm_count() * 2 / kCluster;
  int n = known[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(kCluster * 64);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = kCluster;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n < 1) {
      cudaGetLastError();
      n = sm_count() * 2 / kCluster;
    }
    known[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

// `resident`: clusters of the first pass that run at once, so that it runs in one wave, or where `run`
// bounds a thread's pixels in whole ones
static Plan plan(Params& p, int vec, int size, int resident, int run = 0) {
  p.V = p.C / vec;
  p.vlanes = p.V < kThreads ? p.V : kThreads;
  p.rows = kThreads / p.vlanes;
  const bool fused = p.P * p.C * size <= kFusedBytes;
  int64_t clusters = fused ? 1 : most_clusters(p.B, p.P);
  if (clusters * p.B > resident) clusters = resident / p.B > 0 ? resident / p.B : 1;
  // at least 16 pixels per thread row, so that runs fill
  const int64_t most = ceil_div(p.P, (int64_t)kCluster * p.rows * 16);
  if (clusters > most) clusters = most;
  const int64_t need = run ? ceil_div(p.P, (int64_t)kCluster * p.rows * run) : 0;
  if (need > clusters) {
    clusters = ceil_div(need * p.B, resident) * resident / p.B;
    if (clusters < need) clusters = need;
    const int64_t room = most_grad_clusters(p.B, p.P);
    if (clusters > room) clusters = room;
  }
  p.clusters = (int)clusters;
  p.chunks = kCluster * p.clusters;
  p.chunk = ceil_div(p.P, p.chunks);
  p.direct = p.G <= kDirectGroups;
  return {fused, (unsigned)(ceil_div((int64_t)p.vlanes * p.rows, 32) * 32)};
}

// Launches with clusters of `cluster` CTAs (0: none); dependent: may start before the launch before
// it has ended, and waits for it in the kernel.
static int launch(void (*kernel)(Params), dim3 grid, unsigned threads, size_t smem, int cluster, bool dependent,
                  const Params& p, cudaStream_t st, const char* what) {
  if (smem > 48 * 1024) {
    // the largest size at once, not this call's: another thread may launch the same kernel with another one
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem);
    ZIB_HOST_CHECK(e == cudaSuccess, ZIB_ERR_LAUNCH, "%s: cudaFuncSetAttribute failed: %s", what,
                   cudaGetErrorString(e));
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  int n = 0;
  if (cluster) {
    at[n].id = cudaLaunchAttributeClusterDimension;
    at[n].val.clusterDim.x = cluster;
    at[n].val.clusterDim.y = at[n].val.clusterDim.z = 1;
    ++n;
  }
  if (dependent) {
    at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = at;
  cfg.numAttrs = n;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
  if (e != cudaSuccess) {
    cudaGetLastError();
    zib_set_error("%s: launch failed: %s", what, cudaGetErrorString(e));
    return ZIB_ERR_LAUNCH;
  }
  return ZIB_OK;
}

// the same with x CTAs for each batch entry, which lie along y of the grid: 65535 of them to a launch.
// (Along y and z, with surplus CTAs that leave, the gradients of [4, 447262, 9] took 111 us instead of 99.)
static int launch_batch(void (*kernel)(Params), unsigned x, unsigned threads, size_t smem, int cluster, bool dependent,
                        Params p, cudaStream_t st, const char* what) {
  constexpr int64_t kMost = 65535;
  int rc = ZIB_OK;
  for (p.b0 = 0; p.b0 < p.B && !rc; p.b0 += kMost) {
    const int64_t n = p.B - p.b0 < kMost ? p.B - p.b0 : kMost;
    rc = launch(kernel, dim3(x, (unsigned)n), threads, smem, cluster, dependent, p, st, what);
  }
  return rc;
}

template <typename T, int VEC, int GV>
static int forward_g(Params& p, cudaStream_t st) {
  const char* what = "zib_group_norm";
  static std::atomic<int> known[64];
  const Plan pl = plan(p, VEC, sizeof(T), resident_clusters(stats_kernel<T, VEC, GV, false>, kThreads, 24 * 1024, known));
  const size_t sums = (size_t)p.rows * p.V * (VEC / GV);
  size_t smem = ((p.cpg / GV * p.rows == 1 ? 0 : (size_t)p.G) + sums) * sizeof(double2);
  const size_t stats = (size_t)p.G * (sizeof(double2) + 2 * sizeof(float));
  if (smem < stats) smem = stats;
  ZIB_HOST_CHECK(smem <= kMaxSmem, ZIB_ERR_TOO_LARGE, "%s: %d channels", what, p.C);
  if (pl.fused)
    return launch_batch(stats_kernel<T, VEC, GV, true>, p.chunks, pl.threads, smem, kCluster, false, p, st, what);
  int rc = launch_batch(stats_kernel<T, VEC, GV, false>, p.chunks, pl.threads, smem, kCluster, false, p, st, what);
  if (!rc && !p.direct)
    rc = launch(finish_stats_kernel, dim3((unsigned)ceil_div(p.B * p.G, 8)), 256, 0, 0, true, p, st, what);
  if (!rc) rc = launch_batch(apply_kernel<T, VEC>, 2 * p.chunks, pl.threads, 0, 0, true, p, st, what);
  return rc;
}

template <typename T, int VEC>
static int forward_v(Params& p, cudaStream_t st) {
  const int gv = gcd(p.cpg, VEC);
  if constexpr (VEC == 8) if (gv == 8) return forward_g<T, VEC, 8>(p, st);
  if constexpr (VEC >= 4) if (gv == 4) return forward_g<T, VEC, 4>(p, st);
  if constexpr (VEC >= 2) if (gv == 2) return forward_g<T, VEC, 2>(p, st);
  return forward_g<T, VEC, 1>(p, st);
}

template <typename T, int VEC>
static int backward_v(Params& p, cudaStream_t st) {
  const char* what = "zib_group_norm_backward";
  static std::atomic<int> known[64];
  const Plan pl = plan(p, VEC, 2 * sizeof(T),  // x and dy
                       resident_clusters(grad_stats_kernel<T, VEC, false>, kThreads, 24 * 1024, known), kGradRun);
  size_t smem = ((size_t)p.C + (size_t)p.rows * p.vlanes * VEC) * sizeof(float2);
  const size_t sums = ((size_t)2 * p.C + p.G) * sizeof(float2);
  if (smem < sums) smem = sums;
  const bool params = p.dw || p.db;
  int rc;
  if (pl.fused || !p.out) {
    rc = launch_batch(pl.fused ? grad_stats_kernel<T, VEC, true> : grad_stats_kernel<T, VEC, false>, p.chunks,
                      pl.threads, smem, kCluster, false, p, st, what);
    if (!rc && params)
      rc = launch(param_grad_kernel, dim3((unsigned)ceil_div(p.C, 8)), 256, 0, 0, true, p, st, what);
    return rc;
  }
  rc = launch_batch(grad_stats_kernel<T, VEC, false>, p.chunks, pl.threads, smem, kCluster, false, p, st, what);
  if (!rc && !p.direct)
    rc = launch(finish_grad_kernel, dim3((unsigned)ceil_div(p.B * p.G, 8)), 256, 0, 0, true, p, st, what);
  const unsigned extra = params ? (unsigned)ceil_div(p.C, (int64_t)pl.threads / 32) : 0;
  if (!rc)
    rc = launch_batch(grad_apply_kernel<T, VEC>, p.chunks + extra, pl.threads, 0, 0, true, p, st, what);
  return rc;
}

static int check(const Params& p, int64_t C, int64_t G, int dtype, const char* what) {
  ZIB_HOST_CHECK(known_dtype(dtype) && known_dtype(p.wdtype), ZIB_ERR_INVALID_ARG, "%s: unknown dtype", what);
  ZIB_HOST_CHECK(p.B >= 0 && p.P >= 0 && C >= 1 && G >= 1 && C % G == 0, ZIB_ERR_INVALID_ARG,
                 "%s: %lld channels in %lld groups", what, (long long)C, (long long)G);
  ZIB_HOST_CHECK(C <= kMaxChannels && p.B < (1ll << 31), ZIB_ERR_TOO_LARGE,
                 "%s: at most %d channels and 2^31 - 1 batch entries", what, kMaxChannels);
  ZIB_HOST_CHECK(p.act == ZIB_ACT_NONE || p.act == ZIB_ACT_SILU, ZIB_ERR_INVALID_ARG, "%s: unknown activation %d",
                 what, p.act);
  ZIB_HOST_CHECK(p.eps >= 0.0f, ZIB_ERR_INVALID_ARG, "%s: eps must not be negative", what);
  return ZIB_OK;
}

// elements per access: as many as divide the channels, the strides and the addresses
static int vector_width(const Params& p, int size) {
  auto ok = [&](const void* x, int64_t sb, int64_t sp, int v) {
    return !x || ((uintptr_t)x % (v * size) == 0 && (sb % v == 0 || p.B == 1) && (sp % v == 0 || p.P == 1));
  };
  int v = 16 / size;
  while (v > 1 && !(p.C % v == 0 && ok(p.x, p.xsb, p.xsp, v) && ok(p.dy, p.dsb, p.dsp, v) && ok(p.out, 0, 0, v)))
    v >>= 1;
  return v;
}

template <typename T>
static int forward(Params& p, int v, cudaStream_t st) {
  if constexpr (sizeof(T) == 2) if (v == 8) return forward_v<T, 8>(p, st);
  if (v == 4) return forward_v<T, 4>(p, st);
  if (v == 2) return forward_v<T, 2>(p, st);
  return forward_v<T, 1>(p, st);
}

// four channels per access at most: two inputs, four constants and two sums per channel are registers
template <typename T>
static int backward(Params& p, int v, cudaStream_t st) {
  if (v >= 4) return backward_v<T, 4>(p, st);
  if (v == 2) return backward_v<T, 2>(p, st);
  return backward_v<T, 1>(p, st);
}

}  // namespace gn
}  // namespace zib

using namespace zib;

extern "C" int64_t zib_group_norm_workspace(int64_t B, int64_t P, int64_t C, int64_t G, int backward) {
  if (B < 0 || P < 0 || C < 1 || G < 1) return 0;
  const int64_t n = B * (backward ? gn::most_grad_clusters(B, P) : gn::most_clusters(B, P));
  const int64_t groups = n * G * (int64_t)sizeof(double2);
  return backward ? groups + (n * C + B * G) * (int64_t)sizeof(float2) : groups;
}

extern "C" int zib_group_norm(const void* x, int64_t xsb, int64_t xsp, void* y, const void* w, const void* b,
                              int wdtype, float* mean, float* rstd, void* workspace, int64_t workspace_bytes,
                              int64_t B, int64_t P, int64_t C, int64_t G, int dtype, float eps, int act,
                              void* stream) {
  const char* what = "zib_group_norm";
  gn::Params p{};
  p.x = x; p.xsb = xsb; p.xsp = xsp; p.out = y; p.w = w; p.b = b; p.wdtype = wdtype;
  p.mean = mean; p.rstd = rstd; p.gpart = (double2*)workspace;
  p.B = B; p.P = P; p.act = act; p.eps = eps;
  const int rc = gn::check(p, C, G, dtype, what);
  if (rc) return rc;
  if (B == 0 || P == 0) return ZIB_OK;
  ZIB_HOST_CHECK(x && y && mean && rstd && workspace, ZIB_ERR_INVALID_ARG, "%s: null operand", what);
  ZIB_HOST_CHECK(workspace_bytes >= zib_group_norm_workspace(B, P, C, G, 0) && (uintptr_t)workspace % 16 == 0,
                 ZIB_ERR_INVALID_ARG, "%s: workspace of %lld bytes, 16-byte aligned, needed", what,
                 (long long)zib_group_norm_workspace(B, P, C, G, 0));
  p.C = (int)C; p.G = (int)G; p.cpg = (int)(C / G);
  cudaStream_t st = (cudaStream_t)stream;
  const int v = gn::vector_width(p, dtype_bytes(dtype));
  if (dtype == ZIB_BF16) return gn::forward<__nv_bfloat16>(p, v, st);
  if (dtype == ZIB_F16) return gn::forward<__half>(p, v, st);
  return gn::forward<float>(p, v, st);
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
  const int rc = gn::check(p, C, G, dtype, what);
  if (rc) return rc;
  ZIB_HOST_CHECK(B > 0 && P > 0, ZIB_ERR_INVALID_ARG, "%s: empty input", what);
  ZIB_HOST_CHECK(x && dy && mean && rstd && workspace, ZIB_ERR_INVALID_ARG, "%s: null operand", what);
  ZIB_HOST_CHECK(workspace_bytes >= zib_group_norm_workspace(B, P, C, G, 1) && (uintptr_t)workspace % 16 == 0,
                 ZIB_ERR_INVALID_ARG, "%s: workspace of %lld bytes, 16-byte aligned, needed", what,
                 (long long)zib_group_norm_workspace(B, P, C, G, 1));
  if (!dx && !dw && !db) return ZIB_OK;
  p.C = (int)C; p.G = (int)G; p.cpg = (int)(C / G);
  const int64_t n = B * gn::most_grad_clusters(B, P);
  p.gpart = (double2*)workspace;
  p.cpart = (float2*)(p.gpart + n * G);
  p.coef = p.cpart + n * C;
  cudaStream_t st = (cudaStream_t)stream;
  const int v = gn::vector_width(p, dtype_bytes(dtype));
  if (dtype == ZIB_BF16) return gn::backward<__nv_bfloat16>(p, v, st);
  if (dtype == ZIB_F16) return gn::backward<__half>(p, v, st);
  return gn::backward<float>(p, v, st);
}
