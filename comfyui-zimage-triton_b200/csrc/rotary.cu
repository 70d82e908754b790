// Rotary positions.
//
// Position p turns feature pair j of every head by the angle p f_j:
//   a' = a cos - b sin,  b' = b cos + a sin
// where the pair is (x[2j], x[2j+1]) in the interleaved layout and (x[j], x[j + R/2]) in the half
// layout; features R and up pass through.  Turning by the opposite angle is the transposed map,
// so the gradient is the same kernel with sin negated.
//
// Bound by memory: each element is read and written once (4 bytes in 16-bit types) against three
// fp32 operations.  A thread keeps one unit of a head (VEC pairs in the half layout, VEC features
// in the interleaved one) and walks over the heads of its token, queries and keys alike, so the
// cos and sin of a unit are read once per token, not once per head: at 30 + 30 heads the fp32
// table would otherwise be as many bytes as the data.
#include "zib_async.cuh"
#include "zib_types.cuh"

ZIB_DEFINE_ERROR_READER(zib_err_read_clear_rotary)

namespace zib {
namespace rotary {

struct Heads {  // one tensor [B, S, H, D], element strides; out contiguous over (B, S, H, D)
  const void* x;
  void* out;
  int64_t sb, ss, sh;
  int H;
};

struct Params {
  Heads q, k;
  const float* cos;
  const float* sin;
  int64_t cs_b, cs_l;  // table strides of batch entry and position
  const void* pos;     // positions [B, S] (null: the index s)
  int pos64;           // 1: int64 positions, 0: int32
  int64_t ps_b, ps_s;
  int64_t L;           // table rows
  int64_t S, tokens;   // tokens = B * S
  int D, R;
  int units;           // units per head: rotated ones, then pass-through ones
  int rot_units;
  int head_lanes, token_lanes;
  float sign;
};

// Loads unit u of one head, rotates, stores.
template <typename T, int VEC, bool HALF>
__device__ __forceinline__ void turn(const T* __restrict__ x, T* __restrict__ o, int at, int half, const float* c,
                                     const float* s) {
  using V = Pack<T, VEC>;
  if constexpr (HALF) {
    const V a = *reinterpret_cast<const V*>(x + at), b = *reinterpret_cast<const V*>(x + at + half);
    V ra, rb;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const float fa = to_f32(a.v[i]), fb = to_f32(b.v[i]);
      ra.v[i] = from_f32<T>(fmaf(fa, c[i], -(fb * s[i])));
      rb.v[i] = from_f32<T>(fmaf(fb, c[i], fa * s[i]));
    }
    *reinterpret_cast<V*>(o + at) = ra;
    *reinterpret_cast<V*>(o + at + half) = rb;
  } else {
    const V a = *reinterpret_cast<const V*>(x + at);
    V r;
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) {
      const float fa = to_f32(a.v[2 * i]), fb = to_f32(a.v[2 * i + 1]);
      r.v[2 * i] = from_f32<T>(fmaf(fa, c[i], -(fb * s[i])));
      r.v[2 * i + 1] = from_f32<T>(fmaf(fb, c[i], fa * s[i]));
    }
    *reinterpret_cast<V*>(o + at) = r;
  }
}

// VEC: elements per access.  The interleaved layout turns VEC / 2 pairs per unit, the half layout VEC.
template <typename T, int VEC, bool HALF>
__global__ void __launch_bounds__(1024) rotary_kernel(const Params p) {
  using V = Pack<T, VEC>;
  constexpr int NP = HALF ? VEC : VEC / 2;  // pairs per unit
  const int tid = threadIdx.x;
  const int u = tid % p.units;
  const int hl = (tid / p.units) % p.head_lanes;
  const int64_t token = (int64_t)blockIdx.x * p.token_lanes + tid / (p.units * p.head_lanes);
  if (token >= p.tokens) return;
  const int64_t b = token / p.S, s = token - b * p.S;
  const bool rot = u < p.rot_units;
  float c[NP], sn[NP];
  if (rot) {
    int64_t l = s;
    if (p.pos) {
      const int64_t i = b * p.ps_b + s * p.ps_s;
      l = p.pos64 ? reinterpret_cast<const int64_t*>(p.pos)[i] : (int64_t)reinterpret_cast<const int32_t*>(p.pos)[i];
    }
    if (l < 0 || l >= p.L) {
      // a position outside the table: the rotated features read NaN and the host learns of it
      atomicExch(&g_zib_err_word, (int)ZIB_ERR_INVALID_ARG);
#pragma unroll
      for (int i = 0; i < NP; ++i) c[i] = sn[i] = __uint_as_float(0x7FC00000u);
    } else {
      const float* cp = p.cos + b * p.cs_b + l * p.cs_l + u * NP;
      const float* sp = p.sin + b * p.cs_b + l * p.cs_l + u * NP;
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        c[i] = __ldg(cp + i);
        sn[i] = p.sign * __ldg(sp + i);
      }
    }
  }
  const int at = rot ? u * VEC : p.R + (u - p.rot_units) * VEC;
  const int half = p.R >> 1;
#pragma unroll 1
  for (int t = 0; t < 2; ++t) {
    const Heads& hd = t ? p.k : p.q;
    const T* x = reinterpret_cast<const T*>(hd.x) + b * hd.sb + s * hd.ss;
    T* o = reinterpret_cast<T*>(hd.out) + token * hd.H * p.D;
#pragma unroll 2
    for (int h = hl; h < hd.H; h += p.head_lanes) {
      if (rot) turn<T, VEC, HALF>(x + h * hd.sh, o + (int64_t)h * p.D, at, half, c, sn);
      else *reinterpret_cast<V*>(o + (int64_t)h * p.D + at) = *reinterpret_cast<const V*>(x + h * hd.sh + at);
    }
  }
}

template <typename T, bool HALF>
static void launch(int vec, unsigned grid, int threads, const Params& p, cudaStream_t st) {
  if constexpr (sizeof(T) == 2) {
    if (vec == 8) { rotary_kernel<T, 8, HALF><<<grid, threads, 0, st>>>(p); return; }
  }
  if (vec == 4) { rotary_kernel<T, 4, HALF><<<grid, threads, 0, st>>>(p); return; }
  if (vec == 2) { rotary_kernel<T, 2, HALF><<<grid, threads, 0, st>>>(p); return; }
  if constexpr (HALF) rotary_kernel<T, 1, HALF><<<grid, threads, 0, st>>>(p);
}

// --- tables ------------------------------------------------------------------------

struct TableParams {
  const void* pos;  // null: start, start + 1, ...
  int pos64;
  int64_t ps, start, T;
  int half;          // dim / 2
  int kind;          // zib_rotary_scaling
  double log_theta;  // of the base in use
  double inv_factor, original, beta_fast, beta_slow;
  float mscale;
  float* cos;
  float* sin;
};

// cos and sin of p f_j, f_j = theta^(-2j/dim) scaled.  The angle is formed in turns in fp64 (a far
// position times a frequency needs more than 24 bits), its whole turns are dropped there, and the
// rest is split into an fp32 value and a correction d for the first-order step
// cos(x + d) = cos x - d sin x, so each entry is within about 2 ulp.  A thread keeps one frequency
// and walks over positions, so the fp64 exp is paid once per thread.
__global__ void __launch_bounds__(256) rotary_table_kernel(const TableParams p) {
  const int j = blockIdx.y * blockDim.x + threadIdx.x;
  if (j >= p.half) return;
  double f = exp(-p.log_theta * (double)j / (double)p.half);
  if (p.kind == ZIB_ROTARY_LINEAR) f *= p.inv_factor;
  if (p.kind == ZIB_ROTARY_YARN) {
    // whole turns over the original length: few turns are interpolated, many are kept
    const double turns = p.original * f * 0.15915494309189535;
    const double keep = fmin(1.0, fmax(0.0, (turns - p.beta_slow) / (p.beta_fast - p.beta_slow)));
    f = (1.0 - keep) * f * p.inv_factor + keep * f;
  }
  const double ft = f * 0.15915494309189535;  // turns per position
  const int64_t step = (int64_t)gridDim.x * blockDim.y;
  for (int64_t t = (int64_t)blockIdx.x * blockDim.y + threadIdx.y; t < p.T; t += step) {
    int64_t pos = p.start + t;
    if (p.pos)
      pos = p.pos64 ? reinterpret_cast<const int64_t*>(p.pos)[t * p.ps]
                    : (int64_t)reinterpret_cast<const int32_t*>(p.pos)[t * p.ps];
    const double a = (double)pos * ft;
    const double r = 2.0 * (a - rint(a));  // angle / pi, in [-1, 1]
    const float hi = (float)r;
    const float d = (float)((r - (double)hi) * 3.141592653589793);
    float s, c;
    sincospif(hi, &s, &c);
    p.cos[t * p.half + j] = p.mscale * fmaf(-d, s, c);
    p.sin[t * p.half + j] = p.mscale * fmaf(d, c, s);
  }
}

}  // namespace rotary
}  // namespace zib

using namespace zib;

extern "C" int zib_rotary(const void* q, int64_t q_sb, int64_t q_ss, int64_t q_sh, void* q_out, int64_t Hq,
                          const void* k, int64_t k_sb, int64_t k_ss, int64_t k_sh, void* k_out, int64_t Hk,
                          int dtype, const float* cos, const float* sin, int64_t cs_b, int64_t cs_l, int64_t L,
                          const void* positions, int pos64, int64_t ps_b, int64_t ps_s, int64_t B, int64_t S,
                          int64_t D, int64_t R, int half_layout, int inverse, void* stream) {
  const char* what = "zib_rotary";
  ZIB_HOST_CHECK(known_dtype(dtype), ZIB_ERR_INVALID_ARG, "%s: unknown dtype %d", what, dtype);
  ZIB_HOST_CHECK(B >= 0 && S >= 0 && Hq >= 0 && Hk >= 0, ZIB_ERR_INVALID_ARG, "%s: negative size", what);
  ZIB_HOST_CHECK(D >= 2 && D <= 1024 && R >= 2 && R <= D && R % 2 == 0, ZIB_ERR_INVALID_ARG,
                 "%s: head size %lld (2 to 1024) with %lld rotated features (even, at most the head size)", what,
                 (long long)D, (long long)R);
  if (B == 0 || S == 0 || Hq + Hk == 0) return ZIB_OK;
  ZIB_HOST_CHECK((Hq == 0 || (q && q_out)) && (Hk == 0 || (k && k_out)) && cos && sin, ZIB_ERR_INVALID_ARG,
                 "%s: null operand", what);
  ZIB_HOST_CHECK(L >= 1 && (positions || L >= S), ZIB_ERR_INVALID_ARG, "%s: table of %lld rows for %lld positions",
                 what, (long long)L, (long long)S);
  ZIB_HOST_CHECK(Hq <= (1 << 20) && Hk <= (1 << 20), ZIB_ERR_TOO_LARGE, "%s: head count", what);
  // elements per access: as many as divide the parts of a head, the strides and the addresses
  const int size = dtype_bytes(dtype);
  int vec = 16 / size;
  const int64_t part = half_layout ? R / 2 : R;
  auto fits = [&](int v) {
    auto ok = [&](const void* x, void* o, int64_t sb, int64_t ss, int64_t sh, int64_t H) {
      return H == 0 || ((sb % v == 0 || B == 1) && (ss % v == 0 || S == 1) && (sh % v == 0 || H == 1) &&
                        (uintptr_t)x % (v * size) == 0 && (uintptr_t)o % (v * size) == 0);
    };
    return part % v == 0 && (D - R) % v == 0 && ok(q, q_out, q_sb, q_ss, q_sh, Hq) &&
           ok(k, k_out, k_sb, k_ss, k_sh, Hk);
  };
  while (vec > 1 && !fits(vec)) vec >>= 1;
  ZIB_HOST_CHECK(vec > 1 || half_layout, ZIB_ERR_ALIGNMENT,
                 "%s: the interleaved layout needs even strides, an even head size and operands aligned to a pair",
                 what);
  rotary::Params p;
  p.q = {q, q_out, q_sb, q_ss, q_sh, (int)Hq};
  p.k = {k, k_out, k_sb, k_ss, k_sh, (int)Hk};
  p.cos = cos; p.sin = sin; p.cs_b = cs_b; p.cs_l = cs_l; p.L = L;
  p.pos = positions; p.pos64 = pos64; p.ps_b = ps_b; p.ps_s = ps_s;
  p.S = S; p.tokens = B * S; p.D = (int)D; p.R = (int)R;
  p.rot_units = (int)(part / vec);
  p.units = p.rot_units + (int)((D - R) / vec);
  p.sign = inverse ? -1.0f : 1.0f;
  const int most = (int)(Hq > Hk ? Hq : Hk);
  p.head_lanes = 256 / p.units;
  if (p.head_lanes < 1) p.head_lanes = 1;
  if (p.head_lanes > most) p.head_lanes = most;
  p.token_lanes = 256 / (p.units * p.head_lanes);
  if (p.token_lanes < 1) p.token_lanes = 1;
  const int threads = p.units * p.head_lanes * p.token_lanes;
  const int64_t grid = ceil_div(p.tokens, p.token_lanes);
  ZIB_HOST_CHECK(grid <= 0x7FFFFFFF, ZIB_ERR_TOO_LARGE, "%s: %lld tokens", what, (long long)p.tokens);
  cudaStream_t st = (cudaStream_t)stream;
  const unsigned g = (unsigned)grid;
  if (dtype == ZIB_BF16) {
    if (half_layout) rotary::launch<__nv_bfloat16, true>(vec, g, threads, p, st);
    else rotary::launch<__nv_bfloat16, false>(vec, g, threads, p, st);
  } else if (dtype == ZIB_F16) {
    if (half_layout) rotary::launch<__half, true>(vec, g, threads, p, st);
    else rotary::launch<__half, false>(vec, g, threads, p, st);
  } else {
    if (half_layout) rotary::launch<float, true>(vec, g, threads, p, st);
    else rotary::launch<float, false>(vec, g, threads, p, st);
  }
  return zib_check_launch(what);
}

extern "C" int zib_rotary_table(const void* positions, int pos64, int64_t ps, int64_t start, int64_t T, int64_t dim,
                                double theta, int scaling, double factor, double original, double beta_fast,
                                double beta_slow, double attention_factor, float* cos, float* sin, void* stream) {
  const char* what = "zib_rotary_table";
  ZIB_HOST_CHECK(T >= 0 && dim >= 2 && dim % 2 == 0 && dim <= 65536, ZIB_ERR_INVALID_ARG,
                 "%s: %lld positions, dim %lld (even, at most 65536)", what, (long long)T, (long long)dim);
  ZIB_HOST_CHECK(theta > 0.0 && theta < 1e300, ZIB_ERR_INVALID_ARG, "%s: theta must be positive and finite", what);
  ZIB_HOST_CHECK(scaling >= ZIB_ROTARY_NONE && scaling <= ZIB_ROTARY_YARN, ZIB_ERR_INVALID_ARG,
                 "%s: unknown scaling %d", what, scaling);
  if (scaling != ZIB_ROTARY_NONE)
    ZIB_HOST_CHECK(factor >= 1.0 && factor < 1e9, ZIB_ERR_INVALID_ARG, "%s: scaling factor must be at least 1", what);
  if (scaling == ZIB_ROTARY_NTK)
    ZIB_HOST_CHECK(dim > 2, ZIB_ERR_INVALID_ARG, "%s: ntk scaling needs dim > 2", what);
  if (scaling == ZIB_ROTARY_YARN)
    ZIB_HOST_CHECK(original > 0.0 && beta_fast > beta_slow && attention_factor > 0.0, ZIB_ERR_INVALID_ARG,
                   "%s: yarn scaling needs a positive original length, beta_fast > beta_slow and a positive "
                   "attention factor", what);
  if (T == 0) return ZIB_OK;
  ZIB_HOST_CHECK(cos && sin, ZIB_ERR_INVALID_ARG, "%s: null operand", what);
  rotary::TableParams p;
  p.pos = positions; p.pos64 = pos64; p.ps = ps; p.start = start; p.T = T;
  p.half = (int)(dim / 2);
  p.kind = scaling;
  p.log_theta = log(theta);
  if (scaling == ZIB_ROTARY_NTK) p.log_theta += log(factor) * (double)dim / (double)(dim - 2);
  p.inv_factor = 1.0 / factor;
  p.original = original; p.beta_fast = beta_fast; p.beta_slow = beta_slow;
  p.mscale = scaling == ZIB_ROTARY_YARN ? (float)attention_factor : 1.0f;
  p.cos = cos; p.sin = sin;
  const int bx = p.half >= 64 ? 64 : 32;
  dim3 block(bx, 256 / bx);
  const int64_t gy = ceil_div(p.half, bx);
  int64_t gx = ceil_div(T, (int64_t)block.y * 4);
  const int64_t cap = ceil_div((int64_t)sm_count() * 8, gy);
  if (gx > cap) gx = cap;
  rotary::rotary_table_kernel<<<dim3((unsigned)gx, (unsigned)gy), block, 0, (cudaStream_t)stream>>>(p);
  return zib_check_launch(what);
}
