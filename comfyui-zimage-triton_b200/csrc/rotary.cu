// Rotary positions.
//
// Position p turns feature pair j of every head by the angle p f_j:
//   a' = a cos - b sin,  b' = b cos + a sin
// where the pair is (x[2j], x[2j+1]) in the interleaved layout and (x[j], x[j + R/2]) in the half
// layout; features R and up pass through.  Turning by the opposite angle is the transposed map,
// so the gradient is the same kernel with sin negated.
//
// Bound by memory: each element is read and written once (4 bytes in 16-bit types) against three
// fp32 operations.  A thread keeps one unit of a head (two vectors of VEC features: the halves of
// VEC pairs in the half layout, neighbours where features pass through; one vector in the interleaved
// layout) and walks over heads of its token, queries and keys in one count, so the cos and sin of a
// unit are read once for a few heads: the fp32 table would otherwise be as many bytes as the data.
// A thread's chain is long (position, table row, data), so what hides it is many threads: more loads
// per thread at the price of registers (four heads in flight, 25 to 37% occupancy) measured slower,
// 97 us for [2, 4608, 30 + 30, 128] interleaved (285 MB, 43.6 us at HBM's rate) where this takes 53 us.
#include "zib_async.cuh"
#include "zib_pairs.cuh"

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
  int64_t S;
  int D, R;
  int units;           // units per head: rotated ones, then pass-through ones
  int rot_units;
  int table_vec;       // the tables' rows allow 16-byte (or a unit's) accesses
  float sign;
};

// the tensors that are read are not written by the launch: loads may pass stores
template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> load_vec(const T* p) {
  Pack<T, VEC> r;
  if constexpr (sizeof(r) == 16) *reinterpret_cast<uint4*>(&r) = __ldg(reinterpret_cast<const uint4*>(p));
  else if constexpr (sizeof(r) == 8) *reinterpret_cast<uint2*>(&r) = __ldg(reinterpret_cast<const uint2*>(p));
  else if constexpr (sizeof(r) == 4) *reinterpret_cast<uint32_t*>(&r) = __ldg(reinterpret_cast<const uint32_t*>(p));
  else *reinterpret_cast<uint16_t*>(&r) = __ldg(reinterpret_cast<const uint16_t*>(p));
  return r;
}

// The cos and sin of one unit: per pair of neighbouring features (interleaved) or of pairs (half).
template <int VEC, bool HALF>
struct Angles {
  // interleaved, pair j: c = (cos, cos), s = (-sin, sin): (a, b) c + (b, a) s
  // half, pairs 2j and 2j + 1: c = (cos, cos'), s = (sin, sin')
  static constexpr int N = VEC < 2 ? 1 : VEC / 2;
  f2 c[N], s[N];
  __device__ __forceinline__ void set(int i, float cv, float sv) {  // pair i of the unit
    if constexpr (HALF) {
      float c0, c1, s0, s1;
      px::split(c[i / 2], c0, c1);
      px::split(s[i / 2], s0, s1);
      if (i & 1) c1 = cv, s1 = sv;
      else c0 = cv, s0 = sv;
      c[i / 2] = px::mk(c0, c1);
      s[i / 2] = px::mk(s0, s1);
    } else {
      c[i] = px::mk(cv, cv);
      s[i] = px::mk(-sv, sv);
    }
  }
};

__device__ __forceinline__ f2 negate(f2 v) { return v ^ 0x8000000080000000ull; }
__device__ __forceinline__ f2 swap(f2 v) {
  float a, b;
  px::split(v, a, b);
  return px::mk(b, a);
}

// one head's unit in a (and d: its second vector); each output is one product and one multiply-add
template <typename T, int VEC, bool HALF>
__device__ __forceinline__ void turn(const Angles<VEC, HALF>& w, Pack<T, VEC>& a, Pack<T, VEC>& d) {
  f2 u[kPairs<VEC>], v[kPairs<VEC>];
  unpack<T, VEC>(a, u);
  if constexpr (HALF) {
    unpack<T, VEC>(d, v);
#pragma unroll
    for (int j = 0; j < kPairs<VEC>; ++j) {
      const f2 r = px::fma(u[j], w.c[j], negate(px::mul(v[j], w.s[j])));
      v[j] = px::fma(v[j], w.c[j], px::mul(u[j], w.s[j]));
      u[j] = r;
    }
    d = pack<T, VEC>(v);
  } else {
#pragma unroll
    for (int j = 0; j < kPairs<VEC>; ++j) u[j] = px::fma(u[j], w.c[j], px::mul(swap(u[j]), w.s[j]));
  }
  a = pack<T, VEC>(u);
}

// VEC: elements per access.  The interleaved layout turns VEC / 2 pairs per unit, the half layout VEC.
// threadIdx: (unit, head lane, token lane); blockIdx: (tokens of a batch entry, batch entry).
// ONE: one token lane, so that a token's addresses, position and table row are the block's.
template <typename T, int VEC, bool HALF, bool ONE>
__global__ void __launch_bounds__(512, 3) rotary_kernel(const Params p) {
  using V = Pack<T, VEC>;
  constexpr int NP = HALF ? VEC : VEC / 2;  // pairs per unit
  const int u = threadIdx.x;
  const int64_t s = ONE ? blockIdx.x : (int64_t)blockIdx.x * blockDim.z + threadIdx.z, b = blockIdx.y;
  if (!ONE && s >= p.S) return;
  const bool rot = u < p.rot_units;
  int64_t l = s;
  if (p.pos) {
    const int64_t i = b * p.ps_b + s * p.ps_s;
    l = p.pos64 ? reinterpret_cast<const int64_t*>(p.pos)[i] : (int64_t)reinterpret_cast<const int32_t*>(p.pos)[i];
  }
  // the unit's first vector, the distance to its second one, and whether it has that
  const int at = rot ? u * VEC : p.R + (u - p.rot_units) * VEC;
  const int second = rot ? p.R >> 1 : (p.units - p.rot_units) * VEC;
  const bool two = HALF && at + second < p.D;
  Angles<VEC, HALF> w;
  if (rot) {
    if (l < 0 || l >= p.L) {
      // a position outside the table: the rotated features read NaN and the host learns of it
      atomicExch(&g_zib_err_word, (int)ZIB_ERR_INVALID_ARG);
      const float nan = __uint_as_float(0x7FC00000u);
#pragma unroll
      for (int i = 0; i < NP; ++i) w.set(i, nan, nan);
    } else {
      constexpr int FN = NP >= 4 ? 4 : NP;
      using F = Pack<float, FN>;
      const float* cp = p.cos + b * p.cs_b + l * p.cs_l + u * NP;
      const float* sp = p.sin + b * p.cs_b + l * p.cs_l + u * NP;
#pragma unroll
      for (int i = 0; i < NP; i += FN) {
        F c, t;
        if (p.table_vec) {
          c = *reinterpret_cast<const F*>(cp + i);
          t = *reinterpret_cast<const F*>(sp + i);
        } else {
#pragma unroll
          for (int j = 0; j < FN; ++j) {
            c.v[j] = cp[i + j];
            t.v[j] = sp[i + j];
          }
        }
#pragma unroll
        for (int j = 0; j < FN; ++j) w.set(i + j, c.v[j], p.sign * t.v[j]);
      }
    }
  }
  // this thread's heads, of the queries and then of the keys, one count
  int h = threadIdx.y;
  auto walk = [&](const Heads& hd) {
    const T* x = reinterpret_cast<const T*>(hd.x) + (b * hd.sb + s * hd.ss) + (h * hd.sh + at);
    T* o = reinterpret_cast<T*>(hd.out) + (b * p.S + s) * ((int64_t)hd.H * p.D) + (h * p.D + at);
    const int64_t xstep = blockDim.y * hd.sh, ostep = blockDim.y * p.D;
#pragma unroll 2
    for (; h < hd.H; h += blockDim.y, x += xstep, o += ostep) {
      V a = load_vec<T, VEC>(x), d = a;
      if constexpr (HALF) if (two) d = load_vec<T, VEC>(x + second);
      if (rot) turn<T, VEC, HALF>(w, a, d);
      *reinterpret_cast<V*>(o) = a;
      if constexpr (HALF) if (two) *reinterpret_cast<V*>(o + second) = d;
    }
    h -= hd.H;
  };
  walk(p.q);
  walk(p.k);
}

template <typename T, int VEC, bool HALF>
static void launch_vec(dim3 grid, dim3 threads, const Params& p, cudaStream_t st) {
  if (threads.z == 1) rotary_kernel<T, VEC, HALF, true><<<grid, threads, 0, st>>>(p);
  else rotary_kernel<T, VEC, HALF, false><<<grid, threads, 0, st>>>(p);
}

template <typename T, bool HALF>
static void launch(int vec, dim3 grid, dim3 threads, const Params& p, cudaStream_t st) {
  if constexpr (sizeof(T) == 2) {
    if (vec == 8) { launch_vec<T, 8, HALF>(grid, threads, p, st); return; }
  }
  if (vec == 4) { launch_vec<T, 4, HALF>(grid, threads, p, st); return; }
  if (vec == 2) { launch_vec<T, 2, HALF>(grid, threads, p, st); return; }
  if constexpr (HALF) launch_vec<T, 1, HALF>(grid, threads, p, st);
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

// An angle in fixed point, 2^-64 turns: its nearest multiple of a quarter turn, and the rest, within an
// eighth of a turn, in units of 2^-32 turns as fp32.  The lower word keeps the rest's relative accuracy
// (two roundings) down to 2^-56 turns: the sine of a slow frequency at an early position is as small as
// its angle.
__device__ __forceinline__ uint32_t quarter_of(uint64_t a) { return ((uint32_t)(a >> 32) + 0x20000000u) >> 30; }
__device__ __forceinline__ float high_rest(uint64_t a, uint32_t quarter) {
  return (float)(int32_t)((uint32_t)(a >> 32) - (quarter << 30));
}
__device__ __forceinline__ float low_rest(uint64_t a) { return (float)(uint32_t)a; }
constexpr float kLow = 2.3283064365386963e-10f;     // 2^-32
constexpr float kRadians = 1.4629180792671596e-09f;  // 2 pi / 2^32

// cos and sin of such an angle: the quarter decides which of them is which and their signs, exactly, in
// integers; the rest goes through the Taylor series of sine (to x^9) and cosine (to x^10), whose next
// terms are below 2e-9 and 2e-10 there.  One fp32 for the rest leaves values 2.9e-8 off in the mean (1e-7 at
// most), where the rounding to fp32 alone leaves 2.1e-8; carrying its rounding error too gave 2.2e-8 (6.6e-8) and
// took 35 us instead of 27 for 131072 x 64.
__device__ __forceinline__ void sincos_turns(uint64_t a, float& s, float& c) {
  const uint32_t quarter = quarter_of(a);
  const float x = fmaf(low_rest(a), kLow, high_rest(a, quarter)) * kRadians;
  const float x2 = x * x;
  float ps = 2.7557319e-6f;  // 1 / 9!
  ps = fmaf(ps, x2, -1.9841270e-4f);
  ps = fmaf(ps, x2, 8.3333333e-3f);
  ps = fmaf(ps, x2, -1.6666667e-1f);
  ps = fmaf(ps * x2, x, x);
  float pc = -2.7557319e-7f;  // -1 / 10!
  pc = fmaf(pc, x2, 2.4801587e-5f);
  pc = fmaf(pc, x2, -1.3888889e-3f);
  pc = fmaf(pc, x2, 4.1666667e-2f);
  pc = fmaf(pc, x2, -0.5f);
  pc = fmaf(pc, x2, 1.0f);
  const float u = quarter & 1 ? pc : ps, v = quarter & 1 ? ps : pc;
  s = __uint_as_float(__float_as_uint(u) ^ ((quarter & 2) << 30));
  c = __uint_as_float(__float_as_uint(v) ^ (((quarter + 1) & 2) << 30));
}

// the same of two angles, on packed pairs
__device__ __forceinline__ void sincos_turns2(uint64_t a0, uint64_t a1, float m, float (&s)[2], float (&c)[2]) {
  const uint32_t q[2] = {quarter_of(a0), quarter_of(a1)};
  auto all = [](float v) { return px::mk(v, v); };
  const px::f2 x = px::mul(px::fma(px::mk(low_rest(a0), low_rest(a1)), all(kLow),
                                   px::mk(high_rest(a0, q[0]), high_rest(a1, q[1]))), all(kRadians));
  const px::f2 x2 = px::mul(x, x);
  px::f2 ps = all(2.7557319e-6f);
  ps = px::fma(ps, x2, all(-1.9841270e-4f));
  ps = px::fma(ps, x2, all(8.3333333e-3f));
  ps = px::fma(ps, x2, all(-1.6666667e-1f));
  ps = px::fma(px::mul(ps, x2), x, x);
  px::f2 pc = all(-2.7557319e-7f);
  pc = px::fma(pc, x2, all(2.4801587e-5f));
  pc = px::fma(pc, x2, all(-1.3888889e-3f));
  pc = px::fma(pc, x2, all(4.1666667e-2f));
  pc = px::fma(pc, x2, all(-0.5f));
  pc = px::fma(pc, x2, all(1.0f));
  float sv[2], cv[2];
  px::split(px::mul(ps, all(m)), sv[0], sv[1]);
  px::split(px::mul(pc, all(m)), cv[0], cv[1]);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float u = q[i] & 1 ? cv[i] : sv[i], v = q[i] & 1 ? sv[i] : cv[i];
    s[i] = __uint_as_float(__float_as_uint(u) ^ ((q[i] & 2) << 30));
    c[i] = __uint_as_float(__float_as_uint(v) ^ (((q[i] + 1) & 2) << 30));
  }
}

// cos and sin of p f_j, f_j = theta^(-2j/dim) scaled.  The angle is formed in turns, in fixed point of
// 64 bits: a whole position times a frequency, modulo whole turns, is one wrapping 64-bit product (the
// frequency is rounded to 2^-64 turns, so a position below 2^31 is off by less than 2^-33 turns; the
// fp64 frequency behind it by less than 2^-55 turns a position).  A thread keeps J neighbouring
// frequencies and walks over positions, so the fp64 exp is paid once per thread.
// 131072 x 64 (68 MB, 10.4 us at HBM's rate): 20 us launched alone, 14.3 back to back (a fill of as many
// bytes 10.1; without packed pairs 15.8).  Launched alone, angles in fp64 take 28 us and sincospi of the
// fixed-point angle 26, both short of issue slots.
template <int J>
__global__ void __launch_bounds__(256) rotary_table_kernel(const TableParams p) {
  const int j0 = (blockIdx.y * blockDim.x + threadIdx.x) * J;
  if (j0 >= p.half) return;
  uint64_t turns[J];
#pragma unroll
  for (int i = 0; i < J; ++i) {
    double f = exp(-p.log_theta * (double)(j0 + i) / (double)p.half);
    if (p.kind == ZIB_ROTARY_LINEAR) f *= p.inv_factor;
    if (p.kind == ZIB_ROTARY_YARN) {
      // whole turns over the original length: few turns are interpolated, many are kept
      const double over = p.original * f * 0.15915494309189535;
      const double keep = fmin(1.0, fmax(0.0, (over - p.beta_slow) / (p.beta_fast - p.beta_slow)));
      f = (1.0 - keep) * f * p.inv_factor + keep * f;
    }
    double ft = f * 0.15915494309189535;  // turns per position; whole ones do not matter
    ft -= floor(ft);
    turns[i] = (uint64_t)(ft * 18446744073709551616.0);
  }
  const int64_t step = (int64_t)gridDim.x * blockDim.y;
#pragma unroll 4
  for (int64_t t = (int64_t)blockIdx.x * blockDim.y + threadIdx.y; t < p.T; t += step) {
    int64_t pos = p.start + t;
    if (p.pos)
      pos = p.pos64 ? reinterpret_cast<const int64_t*>(p.pos)[t * p.ps]
                    : (int64_t)reinterpret_cast<const int32_t*>(p.pos)[t * p.ps];
    Pack<float, J> c, s;
    auto angle = [&](int i) { return (uint64_t)pos * turns[i]; };
    if constexpr (J == 2) {
      sincos_turns2(angle(0), angle(1), p.mscale, s.v, c.v);
    } else {
      float sv, cv;
      sincos_turns(angle(0), sv, cv);
      c.v[0] = p.mscale * cv;
      s.v[0] = p.mscale * sv;
    }
    *reinterpret_cast<Pack<float, J>*>(p.cos + t * p.half + j0) = c;
    *reinterpret_cast<Pack<float, J>*>(p.sin + t * p.half + j0) = s;
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
  p.S = S; p.D = (int)D; p.R = (int)R;
  p.rot_units = (int)(part / vec);
  p.units = p.rot_units + (int)ceil_div(D - R, half_layout ? 2 * vec : vec);
  p.sign = inverse ? -1.0f : 1.0f;
  const int np = half_layout ? vec : vec / 2, fn = np >= 4 ? 4 : np;
  p.table_vec = ((uintptr_t)cos % (4 * fn) == 0 && (uintptr_t)sin % (4 * fn) == 0 && cs_l % fn == 0 && cs_b % fn == 0);
  // Heads per thread: one where the tokens alone do not fill the SMs (latency); else as many, up to 16,
  // as leave about 64 threads to a token, which pays for a token's addresses and table row over more
  // heads (256 / 128 / 64 / 32 threads a token: 64 / 59 / 59 / 67 us for [2, 4608, 30 + 30, 128]
  // interleaved, 72 / 64 / 55 / 57 us for [16383, 24 + 6, 128] half, 64 of 128 features).
  const int64_t heads = Hq + Hk;
  int64_t per = 1;
  if (B * S >= 4 * sm_count()) {
    per = (heads * p.units + 32) / 64;
    if (per < 1) per = 1;
    if (per > 16) per = 16;
  }
  int64_t lanes = ceil_div(heads, per);
  if (lanes * p.units > 512) lanes = 512 / p.units;  // units <= 512: a unit has two features at least
  int64_t tokens = 128 / (p.units * lanes);
  if (tokens > S) tokens = S;
  if (tokens > 64) tokens = 64;
  if (tokens < 1) tokens = 1;
  const dim3 threads(p.units, (unsigned)lanes, (unsigned)tokens), g((unsigned)ceil_div(S, tokens), (unsigned)B);
  ZIB_HOST_CHECK(ceil_div(S, tokens) <= 0x7FFFFFFF && B <= 65535, ZIB_ERR_TOO_LARGE,
                 "%s: at most 65535 batch entries, got %lld", what, (long long)B);
  cudaStream_t st = (cudaStream_t)stream;
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
  const bool two = p.half % 2 == 0 && (uintptr_t)cos % 8 == 0 && (uintptr_t)sin % 8 == 0;
  const int cols = two ? p.half / 2 : p.half;
  const int bx = cols > 16 ? 32 : 16;
  dim3 block(bx, 256 / bx);
  const int64_t gy = ceil_div(cols, bx);
  int64_t gx = ceil_div(T, (int64_t)block.y * 4);
  const int64_t cap = ceil_div((int64_t)sm_count() * 6, gy);
  if (gx > cap) gx = cap;
  const dim3 grid((unsigned)gx, (unsigned)gy);
  if (two) rotary::rotary_table_kernel<2><<<grid, block, 0, (cudaStream_t)stream>>>(p);
  else rotary::rotary_table_kernel<1><<<grid, block, 0, (cudaStream_t)stream>>>(p);
  return zib_check_launch(what);
}
