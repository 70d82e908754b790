// Block-scaled 8-bit product on 5th-generation tensor cores (tcgen05) for sm_100a: for any scales by sums in
// registers (kind::f8f6f4), and for powers of two by the tensor cores' own scales (kind::mxf8f6f4, below).
//
//   y[m, n] = sum_b sx[m, b] sw[n / 128, b] sum_{k in block b} q[m, k] w[n, k]  (+ bias[n])
//
// The tensor cores sum one block of 128 products per accumulator; the scales differ from block to
// block, so the sum over blocks is formed outside of them, in fp32 registers, from s = sx sw in fp32 (scales whose
// product leaves fp32's range are not for this kernel).
//
// The accumulators hold fp32's 24 bits, here, with the tensor cores' scales and in mma.sync alike (measured: 2^-23
// beside 1 survives in the same step of 32 products, in another one of its block and in other blocks).  A step
// counts terms down to 2^-25 of its largest and cuts its sum to 24 bits instead of rounding it, so it errs by at
// most 33 2^-25 + 2^-23 of that, less than 32 additions in fp32 may.  One accumulator for all of K is therefore
// fp32 arithmetic too; sums of one sign come out low rather than to either side.
//
// Design (persistent, warp-specialised, clusters of two CTAs, tiles of 256 rows x BN columns):
//   warp 0     TMA producer: 128-byte swizzled K-major boxes, one K-block of 128 per stage (each CTA
//              stages its 128 rows of q and half of the BN rows of w).
//   warp 1     issues tcgen05.mma (cta_group::2, 256 x BN x 32).  Every K-block starts a fresh
//              accumulator; the 512 TMEM columns hold 512 / BN of them, so the MMAs run ahead of the
//              warps that empty them.  The whole warp waits and one elected thread issues: descriptors
//              stay uniform, and four MMAs and two commits take 140 clocks instead of 380.
//   warps 4-11 add s * accumulator to their registers: the warps w and w + 4 share a TMEM lane
//              quarter (32 rows) and take half of the BN columns each.  A thread owns one row, so the
//              row's scale is one value; its BN / 2 columns lie in one block of 128 weight rows, so
//              that scale is one value too: one packed multiply-add per two elements and K-block.
//              The output tile leaves through shared memory and TMA stores that drain while the
//              next tile is summed.
// What bounds the sums in registers at 18432 x 11520 x 3840 (686 us, 2380 TFLOP/s): the way of one accumulator from the MMAs
// to registers and back, 565 ns a K-block with two of them under way (the MMAs alone take 270, the
// operands arrive every 320).  Without the sums between blocks the same pipeline runs at 580 us
// (2810 TFLOP/s), where the library's product with one scale a tensor is too.  Measured on that way:
// release at cluster scope 1805 us, one thread waiting and issuing 840 us, accumulators of 128 columns
// in two halves of the tile 790 us (the rows of q are read twice), tiles of 256 x 128 throughout 1030 us,
// the next accumulator's loads behind the current sums 800 us.  Tiles of 256 x 128 take 285 ns a K-block,
// with 2 to 4 accumulators and 3 to 6 stages alike.
// Every mbarrier wait is bounded; on expiry the CTA records ZIB_ERR_TIMEOUT in a device error word,
// drains its loads and MMAs, frees TMEM and exits.
#include "fp8_quant.cuh"
#include "rot_pack.cuh"
#include "zib_tcgen05.cuh"

ZIB_DEFINE_ERROR_READER(zib_err_read_clear_fp8)

namespace zib {
namespace fp8 {

using namespace tc;

constexpr int kEpiWarps = 8;
constexpr int kThreads = (4 + kEpiWarps) * 32;
constexpr int kTmemCols = 512;
constexpr int kABytes = 128 * kBlock;

template <int BN>
struct Cfg {
  static constexpr int BUFS = kTmemCols / BN;  // accumulators in flight
  // Registers: 384 threads start with 168 each (64512); the first warpgroup keeps REGS_ISSUE, the two
  // that sum take REGS_SUM: 128 * 40 + 256 * 232 = 128 * 56 + 256 * 224 = 64512.
  static constexpr int REGS_ISSUE = BN == 256 ? 40 : 56, REGS_SUM = BN == 256 ? 232 : 224;
  static constexpr int STAGE = kABytes + BN / 2 * kBlock;
  static constexpr int STAGES = BN == 256 ? 5 : 6;
  static constexpr int XWARP = 8192;  // output staging per warp: two boxes of 32 rows x 128 bytes
  // bytes of a warp's copy of its bias; tiles of 256 columns leave no room for one
  static constexpr int BIAS = BN == 128 ? BN / 2 * 4 : 0;
  static constexpr int SMEM = STAGES * STAGE + kEpiWarps * (XWARP + BIAS) + 256 + 1024;
  static_assert(SMEM <= 232448, "shared memory per CTA");
};

// D = f32, A = B = e4m3, both K-major
__host__ __device__ constexpr uint32_t idesc_f8(int M, int N) {
  return (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

struct GemmParams {
  int M, N;
  int num_mb, num_nb, num_kb, num_tiles;
  int n_fast, group;
  const float* sx;
  int64_t sx_m, sx_k;
  const float* sw;
  int64_t sw_n, sw_k;
  const void* bias;
  void* y;
  int64_t ldy;
  int tma_store;  // y's rows are 16-byte aligned
  int where;      // 0: any scales; 1: only where the weight's are not powers of two
};

// one tcgen05.mma of K = 32; acc is a constant after unrolling
__device__ __forceinline__ void umma_f8_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool acc) {
  if (acc)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.eq.u32 p, 0, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, 0, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc)
        : "memory");
}

// true in one thread of a converged warp
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r != 0;
}

// bounded wait of a converged warp: the same answer in every thread
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  return __all_sync(0xFFFFFFFFu, mbar_try_wait(bar, parity) || mbar_wait_bounded(bar, parity, abort_flag));
}

// Arrival on a barrier of the cluster with the default (CTA-scope) release: the accumulator was
// read by completed tcgen05.ld, ordered by the tcgen05 fence before it.  A release at cluster scope
// also waits for the thread's global loads in flight (the coming scales): 1805 -> 840 us at
// 18432 x 11520 x 3840, where every K-block arrives once.
__device__ __forceinline__ void arrive_pair(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

// waits for this thread's TMEM loads; the values are tied in so that no use of them moves above the wait
#define ZIB_R8(r, i) "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3]), "+r"(r[i + 4]), "+r"(r[i + 5]), \
                     "+r"(r[i + 6]), "+r"(r[i + 7])
__device__ __forceinline__ void wait_ld(uint32_t (&a)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" : ZIB_R8(a, 0), ZIB_R8(a, 8), ZIB_R8(a, 16), ZIB_R8(a, 24) : : "memory");
}
// the same tie for a second array of the same wait
__device__ __forceinline__ void after_wait(uint32_t (&a)[32]) {
  asm volatile("" : ZIB_R8(a, 0), ZIB_R8(a, 8), ZIB_R8(a, 16), ZIB_R8(a, 24));
}
#undef ZIB_R8

__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, const void* src, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(smem_u32(src)), "r"(x), "r"(y)
               : "memory");
}

// Launched behind the quantiser that writes q and its scales, the kernel may start before that has
// ended: set-up overlaps its tail (2 to 3 us of a call on few rows), and what reads them waits here.
__device__ __forceinline__ void wait_for_primary() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Tile t -> (M-block, N-block): the fast index runs in groups whose rows stay in L2 while the
// tiles sweep the slow index (the same order as the int8 GEMM's).
__device__ __forceinline__ void tile_at(const GemmParams& p, int tile, int& mb, int& nb) {
  const int nfast = p.n_fast ? p.num_nb : p.num_mb, nslow = p.n_fast ? p.num_mb : p.num_nb;
  const int per_group = p.group * nslow;
  const int g = tile / per_group, r = tile - g * per_group;
  const int gsize = min(p.group, nfast - g * p.group);
  const int f = g * p.group + r % gsize, sl = r / gsize;
  nb = p.n_fast ? f : sl;
  mb = p.n_fast ? sl : f;
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&h);
}

// acc[at .. at + 15] (pairs of columns) += s * r
template <int N2>
__device__ __forceinline__ void add_scaled(px::f2 (&acc)[N2], int at, const uint32_t (&r)[32], px::f2 s2) {
#pragma unroll
  for (int j = 0; j < 16; ++j)
    acc[at + j] = px::fma(px::mk(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1])), s2, acc[at + j]);
}

// This thread's CW columns of row `row` to y, through the warp's staging boxes (32 rows x 128 bytes,
// 16-byte chunk c of row r at c ^ (r & 7): the TMA's 128-byte swizzle).
template <typename T, int CW, bool SB = false>
__device__ __forceinline__ void store_tile(const GemmParams& p, const CUtensorMap* map_y, px::f2 (&acc)[CW / 2],
                                           uint8_t* xw, int row0, int n0, int lane,
                                           const float* sbias = nullptr) {
  constexpr int BOXC = 128 / sizeof(T);            // columns per box
  constexpr int BOXES = CW / BOXC;                 // boxes of this warp's part
  constexpr int PER = BOXES < 2 ? BOXES : 2;       // staged at a time
#pragma unroll
  for (int b0 = 0; b0 < BOXES; b0 += PER) {
    if (p.tma_store) {  // the boxes' previous contents have been read
      if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
    }
    __syncwarp();
#pragma unroll
    for (int b = 0; b < PER; ++b) {
      const int col = (b0 + b) * BOXC;  // first of the box's columns
      uint8_t* line = xw + b * 4096 + lane * 128;
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        constexpr int EC = 16 / sizeof(T);  // columns per 16-byte chunk
        float v[EC];
#pragma unroll
        for (int j = 0; j < EC; j += 2) px::split(acc[(col + c * EC + j) / 2], v[j], v[j + 1]);
        if (SB && p.bias) {  // the bias of these columns is in shared memory
#pragma unroll
          for (int j = 0; j < EC; j += 4) {
            const float4 t = *reinterpret_cast<const float4*>(sbias + col + c * EC + j);
            v[j] += t.x, v[j + 1] += t.y, v[j + 2] += t.z, v[j + 3] += t.w;
          }
        } else if (p.bias) {
          const int n = n0 + col + c * EC;
          const T* from = reinterpret_cast<const T*>(p.bias) + n;
          if (reinterpret_cast<uintptr_t>(p.bias) % 16 == 0 && n + EC <= p.N) {
            const Pack<T, EC> t = *reinterpret_cast<const Pack<T, EC>*>(from);
#pragma unroll
            for (int j = 0; j < EC; ++j) v[j] += to_f32(t.v[j]);
          } else {
#pragma unroll
            for (int j = 0; j < EC; ++j)
              if (n + j < p.N) v[j] += to_f32(from[j]);
          }
        }
        uint4 o;
        if constexpr (sizeof(T) == 2) {
          o = make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
        } else {
          o = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
        }
        *reinterpret_cast<uint4*>(line + ((c ^ (lane & 7)) << 4)) = o;
      }
    }
    if (p.tma_store) {
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0 && row0 < p.M) {
#pragma unroll
        for (int b = 0; b < PER; ++b)
          if (n0 + (b0 + b) * BOXC < p.N) tma_store_2d(map_y, xw + b * 4096, n0 + (b0 + b) * BOXC, row0);
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
      }
    } else {
      __syncwarp();
      // rows that start on any element: single elements, a few rows' reads under way at a time (18226 x 4071 x
      // 640: 100 us, 190 one after the other, 166 in pairs where a row's parity allows)
      constexpr int RUN = 4;
#pragma unroll 1
      for (int r0 = 0; r0 < 32 && row0 + r0 < p.M; r0 += RUN) {
#pragma unroll
        for (int b = 0; b < PER; ++b) {
          const int col = n0 + (b0 + b) * BOXC + lane;
          T v[RUN][BOXC / 32];
#pragma unroll
          for (int i = 0; i < RUN; ++i)
#pragma unroll
            for (int e = 0; e < BOXC / 32; ++e) {
              const int r = r0 + i, at = (lane + 32 * e) * (int)sizeof(T);
              v[i][e] = *reinterpret_cast<const T*>(xw + b * 4096 + r * 128 + (((at >> 4) ^ (r & 7)) << 4) + (at & 15));
            }
          T* dst = reinterpret_cast<T*>(p.y) + (int64_t)(row0 + r0) * p.ldy + col;
#pragma unroll
          for (int i = 0; i < RUN; ++i)
#pragma unroll
            for (int e = 0; e < BOXC / 32; ++e)
              if (row0 + r0 + i < p.M && col + 32 * e < p.N) dst[i * p.ldy + 32 * e] = v[i][e];
        }
      }
      __syncwarp();
    }
  }
}

// every scale of the weight is a normal power of two (all CTAs find the same; the weight's scales are
// not written by the launch before)
__device__ __forceinline__ bool powers_of_two(const GemmParams& p) {
  const int rows = (p.N + kBlock - 1) / kBlock, n = rows * p.num_kb;
  bool ok = true;
#pragma unroll 8
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const int r = i / p.num_kb, k = i - r * p.num_kb;
    const uint32_t b = __float_as_uint(__ldg(p.sw + r * p.sw_n + k * p.sw_k));
    ok &= ((b & 0x7FFFFFu) == 0) & (b - 1 < 0x7F7FFFFFu);
  }
  return __syncthreads_and(ok) != 0;
}

template <typename T, int BN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    gemm_pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                     const __grid_constant__ CUtensorMap map_y, const GemmParams p) {
  using C = Cfg<BN>;
  constexpr int STAGES = C::STAGES, BUFS = C::BUFS, CW = BN / 2;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* xbuf = smem + STAGES * C::STAGE;
  uint64_t* bars = reinterpret_cast<uint64_t*>(xbuf + kEpiWarps * (C::XWARP + C::BIAS));
  uint64_t* full_bar = bars;                       // leader's is used
  uint64_t* empty_bar = bars + STAGES;             // both
  uint64_t* tfull_bar = bars + 2 * STAGES;         // both
  uint64_t* tempty_bar = tfull_bar + BUFS;         // leader's is used
  uint64_t* mma_done_bar = tempty_bar + BUFS;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(mma_done_bar + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  static_assert((2 * STAGES + 2 * BUFS + 1) * 8 + 8 <= 256, "barrier area");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const bool leader = rank == 0;
  const int cluster_id = blockIdx.x >> 1, nclusters = gridDim.x >> 1;
  if (p.where && powers_of_two(p)) return;  // the whole grid

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < BUFS; ++a) {
      mbar_init(&tfull_bar[a], 1);
      mbar_init(&tempty_bar[a], 2 * kEpiWarps);  // epilogue warps of both CTAs
    }
    mbar_init(mma_done_bar, 1);
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&map_a);
    tma_prefetch_desc(&map_b);
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_holder)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // both CTAs' barriers are initialised before any cross-CTA signal
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;
  bool aborted = false;

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::REGS_ISSUE));
    if (warp == 0) {  // ---- TMA producer (both CTAs): the whole warp waits, one elected thread issues
      wait_for_primary();  // q
      int stage = 0;
      uint32_t phase = 0, pend_mask = 0, pend_parity = 0;
      bool ok = true;
      const uint32_t full0 = leader ? smem_u32(full_bar) : mapa_rank(smem_u32(full_bar), 0);
      for (int t = cluster_id; t < p.num_tiles && ok; t += nclusters) {
        int mb, nb;
        tile_at(p, t, mb, nb);
        const int row_a = mb * 256 + (int)rank * 128, row_b = nb * BN + (int)rank * (BN / 2);
        for (int kb = 0; kb < p.num_kb; ++kb) {
          if (!warp_wait(&empty_bar[stage], phase ^ 1u, abort_flag)) { ok = false; break; }
          uint8_t* st = smem + stage * C::STAGE;
          if (elect_one()) {
            if (leader) mbar_arrive_expect_tx(&full_bar[stage], 2 * C::STAGE);
            tma_load_2d_pair(st, &map_a, full0 + 8 * stage, kb * kBlock, row_a);
            tma_load_2d_pair(st + kABytes, &map_b, full0 + 8 * stage, kb * kBlock, row_b);
          }
          __syncwarp();
          pend_mask |= 1u << stage;
          pend_parity = (pend_parity & ~(1u << stage)) | (phase << stage);
          if (++stage == STAGES) { stage = 0; phase ^= 1u; }
        }
      }
      if (!ok) {
        aborted = true;
        if (leader)
          for (int s = 0; s < STAGES; ++s)
            if (pend_mask & (1u << s)) mbar_drain_wait(&full_bar[s], (pend_parity >> s) & 1u);
      }
    }
    if (warp == 1 && leader) {  // ---- MMA issuer: the whole warp waits, one elected thread issues
      int stage = 0, buf = 0;
      uint32_t phase = 0, buf_phase = 0;
      bool ok = true;
      const uint32_t base = smem_u32(smem);
      constexpr uint32_t idesc = idesc_f8(256, BN);
      for (int t = cluster_id; t < p.num_tiles && ok; t += nclusters) {
        for (int kb = 0; kb < p.num_kb; ++kb) {
          if (!warp_wait(&full_bar[stage], phase, abort_flag)) { ok = false; break; }
          const uint64_t adesc = sdesc_sw128(base + stage * C::STAGE);
          const uint64_t bdesc = sdesc_sw128(base + stage * C::STAGE + kABytes);
          if (!warp_wait(&tempty_bar[buf], buf_phase ^ 1u, abort_flag)) { ok = false; break; }
          tc_fence_after();
          const uint32_t d = tmem_base + (uint32_t)(buf * BN);
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < kBlock / 32; ++k)
              umma_f8_pair(d, adesc + (uint64_t)(k * 2), bdesc + (uint64_t)(k * 2), idesc, k != 0);
            umma_commit_pair(&tfull_bar[buf], (uint16_t)3);
            umma_commit_pair(&empty_bar[stage], (uint16_t)3);  // frees the stage in both CTAs
          }
          __syncwarp();
          if (++buf == BUFS) { buf = 0; buf_phase ^= 1u; }
          if (++stage == STAGES) { stage = 0; phase ^= 1u; }
        }
      }
      if (!ok) aborted = true;
      if (elect_one()) {
        umma_commit_pair(mma_done_bar, (uint16_t)1);
        mbar_drain_wait(mma_done_bar, 0);
      }
    }
    __syncwarp();
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::REGS_SUM));
    // ---- sums over K-blocks and output (both CTAs)
    const int quarter = warp & 3, half = (warp - 4) >> 2;
    uint8_t* xw = xbuf + (warp - 4) * C::XWARP;
    float* sbias = reinterpret_cast<float*>(xbuf + kEpiWarps * C::XWARP + (warp - 4) * C::BIAS);
    const uint32_t tempty0 = mapa_rank(smem_u32(tempty_bar), 0);
    const uint32_t t_warp = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(half * CW);
    int buf = 0;
    uint32_t buf_phase = 0;
    bool ok = true;
    // scales of the coming K-block, loaded one ahead
    const float *px_ = nullptr, *pw_ = nullptr;
    int mb = 0, nb = 0;
    float sx = 0.0f, sw = 0.0f;
    auto locate = [&](int t) {
      tile_at(p, t, mb, nb);
      const int row = mb * 256 + (int)rank * 128 + quarter * 32 + lane, n0 = nb * BN + half * CW;
      px_ = row < p.M ? p.sx + row * p.sx_m : nullptr;
      pw_ = n0 < p.N ? p.sw + (n0 / kBlock) * p.sw_n : nullptr;
      sx = px_ ? __ldg(px_) : 0.0f;
      sw = pw_ ? __ldg(pw_) : 0.0f;
    };
    wait_for_primary();  // the scales of q
    if (cluster_id < p.num_tiles) locate(cluster_id);
    for (int t = cluster_id; t < p.num_tiles && ok; t += nclusters) {
      const int row0 = mb * 256 + (int)rank * 128 + quarter * 32, n0 = nb * BN + half * CW;
      if (C::BIAS > 0 && p.bias) {
        __syncwarp();
#pragma unroll
        for (int c = lane; c < CW; c += 32)
          sbias[c] = n0 + c < p.N ? to_f32(reinterpret_cast<const T*>(p.bias)[n0 + c]) : 0.0f;
        __syncwarp();
      }
      px::f2 acc[CW / 2];
#pragma unroll
      for (int j = 0; j < CW / 2; ++j) acc[j] = 0ull;
      for (int kb = 0; kb < p.num_kb; ++kb) {
        const float s = sx * sw;
        const px::f2 s2 = px::mk(s, s);
        if (kb + 1 < p.num_kb) {
          sx = px_ ? __ldg(px_ + (kb + 1) * p.sx_k) : 0.0f;
          sw = pw_ ? __ldg(pw_ + (kb + 1) * p.sw_k) : 0.0f;
        }
        if (!warp_wait(&tfull_bar[buf], buf_phase, abort_flag)) { ok = false; break; }
        tc_fence_after();
        const uint32_t ta = t_warp + (uint32_t)(buf * BN);
        uint32_t r0[32], r1[32];
        tmem_ld32(ta, r0);
        tmem_ld32(ta + 32u, r1);
        wait_ld(r0);
        after_wait(r1);
        if constexpr (CW == 128) {
          add_scaled(acc, 0, r0, s2);
          tmem_ld32(ta + 64u, r0);
          add_scaled(acc, 16, r1, s2);
          tmem_ld32(ta + 96u, r1);
          wait_ld(r0);
          after_wait(r1);
        }
        // read: the accumulator may be filled again
        tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive_pair(tempty0 + 8 * buf);
        add_scaled(acc, CW / 2 - 32, r0, s2);
        add_scaled(acc, CW / 2 - 16, r1, s2);
        if (++buf == BUFS) { buf = 0; buf_phase ^= 1u; }
      }
      if (!ok) break;
      if (t + nclusters < p.num_tiles) locate(t + nclusters);
      store_tile<T, CW, (C::BIAS > 0)>(p, &map_y, acc, xw, row0, n0, lane, sbias);
    }
    if (!ok) aborted = true;
    if (p.tma_store && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    __syncwarp();
  }

  // An aborted CTA gives copies still in flight (the peer's loads complete on the leader's
  // barrier) a bounded grace period before the CTAs leave.
  if (__syncthreads_or(aborted ? 1 : 0)) {
    const unsigned long long t0 = globaltimer();
    while (globaltimer() - t0 < 2000000ull) {
    }
  }
  tc_fence_before();
  cluster_sync_all();  // both CTAs are done with TMEM and with each other's barriers
  tc_fence_after();
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kTmemCols)
                 : "memory");
}

// --- scales that the tensor cores apply -----------------------------------------------

// Where the weight's scales are powers of two as the activations' are, both are exponents: the tensor
// cores multiply them in (tcgen05.mma kind::mxf8f6f4, a scale of 8 exponent bits for each row and 32
// columns; a block of 128 has the same one four times), and the sum over all K-blocks stays in one
// accumulator.
//
// Tiles of 256 x 192 by pairs of CTAs: two accumulators of 192 columns leave 128 of TMEM's 512 for the
// scales of the stages in flight (16 each).
//   warp 0     TMA producer, as above
//   warp 1     MMA issuer
//   warps 4-7  output: TMEM to registers, through shared memory to TMA stores, while the next tile is summed
//   warps 8-11 scales: every stage's 128 exponents of rows (4 columns) and 192 of weight rows (6 columns,
//              each of 32 equal ones) to TMEM, once per lane quarter
// 18432 x 11520 x 3840: 608 us (2680 TFLOP/s; 695 for the sums in registers, timed in turns), 4608 x 3840 x
// 10240: 133 us (174).  Bound by the operands' way from L2 (28 KB an SM and K-block) and, with one
// K-block's scales on their way at a time, by those: 779 us; two 614, four 609, six 608, ten 619, six over
// the ends of tiles (more instructions per K-block) 640; without any loads of scales 579.
// A weight with another scale anywhere is left to the kernel above, launched behind this one, which
// otherwise ends at once.
struct Mx {
  static constexpr int BN = 192;
  static constexpr int STAGES = 6;
  static constexpr int STAGE = kABytes + BN / 2 * kBlock;
  static constexpr int AHEAD = 6;  // K-blocks whose scales are on their way
  static constexpr int XWARP = 8192;
  static constexpr int SCALES = 2 * BN;  // first TMEM column of the scales
  static constexpr int BIAS = BN * 4;  // bytes of a warp's copy of a tile's bias
  static constexpr int SMEM = STAGES * STAGE + 4 * (XWARP + BIAS) + 256 + 1024;
  static_assert(SMEM <= 232448, "shared memory per CTA");
  static_assert(SCALES + 16 * STAGES <= kTmemCols, "TMEM columns");
  // D = f32, A = B = e4m3, both K-major, scales of 8 exponent bits, the first byte of their words
  static constexpr uint32_t IDESC = ((uint32_t)(BN >> 3) << 17) | (1u << 23) | ((uint32_t)(256 >> 7) << 27);
};

__device__ __forceinline__ void umma_mx_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t sa, uint32_t sb, bool acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(Mx::IDESC), "r"(sa), "r"(sb), "r"((uint32_t)acc)
      : "memory");
}
__device__ __forceinline__ void tmem_st4(uint32_t taddr, const uint32_t (&v)[4]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(taddr), "r"(v[0]), "r"(v[1]),
               "r"(v[2]), "r"(v[3])
               : "memory");
}
// the exponent of a power of two (255: NaN), four times
__device__ __forceinline__ uint32_t exponents(float s) {
  return ((__float_as_uint(s) >> 23) & 0xFFu) * 0x01010101u;
}

template <typename T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    gemm_mx_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                   const __grid_constant__ CUtensorMap map_y, const GemmParams p) {
  constexpr int STAGES = Mx::STAGES, BN = Mx::BN;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* xbuf = smem + STAGES * Mx::STAGE;
  uint64_t* bars = reinterpret_cast<uint64_t*>(xbuf + 4 * (Mx::XWARP + Mx::BIAS));
  uint64_t* full_bar = bars;                 // leader's is used
  uint64_t* empty_bar = bars + STAGES;       // both
  uint64_t* tfull_bar = bars + 2 * STAGES;   // both
  uint64_t* tempty_bar = tfull_bar + 2;      // leader's is used
  uint64_t* mma_done_bar = tempty_bar + 2;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(mma_done_bar + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  static_assert((2 * STAGES + 5) * 8 + 8 <= 256, "barrier area");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const bool leader = rank == 0;
  const int cluster_id = blockIdx.x >> 1, nclusters = gridDim.x >> 1;
  if (!powers_of_two(p)) {  // the whole grid; the launch behind this one counts on the quantiser's end
    wait_for_primary();
    return;
  }

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 1 + 2 * 4);  // the operands, the scale warps of both CTAs
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull_bar[a], 1);
      mbar_init(&tempty_bar[a], 2 * 4);  // output warps of both CTAs
    }
    mbar_init(mma_done_bar, 1);
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&map_a);
    tma_prefetch_desc(&map_b);
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_holder)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // both CTAs' barriers are initialised before any cross-CTA signal
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;
  bool ok = true;
  wait_for_primary();  // q and its scales

  if (warp == 0) {  // ---- TMA producer (both CTAs): the whole warp waits, one elected thread issues
    int stage = 0;
    uint32_t phase = 0;
    const uint32_t full0 = leader ? smem_u32(full_bar) : mapa_rank(smem_u32(full_bar), 0);
    for (int t = cluster_id; t < p.num_tiles && ok; t += nclusters) {
      int mb, nb;
      tile_at(p, t, mb, nb);
      const int row_a = mb * 256 + (int)rank * 128, row_b = nb * BN + (int)rank * (BN / 2);
      for (int kb = 0; kb < p.num_kb; ++kb) {
        if (!warp_wait(&empty_bar[stage], phase ^ 1u, abort_flag)) { ok = false; break; }
        uint8_t* st = smem + stage * Mx::STAGE;
        if (elect_one()) {
          if (leader) mbar_arrive_expect_tx(&full_bar[stage], 2 * Mx::STAGE);
          tma_load_2d_pair(st, &map_a, full0 + 8 * stage, kb * kBlock, row_a);
          tma_load_2d_pair(st + kABytes, &map_b, full0 + 8 * stage, kb * kBlock, row_b);
        }
        __syncwarp();
        if (++stage == STAGES) { stage = 0; phase ^= 1u; }
      }
    }
  } else if (warp == 1) {
    if (leader) {  // ---- MMA issuer: the whole warp waits, one elected thread issues
      int stage = 0, buf = 0;
      uint32_t phase = 0, buf_phase = 0;
      const uint32_t base = smem_u32(smem);
      for (int t = cluster_id; t < p.num_tiles && ok; t += nclusters) {
        if (!warp_wait(&tempty_bar[buf], buf_phase ^ 1u, abort_flag)) { ok = false; break; }
        const uint32_t d = tmem_base + (uint32_t)(buf * BN);
        for (int kb = 0; kb < p.num_kb; ++kb) {
          if (!warp_wait(&full_bar[stage], phase, abort_flag)) { ok = false; break; }
          tc_fence_after();
          const uint64_t adesc = sdesc_sw128(base + stage * Mx::STAGE);
          const uint64_t bdesc = sdesc_sw128(base + stage * Mx::STAGE + kABytes);
          const uint32_t sc = tmem_base + (uint32_t)(Mx::SCALES + 16 * stage);
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < kBlock / 32; ++k)
              umma_mx_pair(d, adesc + (uint64_t)(k * 2), bdesc + (uint64_t)(k * 2), sc, sc + 4u, kb + k != 0);
            umma_commit_pair(&empty_bar[stage], (uint16_t)3);  // frees the stage in both CTAs
            if (kb + 1 == p.num_kb) umma_commit_pair(&tfull_bar[buf], (uint16_t)3);
          }
          __syncwarp();
          if (++stage == STAGES) { stage = 0; phase ^= 1u; }
        }
        if (++buf == 2) { buf = 0; buf_phase ^= 1u; }
      }
      if (elect_one()) {
        umma_commit_pair(mma_done_bar, (uint16_t)1);
        mbar_drain_wait(mma_done_bar, 0);
      }
    }
  } else if (warp >= 8) {  // ---- scales (both CTAs)
    const int quarter = warp & 3;
    const uint32_t full0 = mapa_rank(smem_u32(full_bar), 0);
    const uint32_t t_warp = tmem_base + ((uint32_t)(quarter * 32) << 16) + Mx::SCALES;
    int stage = 0;
    uint32_t phase = 0;
    for (int t = cluster_id; t < p.num_tiles && ok; t += nclusters) {
      int mb, nb;
      tile_at(p, t, mb, nb);
      const int row0 = mb * 256 + (int)rank * 128 + lane, n = nb * BN + lane * 32;  // lanes 0 .. 5: a column each
      const float* pa[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) pa[c] = row0 + 32 * c < p.M ? p.sx + (row0 + 32 * c) * p.sx_m : nullptr;
      const float* pb = lane < BN / 32 && n < p.N ? p.sw + (n / kBlock) * p.sw_n : nullptr;
      float a[Mx::AHEAD][4], b[Mx::AHEAD];  // of the coming K-blocks
      auto load = [&](int r, int kb) {
#pragma unroll
        for (int c = 0; c < 4; ++c) a[r][c] = pa[c] && kb < p.num_kb ? __ldg(pa[c] + kb * p.sx_k) : 1.0f;
        b[r] = pb && kb < p.num_kb ? __ldg(pb + kb * p.sw_k) : 1.0f;
      };
#pragma unroll
      for (int r = 0; r < Mx::AHEAD; ++r) load(r, r);
      for (int kb0 = 0; kb0 < p.num_kb && ok; kb0 += Mx::AHEAD) {
#pragma unroll
        for (int r = 0; r < Mx::AHEAD; ++r) {
          if (kb0 + r >= p.num_kb) break;
          uint32_t va[4], b0[4], b1[4];
          const uint32_t e = exponents(b[r]);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            va[c] = exponents(a[r][c]);
            b0[c] = __shfl_sync(0xFFFFFFFFu, e, c);
            b1[c] = __shfl_sync(0xFFFFFFFFu, e, 4 + c);
          }
          load(r, kb0 + r + Mx::AHEAD);
          if (!warp_wait(&empty_bar[stage], phase ^ 1u, abort_flag)) { ok = false; break; }
          tc_fence_after();
          const uint32_t at = t_warp + (uint32_t)(16 * stage);
          tmem_st4(at, va);
          tmem_st4(at + 4u, b0);
          tmem_st4(at + 8u, b1);
          asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
          tc_fence_before();
          __syncwarp();
          if (lane == 0) arrive_pair(full0 + 8 * stage);
          if (++stage == STAGES) { stage = 0; phase ^= 1u; }
        }
      }
    }
  } else if (warp >= 4) {  // ---- output (both CTAs)
    const int quarter = warp & 3;
    uint8_t* xw = xbuf + (warp - 4) * Mx::XWARP;
    float* sbias = reinterpret_cast<float*>(xbuf + 4 * Mx::XWARP + (warp - 4) * Mx::BIAS);
    const uint32_t tempty0 = mapa_rank(smem_u32(tempty_bar), 0);
    int buf = 0;
    uint32_t buf_phase = 0;
    for (int t = cluster_id; t < p.num_tiles && ok; t += nclusters) {
      int mb, nb;
      tile_at(p, t, mb, nb);
      const int row0 = mb * 256 + (int)rank * 128 + quarter * 32, n0 = nb * BN;
      if (p.bias) {
        __syncwarp();
#pragma unroll
        for (int c = lane; c < BN; c += 32)
          sbias[c] = n0 + c < p.N ? to_f32(reinterpret_cast<const T*>(p.bias)[n0 + c]) : 0.0f;
        __syncwarp();
      }
      if (!warp_wait(&tfull_bar[buf], buf_phase, abort_flag)) { ok = false; break; }
      tc_fence_after();
      const uint32_t ta = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(buf * BN);
#pragma unroll 1
      for (int c = 0; c < BN / 64; ++c) {
        uint32_t r0[32], r1[32];
        tmem_ld32(ta + 64u * c, r0);
        tmem_ld32(ta + 64u * c + 32u, r1);
        wait_ld(r0);
        after_wait(r1);
        if (c + 1 == BN / 64) {  // read: the accumulator may be filled again
          tc_fence_before();
          __syncwarp();
          if (lane == 0) arrive_pair(tempty0 + 8 * buf);
        }
        px::f2 v[32];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          v[j] = px::mk(__uint_as_float(r0[2 * j]), __uint_as_float(r0[2 * j + 1]));
          v[16 + j] = px::mk(__uint_as_float(r1[2 * j]), __uint_as_float(r1[2 * j + 1]));
        }
        store_tile<T, 64, true>(p, &map_y, v, xw, row0, n0 + 64 * c, lane, sbias + 64 * c);
      }
      if (++buf == 2) { buf = 0; buf_phase ^= 1u; }
    }
    if (p.tma_store && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    __syncwarp();
  }

  // An aborted CTA gives copies still in flight (the peer's loads complete on the leader's
  // barrier) a bounded grace period before the CTAs leave.
  if (__syncthreads_or(ok ? 0 : 1)) {
    const unsigned long long t0 = globaltimer();
    while (globaltimer() - t0 < 2000000ull) {
    }
  }
  tc_fence_before();
  cluster_sync_all();  // both CTAs are done with TMEM and with each other's barriers
  tc_fence_after();
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kTmemCols)
                 : "memory");
}

// --- host ------------------------------------------------------------------------

// [rows, cols] row-major with row stride ld_bytes, boxes of 128 bytes x box_rows, 128-byte swizzle
static int make_map(CUtensorMap* map, CUtensorMapDataType type, int size, const void* base, int64_t cols,
                    int64_t rows, int64_t ld_bytes, uint32_t box_rows, const char* what) {
  EncodeTiledFn enc = get_encode_fn();
  ZIB_HOST_CHECK(enc, ZIB_ERR_UNSUPPORTED, "%s: cuTensorMapEncodeTiled unavailable", what);
  cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)ld_bytes};
  cuuint32_t box[2] = {(cuuint32_t)(128 / size), box_rows};
  cuuint32_t estr[2] = {1, 1};
  const CUresult r = enc(map, type, 2, const_cast<void*>(base), dims, strides, box, estr,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  ZIB_HOST_CHECK(r == CUDA_SUCCESS, ZIB_ERR_INVALID_ARG, "%s: cuTensorMapEncodeTiled failed (%d)", what, (int)r);
  return ZIB_OK;
}

constexpr int64_t kGroupBudget = 48ll << 20;  // L2 bytes for the operand that every wave re-reads

// MX: the tensor cores apply the scales (BN = Mx::BN), or the launch does nothing where they cannot
template <typename T, int BN, bool MX = false>
static int launch_pair(GemmParams p, const void* q, int64_t ldq, const void* w, int64_t ldw, int64_t K,
                       bool dependent, cudaStream_t st, const char* what) {
  CUtensorMap ta, tb, ty;
  int rc = make_map(&ta, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, q, K, p.M, ldq, 128u, what);
  if (!rc) rc = make_map(&tb, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, w, K, p.N, ldw, BN / 2, what);
  p.tma_store = ((uintptr_t)p.y % 16 == 0 && p.ldy * sizeof(T) % 16 == 0) ? 1 : 0;
  ty = ta;
  if (!rc && p.tma_store)
    rc = make_map(&ty, sizeof(T) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, sizeof(T),
                  p.y, p.N, p.M, p.ldy * (int64_t)sizeof(T), 32u, what);
  if (rc) return rc;
  void (*kernel)(CUtensorMap, CUtensorMap, CUtensorMap, GemmParams);
  int smem;
  if constexpr (MX) kernel = gemm_mx_kernel<T>, smem = Mx::SMEM;
  else kernel = gemm_pair_kernel<T, BN>, smem = Cfg<BN>::SMEM;
  static std::atomic<bool> set[64];
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && !set[dev].load(std::memory_order_relaxed)) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    ZIB_HOST_CHECK(e == cudaSuccess, ZIB_ERR_LAUNCH, "%s: cudaFuncSetAttribute failed: %s", what,
                   cudaGetErrorString(e));
    set[dev].store(true, std::memory_order_relaxed);
  }
  p.num_mb = (int)ceil_div(p.M, 256);
  p.num_nb = (int)ceil_div(p.N, BN);
  p.num_kb = (int)ceil_div(K, kBlock);
  ZIB_HOST_CHECK((int64_t)p.num_mb * p.num_nb < (1ll << 30), ZIB_ERR_TOO_LARGE, "%s: M=%d N=%d", what, p.M, p.N);
  p.num_tiles = p.num_mb * p.num_nb;
  p.n_fast = (int64_t)p.M * K > (int64_t)p.N * K ? 1 : 0;  // the smaller operand is re-read from L2
  const int64_t nfast = p.n_fast ? p.num_nb : p.num_mb;
  const int64_t per = kGroupBudget / ((p.n_fast ? BN : 256) * K);
  const int64_t groups = ceil_div(nfast, per < 1 ? 1 : per);
  p.group = (int)ceil_div(nfast, groups);
  int clusters = sm_count() / 2;
  if (clusters > p.num_tiles) clusters = p.num_tiles;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(2 * clusters);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = dependent ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, ta, tb, ty, p);
  if (e != cudaSuccess) {
    cudaGetLastError();
    zib_set_error("%s: launch failed: %s", what, cudaGetErrorString(e));
    return ZIB_ERR_LAUNCH;
  }
  return ZIB_OK;
}

template <typename T>
static int gemm(GemmParams p, const void* q, int64_t ldq, const void* w, int64_t ldw, int64_t K, bool exponents,
                bool dependent, cudaStream_t st, const char* what) {
  // whole waves of 256 x 256 tiles, or twice as many 256 x 128 ones where those end sooner
  const int64_t pairs = sm_count() / 2, mb = ceil_div(p.M, 256), kb = ceil_div(K, kBlock);
  const int64_t wide = ceil_div(mb * ceil_div(p.N, 256), pairs) * 2, slim = ceil_div(mb * ceil_div(p.N, 128), pairs);
  if (exponents) {
    // The tensor cores apply the scales where that and the second launch, which then ends at once, are sooner.
    // A call there takes 5 us more than here, and each wave 0.27 us a K-block and 0.6 us; here each wave 0.54 us a
    // K-block and 0.6 us (wide) or 0.34 us a K-block (slim).  16-bit rows of y that start on any element leave by
    // elements, there through four warps instead of eight: 1 us more a wave.  Fitted to 1600 calls of 256 to 18226
    // rows, aligned or not, in 16 and 32 bits, both sides timed in turns: by this rule a call takes 0.1 to 0.6% more
    // than on its faster side on average.  bf16 with bias, the tensor cores' scales / sums in registers: 4608 x
    // 2560 -> 3840 56 / 69 us, 4608 x 3840 -> 2560 60 / 76, 768 x 2560 -> 3840 26 / 26, 512 x 3840 -> 7680 38 / 31, 2304 x
    // 512 -> 11520 47 / 41, 18226 x 512 -> 4071 173 / 143, and the wrong way 256 x 3840 -> 11520 34 / 30 (few rows: bound
    // by the weight's way from memory).
    const int64_t mx = ceil_div(mb * ceil_div(p.N, Mx::BN), pairs);
    const int64_t sums = slim < wide ? 34 * kb * slim : (27 * kb + 30) * wide;
    const bool elements = sizeof(T) == 2 && ((uintptr_t)p.y % 16 != 0 || p.ldy * sizeof(T) % 16 != 0);
    if (500 + (27 * kb + (elements ? 160 : 60)) * mx < sums) {
      const int rc = launch_pair<T, Mx::BN, true>(p, q, ldq, w, ldw, K, dependent, st, what);
      if (rc) return rc;
      p.where = 1;
      dependent = false;
    }
  }
  if (slim < wide) return launch_pair<T, 128>(p, q, ldq, w, ldw, K, dependent, st, what);
  return launch_pair<T, 256>(p, q, ldq, w, ldw, K, dependent, st, what);
}

}  // namespace fp8
}  // namespace zib

using namespace zib;

int zib::fp8_gemm(const void* q, int64_t ldq, const float* sx, int64_t sx_m, int64_t sx_k, const void* w, int64_t ldw,
                  const float* sw, int64_t sw_n, int64_t sw_k, const void* bias, void* y, int64_t ldy, int dtype,
                  int64_t M, int64_t N, int64_t K, bool exponents, bool dependent, cudaStream_t st,
                  const char* what) {
  fp8::GemmParams p{};
  p.M = (int)M; p.N = (int)N;
  p.sx = sx; p.sx_m = sx_m; p.sx_k = sx_k;
  p.sw = sw; p.sw_n = sw_n; p.sw_k = sw_k;
  p.bias = bias; p.y = y; p.ldy = ldy;
  if (dtype == ZIB_BF16) return fp8::gemm<__nv_bfloat16>(p, q, ldq, w, ldw, K, exponents, dependent, st, what);
  if (dtype == ZIB_F16) return fp8::gemm<__half>(p, q, ldq, w, ldw, K, exponents, dependent, st, what);
  return fp8::gemm<float>(p, q, ldq, w, ldw, K, exponents, dependent, st, what);
}

extern "C" int zib_fp8_block_gemm(const void* q, int64_t ldq, const float* sx, int64_t sx_m, int64_t sx_k,
                                  const void* w, int64_t ldw, const float* sw, int64_t sw_n, int64_t sw_k,
                                  const void* bias, void* y, int64_t ldy, int dtype, int64_t M, int64_t N, int64_t K,
                                  void* stream) {
  const char* what = "zib_fp8_block_gemm";
  ZIB_HOST_CHECK(known_dtype(dtype), ZIB_ERR_INVALID_ARG, "%s: unknown dtype %d", what, dtype);
  ZIB_HOST_CHECK(M >= 0 && N >= 1 && K >= 1 && ldq >= K && ldw >= K && ldy >= N, ZIB_ERR_INVALID_ARG,
                 "%s: bad shape M=%lld N=%lld K=%lld", what, (long long)M, (long long)N, (long long)K);
  ZIB_HOST_CHECK(M < (1ll << 31) - 512 && N < (1ll << 31) - 512 && K < (1ll << 31) - 512, ZIB_ERR_TOO_LARGE,
                 "%s: M=%lld N=%lld K=%lld", what, (long long)M, (long long)N, (long long)K);
  ZIB_HOST_CHECK(ldq % 16 == 0 && ldw % 16 == 0 && (uintptr_t)q % 16 == 0 && (uintptr_t)w % 16 == 0,
                 ZIB_ERR_ALIGNMENT, "%s: q and w need 16-byte aligned rows", what);
  if (M == 0) return ZIB_OK;
  ZIB_HOST_CHECK(q && sx && w && sw && y, ZIB_ERR_INVALID_ARG, "%s: null operand", what);
  return fp8_gemm(q, ldq, sx, sx_m, sx_k, w, ldw, sw, sw_n, sw_k, bias, y, ldy, dtype, M, N, K, false, false,
                  (cudaStream_t)stream, what);
}
