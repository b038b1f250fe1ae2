// Grouped products with 4-bit expert weights on CTA pairs (tcgen05.mma
// cta_group::2), for experts with many rows.
//
//   gated: h[r, j] = act(a[r] . Wg[e, j]) * (a[r] . Wu[e, j])   stored in the layer dtype
//   down:  y[r, n] = h[r] . W2[e, n]                            stored in fp32
// As in gemm_pair.cu the weights are the MMA's M side (128 rows per CTA, 256
// per pair) and the expert's token rows its N side (up to 256 in steps of 16,
// half of them in each CTA's shared memory).  The weights arrive as 4-bit codes
// (int4.cuh): TMA copies bring a CTA's codes and scales into a ring of their
// own, and code warps turn each word into eight 16-bit values
// scale * (code - 8) and write them where a TMA copy would have put 16-bit
// weights (K-major, 128-byte swizzle).  The product of a code with a scale of
// five significant bits is exact, so scales made by rf_moe_int4_quantize round
// nothing here; a scale with more bits is rounded once per weight, to nearest.
// Gated tiles put 16 gate rows and their 16 up rows into one quadrant of 32
// TMEM lanes, so the epilogue pairs them with one shuffle.
//
// Bound by the MMAs with tiles of 256 tokens: a stage of 128 k takes 1024 cycles
// of them (4096 tokens through eight experts of 4096 x 14336: 1.91-1.93 ms in
// all, 93 % of the measured bf16 peak, 2.21 in a steady run at the power cap;
// 8192 through 64 of 2048 x 1408: 0.73 ms, 72 %, the rest the permutation, the
// combine and unfilled tiles).  With few tokens a stage takes 800-860 cycles
// whatever their number: 32 KB of 16-bit rows are written to shared memory and
// read back, 18 KB of codes pass in and out, about 700 cycles of its bandwidth
// (16 tokens through the same experts: 0.28 ms, 40 % of the HBM rate).  Tried
// without gain there: a ring of tokens of its own, two slots of codes per stage,
// 24 code warps, codes called into L2 ahead.
//
// Roles (a cluster of two CTAs per pair, persistent, 19 warps):
//   warp 0        TMA producer of this CTA's token rows
//   warp 1        first CTA: MMA issuer
//   warps 2-5     epilogue, one per TMEM lane quadrant
//   warps 6-17    codes -> 16-bit rows: four warps (32 rows each) for each of
//                 the ring's three slots, so that three stages are in work at a time
//   warp 18       TMA producer of this CTA's codes and scales
// A stage of the ring holds 128 k: it is full when the token bytes of both CTAs
// and the arrivals of the pair's eight code warps of its slot are in, and empty when
// the MMAs that read it have committed.  Tiles (group, feature block, token
// block; tokens fastest, so that running pairs share weights in L2) go to the
// pairs round robin.  Every wait is bounded (2 s): on expiry the CTA sets the
// device error word, both CTAs stop, let their copies land, drain their MMAs,
// meet at a cluster barrier and free TMEM.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <type_traits>

#include "int4.cuh"
#include "gemm.cuh"

RF_DEVICE_ERROR_WORD();
#include "tc_pair_ptx.cuh"

namespace {

constexpr int Q_BK = 64;                        // swizzle atom depth (elements)
constexpr int Q_KSUB = 2;                       // atoms per stage
constexpr int Q_TOK = 256;                      // token rows per tile
constexpr int Q_A_SUB = 128 * Q_BK * 2;         // 16 KB: this CTA's weight rows
constexpr int Q_B_SUB = (Q_TOK / 2) * Q_BK * 2; // 16 KB: this CTA's token rows
constexpr int Q_STAGES = 3;
constexpr int Q_STAGE_BYTES = Q_KSUB * (Q_A_SUB + Q_B_SUB);
constexpr int Q_EPI_WARPS = 4;
constexpr int Q_CODE_WARPS = 4;                 // code warps of a stage: 32 weight rows each
constexpr int Q_COPY_WARP = 2 + Q_EPI_WARPS + Q_STAGES * Q_CODE_WARPS;  // the last warp
constexpr int Q_THREADS = 32 * (Q_COPY_WARP + 1);
constexpr int Q_BLOCKS = 8;                     // row blocks (16 rows) of a CTA's stage
constexpr int Q_CODE_BYTES = Q_BLOCKS * Q_KSUB * rf::I4_BLOCK;  // 8 KB
constexpr int Q_SCALE_BYTES = Q_BLOCKS * 4 * rf::I4_ROWS * 2;   // 1 KB: up to four groups
constexpr int Q_MAX_E = 1024;
constexpr int Q_NUM_BARS = 4 * Q_STAGES + 5;  // full, empty, tmem full x2, tmem empty x2, drain, codes full, codes empty
constexpr int Q_N_BOXES = 5;                    // token boxes of 8, 16, 32, 64, 128 rows
constexpr unsigned Q_EPI_SLEEP_NS = 256;
constexpr uint64_t Q_ABORT_DRAIN_NS = 1000000;  // pause for copies in flight after an abort
constexpr uint32_t Q_TMEM_COLS = 512;
constexpr size_t Q_SMEM_BYTES =
    1024 + (size_t)Q_STAGES * Q_STAGE_BYTES + (size_t)Q_STAGES * (Q_CODE_BYTES + Q_SCALE_BYTES) + Q_NUM_BARS * 8 + 16 +
    (size_t)(Q_MAX_E + 1) * 4;
static_assert(Q_SMEM_BYTES <= 227 * 1024, "shared memory");
static_assert(Q_CODE_BYTES % 128 == 0 && Q_SCALE_BYTES % 128 == 0, "TMA destinations");
static_assert(Q_A_SUB % 1024 == 0 && Q_B_SUB % 1024 == 0, "swizzle atoms");

struct PairArgs {
  const int32_t *offsets, *counts;
  void *out;
  int E, Kdim, N, n_fb;
  int group, act;
  rf::Int4Shape sh;
};

struct TokMaps {
  CUtensorMap m[Q_N_BOXES];
};

// Arrive on either CTA's barrier with a release of CTA scope.  What it hands
// over stays on this SM: rows in this CTA's shared memory that this SM's tensor
// core reads (ordered by the proxy fence before it), or this CTA's TMEM; only
// the count is kept by the other CTA.  A release of cluster scope here waited
// 1000-1800 cycles, once per stage (clock64, eight experts of 4096 x 14336).
__device__ __forceinline__ void mbar_arrive_remote(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.release.cta.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ uint4 ld_shared_v4(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t ld_shared_u32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

__device__ __forceinline__ void st_shared_v4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(r));
  return r != 0;
}
// sw128_desc of an address, its low word; the high word is the same for all.
constexpr uint32_t SW128_DESC_HI = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t sw128_desc_lo(uint32_t saddr) { return ((saddr >> 4) & 0x3FFFu) | (1u << 16); }
__device__ __forceinline__ void tc_mma_pair_lo(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc,
                                               uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "mov.b64 a, {%1, %5};\n\t"
      "mov.b64 b, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], a, b, %3, p;\n\t}\n" ::"r"(d),
      "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(SW128_DESC_HI)
      : "memory");
}
// Two 16-bit products, each rounded to nearest (exact for short scales).
template <typename T> __device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b);
template <> __device__ __forceinline__ uint32_t mul2<__nv_bfloat16>(uint32_t a, uint32_t b) {
  const __nv_bfloat162 r = __hmul2(*reinterpret_cast<const __nv_bfloat162 *>(&a), *reinterpret_cast<const __nv_bfloat162 *>(&b));
  return *reinterpret_cast<const uint32_t *>(&r);
}
template <> __device__ __forceinline__ uint32_t mul2<__half>(uint32_t a, uint32_t b) {
  const __half2 r = __hmul2(*reinterpret_cast<const __half2 *>(&a), *reinterpret_cast<const __half2 *>(&b));
  return *reinterpret_cast<const uint32_t *>(&r);
}

// 16 token columns of a quadrant: lanes 0-15 hold gate sums, lanes 16-31 the up
// sums of the same 16 features.  Lanes 0-15 finish the even tokens, 16-31 the
// odd ones (out and left are for this lane's first).
template <typename T, int ACT>
__device__ __forceinline__ void store_gated(const uint32_t (&v)[16], int lane, T *out, int N, int left) {
  const bool up = lane >= 16;
  float h[8];  // eight chains at a time: inside the stores' conditions they ran one after another
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t got = __shfl_xor_sync(0xffffffffu, up ? v[2 * i] : v[2 * i + 1], 16);
    const float g = __uint_as_float(up ? got : v[2 * i]);
    const float u = __uint_as_float(up ? v[2 * i + 1] : got);
    h[i] = rf::act_gate_t<ACT>(g) * u;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) asm volatile("" : "+f"(h[i]));
#pragma unroll
  for (int i = 0; i < 8; ++i, out += 2 * (int64_t)N)
    if (2 * i < left) *out = rf::Cvt<T>::from_f(h[i]);
}

// SUBS: scale groups in a stage's 128 k (1, 2 or 4).
template <typename T, bool GATED, int SUBS>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(Q_THREADS, 1)
    int4_pair_gemm(const __grid_constant__ TokMaps tmX, const __grid_constant__ CUtensorMap tmW,
                   const __grid_constant__ CUtensorMap tmS, const PairArgs p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t *sA = smem;
  uint8_t *sB = sA + Q_STAGES * Q_KSUB * Q_A_SUB;
  uint8_t *sQ = sB + Q_STAGES * Q_KSUB * Q_B_SUB;  // [slot] codes, then scales
  uint64_t *bars = reinterpret_cast<uint64_t *>(sQ + Q_STAGES * (Q_CODE_BYTES + Q_SCALE_BYTES));
  uint32_t *tmem_holder = reinterpret_cast<uint32_t *>(bars + Q_NUM_BARS);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_holder + 1);
  int *tile_prefix = reinterpret_cast<int *>(tmem_holder + 4);  // [E+1]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int E = p.E;
  const int pair = (int)cluster_id_x(), npairs = (int)ncluster_x();
  const uint32_t bar0 = smem_u32(bars);
#define FULL(s) (bar0 + 8u * (uint32_t)(s))
#define EMPTY(s) (bar0 + 8u * (uint32_t)(Q_STAGES + (s)))
#define TFULL(a) (bar0 + 8u * (uint32_t)(2 * Q_STAGES + (a)))
#define TEMPTY(a) (bar0 + 8u * (uint32_t)(2 * Q_STAGES + 2 + (a)))
  const uint32_t DRAIN = bar0 + 8u * (uint32_t)(2 * Q_STAGES + 4);
#define CFULL(s) (bar0 + 8u * (uint32_t)(2 * Q_STAGES + 5 + (s)))
#define CEMPTY(s) (bar0 + 8u * (uint32_t)(3 * Q_STAGES + 5 + (s)))
  const uint32_t peer_abort = mapa_shared(smem_u32((const void *)abort_flag), rank ^ 1u);

  // bounded wait with cluster-scope acquire; on expiry both CTAs are told to stop
  auto pwait = [&](uint32_t bar, uint32_t parity, unsigned sleep_ns) -> bool {
    if (mbar_try_cluster(bar, parity)) return true;
    const uint64_t t0 = rf::globaltimer_ns();
    for (uint32_t it = 1;; ++it) {
      if (sleep_ns) __nanosleep(sleep_ns);
      if (mbar_try_cluster(bar, parity)) return true;
      if ((it & 63) == 0) {
        if (*abort_flag) return false;
        if (rf::globaltimer_ns() - t0 > WAIT_LIMIT_NS) {
          *abort_flag = 1;
          st_cluster_u32(peer_abort, 1u);
          rf_report(RF_DEV_WAIT_TIMEOUT);
          return false;
        }
      }
    }
  };

  if (threadIdx.x == 0) {
    for (int s = 0; s < Q_STAGES; ++s) {
      mbar_init(FULL(s), 1 + 2 * Q_CODE_WARPS);  // the first CTA's: its token producer and the pair's code warps
      mbar_init(EMPTY(s), 1);
      mbar_init(CFULL(s), 1);
      mbar_init(CEMPTY(s), Q_CODE_WARPS);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(TFULL(a), 1);
      mbar_init(TEMPTY(a), 2 * Q_EPI_WARPS);
    }
    mbar_init(DRAIN, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (threadIdx.x == 32 * Q_COPY_WARP) {
    asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)&tmW) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)&tmS) : "memory");
  }
  if (threadIdx.x == 32)
    for (int i = 0; i < Q_N_BOXES; ++i) asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)&tmX.m[i]) : "memory");
  for (int e = threadIdx.x; e < E; e += Q_THREADS) tile_prefix[e + 1] = (p.counts[e] + Q_TOK - 1) / Q_TOK * p.n_fb;
  if (warp == 1) {
    tmem_alloc_pair(smem_u32(tmem_holder), Q_TMEM_COLS);
    tmem_relinquish_pair();
  }
  __syncthreads();
  if (warp == 2) {  // inclusive scan of tile counts
    int carry = 0;
    for (int c = 0; c < E; c += 32) {
      int v = c + lane < E ? tile_prefix[c + lane + 1] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
      }
      if (c + lane < E) tile_prefix[c + lane + 1] = carry + v;
      carry += __shfl_sync(0xffffffffu, v, 31);
    }
    if (lane == 0) tile_prefix[0] = 0;
  }
  tc_fence_before();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;
  const int total = tile_prefix[E];
  const int num_kb = (p.Kdim + Q_BK * Q_KSUB - 1) / (Q_BK * Q_KSUB);  // stages per tile

  // tile -> expert, first token row, token count, feature block
  auto decode = [&](int t, int &e, int &row0, int &ntok, int &fb) {
    int lo = 0, hi = E - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (tile_prefix[mid] <= t) lo = mid;
      else hi = mid - 1;
    }
    const int cnt = __ldg(p.counts + lo);
    const int ntb = (cnt + Q_TOK - 1) / Q_TOK;
    const int local = t - tile_prefix[lo];
    fb = local / ntb;
    const int tb = local - fb * ntb;
    e = lo;
    // the rows in equal blocks: 800 rows as 4 x 208 or less, not 3 x 256 and 32
    const int per = ((cnt + ntb - 1) / ntb + 15) & ~15;  // <= Q_TOK, so the last block has rows
    row0 = __ldg(p.offsets + lo) + tb * per;
    ntok = min(per, cnt - tb * per);
  };

  if (warp == 0) {
    // ------------------------------------------------------- token producer
    const uint32_t full0 = mapa_shared(FULL(0), 0);
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int t = pair; t < total && ok; t += npairs) {
      int e, row0, ntok, fb;
      decode(t, e, row0, ntok, fb);
      const int half = ((ntok + 15) & ~15) >> 1;  // token rows per CTA: a multiple of 8
      int bi = 0;
      while ((8 << bi) < half) ++bi;
      const uint32_t bytes = (uint32_t)Q_KSUB * (uint32_t)(8 << bi) * (Q_BK * 2);  // per CTA
      const int xrow = row0 + (rank ? half : 0);
      for (int kb = 0; kb < num_kb; ++kb) {
        ok = __all_sync(0xffffffffu, pwait(EMPTY(stage), phase ^ 1u, 0));
        if (!ok) break;
        if (elect_one()) {
          const uint32_t b_dst = smem_u32(sB + stage * Q_KSUB * Q_B_SUB);
          if (rank == 0) mbar_expect_tx(FULL(stage), 2u * bytes);  // both CTAs load the same box sizes
#pragma unroll
          for (int j = 0; j < Q_KSUB; ++j)
            tma_load_2d_pair(b_dst + (uint32_t)(j * Q_B_SUB), &tmX.m[bi], full0 + 8u * (uint32_t)stage,
                             (kb * Q_KSUB + j) * Q_BK, xrow);
        }
        __syncwarp();
        if (++stage == Q_STAGES) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
    if (!ok) {  // let the copies in flight land before this CTA can exit (bounded pause)
      const uint64_t t0 = rf::globaltimer_ns();
      while (rf::globaltimer_ns() - t0 < Q_ABORT_DRAIN_NS) __nanosleep(1000);
    }
  } else if (warp == 1) {
    if (rank == 0) {
      // ---------------------------------------------------------- MMA issuer
      // The whole warp walks the loop and one elected lane issues: addresses
      // and descriptors stay warp-uniform (inside a one-lane branch an MMA took 88
      // cycles to issue; 16 tokens: 0.42 -> 0.29 ms).
      const uint32_t IDESC = pair_idesc_base<T>();
      const uint32_t peer_bars = mapa_shared(bar0, 1);
      const uint32_t a_desc = sw128_desc_lo(smem_u32(sA)), b_desc = sw128_desc_lo(smem_u32(sB));
      int stage = 0, it = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int t = pair; t < total && ok; t += npairs, ++it) {
        int e, row0, ntok, fb;
        decode(t, e, row0, ntok, fb);
        const uint32_t idesc = IDESC | ((uint32_t)(((ntok + 15) & ~15) >> 3) << 17);
        const int acc = it & 1;
        ok = __all_sync(0xffffffffu, pwait(TEMPTY(acc), (uint32_t)(((it >> 1) & 1) ^ 1), 0));
        if (!ok) break;
        tc_fence_after();
        const uint32_t d = tmem_base + (uint32_t)(acc * 256);
        for (int kb = 0; kb < num_kb; ++kb) {
          ok = __all_sync(0xffffffffu, pwait(FULL(stage), phase, 0));
          if (!ok) break;
          tc_fence_after();
          const uint32_t a0 = a_desc + (uint32_t)(stage * (Q_KSUB * Q_A_SUB >> 4));
          const uint32_t b0 = b_desc + (uint32_t)(stage * (Q_KSUB * Q_B_SUB >> 4));
          if (elect_one()) {
#pragma unroll
            for (int j = 0; j < Q_KSUB; ++j)
#pragma unroll
              for (int k = 0; k < Q_BK / 16; ++k)
                tc_mma_pair_lo(d, a0 + (uint32_t)((j * Q_A_SUB + k * 32) >> 4), b0 + (uint32_t)((j * Q_B_SUB + k * 32) >> 4),
                               idesc, (kb | j | k) ? 1u : 0u);
            tc_commit_pair(EMPTY(stage));  // frees the stage in both CTAs once read
            tc_commit_pair(peer_bars + (EMPTY(stage) - bar0));
            if (kb == num_kb - 1) {
              tc_commit_pair(TFULL(acc));
              tc_commit_pair(peer_bars + (TFULL(acc) - bar0));
            }
          }
          __syncwarp();
          if (++stage == Q_STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      // no MMA may still be running when either CTA releases TMEM or exits
      if (elect_one()) {
        tc_commit_pair(DRAIN);
        mbar_wait_teardown(DRAIN, 0);
      }
      __syncwarp();
    }
  } else if (warp < 2 + Q_EPI_WARPS) {
    // ------------------------------------------------------------ epilogue
    const int wq = warp & 3;  // the TMEM lane quadrant a warp can read
    const uint32_t tempty0 = mapa_shared(TEMPTY(0), 0);
    int it = 0;
    for (int t = pair; t < total; t += npairs, ++it) {
      int e, row0, ntok, fb;
      decode(t, e, row0, ntok, fb);
      const int acc = it & 1;
      int ok = 1;
      if (lane == 0) ok = pwait(TFULL(acc), (uint32_t)((it >> 1) & 1), Q_EPI_SLEEP_NS) ? 1 : 0;
      ok = __shfl_sync(0xffffffffu, ok, 0);
      if (!ok) break;
      tc_fence_after();
      const uint32_t tb = tmem_base + ((uint32_t)(wq * 32) << 16) + (uint32_t)(acc * 256);
      const int np = (ntok + 15) & ~15;
      // gated: lanes 0-15 of the quadrant hold gate rows, 16-31 the same features' up rows
      const int f = GATED ? fb * 128 + (int)rank * 64 + wq * 16 + (lane & 15) : fb * 256 + (int)rank * 128 + wq * 32 + lane;
      for (int c = 0; c < np; c += 16) {
        uint32_t v[16];
        tmem_ld16(tb + (uint32_t)c, v);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i) asm volatile("" : "+r"(v[i]));  // no use of v moves above the wait
        if (c + 16 >= np) {  // the accumulator is free for the pair's tile after next
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_remote(tempty0 + 8u * (uint32_t)acc);
        }
        if constexpr (GATED) {
          T *out = reinterpret_cast<T *>(p.out) + (int64_t)(row0 + c + (lane >> 4)) * p.N + f;
          const int left = f < p.N ? ntok - c - (lane >> 4) : 0;  // tokens of this lane's parity from here on
          if (p.act == RF_ACT_SILU) store_gated<T, RF_ACT_SILU>(v, lane, out, p.N, left);
          else if (p.act == RF_ACT_GELU) store_gated<T, RF_ACT_GELU>(v, lane, out, p.N, left);
          else store_gated<T, RF_ACT_GELU_TANH>(v, lane, out, p.N, left);
        } else {
          float *out = reinterpret_cast<float *>(p.out) + (int64_t)(row0 + c) * p.N + f;
          const int left = f < p.N ? ntok - c : 0;
#pragma unroll
          for (int i = 0; i < 16; ++i, out += p.N)
            if (i < left) *out = __uint_as_float(v[i]);
        }
      }
    }
  } else if (warp == Q_COPY_WARP) {
    // ---------------------------------------------- codes and scales producer
    const int64_t row_blocks = p.sh.row_blocks();
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int t = pair; t < total && ok; t += npairs) {
      int e, row0, ntok, fb;
      decode(t, e, row0, ntok, fb);
      // two boxes of four row blocks: gate and up, or eight in a row; blocks past
      // the weight's own are some other rows or zeros, never stored
      const int rb0 = (int)((int64_t)e * row_blocks) + (GATED ? fb * 8 + (int)rank * 4 : fb * 16 + (int)rank * 8);
      const int rb1 = rb0 + (GATED ? (int)p.sh.half_blocks : 4);
      for (int kb = 0; kb < num_kb; ++kb) {
        ok = __all_sync(0xffffffffu, pwait(CEMPTY(stage), phase ^ 1u, 0));
        if (!ok) break;
        if (elect_one()) {
          const uint32_t dst = smem_u32(sQ) + (uint32_t)(stage * (Q_CODE_BYTES + Q_SCALE_BYTES));
          const uint32_t sdst = dst + Q_CODE_BYTES;
          mbar_expect_tx(CFULL(stage), Q_CODE_BYTES + Q_BLOCKS * SUBS * rf::I4_ROWS * 2);
          tma_load_2d(dst, &tmW, CFULL(stage), kb * (Q_KSUB * rf::I4_BLOCK / 4), rb0);
          tma_load_2d(dst + Q_CODE_BYTES / 2, &tmW, CFULL(stage), kb * (Q_KSUB * rf::I4_BLOCK / 4), rb1);
          tma_load_2d(sdst, &tmS, CFULL(stage), kb * (SUBS * rf::I4_ROWS), rb0);
          tma_load_2d(sdst + Q_SCALE_BYTES / 2, &tmS, CFULL(stage), kb * (SUBS * rf::I4_ROWS), rb1);
        }
        __syncwarp();
        if (++stage == Q_STAGES) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
    if (!ok) {  // let the copies in flight land before this CTA can exit (bounded pause)
      const uint64_t t0 = rf::globaltimer_ns();
      while (rf::globaltimer_ns() - t0 < Q_ABORT_DRAIN_NS) __nanosleep(1000);
    }
  } else {
    // --------------------------------------------------------- code warps
    // Warp cw serves one slot of the rings, so it follows every phase of the
    // barriers that it waits for: stages s = slot, slot + Q_STAGES, ...
    const int cw = warp - 2 - Q_EPI_WARPS;
    const int slot = cw / Q_CODE_WARPS, j = cw % Q_CODE_WARPS;  // its 32 of the CTA's 128 rows
    const int g = lane >> 2, c = lane & 3;
    const uint32_t codes = smem_u32(sQ) + (uint32_t)(slot * (Q_CODE_BYTES + Q_SCALE_BYTES));
    const int steps = pair < total ? ((total - 1 - pair) / npairs + 1) * num_kb : 0;
    // rows g and g + 8 of a block, 16-byte pieces 4 h + c of their 128 bytes,
    // swizzled; the first one written has h = g & 1
    const uint32_t piece0 = (uint32_t)((((4 * (g & 1) + c) ^ g) & 7) * 16), piece1 = piece0 ^ 64u;
    const uint32_t a_dst = smem_u32(sA + slot * Q_KSUB * Q_A_SUB) + (uint32_t)((j * 32 + g) * 128);
    const uint32_t full = mapa_shared(FULL(slot), 0);
    uint32_t phase = 0;
    for (int s = slot; s < steps; s += Q_STAGES, phase ^= 1u) {
      bool ok = __all_sync(0xffffffffu, pwait(CFULL(slot), phase, 0));  // the warp leaves together
      if (!ok) break;
      uint4 q[2][Q_KSUB];
      uint32_t sc[2][SUBS];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        // the tile's rows 32 j .. 32 j + 15 and the next 16: a gate block and
        // its up block, or two neighbours
        const int at = GATED ? 4 * r + j : 2 * j + r;
        const uint32_t src = codes + (uint32_t)(at * Q_KSUB * rf::I4_BLOCK + lane * 16);
        const uint32_t ss = codes + Q_CODE_BYTES +
                            (uint32_t)((at >> 2) * (Q_SCALE_BYTES / 2) + (at & 3) * (SUBS * rf::I4_ROWS * 2) + g * SUBS * 4);
#pragma unroll
        for (int b = 0; b < Q_KSUB; ++b) q[r][b] = ld_shared_v4(src + (uint32_t)(b * rf::I4_BLOCK));
#pragma unroll
        for (int i = 0; i < SUBS; ++i) sc[r][i] = ld_shared_u32(ss + (uint32_t)(i * 4));
      }
      // a proxy fence before the release: copies of the async proxy refill the
      // slot, and without it they overtook reads still under way (the last
      // block's 16 rows came out wrong in most runs of 4096 tokens and more)
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(CEMPTY(slot));  // the codes are in registers
      // 16-bit values of rows g (v[..][0]) and g + 8, before the wait: only
      // the stores stay between a slot's release and its next use
      uint32_t v[2][Q_KSUB][2][2][4];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
#pragma unroll
        for (int b = 0; b < Q_KSUB; ++b) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            // even rows write their halves in order, odd rows the second one
            // first: eight neighbouring lanes then cover all 32 banks
            const int h = i ^ (g & 1);
            const uint32_t lo = h ? q[r][b].y : q[r][b].x, hi = h ? q[r][b].w : q[r][b].z;
            // SUBS 4: a group is one half (32 k); 2: one block; 1: the stage
            const uint32_t sv = SUBS == 4 ? (h ? sc[r][(2 * b + 1) % SUBS] : sc[r][(2 * b) % SUBS]) : sc[r][b * SUBS / 2];
            const uint32_t s_lo = __byte_perm(sv, sv, 0x1010), s_hi = __byte_perm(sv, sv, 0x3232);
#pragma unroll
            for (int m = 0; m < 4; ++m) {
              v[r][b][i][0][m] = mul2<T>(rf::int4_pair<T>(lo, m), s_lo);
              v[r][b][i][1][m] = mul2<T>(rf::int4_pair<T>(hi, m), s_hi);
              asm volatile("" : "+r"(v[r][b][i][0][m]), "+r"(v[r][b][i][1][m]));  // computed here
            }
          }
        }
      }
      ok = __all_sync(0xffffffffu, pwait(EMPTY(slot), phase ^ 1u, 0));
      if (!ok) break;
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int b = 0; b < Q_KSUB; ++b)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t at = a_dst + (uint32_t)(b * Q_A_SUB + r * 16 * 128) + (i ? piece1 : piece0);
            const uint32_t(&w)[2][4] = v[r][b][i];
            st_shared_v4(at, w[0][0], w[0][1], w[0][2], w[0][3]);
            st_shared_v4(at + 8 * 128, w[1][0], w[1][1], w[1][2], w[1][3]);
          }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the MMA reads through the async proxy
      __syncwarp();
      if (lane == 0) mbar_arrive_remote(full);
    }
  }
  // ---------------------------------------------------------------- teardown
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // no CTA of the pair leaves while the other may still reach into it
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, Q_TMEM_COLS);
  }
#undef CFULL
#undef CEMPTY
#undef FULL
#undef EMPTY
#undef TFULL
#undef TEMPTY
}

template <typename T, bool GATED, int SUBS>
int launch_pair_t(const TokMaps &mx, const CUtensorMap &mw, const CUtensorMap &ms, const PairArgs &p, cudaStream_t st) {
  auto kern = int4_pair_gemm<T, GATED, SUBS>;
  static rf::PerDevice fit;
  const int clusters = fit.get(rf::current_device(), [&]() -> int {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Q_SMEM_BYTES) != cudaSuccess) return 0;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2 * std::max(1, rf::num_sms() / 2), 1, 1);
    cfg.blockDim = dim3(Q_THREADS, 1, 1);
    cfg.dynamicSmemBytes = Q_SMEM_BYTES;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = 2;
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    int n = 0;
    return cudaOccupancyMaxActiveClusters(&n, (void *)kern, &cfg) == cudaSuccess ? n : 0;
  });
  if (clusters < 1) {
    cudaGetLastError();
    return rf::fail(RF_ERR_CUDA, "4-bit products: the CTA-pair kernel does not fit this device");
  }
  kern<<<2 * clusters, Q_THREADS, Q_SMEM_BYTES, st>>>(mx, mw, ms, p);
  return rf::check_launch(GATED ? "4-bit gated products (CTA pairs)" : "4-bit down products (CTA pairs)");
}

template <typename T, bool GATED>
int launch_pair_g(const TokMaps &mx, const CUtensorMap &mw, const CUtensorMap &ms, const PairArgs &p, cudaStream_t st) {
  if (p.group == 32) return launch_pair_t<T, GATED, 4>(mx, mw, ms, p, st);
  if (p.group == 64) return launch_pair_t<T, GATED, 2>(mx, mw, ms, p, st);
  return launch_pair_t<T, GATED, 1>(mx, mw, ms, p, st);
}

}  // namespace

namespace rf {

int launch_int4_pair(const Int4Gemm &g, bool gated, cudaStream_t st) {
  TokMaps mx;
  const cuuint64_t dX[2] = {(cuuint64_t)g.Kdim, (cuuint64_t)g.rows};
  const cuuint64_t sX[1] = {(cuuint64_t)g.Kdim * 2};
  for (int i = 0; i < Q_N_BOXES; ++i) {
    const cuuint32_t bX[2] = {Q_BK, (cuuint32_t)(8 << i)};
    if (!tma_encode(&mx.m[i], g.dtype, 2, g.a, dX, sX, bX))
      return rf::fail(RF_ERR_CUDA, "4-bit products: the token rows' tensor map could not be encoded");
  }
  PairArgs p;
  p.offsets = g.offsets;
  p.counts = g.counts;
  p.out = g.out;
  p.E = g.E;
  p.Kdim = g.Kdim;
  p.N = g.N;
  p.n_fb = gated ? (g.N + 127) / 128 : (g.N + 255) / 256;
  p.group = g.group;
  p.act = g.act;
  p.sh = int4_shape(gated ? 2 * (int64_t)g.N : g.N, g.Kdim, g.group, gated);
  // codes as [E * row blocks][k blocks * 128] words, scales as [E * row blocks][padded groups * 16]
  const uint64_t rows = (uint64_t)g.E * (uint64_t)p.sh.row_blocks();
  const uint32_t scale_cols = (uint32_t)(Q_KSUB * Q_BK / g.group * rf::I4_ROWS);
  CUtensorMap mw, ms;
  if (!tma_encode_plain(&mw, CU_TENSOR_MAP_DATA_TYPE_UINT32, g.w, (uint64_t)p.sh.k_blocks * (I4_BLOCK / 4), rows,
                        (uint64_t)p.sh.k_blocks * I4_BLOCK, Q_KSUB * I4_BLOCK / 4, 4) ||
      !tma_encode_plain(&ms, CU_TENSOR_MAP_DATA_TYPE_UINT16, g.scales, (uint64_t)p.sh.groups * I4_ROWS, rows,
                        (uint64_t)p.sh.groups * I4_ROWS * 2, scale_cols, 4))
    return rf::fail(RF_ERR_CUDA, "4-bit products: the weights' tensor maps could not be encoded");
  if (g.dtype == RF_F16)
    return gated ? launch_pair_g<__half, true>(mx, mw, ms, p, st) : launch_pair_g<__half, false>(mx, mw, ms, p, st);
  return gated ? launch_pair_g<__nv_bfloat16, true>(mx, mw, ms, p, st)
               : launch_pair_g<__nv_bfloat16, false>(mx, mw, ms, p, st);
}

}  // namespace rf
