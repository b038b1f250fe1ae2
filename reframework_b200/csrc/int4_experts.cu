// The routed experts of a MoE layer with 4-bit weights (int4.cuh).
//
//   h[r, j] = act(x[r] . W1g[e, j]) * (x[r] . W1u[e, j])      rounded to the layer dtype
//   y[r, n] = h[r] . W2[e, n]                                 fp32
//   out[t]  = round(sum_k w[t, k] y[row(t, k)] + shared_scale * shared_y + residual)
// for the rows r that the permute gives expert e.  h is rounded because it is
// the second product's 16-bit operand; everything else stays fp32 up to out.
//
// Few pairs (T * K <= 1024, few rows per expert): int4_few_kernel, bound by
// reading the weights, half a byte each, and by the instructions that unpack
// them (about 14 for 256 weights of a warp, of which 7 shift and mask).  A job is
// 32 weight rows a warp group (gated: 16 gate and their 16 up rows) of one
// expert over the whole reduction, against 8 of its tokens.  A lane's 16-byte
// word of the stored layout is its fragment of four 16 x 16 tiles of mma.sync,
// the codes as exact 16-bit integers; the tokens are read straight from their
// rows.  A group's sums are scaled in fp32 after its products.  The warps'
// partial sums meet in shared memory in warp order, so results do not depend on
// timing.  There is no permutation: every block finds the experts' pairs in the
// ids, h and y rows are the pairs themselves, and the three launches (gated,
// down, combine) are chained by programmatic dependent launch, each waiting for
// its predecessor's rows only after its ids and first weights are on the way.
// Measured: 7 tokens through eight experts of 4096 x 14336, groups of 32, 146 us
// where they reach six experts, 178 at 7.3 (62 % of the measured HBM rate), one
// token 58 us; 64 tokens through 60 experts of 2048 x 1408 85 us, one token 15 us.
// Many rows per expert: permute with the row gather, then int4_pair.cu.
#include <algorithm>
#include <string>
#include <type_traits>

#include "gemm.cuh"
#include "int4.cuh"

RF_DEVICE_ERROR_WORD();

namespace {

constexpr int FW_WARPS = 8;
constexpr int FW_THREADS = FW_WARPS * 32;
// Pairs that a block's list holds; more take the CTA-pair kernel whatever their
// rows.  Not a crossover: 256 experts of 2048 x 512, 4 rows each (1024 pairs) 133 us
// here, 199 there; 5 and 8 rows (1280, 2048 pairs) take 202 and 204 there.
constexpr int FW_PAIRS = 1024;
constexpr int FW_STEP = rf::I4_STEP;
constexpr int FW_AHEAD = 4;     // a power of two: ring slots of a warp: steps of codes on their way, and the one in use
// 32-row units (times experts) from which two warps share a unit's k instead of
// eight: longer runs per job, while below it jobs of four units would leave blocks
// idle (2368 units are two jobs for each of 296 resident blocks).  Measured at one
// shape: 64 tokens through 60 experts of 2048 x 1408, 111 us with eight, 101 with two.
constexpr int FW_MANY_JOBS = 2368;
constexpr int KMAX = 16;

struct FewArgs {
  const void *a;         // x [T, Kd] (gated) or h [pairs, Kd]
  const uint8_t *w;
  const void *scales;
  void *out;             // h [pairs, N] in T (gated) or y [pairs, N] fp32
  const int32_t *ids;    // [pairs]
  int pairs, topk, E, N, Kd, act, units;  // units: 32-row units times the row groups of a job, rounded up
  rf::Int4Shape sh;
};

// d = a . b + c, c four registers or zeros
template <typename T>
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1,
                                          const float (&c)[4]) {
  if constexpr (std::is_same<T, __half>::value)
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
  else
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}

__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
// Waits until the launch before this one is complete and its writes visible.
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Two neighbouring 16-bit scales (rows r and r + 8) as floats.
template <typename T>
__device__ __forceinline__ float2 scale_pair(uint32_t v) {
  if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2 *>(&v));
  else return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}

struct FewShared {
  uint4 ring[FW_WARPS][FW_AHEAD][4][32];   // codes on their way, by lane
  uint32_t scale[FW_WARPS][FW_AHEAD][2][32];  // and their scales (8 rows x up to 4 groups)
  float red[FW_WARPS][2 * 4 * 32];
  int count[1024];          // pairs of each expert
  int prefix[1025];         // passes (8 pairs each) before the y-th expert that has pairs
  int list[FW_PAIRS];       // the current expert's pairs, ascending
  uint16_t expert[1024];    // the experts that have pairs, ascending
  int active, part[FW_WARPS];
};

// A job is 32 weight rows for each of the block's row groups, of one expert,
// against 8 of its tokens; a launch's jobs in the order expert, unit, pass.
struct FewJob {
  int y, unit, pass;
};

// Counts each expert's pairs; the experts that have any, with their passes summed up.
__device__ __forceinline__ void count_experts(const FewArgs &p, FewShared &s, const int (&id)[FW_PAIRS / FW_THREADS]) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int e = tid; e < p.E; e += FW_THREADS) s.count[e] = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < FW_PAIRS / FW_THREADS; ++i)
    if (id[i] >= 0) atomicAdd(&s.count[id[i]], 1);
  __syncthreads();
  if (warp == 0) {
    int n = 0, passes = 0;
    for (int e0 = 0; e0 < p.E; e0 += 32) {
      const int cnt = e0 + lane < p.E ? s.count[e0 + lane] : 0;
      const unsigned b = __ballot_sync(0xffffffffu, cnt > 0);
      const int mine = (cnt + 7) / 8;
      int upto = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += u;
      }
      if (cnt > 0) {
        const int y = n + __popc(b & ((1u << lane) - 1u));
        s.expert[y] = (uint16_t)(e0 + lane);
        s.prefix[y] = passes + upto - mine;
      }
      n += __popc(b);
      passes += __shfl_sync(0xffffffffu, upto, 31);
    }
    if (lane == 0) {
      s.active = n;
      s.prefix[n] = passes;
    }
  }
  __syncthreads();
}

// The pairs of expert e, ascending, into s.list.
__device__ __forceinline__ void list_pairs(const FewArgs &p, FewShared &s, const int (&id)[FW_PAIRS / FW_THREADS], int e) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int base = 0;
  __syncthreads();  // the previous expert's list has been read
#pragma unroll
  for (int i = 0; i < FW_PAIRS / FW_THREADS; ++i) {
    if (i * FW_THREADS >= p.pairs) break;
    const unsigned b = __ballot_sync(0xffffffffu, id[i] == e);
    if (lane == 0) s.part[warp] = __popc(b);
    __syncthreads();
    int at = base;
#pragma unroll
    for (int w = 0; w < FW_WARPS; ++w) {
      at += w < warp ? s.part[w] : 0;
      base += s.part[w];
    }
    if (id[i] == e) s.list[at + __popc(b & ((1u << lane) - 1u))] = i * FW_THREADS + tid;
    __syncthreads();
  }
}

// Bytes to shared address dst; 16 bypass L1.
template <int BYTES>
__device__ __forceinline__ void copy_bytes(uint32_t dst, const void *src) {
  if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }

// SUBS: scale groups in a step's 128 k (1, 2 or 4).  KS: warps that share a
// row group's k; the block's 8 / KS row groups are 32 weight rows each.
//
// The codes go to the tensor cores as code + B (B = 128 in bf16, 16 in fp16: a
// shift and one three-input logic operation per pair), and a group's sums start
// from -(B + 8) * sum x, itself a product, with a matrix of -(B + 8), that the two
// row blocks share: sum x (code + B) - (B + 8) sum x = sum x (code - 8).
// Subtracting B + 8 from every code instead took 4 of 15 instructions a word.
// What the larger terms cost: a group's sum passes through two chains of
// 8 / SUBS dependent products each, whose partial sums reach (B + 8) sum |x|.  If
// each truncates its 17 addends at 2^-23 of the largest, at most (B + 15) |x|, the
// sum is off by up to (16 / SUBS) * 17 * 2^-23 * (B + 15) sum |x|, times the scale:
// it follows sum |x|, not sum |x w|.  A channel whose codes are all 8 adds nothing
// in the definition but its share of that here.  Measured, two such channels of
// 2048, the others N(0, 1), the output's error against fp64: bf16 0.0023 with
// channels of up to 1000, as in the CTA-pair kernel, where they add exactly 0;
// 0.0031 with 10000, 0.015 with 50000; fp16 0.00029, 0.0004, 0.0044.
//
// Each warp copies its codes into a ring of its own, FW_AHEAD - 1 steps before
// their use and across the ends of jobs: a job is only a few steps long per
// warp (4 at K = 4096), and the memory would idle at each end.
template <typename T, bool GATED, int SUBS, int KS>
__global__ void __launch_bounds__(FW_THREADS, 2) int4_few_kernel(const FewArgs p) {
  extern __shared__ __align__(16) uint8_t few_smem[];
  FewShared &sm = *reinterpret_cast<FewShared *>(few_smem);
  constexpr uint32_t OFFSET = std::is_same<T, __half>::value ? 0xce00ce00u : 0xc308c308u;  // -24, -136 twice
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, c = lane & 3;
  launch_dependents();
  int id[FW_PAIRS / FW_THREADS];  // this thread's pairs' experts
#pragma unroll
  for (int i = 0; i < FW_PAIRS / FW_THREADS; ++i) {
    const int at = i * FW_THREADS + (int)threadIdx.x;
    id[i] = at < p.pairs ? p.ids[at] : -1;
    if (at < p.pairs && (unsigned)id[i] >= (unsigned)p.E) {
      if (GATED && blockIdx.x == 0) rf_report(RF_DEV_BAD_EXPERT_ID);
      id[i] = -1;
    }
  }
  count_experts(p, sm, id);
  const int n = sm.active;
  const int64_t jobs = (int64_t)sm.prefix[n] * p.units;
  const int j0 = (int)(jobs * blockIdx.x / gridDim.x), j1 = (int)(jobs * (blockIdx.x + 1) / gridDim.x);
  if (j0 >= j1) {
    if (!GATED) wait_for_previous();  // no launch of the chain ends before the one in front of it
    return;
  }
  const int steps = (int)p.sh.k_blocks / 2;
  constexpr int RG = FW_WARPS / KS;
  const int rg = warp / KS, ks = warp % KS;
  const int st0 = steps * ks / KS, mine = steps * (ks + 1) / KS - st0;  // this warp's steps of a job

  auto passes_of = [&](int y) { return sm.prefix[y + 1] - sm.prefix[y]; };
  auto job_at = [&](int j) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if ((int64_t)sm.prefix[mid] * p.units <= j) lo = mid;
      else hi = mid - 1;
    }
    const int at = j - sm.prefix[lo] * p.units, np = passes_of(lo);
    return FewJob{lo, at / np, at % np};
  };
  auto next_job = [&](FewJob &b) {
    if (++b.pass < passes_of(b.y)) return;
    b.pass = 0;
    if (++b.unit < p.units) return;
    b.unit = 0;
    ++b.y;
  };

  // ---- the copy cursor: step cst of job cj, for this lane
  FewJob cb = job_at(j0);
  int cj = j0, cst = 0, cslot = 0;
  const uint4 *wp[2];
  const uint32_t *sp[2];
  auto open_job = [&]() {
    if (cj >= j1) return;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      // rows past the weight's own read its last block: never stored
      const int64_t u = cb.unit * RG + rg;
      int64_t rb = GATED ? min(u, p.sh.half_blocks - 1) + r * p.sh.half_blocks : min(2 * u + r, p.sh.half_blocks - 1);
      rb += (int64_t)sm.expert[cb.y] * p.sh.row_blocks();
      wp[r] = reinterpret_cast<const uint4 *>(p.w + (rb * p.sh.k_blocks + 2 * st0) * rf::I4_BLOCK) + lane;
      sp[r] = reinterpret_cast<const uint32_t *>(reinterpret_cast<const T *>(p.scales) +
                                                 (rb * p.sh.groups + st0 * SUBS) * rf::I4_ROWS) + g * SUBS;
    }
  };
  const uint32_t ring0 = (uint32_t)__cvta_generic_to_shared(&sm.ring[warp][0][0][lane]);
  const uint32_t scale0 = (uint32_t)__cvta_generic_to_shared(&sm.scale[warp][0][0][g * SUBS]);
  auto copy_step = [&]() {
    if (cj < j1) {
      const uint32_t rd = ring0 + (uint32_t)cslot * (4 * 32 * 16), sd = scale0 + (uint32_t)cslot * (2 * 32 * 4);
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        copy_bytes<16>(rd + (2 * r) * 512, wp[r]);
        copy_bytes<16>(rd + (2 * r + 1) * 512, wp[r] + 32);
        if (c == 0) copy_bytes<4 * SUBS>(sd + r * 128, sp[r]);  // its row's scales, for the row's four lanes
        wp[r] += 64;
        sp[r] += 8 * SUBS;
      }
      if (++cst == mine) {
        cst = 0;
        ++cj;
        next_job(cb);
        open_job();
      }
    }
    copies_commit();
    cslot = (cslot + 1) % FW_AHEAD;
  };
  if (mine > 0) {
    open_job();
    for (int i = 0; i < FW_AHEAD - 1; ++i) copy_step();
  }
  if (!GATED) wait_for_previous();  // the rows of h come from the launch before

  FewJob b = job_at(j0);
  int y = -1, cnt = 0, slot = 0;
  for (int j = j0; j < j1; ++j, next_job(b)) {
    if (b.y != y) {
      y = b.y;
      cnt = sm.count[sm.expert[y]];
      list_pairs(p, sm, id, sm.expert[y]);
    }
    const int c0 = 8 * b.pass;
    // token columns past the count repeat the last one and are not stored
    const int pair = sm.list[min(c0 + g, cnt - 1)];
    const T *xp = reinterpret_cast<const T *>(p.a) + (int64_t)(GATED ? pair / p.topk : pair) * p.Kd + 8 * c;
    uint4 x[2][2];
    auto load_tokens = [&](int st) {
      const T *q = xp + st * FW_STEP;
      if ((st + 1) * FW_STEP <= p.Kd) {
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k >> 1][k & 1] = *reinterpret_cast<const uint4 *>(q + 32 * k);
      } else {  // past the row's end: zeros
#pragma unroll
        for (int k = 0; k < 4; ++k)
          x[k >> 1][k & 1] = st * FW_STEP + 32 * k + 8 * c < p.Kd ? *reinterpret_cast<const uint4 *>(q + 32 * k)
                                                               : make_uint4(0u, 0u, 0u, 0u);
      }
    };
    float acc[2][4];
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[r][i] = 0.f;
    for (int s = 0; s < mine; ++s) {
      load_tokens(st0 + s);
      copies_wait<FW_AHEAD - 2>();
      __syncwarp();  // a lane's scales were copied by another one
      copy_step();
      constexpr int PER = 4 / SUBS;  // 32-k pieces of a group
      uint4 q[2][2];
      uint32_t sc[2][SUBS];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        q[r][0] = sm.ring[warp][slot][2 * r][lane];
        q[r][1] = sm.ring[warp][slot][2 * r + 1][lane];
#pragma unroll
        for (int i = 0; i < SUBS; ++i) sc[r][i] = sm.scale[warp][slot][r][g * SUBS + i];
      }
      slot = (slot + 1) % FW_AHEAD;
#pragma unroll
      for (int i = 0; i < SUBS; ++i) {
        float start[4];  // -(B + 8) sum x, by token column
        const float zero[4] = {0.f, 0.f, 0.f, 0.f};
        const uint32_t offset[4] = {OFFSET, OFFSET, OFFSET, OFFSET};
#pragma unroll
        for (int k = 0; k < PER; ++k) {
          const uint4 xv = x[(i * PER + k) >> 1][(i * PER + k) & 1];
          if (k == 0) mma_16816<T>(start, offset, xv.x, xv.y, zero);
          else mma_16816<T>(start, offset, xv.x, xv.y, start);
          mma_16816<T>(start, offset, xv.z, xv.w, start);
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float d[4];
#pragma unroll
          for (int k = 0; k < PER; ++k) {
            const int bl = (i * PER + k) >> 1, h = (i * PER + k) & 1;
            const uint32_t lo = h ? q[r][bl].y : q[r][bl].x, hi = h ? q[r][bl].w : q[r][bl].z;
            const uint4 xv = x[bl][h];
#pragma unroll
            for (int m = 0; m < 2; ++m) {
              const uint32_t fr[4] = {rf::int4_raw<T>(lo, 2 * m), rf::int4_raw<T>(hi, 2 * m),
                                      rf::int4_raw<T>(lo, 2 * m + 1), rf::int4_raw<T>(hi, 2 * m + 1)};
              if (k + m == 0) mma_16816<T>(d, fr, xv.x, xv.y, start);
              else mma_16816<T>(d, fr, m ? xv.z : xv.x, m ? xv.w : xv.y, d);
            }
          }
          const float2 f = scale_pair<T>(sc[r][i]);
          acc[r][0] = fmaf(d[0], f.x, acc[r][0]);
          acc[r][1] = fmaf(d[1], f.x, acc[r][1]);
          acc[r][2] = fmaf(d[2], f.y, acc[r][2]);
          acc[r][3] = fmaf(d[3], f.y, acc[r][3]);
        }
      }
    }
    // ---- the warps' partial sums, in warp order
    __syncthreads();  // the previous job's sums have been read
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int i = 0; i < 4; ++i) sm.red[warp][(r * 4 + i) * 32 + lane] = acc[r][i];
    __syncthreads();
    constexpr int PER = GATED ? 16 : 32;  // features of a row group
#pragma unroll
    for (int i = threadIdx.x; i < RG * PER * 8; i += FW_THREADS) {
      const int f = i % (RG * PER), col = i / (RG * PER);  // feature, token of the job
      const int r16 = f & 15, w0 = f / PER * KS;
      const int at = ((col & 1) + 2 * (r16 >> 3)) * 32 + (r16 & 7) * 4 + (col >> 1);
      const int64_t feat = (int64_t)b.unit * (RG * PER) + f;
      if (c0 + col >= cnt || feat >= p.N) continue;
      const int64_t row = sm.list[c0 + col];
      if constexpr (GATED) {
        float gt = 0.f, up = 0.f;
#pragma unroll
        for (int w = 0; w < KS; ++w) {
          gt += sm.red[w0 + w][at];
          up += sm.red[w0 + w][at + 4 * 32];
        }
        reinterpret_cast<T *>(p.out)[row * p.N + feat] = rf::Cvt<T>::from_f(rf::act_gate(p.act, gt) * up);
      } else {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < KS; ++w) v += sm.red[w0 + w][at + (f >> 4 & 1) * 4 * 32];
        reinterpret_cast<float *>(p.out)[row * p.N + feat] = v;
      }
    }
  }
  copies_wait<0>();
}

// Launches `kern` so that it may start while the previous launch on the stream
// drains (it waits for it itself, wait_for_previous).
template <typename... Params, typename... Args>
int launch_chained(const char *what, void (*kern)(Params...), dim3 grid, int threads, size_t smem, bool chained,
                   cudaStream_t st, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = chained ? 1 : 0;
  const cudaError_t err = cudaLaunchKernelEx(&cfg, kern, Params(args)...);
  if (err != cudaSuccess) {
    cudaGetLastError();
    return rf::fail(RF_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(err));
  }
  return RF_OK;
}

template <typename T, bool GATED, int SUBS, int KS>
int launch_few_k(FewArgs p, cudaStream_t st) {
  auto kern = int4_few_kernel<T, GATED, SUBS, KS>;
  const char *what = GATED ? "4-bit gated products (few rows)" : "4-bit down products (few rows)";
  static rf::PerDevice fit;
  const int resident = fit.get(rf::current_device(), [&]() -> int {
    int n = 0;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(FewShared)) != cudaSuccess) return 0;
    return cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, FW_THREADS, sizeof(FewShared)) == cudaSuccess ? n : 0;
  });
  if (resident < 1) {
    cudaGetLastError();
    return rf::fail(RF_ERR_CUDA, std::string(what) + ": the kernel does not fit this device");
  }
  p.units = (p.units + FW_WARPS / KS - 1) / (FW_WARPS / KS);
  // as many blocks as run at once share the jobs (at most units * pairs) evenly
  const int64_t most = (int64_t)p.units * p.pairs;
  const int64_t blocks = std::min<int64_t>(most, (int64_t)rf::num_sms() * resident);
  return launch_chained(what, kern, dim3((unsigned)blocks), FW_THREADS, sizeof(FewShared), !GATED, st, p);
}

template <typename T, bool GATED, int SUBS>
int launch_few_s(const FewArgs &p, cudaStream_t st) {
  const int64_t jobs = (int64_t)p.units * std::min(p.E, p.pairs);
  if (jobs >= FW_MANY_JOBS) return launch_few_k<T, GATED, SUBS, 2>(p, st);
  return launch_few_k<T, GATED, SUBS, 8>(p, st);
}

template <typename T, bool GATED>
int launch_few_t(const FewArgs &p, int group, cudaStream_t st) {
  if (group == 32) return launch_few_s<T, GATED, 4>(p, st);
  if (group == 64) return launch_few_s<T, GATED, 2>(p, st);
  return launch_few_s<T, GATED, 1>(p, st);
}

int launch_few(const rf::Int4Gemm &g, bool gated, const int32_t *ids, int topk, cudaStream_t st) {
  const rf::Int4Shape sh = rf::int4_shape(gated ? 2 * (int64_t)g.N : g.N, g.Kdim, g.group, gated);
  const int units = (int)(gated ? sh.half_blocks : (sh.row_blocks() + 1) / 2);
  const FewArgs p{g.a, g.w, g.scales, g.out, ids, (int)g.rows, topk, g.E, g.N, g.Kdim, g.act, units, sh};
  if (g.dtype == RF_F16) return gated ? launch_few_t<__half, true>(p, g.group, st) : launch_few_t<__half, false>(p, g.group, st);
  return gated ? launch_few_t<__nv_bfloat16, true>(p, g.group, st) : launch_few_t<__nv_bfloat16, false>(p, g.group, st);
}

// ------------------------------------------------------------------ combine
constexpr int CB_THREADS = 128;

struct CombineArgs {
  const float *y;
  const int32_t *row_of_slot;  // y's row of a pair (-1: none), or
  const int32_t *ids;          // the pair itself unless its id names no expert
  const float *w;
  const void *shared_y;
  const float *shared_scale;
  const void *residual;
  void *out;
  int64_t T;
  int K, H, E;
};

// One block per (token, 128 * 8 columns): fp32 sums in slot order, one
// rounding at the end.
template <typename T>
__global__ void __launch_bounds__(CB_THREADS) int4_combine_kernel(const CombineArgs a) {
  const int col = (blockIdx.y * CB_THREADS + threadIdx.x) * 8;
  wait_for_previous();
  if (col >= a.H) return;
  for (int64_t t = blockIdx.x; t < a.T; t += gridDim.x) {
    float acc[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = 0.f;
    for (int k = 0; k < a.K; ++k) {
      int64_t r = t * a.K + k;
      if (a.ids) r = (unsigned)a.ids[r] < (unsigned)a.E ? r : -1;
      else r = a.row_of_slot[r];
      if (r < 0) continue;  // an id that names no expert
      const float w = a.w[t * a.K + k];
      const float4 *p = reinterpret_cast<const float4 *>(a.y + r * a.H + col);
      const float4 u = p[0], v = p[1];
      const float f[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] = fmaf(w, f[i], acc[i]);
    }
    const int64_t at = t * a.H + col;
    float f[8];
    // ordinary loads, not the read-only path: out may be residual
    if (a.shared_y) {
      rf::unpack16<T>(__ldcg(reinterpret_cast<const uint4 *>(reinterpret_cast<const T *>(a.shared_y) + at)), f);
      const float s = a.shared_scale ? a.shared_scale[t] : 1.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] = fmaf(s, f[i], acc[i]);
    }
    if (a.residual) {
      rf::unpack16<T>(__ldcg(reinterpret_cast<const uint4 *>(reinterpret_cast<const T *>(a.residual) + at)), f);
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] += f[i];
    }
    *reinterpret_cast<uint4 *>(reinterpret_cast<T *>(a.out) + at) =
        make_uint4(rf::pack2<T>(acc[0], acc[1]), rf::pack2<T>(acc[2], acc[3]), rf::pack2<T>(acc[4], acc[5]),
                   rf::pack2<T>(acc[6], acc[7]));
  }
}

template <typename T>
int launch_combine(const CombineArgs &a, cudaStream_t st) {
  const int64_t gy = (a.H + CB_THREADS * 8 - 1) / (CB_THREADS * 8);
  const int64_t gx = std::min<int64_t>(a.T, std::max<int64_t>(1, (int64_t)rf::num_sms() * 16 / gy));
  return launch_chained("4-bit combine", int4_combine_kernel<T>, dim3((unsigned)gx, (unsigned)gy), CB_THREADS, 0, a.ids != nullptr,
                        st, a);
}

// ------------------------------------------------------------------ workspace
struct Layout {
  size_t offsets, counts, row_of_slot, src, permute, permute_bytes, x, h, y, total;
  int64_t rows;
};

size_t aligned(size_t v) { return (v + 255) & ~(size_t)255; }

Layout make_layout(int64_t T, int64_t K, int64_t E, int64_t H, int64_t I) {
  Layout l;
  l.rows = T * K;
  l.permute_bytes = rf_moe_permute_workspace_size(T * K, E);
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += aligned(bytes);
    return here;
  };
  l.offsets = take((size_t)(E + 1) * 4);
  l.counts = take((size_t)E * 4);
  l.row_of_slot = take((size_t)l.rows * 4);
  l.src = take((size_t)l.rows * 4);
  l.permute = take(l.permute_bytes);
  l.x = take((size_t)l.rows * (size_t)H * 2);
  l.h = take((size_t)l.rows * (size_t)I * 2);
  l.y = take((size_t)l.rows * (size_t)H * 4);
  l.total = at;
  return l;
}

bool sizes_ok(int64_t T, int64_t K, int64_t E, int64_t H, int64_t I) {
  return T >= 0 && K >= 1 && K <= KMAX && E >= 1 && E <= 1024 && H > 0 && I > 0 && H % 8 == 0 && I % 8 == 0 &&
         H <= ((int64_t)1 << 20) && I <= ((int64_t)1 << 20) && T <= 0x7fffffff / K;
}

// The CTA-pair kernel from this many rows per expert on (the mean over the
// experts that can have any: the counts are on the device).  Either side of it,
// us of few rows / CTA pairs: 60 experts of 2048 x 1408, 6.4 rows 95 / 119, 8.5
// rows 112 / 119, 12.8 rows 150 / 120; eight of 4096 x 14336, 8 rows 266 / 282,
// 12 rows 332 / 282; 64 experts, 9.4 rows 129 / 127.
constexpr int64_t PAIR_ROWS = 9;

bool use_pair(int64_t T, int64_t K, int64_t E) {
  const int impl = rf::gemm_impl();
  if (T * K > FW_PAIRS || impl == 5) return true;
  if (impl == 1) return false;
  return T * K >= PAIR_ROWS * std::min(E, T * K);
}

}  // namespace

extern "C" size_t rf_moe_int4_experts_workspace_size(int64_t T, int64_t K, int64_t E, int64_t H, int64_t I) {
  if (T <= 0 || !sizes_ok(T, K, E, H, I)) return 256;
  return make_layout(T, K, E, H, I).total;
}

extern "C" int rf_moe_int4_experts(const void *x, int dtype, const void *w1, const void *w1_scales,
                                   int64_t w1_group, const void *w2, const void *w2_scales, int64_t w2_group,
                                   const float *topk_weights, const int32_t *topk_ids, int64_t T, int64_t K, int64_t E,
                                   int64_t H, int64_t I, int activation, const void *shared_y,
                                   const float *shared_scale, const void *residual, void *out, void *workspace,
                                   size_t workspace_bytes, rf_stream_t stream) {
  RF_CHECK_ARG(dtype == RF_F16 || dtype == RF_BF16, "rf_moe_int4_experts: 4-bit experts serve bf16 and fp16 layers");
  RF_CHECK_ARG(activation >= RF_ACT_SILU && activation <= RF_ACT_GELU_TANH, "rf_moe_int4_experts: unknown activation");
  RF_CHECK_ARG(sizes_ok(T, K, E, H, I),
               "rf_moe_int4_experts: bad sizes (K <= 16, E <= 1024, H and I multiples of 8 up to 2^20, T * K < 2^31)");
  RF_CHECK_ARG(rf::int4_valid(2 * I, H, w1_group, true) && rf::int4_valid(H, I, w2_group, false),
               "rf_moe_int4_experts: group sizes must be 32, 64 or 128");
  RF_CHECK_ARG(w1 && w1_scales && w2 && w2_scales, "rf_moe_int4_experts: null weights");
  RF_CHECK_ARG(T == 0 || (x && topk_weights && topk_ids && out), "rf_moe_int4_experts: null pointer");
  RF_CHECK_ARG((uintptr_t)x % 16 == 0 && (uintptr_t)w1 % 16 == 0 && (uintptr_t)w1_scales % 16 == 0 &&
                   (uintptr_t)w2 % 16 == 0 && (uintptr_t)w2_scales % 16 == 0 && (uintptr_t)shared_y % 16 == 0 &&
                   (uintptr_t)residual % 16 == 0 && (uintptr_t)out % 16 == 0,
               "rf_moe_int4_experts: buffers must be 16-byte aligned");
  if (T == 0) return RF_OK;
  const Layout l = make_layout(T, K, E, H, I);
  RF_CHECK_ARG(workspace && workspace_bytes >= l.total && (uintptr_t)workspace % 256 == 0,
               "rf_moe_int4_experts: workspace too small (see rf_moe_int4_experts_workspace_size) or not 256-byte aligned");
  uint8_t *ws = (uint8_t *)workspace;
  int32_t *offsets = (int32_t *)(ws + l.offsets), *counts = (int32_t *)(ws + l.counts);
  int32_t *ros = (int32_t *)(ws + l.row_of_slot), *src = (int32_t *)(ws + l.src);
  cudaStream_t st = (cudaStream_t)stream;
  const bool pair = use_pair(T, K, E);
  const rf::Int4Gemm g{pair ? ws + l.x : x, (const uint8_t *)w1, w1_scales, ws + l.h, offsets, counts, l.rows, (int)E,
                       (int)H, (int)I, (int)w1_group, dtype, activation};
  const rf::Int4Gemm d{ws + l.h, (const uint8_t *)w2, w2_scales, ws + l.y, offsets, counts, l.rows, (int)E,
                       (int)I, (int)H, (int)w2_group, dtype, activation};
  int rc;
  if (pair) {
    rc = rf_moe_permute(topk_ids, T, K, E, 1, x, dtype, H, offsets, counts, ros, src, ws + l.x, ws + l.permute,
                        l.permute_bytes, stream);
    if (!rc) rc = rf::launch_int4_pair(g, true, st);
    if (!rc) rc = rf::launch_int4_pair(d, false, st);
  } else {
    rc = launch_few(g, true, topk_ids, (int)K, st);
    if (!rc) rc = launch_few(d, false, topk_ids, 1, st);
  }
  if (rc) return rc;
  const CombineArgs cb{(const float *)(ws + l.y), pair ? ros : nullptr, pair ? nullptr : topk_ids, topk_weights, shared_y,
                       shared_scale, residual, out, T, (int)K, (int)H, (int)E};
  return dtype == RF_F16 ? launch_combine<__half>(cb, st) : launch_combine<__nv_bfloat16>(cb, st);
}
