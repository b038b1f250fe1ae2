// The routed experts of a MoE layer with 4-bit weights (int4.cuh).
//
//   h[r, j] = act(x[r] . W1g[e, j]) * (x[r] . W1u[e, j])      rounded to the layer dtype
//   y[r, n] = h[r] . W2[e, n]                                 fp32
//   out[t]  = round(sum_k w[t, k] y[row(t, k)] + shared_scale * shared_y + residual)
// for the rows r that the permute gives expert e.  h is rounded because it is
// the second product's 16-bit operand; everything else stays fp32 up to out.
//
// Few rows per expert (int4_skinny_kernel): bound by reading the weights, half
// a byte each.  A block takes 32 weight rows (gated: 16 gate and their 16 up
// rows) of one expert over the whole reduction, its eight warps one eighth of
// it each; a lane's 16-byte word of the stored layout is its fragment of four
// 16 x 16 tiles of mma.sync, the codes as exact 16-bit integers, and the
// tokens (8 to a tile) are read straight from their rows.  A group's sums are
// scaled in fp32 after its products.  The eight partial sums meet in shared
// memory in warp order, so results do not depend on timing.
#include <algorithm>
#include <string>

#include "gemm.cuh"
#include "int4.cuh"

RF_DEVICE_ERROR_WORD();

namespace {

constexpr int SK_WARPS = 8;
constexpr int SK_THREADS = SK_WARPS * 32;
constexpr int SK_UNROLL = 4;  // k blocks whose loads are in flight together
constexpr int KMAX = 16;

struct SkinnyArgs {
  const void *a;        // x [tokens, Kd] (gated) or h [rows, Kd]
  const uint8_t *w;
  const void *scales;
  void *out;            // h [rows, N] in T (gated) or y [rows, N] fp32
  const int32_t *offsets, *counts;
  const int32_t *src;   // gated: row -> token * topk + slot
  int topk, E, N, Kd, group, act;
  rf::Int4Shape sh;
};

template <typename T>
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma_16816<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma_16816<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint4 ldg_stream(const uint4 *p) {  // weights pass through once: not kept in L1
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

// The y-th expert (ascending) that has rows, or -1.
__device__ __forceinline__ int nth_active(const int32_t *counts, int E, int y) {
  const int lane = threadIdx.x & 31;
  for (int c = 0; c < E; c += 32) {
    const unsigned b = __ballot_sync(0xffffffffu, c + lane < E && counts[c + lane] > 0);
    const int n = __popc(b);
    if (y < n) return c + (int)__fns(b, 0, y + 1);
    y -= n;
  }
  return -1;
}

// Two neighbouring 16-bit scales (rows r and r + 8) as floats.
template <typename T>
__device__ __forceinline__ float2 scale_pair(uint32_t v) {
  if constexpr (sizeof(T) == 2 && std::is_same<T, __half>::value) {
    return __half22float2(*reinterpret_cast<const __half2 *>(&v));
  } else {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  }
}

// SUB: scale groups in a 64-k block (2 for groups of 32, else 1).
template <typename T, int NT, bool GATED, int SUB>
__global__ void __launch_bounds__(SK_THREADS) int4_skinny_kernel(const SkinnyArgs p) {
  __shared__ float red[SK_WARPS][2 * NT * 4 * 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, c = lane & 3;
  const int e = nth_active(p.counts, p.E, blockIdx.y);
  if (e < 0) return;
  const int row0 = p.offsets[e], cnt = p.counts[e];
  const int unit = blockIdx.x;
  const int KB = (int)p.sh.k_blocks, groups = (int)p.sh.groups;
  const int64_t rb1 = GATED ? p.sh.half_blocks + unit : min((int64_t)(2 * unit + 1), p.sh.row_blocks() - 1);
  const uint4 *wp[2];
  const uint32_t *sp[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int64_t b = (int64_t)e * p.sh.row_blocks() + (r ? rb1 : (int64_t)(GATED ? unit : 2 * unit));
    wp[r] = reinterpret_cast<const uint4 *>(p.w + b * KB * rf::I4_BLOCK) + lane;
    sp[r] = reinterpret_cast<const uint32_t *>(reinterpret_cast<const T *>(p.scales) + b * groups * rf::I4_ROWS) + g;
  }
  const int kb0 = KB * warp / SK_WARPS, kb1 = KB * (warp + 1) / SK_WARPS;
  const T *a = reinterpret_cast<const T *>(p.a);
  for (int c0 = 0; c0 < cnt; c0 += 8 * NT) {
    const T *xp[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = c0 + 8 * n + g;
      xp[n] = nullptr;
      if (r < cnt) xp[n] = a + (int64_t)(GATED ? p.src[row0 + r] / p.topk : row0 + r) * p.Kd;
    }
    float acc[2][NT][4];
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[r][n][j] = 0.f;
    for (int kb = kb0; kb < kb1; kb += SK_UNROLL) {
      uint4 q[SK_UNROLL][2], x[SK_UNROLL][NT][2];
      uint32_t s[SK_UNROLL][2][SUB];
#pragma unroll
      for (int u = 0; u < SK_UNROLL; ++u) {
        const bool in = kb + u < kb1;
        const int k = (kb + u) * rf::I4_K;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          q[u][r] = in ? ldg_stream(wp[r] + (int64_t)(kb + u) * 32) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
          for (int h = 0; h < SUB; ++h) {
            const int gr = (k + 32 * h) / p.group;  // past the last group only where the codes are padding
            s[u][r][h] = in && gr < groups ? __ldg(sp[r] + (int64_t)gr * 8) : 0u;
          }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int kx = k + 32 * h + 8 * c;
            x[u][n][h] = in && xp[n] && kx < p.Kd ? __ldg(reinterpret_cast<const uint4 *>(xp[n] + kx))
                                                 : make_uint4(0u, 0u, 0u, 0u);
          }
      }
#pragma unroll
      for (int u = 0; u < SK_UNROLL; ++u) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float d[NT][4];
#pragma unroll
          for (int h = 0; h < 2; ++h) {  // the block's halves: words h of rows g and g + 8
            if (h == 0 || SUB == 2) {
#pragma unroll
              for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int j = 0; j < 4; ++j) d[n][j] = 0.f;
            }
            const uint32_t lo = h ? q[u][r].y : q[u][r].x, hi = h ? q[u][r].w : q[u][r].z;
#pragma unroll
            for (int m = 0; m < 2; ++m) {
              const uint32_t fr[4] = {rf::int4_pair<T>(lo, 2 * m), rf::int4_pair<T>(hi, 2 * m),
                                      rf::int4_pair<T>(lo, 2 * m + 1), rf::int4_pair<T>(hi, 2 * m + 1)};
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                const uint4 xv = x[u][n][h];
                mma_16816<T>(d[n], fr, m ? xv.z : xv.x, m ? xv.w : xv.y);
              }
            }
            if (h == 1 || SUB == 2) {
              const float2 f = scale_pair<T>(s[u][r][SUB == 2 ? h : 0]);
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                acc[r][n][0] = fmaf(d[n][0], f.x, acc[r][n][0]);
                acc[r][n][1] = fmaf(d[n][1], f.x, acc[r][n][1]);
                acc[r][n][2] = fmaf(d[n][2], f.y, acc[r][n][2]);
                acc[r][n][3] = fmaf(d[n][3], f.y, acc[r][n][3]);
              }
            }
          }
        }
      }
    }
    // ---- the warps' partial sums, in warp order
    __syncthreads();  // the previous chunk's sums have been read
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) red[warp][((r * NT + n) * 4 + j) * 32 + lane] = acc[r][n][j];
    __syncthreads();
    constexpr int PER = GATED ? 16 : 32;  // features of a unit
    for (int i = threadIdx.x; i < PER * 8 * NT; i += SK_THREADS) {
      const int f = i % PER, col = i / PER;  // feature, token of the chunk
      const int r16 = f & 15;
      const int at = ((col >> 3) * 4 + (col & 1) + 2 * (r16 >> 3)) * 32 + (r16 & 7) * 4 + ((col & 7) >> 1);
      if (c0 + col >= cnt) continue;
      const int64_t row = row0 + c0 + col;
      if constexpr (GATED) {
        float gt = 0.f, up = 0.f;
#pragma unroll
        for (int w = 0; w < SK_WARPS; ++w) {
          gt += red[w][at];
          up += red[w][at + NT * 4 * 32];
        }
        const int64_t feat = (int64_t)unit * 16 + f;
        if (feat < p.N) reinterpret_cast<T *>(p.out)[row * p.N + feat] = rf::Cvt<T>::from_f(rf::act_gate(p.act, gt) * up);
      } else {
        float y = 0.f;
#pragma unroll
        for (int w = 0; w < SK_WARPS; ++w) y += red[w][at + (f >> 4) * NT * 4 * 32];
        const int64_t feat = (int64_t)unit * 32 + f;
        if (feat < p.N) reinterpret_cast<float *>(p.out)[row * p.N + feat] = y;
      }
    }
  }
}

template <typename T, int NT>
int launch_skinny_t(const SkinnyArgs &p, bool gated, int max_active, cudaStream_t st) {
  const int units = (int)(gated ? p.sh.half_blocks : (p.sh.row_blocks() + 1) / 2);
  const dim3 grid(units, max_active);
  if (gated) {
    if (p.group == 32) int4_skinny_kernel<T, NT, true, 2><<<grid, SK_THREADS, 0, st>>>(p);
    else int4_skinny_kernel<T, NT, true, 1><<<grid, SK_THREADS, 0, st>>>(p);
  } else {
    if (p.group == 32) int4_skinny_kernel<T, NT, false, 2><<<grid, SK_THREADS, 0, st>>>(p);
    else int4_skinny_kernel<T, NT, false, 1><<<grid, SK_THREADS, 0, st>>>(p);
  }
  return rf::check_launch(gated ? "4-bit gated products" : "4-bit down products");
}

int launch_skinny(const rf::Int4Gemm &g, bool gated, const int32_t *src, int topk, int max_active, cudaStream_t st) {
  const SkinnyArgs p{g.a, g.w, g.scales, g.out, g.offsets, g.counts, src, topk, g.E, g.N, g.Kdim, g.group, g.act,
                     rf::int4_shape(gated ? 2 * (int64_t)g.N : g.N, g.Kdim, g.group, gated)};
  if (g.dtype == RF_F16) return launch_skinny_t<__half, 1>(p, gated, max_active, st);
  return launch_skinny_t<__nv_bfloat16, 1>(p, gated, max_active, st);
}

// ------------------------------------------------------------------ combine
constexpr int CB_THREADS = 128;

struct CombineArgs {
  const float *y;
  const int32_t *row_of_slot;
  const float *w;
  const void *shared_y;
  const float *shared_scale;
  const void *residual;
  void *out;
  int64_t T;
  int K, H;
};

// One block per (token, 128 * 8 columns): fp32 sums in slot order, one
// rounding at the end.
template <typename T>
__global__ void __launch_bounds__(CB_THREADS) int4_combine_kernel(const CombineArgs a) {
  const int col = (blockIdx.y * CB_THREADS + threadIdx.x) * 8;
  if (col >= a.H) return;
  for (int64_t t = blockIdx.x; t < a.T; t += gridDim.x) {
    float acc[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = 0.f;
    for (int k = 0; k < a.K; ++k) {
      const int r = a.row_of_slot[t * a.K + k];
      if (r < 0) continue;  // an id that names no expert
      const float w = a.w[t * a.K + k];
      const float4 *p = reinterpret_cast<const float4 *>(a.y + (int64_t)r * a.H + col);
      const float4 u = __ldg(p), v = __ldg(p + 1);
      const float f[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] = fmaf(w, f[i], acc[i]);
    }
    const int64_t at = t * a.H + col;
    float f[8];
    if (a.shared_y) {
      rf::unpack16<T>(__ldg(reinterpret_cast<const uint4 *>(reinterpret_cast<const T *>(a.shared_y) + at)), f);
      const float s = a.shared_scale ? a.shared_scale[t] : 1.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] = fmaf(s, f[i], acc[i]);
    }
    if (a.residual) {
      rf::unpack16<T>(__ldg(reinterpret_cast<const uint4 *>(reinterpret_cast<const T *>(a.residual) + at)), f);
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
  int4_combine_kernel<T><<<dim3((unsigned)gx, (unsigned)gy), CB_THREADS, 0, st>>>(a);
  return rf::check_launch("4-bit combine");
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
         H < ((int64_t)1 << 28) && I < ((int64_t)1 << 28) && T <= 0x7fffffff / K;
}

// The CTA-pair kernel from this many rows per expert on (the mean over the
// experts that can have any: the counts are on the device).
constexpr int64_t PAIR_ROWS = 8;

bool use_pair(int64_t T, int64_t K, int64_t E) {
  const int impl = rf::gemm_impl();
  if (impl == 1) return false;
  if (impl == 5) return true;
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
               "rf_moe_int4_experts: bad sizes (K <= 16, E <= 1024, H and I multiples of 8, T * K < 2^31)");
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
  int rc = rf_moe_permute(topk_ids, T, K, E, 1, pair ? x : nullptr, dtype, pair ? H : 0, offsets, counts, ros, src,
                          pair ? ws + l.x : nullptr, ws + l.permute, l.permute_bytes, stream);
  if (rc) return rc;
  const rf::Int4Gemm g{pair ? ws + l.x : x, (const uint8_t *)w1, w1_scales, ws + l.h, offsets, counts, l.rows, (int)E,
                       (int)H, (int)I, (int)w1_group, dtype, activation};
  const rf::Int4Gemm d{ws + l.h, (const uint8_t *)w2, w2_scales, ws + l.y, offsets, counts, l.rows, (int)E,
                       (int)I, (int)H, (int)w2_group, dtype, activation};
  const int max_active = (int)std::min<int64_t>(E, T * K);
  rc = pair ? rf::launch_int4_pair(g, true, st) : launch_skinny(g, true, src, (int)K, max_active, st);
  if (rc) return rc;
  rc = pair ? rf::launch_int4_pair(d, false, st) : launch_skinny(d, false, nullptr, 1, max_active, st);
  if (rc) return rc;
  const CombineArgs cb{(const float *)(ws + l.y), ros, topk_weights, shared_y, shared_scale, residual, out, T, (int)K, (int)H};
  return dtype == RF_F16 ? launch_combine<__half>(cb, st) : launch_combine<__nv_bfloat16>(cb, st);
}
