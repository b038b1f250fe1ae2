// Residual addition + RMSNorm + e4m3 output with scales, one pass over the rows.
//
// Per row (reframework/layers/norm.py:27-53 up to the last step):
//   r = round(x + residual)                 in the layer dtype (r = x without a residual)
//   z = r * 1/sqrt(mean(r^2) + eps) * w (+ b)   in fp32, on the stored r
//   per group of g columns (g = H: the whole row):
//     scale = max|z| / 448, q = e4m3(z / scale)   (448: the largest e4m3)
// An all-zero group has scale 1; a group holding a NaN or an infinity has
// scale NaN and zero codes, so that every value it stands for is NaN.
//
// Each input element is read once and kept in registers across the reductions (sum
// of squares, then max|z|), each output written once.  The sums and z are fp32; the
// roundings are those of the outputs' types.  A row belongs to TPR threads (a warp,
// or a small block) with up to four 16-byte vectors each: few threads per barrier,
// many independent rows per SM.  A block has nothing on its way behind its own
// row's loads: 8192 x 2048 with groups of 128 and the 16-bit row takes 31.5-33 us,
// 70-74 % of the measured HBM rate (one barrier a row, 3.5 waves of blocks, issue
// slots 64 % busy); blocks of 256 threads a row took 44, a warp of eight vectors 45.
#include <cuda_fp8.h>

#include "common.cuh"

namespace {

constexpr float E4M3_MAX = 448.0f;
constexpr float MIN_SCALE = 0x1p-126f;  // keeps 1 / scale finite
constexpr unsigned FULL = 0xffffffffu;

struct NormArgs {
  const void *x;
  const void *residual;  // may be NULL
  const float *w;
  const float *b;        // may be NULL
  void *residual_out;    // may be NULL without a residual
  void *normed;          // may be NULL
  uint8_t *q;            // [T, H] e4m3; may be NULL (then so is scales)
  float *scales;         // [T, H / g]
  int64_t T;
  int H;
  int lanes;             // threads that share a group: g / V (0: the whole row)
  int n_groups;          // H / g
  float eps;
};

// Over the threads of a row: a warp, or the block's warps in warp order.
template <int WARPS>
__device__ __forceinline__ float row_sum(float v, float *red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(FULL, v, o);
  if constexpr (WARPS > 1) {
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) v += red[w];
  }
  return v;
}
template <int WARPS>
__device__ __forceinline__ uint32_t row_max(uint32_t v, uint32_t *red) {
  v = __reduce_max_sync(FULL, v);
  if constexpr (WARPS > 1) {
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int w = 1; w < WARPS; ++w) v = max(v, red[w]);
  }
  return v;
}

// Magnitudes are compared as the integers of their bits: the same order, and a
// NaN (above the infinity's bits) is not lost as in a float maximum.
constexpr uint32_t INF_BITS = 0x7f800000u;
__device__ __forceinline__ uint32_t mag_bits(float z) { return __float_as_uint(z) & 0x7fffffffu; }

// max|z| of a group -> its scale, and 1 / scale (0 for a group that is not finite).
__device__ __forceinline__ float scale_of(uint32_t top) {
  if (top == 0u) return 1.f;
  if (top >= INF_BITS) return NAN;
  return fmaxf(__uint_as_float(top) / E4M3_MAX, MIN_SCALE);
}
__device__ __forceinline__ float inverse_of(uint32_t top) {
  const float amax = __uint_as_float(top);
  if (amax > 0x1p-100f && amax < 0x1p100f) return __fdividef(E4M3_MAX, amax);  // within 2 ulp
  if (top >= INF_BITS) return 0.f;
  return top == 0u ? 1.f : 1.0f / scale_of(top);
}

template <typename T, int V>
__device__ __forceinline__ void store_vec(T *p, const float *f) {
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4 *>(p) = make_float4(f[0], f[1], f[2], f[3]);
  } else {
    *reinterpret_cast<uint4 *>(p) =
        make_uint4(rf::pack2<T>(f[0], f[1]), rf::pack2<T>(f[2], f[3]), rf::pack2<T>(f[4], f[5]), rf::pack2<T>(f[6], f[7]));
  }
}

template <int V>
__device__ __forceinline__ void load_f32(const float *p, int at, float (&f)[V]) {
  if ((reinterpret_cast<uintptr_t>(p) & 15) == 0) {
#pragma unroll
    for (int i = 0; i < V; i += 4) {
      const float4 v = __ldg(reinterpret_cast<const float4 *>(p + at + i));
      f[i] = v.x, f[i + 1] = v.y, f[i + 2] = v.z, f[i + 3] = v.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = __ldg(p + at + i);
  }
}

__device__ __forceinline__ uint32_t e4m3x4(const float *z, float inv) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(z[0] * inv, z[1] * inv), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(z[2] * inv, z[3] * inv), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}

// WARPS warps per row, up to VPT 16-byte vectors per thread; a block holds one
// row, or four where a row is a warp's.
template <typename T, int WARPS, int VPT>
__global__ void __launch_bounds__(WARPS == 1 ? 128 : WARPS * 32) add_rmsnorm_q8_kernel(const NormArgs a) {
  constexpr int V = 16 / sizeof(T);
  constexpr int TPR = WARPS * 32;  // threads of a row
  __shared__ float sum_red[WARPS];
  __shared__ uint32_t max_red[WARPS];
  const int tid = WARPS == 1 ? (threadIdx.x & 31) : threadIdx.x;
  const int nvec = a.H / V;
  const T *x = reinterpret_cast<const T *>(a.x);
  const T *res = reinterpret_cast<const T *>(a.residual);
  const int64_t t = WARPS == 1 ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5) : (int64_t)blockIdx.x;
  if (t >= a.T) return;
  {
    float z[VPT][V];
    uint4 xv[VPT], rv[VPT];
#pragma unroll
    for (int u = 0; u < VPT; ++u) {
      const int v = tid + u * TPR;
      const int64_t at = t * a.H + (int64_t)v * V;
      // not the read-only path: residual_out may be either buffer.  Past L1, as that
      // path is; through L1 8192 x 2048 rows took 34.0 us, not 31.5.
      xv[u] = v < nvec ? __ldcg(reinterpret_cast<const uint4 *>(x + at)) : make_uint4(0u, 0u, 0u, 0u);
      if (res) rv[u] = v < nvec ? __ldcg(reinterpret_cast<const uint4 *>(res + at)) : make_uint4(0u, 0u, 0u, 0u);
    }
    float ss = 0.f;
#pragma unroll
    for (int u = 0; u < VPT; ++u) {
      const int v = tid + u * TPR;
      rf::unpack16<T>(xv[u], z[u]);
      if (res) {
        float f[V];
        rf::unpack16<T>(rv[u], f);
#pragma unroll
        for (int i = 0; i < V; ++i) z[u][i] = rf::round_to<T>(__fadd_rn(z[u][i], f[i]));
      }
      if (a.residual_out && v < nvec)
        store_vec<T, V>(reinterpret_cast<T *>(a.residual_out) + t * a.H + (int64_t)v * V, z[u]);
#pragma unroll
      for (int i = 0; i < V; ++i) ss = fmaf(z[u][i], z[u][i], ss);
    }
    const float inv = 1.0f / sqrtf(row_sum<WARPS>(ss, sum_red) / (float)a.H + a.eps);
    uint32_t top = 0u;  // of this thread's columns (the whole row is one group)
    uint32_t vmax[VPT]; // of one vector
#pragma unroll
    for (int u = 0; u < VPT; ++u) {
      const int v = tid + u * TPR;
      vmax[u] = 0u;
      if (v < nvec) {
        float w[V], bias[V];
        load_f32<V>(a.w, v * V, w);
        if (a.b) load_f32<V>(a.b, v * V, bias);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          z[u][i] = z[u][i] * inv * w[i];
          if (a.b) z[u][i] += bias[i];
          vmax[u] = max(vmax[u], mag_bits(z[u][i]));
        }
      }
      top = max(top, vmax[u]);
    }
    float is[VPT];
    if (a.lanes == 0) {
      top = row_max<WARPS>(top, max_red);
      is[0] = inverse_of(top);
#pragma unroll
      for (int u = 1; u < VPT; ++u) is[u] = is[0];
      if (tid == 0 && a.q) a.scales[t] = scale_of(top);
    } else {
#pragma unroll
      for (int u = 0; u < VPT; ++u) {
        for (int o = a.lanes >> 1; o > 0; o >>= 1) vmax[u] = max(vmax[u], __shfl_xor_sync(FULL, vmax[u], o));
        is[u] = inverse_of(vmax[u]);
        const int v = tid + u * TPR;
        if (v < nvec && v % a.lanes == 0 && a.q) a.scales[t * a.n_groups + v / a.lanes] = scale_of(vmax[u]);
      }
    }
#pragma unroll
    for (int u = 0; u < VPT; ++u) {
      const int v = tid + u * TPR;
      if (v >= nvec) continue;
      const int64_t at = t * a.H + (int64_t)v * V;
      if (a.normed) store_vec<T, V>(reinterpret_cast<T *>(a.normed) + at, z[u]);
      if (!a.q) continue;
      uint32_t q[V / 4];
#pragma unroll
      for (int i = 0; i < V / 4; ++i) q[i] = is[u] != 0.f ? e4m3x4(z[u] + 4 * i, is[u]) : 0u;
      if constexpr (V == 8) *reinterpret_cast<uint2 *>(a.q + at) = make_uint2(q[0], q[1]);
      else *reinterpret_cast<uint32_t *>(a.q + at) = q[0];
    }
  }
}

template <typename T, int WARPS, int VPT>
int launch_v(const NormArgs &a, cudaStream_t st) {
  const int64_t blocks = WARPS == 1 ? (a.T + 3) / 4 : a.T;
  add_rmsnorm_q8_kernel<T, WARPS, VPT><<<(unsigned)blocks, WARPS == 1 ? 128 : WARPS * 32, 0, st>>>(a);
  return rf::check_launch("rf_moe_add_rmsnorm_q8");
}

// Few rows leave SMs idle, so a row gets twice the threads (64 rows of 4096:
// 3.5 us against 4.2); with many, four vectors a thread keep more bytes in
// flight for each barrier (2047 rows of 6144: 15.8 us against 19.1; 16.4-17.4
// with inputs from HBM: two barriers a row, 2.8 waves).
template <typename T>
int launch_t(const NormArgs &a, cudaStream_t st) {
  const int nvec = a.H / (16 / (int)sizeof(T));
  if (nvec <= 32) return launch_v<T, 1, 1>(a, st);
  if (nvec <= 64) return launch_v<T, 1, 2>(a, st);
  if (a.T <= 2 * rf::num_sms() && nvec <= 1024) {
    if (nvec <= 128) return launch_v<T, 2, 2>(a, st);
    if (nvec <= 256) return launch_v<T, 4, 2>(a, st);
    if (nvec <= 512) return launch_v<T, 8, 2>(a, st);
    return launch_v<T, 16, 2>(a, st);
  }
  switch ((nvec + 127) / 128) {
    case 1: return launch_v<T, 1, 4>(a, st);
    case 2: return launch_v<T, 2, 4>(a, st);
    case 3: return launch_v<T, 3, 4>(a, st);
    case 4: return launch_v<T, 4, 4>(a, st);
    case 5: return launch_v<T, 5, 4>(a, st);
    case 6: return launch_v<T, 6, 4>(a, st);
    case 7: return launch_v<T, 7, 4>(a, st);
    case 8: return launch_v<T, 8, 4>(a, st);
    default: break;
  }
  if (nvec <= 2048) return launch_v<T, 16, 4>(a, st);
  return launch_v<T, 32, 4>(a, st);  // up to 65536 bytes
}

}  // namespace

extern "C" int rf_moe_add_rmsnorm_q8(const void *x, const void *residual, int64_t T, int64_t H, int dtype,
                                     const float *norm_weight, const float *norm_bias, float eps,
                                     int64_t group_size, void *residual_out, void *normed_out, void *q,
                                     float *scales, rf_stream_t stream) {
  RF_CHECK_ARG(rf::valid_dtype(dtype), "rf_moe_add_rmsnorm_q8: unknown dtype");
  RF_CHECK_ARG(T >= 0 && T <= 0x7fffffff && H > 0 && H < ((int64_t)1 << 30), "rf_moe_add_rmsnorm_q8: bad sizes");
  const int64_t esz = (int64_t)rf::dtype_size(dtype);
  RF_CHECK_ARG((H * esz) % 16 == 0, "rf_moe_add_rmsnorm_q8: H * element size must be a multiple of 16 bytes");
  RF_CHECK_ARG(eps >= 0.f, "rf_moe_add_rmsnorm_q8: eps must be >= 0");
  RF_CHECK_ARG(group_size == 0 || ((group_size == 32 || group_size == 64 || group_size == 128) && H % group_size == 0),
               "rf_moe_add_rmsnorm_q8: group_size must be 0 (the row), 32, 64 or 128 and divide H");
  if (H * esz > 65536) return rf::fail(RF_ERR_UNSUPPORTED, "rf_moe_add_rmsnorm_q8: a row holds at most 65536 bytes");
  RF_CHECK_ARG(T == 0 || (x && norm_weight && !q == !scales && (q || normed_out) && (residual_out || !residual)),
               "rf_moe_add_rmsnorm_q8: null pointer");
  RF_CHECK_ARG((uintptr_t)x % 16 == 0 && (uintptr_t)residual % 16 == 0 && (uintptr_t)residual_out % 16 == 0 &&
                   (uintptr_t)normed_out % 16 == 0 && (uintptr_t)q % 16 == 0,
               "rf_moe_add_rmsnorm_q8: buffers must be 16-byte aligned");
  RF_CHECK_ARG(T == 0 || ((!q || (q != residual_out && q != normed_out)) && (!normed_out || normed_out != residual_out)),
               "rf_moe_add_rmsnorm_q8: the outputs must not alias");
  if (T == 0) return RF_OK;
  NormArgs a{x, residual, norm_weight, norm_bias, residual_out, normed_out, (uint8_t *)q, scales, T, (int)H, 0, 1, eps};
  if (group_size) {
    a.lanes = (int)(group_size * esz / 16);
    a.n_groups = (int)(H / group_size);
  }
  cudaStream_t st = (cudaStream_t)stream;
  switch (dtype) {
    case RF_F32: return launch_t<float>(a, st);
    case RF_F16: return launch_t<__half>(a, st);
    default: return launch_t<__nv_bfloat16>(a, st);
  }
}
