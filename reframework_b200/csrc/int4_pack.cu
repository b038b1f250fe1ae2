// Laying out 4-bit expert weights (int4.cuh): from codes and scales, from
// 16- or 32-bit weights (quantising them), and back to the layer dtype.
//
// Quantisation, per row and group of g along the reduction axis:
//   s = max|w| / 7 rounded to five significant bits (in the layer dtype),
//   code = clamp(round(w / s), -8, 7) + 8
// Five bits times the code's three is at most eight significant bits, so
// s * (code - 8) is exact in bf16 and fp16: the tensor-core form, whose
// operand is that product, then rounds no weight.  A group of zeros, or of
// magnitudes whose scale underflows the layer dtype, has s = 0.
// These run once per loaded weight; they are bound by reading it.
#include <cuda_bf16.h>

#include "int4.cuh"

namespace {

constexpr int THREADS = 256;

struct PackArgs {
  const uint8_t *codes;   // [S, N, K/2]
  const void *scales_in;  // [S, N, groups] in T
  const void *w;          // [S, N, K]
  uint8_t *data;
  void *scales;
  void *out;              // dequantize: [S, N, K]
  int64_t S, N, K;
  int group;
  rf::Int4Shape sh;
};

// Source row of packed row `r16` of row block rb (-1: padding).
__device__ __forceinline__ int64_t source_row(const rf::Int4Shape &sh, int64_t rb, int r16) {
  const int64_t half = rb / sh.half_blocks;
  const int64_t r = (rb - half * sh.half_blocks) * rf::I4_ROWS + r16;
  return r < sh.half_rows ? half * sh.half_rows + r : -1;
}

__device__ __forceinline__ uint32_t place(uint32_t word, int k, uint32_t code) {  // k = 0..7 in the word
  return word | (code << (4 * (k / 2 + 4 * (k & 1))));
}

// The k inside a block of a lane's j-th code of a row (j = 0..15).
__device__ __forceinline__ int lane_k(int lane, int j) { return 32 * (j >> 3) + 8 * (lane & 3) + (j & 7); }

// One thread per (slot, row block, k block, lane): 16 bytes of codes.
__global__ void __launch_bounds__(THREADS) int4_pack_kernel(const PackArgs a) {
  const int64_t n = a.S * a.sh.row_blocks() * a.sh.k_blocks * 32;
  for (int64_t i = (int64_t)blockIdx.x * THREADS + threadIdx.x; i < n; i += (int64_t)gridDim.x * THREADS) {
    const int lane = (int)(i & 31);
    const int64_t block = i >> 5;
    const int64_t kb = block % a.sh.k_blocks;
    const int64_t rbs = block / a.sh.k_blocks;
    const int64_t rb = rbs % a.sh.row_blocks(), s = rbs / a.sh.row_blocks();
    uint32_t word[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int64_t row = source_row(a.sh, rb, (lane >> 2) + 8 * h);
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const int64_t k = kb * rf::I4_K + lane_k(lane, j);
        uint32_t code = 8u;
        if (row >= 0 && k < a.K) {
          const uint8_t b = a.codes[((s * a.N + row) * a.K + k) >> 1];
          code = (k & 1) ? (uint32_t)(b >> 4) : (uint32_t)(b & 15);
        }
        word[2 * h + (j >> 3)] = place(word[2 * h + (j >> 3)], j & 7, code);
      }
    }
    reinterpret_cast<uint4 *>(a.data)[i] = make_uint4(word[0], word[1], word[2], word[3]);
  }
}

// One thread per (slot, row block, group, row).
template <typename T>
__global__ void __launch_bounds__(THREADS) int4_scales_kernel(const PackArgs a) {
  const int64_t n = a.S * a.sh.slot_scales();
  for (int64_t i = (int64_t)blockIdx.x * THREADS + threadIdx.x; i < n; i += (int64_t)gridDim.x * THREADS) {
    const int r16 = (int)(i % rf::I4_ROWS);
    const int64_t g = i / rf::I4_ROWS % a.sh.groups;
    const int64_t rbs = i / rf::I4_ROWS / a.sh.groups;
    const int64_t rb = rbs % a.sh.row_blocks(), s = rbs / a.sh.row_blocks();
    const int64_t row = source_row(a.sh, rb, r16);
    const int64_t groups = (a.K + a.group - 1) / a.group;
    reinterpret_cast<T *>(a.scales)[rbs * a.sh.groups * rf::I4_ROWS + rf::int4_scale_at(r16, g, rf::I4_STEP / a.group)] =
        row >= 0 && g < groups ? reinterpret_cast<const T *>(a.scales_in)[(s * a.N + row) * groups + g]
                               : rf::Cvt<T>::from_f(0.f);
  }
}

// A block handles one (slot, row block), its k in steps of 128: a warp takes
// every eighth row, its lanes the row's k (32 consecutive k are in one group),
// and the codes pass through shared memory into the stored order.
template <typename TW, typename T>
__global__ void __launch_bounds__(THREADS) int4_quantize_kernel(const PackArgs a) {
  __shared__ uint8_t code[rf::I4_ROWS][128];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t rbs = blockIdx.x;
  const int64_t rb = rbs % a.sh.row_blocks(), s = rbs / a.sh.row_blocks();
  const TW *w = reinterpret_cast<const TW *>(a.w);
  T *scales = reinterpret_cast<T *>(a.scales) + rbs * a.sh.groups * rf::I4_ROWS;
  uint8_t *data = a.data + rbs * a.sh.k_blocks * rf::I4_BLOCK;
  for (int64_t k0 = 0; k0 < a.sh.k_blocks * rf::I4_K; k0 += 128) {
    for (int r16 = warp; r16 < rf::I4_ROWS; r16 += THREADS / 32) {
      const int64_t row = source_row(a.sh, rb, r16);
      float v[4];  // k0 + lane + 32 i: 32 consecutive k belong to one group
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int64_t k = k0 + lane + 32 * i;
        v[i] = row >= 0 && k < a.K ? rf::Cvt<TW>::to_f(w[(s * a.N + row) * a.K + k]) : 0.f;
      }
      float m[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        m[i] = fabsf(v[i]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m[i] = fmaxf(m[i], __shfl_xor_sync(0xffffffffu, m[i], o));
      }
      const int per = a.group / 32;  // 32-wide pieces in a group: 1, 2 or 4
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float top = m[i];
        for (int j = 0; j < 4; ++j)
          if (j / per == i / per) top = fmaxf(top, m[j]);
        float sc = 0.f;
        if (top > 0.f) {
          int ex;
          const float f = frexpf(top / 7.f, &ex);
          sc = rf::Cvt<T>::to_f(rf::Cvt<T>::from_f(ldexpf(rintf(f * 32.f), ex - 5)));
        }
        const float q = sc > 0.f ? fminf(fmaxf(rintf(v[i] / sc), -8.f), 7.f) : 0.f;
        code[r16][lane + 32 * i] = (uint8_t)((int)q + 8);
        const int64_t g = (k0 + 32 * i) / a.group;
        if (lane == 0 && (32 * i) % a.group == 0 && g < a.sh.groups)
          scales[rf::int4_scale_at(r16, g, rf::I4_STEP / a.group)] = rf::Cvt<T>::from_f(row >= 0 ? sc : 0.f);
      }
    }
    __syncthreads();
    if (threadIdx.x < 64) {
      const int64_t kb = k0 / rf::I4_K + (threadIdx.x >> 5);
      if (kb < a.sh.k_blocks) {
        uint32_t word[4] = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int j = 0; j < 16; ++j)
            word[2 * h + (j >> 3)] = place(word[2 * h + (j >> 3)], j & 7,
                                           code[(lane >> 2) + 8 * h][(threadIdx.x >> 5) * 64 + lane_k(lane, j)]);
        reinterpret_cast<uint4 *>(data + kb * rf::I4_BLOCK)[lane] = make_uint4(word[0], word[1], word[2], word[3]);
      }
    }
    __syncthreads();
  }
}

// The stored weights as scale * (code - 8) in T.
template <typename T>
__global__ void __launch_bounds__(THREADS) int4_dequantize_kernel(const PackArgs a) {
  const int64_t n = a.S * a.sh.row_blocks() * a.sh.k_blocks * 32;
  for (int64_t i = (int64_t)blockIdx.x * THREADS + threadIdx.x; i < n; i += (int64_t)gridDim.x * THREADS) {
    const int lane = (int)(i & 31);
    const int64_t block = i >> 5;
    const int64_t kb = block % a.sh.k_blocks;
    const int64_t rbs = block / a.sh.k_blocks;
    const int64_t rb = rbs % a.sh.row_blocks(), s = rbs / a.sh.row_blocks();
    const uint4 q = reinterpret_cast<const uint4 *>(a.data)[i];
    const uint32_t word[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int64_t row = source_row(a.sh, rb, (lane >> 2) + 8 * h);
      if (row < 0) continue;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const int64_t k = kb * rf::I4_K + lane_k(lane, j);
        if (k >= a.K) continue;
        const uint32_t w = word[2 * h + (j >> 3)];
        const int code = (int)(w >> (4 * ((j & 7) / 2 + 4 * (j & 1))) & 15u);
        const float sc = rf::Cvt<T>::to_f(
            reinterpret_cast<const T *>(a.scales)[rbs * a.sh.groups * rf::I4_ROWS +
                                                  rf::int4_scale_at((lane >> 2) + 8 * h, k / a.group, rf::I4_STEP / a.group)]);
        reinterpret_cast<T *>(a.out)[(s * a.N + row) * a.K + k] = rf::Cvt<T>::from_f(sc * (float)(code - 8));
      }
    }
  }
}

int blocks_for(int64_t n) {
  const int64_t b = (n + THREADS - 1) / THREADS, cap = (int64_t)rf::num_sms() * 32;
  return (int)(b < cap ? b : cap);
}

template <typename TW>
void launch_quantize(const PackArgs &a, int dtype, cudaStream_t st) {
  const int blocks = (int)(a.S * a.sh.row_blocks());
  if (dtype == RF_F16) int4_quantize_kernel<TW, __half><<<blocks, THREADS, 0, st>>>(a);
  else int4_quantize_kernel<TW, __nv_bfloat16><<<blocks, THREADS, 0, st>>>(a);
}

}  // namespace

#define RF_CHECK_INT4(what)                                                                                   \
  RF_CHECK_ARG(dtype == RF_F16 || dtype == RF_BF16, what ": 4-bit weights serve bf16 and fp16 layers");        \
  RF_CHECK_ARG(S > 0 && rf::int4_valid(N, K, group_size, gated != 0),                                          \
               what ": rows (of each half) and K must be multiples of 8, group_size 32, 64 or 128");          \
  const rf::Int4Shape sh = rf::int4_shape(N, K, group_size, gated != 0);                                       \
  RF_CHECK_ARG(S <= 0x7fffffff / sh.row_blocks(), what ": too many rows")

extern "C" int64_t rf_moe_int4_data_size(int64_t S, int64_t N, int64_t K, int64_t group_size, int gated) {
  if (S <= 0 || !rf::int4_valid(N, K, group_size, gated != 0)) return -1;
  return S * rf::int4_shape(N, K, group_size, gated != 0).slot_bytes();
}

extern "C" int64_t rf_moe_int4_scales_count(int64_t S, int64_t N, int64_t K, int64_t group_size, int gated) {
  if (S <= 0 || !rf::int4_valid(N, K, group_size, gated != 0)) return -1;
  return S * rf::int4_shape(N, K, group_size, gated != 0).slot_scales();
}

extern "C" int rf_moe_int4_pack(const void *codes, const void *scales, int dtype, int64_t S, int64_t N, int64_t K,
                                int64_t group_size, int gated, void *data, void *packed_scales,
                                rf_stream_t stream) {
  RF_CHECK_INT4("rf_moe_int4_pack");
  RF_CHECK_ARG(codes && scales && data && packed_scales && (uintptr_t)data % 16 == 0 && (uintptr_t)packed_scales % 16 == 0,
               "rf_moe_int4_pack: null or unaligned pointer");
  PackArgs a{(const uint8_t *)codes, scales, nullptr, (uint8_t *)data, packed_scales, nullptr, S, N, K, (int)group_size, sh};
  cudaStream_t st = (cudaStream_t)stream;
  int4_pack_kernel<<<blocks_for(S * sh.slot_bytes() / 16), THREADS, 0, st>>>(a);
  if (dtype == RF_F16) int4_scales_kernel<__half><<<blocks_for(S * sh.slot_scales()), THREADS, 0, st>>>(a);
  else int4_scales_kernel<__nv_bfloat16><<<blocks_for(S * sh.slot_scales()), THREADS, 0, st>>>(a);
  return rf::check_launch("rf_moe_int4_pack");
}

extern "C" int rf_moe_int4_quantize(const void *w, int w_dtype, int dtype, int64_t S, int64_t N, int64_t K,
                                    int64_t group_size, int gated, void *data, void *packed_scales,
                                    rf_stream_t stream) {
  RF_CHECK_ARG(rf::valid_dtype(w_dtype), "rf_moe_int4_quantize: unknown dtype");
  RF_CHECK_INT4("rf_moe_int4_quantize");
  RF_CHECK_ARG(w && data && packed_scales && (uintptr_t)data % 16 == 0 && (uintptr_t)packed_scales % 16 == 0,
               "rf_moe_int4_quantize: null or unaligned pointer");
  PackArgs a{nullptr, nullptr, w, (uint8_t *)data, packed_scales, nullptr, S, N, K, (int)group_size, sh};
  cudaStream_t st = (cudaStream_t)stream;
  switch (w_dtype) {
    case RF_F32: launch_quantize<float>(a, dtype, st); break;
    case RF_F16: launch_quantize<__half>(a, dtype, st); break;
    default: launch_quantize<__nv_bfloat16>(a, dtype, st); break;
  }
  return rf::check_launch("rf_moe_int4_quantize");
}

extern "C" int rf_moe_int4_dequantize(const void *data, const void *packed_scales, int dtype, int64_t S, int64_t N,
                                      int64_t K, int64_t group_size, int gated, void *w, rf_stream_t stream) {
  RF_CHECK_INT4("rf_moe_int4_dequantize");
  RF_CHECK_ARG(w && data && packed_scales && (uintptr_t)data % 16 == 0 && (uintptr_t)packed_scales % 16 == 0,
               "rf_moe_int4_dequantize: null or unaligned pointer");
  PackArgs a{nullptr, nullptr, nullptr, (uint8_t *)data, (void *)packed_scales, w, S, N, K, (int)group_size, sh};
  cudaStream_t st = (cudaStream_t)stream;
  const int blocks = blocks_for(S * sh.slot_bytes() / 16);
  if (dtype == RF_F16) int4_dequantize_kernel<__half><<<blocks, THREADS, 0, st>>>(a);
  else int4_dequantize_kernel<__nv_bfloat16><<<blocks, THREADS, 0, st>>>(a);
  return rf::check_launch("rf_moe_int4_dequantize");
}
