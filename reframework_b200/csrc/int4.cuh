// 4-bit expert weights with group scales: the stored layout and the device
// code that turns codes into 16-bit values.
//
// A weight is scale[n, k / g] * (code[n, k] - 8), code in 0..15, g in
// {32, 64, 128} along the reduction axis.  Stored per expert slot:
//   data   [row blocks][k blocks][512 bytes]        16 rows x 64 k to a block
//   scales [row blocks][steps][8][128 / g][2]       in the layer dtype
// with an even number of k blocks, two to a step of 128 k,
// so that a warp reads a block as 32 consecutive 16-byte words.  Lane
// 4 * r + c (r = 0..7, c = 0..3) holds, as four 32-bit words of 8 codes: row
// r's k = 8 c .. 8 c + 7, its k = 32 + 8 c .. 32 + 8 c + 7, and the same of row
// r + 8.  Those are the rows and, with k renamed the same way for the other
// operand, the k of the lane's fragments of two 16 x 16 tiles of mma.sync per
// half of the block (a scale group of 32 is a half), and four 16-byte pieces
// of a K-major shared-memory tile.  In a word, code 2 i sits in nibble i and
// code 2 i + 1 in nibble i + 4, so that one shift and one mask give the
// neighbouring pair as two 16-bit halves.  The scales of a step are stored row r
// = 0..7 first, then group, then row r or r + 8: a lane's are one word to 16 bytes.
// Rows and k past the weight's own are stored as code 8 (zero) with scale 0;
// a gated weight's gate and up halves are padded to whole row blocks each.
#pragma once

#include <type_traits>

#include "common.cuh"
#include "per_device.cuh"

namespace rf {

constexpr int I4_ROWS = 16, I4_K = 64, I4_BLOCK = 512, I4_STEP = 128;

struct Int4Shape {
  int64_t half_rows;   // rows of one half (N, or N / 2 gated)
  int halves;          // 2 gated, 1 otherwise
  int64_t half_blocks; // row blocks of one half
  int64_t k_blocks;    // even
  int64_t groups;      // scale groups along K, padded to whole steps

  __host__ __device__ int64_t row_blocks() const { return half_blocks * halves; }
  __host__ __device__ int64_t slot_bytes() const { return row_blocks() * k_blocks * I4_BLOCK; }
  __host__ __device__ int64_t slot_scales() const { return row_blocks() * groups * I4_ROWS; }
};

inline __host__ __device__ Int4Shape int4_shape(int64_t N, int64_t K, int64_t group, bool gated) {
  Int4Shape s;
  s.halves = gated ? 2 : 1;
  s.half_rows = N / s.halves;
  s.half_blocks = (s.half_rows + I4_ROWS - 1) / I4_ROWS;
  const int64_t steps = (K + I4_STEP - 1) / I4_STEP;
  s.k_blocks = steps * (I4_STEP / I4_K);
  s.groups = steps * (I4_STEP / group);
  return s;
}

// Where the scale of row r16 of a row block and group gr (of subs to a step)
// stands among the block's scales.
inline __host__ __device__ int64_t int4_scale_at(int r16, int64_t gr, int subs) {
  return gr / subs * (I4_ROWS * subs) + ((r16 & 7) * subs + (int)(gr % subs)) * 2 + (r16 >> 3);
}

// Sizes, group and dtype of a 4-bit weight that the kernels take.
inline bool int4_valid(int64_t N, int64_t K, int64_t group, bool gated) {
  return N > 0 && K > 0 && K % 8 == 0 && (N / (gated ? 2 : 1)) % 8 == 0 && (!gated || N % 2 == 0) &&
         (group == 32 || group == 64 || group == 128) && N < ((int64_t)1 << 30) && K < ((int64_t)1 << 30);
}

// The pair of codes (2 i, 2 i + 1) of a word as two 16-bit values code + B,
// exact, by placing the codes in the mantissas of B (published by Kim, Henry,
// Fahim and Awadalla, "Who Says Elephants Can't Run", 2022, with the order of the
// codes that it needs).  bf16: the last mantissa bits of 128.0, B = 128.  fp16:
// the first ones of 16.0, B = 16, a shift more: the last bits of 1024.0 made a
// product's terms 40 times as large, and an fp16 layer came out off by 0.00033,
// not 0.00029.
template <typename T> __device__ __forceinline__ uint32_t int4_raw(uint32_t word, int i) {
  constexpr bool HALF = std::is_same<T, __half>::value;
  constexpr int AT = HALF ? 6 : 0;  // the code's place in the mantissa
  constexpr uint32_t MASK = 0x000f000fu << AT, BASE = HALF ? 0x4c004c00u : 0x43004300u;
  const uint32_t w = 4 * i < AT ? word << (AT - 4 * i) : word >> (4 * i - AT);
  uint32_t r;  // (word & mask) | base; in C++ 7 tokens through eight experts of 4096 x 14336 took 178 us, so 144
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(w), "r"(MASK), "r"(BASE));
  return r;
}
// The same pair as code - 8, exact: B + 8 = 136 or 24 less.
template <typename T> __device__ __forceinline__ uint32_t int4_pair(uint32_t word, int i);
template <> __device__ __forceinline__ uint32_t int4_pair<__nv_bfloat16>(uint32_t word, int i) {
  const uint32_t b = int4_raw<__nv_bfloat16>(word, i);
  const __nv_bfloat162 off = __nv_bfloat162(__ushort_as_bfloat16(0x4308), __ushort_as_bfloat16(0x4308));
  const __nv_bfloat162 v = __hsub2(*reinterpret_cast<const __nv_bfloat162 *>(&b), off);
  return *reinterpret_cast<const uint32_t *>(&v);
}
template <> __device__ __forceinline__ uint32_t int4_pair<__half>(uint32_t word, int i) {
  const uint32_t b = int4_raw<__half>(word, i);
  const __half2 off = __half2(__ushort_as_half(0x4e00), __ushort_as_half(0x4e00));
  const __half2 v = __hsub2(*reinterpret_cast<const __half2 *>(&b), off);
  return *reinterpret_cast<const uint32_t *>(&v);
}

inline int current_device() {
  int dev = -1;
  return cudaGetDevice(&dev) == cudaSuccess ? dev : -1;
}

// One grouped product over all experts, rows in permuted order.
struct Int4Gemm {
  const void *a;                   // [rows, Kdim] in dtype
  const uint8_t *w;
  const void *scales;
  void *out;                       // gated: [rows, N] in dtype; down: [rows, N] fp32
  const int32_t *offsets, *counts; // [E+1], [E]
  int64_t rows;
  int E, Kdim, N;                  // N: output columns (I gated, H down)
  int group, dtype, act;
};

// On CTA pairs (int4_pair.cu).
int launch_int4_pair(const Int4Gemm &g, bool gated, cudaStream_t st);

}  // namespace rf
