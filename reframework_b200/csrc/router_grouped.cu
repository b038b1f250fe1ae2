// Grouped routing: softmax or sigmoid scores, a selection bias, expert groups,
// top-k, renormalised and scaled weights.
//
// Per token with logits l[0..E) (from router_logits, or given):
//   s = softmax(l) or sigmoid(l)
//   c = s + b            b: selection bias (load balance), never in the weights;
//                        b[e] = -inf closes an expert
//   score of a group of E/G consecutive experts = max c, or the sum of its two
//   largest c; the topk_groups best groups stay (ties: the lower group) and the
//   others' c becomes -inf
//   ids = the K largest c, in that order (ties: the lower id; a NaN c counts as
//   -inf); w = s[ids], divided by max(sum w, 1e-20) when renormalising, * scale
//
// The order is that of the exact scores, not of their fp32 roundings: experts
// are picked by fp32 values with a bound on their error, and where a decision
// hangs on a gap within that bound the candidates are put in order by their
// fp64 scores (without a bias c is monotone in l, so logits are compared then).
// The weights are computed again from the chosen logits, with expf.  A softmax
// score is then divided by the sum over all experts, which is one of __expf.  A
// term e^-d of it, d = m - l, is off by (2 + 1.173 d + d / 2) * 2^-23 of itself,
// and the mean of d over a softmax is at most ln E, so the sum is off by at most
// (27.2 + NV + 5) * 2^-24 of itself (E = 1024; NV + 5 additions).  A score is that
// and d + 5 roundings off; renormalised, the sum cancels and d + 5 twice stay.
//
// One warp per token: lane i holds the nv consecutive experts from i * nv as
// order-preserving integer keys, sorted, nv being a divisor of the group size
// wherever one fits, so that a group is a run of whole lanes and its score a
// segmented shuffle reduction over the lanes' first keys.  A pick is one
// redux.sync over the lanes' first keys and a shift in the lane that had it.
// The place within a lane is kept in a key's low bits (part of the error
// bound).  Sizes without such an nv, e.g. groups of 37, take an fp64 form.
// Bound by latency: a chain of dependent reductions per pick, 6.8 warps a
// scheduler (64 registers: 8 blocks an SM, 1.73 waves of 8192 tokens), issue slots
// 46 % busy.  256 experts, K = 8, 8 groups: 1263 instructions a token, of which 8
// sigmoids a lane, a sort of 8 and 13 picks or reductions; 8192 tokens take 18 us
// (their bytes alone 1.4), one of 64 experts 3.8, nearly all of it the launch.
#include "router.cuh"

namespace {

constexpr int GR_WARPS = 4;
constexpr int GR_THREADS = GR_WARPS * 32;
constexpr unsigned FULL = 0xffffffffu;
constexpr uint32_t KEY_NEG_INF = 0x007fffffu;  // order_key(-inf)
// Keys below it: 0 for a taken expert or a place past E, and KEY_MASKED for a
// NaN or a dropped group where logits are compared (there -inf stands for a
// score of 0, which comes before a masked one).  Where scores are compared
// NaN and dropped groups are -inf itself, like a closed expert.  (64: above the
// place bits.)
constexpr uint32_t KEY_MASKED = 64u;

struct GroupedArgs {
  const void *x;         // logits [T, E] when partial is NULL
  const float *partial;  // [slices][T][ld]
  int slices;
  int64_t ld;
  const float *bias;         // added to the logits
  const float *select_bias;  // added to the scores, for the selection
  float *shared_scale;
  float *topk_w;
  int32_t *ids32;
  int64_t *ids64;
  float *logits_out;
  int64_t T;
  int E, K, G, keep, per;  // per = E / G
  int nv;                  // experts per lane (0: every token in fp64)
  int sigmoid, top2, renormalize, round_dtype, has_shared;
  float scale;
};

// Unsigned integers in the order of the floats, -0 as 0; `low` for NaN.
__device__ __forceinline__ uint32_t order_key(float c, uint32_t low) {
  if (!(c == c)) return low;
  const uint32_t u = __float_as_uint(c + 0.0f);
  return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k ^ ((k & 0x80000000u) ? 0x80000000u : 0xffffffffu));
}

template <typename TX>
__device__ __forceinline__ float logit_of(const GroupedArgs &a, int64_t t, int e) {
  float v = a.partial ? rf::sum_slices(a.partial + t * a.ld + e, a.T * a.ld, a.slices)
                      : rf::Cvt<TX>::to_f(reinterpret_cast<const TX *>(a.x)[t * a.E + e]);
  if (a.round_dtype >= 0) v = rf::round_dt(a.round_dtype, v);
  if (a.bias) {
    v += a.bias[e];
    if (a.round_dtype >= 0) v = rf::round_dt(a.round_dtype, v);
  }
  return v;
}

__device__ __forceinline__ double warp_max(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmax(v, __shfl_xor_sync(FULL, v, o));
  return v;
}

// The whole selection of one token in fp64; sc is this warp's [E] scratch.
// Lane k gets choice k and its score.
template <typename TX>
__device__ __noinline__ void route_exact(const GroupedArgs &a, int64_t t, double *sc, int *my_id, float *my_s) {
  const int lane = threadIdx.x & 31;
  const double ninf = -(double)INFINITY;
  double m = ninf, sum = 1.0;
  __syncwarp();
  if (!a.sigmoid) {
    for (int e = lane; e < a.E; e += 32) m = fmax(m, (double)logit_of<TX>(a, t, e));
    m = warp_max(m);
    sum = 0.0;
    for (int e = lane; e < a.E; e += 32) sum += exp((double)logit_of<TX>(a, t, e) - m);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(FULL, sum, o);
  }
  auto score_of = [&](double l) -> double { return a.sigmoid ? 1.0 / (1.0 + exp(-l)) : exp(l - m) / sum; };
  // with a bias the scores are compared, without one the logits (the same
  // order; a logit of -inf still comes before what is masked)
  const double least = -1e300;
  for (int e = lane; e < a.E; e += 32) {
    const double l = logit_of<TX>(a, t, e);
    const double c = a.select_bias ? score_of(l) + (double)a.select_bias[e] : l > least ? l : least;
    sc[e] = c == c && l == l && sum == sum ? c : ninf;
  }
  __syncwarp();
  if (a.G > 1) {
    double gs = ninf;
    if (lane < a.G) {
      double c1 = ninf, c2 = ninf;
      for (int i = 0; i < a.per; ++i) {
        const double c = sc[lane * a.per + i];
        c2 = fmax(c2, fmin(c1, c));
        c1 = fmax(c1, c);
      }
      gs = c1;
      if (a.top2) {
        if (!a.select_bias) {
          c1 = c1 > ninf ? score_of(c1) : ninf;
          c2 = c2 > ninf ? score_of(c2) : ninf;
        }
        gs = c1 + c2;
      }
      if (!(gs == gs)) gs = ninf;
    }
    int before = 0;
    for (int g = 0; g < a.G; ++g) {
      const double o = __shfl_sync(FULL, gs, g);
      before += (o > gs || (o == gs && g < lane)) ? 1 : 0;
    }
    const unsigned kept = __ballot_sync(FULL, lane < a.G && before < a.keep);
    for (int e = lane; e < a.E; e += 32)
      if (!(kept >> (e / a.per) & 1u)) sc[e] = ninf;
    __syncwarp();
  }
  int id = 0;
  for (int k = 0; k < a.K; ++k) {  // a taken expert becomes NaN, which no comparison prefers
    double best = ninf;
    int bi = 0x7fffffff;
    for (int e = lane; e < a.E; e += 32) {
      const double c = sc[e];
      if (c > best || (c == best && e < bi)) {
        best = c;
        bi = e;
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const double ob = __shfl_xor_sync(FULL, best, o);
      const int oi = __shfl_xor_sync(FULL, bi, o);
      if (ob > best || (ob == best && oi < bi)) {
        best = ob;
        bi = oi;
      }
    }
    if (lane == k) id = bi;
    __syncwarp();
    if (lane == 0) sc[bi] = (double)NAN;
    __syncwarp();
  }
  *my_id = id;
  *my_s = lane < a.K ? (float)score_of((double)logit_of<TX>(a, t, id)) : 0.f;
}

// Descending, NV a power of two (bitonic: every comparison a min and a max).
template <int NV>
__device__ __forceinline__ void sort_keys(uint32_t (&k)[NV]) {
#pragma unroll
  for (int size = 2; size <= NV; size <<= 1)
#pragma unroll
    for (int d = size >> 1; d > 0; d >>= 1)
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int j = i ^ d;
        if (j > i) {
          const uint32_t hi = max(k[i], k[j]), lo = min(k[i], k[j]);
          const bool down = (i & size) == 0;
          k[i] = down ? hi : lo;
          k[j] = down ? lo : hi;
        }
      }
}

// A score to within 7 * 2^-24 (sigmoid): __expf is off by (2 + 1.173 |l|) ulp,
// of which the score sees s (1 - s), at most 0.77 ulp of 1 in all; the quotient
// adds 2 and the sum half an ulp.
__device__ __forceinline__ float fast_sigmoid(float l) { return __fdividef(1.0f, 1.0f + __expf(-l)); }

// n candidates, one per lane (the first n_open of them neither masked nor
// closed), in the order of their exact values; returns the id of this lane's place.
template <typename TX>
__device__ __noinline__ int settle(const GroupedArgs &a, int64_t t, int id, int n, int n_open, float m) {
  const int lane = threadIdx.x & 31;
  const double ninf = -(double)INFINITY;
  double v = lane < n ? (double)logit_of<TX>(a, t, id) : 0.0;
  if (a.select_bias) {
    double total = 1.0;
    if (!a.sigmoid) {
      total = 0.0;
      for (int e = lane; e < a.E; e += 32) total += exp((double)logit_of<TX>(a, t, e) - (double)m);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(FULL, total, o);
    }
    v = (a.sigmoid ? 1.0 / (1.0 + exp(-v)) : exp(v - (double)m) / total) + (lane < n ? (double)a.select_bias[id] : 0.0);
  }
  v = lane >= n_open ? ninf : a.select_bias ? v : fmax(v, -1e300);  // a logit of -inf comes before what is masked
  int rank = 0;
  for (int j = 0; j < n; ++j) {
    const double o = __shfl_sync(FULL, v, j);
    const int oi = __shfl_sync(FULL, id, j);
    rank += (o > v || (o == v && oi < id)) ? 1 : 0;
  }
  int mine = 0;
  for (int j = 0; j < n; ++j) {
    const int r = __shfl_sync(FULL, rank, j), oi = __shfl_sync(FULL, id, j);
    if (lane == r) mine = oi;
  }
  return mine;
}

// WHOLE: every lane's nv experts are NV or none (nv == NV, E a multiple of NV),
// read as 16-byte vectors where the type has that many.
template <int NV, typename TX, bool WHOLE>
__global__ void __launch_bounds__(GR_THREADS) router_grouped_kernel(const GroupedArgs a) {
  extern __shared__ double s_exact[];  // [GR_WARPS][E], for route_exact
  constexpr uint32_t PLACE = NV - 1;   // the low bits of a key: NV - 1 - place in the lane
  constexpr int V = 16 / sizeof(TX);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int nv = WHOLE ? NV : a.nv;
  const int e0 = lane * nv;
  const bool by_score = a.select_bias != nullptr;  // else experts are compared by their logits
  const uint32_t low = (by_score ? KEY_NEG_INF : KEY_MASKED) & ~PLACE;
  const int64_t t = (int64_t)blockIdx.x * GR_WARPS + warp;
  if (t >= a.T) return;
  if (a.has_shared && lane == 0) {
    const float z = rf::sum_slices(a.partial + t * a.ld + a.E, a.T * a.ld, a.slices);
    a.shared_scale[t] = 1.0f / (1.0f + expf(-z));
  }
  if (a.logits_out)
    for (int e = lane; e < a.E; e += 32) a.logits_out[t * a.E + e] = logit_of<TX>(a, t, e);
  auto inside = [&](int j) { return WHOLE ? e0 < a.E : j < nv && e0 + j < a.E; };
  int my_id = 0;
  float my_s = 0.f;
  bool exact = a.nv == 0;  // every decision of this token in fp64
  float m = 0.f, sum = 1.f;  // softmax: the largest logit, the sum
  if (!exact) {
    float l[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) l[j] = -INFINITY;
    if (WHOLE && NV >= V && !a.partial) {
      if (e0 < a.E) {
        const TX *row = reinterpret_cast<const TX *>(a.x) + t * a.E + e0;
#pragma unroll
        for (int j = 0; j + V <= NV; j += V) rf::unpack16<TX>(__ldg(reinterpret_cast<const uint4 *>(row + j)), l + j);
        if (a.round_dtype >= 0 || a.bias) {
#pragma unroll
          for (int j = 0; j < NV; ++j) {
            if (a.round_dtype >= 0) l[j] = rf::round_dt(a.round_dtype, l[j]);
            if (a.bias) {
              l[j] += a.bias[e0 + j];
              if (a.round_dtype >= 0) l[j] = rf::round_dt(a.round_dtype, l[j]);
            }
          }
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (inside(j)) l[j] = logit_of<TX>(a, t, e0 + j);
    }
    bool row_nan = false;
    if (!a.sigmoid) {
      m = l[0];
#pragma unroll
      for (int j = 1; j < NV; ++j) m = fmaxf(m, l[j]);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(FULL, m, o));
      sum = 0.f;
#pragma unroll
      for (int j = 0; j < NV; ++j) sum += inside(j) ? __expf(l[j] - m) : 0.f;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(FULL, sum, o);
      row_nan = !(sum == sum);
    }
    // Errors: of a score, absolute (softmax: __expf within 2 + 1.173 |l - m| ulp
    // and its argument's rounding, worth 3 ulp of the largest score; the sum's,
    // with |l - m| at most 8 on average, and its NV + 5 additions; a product);
    // of a key, relative to its value (a rounding, and the place bits).
    const float inv = 1.0f / sum;
    const float eps = a.sigmoid ? 7.f * 0x1p-24f : (NV + 48) * 0x1p-24f * inv;
    constexpr float KEY_EPS = (NV > 1 ? 2 * NV : 1) * 0x1p-24f;
    // 16-bit logits have no bits where the place goes: their keys are exact
    const bool exact_keys = !by_score && (NV == 1 || (sizeof(TX) == 2 && !a.bias));
    // Two values no further apart than this may be in the other order exactly.
    const float tol0 = by_score ? 2.f * eps : 0.f, tol1 = exact_keys ? 0.f : 2.f * KEY_EPS;
    auto tolerance = [&](float u, float v) { return fmaf(tol1, fmaxf(fabsf(u), fabsf(v)), tol0); };
    // ---- keys
    if (by_score) {
      float sb[NV];
#pragma unroll
      for (int j = 0; j < NV; ++j) sb[j] = 0.f;
      if (WHOLE && NV >= 4 && ((uintptr_t)a.select_bias & 15) == 0) {
        if (e0 < a.E) {
#pragma unroll
          for (int j = 0; j + 4 <= NV; j += 4)
            rf::unpack16<float>(__ldg(reinterpret_cast<const uint4 *>(a.select_bias + e0 + j)), sb + j);
        }
      } else {
#pragma unroll
        for (int j = 0; j < NV; ++j)
          if (inside(j)) sb[j] = a.select_bias[e0 + j];
      }
#pragma unroll
      for (int j = 0; j < NV; ++j)  // a place past the lane's experts stays -inf: a group's top-2 sum sees all NV
        if (inside(j)) l[j] = (a.sigmoid ? fast_sigmoid(l[j]) : __expf(l[j] - m) * inv) + sb[j];
    }
    uint32_t key[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) key[j] = inside(j) ? (order_key(l[j], low) & ~PLACE) | (PLACE - j) : 0u;
    if (row_nan) {
#pragma unroll
      for (int j = 0; j < NV; ++j) key[j] = inside(j) ? low | (PLACE - j) : 0u;
    }
    sort_keys<NV>(key);
    // ---- groups: runs of `lanes` lanes, scored by their first keys
    if (a.G > 1) {
      const int lanes = a.per / nv;
      const int pos = lane % lanes;
      uint32_t gk;
      float gtol = 0.f;  // top-2 scores
      if (!a.top2) {
        uint32_t k1 = key[0] & ~PLACE;
        // after step o a lane covers itself and the min(2 o, rest) - 1 lanes
        // above it inside its group; the group's first lane ends with all
        for (int o = 1; o < lanes; o <<= 1) {
          const uint32_t up = __shfl_down_sync(FULL, k1, o);
          if (pos + o < lanes) k1 = max(k1, up);
        }
        gk = __shfl_sync(FULL, k1, min(lane * lanes, 31));  // lane g takes group g's score
      } else {
        // l holds the selection scores, or the logits, whose two largest give the scores
        float c1 = -INFINITY, c2 = -INFINITY;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          const float c = l[j] == l[j] && !row_nan ? l[j] : -INFINITY;
          c2 = fmaxf(c2, fminf(c1, c));
          c1 = fmaxf(c1, c);
        }
        if (!by_score) {  // past the lane's own experts, and for NaN: -inf, a logit of -inf: 0
          c1 = key[0] >= low + NV ? a.sigmoid ? fast_sigmoid(c1) : __expf(c1 - m) * inv : -INFINITY;
          c2 = NV > 1 && key[NV > 1 ? 1 : 0] >= low + NV ? a.sigmoid ? fast_sigmoid(c2) : __expf(c2 - m) * inv : -INFINITY;
        }
        for (int o = 1; o < lanes; o <<= 1) {
          const float o1 = __shfl_down_sync(FULL, c1, o), o2 = __shfl_down_sync(FULL, c2, o);
          if (pos + o < lanes) {
            c2 = fmaxf(fmaxf(c2, o2), fminf(c1, o1));
            c1 = fmaxf(c1, o1);
          }
        }
        const int src = min(lane * lanes, 31);
        c1 = __shfl_sync(FULL, c1, src);
        c2 = __shfl_sync(FULL, c2, src);
        gk = order_key(c1 + c2, KEY_NEG_INF);
        // twice a score's error for each of two sums, and roundings of values up to big
        float big = fabsf(c1) < INFINITY ? fabsf(c1) : 0.f;
        if (fabsf(c2) < INFINITY) big = fmaxf(big, fabsf(c2));
        big = __uint_as_float(__reduce_max_sync(FULL, __float_as_uint(lane < a.G ? big : 0.f)));
        gtol = 4.f * eps + 0x1p-21f * big;
      }
      int before = 0;
      for (int g = 0; g < a.G; ++g) {
        const uint32_t o = __shfl_sync(FULL, gk, g);
        before += (o > gk || (o == gk && g < lane)) ? 1 : 0;
      }
      const bool stays = lane < a.G && before < a.keep;
      const unsigned kept = __ballot_sync(FULL, stays);
      if (a.keep < a.G && !(exact_keys && !a.top2)) {
        const uint32_t in = __reduce_min_sync(FULL, stays ? gk : 0xffffffffu);
        const uint32_t out = __reduce_max_sync(FULL, !stays && lane < a.G ? gk : 0u);
        const float vi = key_value(in), vo = key_value(out);
        if (out > KEY_NEG_INF && vi - vo <= (a.top2 ? gtol : tolerance(vi, vo))) exact = true;
      }
      if (!(kept >> min(lane / lanes, 31) & 1u)) {
#pragma unroll
        for (int j = 0; j < NV; ++j) key[j] = inside(j) ? low | (PLACE - j) : 0u;
      }
    }
    // ---- K picks, and on to the first gap that is certain
    int n = 0, n_open = 0;
    bool unsure = false;
    float last = INFINITY;
    while (!exact) {
      const uint32_t mine = key[0] & ~PLACE;
      const uint32_t best = __reduce_max_sync(FULL, mine);
      const float v = key_value(best);
      // (the first gap is infinite, one down to a masked or closed expert NaN or infinite)
      const bool close = !exact_keys && last - v <= tolerance(last, v) && n > 0 && best > KEY_NEG_INF;
      if (n >= a.K && (!close || n == 32)) {
        exact = close;  // more than a warp of candidates in a row
        break;
      }
      const unsigned holders = __ballot_sync(FULL, mine == best && key[0] != 0u);
      if (holders == 0u) break;  // every expert is picked
      unsure |= close;
      last = v;
      n_open += best > low ? 1 : 0;
      const int owner = __ffs(holders) - 1;
      const int at = owner * nv + (int)(~__shfl_sync(FULL, key[0], owner) & PLACE);
      if (lane == n) my_id = at;
      const bool pop = lane == owner;
#pragma unroll
      for (int j = 0; j + 1 < NV; ++j) key[j] = pop ? key[j + 1] : key[j];
      key[NV - 1] = pop ? 0u : key[NV - 1];
      ++n;
    }
    if (unsure && !exact) my_id = settle<TX>(a, t, my_id, n, n_open, m);
    if (!exact && lane < a.K) {  // the scores of the chosen, from their logits
      const float lc = logit_of<TX>(a, t, my_id);
      my_s = a.sigmoid ? 1.0f / (1.0f + expf(-lc)) : expf(lc - m) / sum;
    }
  }
  if (exact) route_exact<TX>(a, t, s_exact + warp * a.E, &my_id, &my_s);
  // ---- weights
  if (lane >= a.K) my_s = 0.f;
  float w = my_s;
  if (a.renormalize) {
    float total = my_s;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) total += __shfl_xor_sync(FULL, total, o);  // K <= 16
    w = my_s / (total < 1e-20f ? 1e-20f : total);
  }
  if (lane < a.K) {
    a.topk_w[t * a.K + lane] = w * a.scale;
    if (a.ids32) a.ids32[t * a.K + lane] = my_id;
    if (a.ids64) a.ids64[t * a.K + lane] = my_id;
  }
}

template <int NV, typename TX>
int launch_nv(const GroupedArgs &a, cudaStream_t st) {
  const int64_t blocks = (a.T + GR_WARPS - 1) / GR_WARPS;
  // fp64 scratch: 32 KB at most (E <= 1024)
  const size_t smem = (size_t)GR_WARPS * a.E * sizeof(double);
  if (a.nv == NV && a.E % NV == 0) router_grouped_kernel<NV, TX, true><<<(unsigned)blocks, GR_THREADS, smem, st>>>(a);
  else router_grouped_kernel<NV, TX, false><<<(unsigned)blocks, GR_THREADS, smem, st>>>(a);
  return rf::check_launch("rf_moe_router_grouped_topk(selection)");
}

template <typename TX>
int launch_tx(const GroupedArgs &a, cudaStream_t st) {
  if (a.nv <= 1) return launch_nv<1, TX>(a, st);
  if (a.nv == 2) return launch_nv<2, TX>(a, st);
  if (a.nv <= 4) return launch_nv<4, TX>(a, st);
  if (a.nv <= 8) return launch_nv<8, TX>(a, st);
  if (a.nv <= 16) return launch_nv<16, TX>(a, st);
  return launch_nv<32, TX>(a, st);
}

// Experts per lane: at least ceil(E / 32) and, with groups, a divisor of the
// group size, so that groups are whole lanes; 0 if there is none up to 32.
int experts_per_lane(int E, int per, int G) {
  int nv = (E + 31) / 32;
  if (G > 1)
    while (nv <= 32 && per % nv != 0) ++nv;
  return nv <= 32 ? nv : 0;
}

}  // namespace

extern "C" int rf_moe_router_grouped_topk(const void *x, int x_dtype, const void *gate, int gate_dtype,
                                          const float *bias, int64_t T, int64_t H, int64_t E, int64_t K,
                                          int scoring, const float *select_bias, int64_t num_groups,
                                          int64_t topk_groups, int group_score, int renormalize, float scale,
                                          int round_dtype, const void *shared_gate, float *shared_scale,
                                          float *topk_weights, int32_t *topk_ids32, int64_t *topk_ids64,
                                          float *logits, void *workspace, size_t workspace_bytes,
                                          rf_stream_t stream) {
  RF_CHECK_ARG(rf::valid_dtype(x_dtype) && rf::valid_dtype(gate_dtype),
               "rf_moe_router_grouped_topk: unknown dtype");
  RF_CHECK_ARG(round_dtype < 0 || rf::valid_dtype(round_dtype), "rf_moe_router_grouped_topk: bad round_dtype");
  RF_CHECK_ARG(scoring == RF_SCORE_SOFTMAX || scoring == RF_SCORE_SIGMOID,
               "rf_moe_router_grouped_topk: unknown scoring");
  RF_CHECK_ARG(group_score == RF_GROUP_MAX || group_score == RF_GROUP_TOP2,
               "rf_moe_router_grouped_topk: unknown group_score");
  RF_CHECK_ARG(T >= 0 && T <= 0x7fffffff && H > 0 && E > 0, "rf_moe_router_grouped_topk: sizes must be positive");
  RF_CHECK_ARG(E <= rf::ROUTER_EMAX, "rf_moe_router_grouped_topk: at most 1024 experts");
  RF_CHECK_ARG(num_groups >= 1 && num_groups <= 32 && E % num_groups == 0,
               "rf_moe_router_grouped_topk: num_groups must be 1..32 and divide the experts");
  RF_CHECK_ARG(topk_groups >= 1 && topk_groups <= num_groups,
               "rf_moe_router_grouped_topk: need 1 <= topk_groups <= num_groups");
  RF_CHECK_ARG(num_groups == 1 || group_score == RF_GROUP_MAX || E / num_groups >= 2,
               "rf_moe_router_grouped_topk: a top-2 group score needs two experts in a group");
  RF_CHECK_ARG(K >= 1 && K <= rf::ROUTER_KMAX && K <= topk_groups * (E / num_groups),
               "rf_moe_router_grouped_topk: need 1 <= K <= min(16, experts in the kept groups)");
  RF_CHECK_ARG(scale == scale && scale - scale == 0.f, "rf_moe_router_grouped_topk: scale must be finite");
  RF_CHECK_ARG(!gate || H % 8 == 0, "rf_moe_router_grouped_topk: hidden size must be a multiple of 8");
  RF_CHECK_ARG(gate || (H == E && !shared_gate),
               "rf_moe_router_grouped_topk: without a gate, x holds the [T,E] logits (H == E)");
  RF_CHECK_ARG(T == 0 || (topk_weights && (topk_ids32 || topk_ids64)),
               "rf_moe_router_grouped_topk: missing outputs");
  RF_CHECK_ARG(T == 0 || x, "rf_moe_router_grouped_topk: null input");
  RF_CHECK_ARG(T == 0 || !shared_gate || shared_scale,
               "rf_moe_router_grouped_topk: shared_gate needs shared_scale");
  RF_CHECK_ARG((uintptr_t)x % 16 == 0 && (uintptr_t)gate % 16 == 0 && (uintptr_t)shared_gate % 16 == 0,
               "rf_moe_router_grouped_topk: x / gate must be 16-byte aligned");
  if (T == 0) return RF_OK;
  cudaStream_t st = (cudaStream_t)stream;
  GroupedArgs a;
  a.x = x;
  a.partial = nullptr;
  a.slices = 1;
  a.ld = E;
  a.bias = bias;
  a.select_bias = select_bias;
  a.shared_scale = shared_scale;
  a.topk_w = topk_weights;
  a.ids32 = topk_ids32;
  a.ids64 = topk_ids64;
  a.logits_out = logits;
  a.T = T;
  a.E = (int)E;
  a.K = (int)K;
  a.G = (int)num_groups;
  a.keep = (int)topk_groups;
  a.per = (int)(E / num_groups);
  a.nv = experts_per_lane(a.E, a.per, a.G);
  a.sigmoid = scoring == RF_SCORE_SIGMOID;
  a.top2 = group_score == RF_GROUP_TOP2 && num_groups > 1;
  a.renormalize = renormalize;
  a.round_dtype = round_dtype;
  a.has_shared = shared_gate ? 1 : 0;
  a.scale = scale;
  if (gate) {
    rf::RouterLogits lg;
    const int rc = rf::router_logits("rf_moe_router_grouped_topk", x, x_dtype, gate, gate_dtype, shared_gate, T, H, E,
                                     workspace, workspace_bytes, st, &lg);
    if (rc) return rc;
    a.partial = lg.partial;
    a.slices = lg.slices;
    a.ld = lg.ld;
    return launch_tx<float>(a, st);
  }
  switch (x_dtype) {
    case RF_F32: return launch_tx<float>(a, st);
    case RF_F16: return launch_tx<__half>(a, st);
    default: return launch_tx<__nv_bfloat16>(a, st);
  }
}
