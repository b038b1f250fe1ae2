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
// The order is that of the exact scores, not of their fp32 roundings:
//   * without a bias c is monotone in l, so experts (and groups by their
//     maximum) are compared by their logits, which are exact;
//   * otherwise c is computed in fp32 with a bound on its error, and a token
//     whose decision hangs on a gap within that bound is decided again in fp64
//     (route_exact: one token in some thousands, at its warp's expense alone).
// One warp per token: lane i holds the nv consecutive experts from i * nv, in
// registers, nv being a divisor of the group size wherever one fits, so that a
// group is a run of whole lanes: its score is a segmented shuffle reduction,
// and a choice is one redux.sync over order-preserving integer keys, the
// lowest lane with the largest key holding the lowest id.  (Sizes without such
// an nv, e.g. groups of 37, take the fp64 form for every token.)
#include <algorithm>

#include "router.cuh"

RF_DEVICE_ERROR_WORD();

namespace {

constexpr int GR_WARPS = 4;
constexpr int GR_THREADS = GR_WARPS * 32;
constexpr unsigned FULL = 0xffffffffu;
constexpr uint32_t KEY_NEG_INF = 0x007fffffu;  // order_key(-inf)
// Keys below it: 0 for a taken expert or a place past E, and KEY_MASKED for a
// NaN or a dropped group where logits are compared (there -inf stands for a
// score of 0, which comes before a masked one).  Where scores are compared
// NaN and dropped groups are -inf itself, like a closed expert.
constexpr uint32_t KEY_MASKED = 1u;

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

// nv consecutive logits from element e of row t (e a multiple of nv).
template <int NV, typename TX>
__device__ __forceinline__ void load_logits(const GroupedArgs &a, int64_t t, int e0, int nv, float (&l)[NV]) {
  constexpr int V = 16 / sizeof(TX);
  if constexpr (NV >= V) {
    // whole 16-byte vectors: uniform over the launch
    if (!a.partial && nv == NV && a.E % V == 0) {
      const TX *row = reinterpret_cast<const TX *>(a.x) + t * a.E + e0;
#pragma unroll
      for (int j = 0; j < NV; j += V) {
        if (e0 + j < a.E) rf::unpack16<TX>(__ldg(reinterpret_cast<const uint4 *>(row + j)), l + j);
      }
      if (a.round_dtype >= 0 || a.bias) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          if (e0 + j >= a.E) continue;
          if (a.round_dtype >= 0) l[j] = rf::round_dt(a.round_dtype, l[j]);
          if (a.bias) {
            l[j] += a.bias[e0 + j];
            if (a.round_dtype >= 0) l[j] = rf::round_dt(a.round_dtype, l[j]);
          }
        }
      }
      return;
    }
  }
#pragma unroll
  for (int j = 0; j < NV; ++j)
    if (j < nv && e0 + j < a.E) l[j] = logit_of<TX>(a, t, e0 + j);
}

template <int NV, typename TX>
__global__ void __launch_bounds__(GR_THREADS) router_grouped_kernel(const GroupedArgs a) {
  extern __shared__ double s_exact[];  // [GR_WARPS][E], for route_exact
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int nv = a.nv;
  const int e0 = lane * nv;
  const bool by_score = a.select_bias != nullptr;  // else experts are compared by their logits
  const bool group_by_score = by_score || a.top2;
  const uint32_t low = by_score ? KEY_NEG_INF : KEY_MASKED;
  for (int64_t t = (int64_t)blockIdx.x * GR_WARPS + warp; t < a.T; t += (int64_t)gridDim.x * GR_WARPS) {
    if (a.has_shared && lane == 0) {
      const float z = rf::sum_slices(a.partial + t * a.ld + a.E, a.T * a.ld, a.slices);
      a.shared_scale[t] = 1.0f / (1.0f + expf(-z));
    }
    if (a.logits_out)
      for (int e = lane; e < a.E; e += 32) a.logits_out[t * a.E + e] = logit_of<TX>(a, t, e);
    int my_id = 0;
    float my_s = 0.f;
    bool exact = nv == 0;
    if (!exact) {
      // ---- scores
      float l[NV], s[NV];
      uint32_t key[NV];
#pragma unroll
      for (int j = 0; j < NV; ++j) l[j] = -INFINITY;
      load_logits<NV, TX>(a, t, e0, nv, l);
      float eps, smax;  // relative error of a score (see below), an upper bound of the scores
      bool row_nan = false;
      if (a.sigmoid) {
        smax = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          s[j] = 1.0f / (1.0f + expf(-l[j]));
          smax = fmaxf(smax, s[j]);
        }
        // expf within 2 ulp, one addition, one division
        eps = 6.0f * 0x1p-24f;
      } else {
        float m = l[0];
#pragma unroll
        for (int j = 1; j < NV; ++j) m = fmaxf(m, l[j]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(FULL, m, o));
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          s[j] = j < nv && e0 + j < a.E ? expf(l[j] - m) : 0.f;
          sum += s[j];
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(FULL, sum, o);
        row_nan = !(sum == sum);
        smax = 1.0f / sum;
#pragma unroll
        for (int j = 0; j < NV; ++j) s[j] = s[j] / sum;
        // expf within 2 ulp (its argument's own rounding is worth less than
        // one more: x e^-x < 0.37), NV + 5 additions, one division
        eps = (NV + 5 + 8) * 0x1p-24f;
      }
      // ---- what experts are compared by
      float cabs = 0.f;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int e = e0 + j;
        float c = l[j];
        if (by_score && j < nv && e < a.E) c = s[j] + a.select_bias[e];
        if (fabsf(c) < INFINITY) cabs = fmaxf(cabs, fabsf(c));
        key[j] = j < nv && e < a.E ? (row_nan ? low : order_key(c, low)) : 0u;
      }
      // Two fp32 scores closer than tol may be in the other order exactly:
      // each is off by at most eps * smax + 2^-24 * |c|.
      float tol = -1.f, gtol = -1.f;
      if (group_by_score) {
        smax = __uint_as_float(__reduce_max_sync(FULL, __float_as_uint(fmaxf(smax, 0.f))));
        cabs = __uint_as_float(__reduce_max_sync(FULL, __float_as_uint(by_score ? cabs : smax)));
        const float one = eps * smax + 0x1p-24f * cabs;
        if (by_score) tol = 2.f * one;
        gtol = a.top2 ? 4.f * one + 0x1p-22f * cabs : 2.f * one;
      }
      // ---- groups: runs of `lanes` lanes
      if (a.G > 1) {
        const int lanes = a.per / nv;
        uint32_t k1 = 0u;       // by maximum, as keys
        float c1 = -INFINITY, c2 = -INFINITY;  // by the two largest
        if (!a.top2) {
#pragma unroll
          for (int j = 0; j < NV; ++j) k1 = max(k1, key[j]);
        } else {
#pragma unroll
          for (int j = 0; j < NV; ++j) {
            const float c = key[j] > low ? (by_score ? key_value(key[j]) : s[j]) : -INFINITY;
            c2 = fmaxf(c2, fminf(c1, c));
            c1 = fmaxf(c1, c);
          }
        }
        // after step o a lane covers itself and the min(2 o, rest) - 1 lanes
        // above it inside its group; the group's first lane ends with all
        const int pos = lane % lanes;
        for (int o = 1; o < lanes; o <<= 1) {
          const uint32_t ok = __shfl_down_sync(FULL, k1, o);
          const float o1 = __shfl_down_sync(FULL, c1, o), o2 = __shfl_down_sync(FULL, c2, o);
          if (pos + o < lanes && lane + o < 32) {
            k1 = max(k1, ok);
            c2 = fmaxf(fmaxf(c2, o2), fminf(c1, o1));
            c1 = fmaxf(c1, o1);
          }
        }
        // lane g takes group g's score
        const int src = min(lane * lanes, 31);
        k1 = __shfl_sync(FULL, k1, src);
        c1 = __shfl_sync(FULL, c1, src);
        c2 = __shfl_sync(FULL, c2, src);
        const uint32_t gk = a.top2 ? order_key(c1 + c2, KEY_NEG_INF) : k1;
        int before = 0;
        for (int g = 0; g < a.G; ++g) {
          const uint32_t o = __shfl_sync(FULL, gk, g);
          before += (o > gk || (o == gk && g < lane)) ? 1 : 0;
        }
        const bool stays = lane < a.G && before < a.keep;
        const unsigned kept = __ballot_sync(FULL, stays);
        if (group_by_score && a.keep < a.G) {
          const uint32_t in = __reduce_min_sync(FULL, stays ? gk : 0xffffffffu);
          const uint32_t out = __reduce_max_sync(FULL, !stays && lane < a.G ? gk : 0u);
          if (out > KEY_NEG_INF && key_value(in) - key_value(out) <= gtol) exact = true;
        }
        if (!(kept >> min(lane / lanes, 31) & 1u)) {
#pragma unroll
          for (int j = 0; j < NV; ++j) key[j] = min(key[j], low);
        }
      }
      // ---- K choices, and one more that only shows its distance
      uint32_t mine = 0u, last = 0u;
#pragma unroll
      for (int j = 0; j < NV; ++j) mine = max(mine, key[j]);
      const int rounds = by_score ? min(a.K + 1, a.E) : a.K;
      for (int k = 0; k < rounds && !exact; ++k) {
        const uint32_t best = __reduce_max_sync(FULL, mine);
        if (by_score) {
          if (k > 0 && best > KEY_NEG_INF && key_value(last) - key_value(best) <= tol) exact = true;
          last = best;
          if (k == a.K) break;
        }
        const int owner = __ffs(__ballot_sync(FULL, mine == best)) - 1;
        int at = 0;
        float sv = 0.f;
        if (lane == owner) {
          mine = 0u;
          bool found = false;
#pragma unroll
          for (int j = 0; j < NV; ++j) {
            if (!found && key[j] == best) {
              found = true;
              at = e0 + j;
              sv = s[j];
              key[j] = 0u;
            }
            mine = max(mine, key[j]);
          }
        }
        at = __shfl_sync(FULL, at, owner);
        sv = __shfl_sync(FULL, sv, owner);
        if (lane == k) {
          my_id = at;
          my_s = sv;
        }
      }
    }
    if (exact) route_exact<TX>(a, t, s_exact + warp * a.E, &my_id, &my_s);
    // ---- weights
    float w = my_s;
    if (a.renormalize) {
      float sum = 0.f;
      for (int k = 0; k < a.K; ++k) sum += __shfl_sync(FULL, my_s, k);
      w = my_s / (sum < 1e-20f ? 1e-20f : sum);
    }
    if (lane < a.K) {
      a.topk_w[t * a.K + lane] = w * a.scale;
      if (a.ids32) a.ids32[t * a.K + lane] = my_id;
      if (a.ids64) a.ids64[t * a.K + lane] = my_id;
    }
  }
}

template <int NV, typename TX>
int launch_nv(const GroupedArgs &a, cudaStream_t st) {
  const int64_t blocks = std::min<int64_t>((a.T + GR_WARPS - 1) / GR_WARPS, (int64_t)rf::num_sms() * 16);
  // fp64 scratch only where a token can need it: 32 KB at most (E <= 1024)
  const bool may_be_exact = a.nv == 0 || a.select_bias || (a.top2 && a.G > 1);
  const size_t smem = may_be_exact ? (size_t)GR_WARPS * a.E * sizeof(double) : 0;
  router_grouped_kernel<NV, TX><<<(int)blocks, GR_THREADS, smem, st>>>(a);
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
  RF_CHECK_ARG(T >= 0 && H > 0 && E > 0, "rf_moe_router_grouped_topk: sizes must be positive");
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
