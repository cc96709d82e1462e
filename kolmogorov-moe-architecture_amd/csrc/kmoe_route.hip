// Routing of logits to experts, and its backward.
//   score   s_e = softmax(l)_e or sigmoid(l_e)       (a logit of -inf masks its expert: s 0)
//   choice  c_e = s_e + b_e, -inf for a masked expert; NaN ranks above everything
//   groups  G equal runs of experts; a group's value is the sum of its best one or two
//           unmasked choices (-inf without any), the best `topk_groups` groups stay
//   idx     the k largest c among the experts of those groups, equal c lowest index first
//   weight  w_j = a s_j / (sum_i s_i + 1e-20) over the chosen i, or a s_j
// The bias moves the choice only, so it gets no gradient.  Backward, from dw:
//   ds_j = a / S (dw_j - sum_i dw_i s_i / S), S = sum_i s_i + 1e-20   (or a dw_j)
//   sigmoid: dl_j = ds_j s_j (1 - s_j);  softmax: dl_e = s_e (ds_e - sum_j ds_j s_j)
//
// Two choices may be closer than 32-bit rounding, and the experts picked are those of the
// definition: a token is ranked in f32, and again in 64 bits where two neighbours of that
// order (or the last kept and the first dropped group) are closer than the f32 error.  That error
// is the largest of the token's choices, so the wider the logits spread the more tokens need 64
// bits: of softmax scores of 64 experts, top-8, 0.1 % at a standard deviation of 1.5, 7 % at 5, 34 % at 8.
#include <type_traits>

#include "kmoe_common.h"

namespace {

constexpr double ROUTE_TINY = 1e-20;
constexpr int MAX_K = 8;

// Order-preserving integer of a double, NaN on top.
__device__ __forceinline__ int64_t key_of(double v) {
  if (v != v) return INT64_MAX;
  const int64_t b = __double_as_longlong(v == 0.0 ? 0.0 : v);  // -0 and 0 are equal
  return b < 0 ? (int64_t)(~(uint64_t)b ^ 0x8000000000000000ull) : b;
}

// The value of the lane whose place in its group of 2 S lanes is mirrored (S 4, 8) or S lanes
// away (S 1, 2, 16, 32), by lane moves instead of LDS permutes: in a reduction that has made
// the groups of S lanes uniform both are the other group's.
template <int S>
__device__ __forceinline__ int across(int v) {
  if constexpr (S == 1)
    return __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xF, 0xF, false);  // quad_perm 1 0 3 2
  else if constexpr (S == 2)
    return __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xF, 0xF, false);  // quad_perm 2 3 0 1
  else if constexpr (S == 4)
    return __builtin_amdgcn_update_dpp(0, v, 0x141, 0xF, 0xF, false);  // row_half_mirror
  else if constexpr (S == 8)
    return __builtin_amdgcn_update_dpp(0, v, 0x140, 0xF, 0xF, false);  // row_mirror
  else
    return __shfl_xor(v, S, 64);
}
template <int L, class Op>
__device__ __forceinline__ float group_reduce(float v, Op op) {
  auto step = [&](auto s) { v = op(v, __int_as_float(across<decltype(s)::value>(__float_as_int(v)))); };
  if constexpr (L >= 2) step(std::integral_constant<int, 1>{});
  if constexpr (L >= 4) step(std::integral_constant<int, 2>{});
  if constexpr (L >= 8) step(std::integral_constant<int, 4>{});
  if constexpr (L >= 16) step(std::integral_constant<int, 8>{});
  if constexpr (L >= 32) step(std::integral_constant<int, 16>{});
  if constexpr (L >= 64) step(std::integral_constant<int, 32>{});
  return v;
}
template <int L>
__device__ __forceinline__ float group_sum(float v) {
  return group_reduce<L>(v, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ double wave_sum(double v) {
  auto step = [&](auto s) {
    constexpr int S = decltype(s)::value;
    const int64_t b = __double_as_longlong(v);
    const uint64_t hi = (uint32_t)across<S>((int)(b >> 32)), lo = (uint32_t)across<S>((int)b);
    v += __longlong_as_double((int64_t)(hi << 32 | lo));
  };
  step(std::integral_constant<int, 1>{});
  step(std::integral_constant<int, 2>{});
  step(std::integral_constant<int, 4>{});
  step(std::integral_constant<int, 8>{});
  step(std::integral_constant<int, 16>{});
  step(std::integral_constant<int, 32>{});
  return v;
}
// Maximum over the L lanes of a token, NaN if there is one.
template <int L>
__device__ __forceinline__ float group_max(float v) {
  return group_reduce<L>(v, [](float a, float b) { return a != a ? a : (b != b || b > a ? b : a); });
}
// Maximum of numbers.
template <int L>
__device__ __forceinline__ float group_top(float v) {
  return group_reduce<L>(v, [](float a, float b) { return fmaxf(a, b); });
}

// LDS written by this wave is read by this wave: no workgroup barrier.
__device__ __forceinline__ void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

struct RouteArgs {
  const float* logits;
  int64_t T;
  int E, k;
  bool sigmoid;
  const float* bias;
  int groups, topk_groups, group_top;
  bool renorm;
  float scale;
  int64_t* idx;
  float* w;
  int32_t* block_counts;
  int hb;  // tokens of a workgroup: the histogram's block
};

constexpr int LANES = 16;         // lanes of a token: its reductions are moves within a row of lanes

// What a token keeps in LDS.
struct RouteLds {
  int64_t key[KMOE_MAX_EXPERTS];   // (64: a lane's place each)
  int64_t gkey[KMOE_MAX_EXPERTS];
  float pick[MAX_K];  // chosen scores
};

// Scores of a token's logits l (expert sub EPL + i of the lane) in f32; rel: bounds of their
// relative errors: exp 2 half steps (2^-24) and, for softmax, the rounding of l - max, |l - max|
// half steps; the sum of the token's exponentials the same, at most 16 half steps where it
// matters (smaller ones add less than their error), and its additions 2 + log2 16; the quotient
// one: (|l - max| + 32) 2^-24.  Sigmoid: exp, sum, quotient, under 8 2^-24.
template <int EPL>
__device__ __forceinline__ void scores_of(const float (&l)[EPL], bool sigmoid, float (&s)[EPL], float (&rel)[EPL]) {
  if (sigmoid) {
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      s[i] = 1.0f / (1.0f + expf(-l[i]));  // 0 for -inf
      rel[i] = 0x1p-21f;
    }
    return;
  }
  float m = l[0];
#pragma unroll
  for (int i = 1; i < EPL; ++i) m = m != m ? m : (l[i] != l[i] || l[i] > m ? l[i] : m);
  m = group_max<LANES>(m);
  float z = 0.0f;
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    s[i] = m == -INFINITY ? 0.0f : expf(l[i] - m);
    rel[i] = (m - l[i] + 32.0f) * 0x1p-24f;
    z += s[i];
  }
  z = group_sum<LANES>(z);
#pragma unroll
  for (int i = 0; i < EPL; ++i) s[i] = m == -INFINITY ? 0.0f : s[i] / z;
}

// Groups kept by their values val[g] in LDS (equal values: lowest group first), as a mask;
// low and high: the least value kept and the greatest dropped among the lane's groups.
__device__ __forceinline__ uint64_t keep_groups(const RouteArgs& a, const float* val, int sub, float& low, float& high) {
  uint64_t kept = 0;
  for (int g = sub; g < a.groups; g += LANES) {
    const float v = val[g];
    int rank = 0;
#pragma unroll 8
    for (int j = 0; j < a.groups; ++j) {
      const float o = val[j];
      rank += o > v || (o == v && j < g);
    }
    if (rank < a.topk_groups) {
      kept |= 1ull << g;
      low = v < low ? v : low;
    } else {
      high = v > high ? v : high;
    }
  }
#pragma unroll
  for (int o = 1; o < LANES; o *= 2) kept |= __shfl_xor(kept, o, 64);
  return kept;
}
// Order-preserving integer of a float's bits, and back.
__device__ __forceinline__ int ordered(int b) { return b ^ ((b >> 31) & 0x7fffffff); }
__device__ __forceinline__ int row_max(int v) {
  v = max(v, across<1>(v));
  v = max(v, across<2>(v));
  v = max(v, across<4>(v));
  return max(v, across<8>(v));
}

// A token's order in 64 bits, by the whole wave: lane e holds expert e, its logit l and bias b
// (e >= E: l -inf).  The place of the lane's expert; its score in the token's pick if that is < k.
__device__ __forceinline__ int rank64(const RouteArgs& a, RouteLds& s, float l, float b, int lane, int gs) {
  double sc;
  if (a.sigmoid) {
    sc = 1.0 / (1.0 + exp(-(double)l));  // 0 for -inf
  } else {
    const float m = group_max<64>(l);
    sc = m == -INFINITY ? 0.0 : exp((double)l - (double)m);
    const double z = wave_sum(sc);
    sc = m == -INFINITY ? 0.0 : sc / z;
  }
  const double c = l == -INFINITY ? -INFINITY : sc + (double)b;
  int64_t key = lane < a.E ? key_of(c) : INT64_MIN;
  if (a.groups > 1) {
    s.key[lane] = __double_as_longlong(c);
    wave_lds_fence();
    int64_t mine = INT64_MIN;
    if (lane < a.groups) {
      double b1 = -INFINITY, b2 = -INFINITY;
      bool nan = false;
#pragma unroll 8
      for (int j = 0; j < gs; ++j) {
        const double v = __longlong_as_double(s.key[lane * gs + j]);
        nan |= v != v;
        if (v > b1) {
          b2 = b1;
          b1 = v;
        } else if (v > b2) {
          b2 = v;
        }
      }
      if (a.group_top == 2 && b2 > -INFINITY) b1 += b2;
      mine = nan ? INT64_MAX : key_of(b1);
    }
    s.gkey[lane] = mine;
    wave_lds_fence();
    int rank = 0;
#pragma unroll 8
    for (int j = 0; j < a.groups; ++j) {
      const int64_t o = s.gkey[j];
      rank += o > mine || (o == mine && j < lane);
    }
    const uint64_t kept = __ballot(lane < a.groups && rank < a.topk_groups);
    if (!((kept >> (lane / gs)) & 1)) key = INT64_MIN;  // behind masked experts
  }
  s.key[lane] = key;
  wave_lds_fence();
  int rank = 0;
#pragma unroll 8
  for (int j = 0; j < a.E; ++j) {
    const int64_t o = s.key[j];
    rank += o > key || (o == key && j < lane);
  }
  if (lane < a.E && rank < a.k) s.pick[rank] = l == -INFINITY ? 0.0f : (float)sc;
  return lane < a.E ? rank : MAX_K;
}

// One workgroup per histogram block, its waves independent of each other; 16 lanes hold a
// token, EPL experts each.  The time is that of one token's chain of dependent steps, so a
// wave works on four and a workgroup on 64 at once: 16384 tokens, 64 experts, 8 groups, top-8
// 11.9 us (64 lanes a token, four tokens a wave one after the other: 27), 64 tokens 5.5; with
// choices so far apart that no token needs the 64-bit order 8.6 and 5.5.  That order takes the
// whole wave for one token (with its 16 lanes, the wave's four tokens together, 12.9; where every
// token needs it, all logits alike, 29 against 17).  At standard deviations of the logits of
// 1.5 / 5 / 8 sigmoid 10 / 17 / 27 in a replayed graph, softmax 12 / 19 / 27.
template <int EPL>
__global__ __launch_bounds__(1024) void route_kernel(RouteArgs a) {
  __shared__ RouteLds lds[64];
  __shared__ int count[64];
  const int tid = threadIdx.x, sub = tid % LANES, slot = tid / LANES, base = tid & 63 & ~(LANES - 1);
  if (tid < 64) count[tid] = 0;
  __syncthreads();
  RouteLds& s = lds[slot];
  const int64_t t = (int64_t)blockIdx.x * a.hb + slot;  // blockDim.x = LANES hb
  const bool live = t < a.T;
  const int gs = a.E / a.groups;
  float l[EPL], b[EPL], sc[EPL], x[EPL];
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    const int e = sub * EPL + i;
    const bool on = live && e < a.E;
    l[i] = on ? a.logits[t * a.E + e] : -INFINITY;
    b[i] = on && a.bias ? a.bias[e] : 0.0f;
  }
  if (!__any(live)) goto done;
  {
    float rel[EPL];  // more than the scores' relative errors
    scores_of<EPL>(l, a.sigmoid, sc, rel);
    bool sure = true;
    float err = 0.0f;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      x[i] = l[i] == -INFINITY ? -INFINITY : sc[i] + b[i];
      if (l[i] != -INFINITY) {
        sure = sure && fabsf(x[i]) < INFINITY;  // NaN and infinities are left to the 64-bit order
        err = fmaxf(err, sc[i] * rel[i] + fabsf(x[i]) * 0x1p-23f);
      }
    }
    err = group_top<LANES>(err);  // more than the error of any choice of the token
    if (a.groups > 1) {
      // (the 64-bit order's keys are not in use yet)
      float* const cv = reinterpret_cast<float*>(s.key);
      float* const gv = reinterpret_cast<float*>(s.gkey);
#pragma unroll
      for (int i = 0; i < EPL; ++i) cv[sub * EPL + i] = x[i];
      wave_lds_fence();
      for (int g = sub; g < a.groups; g += LANES) {
        float v = -INFINITY, b2 = -INFINITY;
#pragma unroll 8
        for (int j = 0; j < gs; ++j) {
          const float u = cv[g * gs + j];
          b2 = fmaxf(b2, fminf(v, u));
          v = fmaxf(v, u);
        }
        if (a.group_top == 2 && b2 > -INFINITY) v += b2;
        gv[g] = v;
      }
      wave_lds_fence();
      float low = INFINITY, high = -INFINITY;
      const uint64_t kept = keep_groups(a, gv, sub, low, high);
      low = -group_top<LANES>(-low);
      high = group_top<LANES>(high);
      // a group's value is the sum of up to two choices
      sure = sure && (a.topk_groups == a.groups || low - high > 4.0f * err);
#pragma unroll
      for (int i = 0; i < EPL; ++i)
        if (!((kept >> ((sub * EPL + i) / gs)) & 1)) x[i] = -INFINITY;
      wave_lds_fence();
    }
    // k rounds of the largest choice, and one more for the gap behind the last, on integers of
    // the floats' order.  Equal choices go in one round: more than k are then gone.
    int rank[EPL], key[EPL];
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      rank[i] = MAX_K;
      key[i] = ordered(__float_as_int(x[i]));
    }
    float last = INFINITY;
    auto round = [&](int r, bool take) {
      int m = key[0];
#pragma unroll
      for (int i = 1; i < EPL; ++i) m = max(m, key[i]);
      m = row_max(m);
      const float best = __int_as_float(ordered(m));
      sure = sure && last - best > 2.0f * err && (best > -INFINITY || !take);
      last = best;
      if (take) {
#pragma unroll
        for (int i = 0; i < EPL; ++i) {
          const bool hit = key[i] == m;
          rank[i] = hit ? r : rank[i];
          key[i] = hit ? INT_MIN : key[i];
        }
      }
    };
    for (int r = 0; r < a.k; ++r) round(r, true);
    if (a.k < a.E) round(a.k, false);
    float gone = 0.0f;
#pragma unroll
    for (int i = 0; i < EPL; ++i)
      if (rank[i] < a.k) {
        gone += 1.0f;
        s.pick[rank[i]] = sc[i];
      }
    sure = sure && group_sum<LANES>(gone) == (float)a.k;
    wave_lds_fence();
    const uint64_t open = __ballot(live && !sure);  // lanes of the tokens to order in 64 bits
    if (open) {
      float* const lv = reinterpret_cast<float*>(s.key);
#pragma unroll
      for (int i = 0; i < EPL; ++i) lv[sub * EPL + i] = l[i];
      wave_lds_fence();
      const int lane = tid & 63;
      for (int j = 0; j < 64 / LANES; ++j)
        if ((open >> (j * LANES)) & 0xffffu) {
          const int tok = (tid >> 6) * (64 / LANES) + j;
          RouteLds& o = lds[tok];
          const float le = lane < a.E ? reinterpret_cast<const float*>(o.key)[lane] : -INFINITY;
          const float be = lane < a.E && a.bias ? a.bias[lane] : 0.0f;
          wave_lds_fence();
          const int r = rank64(a, o, le, be, lane, gs);
          if (r < a.k) {
            a.idx[((int64_t)blockIdx.x * a.hb + tok) * a.k + r] = lane;
            if (a.block_counts) atomicAdd(&count[lane], 1);
          }
        }
      wave_lds_fence();
      if ((open >> base) & 0xffffu)
#pragma unroll
        for (int i = 0; i < EPL; ++i) rank[i] = MAX_K;  // written above
    }
#pragma unroll
    for (int i = 0; i < EPL; ++i)
      if (live && rank[i] < a.k) {
        a.idx[t * a.k + rank[i]] = sub * EPL + i;
        if (a.block_counts) atomicAdd(&count[sub * EPL + i], 1);
      }
    const float p = sub < a.k ? s.pick[sub] : 0.0f;
    const float sum = group_sum<LANES>(p) + (float)ROUTE_TINY;
    if (live && sub < a.k) a.w[t * a.k + sub] = a.scale * (a.renorm ? p / sum : p);
  }
done:
  if (a.block_counts) {
    __syncthreads();
    if (tid < a.E) a.block_counts[(int64_t)blockIdx.x * a.E + tid] = count[tid];
  }
}

// v of lane J of the lane's row of 16 (L 8: of its half row).
template <int L, int J>
__device__ __forceinline__ int entry(int v) {
  const int lo = __builtin_amdgcn_update_dpp(0, v, 0x150 + J, 0xF, 0xF, false);  // row_newbcast
  if constexpr (L >= 16) return lo;
  const int hi = __builtin_amdgcn_update_dpp(0, v, 0x150 + J + 8, 0xF, 0xF, false);
  return threadIdx.x & 8 ? hi : lo;
}
// f(j) for the entries j < k, two at a time (with an odd k one past it, an entry without an expert).
template <int J = 0, class Fn>
__device__ __forceinline__ void each_entry(int k, Fn&& f) {
  if constexpr (J < MAX_K) {
    if (J >= k) return;
    f(std::integral_constant<int, J>{});
    f(std::integral_constant<int, J + 1>{});
    each_entry<J + 2>(k, f);
  }
}

// dlogits (accumulate: added to).  L lanes per token; f32 throughout: no comparisons.  Differences of
// sums that nearly cancel are written as sums of differences, with P = sum of the chosen s, S = P + tiny,
// D_e = sum_i s_i (dw_e - dw_i) over the chosen i, m = sum_i s_i dw_i / S:
//   renorm   ds_e = a / S (D_e + tiny dw_e) / S;  sum_i ds_i s_i = a tiny m / S
//   without  softmax: ds_e - sum_i ds_i s_i = a (D_e + dw_e U), U the sum of the other experts' s
// so that gradients that vanish (one expert, or equal dw, renormalised) are not the roundings of
// the terms: sigmoid, 16 experts, top-1 had up to 5e-7 of those.  s (1 - s) of the sigmoid
// comes from exp(-|l|) for the same reason.  A lane loads one entry of the choice, and the
// others come by moves within its row of lanes.  A launch's latency and one chain of reductions: 4099
// tokens, 48 experts, top-6 in a replayed graph 3.5 us (with sums over the lanes in
// place of the entries 3.8), 16384 tokens, 64 experts, top-8 6.5 (8.3).
template <int L>
__global__ __launch_bounds__(256) void route_bwd_kernel(const float* __restrict__ logits, const int64_t* __restrict__ idx,
                                                        const float* __restrict__ dw, int64_t T, int E, int k, bool sigmoid,
                                                        bool renorm, float scale, bool accumulate,
                                                        float* __restrict__ dlogits) {
  const int e = threadIdx.x % L;
  const int64_t t = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
  const bool live = t < T, on = live && e < E;
  const float l = on ? logits[t * E + e] : -INFINITY;
  // the token's choice, one entry j a lane (copies in each row of 16 lanes): its expert (an id out of
  // range: none) and the gradient of its weight
  constexpr int ROW = L < 16 ? L : 16;
  const int j0 = threadIdx.x % ROW;
  const int64_t id = live && j0 < k ? idx[t * k + j0] : -1;
  const int ej = id >= 0 && id < E ? (int)id : -1;
  const float gj = ej >= 0 ? dw[t * k + j0] : 0.0f;
  // this lane's own gradient, 0 where it was not chosen
  float g = 0.0f;
  bool chosen = false;
  each_entry(k, [&](auto j) {  // (the broadcasts by all lanes: none under a condition of the lane's own)
    const int ev = entry<L, decltype(j)::value>(ej);
    const float gv = __int_as_float(entry<L, decltype(j)::value>(__float_as_int(gj)));
    g = ev == e ? gv : g;
    chosen = chosen || ev == e;
  });
  float s, ds_dl = 0.0f;  // score; its own derivative (sigmoid)
  if (sigmoid) {
    const float q = expf(-fabsf(l)), r = 1.0f / (1.0f + q);
    s = on ? (l < 0.0f ? q * r : r) : 0.0f;
    ds_dl = q * r * r;
  } else {
    const float m = group_max<L>(l);
    s = on && m != -INFINITY ? expf(l - m) : 0.0f;
    const float z = group_sum<L>(s);
    s = m == -INFINITY ? 0.0f : s / z;
  }
  const float si = __shfl(s, max(ej, 0), L), sj = ej >= 0 ? si : 0.0f;
  float S = 0.0f, D = 0.0f, M = 0.0f;
  each_entry(k, [&](auto j) {  // entries without an expert add zeros
    const float sv = __int_as_float(entry<L, decltype(j)::value>(__float_as_int(sj)));
    const float gv = __int_as_float(entry<L, decltype(j)::value>(__float_as_int(gj)));
    S += sv;
    D = fmaf(sv, g - gv, D);
    M = fmaf(sv, gv, M);
  });
  float dl;
  if (renorm) {
    // (s / S and ds_dl / S are at most 1 for a chosen expert, also where S is tiny)
    S += (float)ROUTE_TINY;
    const float c = chosen ? fmaf(g, (float)ROUTE_TINY, D) / S : 0.0f;
    dl = !sigmoid ? scale * (s / S) * (c - M / S * (float)ROUTE_TINY) : chosen ? scale * (ds_dl / S) * c : 0.0f;
  } else if (sigmoid) {
    dl = chosen ? scale * g * ds_dl : 0.0f;
  } else {
    const float U = group_sum<L>(chosen ? 0.0f : s);
    dl = scale * s * fmaf(g, U, D);
  }
  if (on) dlogits[t * E + e] = accumulate ? dlogits[t * E + e] + dl : dl;
}

int lanes_of(int E) {
  int l = 8;
  while (l < E) l *= 2;
  return l;
}

}  // namespace

extern "C" int kmoe_route_topk(const float* logits, int64_t T, int E, int k, int scores, const float* bias, int groups,
                               int topk_groups, int group_top, int renorm, float scale, int64_t* topk_idx, float* topk_w,
                               int32_t* block_counts, void* stream) {
  KMOE_REQUIRE(T == 0 || (logits && topk_idx && topk_w), KMOE_ERR_NULL, "kmoe_route_topk: null buffer");
  KMOE_REQUIRE(T >= 0 && E >= 1 && E <= KMOE_MAX_EXPERTS, KMOE_ERR_SHAPE, "kmoe_route_topk: T=%lld, E=%d (1..%d)",
               (long long)T, E, KMOE_MAX_EXPERTS);
  KMOE_REQUIRE(groups >= 1 && E % groups == 0 && topk_groups >= 1 && topk_groups <= groups, KMOE_ERR_SHAPE,
               "kmoe_route_topk: groups=%d must divide E=%d and topk_groups=%d lie in 1..groups", groups, E, topk_groups);
  KMOE_REQUIRE(k >= 1 && k <= MAX_K && k <= topk_groups * (E / groups), KMOE_ERR_SHAPE,
               "kmoe_route_topk: k=%d must lie in 1..%d and not exceed the experts of the kept groups (%d)", k, MAX_K,
               topk_groups * (E / groups));
  KMOE_REQUIRE(scores == KMOE_SCORES_SOFTMAX || scores == KMOE_SCORES_SIGMOID, KMOE_ERR_UNSUPPORTED,
               "kmoe_route_topk: scores=%d", scores);
  KMOE_REQUIRE(group_top == 1 || group_top == 2, KMOE_ERR_SHAPE, "kmoe_route_topk: group_top=%d must be 1 or 2", group_top);
  if (T == 0) return KMOE_OK;
  const int hb = kmoe::router_block_tokens(T);
  const int64_t blocks = kmoe::ceil_div<int64_t>(T, hb);
  KMOE_REQUIRE(blocks < 1 << 22, KMOE_ERR_SHAPE, "kmoe_route_topk: T=%lld is too large", (long long)T);
  const RouteArgs a{logits, T,    E,           k,      scores == KMOE_SCORES_SIGMOID, bias, groups, topk_groups, group_top,
                    renorm != 0, scale, topk_idx, topk_w, block_counts, hb};
  hipStream_t s = kmoe::as_stream(stream);
  const dim3 grid((unsigned)blocks), block(LANES * hb);  // 512 or 1024 threads
  if (E <= LANES)
    hipLaunchKernelGGL(route_kernel<1>, grid, block, 0, s, a);
  else if (E <= 2 * LANES)
    hipLaunchKernelGGL(route_kernel<2>, grid, block, 0, s, a);
  else
    hipLaunchKernelGGL(route_kernel<4>, grid, block, 0, s, a);
  return kmoe::check_launch("kmoe_route_topk");
}

extern "C" int kmoe_route_topk_bwd(const float* logits, const int64_t* topk_idx, const float* dw, int64_t T, int E, int k,
                                   int scores, int renorm, float scale, int accumulate, float* dlogits, void* stream) {
  KMOE_REQUIRE(T == 0 || (logits && topk_idx && dw && dlogits), KMOE_ERR_NULL, "kmoe_route_topk_bwd: null buffer");
  KMOE_REQUIRE(T >= 0 && E >= 1 && E <= KMOE_MAX_EXPERTS && k >= 1 && k <= MAX_K && k <= E, KMOE_ERR_SHAPE,
               "kmoe_route_topk_bwd: T=%lld, E=%d, k=%d", (long long)T, E, k);
  KMOE_REQUIRE(scores == KMOE_SCORES_SOFTMAX || scores == KMOE_SCORES_SIGMOID, KMOE_ERR_UNSUPPORTED,
               "kmoe_route_topk_bwd: scores=%d", scores);
  if (T == 0) return KMOE_OK;
  const int L = lanes_of(E);
  const int64_t blocks = kmoe::ceil_div<int64_t>(T, 256 / L);
  KMOE_REQUIRE(blocks < 1 << 24, KMOE_ERR_SHAPE, "kmoe_route_topk_bwd: T=%lld is too large", (long long)T);
  hipStream_t s = kmoe::as_stream(stream);
  const bool sig = scores == KMOE_SCORES_SIGMOID;
#define KMOE_ROUTE_BWD(L_)                                                                                                  \
  hipLaunchKernelGGL(route_bwd_kernel<L_>, dim3((unsigned)blocks), dim3(256), 0, s, logits, topk_idx, dw, T, E, k, sig,      \
                     renorm != 0, scale, accumulate != 0, dlogits)
  switch (L) {
    case 8: KMOE_ROUTE_BWD(8); break;
    case 16: KMOE_ROUTE_BWD(16); break;
    case 32: KMOE_ROUTE_BWD(32); break;
    default: KMOE_ROUTE_BWD(64);
  }
#undef KMOE_ROUTE_BWD
  return kmoe::check_launch("kmoe_route_topk_bwd");
}
