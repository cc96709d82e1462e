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
// Two choices may be closer than 32-bit rounding: choices and group values are computed and
// compared in 64 bits, so the experts picked are those of the definition.
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

template <int L, class V>
__device__ __forceinline__ V group_sum(V v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
// maximum over the L lanes of a token, NaN if there is one
template <int L>
__device__ __forceinline__ float group_max(float v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) {
    const float u = __shfl_xor(v, o, 64);
    v = v != v ? v : (u != u || u > v ? u : v);
  }
  return v;
}

// Score of lane e's logit (64 bits); every lane of the token's L takes part.
template <int L>
__device__ __forceinline__ double score(float l, bool on, bool sigmoid) {
  if (sigmoid) return on ? 1.0 / (1.0 + exp(-(double)l)) : 0.0;
  const float m = group_max<L>(on ? l : -INFINITY);
  if (m == -INFINITY) return 0.0;
  const double p = on ? exp((double)l - (double)m) : 0.0;
  return p / group_sum<L>(p);
}

struct RouteArgs {
  const float* logits;
  int64_t T;
  int E, k;
  bool sigmoid;
  const float* bias;
  int groups, topk_groups, group_top;
  bool renorm;
  double scale;
  int64_t* idx;
  float* w;
  int32_t* block_counts;
  int hb;  // tokens of a workgroup: the histogram's block
};

// One workgroup per histogram block; L lanes (a power of two >= E) hold a token's experts.
// Ranks are counted: an expert's place is the number of experts ahead of it, read from LDS
// as broadcasts, so no step depends on the one before.
template <int L>
__global__ __launch_bounds__(1024) void route_kernel(RouteArgs a) {
  __shared__ int64_t key[1024];
  __shared__ int64_t gkey[1024];
  __shared__ double pick[1024 / L][MAX_K];
  __shared__ int count[64];
  const int tid = threadIdx.x, e = tid % L, slot = tid / L, per = blockDim.x / L;
  const int64_t t_begin = (int64_t)blockIdx.x * a.hb;
  if (tid < 64) count[tid] = 0;
  const int gs = a.E / a.groups;
  for (int p = 0; p < a.hb; p += per) {  // the same trip count for every thread
    const int64_t t = t_begin + p + slot;
    const bool live = p + slot < a.hb && t < a.T;
    const bool on = live && e < a.E;
    const float l = on ? a.logits[t * a.E + e] : -INFINITY;
    const double s = score<L>(l, on, a.sigmoid);
    const bool masked = !on || l == -INFINITY;
    const double c = masked ? -INFINITY : s + (a.bias ? (double)a.bias[e] : 0.0);
    int64_t kc = key_of(c);
    const int64_t none = key_of(-INFINITY);
    bool in = on;
    if (a.groups > 1) {
      __syncthreads();
      key[tid] = __double_as_longlong(c);
      __syncthreads();
      if (e < a.groups) {
        double b1 = -INFINITY, b2 = -INFINITY;
        bool nan = false;
        for (int j = 0; j < gs; ++j) {
          const double v = __longlong_as_double(key[slot * L + e * gs + j]);
          nan |= v != v;
          if (v > b1) {
            b2 = b1;
            b1 = v;
          } else if (v > b2) {
            b2 = v;
          }
        }
        if (a.group_top == 2 && b2 > -INFINITY) b1 += b2;
        gkey[tid] = nan ? INT64_MAX : key_of(b1);
      }
      __syncthreads();
      if (on) {
        const int g = e / gs;
        const int64_t mine = gkey[slot * L + g];
        int rank = 0;
        for (int j = 0; j < a.groups; ++j) {
          const int64_t o = gkey[slot * L + j];
          rank += o > mine || (o == mine && j < g);
        }
        in = rank < a.topk_groups;
      }
    }
    __syncthreads();
    // experts of dropped groups rank behind masked ones
    key[tid] = in ? kc : INT64_MIN;
    if (!in) kc = INT64_MIN;
    __syncthreads();
    if (on && in) {
      int rank = 0;
      for (int j = 0; j < a.E; ++j) {
        const int64_t o = key[slot * L + j];
        rank += o > kc || (o == kc && j < e);
      }
      if (rank < a.k) {
        pick[slot][rank] = kc == none ? 0.0 : s;
        a.idx[t * a.k + rank] = e;
        if (a.block_counts) atomicAdd(&count[e], 1);
      }
    }
    __syncthreads();
    if (live && e < a.k) {
      double w = pick[slot][e];
      if (a.renorm) {
        double sum = ROUTE_TINY;
        for (int j = 0; j < a.k; ++j) sum += pick[slot][j];
        w /= sum;
      }
      a.w[t * a.k + e] = (float)(a.scale * w);
    }
  }
  if (a.block_counts) {
    __syncthreads();
    if (tid < a.E) a.block_counts[(int64_t)blockIdx.x * a.E + tid] = count[tid];
  }
}

// dlogits (accumulate: added to).  L lanes per token; f32 throughout: no comparisons.
template <int L>
__global__ __launch_bounds__(256) void route_bwd_kernel(const float* __restrict__ logits, const int64_t* __restrict__ idx,
                                                        const float* __restrict__ dw, int64_t T, int E, int k, bool sigmoid,
                                                        bool renorm, float scale, bool accumulate,
                                                        float* __restrict__ dlogits) {
  const int e = threadIdx.x % L;
  const int64_t t = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
  const bool live = t < T, on = live && e < E;
  const float l = on ? logits[t * E + e] : -INFINITY;
  float s;
  if (sigmoid) {
    s = on ? 1.0f / (1.0f + expf(-l)) : 0.0f;
  } else {
    const float m = group_max<L>(l);
    s = on && m != -INFINITY ? expf(l - m) : 0.0f;
    const float z = group_sum<L>(s);
    s = m == -INFINITY ? 0.0f : s / z;
  }
  // this lane's gradient of the weight, 0 where it was not chosen
  float g = 0.0f;
  bool chosen = false;
  if (on)
    for (int j = 0; j < k; ++j)
      if (idx[t * k + j] == e) {
        g = dw[t * k + j];
        chosen = true;
      }
  float ds = scale * g;
  if (renorm) {
    const float S = group_sum<L>(chosen ? s : 0.0f) + (float)ROUTE_TINY;
    const float mean = group_sum<L>(chosen ? g * s : 0.0f) / S;
    ds = chosen ? scale / S * (g - mean) : 0.0f;
  }
  float dl;
  if (sigmoid) {
    dl = chosen ? ds * s * (1.0f - s) : 0.0f;
  } else {
    const float q = group_sum<L>(chosen ? ds * s : 0.0f);
    dl = s * (ds - q);
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
                    renorm != 0, (double)scale, topk_idx, topk_w, block_counts, hb};
  hipStream_t s = kmoe::as_stream(stream);
  const int L = lanes_of(E);
  const int threads = hb * L < 1024 ? hb * L : 1024;
  switch (L) {
    case 8: hipLaunchKernelGGL(route_kernel<8>, dim3((unsigned)blocks), dim3(threads), 0, s, a); break;
    case 16: hipLaunchKernelGGL(route_kernel<16>, dim3((unsigned)blocks), dim3(threads), 0, s, a); break;
    case 32: hipLaunchKernelGGL(route_kernel<32>, dim3((unsigned)blocks), dim3(threads), 0, s, a); break;
    default: hipLaunchKernelGGL(route_kernel<64>, dim3((unsigned)blocks), dim3(threads), 0, s, a);
  }
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
