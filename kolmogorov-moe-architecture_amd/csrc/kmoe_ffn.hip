// The gated feed-forward block and adapted projections without gradients in one native call, and
// the projection of few rows, which streams the weights once.
#include "kmoe_dense_launch.h"
#include "kmoe_few.h"

using namespace kmoe_dense;

namespace {

// ---------------------------------------------------------------- few rows
// y = x w^T of T <= 16 rows.  A workgroup takes ROWS weight rows and all of x; its W waves share K and
// their sums meet in LDS.  Bound by the weights' bytes, and below some 10 MB by latency (one row,
// weights from HBM: 5632 x 2048 9.7 us, 2048 x 5632 8.2; the gate and up rows of the block are
// enough for the tiles of 64 x 64, 11.7 against 14.1 us).  An adapter is added in f32: a thread sums
// all ranks of one result, its factors on their way with the first weights.
// Of at most 8 rows what they lost by their rounding goes into the upper 8 of the MFMA's 16.
constexpr int FEW = 16, FEW_LOST = 8;

template <int ROWS, bool ADAPT>
__global__ __launch_bounds__(512) void few_kernel(Args g) {
  constexpr int W = 8, D = 4;
  __shared__ f32x4_t part[W][64];
  __shared__ float extra[16][ADAPT ? 17 : 1];  // [row of x][weight row]
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, lq = lane >> 4;
  const int n0 = blockIdx.x * ROWS;
  const int at = tid & 15, an = tid >> 4;
  int id = -1;
  if (ADAPT && at < g.M && an < ROWS && n0 + an < g.N) id = g.ad.ids[at];
  Stream16<1, W, D> st;
  st.w[0] = g.b[0] + (int64_t)n0 * g.ldb, st.x = g.a[0], st.K = g.K;
  st.woff[0] = l16 < ROWS && n0 + l16 < g.N ? (uint32_t)(l16 * g.ldb) * 2 : NOWHERE;
  const int lost = g.fold ? l16 - 8 : -1;  // (less than 2^27 bytes behind)
  st.xoff = l16 < g.M                  ? (uint32_t)(l16 * g.lda) * 2
            : lost >= 0 && lost < g.M  ? (uint32_t)(g.fold + lost * g.lda) * 2
                                       : NOWHERE;
  f32x4_t acc[1] = {f32x4_t{0.0f, 0.0f, 0.0f, 0.0f}};
  st.start(wave, lane);
  if constexpr (ADAPT) {
    float sum = 0.0f;
    if ((unsigned)id < (unsigned)g.ad.n) {
      const uint16_t* const b = g.ad.b[0] + ((int64_t)id * g.N + n0 + an) * g.ad.r;
      const uint16_t* const v = g.ad.v[0] + at * g.ad.r;
      for (int s = 0; s < g.ad.r; s += 32) {
        i32x4_t bv[4], vv[4], lv[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int j = s + 8 * q < g.ad.r ? s + 8 * q : s;
          bv[q] = *reinterpret_cast<const i32x4_t*>(b + j);
          vv[q] = *reinterpret_cast<const i32x4_t*>(v + j);
          lv[q] = *reinterpret_cast<const i32x4_t*>(v + g.M * g.ad.r + j);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          if (s + 8 * q >= g.ad.r) break;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            auto half = [&](const i32x4_t& w, int i) {
              return __uint_as_float(i ? (uint32_t)w[c] & 0xffff0000u : (uint32_t)w[c] << 16);
            };
            sum += half(bv[q], 0) * (half(vv[q], 0) + half(lv[q], 0)) + half(bv[q], 1) * (half(vv[q], 1) + half(lv[q], 1));
          }
        }
      }
    }
    if (an < 16) extra[at][an] = sum;
  }
  st.run(wave, lane, acc);
  part[wave][lane] = acc[0];
  __syncthreads();
  // row l % 16, columns n0 + 4 (l / 16) .. + 3
  const int n = n0 + 4 * lq;
  if (wave) return;
  f32x4_t s = part[0][lane];
#pragma unroll
  for (int k = 1; k < W; ++k) s += part[k][lane];
  if (g.fold) {
#pragma unroll
    for (int c = 0; c < 4; ++c) s[c] = with_lost(s[c], __shfl(s[c], lane | 8, 64));
  }
  if (l16 >= g.M || 4 * lq >= ROWS || n >= g.N) return;
  if constexpr (ADAPT) {
#pragma unroll
    for (int c = 0; c < 4; ++c) s[c] += extra[l16][4 * lq + c];
  }
  *reinterpret_cast<i32x2_t*>(static_cast<uint16_t*>(g.c) + l16 * g.ldc + n) = pack4(s[0], s[1], s[2], s[3]);
}

template <bool ADAPT>
int launch_few(const Args& g, hipStream_t s) {
  KMOE_REQUIRE(g.K < 1 << 22, KMOE_ERR_SHAPE, "kmoe product of few rows: rows of %d values (below 2^22)", g.K);
  // (8 weight rows a workgroup where 16 would leave units idle: 2048 x 5632 8.2 against 9.4 us, 5632 x
  // 2048 10.6 against 9.7)
  if (kmoe::ceil_div(g.N, 16) < kmoe::cu_count())
    hipLaunchKernelGGL((few_kernel<8, ADAPT>), dim3((unsigned)kmoe::ceil_div(g.N, 8)), dim3(512), 0, s, g);
  else
    hipLaunchKernelGGL((few_kernel<16, ADAPT>), dim3((unsigned)kmoe::ceil_div(g.N, 16)), dim3(512), 0, s, g);
  return kmoe::check_launch("kmoe product of few rows");
}

// Runs of K in which a projection of more rows is computed, where its tiles leave units idle: partial
// sums in f32, summed by a second launch (some 5 us with the partial sums' way).  1: in one.
int linear_runs(int64_t T, int K, int N, bool lost) {
  if (T <= (lost ? FEW_LOST : FEW)) return 1;
  const int64_t tiles = kmoe::ceil_div<int64_t>(T, 64) * kmoe::ceil_div(N, 64), cus = kmoe::cu_count();
  const int steps = kmoe::ceil_div(K, 64);
  double least;
  choose_tile(T, N, steps, T256, &least);
  int64_t best = 1;
  for (int side = 1; side <= 2; ++side) {
    int64_t runs = side * cus / tiles;
    runs = runs < 16 ? runs : 16;
    runs = runs < steps / 4 ? runs : steps / 4;
    if (runs < 2) continue;
    const double us = (tiles * runs > cus ? 0.50 : 0.33) * kmoe::ceil_div<int64_t>(steps, runs) + 2.0 + 5.0;
    if (us < least) least = us, best = runs;
  }
  return (int)best;
}
int64_t run_of(int K, int runs) { return kmoe::ceil_div(kmoe::ceil_div(K, 64), runs) * 64; }

const uint16_t* bf(const void* p) { return static_cast<const uint16_t*>(p); }
bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
size_t piece(int64_t bytes) { return (size_t)((bytes + 255) / 256 * 256); }

int check_adapter(const char* who, const kmoe_adapter* a, int n, int64_t T) {
  if (!a) return KMOE_OK;
  KMOE_REQUIRE(T <= ADAPTED_ROWS, KMOE_ERR_SHAPE, "%s: %lld rows with adapters (at most %lld)", who, (long long)T,
               (long long)ADAPTED_ROWS);
  KMOE_REQUIRE(a->a && a->b, KMOE_ERR_NULL, "%s: null adapter buffer", who);
  KMOE_REQUIRE(n > 0 && a->rank > 0 && a->rank <= KMOE_MAX_RANK && a->rank % 8 == 0, KMOE_ERR_SHAPE,
               "%s: %d adapters of rank %d (a multiple of 8, at most %d)", who, n, a->rank, KMOE_MAX_RANK);
  KMOE_REQUIRE(aligned(a->a) && aligned(a->b), KMOE_ERR_SHAPE, "%s: adapters are aligned to 16 bytes", who);
  return KMOE_OK;
}

size_t runs_bytes(int64_t T, int K, int N, bool lost) {
  const int runs = T > 0 && K > 0 && N > 0 ? linear_runs(T, K, N, lost) : 1;
  return runs > 1 ? piece((int64_t)runs * T * N * 4) : 0;
}

// y = x w^T with the adapter's outer product, whose inner products v are there; part: runs_bytes.
// lost: x is (2, T, K), the second T rows what the first ones lost.
int project(const void* x, bool lost, int64_t T, int K, const void* w, int N, const int32_t* ids, int n,
            const kmoe_adapter* ad, const void* v, void* y, void* part, hipStream_t s) {
  Args g{};
  g.a[0] = bf(x), g.b[0] = bf(w), g.K = K, g.lda = K, g.ldb = K, g.M = T, g.N = N, g.ldc = N, g.c = y;
  g.fold = lost ? T * K : 0;
  if (ad) g.ad = {ids, {bf(v), nullptr}, {bf(ad->b), nullptr}, n, ad->rank};
  if (T <= (lost ? FEW_LOST : FEW)) return ad ? launch_few<true>(g, s) : launch_few<false>(g, s);
  const int runs = linear_runs(T, K, N, lost);
  if (runs == 1) return ad ? launch_linear_adapt(g, s) : launch_linear(g, s);
  g.k_run = (int)run_of(K, runs), g.c = part, g.c_f32 = 1;
  if (const int rc = ad ? launch_linear_runs_adapt(g, s) : launch_linear_runs(g, s)) return rc;
  return launch_sum_runs(static_cast<const float*>(part), kmoe::ceil_div(K, g.k_run), T * N, static_cast<uint16_t*>(y), s);
}

}  // namespace

extern "C" size_t kmoe_adapted_linear_workspace_bytes(int64_t T, int K, int N, int rank) {
  if (T <= 0) return 0;
  return piece(T * (rank > 0 ? rank : 0) * 4) + runs_bytes(T, K, N, false);
}

extern "C" int kmoe_adapted_linear(const void* x, int64_t T, int K, const void* w, int N, const int32_t* ids, int n_adapters,
                                   const kmoe_adapter* adapter, void* y, void* workspace, size_t workspace_bytes,
                                   void* stream) {
  KMOE_REQUIRE(T >= 0 && T < ((int64_t)1 << 31) && K > 0 && N > 0 && K % 8 == 0 && N % 8 == 0, KMOE_ERR_SHAPE,
               "kmoe_adapted_linear: %lld rows of %d and %d values (positive multiples of 8)", (long long)T, K, N);
  if (const int rc = check_adapter("kmoe_adapted_linear", adapter, n_adapters, T)) return rc;
  if (T == 0) return KMOE_OK;
  KMOE_REQUIRE(x && w && y && (ids || !adapter), KMOE_ERR_NULL, "kmoe_adapted_linear: null buffer");
  KMOE_REQUIRE(aligned(x) && aligned(w) && aligned(y) && aligned(workspace), KMOE_ERR_SHAPE,
               "kmoe_adapted_linear: buffers are aligned to 16 bytes");
  const size_t need = kmoe_adapted_linear_workspace_bytes(T, K, N, adapter ? adapter->rank : 0);
  KMOE_REQUIRE((workspace || !need) && workspace_bytes >= need, KMOE_ERR_WORKSPACE,
               "kmoe_adapted_linear: workspace of %zu bytes, %zu are needed", workspace_bytes, need);
  if (adapter) {
    const int rc = adapter_inner(x, T, K, ids, n_adapters, adapter->rank, adapter->a, adapter->scale, workspace, nullptr,
                                 nullptr, nullptr, stream);
    if (rc) return rc;
  }
  return project(x, false, T, K, w, N, ids, n_adapters, adapter, workspace, y,
                 static_cast<uint8_t*>(workspace) + piece(T * (adapter ? adapter->rank : 0) * 4), kmoe::as_stream(stream));
}

extern "C" size_t kmoe_gated_ffn_workspace_bytes(int64_t T, int d, int F, int rank_gate_up, int rank_down) {
  if (T <= 0) return 0;
  const bool lost = T <= LOST_ROWS;
  return piece(T * F * (lost ? 4 : 2)) + 2 * piece(T * rank_gate_up * 4) + piece(T * rank_down * 4) + runs_bytes(T, F, d, lost);
}

extern "C" int kmoe_gated_ffn(const void* x, int64_t T, int d, int F, const void* w_gate, const void* w_up,
                              const void* w_down, int act, const int32_t* ids, int n_adapters, const kmoe_adapter* gate,
                              const kmoe_adapter* up, const kmoe_adapter* down, void* y, void* workspace,
                              size_t workspace_bytes, void* stream) {
  KMOE_REQUIRE(T >= 0 && T < ((int64_t)1 << 31) && d > 0 && F > 0 && d % 8 == 0 && F % 8 == 0, KMOE_ERR_SHAPE,
               "kmoe_gated_ffn: %lld rows, d=%d, F=%d (positive multiples of 8)", (long long)T, d, F);
  KMOE_REQUIRE(act >= KMOE_ACT_SILU && act <= KMOE_ACT_RELU, KMOE_ERR_UNSUPPORTED, "kmoe_gated_ffn: activation %d", act);
  for (const kmoe_adapter* a : {gate, up, down})
    if (const int rc = check_adapter("kmoe_gated_ffn", a, n_adapters, T)) return rc;
  KMOE_REQUIRE(!gate || !up || gate->rank == up->rank, KMOE_ERR_SHAPE,
               "kmoe_gated_ffn: the gate's and the up projection's adapters have one rank, got %d and %d", gate->rank, up->rank);
  if (T == 0) return KMOE_OK;
  const bool any = gate || up || down;
  KMOE_REQUIRE(x && w_gate && w_up && w_down && y && workspace && (ids || !any), KMOE_ERR_NULL, "kmoe_gated_ffn: null buffer");
  KMOE_REQUIRE(aligned(x) && aligned(w_gate) && aligned(w_up) && aligned(w_down) && aligned(y) && aligned(workspace),
               KMOE_ERR_SHAPE, "kmoe_gated_ffn: buffers are aligned to 16 bytes");
  const int rgu = gate ? gate->rank : up ? up->rank : 0, rd = down ? down->rank : 0;
  KMOE_REQUIRE(workspace_bytes >= kmoe_gated_ffn_workspace_bytes(T, d, F, rgu, rd), KMOE_ERR_WORKSPACE,
               "kmoe_gated_ffn: workspace of %zu bytes, %zu are needed", workspace_bytes,
               kmoe_gated_ffn_workspace_bytes(T, d, F, rgu, rd));
  uint8_t* w = static_cast<uint8_t*>(workspace);
  void* const h = w;
  const bool lost = T <= LOST_ROWS;
  void* const vg = w += piece(T * F * (lost ? 4 : 2));
  void* const vu = w += piece(T * rgu * 4);
  void* const vd = w += piece(T * rgu * 4);
  void* const part = w += piece(T * rd * 4);
  hipStream_t s = kmoe::as_stream(stream);
  int rc = KMOE_OK;
  if (rgu) {
    if (gate && up)
      rc = adapter_inner(x, T, d, ids, n_adapters, rgu, gate->a, gate->scale, vg, up->a, up->scale, vu, stream);
    else
      rc = adapter_inner(x, T, d, ids, n_adapters, rgu, (gate ? gate : up)->a, (gate ? gate : up)->scale, gate ? vg : vu,
                              nullptr, nullptr, nullptr, stream);
    if (rc) return rc;
  }
  Args g{};
  g.a[0] = bf(x), g.b[0] = bf(w_gate), g.b[1] = bf(w_up), g.K = d, g.lda = d, g.ldb = d, g.M = T, g.N = F;
  g.ldc = F, g.c = h, g.lost = lost ? T * F : 0, g.act = act;
  if (rgu)
    g.ad = {ids, {gate ? bf(vg) : nullptr, up ? bf(vu) : nullptr}, {gate ? bf(gate->b) : nullptr, up ? bf(up->b) : nullptr},
            n_adapters, rgu};
  rc = rgu ? launch_gated_adapt(g, s) : launch_gated(g, s);
  if (rc) return rc;
  if (down) {
    rc = adapter_inner(h, T, F, ids, n_adapters, rd, down->a, down->scale, vd, nullptr, nullptr, nullptr, stream);
    if (rc) return rc;
  }
  return project(h, lost, T, F, w_down, d, ids, n_adapters, down, vd, y, part, s);
}
