// The gated feed-forward block and adapted projections without gradients in one native call, and
// the products of few rows, which stream the weights once.
#include "kmoe_dense_launch.h"

using namespace kmoe_dense;

namespace {

// ---------------------------------------------------------------- few rows
// A workgroup takes 16 weight rows (GATED: 16 gate and the same 16 up rows) and all T <= 64 rows of
// x; its waves share K, 64 at a time, each lane reading 16 bytes of a weight row and of an x row
// straight into the MFMA's operands: every weight byte is read once, by one wave, two 64-byte
// halves of a line one after the other.  The waves' sums meet in LDS.  Bound by the weights'
// bytes, and below some 10 MB by latency.  Adapters are added by the lanes that hold the results,
// rank by rank in f32 (few rows: their factors are read once, like the weights).
constexpr int FEW = 64;

template <int TB, int W, bool GATED, bool ADAPT>
__global__ __launch_bounds__(W * 64) void few_kernel(Args g) {
  constexpr int G = GATED ? 2 : 1;
  __shared__ f32x4_t part[W][G][TB][64];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, lq = lane >> 4;
  const int n0 = blockIdx.x * 16;
  const int wrow = n0 + l16 < g.N ? n0 + l16 : g.N - 1;
  const uint16_t* wp[G];
#pragma unroll
  for (int y = 0; y < G; ++y) wp[y] = g.b[y] + (int64_t)wrow * g.ldb;
  const uint16_t* xp[TB];
#pragma unroll
  for (int b = 0; b < TB; ++b) {
    const int64_t t = b * 16 + l16 < g.M ? b * 16 + l16 : g.M - 1;
    xp[b] = g.a[0] + t * g.lda;
  }
  f32x4_t acc[G][TB];
#pragma unroll
  for (int y = 0; y < G; ++y)
#pragma unroll
    for (int b = 0; b < TB; ++b) acc[y][b] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  auto step = [&](int k, bool in) {
    bf16x8_t fw[G], fx[TB];
#pragma unroll
    for (int y = 0; y < G; ++y) {
      fw[y] = *reinterpret_cast<const bf16x8_t*>(wp[y] + (in ? k : 0));
      if (!in) fw[y] = bf16x8_t{};
    }
#pragma unroll
    for (int b = 0; b < TB; ++b) {
      fx[b] = *reinterpret_cast<const bf16x8_t*>(xp[b] + (in ? k : 0));
      if (!in) fx[b] = bf16x8_t{};
    }
#pragma unroll
    for (int y = 0; y < G; ++y)
#pragma unroll
      for (int b = 0; b < TB; ++b) acc[y][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fw[y], fx[b], acc[y][b], 0, 0, 0);
  };
  const int full = g.K & ~63;
#pragma unroll 4
  for (int k0 = wave * 64; k0 < full; k0 += W * 64) {
    step(k0 + 8 * lq, true);
    step(k0 + 32 + 8 * lq, true);
  }
  if (full < g.K && (full / 64) % W == wave) {
    step(full + 8 * lq, full + 8 * lq < g.K);
    step(full + 32 + 8 * lq, full + 32 + 8 * lq < g.K);
  }
#pragma unroll
  for (int y = 0; y < G; ++y)
#pragma unroll
    for (int b = 0; b < TB; ++b) part[wave][y][b][lane] = acc[y][b];
  __syncthreads();
  // thread: row 16 (tid / 64) + l % 16, columns n0 + 4 (l / 16) .. + 3
  if (tid >= TB * 64) return;
  const int64_t t = wave * 16 + l16;
  const int n = n0 + 4 * lq;
  if (t >= g.M || n >= g.N) return;
  f32x4_t s[G];
#pragma unroll
  for (int y = 0; y < G; ++y) {
    s[y] = part[0][y][wave][lane];
#pragma unroll
    for (int w = 1; w < W; ++w) s[y] += part[w][y][wave][lane];
  }
  if constexpr (ADAPT) {
    const int id = g.ad.ids[t];
    if ((unsigned)id < (unsigned)g.ad.n) {
#pragma unroll
      for (int y = 0; y < G; ++y) {
        if (!g.ad.b[y]) continue;
        const uint16_t* const b = g.ad.b[y] + ((int64_t)id * g.N + n) * g.ad.r;
        const uint16_t* const v = g.ad.v[y] + t * g.ad.r;
        float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int j = 0; j < g.ad.r; j += 8) {
          const i32x4_t vv = *reinterpret_cast<const i32x4_t*>(v + j);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const i32x4_t bv = *reinterpret_cast<const i32x4_t*>(b + c * g.ad.r + j);
#pragma unroll
            for (int q = 0; q < 4; ++q)
              d[c] += __uint_as_float((uint32_t)vv[q] << 16) * __uint_as_float((uint32_t)bv[q] << 16) +
                      __uint_as_float((uint32_t)vv[q] & 0xffff0000u) * __uint_as_float((uint32_t)bv[q] & 0xffff0000u);
          }
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) s[y][c] += d[c];
      }
    }
  }
  float o[4];
  if constexpr (GATED) {
    with_act(g.act, [&](auto tag) {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        float a, da;
        act_at<decltype(tag)::value>(s[0][c], a, da);
        o[c] = a * s[G - 1][c];
      }
    });
  } else {
#pragma unroll
    for (int c = 0; c < 4; ++c) o[c] = s[0][c];
  }
  *reinterpret_cast<i32x2_t*>(static_cast<uint16_t*>(g.c) + t * g.ldc + n) = pack4(o[0], o[1], o[2], o[3]);
}

template <bool GATED, bool ADAPT>
int launch_few(const Args& g, hipStream_t s) {
  const dim3 grid((unsigned)kmoe::ceil_div(g.N, 16));
  constexpr int W = 8;
  switch (kmoe::ceil_div<int64_t>(g.M, 16)) {
    case 1: hipLaunchKernelGGL((few_kernel<1, W, GATED, ADAPT>), grid, dim3(W * 64), 0, s, g); break;
    case 2: hipLaunchKernelGGL((few_kernel<2, W, GATED, ADAPT>), grid, dim3(W * 64), 0, s, g); break;
    case 3: hipLaunchKernelGGL((few_kernel<3, W, GATED, ADAPT>), grid, dim3(W * 64), 0, s, g); break;
    default: hipLaunchKernelGGL((few_kernel<4, W, GATED, ADAPT>), grid, dim3(W * 64), 0, s, g);
  }
  return kmoe::check_launch("kmoe product of few rows");
}

const uint16_t* bf(const void* p) { return static_cast<const uint16_t*>(p); }
bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
size_t piece(int64_t bytes) { return (size_t)((bytes + 255) / 256 * 256); }

int check_adapter(const char* who, const kmoe_adapter* a, int n) {
  if (!a) return KMOE_OK;
  KMOE_REQUIRE(a->a && a->b, KMOE_ERR_NULL, "%s: null adapter buffer", who);
  KMOE_REQUIRE(n > 0 && a->rank > 0 && a->rank <= KMOE_MAX_RANK && a->rank % 8 == 0, KMOE_ERR_SHAPE,
               "%s: %d adapters of rank %d (a multiple of 8, at most %d)", who, n, a->rank, KMOE_MAX_RANK);
  KMOE_REQUIRE(aligned(a->a) && aligned(a->b), KMOE_ERR_SHAPE, "%s: adapters are aligned to 16 bytes", who);
  return KMOE_OK;
}

// y = x w^T with the adapter's outer product, whose inner products v are there.
int project(const void* x, int64_t T, int K, const void* w, int N, const int32_t* ids, int n, const kmoe_adapter* ad,
            const void* v, void* y, hipStream_t s) {
  if (T > FEW)
    return kmoe_dense_linear(x, T, K, w, N, ad ? ids : nullptr, n, ad ? ad->rank : 0, v, ad ? ad->b : nullptr, y, s);
  Args g{};
  g.a[0] = bf(x), g.b[0] = bf(w), g.K = K, g.lda = K, g.ldb = K, g.M = T, g.N = N, g.ldc = N, g.c = y;
  if (!ad) return launch_few<false, false>(g, s);
  g.ad = {ids, {bf(v), nullptr}, {bf(ad->b), nullptr}, n, ad->rank};
  return launch_few<false, true>(g, s);
}

}  // namespace

extern "C" size_t kmoe_adapted_linear_workspace_bytes(int64_t T, int rank) { return piece(T * (rank > 0 ? rank : 0) * 2); }

extern "C" int kmoe_adapted_linear(const void* x, int64_t T, int K, const void* w, int N, const int32_t* ids, int n_adapters,
                                   const kmoe_adapter* adapter, void* y, void* workspace, size_t workspace_bytes,
                                   void* stream) {
  KMOE_REQUIRE(T >= 0 && T < ((int64_t)1 << 31) && K > 0 && N > 0 && K % 8 == 0 && N % 8 == 0, KMOE_ERR_SHAPE,
               "kmoe_adapted_linear: %lld rows of %d and %d values (positive multiples of 8)", (long long)T, K, N);
  if (const int rc = check_adapter("kmoe_adapted_linear", adapter, n_adapters)) return rc;
  if (T == 0) return KMOE_OK;
  KMOE_REQUIRE(x && w && y && (ids || !adapter), KMOE_ERR_NULL, "kmoe_adapted_linear: null buffer");
  KMOE_REQUIRE(aligned(x) && aligned(w) && aligned(y) && aligned(workspace), KMOE_ERR_SHAPE,
               "kmoe_adapted_linear: buffers are aligned to 16 bytes");
  if (adapter) {
    KMOE_REQUIRE(workspace && workspace_bytes >= kmoe_adapted_linear_workspace_bytes(T, adapter->rank), KMOE_ERR_WORKSPACE,
                 "kmoe_adapted_linear: workspace of %zu bytes, %zu are needed", workspace_bytes,
                 kmoe_adapted_linear_workspace_bytes(T, adapter->rank));
    const int rc = kmoe_adapter_inner(x, T, K, ids, n_adapters, adapter->rank, adapter->a, adapter->scale, workspace, nullptr,
                                      nullptr, nullptr, stream);
    if (rc) return rc;
  }
  return project(x, T, K, w, N, ids, n_adapters, adapter, workspace, y, kmoe::as_stream(stream));
}

extern "C" size_t kmoe_gated_ffn_workspace_bytes(int64_t T, int F, int rank_gate_up, int rank_down) {
  return piece(T * F * 2) + 2 * piece(T * rank_gate_up * 2) + piece(T * rank_down * 2);
}

extern "C" int kmoe_gated_ffn(const void* x, int64_t T, int d, int F, const void* w_gate, const void* w_up,
                              const void* w_down, int act, const int32_t* ids, int n_adapters, const kmoe_adapter* gate,
                              const kmoe_adapter* up, const kmoe_adapter* down, void* y, void* workspace,
                              size_t workspace_bytes, void* stream) {
  KMOE_REQUIRE(T >= 0 && T < ((int64_t)1 << 31) && d > 0 && F > 0 && d % 8 == 0 && F % 8 == 0, KMOE_ERR_SHAPE,
               "kmoe_gated_ffn: %lld rows, d=%d, F=%d (positive multiples of 8)", (long long)T, d, F);
  KMOE_REQUIRE(act >= KMOE_ACT_SILU && act <= KMOE_ACT_RELU, KMOE_ERR_UNSUPPORTED, "kmoe_gated_ffn: activation %d", act);
  for (const kmoe_adapter* a : {gate, up, down})
    if (const int rc = check_adapter("kmoe_gated_ffn", a, n_adapters)) return rc;
  KMOE_REQUIRE(!gate || !up || gate->rank == up->rank, KMOE_ERR_SHAPE,
               "kmoe_gated_ffn: the gate's and the up projection's adapters have one rank, got %d and %d", gate->rank, up->rank);
  if (T == 0) return KMOE_OK;
  const bool any = gate || up || down;
  KMOE_REQUIRE(x && w_gate && w_up && w_down && y && workspace && (ids || !any), KMOE_ERR_NULL, "kmoe_gated_ffn: null buffer");
  KMOE_REQUIRE(aligned(x) && aligned(w_gate) && aligned(w_up) && aligned(w_down) && aligned(y) && aligned(workspace),
               KMOE_ERR_SHAPE, "kmoe_gated_ffn: buffers are aligned to 16 bytes");
  const int rgu = gate ? gate->rank : up ? up->rank : 0, rd = down ? down->rank : 0;
  KMOE_REQUIRE(workspace_bytes >= kmoe_gated_ffn_workspace_bytes(T, F, rgu, rd), KMOE_ERR_WORKSPACE,
               "kmoe_gated_ffn: workspace of %zu bytes, %zu are needed", workspace_bytes,
               kmoe_gated_ffn_workspace_bytes(T, F, rgu, rd));
  uint8_t* w = static_cast<uint8_t*>(workspace);
  void* const h = w;
  void* const vg = w += piece(T * F * 2);
  void* const vu = w += piece(T * rgu * 2);
  void* const vd = w += piece(T * rgu * 2);
  hipStream_t s = kmoe::as_stream(stream);
  int rc = KMOE_OK;
  if (rgu) {
    if (gate && up)
      rc = kmoe_adapter_inner(x, T, d, ids, n_adapters, rgu, gate->a, gate->scale, vg, up->a, up->scale, vu, stream);
    else
      rc = kmoe_adapter_inner(x, T, d, ids, n_adapters, rgu, (gate ? gate : up)->a, (gate ? gate : up)->scale, gate ? vg : vu,
                              nullptr, nullptr, nullptr, stream);
    if (rc) return rc;
  }
  if (T > FEW) {
    rc = kmoe_dense_gate_up(x, T, d, w_gate, w_up, F, act, rgu ? ids : nullptr, n_adapters, rgu, gate ? vg : nullptr,
                            gate ? gate->b : nullptr, up ? vu : nullptr, up ? up->b : nullptr, h, nullptr, stream);
  } else {
    Args g{};
    g.a[0] = bf(x), g.b[0] = bf(w_gate), g.b[1] = bf(w_up), g.K = d, g.lda = d, g.ldb = d, g.M = T, g.N = F;
    g.ldc = F, g.c = h, g.act = act;
    if (rgu)
      g.ad = {ids, {gate ? bf(vg) : nullptr, up ? bf(vu) : nullptr}, {gate ? bf(gate->b) : nullptr, up ? bf(up->b) : nullptr},
              n_adapters, rgu};
    rc = rgu ? launch_few<true, true>(g, s) : launch_few<true, false>(g, s);
  }
  if (rc) return rc;
  if (down) {
    rc = kmoe_adapter_inner(h, T, F, ids, n_adapters, rd, down->a, down->scale, vd, nullptr, nullptr, nullptr, stream);
    if (rc) return rc;
  }
  return project(h, T, F, w_down, d, ids, n_adapters, down, vd, y, s);
}
