// Low-rank adapters of many requests: the inner products, and the gradients of both factors.
#include "kmoe_dense_launch.h"
#include "kmoe_few.h"

using kmoe_dense::NOWHERE;
using kmoe_dense::pack4;
using kmoe_dense::Stream16;
using kmoe_dense::tr4_t;

namespace {

// ---------------------------------------------------------------- inner products
// v[t, j] = scale[i] sum_k x[t, k] a[i, j, k], i = ids[t], rounded to bf16: an operand of the outer
// product's MFMAs, one rounding (half a step of 2^-8) of a term that adds to the projection's.
// A workgroup takes 16 rows, RB blocks of 16 ranks and every gridDim.y-th of the adapters that the rows
// have (few rows with an adapter each: a workgroup an adapter); its 8 waves share K.  Each
// adapter's product is computed for all 16 rows and kept for those that have it: bound by reading
// x and the adapters, not by the products, and no row's values meet another's adapter.  Few
// rows take a workgroup a block of ranks: latency counts and x is small.
constexpr int SW = 8;  // waves

struct Shrink {
  const uint16_t* x;
  int64_t T;
  int K;
  const int32_t* ids;
  int n, r;
  int sides;      // 1 or 2 sets of adapters; blockIdx.z = the first of its RB blocks of ranks * sides + set
  const uint16_t* a[2];
  const float* scale[2];
  uint16_t* v[2];
};

template <int RB, int D>
__global__ __launch_bounds__(SW * 64) void shrink_kernel(Shrink g) {
  __shared__ f32x4_t part[SW][RB][64];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, lq = lane >> 4;
  const int64_t t0 = (int64_t)blockIdx.x * 16;
  const int z = blockIdx.z % g.sides, j0 = blockIdx.z / g.sides * (RB * 16);
  int id = t0 + l16 < g.T ? g.ids[t0 + l16] : -1;
  if ((unsigned)id >= (unsigned)g.n) id = -1;
  bool first = lane < 16 && id >= 0;
#pragma unroll
  for (int t = 0; t < 15; ++t) {
    const int o = __builtin_amdgcn_readlane(id, t);
    if (t < lane && o == id) first = false;
  }
  uint64_t todo = __ballot(first);
  Stream16<RB, SW, D> st;
  st.x = g.x + t0 * g.K, st.K = g.K;
  st.xoff = t0 + l16 < g.T ? (uint32_t)(l16 * g.K) * 2 : NOWHERE;
#pragma unroll
  for (int b = 0; b < RB; ++b) {
    const int j = j0 + b * 16 + l16;
    st.woff[b] = j < g.r ? (uint32_t)(j * g.K) * 2 : NOWHERE;
  }
  for (int c = 0; todo; ++c, todo &= todo - 1) {
    if (c % (int)gridDim.y != (int)blockIdx.y) continue;
    const int cur = __builtin_amdgcn_readlane(id, __builtin_ctzll(todo));
    f32x4_t acc[RB];
#pragma unroll
    for (int b = 0; b < RB; ++b) {
      st.w[b] = g.a[z] + (int64_t)cur * g.r * g.K;
      acc[b] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    }
    st.start(wave, lane);
    st.run(wave, lane, acc);
#pragma unroll
    for (int b = 0; b < RB; ++b) part[wave][b][lane] = acc[b];
    __syncthreads();
    // thread: ranks 4 (l / 16) .. + 3 of block tid / 64, row l % 16
    if (tid < RB * 64) {
      f32x4_t s = part[0][wave][lane];
#pragma unroll
      for (int w = 1; w < SW; ++w) s += part[w][wave][lane];
      const int j = j0 + wave * 16 + 4 * lq;
      if (id == cur && j < g.r) {
        const float f = g.scale[z] ? g.scale[z][cur] : 1.0f;
        *reinterpret_cast<i32x2_t*>(g.v[z] + (t0 + l16) * g.r + j) = pack4(f * s[0], f * s[1], f * s[2], f * s[3]);
      }
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------- gradients of the factors
// out[i][j, c] = sum over rows t with ids[t] = i of l[t, j] m[t, c], l (T, r), m (T, C), f32 sums.
// A workgroup takes an adapter, 128 columns (32 a wave) and a run of rows; of the run it visits the
// groups of 32 rows in which the adapter occurs, other rows in them read as zeros in both
// operands.  Operands along t come from LDS by transposing reads.  Runs of rows are summed by
// a second kernel, in order.  OUTER: out[i] is (C, r), the outer factor, instead of (r, C).
constexpr int GC = 128, GR = 32;     // columns of a workgroup, rows of a group
constexpr int GMAXRUN = 64 * 1024;   // rows of a run at most: a bit a group in LDS

struct FactorGrad {
  const uint16_t* l;
  const uint16_t* m;
  const int32_t* ids;
  int64_t T, run;
  int n, r, C;
  int runs;
  float* part;     // (runs, n, ...) when runs > 1
  uint16_t* out;
};

// byte of 8-byte piece at column col (a multiple of 4) of row t in a tile of ROWB-byte rows
template <int ROWB>
__device__ __forceinline__ int gpos(int t, int col) {
  return t * ROWB + (((col >> 3) ^ (ROWB >= 128 ? kmoe_dense::strided_swz<ROWB>(t) << 1 : 0)) << 4) + (col & 4) * 2;
}
template <int ROWB>
__device__ __forceinline__ bf16x8_t gfrag(const uint8_t* p, int col0, int lane) {
  const int i16 = lane & 15, t = 8 * (lane >> 4) + (i16 >> 2), col = col0 + 4 * (i16 & 3);
  const tr4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((KMOE_LDS tr4_t*)(p + gpos<ROWB>(t, col)));
  const tr4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((KMOE_LDS tr4_t*)(p + gpos<ROWB>(t + 4, col)));
  return __builtin_bit_cast(bf16x8_t, (short __attribute__((ext_vector_type(8)))){lo[0], lo[1], lo[2], lo[3], hi[0], hi[1],
                                                                                 hi[2], hi[3]});
}

template <int RB, bool OUTER>
__global__ __launch_bounds__(256) void factor_grad_kernel(FactorGrad g) {
  constexpr int LROWB = RB * 32, MROWB = GC * 2;
  __shared__ __attribute__((aligned(16))) uint8_t lt[GR * LROWB];
  __shared__ __attribute__((aligned(16))) uint8_t mt[GR * MROWB];
  __shared__ uint32_t occurs[GMAXRUN / GR / 32];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, lq = lane >> 4;
  const int c0 = blockIdx.x * GC, me = blockIdx.y;
  const int64_t r0 = (int64_t)blockIdx.z * g.run, r1 = r0 + g.run < g.T ? r0 + g.run : g.T;
  const int groups = r1 > r0 ? (int)((r1 - r0 + GR - 1) / GR) : 0;
  for (int w = tid; w < (groups + 31) / 32; w += 256) occurs[w] = 0;
  __syncthreads();
  // a wave looks at 64 rows, two groups, at a time
  for (int64_t t = r0 + wave * 64; t < r1; t += 256) {
    const uint64_t hit = __ballot(t + lane < r1 && g.ids[t + lane] == me);
    const int gi = (int)((t - r0) / GR);
    const uint32_t bits = ((uint32_t)hit ? 1u : 0u) | ((hit >> 32) ? 2u : 0u);
    if (lane == 0 && bits) atomicOr(&occurs[gi >> 5], bits << (gi & 31));
  }
  __syncthreads();
  f32x4_t acc[RB][2];
#pragma unroll
  for (int b = 0; b < RB; ++b) acc[b][0] = acc[b][1] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  for (int w = 0; w < (groups + 31) / 32; ++w) {
    uint32_t bits = __builtin_amdgcn_readfirstlane(occurs[w]);
    for (; bits; bits &= bits - 1) {
      const int64_t t0 = r0 + (int64_t)(w * 32 + __builtin_ctz(bits)) * GR;
      // 32 rows x 16 chunks of m, 32 x 2 RB of l
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int t = (tid >> 4) + 16 * q, ch = tid & 15;
        const bool in = t0 + t < r1 && g.ids[t0 + t] == me && c0 + ch * 8 < g.C;
        i32x4_t v{0, 0, 0, 0};
        if (in) v = *reinterpret_cast<const i32x4_t*>(g.m + (t0 + t) * g.C + c0 + ch * 8);
        *reinterpret_cast<i32x4_t*>(mt + gpos<MROWB>(t, ch * 8)) = v;
      }
      for (int e = tid; e < GR * 2 * RB; e += 256) {
        const int t = e / (2 * RB), ch = e % (2 * RB);
        const bool in = t0 + t < r1 && g.ids[t0 + t] == me && ch * 8 < g.r;
        i32x4_t v{0, 0, 0, 0};
        if (in) v = *reinterpret_cast<const i32x4_t*>(g.l + (t0 + t) * g.r + ch * 8);
        *reinterpret_cast<i32x4_t*>(lt + gpos<LROWB>(t, ch * 8)) = v;
      }
      __syncthreads();
      bf16x8_t fm[2];
#pragma unroll
      for (int y = 0; y < 2; ++y) fm[y] = gfrag<MROWB>(mt, wave * 32 + y * 16, lane);
#pragma unroll
      for (int b = 0; b < RB; ++b) {
        const bf16x8_t fl = gfrag<LROWB>(lt, b * 16, lane);
#pragma unroll
        for (int y = 0; y < 2; ++y)
          acc[b][y] = OUTER ? __builtin_amdgcn_mfma_f32_16x16x32_bf16(fl, fm[y], acc[b][y], 0, 0, 0)
                            : __builtin_amdgcn_mfma_f32_16x16x32_bf16(fm[y], fl, acc[b][y], 0, 0, 0);
      }
      __syncthreads();
    }
  }
  // OUTER: a lane holds column l % 16, ranks 4 (l / 16) .. + 3; else rank l % 16, four columns
  const int64_t size = (int64_t)g.r * g.C;
#pragma unroll
  for (int b = 0; b < RB; ++b)
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      const int c = c0 + wave * 32 + y * 16 + (OUTER ? l16 : 4 * lq), j = b * 16 + (OUTER ? 4 * lq : l16);
      if (c >= g.C || j >= g.r) continue;
      const int64_t at = OUTER ? (int64_t)c * g.r + j : (int64_t)j * g.C + c;
      const f32x4_t v = acc[b][y];
      if (g.runs > 1)
        *reinterpret_cast<f32x4_t*>(g.part + ((int64_t)blockIdx.z * g.n + me) * size + at) = v;
      else
        *reinterpret_cast<i32x2_t*>(g.out + me * size + at) = pack4(v[0], v[1], v[2], v[3]);
    }
}

__global__ __launch_bounds__(256) void sum_runs_kernel(const float* __restrict__ part, int runs, int64_t total,
                                                       uint16_t* __restrict__ out) {
  const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (at >= total) return;
  f32x4_t s = *reinterpret_cast<const f32x4_t*>(part + at);
  for (int k = 1; k < runs; ++k) s += *reinterpret_cast<const f32x4_t*>(part + (int64_t)k * total + at);
  *reinterpret_cast<i32x2_t*>(out + at) = pack4(s[0], s[1], s[2], s[3]);
}

// Runs of rows: as many as give every compute unit two workgroups, of at least 256 rows.
int64_t runs_of(int64_t T, int n, int C) {
  const int64_t blocks = (int64_t)n * kmoe::ceil_div(C, GC);
  int64_t runs = kmoe::ceil_div<int64_t>(512, blocks);
  runs = runs < kmoe::ceil_div<int64_t>(T, 256) ? runs : kmoe::ceil_div<int64_t>(T, 256);
  const int64_t least = kmoe::ceil_div<int64_t>(T, GMAXRUN);
  return runs > least ? runs : (least > 1 ? least : 1);
}

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace

int kmoe_dense::launch_sum_runs(const float* part, int runs, int64_t total, uint16_t* out, hipStream_t s) {
  hipLaunchKernelGGL(sum_runs_kernel, dim3((unsigned)kmoe::ceil_div<int64_t>(total, 1024)), dim3(256), 0, s, part, runs, total,
                     out);
  return kmoe::check_launch("kmoe sum of runs");
}

extern "C" int kmoe_adapter_inner(const void* x, int64_t T, int K, const int32_t* ids, int n, int rank, const void* a,
                                  const float* scale, void* v, const void* a2, const float* scale2, void* v2,
                                  void* stream) {
  KMOE_REQUIRE(T >= 0 && T < ((int64_t)1 << 31) && K > 0 && K % 8 == 0, KMOE_ERR_SHAPE,
               "kmoe_adapter_inner: %lld rows of %d values (a positive multiple of 8)", (long long)T, K);
  KMOE_REQUIRE(n > 0 && rank > 0 && rank <= KMOE_MAX_RANK && rank % 8 == 0, KMOE_ERR_SHAPE,
               "kmoe_adapter_inner: %d adapters of rank %d (a multiple of 8, at most %d)", n, rank, KMOE_MAX_RANK);
  if (T == 0) return KMOE_OK;
  KMOE_REQUIRE(x && ids && a && v && !a2 == !v2, KMOE_ERR_NULL, "kmoe_adapter_inner: null buffer");
  KMOE_REQUIRE(aligned(x) && aligned(a) && aligned(v) && aligned(a2) && aligned(v2), KMOE_ERR_SHAPE,
               "kmoe_adapter_inner: buffers are aligned to 16 bytes");
  KMOE_REQUIRE(K < 1 << 22, KMOE_ERR_SHAPE, "kmoe_adapter_inner: rows of %d values (below 2^22)", K);
  Shrink g{static_cast<const uint16_t*>(x), T, K, ids, n, rank, a2 ? 2 : 1,
           {static_cast<const uint16_t*>(a), static_cast<const uint16_t*>(a2)}, {scale, scale2},
           {static_cast<uint16_t*>(v), static_cast<uint16_t*>(v2)}};
  const int64_t tiles = kmoe::ceil_div<int64_t>(T, 16);
  int64_t y = kmoe::ceil_div<int64_t>(1024, tiles);
  y = y < 16 ? y : 16;
  y = y < n ? y : n;
  const int blocks = kmoe::ceil_div(rank, 16);
  // (blocks of ranks side by side read x again each: up to a place for every workgroup)
  const int rb = tiles * y * blocks * g.sides <= 2 * kmoe::cu_count() || blocks == 1 ? 1 : blocks == 2 ? 2 : 4;
  const dim3 grid((unsigned)tiles, (unsigned)y, kmoe::ceil_div(blocks, rb) * g.sides), block(SW * 64);
  hipStream_t s = kmoe::as_stream(stream);
  if (rb == 1)
    hipLaunchKernelGGL((shrink_kernel<1, 4>), grid, block, 0, s, g);
  else if (rb == 2)
    hipLaunchKernelGGL((shrink_kernel<2, 4>), grid, block, 0, s, g);
  else
    hipLaunchKernelGGL((shrink_kernel<4, 2>), grid, block, 0, s, g);
  return kmoe::check_launch("kmoe_adapter_inner");
}

extern "C" size_t kmoe_adapter_grad_workspace_bytes(int64_t T, int n, int rank, int C) {
  if (T <= 0 || n <= 0 || rank <= 0 || C <= 0) return 0;
  const int64_t runs = runs_of(T, n, C);
  return runs > 1 ? (size_t)runs * n * rank * C * sizeof(float) : 0;
}

extern "C" int kmoe_adapter_grad(const void* l, const void* m, int64_t T, const int32_t* ids, int n, int rank, int C,
                                 int outer, void* out, void* workspace, size_t workspace_bytes, void* stream) {
  KMOE_REQUIRE(T >= 0 && T < ((int64_t)1 << 31) && C > 0 && C % 8 == 0, KMOE_ERR_SHAPE,
               "kmoe_adapter_grad: %lld rows of %d values (a positive multiple of 8)", (long long)T, C);
  KMOE_REQUIRE(n > 0 && n <= 65535 && rank > 0 && rank <= KMOE_MAX_RANK && rank % 8 == 0, KMOE_ERR_SHAPE,
               "kmoe_adapter_grad: %d adapters (at most 65535) of rank %d (a multiple of 8, at most %d)", n, rank,
               KMOE_MAX_RANK);
  KMOE_REQUIRE(out && (T == 0 || (l && m && ids)), KMOE_ERR_NULL, "kmoe_adapter_grad: null buffer");
  KMOE_REQUIRE(aligned(l) && aligned(m) && aligned(out) && aligned(workspace), KMOE_ERR_SHAPE,
               "kmoe_adapter_grad: buffers are aligned to 16 bytes");
  KMOE_REQUIRE(workspace_bytes >= kmoe_adapter_grad_workspace_bytes(T, n, rank, C), KMOE_ERR_WORKSPACE,
               "kmoe_adapter_grad: workspace of %zu bytes, %zu are needed", workspace_bytes,
               kmoe_adapter_grad_workspace_bytes(T, n, rank, C));
  const int64_t runs = T > 0 ? runs_of(T, n, C) : 1;
  KMOE_REQUIRE(runs <= 65535, KMOE_ERR_SHAPE, "kmoe_adapter_grad: %lld rows", (long long)T);
  // (a run is whole groups: a wave looks at two of them at a time)
  const int64_t run = kmoe::ceil_div<int64_t>(kmoe::ceil_div<int64_t>(T, runs), 64) * 64;
  FactorGrad g{static_cast<const uint16_t*>(l), static_cast<const uint16_t*>(m), ids, T, run, n, rank, C, (int)runs,
               static_cast<float*>(workspace), static_cast<uint16_t*>(out)};
  const dim3 grid((unsigned)kmoe::ceil_div(C, GC), (unsigned)n, (unsigned)runs), block(256);
  hipStream_t s = kmoe::as_stream(stream);
  const int rb = kmoe::ceil_div(rank, 16);
#define KMOE_FACTOR(RB)                                                            \
  do {                                                                             \
    if (outer)                                                                     \
      hipLaunchKernelGGL((factor_grad_kernel<RB, true>), grid, block, 0, s, g);    \
    else                                                                           \
      hipLaunchKernelGGL((factor_grad_kernel<RB, false>), grid, block, 0, s, g);   \
  } while (0)
  if (rb == 1)
    KMOE_FACTOR(1);
  else if (rb == 2)
    KMOE_FACTOR(2);
  else if (rb <= 4)
    KMOE_FACTOR(4);
  else
    KMOE_FACTOR(8);
#undef KMOE_FACTOR
  int rc = kmoe::check_launch("kmoe_adapter_grad");
  if (rc != KMOE_OK || runs == 1) return rc;
  const int64_t total = (int64_t)n * rank * C;
  return kmoe_dense::launch_sum_runs(g.part, (int)runs, total, g.out, s);
}
