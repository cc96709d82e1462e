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
// product's MFMAs, one rounding (half a step of 2^-8) of a term that adds to the projection's.  What
// it loses is kept behind, for the factors' gradients, of which it is the whole operand.
// A workgroup takes 16 rows, RB blocks of 16 ranks and every gridDim.y-th of the adapters that the rows
// have (few rows with an adapter each: a workgroup an adapter); its W waves share K.  Rows that have
// another adapter than the one in turn read as zeros, for nothing (512 rows with 16 adapters in
// turn, rank 16: 13.8 us; read and not kept 20).  Bound by reading x and the adapters and by latency, not
// by the products; few rows take a workgroup a block of ranks.  K 2048, rank 16: one row 5 us, 48
// rows with an adapter each 7; 4099 rows of prompts, rank 32, 14.5 (x alone 3.5 at HBM's rate).
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

template <int RB, int W, int D>
__global__ __launch_bounds__(W * 64) void shrink_kernel(Shrink g) {
  __shared__ f32x4_t part[W][RB][64];
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
  Stream16<RB, W, D> st;
  st.x = g.x + t0 * g.K, st.K = g.K;
#pragma unroll
  for (int b = 0; b < RB; ++b) {
    const int j = j0 + b * 16 + l16;
    st.woff[b] = j < g.r ? (uint32_t)(j * g.K) * 2 : NOWHERE;
  }
  for (int c = 0; todo; ++c, todo &= todo - 1) {
    if (c % (int)gridDim.y != (int)blockIdx.y) continue;
    const int cur = __builtin_amdgcn_readlane(id, __builtin_ctzll(todo));
    st.xoff = id == cur ? (uint32_t)(l16 * g.K) * 2 : NOWHERE;
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
      for (int w = 1; w < W; ++w) s += part[w][wave][lane];
      const int j = j0 + wave * 16 + 4 * lq;
      if (id == cur && j < g.r) {
        const float f = g.scale[z] ? g.scale[z][cur] : 1.0f;
        const float o[4] = {f * s[0], f * s[1], f * s[2], f * s[3]};
        const i32x2_t w = pack4(o[0], o[1], o[2], o[3]);
        uint16_t* const to = g.v[z] + (t0 + l16) * g.r + j;
        *reinterpret_cast<i32x2_t*>(to) = w;
        kmoe_dense::store_lost(to + g.T * g.r, o, w);
      }
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------- gradients of the factors
// out[i][j, c] = sum over rows t with ids[t] = i of l[t, j] m[t, c], l (2, T, r) (the second T rows what the
// first lost by their rounding), m (T, C), f32 sums.
// A workgroup takes an adapter, 128 columns (32 a wave) and a run of rows; of the run it visits the
// groups of 32 rows in which the adapter occurs, other rows in them read as zeros in both
// operands.  Operands along t come from LDS by transposing reads, a group's while the next one's rows
// are on their way.  Runs of rows are summed by a second kernel, in order.  `outer`: out[i] is
// (C, r), the outer factor's, instead of (r, C).  Both factors' gradients share a launch; each
// reads its m once, which bounds it (2042 rows, 4 adapters of rank 16, C 2048 and 2816: 15 us and 4 for
// the sum of runs).
constexpr int GC = 128, GR = 32;     // columns of a workgroup, rows of a group
constexpr int GMAXRUN = 64 * 1024;   // rows of a run at most: a bit a group in LDS

struct FactorJob {
  const uint16_t* l;
  const uint16_t* m;
  uint16_t* out;
  int64_t first;   // of its partial sums among a run's
  int C, blocks, outer;
};
struct FactorGrad {
  FactorJob job[2];  // the second one's blocks come after the first one's
  const int32_t* ids;
  int64_t T, run, total;  // total: values of a run's partial sums
  int n, r, runs;
  float* part;            // (runs, total) when runs > 1
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
__device__ __forceinline__ void factor_grad(const FactorGrad& g, const FactorJob& job, int block, uint8_t* lds, uint32_t* occurs) {
  constexpr int LROWB = RB * 32, MROWB = GC * 2, LT = GR * LROWB, STAGE = 2 * LT + GR * MROWB;
  constexpr int NL = RB > 2 ? RB / 2 : 1;  // 16-byte pieces of l a thread holds (of m: 2)
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, lq = lane >> 4;
  const int c0 = block * GC, me = blockIdx.y;
  const int64_t r0 = (int64_t)blockIdx.z * g.run, r1 = r0 + g.run < g.T ? r0 + g.run : g.T;
  const int groups = r1 > r0 ? (int)((r1 - r0 + GR - 1) / GR) : 0, words = (groups + 31) / 32;
  for (int w = tid; w < words; w += 256) occurs[w] = 0;
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
  int word = -1;
  uint32_t bits = 0;
  auto next_group = [&]() -> int64_t {  // its first row, -1 past the last one
    while (!bits && ++word < words) bits = __builtin_amdgcn_readfirstlane(occurs[word]);
    if (!bits) return -1;
    const int64_t t0 = r0 + (int64_t)(word * 32 + __builtin_ctz(bits)) * GR;
    bits &= bits - 1;
    return t0;
  };
  i32x4_t mv[2], lv[NL];
  int mid[2], lid[NL];
  auto row_at = [&](int64_t t) { return t < r1 ? t : r1 - 1; };
  auto fetch = [&](int64_t t0) {  // 32 rows x 16 pieces of m, 64 x 2 RB of l (those not to be used are some row's)
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int64_t t = t0 + (tid >> 4) + 16 * q, at = row_at(t);
      const int c = c0 + (tid & 15) * 8;
      mid[q] = t < r1 && c < job.C ? g.ids[at] : -1;
      mv[q] = *reinterpret_cast<const i32x4_t*>(job.m + at * job.C + (c < job.C ? c : 0));
    }
#pragma unroll
    for (int q = 0; q < NL; ++q) {
      const int e = tid + 256 * q, j = e % (2 * RB) * 8;
      const int64_t t = t0 + e / (2 * RB) % GR, at = row_at(t);
      lid[q] = t < r1 && j < g.r ? g.ids[at] : -1;
      lv[q] = *reinterpret_cast<const i32x4_t*>(job.l + (at + (e < GR * 2 * RB ? 0 : g.T)) * g.r + (j < g.r ? j : 0));
    }
  };
  int64_t t0 = next_group();
  if (t0 >= 0) fetch(t0);
  for (int stage = 0; t0 >= 0; stage ^= 1) {
    uint8_t* const lt = lds + stage * STAGE;
    uint8_t* const mt = lt + 2 * LT;
    const i32x4_t zero{0, 0, 0, 0};
#pragma unroll
    for (int q = 0; q < 2; ++q)
      *reinterpret_cast<i32x4_t*>(mt + gpos<MROWB>((tid >> 4) + 16 * q, (tid & 15) * 8)) = mid[q] == me ? mv[q] : zero;
#pragma unroll
    for (int q = 0; q < NL; ++q) {
      const int e = tid + 256 * q;
      if (e < 2 * GR * 2 * RB)
        *reinterpret_cast<i32x4_t*>(lt + e / (GR * 2 * RB) * LT + gpos<LROWB>(e / (2 * RB) % GR, e % (2 * RB) * 8)) =
            lid[q] == me ? lv[q] : zero;
    }
    t0 = next_group();
    if (t0 >= 0) fetch(t0);
    __syncthreads();  // (the stage before this one is written again past the next one)
    bf16x8_t fm[2];
#pragma unroll
    for (int y = 0; y < 2; ++y) fm[y] = gfrag<MROWB>(mt, wave * 32 + y * 16, lane);
#pragma unroll
    for (int b = 0; b < 2 * RB; ++b) {
      const bf16x8_t fl = gfrag<LROWB>(lt + b / RB * LT, b % RB * 16, lane);
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        f32x4_t& a = acc[b % RB][y];
        a = OUTER ? __builtin_amdgcn_mfma_f32_16x16x32_bf16(fl, fm[y], a, 0, 0, 0)
                  : __builtin_amdgcn_mfma_f32_16x16x32_bf16(fm[y], fl, a, 0, 0, 0);
      }
    }
  }
  // OUTER: a lane holds column l % 16, ranks 4 (l / 16) .. + 3; else rank l % 16, four columns
  const int64_t size = (int64_t)g.r * job.C;
#pragma unroll
  for (int b = 0; b < RB; ++b)
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      const int c = c0 + wave * 32 + y * 16 + (OUTER ? l16 : 4 * lq), j = b * 16 + (OUTER ? 4 * lq : l16);
      if (c >= job.C || j >= g.r) continue;
      const int64_t at = me * size + (OUTER ? (int64_t)c * g.r + j : (int64_t)j * job.C + c);
      const f32x4_t v = acc[b][y];
      if (g.runs > 1)
        *reinterpret_cast<f32x4_t*>(g.part + blockIdx.z * g.total + job.first + at) = v;
      else
        *reinterpret_cast<i32x2_t*>(job.out + at) = pack4(v[0], v[1], v[2], v[3]);
    }
}

template <int RB>
__global__ __launch_bounds__(256) void factor_grad_kernel(FactorGrad g) {
  __shared__ __attribute__((aligned(16))) uint8_t lds[2 * GR * (2 * RB * 32 + GC * 2)];
  __shared__ uint32_t occurs[GMAXRUN / GR / 32];
  const bool second = (int)blockIdx.x >= g.job[0].blocks;
  const FactorJob& job = g.job[second];
  const int block = blockIdx.x - (second ? g.job[0].blocks : 0);
  if (job.outer)
    factor_grad<RB, true>(g, job, block, lds, occurs);
  else
    factor_grad<RB, false>(g, job, block, lds, occurs);
}

// out0 takes the first n0 values of the sums, out1 those after them
__global__ __launch_bounds__(256) void sum_runs_kernel(const float* __restrict__ part, int runs, int64_t total, int64_t n0,
                                                       uint16_t* __restrict__ out0, uint16_t* __restrict__ out1) {
  const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (at >= total) return;
  f32x4_t s = *reinterpret_cast<const f32x4_t*>(part + at);
  for (int k = 1; k < runs; ++k) s += *reinterpret_cast<const f32x4_t*>(part + (int64_t)k * total + at);
  *reinterpret_cast<i32x2_t*>(at < n0 ? out0 + at : out1 + (at - n0)) = pack4(s[0], s[1], s[2], s[3]);
}

// dst[i] (C, R) = src[i] (R, C) transposed, for both of an adapter's factors in one launch: those that the
// backward reads the other way round.
struct Turn {
  const uint16_t* src[2];
  uint16_t* dst[2];
  int R[2], C[2], n;
};
__global__ __launch_bounds__(256) void turn_kernel(Turn g) {
  __shared__ uint16_t tile[64][66];
  const int which = (int)blockIdx.y >= g.n, i = blockIdx.y - which * g.n, tid = threadIdx.x;
  const int R = g.R[which], C = g.C[which], nc = (C + 63) / 64;
  const int r0 = (int)(blockIdx.x / nc) * 64, c0 = (int)(blockIdx.x % nc) * 64;
  if (r0 >= R) return;
  const uint16_t* const src = g.src[which] + (int64_t)i * R * C;
  uint16_t* const dst = g.dst[which] + (int64_t)i * R * C;
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int r = tid / 8 + 32 * q, c = tid % 8 * 8;
    if (r0 + r < R && c0 + c < C) {
      const i32x4_t v = *reinterpret_cast<const i32x4_t*>(src + (int64_t)(r0 + r) * C + c0 + c);
#pragma unroll
      for (int k = 0; k < 8; ++k) tile[r][c + k] = (uint16_t)((uint32_t)v[k / 2] >> (16 * (k % 2)));
    }
  }
  __syncthreads();
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int c = tid / 8 + 32 * q, r = tid % 8 * 8;
    if (c0 + c < C && r0 + r < R) {
      i32x4_t v;
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = (int)(tile[r + 2 * k][c] | (uint32_t)tile[r + 2 * k + 1][c] << 16);
      *reinterpret_cast<i32x4_t*>(dst + (int64_t)(c0 + c) * R + r0 + r) = v;
    }
  }
}

// The runs of rows in which a launch computes the gradients of factors of C and C2 columns (C2 = 0: of
// one factor), and the bytes of their partial sums: as many runs as give every compute unit two
// workgroups, of at least 256 rows.  One factor alone has fewer blocks, so it may take more runs than both.
struct Runs {
  int64_t n;
  size_t bytes;
};
Runs runs_of(int64_t T, int n, int rank, int C, int C2) {
  if (T <= 0) return {1, 0};
  const int64_t blocks = (int64_t)n * (kmoe::ceil_div(C, GC) + kmoe::ceil_div(C2, GC));
  int64_t runs = kmoe::ceil_div<int64_t>(512, blocks);
  runs = runs < kmoe::ceil_div<int64_t>(T, 256) ? runs : kmoe::ceil_div<int64_t>(T, 256);
  const int64_t least = kmoe::ceil_div<int64_t>(T, GMAXRUN);
  runs = runs > least ? runs : (least > 1 ? least : 1);
  return {runs, runs > 1 ? (size_t)runs * n * rank * ((size_t)C + C2) * sizeof(float) : 0};
}

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace

int kmoe_dense::launch_sum_runs(const float* part, int runs, int64_t total, uint16_t* out, hipStream_t s) {
  hipLaunchKernelGGL(sum_runs_kernel, dim3((unsigned)kmoe::ceil_div<int64_t>(total, 1024)), dim3(256), 0, s, part, runs, total,
                     total, out, out);
  return kmoe::check_launch("kmoe sum of runs");
}

int kmoe_dense::adapter_inner(const void* x, int64_t T, int K, const int32_t* ids, int n, int rank, const void* a,
                              const float* scale, void* v, const void* a2, const float* scale2, void* v2, void* stream) {
  KMOE_REQUIRE(K < 1 << 22, KMOE_ERR_SHAPE, "kmoe adapters: rows of %d values (below 2^22)", K);
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
  const dim3 grid((unsigned)tiles, (unsigned)y, kmoe::ceil_div(blocks, rb) * g.sides);
  hipStream_t s = kmoe::as_stream(stream);
  if (rb == 1)
    hipLaunchKernelGGL((shrink_kernel<1, 8, 4>), grid, dim3(512), 0, s, g);
  else if (rb == 2)
    hipLaunchKernelGGL((shrink_kernel<2, 8, 2>), grid, dim3(512), 0, s, g);
  else
    hipLaunchKernelGGL((shrink_kernel<4, 8, 2>), grid, dim3(512), 0, s, g);
  return kmoe::check_launch("kmoe adapters");
}

namespace {

size_t piece(int64_t bytes) { return (size_t)((bytes + 255) / 256 * 256); }

// Of both factors or of either one alone, whichever takes most.
size_t grads_bytes(int64_t T, int n, int rank, int K, int N) {
  const size_t both = runs_of(T, n, rank, K, N).bytes, inner = runs_of(T, n, rank, K, 0).bytes,
               outer = runs_of(T, n, rank, N, 0).bytes, one = inner > outer ? inner : outer;
  return both > one ? both : one;
}

// The gradients of up to two factors (C2 = 0: one) of adapters with rows ids.
int factor_grads(FactorGrad g, int C, int C2, void* workspace, size_t workspace_bytes, hipStream_t s) {
  const auto [runs, bytes] = runs_of(g.T, g.n, g.r, C, C2);
  KMOE_REQUIRE(bytes <= workspace_bytes, KMOE_ERR_WORKSPACE,
               "kmoe_adapted_linear_backward: %zu bytes are left for partial sums, %zu are needed", workspace_bytes, bytes);
  KMOE_REQUIRE(runs <= 65535, KMOE_ERR_SHAPE, "kmoe_adapted_linear_backward: %lld rows", (long long)g.T);
  // (a run is whole groups: a wave looks at two of them at a time)
  g.run = kmoe::ceil_div<int64_t>(kmoe::ceil_div<int64_t>(g.T, runs), 64) * 64;
  g.runs = (int)runs, g.part = static_cast<float*>(workspace);
  const int64_t first = (int64_t)g.n * g.r * C;
  g.job[0].C = C, g.job[0].blocks = kmoe::ceil_div(C, GC), g.job[0].first = 0;
  g.job[1].C = C2, g.job[1].blocks = kmoe::ceil_div(C2, GC), g.job[1].first = first;
  g.total = first + (int64_t)g.n * g.r * C2;
  const dim3 grid((unsigned)(g.job[0].blocks + g.job[1].blocks), (unsigned)g.n, (unsigned)runs), block(256);
  const int rb = kmoe::ceil_div(g.r, 16);
  if (rb == 1)
    hipLaunchKernelGGL(factor_grad_kernel<1>, grid, block, 0, s, g);
  else if (rb == 2)
    hipLaunchKernelGGL(factor_grad_kernel<2>, grid, block, 0, s, g);
  else if (rb <= 4)
    hipLaunchKernelGGL(factor_grad_kernel<4>, grid, block, 0, s, g);
  else
    hipLaunchKernelGGL(factor_grad_kernel<8>, grid, block, 0, s, g);
  const int rc = kmoe::check_launch("kmoe_adapted_linear_backward");
  if (rc != KMOE_OK || runs == 1) return rc;
  hipLaunchKernelGGL(sum_runs_kernel, dim3((unsigned)kmoe::ceil_div<int64_t>(g.total, 1024)), dim3(256), 0, s, g.part, (int)runs,
                     g.total, first, g.job[0].out, g.job[1].out);
  return kmoe::check_launch("kmoe_adapted_linear_backward");
}

}  // namespace

extern "C" size_t kmoe_adapted_linear_backward_workspace_bytes(int64_t T, int K, int N, int n_adapters, int rank) {
  if (T < 0 || K <= 0 || N <= 0 || n_adapters <= 0 || rank <= 0) return 0;
  return piece(T * rank * 4) + piece((int64_t)n_adapters * rank * K * 2) + piece((int64_t)n_adapters * rank * N * 2) +
         grads_bytes(T, n_adapters, rank, K, N);
}

extern "C" int kmoe_adapted_linear_backward(const void* dy, const void* x, int64_t T, int K, const void* w, int N,
                                            const int32_t* ids, int n_adapters, const kmoe_adapter* adapter, const void* v,
                                            void* dx, void* da, void* db, void* workspace, size_t workspace_bytes,
                                            void* stream) {
  KMOE_REQUIRE(T >= 0 && T <= kmoe_dense::ADAPTED_ROWS && K > 0 && N > 0 && K % 8 == 0 && N % 8 == 0, KMOE_ERR_SHAPE,
               "kmoe_adapted_linear_backward: %lld rows (at most %lld) of %d and %d values (positive multiples of 8)", (long long)T,
               (long long)kmoe_dense::ADAPTED_ROWS, K, N);
  KMOE_REQUIRE(adapter && adapter->a && adapter->b, KMOE_ERR_NULL, "kmoe_adapted_linear_backward: null adapter buffer");
  const int r = adapter->rank;
  KMOE_REQUIRE(n_adapters > 0 && n_adapters <= 32767 && r > 0 && r <= KMOE_MAX_RANK && r % 8 == 0, KMOE_ERR_SHAPE,
               "kmoe_adapted_linear_backward: %d adapters (at most 32767) of rank %d (a multiple of 8, at most %d)", n_adapters, r,
               KMOE_MAX_RANK);
  KMOE_REQUIRE(T == 0 || (dy && x && w && ids && (v || !db)), KMOE_ERR_NULL, "kmoe_adapted_linear_backward: null buffer");
  for (const void* p : {dy, x, w, adapter->a, adapter->b, v, (const void*)dx, (const void*)da, (const void*)db,
                        (const void*)workspace})
    KMOE_REQUIRE(aligned(p), KMOE_ERR_SHAPE, "kmoe_adapted_linear_backward: buffers are aligned to 16 bytes");
  const size_t need = kmoe_adapted_linear_backward_workspace_bytes(T, K, N, n_adapters, r);
  KMOE_REQUIRE((workspace || !need) && workspace_bytes >= need, KMOE_ERR_WORKSPACE,
               "kmoe_adapted_linear_backward: workspace of %zu bytes, %zu are needed", workspace_bytes, need);
  uint8_t* at = static_cast<uint8_t*>(workspace);
  uint16_t* const u = reinterpret_cast<uint16_t*>(at);
  uint16_t* const bt = reinterpret_cast<uint16_t*>(at += piece(T * r * 4));
  uint16_t* const a_t = reinterpret_cast<uint16_t*>(at += piece((int64_t)n_adapters * r * N * 2));
  void* const part = at + piece((int64_t)n_adapters * r * K * 2);
  hipStream_t s = kmoe::as_stream(stream);
  if (T > 0 && (dx || da)) {
    Turn g{{static_cast<const uint16_t*>(adapter->b), static_cast<const uint16_t*>(adapter->a)}, {bt, a_t}, {N, r}, {r, K},
           n_adapters};
    const int nr = kmoe::ceil_div(r, 64), blocks = nr * kmoe::ceil_div(N > K ? N : K, 64);
    hipLaunchKernelGGL(turn_kernel, dim3((unsigned)blocks, (unsigned)(dx ? 2 * n_adapters : n_adapters)), dim3(256), 0, s, g);
    if (const int rc = kmoe::check_launch("kmoe_adapted_linear_backward")) return rc;
    if (const int rc = kmoe_dense::adapter_inner(dy, T, N, ids, n_adapters, r, bt, adapter->scale, u, nullptr, nullptr, nullptr, stream))
      return rc;
  }
  if (T > 0 && dx) {
    kmoe_dense::Args g{};
    g.a[0] = static_cast<const uint16_t*>(dy), g.b[0] = static_cast<const uint16_t*>(w);
    g.K = N, g.lda = N, g.ldb = K, g.M = T, g.N = K, g.ldc = K, g.c = dx;
    g.ad = {ids, {u, nullptr}, {a_t, nullptr}, n_adapters, r};
    if (const int rc = kmoe_dense::launch_dx_adapt(g, s)) return rc;
  }
  if (!da && !db) return KMOE_OK;
  FactorGrad g{};
  FactorJob inner{u, static_cast<const uint16_t*>(x), static_cast<uint16_t*>(da), 0, 0, 0, 0};
  FactorJob outer{static_cast<const uint16_t*>(v), static_cast<const uint16_t*>(dy), static_cast<uint16_t*>(db), 0, 0, 0, 1};
  g.ids = ids, g.T = T, g.n = n_adapters, g.r = r;
  g.job[0] = da ? inner : outer, g.job[1] = outer;
  return factor_grads(g, da ? K : N, da && db ? N : 0, part,
                      workspace_bytes - (static_cast<uint8_t*>(part) - static_cast<uint8_t*>(workspace)), s);
}
