// Routed tokens through the microscaled experts as one call: dispatch, row quantisation, the
// two products and the combine launched from here, their intermediates in one workspace.
// From Python the five calls, their argument conversions and a dozen allocations took 66 us a
// pass at one token, more than the kernels.
#include "kmoe_mx.h"

using namespace kmoe_mx;

namespace {

constexpr int FEW = 1024;  // threads of the workgroup that dispatches
constexpr int MAX_ROUNDS = 4;
// Rounds of FEW assignments that one workgroup dispatches: an expert and round cost a ballot.  A
// whole pass with this dispatch / with kmoe_dispatch and the quantisation, us: 16 experts, 96
// assignments 18.4 / 23.7, 1536 27.2 / 31.9, 3000 37.7 / 38.9, 4080 47.4 / 46.7; 8 experts, 4080
// 44.7 / 46.0; 32 experts, 2000 27.8 / 30.4, 3000 33.2 / 31.1; 64 experts, 2000 34.6 / 38.8.
int few_rounds(int E) { return E <= 16 ? MAX_ROUNDS : 2; }

// Dispatch of at most R FEW assignments (the tables of kmoe_dispatch, same order) by workgroup
// 0, the quantisation of the T rows x[row_index[t]] by the others: one launch in place of
// three, whose latencies are the time at these sizes.  A thread holds assignments R tid ..
// R tid + R - 1; a rank is counted by ballots in its wave and summed over the waves before it.
// 96 assignments of 16 experts and 48 x 2048 rows 4.0 us (kmoe_dispatch and the quantisation 8.0),
// 1554 and 777 6.2 (9.1).
template <bool FP4, int R>
__global__ __launch_bounds__(FEW) void tables_kernel(const int64_t* __restrict__ idx, const void* __restrict__ wsrc,
                                                     bool w_f32, int T, int k, int E, int64_t capacity,
                                                     int32_t* __restrict__ counts, int32_t* __restrict__ offsets,
                                                     int32_t* __restrict__ row_token, int32_t* __restrict__ slot_row,
                                                     float* __restrict__ slot_w, const uint16_t* __restrict__ x,
                                                     const int32_t* __restrict__ row_index, int d, uint8_t* __restrict__ q,
                                                     uint8_t* __restrict__ scale) {
  const int tid = threadIdx.x;
  if (blockIdx.x > 0) {
    const int dp = round_up(d, STEP), cpr = dp / 8;
    const int64_t i = (int64_t)(blockIdx.x - 1) * FEW + tid;
    if (i >= (int64_t)T * cpr) return;  // a multiple of 16: blocks of four lanes stay whole
    const int64_t t = i / cpr;
    const int c = (int)(i - t * cpr);
    float v[8] = {};
    const int64_t src = row_index ? (int64_t)row_index[t] : t;
    if (c * 8 < d && src >= 0) unpack8(*reinterpret_cast<const i32x4_t*>(x + src * d + c * 8), v);
    uint32_t code;
    const Codes<FP4, 8> o = encode_quad<FP4>(v, code);
    if constexpr (FP4)
      *reinterpret_cast<uint32_t*>(q + t * (dp / 2) + c * 4) = o.w[0];
    else
      *reinterpret_cast<i32x2_t*>(q + t * dp + c * 8) = i32x2_t{(int)o.w[0], (int)o.w[1]};
    if ((c & 3) == 0) scale[t * scale_bytes(d) + c / 4] = (uint8_t)code;
    return;
  }
  constexpr int NW = FEW / 64;
  __shared__ int cnt[NW][KMOE_MAX_EXPERTS];
  __shared__ int off[KMOE_MAX_EXPERTS];
  const int lane = tid & 63, wave = tid >> 6, A = T * k;
  int e[R], rank[R];
  float w[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int a = tid * R + r;
    e[r] = -1;
    rank[r] = 0;
    w[r] = 0.0f;
    if (a < A) {
      const int64_t v = idx[a];
      e[r] = v >= 0 && v < E ? (int)v : -1;  // ids out of range are dropped
      w[r] = w_f32 ? static_cast<const float*>(wsrc)[a] : bf16_to_f32(static_cast<const uint16_t*>(wsrc)[a]);
    }
  }
  const uint64_t before = lane == 0 ? 0ull : ~0ull >> (64 - lane);
  for (int ee = 0; ee < E; ++ee) {
    int at = 0, all = 0;  // of the lanes before, of the wave
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const uint64_t m = __ballot(e[r] == ee);
      at += __popcll(m & before);
      all += __popcll(m);
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (e[r] == ee) rank[r] = at++;
    if (lane == 0) cnt[wave][ee] = all;
  }
  __syncthreads();
  if (wave == 0) {
    // lane: an expert; cnt becomes the count of the waves before
    int c = 0;
    if (lane < E) {
      int n[NW];
#pragma unroll
      for (int v = 0; v < NW; ++v) n[v] = cnt[v][lane];
#pragma unroll
      for (int v = 0; v < NW; ++v) {
        cnt[v][lane] = c;
        c += n[v];
      }
    }
    const int kept = capacity > 0 && c > capacity ? (int)capacity : c;
    int incl = kept;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int u = __shfl_up(incl, o, 64);
      if (lane >= o) incl += u;
    }
    if (lane < E) {
      off[lane] = incl - kept;
      counts[lane] = c;
      offsets[lane] = incl - kept;
    }
    if (lane == E - 1) offsets[E] = incl;
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int a = tid * R + r;
    if (a < A) {
      int row = -1;
      if (e[r] >= 0) {
        const int at = rank[r] + cnt[wave][e[r]];
        if (capacity <= 0 || at < capacity) {
          row = off[e[r]] + at;
          row_token[row] = a / k;
        }
      }
      slot_row[a] = row;
      slot_w[a] = w[r];
    }
  }
}

// Buffers of one call in the workspace, 256-byte aligned.  yperm, the experts' rows of y, is bf16 as the
// other experts' is: 2 bytes a value written and read (at 16384 tokens, top-2, d 2048 f32 rows
// would add 256 MiB, about 55 us of 523) for one rounding more, 0.0024 relative to 64 bits in place of 0.0017.
struct Buffers {
  size_t offsets, row_token, slot_row, slot_w, dispatch, xq, xs, hq, hs, yperm, total;
};
Buffers layout(int64_t T, int d, int E, int k, int F, bool fp4, bool coded) {
  Buffers b{};
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t p = at;
    at += (bytes + 255) / 256 * 256;
    return p;
  };
  const size_t A = (size_t)T * k;
  b.offsets = take((size_t)(E + 1) * 4);
  b.row_token = take(A * 4);
  b.slot_row = take(A * 4);
  b.slot_w = take(A * 4);
  b.dispatch = take(kmoe_dispatch_workspace_bytes(T, k, E));
  b.xq = take(coded ? 0 : (size_t)T * row_bytes(fp4, d));
  b.xs = take(coded ? 0 : (size_t)T * scale_bytes(d));
  b.hq = take(A * row_bytes(fp4, F));
  b.hs = take(A * scale_bytes(F));
  b.yperm = take(A * (size_t)d * 2);
  b.total = at;
  return b;
}
bool valid(int64_t T, int d, int E, int k, int F, int fmt) {
  return T > 0 && T <= (int64_t)1 << 31 && d > 0 && d % 64 == 0 && E >= 1 && E <= KMOE_MAX_EXPERTS && k >= 1 && k <= 8 &&
         k <= E && F > 0 && T * k < (int64_t)1 << 31 && (fmt == KMOE_DTYPE_FP8_E4M3 || fmt == KMOE_DTYPE_FP4_E2M1);
}

}  // namespace

extern "C" size_t kmoe_mx_experts_workspace_bytes(int64_t T, int d, int E, int k, int F, int fmt, int coded) {
  return valid(T, d, E, k, F, fmt) ? layout(T, d, E, k, F, fmt == KMOE_DTYPE_FP4_E2M1, coded != 0).total : 0;
}

extern "C" int kmoe_mx_experts(const void* x, const int32_t* row_index, int64_t T, int d, int fmt, const void* xq,
                               const uint8_t* x_scale, const int64_t* topk_idx, const void* topk_w, int w_dtype, int k,
                               int E, int64_t capacity, const int32_t* block_counts, const float* partials, float w_lb,
                               float w_z, float* aux_out, const void* w13_packed, const uint8_t* w13_scale,
                               const void* w3_packed, const uint8_t* w3_scale, int F, const int32_t* out_map,
                               const float* out_scale, const void* residual, int64_t T_out, void* y, int y_dtype,
                               int32_t* counts, void* workspace, size_t workspace_bytes, void* stream) {
  KMOE_REQUIRE(x && topk_idx && topk_w && w13_packed && w13_scale && w3_packed && w3_scale && counts && workspace &&
                   (y || T_out == 0),
               KMOE_ERR_NULL, "kmoe_mx_experts: null buffer");
  KMOE_REQUIRE(valid(T, d, E, k, F, fmt), KMOE_ERR_SHAPE, "kmoe_mx_experts: T=%lld d=%d E=%d k=%d F=%d fmt=%d", (long long)T,
               d, E, k, F, fmt);
  KMOE_REQUIRE(w_dtype == KMOE_DTYPE_BF16 || w_dtype == KMOE_DTYPE_F32, KMOE_ERR_DTYPE, "kmoe_mx_experts: topk_w dtype %d",
               w_dtype);
  KMOE_REQUIRE(!xq == !x_scale && (!xq || !row_index), KMOE_ERR_NULL,
               "kmoe_mx_experts: xq and x_scale go together, without row_index");
  KMOE_REQUIRE(!aux_out || (block_counts && partials), KMOE_ERR_NULL, "kmoe_mx_experts: aux losses need block_counts, partials");
  KMOE_REQUIRE(out_map || T_out == T, KMOE_ERR_SHAPE, "kmoe_mx_experts: T_out=%lld without out_map", (long long)T_out);
  const bool fp4 = fmt == KMOE_DTYPE_FP4_E2M1;
  const Buffers b = layout(T, d, E, k, F, fp4, xq != nullptr);
  KMOE_REQUIRE(workspace_bytes >= b.total, KMOE_ERR_WORKSPACE, "kmoe_mx_experts: workspace %zu < %zu bytes",
               workspace_bytes, b.total);
  uint8_t* const ws = static_cast<uint8_t*>(workspace);
  auto i32 = [&](size_t at) { return reinterpret_cast<int32_t*>(ws + at); };
  float* const slot_w = reinterpret_cast<float*>(ws + b.slot_w);
  const int64_t A = T * k;
  const bool quant = !xq;
  int rc;
  if (A <= (int64_t)FEW * few_rounds(E) && !aux_out) {
    const int64_t chunks = quant ? T * (round_up(d, STEP) / 8) : 0;
    const dim3 grid((unsigned)(1 + kmoe::ceil_div<int64_t>(chunks, FEW)));
    const uint16_t* xp = static_cast<const uint16_t*>(x);
    hipStream_t s = kmoe::as_stream(stream);
#define KMOE_TABLES(FP4_, R_)                                                                                             \
  hipLaunchKernelGGL((tables_kernel<FP4_, R_>), grid, dim3(FEW), 0, s, topk_idx, topk_w, w_dtype == KMOE_DTYPE_F32, (int)T, k, \
                     E, capacity, counts, i32(b.offsets), i32(b.row_token), i32(b.slot_row), slot_w, xp, row_index, d,       \
                     ws + b.xq, ws + b.xs)
#define KMOE_TABLES_FMT(R_)    \
  if (fp4)                     \
    KMOE_TABLES(true, R_);     \
  else                         \
    KMOE_TABLES(false, R_)
    if (A <= FEW) {
      KMOE_TABLES_FMT(1);
    } else if (A <= 2 * FEW) {
      KMOE_TABLES_FMT(2);
    } else {
      KMOE_TABLES_FMT(MAX_ROUNDS);
    }
#undef KMOE_TABLES_FMT
#undef KMOE_TABLES
    rc = kmoe::check_launch("kmoe_mx_experts");
    if (rc) return rc;
  } else {
    const size_t dws = kmoe_dispatch_workspace_bytes(T, k, E);
    if (aux_out)
      rc = kmoe_dispatch_counted_aux(x, row_index, T, d, topk_idx, topk_w, w_dtype, k, E, capacity, block_counts, counts,
                                     i32(b.offsets), i32(b.row_token), i32(b.slot_row), slot_w, nullptr, KMOE_DTYPE_BF16,
                                     nullptr, ws + b.dispatch, dws, partials, w_lb, w_z, aux_out, stream);
    else if (block_counts)
      rc = kmoe_dispatch_counted(x, row_index, T, d, topk_idx, topk_w, w_dtype, k, E, capacity, block_counts, counts,
                                 i32(b.offsets), i32(b.row_token), i32(b.slot_row), slot_w, nullptr, KMOE_DTYPE_BF16,
                                 nullptr, ws + b.dispatch, dws, stream);
    else
      rc = kmoe_dispatch(x, row_index, T, d, topk_idx, topk_w, w_dtype, k, E, capacity, counts, i32(b.offsets),
                         i32(b.row_token), i32(b.slot_row), slot_w, nullptr, KMOE_DTYPE_BF16, nullptr, ws + b.dispatch,
                         dws, stream);
    if (rc) return rc;
    if (quant) {
      rc = kmoe_quant_rows_mx(x, row_index, T, nullptr, d, fmt, ws + b.xq, ws + b.xs, stream);
      if (rc) return rc;
    }
  }
  rc = kmoe_gemm_gate_up_mx(quant ? ws + b.xq : xq, quant ? ws + b.xs : x_scale, fmt, T, i32(b.row_token), i32(b.offsets), E,
                            d, F, A, w13_packed, w13_scale, ws + b.hq, ws + b.hs, nullptr, stream);
  if (rc) return rc;
  rc = kmoe_gemm_down_mx(ws + b.hq, ws + b.hs, fmt, i32(b.offsets), E, d, F, A, w3_packed, w3_scale, ws + b.yperm, stream);
  if (rc) return rc;
  return kmoe_combine_residual(ws + b.yperm, d, i32(b.slot_row), slot_w, k, out_map, out_scale, residual, T_out, y, y_dtype,
                               stream);
}
