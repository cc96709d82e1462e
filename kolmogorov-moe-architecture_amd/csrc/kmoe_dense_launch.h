// Launches of the dense products, one source file for each kind: their instances compile side by side.
#pragma once

#include "kmoe_dense.h"

namespace kmoe_dense {

int launch_gated(const Args& g, hipStream_t s);         // act(a b0^T) * (a b1^T)
int launch_gated_adapt(const Args& g, hipStream_t s);
int launch_linear(const Args& g, hipStream_t s);        // a b^T
int launch_linear_adapt(const Args& g, hipStream_t s);
int launch_dh(const Args& g, hipStream_t s);            // (a b) p, (a b) q
int launch_dx(const Args& g, hipStream_t s);            // a b
int launch_dx_two(const Args& g, hipStream_t s);        // a0 b0 + a1 b1
int launch_dx_adapt(const Args& g, hipStream_t s);
int launch_wgrad(const Args& g, hipStream_t s);         // a^T b
int launch_wgrad_two(const Args& g, hipStream_t s);     // a0^T b0 + a1^T b1
// a b^T of few rows in runs of K (kmoe_ffn.hip)
int launch_linear_runs(const Args& g, hipStream_t s);
int launch_linear_runs_adapt(const Args& g, hipStream_t s);
// The adapters' rows of one call: a launch of the inner products (a workgroup of 512 a 16 rows) has fewer than
// 2^32 threads.
constexpr int64_t ADAPTED_ROWS = (((int64_t)1 << 32) / 512 - 1) * 16;
// v (2, T, rank): the scaled inner products of x with a, then what these lost by their rounding (and v2 with a2, of
// one rank); rows without an adapter are left.  The caller has checked the sizes.
int adapter_inner(const void* x, int64_t T, int K, const int32_t* ids, int n, int rank, const void* a, const float* scale,
                  void* v, const void* a2, const float* scale2, void* v2, void* stream);
// out = the sum of `runs` arrays of `total` f32 in their order, as bf16
int launch_sum_runs(const float* part, int runs, int64_t total, uint16_t* out, hipStream_t s);

// The tile, by the time that each would take: rounds of workgroups over the compute units, a round's
// time for 64 of K with every place taken and with one workgroup a unit, and what a round costs
// besides (us; from the down product of 16384 to 48 rows, d 2048, F 5632, and the others of these sizes).
// 256 x 256 and 192 x 256 lie alone on a unit, a fuller chip clocks lower; 128 x 128 two side by side, or
// one with twice the stages; 64 x 128 and 64 x 64 two side by side.  The rates are those of the first
// milliseconds after a pause; measured 60 ms back to back, at the clocks that the chip then holds, us:
//                        256x256 192x256 128x128 128x128/4  64x128  64x64
//   16384 rows, gate up    563     605     664       794      859     1071
//   16384 rows, down       259     298     322       355      429      559
//    2042 rows, gate up     92      82      90       108      110      137
//    2042 rows, down        99      85      61        46       56       71
//     777 rows, gate up     42      38      50        51       49       58
//     777 rows, down        98      82      54        37       29       35
//     128 rows, gate up     43      41      30        23       18       21
//      48 rows, gate up     42      40      30        18       18       12
enum Tile { T256, T192, T128, T128_DEEP, T64X128, T64 };
inline Tile choose_tile(int64_t M, int64_t cols, double steps, int from = T256, double* us = nullptr) {
  struct Rate {
    int bm, bn, side;
    double full, few, besides;
  };
  constexpr Rate rates[] = {{256, 256, 1, 1.63, 1.25, 7.0}, {192, 256, 1, 1.27, 1.05, 6.0}, {128, 128, 2, 1.08, 0.62, 3.0},
                            {128, 128, 1, 0.57, 0.57, 3.0}, {64, 128, 2, 0.72, 0.42, 2.5},  {64, 64, 2, 0.50, 0.33, 2.0}};
  const int64_t cus = kmoe::cu_count();
  int best = from;
  double least = 0;
  for (int i = from; i < 6; ++i) {
    const Rate& r = rates[i];
    const int64_t tiles = kmoe::ceil_div<int64_t>(M, r.bm) * kmoe::ceil_div<int64_t>(cols, r.bn);
    const int64_t rounds = tiles / (cus * r.side), rest = tiles - rounds * cus * r.side;
    double t = rounds * (r.full * steps + r.besides);
    if (rest > cus)
      t += r.full * steps + r.besides;
    else if (rest > 0)
      t += (r.side == 1 ? r.few + (r.full - r.few) * rest / cus : r.few) * steps + r.besides;
    if (i == from || t < least) best = i, least = t;
  }
  if (us) *us = least;
  return (Tile)best;
}

template <int BM, int BN, int KS, int STAGES, bool SA, bool SB, int EPI, bool ADAPT>
int launch_tile(const Args& g, hipStream_t s) {
  constexpr int CN = EPI == EPI_GATED ? BN / 2 : BN;
  const int64_t n_mt = kmoe::ceil_div<int64_t>(g.M, BM), n_nt = kmoe::ceil_div(g.N, CN);
  // (a launch has fewer than 2^32 threads)
  KMOE_REQUIRE(n_mt * n_nt < ((int64_t)1 << 32) / THREADS, KMOE_ERR_SHAPE, "kmoe dense product: %lld x %d results in one call",
               (long long)g.M, g.N);
  // (a tile's 32-bit offsets: 256 rows of a K-contiguous operand, 64 of a K-strided one, an adapter's rows)
  KMOE_REQUIRE(g.lda < (int64_t)1 << 22 && g.ldb < (int64_t)1 << 22, KMOE_ERR_SHAPE,
               "kmoe dense product: rows of %lld and %lld values (below 2^22)", (long long)g.lda, (long long)g.ldb);
  KMOE_REQUIRE(!ADAPT || (int64_t)g.N * g.ad.r < (int64_t)1 << 30, KMOE_ERR_SHAPE,
               "kmoe dense product: adapters of %d x %d values (below 2^30)", g.N, g.ad.r);
  const int runs = g.k_run ? kmoe::ceil_div(g.K, g.k_run) : 1;
  hipLaunchKernelGGL((dense_kernel<BM, BN, KS, STAGES, SA, SB, EPI, ADAPT>), dim3((unsigned)(n_mt * n_nt), runs),
                     dim3(THREADS), 0, s, g, (int)n_mt, (int)n_nt);
  return kmoe::check_launch("kmoe dense product");
}

template <bool SA, bool SB, int EPI, bool ADAPT = false>
int launch_any(const Args& g, hipStream_t s) {
  if (g.fold) {
    KMOE_REQUIRE(g.M <= LOST_ROWS, KMOE_ERR_SHAPE, "kmoe dense product: %lld rows with what they lost (at most %d)",
                 (long long)g.M, LOST_ROWS);
    return launch_tile<64, 64, 2, 4, SA, SB, EPI, ADAPT>(g, s);
  }
  const double steps = (double)kmoe::ceil_div(g.K, 64) * (EPI == EPI_TWO ? 2 : 1);
  // (with adapters not the largest tile: its sums fill the registers)
  switch (choose_tile(g.M, (int64_t)g.N * (EPI == EPI_GATED ? 2 : 1), steps, ADAPT ? T192 : T256)) {
    case T256:
      if constexpr (!ADAPT) return launch_tile<256, 256, 2, 2, SA, SB, EPI, ADAPT>(g, s);
      [[fallthrough]];
    case T192: return launch_tile<192, 256, 2, 2, SA, SB, EPI, ADAPT>(g, s);
    // (weight gradients: steps of 32 of K lie as well, and two more stages fit; 2042 rows 57 against 61 us)
    case T128: return launch_tile<128, 128, SA ? 1 : 2, SA ? 4 : 2, SA, SB, EPI, ADAPT>(g, s);
    case T128_DEEP: return launch_tile<128, 128, 2, 4, SA, SB, EPI, ADAPT>(g, s);
    case T64X128: return launch_tile<64, 128, 2, 3, SA, SB, EPI, ADAPT>(g, s);
    default: return launch_tile<64, 64, 2, 4, SA, SB, EPI, ADAPT>(g, s);
  }
}

}  // namespace kmoe_dense
