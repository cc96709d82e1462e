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

template <int BM, int BN, int KS, int STAGES, bool SA, bool SB, int EPI, bool ADAPT>
int launch_tile(const Args& g, hipStream_t s) {
  constexpr int CN = EPI == EPI_GATED ? BN / 2 : BN;
  const int64_t n_mt = kmoe::ceil_div<int64_t>(g.M, BM), n_nt = kmoe::ceil_div(g.N, CN);
  KMOE_REQUIRE(n_mt * n_nt < (int64_t)1 << 31, KMOE_ERR_SHAPE, "kmoe dense product: %lld x %d results in one call",
               (long long)g.M, g.N);
  // (a tile's 32-bit offsets: 256 rows of a K-contiguous operand, 64 of a K-strided one)
  KMOE_REQUIRE(g.lda < (int64_t)1 << 22 && g.ldb < (int64_t)1 << 22, KMOE_ERR_SHAPE,
               "kmoe dense product: rows of %lld and %lld values (below 2^22)", (long long)g.lda, (long long)g.ldb);
  hipLaunchKernelGGL((dense_kernel<BM, BN, KS, STAGES, SA, SB, EPI, ADAPT>), dim3((unsigned)(n_mt * n_nt)), dim3(THREADS), 0,
                     s, g, (int)n_mt, (int)n_nt);
  return kmoe::check_launch("kmoe dense product");
}

// The tile, by the time that each would take: rounds of workgroups over the compute units, a round's
// time for 64 of K with every place taken and with one workgroup a unit, and what a round costs
// besides (us, down product of 16384 to 200 rows, d 2048, F 5632: 256 x 256 alone on a unit 1.69, 1.15 where
// few are and the chip clocks higher; 128 x 128 two side by side 1.08, one 0.65; the same with
// twice the stages, alone, 0.59; 64 x 128 two side by side 0.70, one 0.36).  So 16384 rows take the
// large tile (297 us; 381, 414, 495 with the others), 2042 the third (51; 103, 66, 59), 777 the fourth
// (30; 98, 55, 40).
template <bool SA, bool SB, int EPI, bool ADAPT = false>
int launch_any(const Args& g, hipStream_t s) {
  const int cus = kmoe::cu_count();
  const int64_t cols = (int64_t)g.N * (EPI == EPI_GATED ? 2 : 1);
  const double steps = (double)kmoe::ceil_div(g.K, 64) * (EPI == EPI_TWO ? 2 : 1);
  auto cost = [&](int bm, int bn, int side, double full, double few, double besides) {
    const int64_t tiles = kmoe::ceil_div<int64_t>(g.M, bm) * kmoe::ceil_div<int64_t>(cols, bn);
    const int64_t rounds = tiles / (cus * side), rest = tiles - rounds * cus * side;
    double t = rounds * (full * steps + besides);
    if (rest > cus)
      t += full * steps + besides;
    else if (rest > 0)
      t += (side == 1 ? few + (full - few) * rest / cus : few) * steps + besides;
    return t;
  };
  const double big = cost(256, 256, 1, 1.69, 1.15, 7.0), two = cost(128, 128, 2, 1.08, 0.65, 3.0);
  const double deep = cost(128, 128, 1, 0.59, 0.44, 3.0), small = cost(64, 128, 2, 0.70, 0.36, 2.5);
  if (big <= two && big <= deep && big <= small) return launch_tile<256, 256, 2, 2, SA, SB, EPI, ADAPT>(g, s);
  // (weight gradients: steps of 32 of K lie as well, and two more stages fit; 2042 rows 57 against 61 us)
  if (two <= deep && two <= small) return launch_tile<128, 128, SA ? 1 : 2, SA ? 4 : 2, SA, SB, EPI, ADAPT>(g, s);
  if (deep <= small) return launch_tile<128, 128, 2, 4, SA, SB, EPI, ADAPT>(g, s);
  return launch_tile<64, 128, 2, 3, SA, SB, EPI, ADAPT>(g, s);
}

}  // namespace kmoe_dense
