// Launches of the dense products, one source file for each kind: their instances compile side by side.
#pragma once

#include "kmoe_dense.h"

namespace kmoe_dense {

int launch_gated(const Args& g, hipStream_t s);         // act(a b0^T) * (a b1^T)
int launch_gated_adapt(const Args& g, hipStream_t s);
int launch_linear(const Args& g, hipStream_t s);        // a b^T
int launch_linear_adapt(const Args& g, hipStream_t s);
int launch_dh(const Args& g, hipStream_t s);            // (a b) p, (a b) q
int launch_dx(const Args& g, hipStream_t s);            // a0 b0 (+ a1 b1)
int launch_dx_adapt(const Args& g, hipStream_t s);
int launch_wgrad(const Args& g, hipStream_t s);         // a^T b

template <int BM, int BN, bool SA, bool SB, int EPI, int NST, bool ADAPT>
int launch_tile(const Args& g, hipStream_t s) {
  constexpr int CN = EPI == EPI_GATED ? BN / 2 : BN;
  const int64_t n_mt = kmoe::ceil_div<int64_t>(g.M, BM), n_nt = kmoe::ceil_div(g.N, CN);
  KMOE_REQUIRE(n_mt * n_nt < (int64_t)1 << 31, KMOE_ERR_SHAPE, "kmoe dense product: %lld x %d results in one call",
               (long long)g.M, g.N);
  hipLaunchKernelGGL((dense_kernel<BM, BN, SA, SB, EPI, NST, ADAPT>), dim3((unsigned)(n_mt * n_nt)), dim3(THREADS), 0, s, g,
                     (int)n_mt, (int)n_nt);
  return kmoe::check_launch("kmoe dense product");
}

// The tile: rounds of workgroups over the compute units, each worth its area over the rate that the
// tile reaches (a 256 x 256 tile fills a compute unit, of the others two run side by side).
template <bool SA, bool SB, int EPI, bool ADAPT = false>
int launch_any(const Args& g, hipStream_t s) {
  const int cus = kmoe::cu_count();
  const int64_t cols = (int64_t)g.N * (EPI == EPI_GATED ? 2 : 1);
  auto cost = [&](int bm, int bn, int side, double rate) {
    const int64_t tiles = kmoe::ceil_div<int64_t>(g.M, bm) * kmoe::ceil_div<int64_t>(cols, bn);
    const int64_t rounds = tiles / (cus * side), rest = tiles - rounds * cus * side;
    return ((double)rounds * side + (rest > cus ? side : rest > 0 ? 1.2 : 0.0)) * bm * bn / rate;
  };
  const double big = cost(256, 256, 1, 1.0), mid = cost(128, 128, 2, 0.86), small = cost(64, 128, 2, 0.66);
  if (big <= mid && big <= small) return launch_tile<256, 256, SA, SB, EPI, 2, ADAPT>(g, s);
  if (mid <= small) return launch_tile<128, 128, SA, SB, EPI, 2, ADAPT>(g, s);
  return launch_tile<64, 128, SA, SB, EPI, 3, ADAPT>(g, s);
}

}  // namespace kmoe_dense
