// Products of 16 rows with rows that are streamed once, from memory straight into the MFMAs.
#pragma once

#include "kmoe_dense.h"

namespace kmoe_dense {

// acc[y] += w[y] x^T over all of K for 16 rows of each w[y] and of x: this wave of W takes 64 of K at a
// time, a lane 16 bytes of a row twice, D such steps in flight.  Bases are uniform; woff, xoff: the
// lane's row l % 16, in bytes, or NOWHERE.  What is past K's end reads as zeros in both.
template <int G, int W, int D>
__device__ __forceinline__ void stream16(const void* const (&w)[G], const uint32_t (&woff)[G], const void* x, uint32_t xoff,
                                         int K, int wave, int lane, f32x4_t (&acc)[G], bool loaded,
                                         bf16x8_t (&fw)[D][2][G], bf16x8_t (&fx)[D][2]) {
  auto load = [&](int d, int it) {
    const int k = (it * W + wave) * 64 + 8 * (lane >> 4);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t at = k + 32 * h < K ? (uint32_t)(k + 32 * h) * 2 : NOWHERE;
#pragma unroll
      for (int y = 0; y < G; ++y) fw[d][h][y] = load16(w[y], (woff[y] | at) & NOWHERE ? NOWHERE : woff[y] + at);
      fx[d][h] = load16(x, at & NOWHERE ? NOWHERE : xoff + at);
    }
  };
  if (!loaded) {
#pragma unroll
    for (int d = 0; d < D; ++d) load(d, d);
    return;
  }
  const int n = (K + 64 * W - 1) / (64 * W);
#pragma unroll 1
  for (int it = 0; it < n; it += D)
    static_for<0, D>([&](auto dt) {
      constexpr int d = decltype(dt)::value;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int y = 0; y < G; ++y)
          acc[y] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fw[d][h][y], fx[d][h], acc[y], 0, 0, 0);
      load(d, it + d + D);
    });
}

}  // namespace kmoe_dense
