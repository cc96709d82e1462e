// Products of 16 rows with rows that are streamed once, from memory straight into the MFMAs.
#pragma once

#include "kmoe_dense.h"

namespace kmoe_dense {

// acc[y] += w[y] x^T over all of K for 16 rows of each w[y] and of x: this wave of W takes 64 of K at a
// time, a lane 16 bytes of a row twice, D such steps in flight.  Bases are uniform; woff, xoff: the
// lane's row l % 16, in bytes, or NOWHERE.  What is past K's end reads as zeros in both.
template <int G, int W, int D>
struct Stream16 {
  const void* w[G];
  const void* x;
  uint32_t woff[G], xoff;
  int K;
  bf16x8_t fw[D][2][G], fx[D][2];

  __device__ __forceinline__ void load(int d, int it, int wave, int lane) {
    const int k = (it * W + wave) * 64 + 8 * (lane >> 4);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t at = k + 32 * h < K ? (uint32_t)(k + 32 * h) * 2 : NOWHERE;
#pragma unroll
      for (int y = 0; y < G; ++y) fw[d][h][y] = load16(w[y], (woff[y] | at) & NOWHERE ? NOWHERE : woff[y] + at);
      fx[d][h] = load16(x, (xoff | at) & NOWHERE ? NOWHERE : xoff + at);
    }
  }
  __device__ __forceinline__ int steps() const { return (K + 64 * W - 1) / (64 * W); }
  __device__ __forceinline__ void start(int wave, int lane) {
    const int n = steps();
    static_for<0, D>([&](auto dt) {
      constexpr int d = decltype(dt)::value;
      if (d < n) load(d, d, wave, lane);
    });
  }
  // (the loop has no conditions, so that a step waits for its own loads only; loads that read nothing
  // would still take their turn in the unit's address path)
  __device__ __forceinline__ void run(int wave, int lane, f32x4_t (&acc)[G]) {
    const int n = steps();
    auto add = [&](auto dt) {
      constexpr int d = decltype(dt)::value;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int y = 0; y < G; ++y)
          acc[y] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fw[d][h][y], fx[d][h], acc[y], 0, 0, 0);
    };
    int it = 0;
#pragma unroll 1
    for (; it + 2 * D <= n; it += D)
      static_for<0, D>([&](auto dt) {
        add(dt);
        load(decltype(dt)::value, it + decltype(dt)::value + D, wave, lane);
      });
    static_for<0, D>([&](auto dt) {
      constexpr int d = decltype(dt)::value;
      if (it + d < n) add(dt);
      if (it + d + D < n) load(d, it + d + D, wave, lane);
    });
    static_for<0, D>([&](auto dt) {
      if (it + D + decltype(dt)::value < n) add(dt);
    });
  }
};

}  // namespace kmoe_dense
