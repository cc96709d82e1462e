// Microscaled numbers (OCP Microscaling Formats v1.0): blocks of 32 values along K share a
// power-of-two scale (e8m0: byte c stands for 2^(c - 127), 255 for NaN), the elements are
// e4m3 or e2m1.  A block's scale is 2^(floor(log2(largest magnitude)) - emax), emax 8 (e4m3)
// and 2 (e2m1), at least 2^-127; elements are value / scale rounded to nearest even and
// saturated (448, 6).  A block that holds a NaN or an infinity gets the scale NaN and zero
// elements, so it stands for NaN throughout, in either element type.
//
// Packed 4-bit weights (kmoe_pack_weights_mx): MFMA operand order.  The unit is the block of
// 32 weight rows (output columns) x 64 of K, 1 KiB: lane l of a wave holds row l % 32, K
// 32 (l / 32) .. + 31 as 16 bytes at 16 l, the even K in the low nibble.  A weight tile is
// 256 rows; per 128 of K it holds its eight 32-row blocks, each with its two K halves: 16
// KiB, and the tile's steps follow each other, so a product streams memory in order.  The
// scales of the same tile step are 1 KiB: per 32-row block and lane two bytes (the K halves).
//   w13: E x Fp/128 tiles x dk/128 steps; block 2 j holds 32 gate columns, 2 j + 1 the up
//        columns of the same f (so a wave that owns both has h in its registers)
//   w3:  E x dp/256 tiles x Fp/128 steps; block j holds output columns 32 j ..
// Fp = round_up(F, 128), dk = round_up(d, 128), dp = round_up(d, 256); padding is zeros.
#pragma once

#include "kmoe_common.h"

namespace kmoe_mx {

constexpr int BLOCK = 32;              // values that share a scale
constexpr int STEP = 128;              // K of one pipeline step
constexpr int TILE_ROWS = 256;         // weight rows of a tile
constexpr int TILE_STEP = 16 * 1024;   // bytes of a weight tile per step
constexpr int SCALE_STEP = 1024;       // scale bytes of a weight tile per step

__host__ __device__ inline int round_up(int a, int b) { return (a + b - 1) / b * b; }
// bytes of a row of K values (K rounded up to the step) and of its scales
__host__ __device__ inline int64_t row_bytes(bool fp4, int K) { return round_up(K, STEP) / (fp4 ? 2 : 1); }
__host__ __device__ inline int64_t scale_bytes(int K) { return round_up(K, STEP) / BLOCK; }

// Scale byte of a block whose largest magnitude is amax (not negative; NaN or infinity: 255).
// The exponent bits of a float are floor(log2) + 127; subnormal floats count as 2^-127.
template <bool FP4>
__device__ __forceinline__ uint32_t scale_code(float amax) {
  const uint32_t ef = __float_as_uint(amax) >> 23;
  constexpr uint32_t EMAX = FP4 ? 2 : 8;
  return ef >= 255u ? 255u : (ef > EMAX ? ef - EMAX : 0u);
}
// 1 / scale of scale byte c < 255 (a power of two, 2^127 at most); 0 for 255
__device__ __forceinline__ float inv_scale(uint32_t c) { return c == 255u ? 0.0f : __uint_as_float((254u - c) << 23); }
// The scale itself (2^-127 is a subnormal float)
__device__ __forceinline__ float scale_value(uint32_t c) {
  return c == 255u ? __uint_as_float(0x7fc00000u) : c == 0u ? __uint_as_float(0x00400000u) : __uint_as_float(c << 23);
}

// Largest magnitude, with every NaN counted as an infinity (fmaxf would drop it).
__device__ __forceinline__ float amax_nan(float m, float v) {
  const float a = fabsf(v);
  return fmaxf(m, a != a ? __uint_as_float(0x7f800000u) : a);
}

// e2m1 code of v (finite): thresholds are the midpoints of 0, .5, 1, 1.5, 2, 3, 4, 6, a tie
// goes to the even code.
__device__ __forceinline__ uint32_t e2m1(float v) {
  const float a = fabsf(v);
  const uint32_t c = (uint32_t)(a > 0.25f) + (uint32_t)(a >= 0.75f) + (uint32_t)(a > 1.25f) + (uint32_t)(a >= 1.75f) +
                     (uint32_t)(a > 2.5f) + (uint32_t)(a >= 3.5f) + (uint32_t)(a > 5.0f);
  return c | (__float_as_uint(v) >> 31 << 3);
}
__device__ __forceinline__ float e2m1_value(uint32_t c) {
  const uint32_t m = c & 7u;
  // exponent field m / 2, mantissa m % 2; field 0 is 0 and 0.5
  const float v = m < 2u ? 0.5f * (float)m : __uint_as_float(((m >> 1) + 126u) << 23 | (m & 1u) << 22);
  return c & 8u ? -v : v;
}

// Codes of v[0 .. N) / scale: N bytes (e4m3) or N / 2 (e2m1, the first value in the low nibble).
template <bool FP4, int N>
struct Codes {
  uint32_t w[FP4 ? N / 8 : N / 4];
};
template <bool FP4, int N>
__device__ __forceinline__ Codes<FP4, N> encode(const float (&v)[N], uint32_t code) {
  Codes<FP4, N> out;
  const float inv = inv_scale(code);
  const bool none = code == 255u;
  if constexpr (FP4) {
#pragma unroll
    for (int i = 0; i < N / 8; ++i) {
      uint32_t w = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) w |= e2m1(v[8 * i + j] * inv) << (4 * j);
      out.w[i] = none ? 0u : w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      int r = __builtin_amdgcn_cvt_pk_fp8_f32(sat448(v[4 * i] * inv), sat448(v[4 * i + 1] * inv), 0, false);
      r = __builtin_amdgcn_cvt_pk_fp8_f32(sat448(v[4 * i + 2] * inv), sat448(v[4 * i + 3] * inv), r, true);
      out.w[i] = none ? 0u : (uint32_t)r;
    }
  }
  return out;
}

// 8 consecutive values of a bf16 row
__device__ __forceinline__ void unpack8(const i32x4_t& a, float (&v)[8]) {
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    v[2 * q] = __uint_as_float(((uint32_t)a[q]) << 16);
    v[2 * q + 1] = __uint_as_float(((uint32_t)a[q]) & 0xffff0000u);
  }
}

// Quantises 8 values per lane, the blocks being groups of four lanes (all active): codes
// and the group's scale byte.
template <bool FP4>
__device__ __forceinline__ Codes<FP4, 8> encode_quad(const float (&v)[8], uint32_t& code) {
  float m = 0.0f;
#pragma unroll
  for (int q = 0; q < 8; ++q) m = amax_nan(m, v[q]);
  m = fmaxf(m, quad_xor<1>(m));
  m = fmaxf(m, quad_xor<2>(m));
  code = scale_code<FP4>(m);
  return encode<FP4, 8>(v, code);
}

}  // namespace kmoe_mx
