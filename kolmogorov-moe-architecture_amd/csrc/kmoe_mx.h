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
// scales of the same tile step are 1 KiB: 16 bytes, one for each 16 weight rows of the tile, of
// row r of those and K 32 b .. at 16 (16 b + r), so one load of a lane has all that it needs.
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
// Bytes of a row of K values (K rounded up to the step) and of its scales (rounded up to 16:
// four steps, which the products load at once).
__host__ __device__ inline int64_t row_bytes(bool fp4, int K) { return round_up(K, STEP) / (fp4 ? 2 : 1); }
__host__ __device__ inline int64_t scale_bytes(int K) { return round_up(K, 4 * STEP) / BLOCK; }

// Scale byte of a block whose largest magnitude has the bits amax (NaN or infinity: 255).
// The exponent bits of a float are floor(log2) + 127; subnormal floats count as 2^-127.
template <bool FP4>
__device__ __forceinline__ uint32_t scale_code(uint32_t amax) {
  const uint32_t ef = amax >> 23;
  constexpr uint32_t EMAX = FP4 ? 2 : 8;
  return ef >= 255u ? 255u : (ef > EMAX ? ef - EMAX : 0u);
}
// 1 / scale of scale byte c < 255 (a power of two, 2^127 at most); 0 for 255
__device__ __forceinline__ float inv_scale(uint32_t c) { return c == 255u ? 0.0f : __uint_as_float((254u - c) << 23); }
// The scale itself (2^-127 is a subnormal float)
__device__ __forceinline__ float scale_value(uint32_t c) {
  return c == 255u ? __uint_as_float(0x7fc00000u) : c == 0u ? __uint_as_float(0x00400000u) : __uint_as_float(c << 23);
}

// Largest magnitude as float bits, which order as integers do; a NaN's are above infinity's.
__device__ __forceinline__ uint32_t amax_bits(uint32_t m, float v) { return max(m, __float_as_uint(v) & 0x7fffffffu); }

// Two finite values as e2m1 codes (a in bits 0 .. 3): the hardware converter, whose rounding
// (nearest, ties to the even code, 6 from above 5) equals the thresholds .25 .75 1.25 1.75 2.5
// 3.5 5 on every finite float (checked exhaustively on gfx950).  SEL: byte of `old` to write.
template <int SEL>
__device__ __forceinline__ uint32_t e2m1x2(uint32_t old, float a, float b) {
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(old, a, b, 1.0f, SEL);
}
// The values of the two codes in byte SEL of w
template <int SEL>
__device__ __forceinline__ f32x2_t e2m1x2_values(uint32_t w) {
  const auto v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, SEL);
  return f32x2_t{v[0], v[1]};
}
__device__ __forceinline__ float clamp448(float v) { return __builtin_amdgcn_fmed3f(v, -448.0f, 448.0f); }

// Codes of v[0 .. N) / scale: N bytes (e4m3) or N / 2 (e2m1, the first value in the low nibble).
template <bool FP4, int N>
struct Codes {
  uint32_t w[FP4 ? N / 8 : N / 4];
};
template <bool FP4, int N>
__device__ __forceinline__ Codes<FP4, N> encode(const float (&v)[N], uint32_t code) {
  Codes<FP4, N> out;
  const float inv = inv_scale(code);
  const bool none = code == 255u;  // inv 0: NaN and infinity times 0 are NaN, replaced below
  if constexpr (FP4) {
#pragma unroll
    for (int i = 0; i < N / 8; ++i) {
      uint32_t w = e2m1x2<0>(0u, v[8 * i] * inv, v[8 * i + 1] * inv);
      w = e2m1x2<1>(w, v[8 * i + 2] * inv, v[8 * i + 3] * inv);
      w = e2m1x2<2>(w, v[8 * i + 4] * inv, v[8 * i + 5] * inv);
      w = e2m1x2<3>(w, v[8 * i + 6] * inv, v[8 * i + 7] * inv);
      out.w[i] = none ? 0u : w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      int r = __builtin_amdgcn_cvt_pk_fp8_f32(clamp448(v[4 * i] * inv), clamp448(v[4 * i + 1] * inv), 0, false);
      r = __builtin_amdgcn_cvt_pk_fp8_f32(clamp448(v[4 * i + 2] * inv), clamp448(v[4 * i + 3] * inv), r, true);
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
  uint32_t m = 0;
#pragma unroll
  for (int q = 0; q < 8; ++q) m = amax_bits(m, v[q]);
  m = max(m, (uint32_t)quad_xor<1>((int)m));
  m = max(m, (uint32_t)quad_xor<2>((int)m));
  code = scale_code<FP4>(m);
  return encode<FP4, 8>(v, code);
}

}  // namespace kmoe_mx
