// Microscaled rows and weights: quantisation, the values back, and the packed 4-bit weights
// (kmoe_mx.h has the formats and layouts).  All of it moves memory: each value is read once
// and each result written once.
#include <algorithm>

#include "kmoe_mx.h"

using namespace kmoe_mx;

namespace {

unsigned grid_of(int64_t items, int per_block) {
  return (unsigned)std::min<int64_t>(kmoe::ceil_div<int64_t>(items, per_block), 1 << 20);
}

// Rows of x (bf16, K a multiple of 32) to codes and scales, both padded to the 128-step of
// K with zeros.  A lane takes 8 values, four lanes a block; row r is x[row_index[r]],
// zeros for -1.  16384 x 2048 to e4m3 18 us (5.7 TB/s), to e2m1 15.4.
template <bool FP4>
__global__ __launch_bounds__(256) void quant_rows_kernel(const uint16_t* __restrict__ x, const int32_t* __restrict__ row_index,
                                                         int64_t rows, const int32_t* __restrict__ n_rows_dev, int K,
                                                         uint8_t* __restrict__ q, uint8_t* __restrict__ scale) {
  const int64_t nr = n_rows_dev ? min<int64_t>(rows, (int64_t)*n_rows_dev) : rows;
  const int Kp = round_up(K, STEP), cpr = Kp / 8, spr = (int)scale_bytes(K);
  const int64_t total = nr * cpr;  // a multiple of 16: the lanes of a block stay together
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / cpr;
    const int c = (int)(i - r * cpr);
    float v[8] = {};
    const int64_t src = row_index ? (int64_t)row_index[r] : r;
    if (c * 8 < K && src >= 0) unpack8(*reinterpret_cast<const i32x4_t*>(x + src * K + c * 8), v);
    uint32_t code;
    const Codes<FP4, 8> o = encode_quad<FP4>(v, code);
    if constexpr (FP4)
      *reinterpret_cast<uint32_t*>(q + r * (Kp / 2) + c * 4) = o.w[0];
    else
      *reinterpret_cast<i32x2_t*>(q + r * Kp + c * 8) = i32x2_t{(int)o.w[0], (int)o.w[1]};
    if ((c & 3) == 0) scale[r * spr + c / 4] = (uint8_t)code;
  }
}

// 8 values of codes at p, times the scale
template <bool FP4>
__device__ __forceinline__ void decode8(const uint8_t* p, float s, float (&v)[8]) {
  if constexpr (FP4) {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(p);
    const f32x2_t a = e2m1x2_values<0>(w), b = e2m1x2_values<1>(w), c = e2m1x2_values<2>(w), d = e2m1x2_values<3>(w);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      v[j] = a[j] * s;
      v[2 + j] = b[j] * s;
      v[4 + j] = c[j] * s;
      v[6 + j] = d[j] * s;
    }
  } else {
    const i32x2_t w = *reinterpret_cast<const i32x2_t*>(p);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(w[j], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w[j], true);
      v[4 * j] = lo[0] * s;
      v[4 * j + 1] = lo[1] * s;
      v[4 * j + 2] = hi[0] * s;
      v[4 * j + 3] = hi[1] * s;
    }
  }
}
__device__ __forceinline__ i32x4_t pack8(const float (&v)[8]) {
  i32x4_t a;
#pragma unroll
  for (int q = 0; q < 4; ++q) a[q] = (int)((uint32_t)f32_to_bf16(v[2 * q]) | ((uint32_t)f32_to_bf16(v[2 * q + 1]) << 16));
  return a;
}

// The values of coded rows in bf16 (exact: 4 and 2 significant bits); row r is coded row
// row_index[r], zeros for -1.  K a multiple of 8.  16384 x 2048 from e4m3 21 us (4.9 TB/s; with
// the codes taken apart by integer operations and not by the converter 26), from e2m1 19.
template <bool FP4>
__global__ __launch_bounds__(256) void dequant_rows_kernel(const uint8_t* __restrict__ q, const uint8_t* __restrict__ scale,
                                                           const int32_t* __restrict__ row_index, int64_t rows,
                                                           const int32_t* __restrict__ n_rows_dev, int K,
                                                           uint16_t* __restrict__ out) {
  const int64_t nr = n_rows_dev ? min<int64_t>(rows, (int64_t)*n_rows_dev) : rows;
  const int Kp = round_up(K, STEP), cpr = K / 8, spr = (int)scale_bytes(K);
  const int64_t total = nr * cpr;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / cpr;
    const int c = (int)(i - r * cpr);
    const int64_t src = row_index ? (int64_t)row_index[r] : r;
    float v[8] = {};
    if (src >= 0) {
      const float s = scale_value(scale[src * spr + c / 4]);
      decode8<FP4>(q + (FP4 ? src * (Kp / 2) + c * 4 : src * Kp + c * 8), s, v);
    }
    *reinterpret_cast<i32x4_t*>(out + r * K + c * 8) = pack8(v);
  }
}

// The 32 values of K from k0 on of C columns n .. of w (K, N) (C a divisor of N with aligned
// rows, or 1), zeros past K and N: v[j][c].
template <bool F32, int C>
struct WBlock {
  float v[BLOCK][C];
};
template <bool F32, int C>
__device__ __forceinline__ void load_block(const void* __restrict__ w, int64_t base, int k0, int K, int N, bool on,
                                           WBlock<F32, C>& o) {
#pragma unroll
  for (int j = 0; j < BLOCK; ++j) {
    const bool in = on && k0 + j < K;
    const int64_t i = base + (int64_t)j * N;
    if constexpr (C == 1) {
      o.v[j][0] = !in ? 0.0f : F32 ? static_cast<const float*>(w)[i] : bf16_to_f32(static_cast<const uint16_t*>(w)[i]);
    } else if constexpr (F32) {
      const f32x4_t z = {0.0f, 0.0f, 0.0f, 0.0f};
      const f32x4_t a = in ? *reinterpret_cast<const f32x4_t*>(static_cast<const float*>(w) + i) : z;
#pragma unroll
      for (int c = 0; c < 4; ++c) o.v[j][c] = a[c];
    } else {
      const i32x2_t a = in ? *reinterpret_cast<const i32x2_t*>(static_cast<const uint16_t*>(w) + i) : i32x2_t{0, 0};
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        o.v[j][2 * c] = __uint_as_float((uint32_t)a[c] << 16);
        o.v[j][2 * c + 1] = __uint_as_float((uint32_t)a[c] & 0xffff0000u);
      }
    }
  }
}
template <bool F32, int C>
__device__ __forceinline__ uint32_t column_code(const WBlock<F32, C>& o, int c) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < BLOCK; ++j) m = amax_bits(m, o.v[j][c]);
  return scale_code<true>(m);
}

// w (E, K, N) to the values its e2m1 blocks along K stand for, bf16.  A thread takes C columns
// of a block: with four (8 bytes of a bf16 row a lane) E 16, K 2048, N 2816 take 71 us
// (5.2 TB/s, a copy's rate), with one 174.
template <bool F32, int C>
__global__ __launch_bounds__(256) void fake_quant_kernel(const void* __restrict__ w, int E, int K, int N,
                                                         uint16_t* __restrict__ out) {
  const int nb = (K + BLOCK - 1) / BLOCK, per = N / C;
  const int64_t total = (int64_t)E * nb * per;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t eb = i / per;
    const int n = (int)(i - eb * per) * C;
    const int64_t e = eb / nb;
    const int k0 = (int)(eb - e * nb) * BLOCK;
    const int64_t base = (e * K + k0) * N + n;
    WBlock<F32, C> o;
    load_block<F32, C>(w, base, k0, K, N, true, o);
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const uint32_t code = column_code<F32, C>(o, c);
      const float inv = inv_scale(code), s = scale_value(code);
#pragma unroll
      for (int j = 0; j < BLOCK; j += 2) {
        const f32x2_t q = e2m1x2_values<0>(e2m1x2<0>(0u, o.v[j][c] * inv, o.v[j + 1][c] * inv));
        o.v[j][c] = code == 255u ? s : q[0] * s;
        o.v[j + 1][c] = code == 255u ? s : q[1] * s;
      }
    }
#pragma unroll
    for (int j = 0; j < BLOCK; ++j)
      if (k0 + j < K) {
        if constexpr (C == 1) {
          out[base + (int64_t)j * N] = f32_to_bf16(o.v[j][0]);
        } else {
          // exact, so the upper halves of the floats are the bf16 values (a NaN's too)
          auto hi = [&](int c) { return __float_as_uint(o.v[j][c]); };
          *reinterpret_cast<i32x2_t*>(out + base + (int64_t)j * N) =
              i32x2_t{(int)(hi(0) >> 16 | (hi(1) & 0xffff0000u)), (int)(hi(2) >> 16 | (hi(3) & 0xffff0000u))};
        }
      }
  }
}

// One matrix w (E, K, N) into a packed weight: output column n of an expert goes to row
// `row(n)` of its tiles.  gate_up: tile n / 128, 32-row block 2 ((n % 128) / 32) + half; else
// tile n / 256, block (n % 256) / 32.  A thread quantises the 32 values of K of C columns
// (16 bytes of C neighbouring lanes of an MFMA block); N and K run over the padded sizes.  The
// three matrices of 16 experts, d 2048, F 2816: bf16 156 us (4.5 TB/s), f32 260 (4.8).
template <bool F32, int C>
__global__ __launch_bounds__(256) void pack_mx_kernel(const void* __restrict__ w, int E, int K, int N, int Np, bool gate_up,
                                                      int half, int tiles, uint8_t* __restrict__ q,
                                                      uint8_t* __restrict__ scale) {
  const int Kp = round_up(K, STEP), nb = Kp / BLOCK, per = Np / C;
  const int64_t total = (int64_t)E * nb * per;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t eb = i / per;
    const int n0 = (int)(i - eb * per) * C;
    const int64_t e = eb / nb;
    const int b = (int)(eb - e * nb), k0 = b * BLOCK;
    WBlock<F32, C> o;
    load_block<F32, C>(w, (e * K + k0) * N + n0, k0, K, N, n0 < N, o);
    const int tile = gate_up ? n0 / 128 : n0 / 256;
    const int blk = gate_up ? 2 * ((n0 & 127) / 32) + half : (n0 & 255) / 32;
    const int step = b / 4, sub = (b >> 1) & 1, lane = (b & 1) * 32 + (n0 & 31);
    const int64_t ts = (e * tiles + tile) * (Kp / STEP) + step;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const uint32_t code = column_code<F32, C>(o, c);
      float v[BLOCK];
#pragma unroll
      for (int j = 0; j < BLOCK; ++j) v[j] = o.v[j][c];
      const Codes<true, BLOCK> d = encode<true, BLOCK>(v, code);
      *reinterpret_cast<i32x4_t*>(q + ts * TILE_STEP + blk * 2048 + sub * 1024 + (lane + c) * 16) =
          i32x4_t{(int)d.w[0], (int)d.w[1], (int)d.w[2], (int)d.w[3]};
      scale[ts * SCALE_STEP + ((b & 3) * 16 + (n0 & 15) + c) * 16 + 2 * blk + (n0 >> 4 & 1)] = (uint8_t)code;
    }
  }
}

// Whether four columns at a time can be loaded: rows of whole, aligned quadruples.
bool four_columns(const void* p, bool f32, int N) { return N % 4 == 0 && reinterpret_cast<uintptr_t>(p) % (f32 ? 16 : 8) == 0; }

bool is_float(int dt) { return dt == KMOE_DTYPE_BF16 || dt == KMOE_DTYPE_F32; }
bool is_mx(int dt) { return dt == KMOE_DTYPE_FP8_E4M3 || dt == KMOE_DTYPE_FP4_E2M1; }

}  // namespace

extern "C" size_t kmoe_mx_row_bytes(int K, int fmt) {
  return K > 0 && is_mx(fmt) ? (size_t)row_bytes(fmt == KMOE_DTYPE_FP4_E2M1, K) : 0;
}
extern "C" size_t kmoe_mx_scale_bytes(int K) { return K > 0 ? (size_t)scale_bytes(K) : 0; }

extern "C" int kmoe_quant_rows_mx(const void* x, const int32_t* row_index, int64_t rows, const int32_t* n_rows_dev, int K,
                                  int fmt, void* q, uint8_t* scale, void* stream) {
  KMOE_REQUIRE(rows == 0 || (x && q && scale), KMOE_ERR_NULL, "kmoe_quant_rows_mx: null buffer");
  KMOE_REQUIRE(is_mx(fmt), KMOE_ERR_DTYPE, "kmoe_quant_rows_mx: element type %d is neither e4m3 nor e2m1", fmt);
  KMOE_REQUIRE(rows >= 0 && rows < (int64_t)1 << 31 && K > 0 && K % BLOCK == 0, KMOE_ERR_SHAPE,
               "kmoe_quant_rows_mx: rows=%lld, K=%d must be a positive multiple of %d", (long long)rows, K, BLOCK);
  if (rows == 0) return KMOE_OK;
  const unsigned grid = grid_of(rows * (round_up(K, STEP) / 8), 256);
  hipStream_t s = kmoe::as_stream(stream);
  const uint16_t* xp = static_cast<const uint16_t*>(x);
  uint8_t* qp = static_cast<uint8_t*>(q);
  if (fmt == KMOE_DTYPE_FP4_E2M1)
    hipLaunchKernelGGL(quant_rows_kernel<true>, dim3(grid), dim3(256), 0, s, xp, row_index, rows, n_rows_dev, K, qp, scale);
  else
    hipLaunchKernelGGL(quant_rows_kernel<false>, dim3(grid), dim3(256), 0, s, xp, row_index, rows, n_rows_dev, K, qp, scale);
  return kmoe::check_launch("kmoe_quant_rows_mx");
}

extern "C" int kmoe_dequant_rows_mx(const void* q, const uint8_t* scale, const int32_t* row_index, int64_t rows,
                                    const int32_t* n_rows_dev, int K, int fmt, void* out, void* stream) {
  KMOE_REQUIRE(rows == 0 || (q && scale && out), KMOE_ERR_NULL, "kmoe_dequant_rows_mx: null buffer");
  KMOE_REQUIRE(is_mx(fmt), KMOE_ERR_DTYPE, "kmoe_dequant_rows_mx: element type %d is neither e4m3 nor e2m1", fmt);
  KMOE_REQUIRE(rows >= 0 && rows < (int64_t)1 << 31 && K > 0 && K % BLOCK == 0, KMOE_ERR_SHAPE,
               "kmoe_dequant_rows_mx: rows=%lld, K=%d must be a positive multiple of %d", (long long)rows, K, BLOCK);
  if (rows == 0) return KMOE_OK;
  const unsigned grid = grid_of(rows * (K / 8), 256);
  hipStream_t s = kmoe::as_stream(stream);
  const uint8_t* qp = static_cast<const uint8_t*>(q);
  uint16_t* op = static_cast<uint16_t*>(out);
  if (fmt == KMOE_DTYPE_FP4_E2M1)
    hipLaunchKernelGGL(dequant_rows_kernel<true>, dim3(grid), dim3(256), 0, s, qp, scale, row_index, rows, n_rows_dev, K, op);
  else
    hipLaunchKernelGGL(dequant_rows_kernel<false>, dim3(grid), dim3(256), 0, s, qp, scale, row_index, rows, n_rows_dev, K,
                       op);
  return kmoe::check_launch("kmoe_dequant_rows_mx");
}

extern "C" int kmoe_fake_quant_mx_cols(const void* w, int w_dtype, int E, int K, int N, void* out, void* stream) {
  KMOE_REQUIRE(w && out, KMOE_ERR_NULL, "kmoe_fake_quant_mx_cols: null buffer");
  KMOE_REQUIRE(is_float(w_dtype), KMOE_ERR_DTYPE, "kmoe_fake_quant_mx_cols: dtype %d", w_dtype);
  KMOE_REQUIRE(E > 0 && K > 0 && N > 0, KMOE_ERR_SHAPE, "kmoe_fake_quant_mx_cols: E=%d K=%d N=%d", E, K, N);
  hipStream_t s = kmoe::as_stream(stream);
  const bool f32 = w_dtype == KMOE_DTYPE_F32;
  const int C = four_columns(w, f32, N) && reinterpret_cast<uintptr_t>(out) % 8 == 0 ? 4 : 1;
  const dim3 grid(grid_of((int64_t)E * kmoe::ceil_div(K, BLOCK) * (N / C), 256));
  uint16_t* op = static_cast<uint16_t*>(out);
  if (f32 && C == 4)
    hipLaunchKernelGGL((fake_quant_kernel<true, 4>), grid, dim3(256), 0, s, w, E, K, N, op);
  else if (f32)
    hipLaunchKernelGGL((fake_quant_kernel<true, 1>), grid, dim3(256), 0, s, w, E, K, N, op);
  else if (C == 4)
    hipLaunchKernelGGL((fake_quant_kernel<false, 4>), grid, dim3(256), 0, s, w, E, K, N, op);
  else
    hipLaunchKernelGGL((fake_quant_kernel<false, 1>), grid, dim3(256), 0, s, w, E, K, N, op);
  return kmoe::check_launch("kmoe_fake_quant_mx_cols");
}

namespace {
struct PackedSizes {
  int64_t w13, s13, w3, s3;
};
PackedSizes packed_sizes(int E, int d, int F) {
  const int64_t Fp = round_up(F, 128), dk = round_up(d, STEP), dp = round_up(d, 256);
  const int64_t t13 = E * (Fp / 128) * (dk / STEP), t3 = E * (dp / 256) * (Fp / STEP);
  return {t13 * TILE_STEP, t13 * SCALE_STEP, t3 * TILE_STEP, t3 * SCALE_STEP};
}
bool packed_ok(int E, int d, int F) { return E >= 1 && E <= KMOE_MAX_EXPERTS && d > 0 && d % 64 == 0 && F > 0; }
}  // namespace

extern "C" size_t kmoe_packed_mx_bytes(int E, int d, int F, int which) {
  if (!packed_ok(E, d, F)) return 0;
  const PackedSizes z = packed_sizes(E, d, F);
  return (size_t)(which == 0 ? z.w13 : which == 1 ? z.s13 : which == 2 ? z.w3 : which == 3 ? z.s3 : 0);
}

extern "C" int kmoe_pack_weights_mx(const void* w1, const void* w2, const void* w3, int w_dtype, int E, int d, int F,
                                    void* w13_packed, uint8_t* w13_scale, void* w3_packed, uint8_t* w3_scale,
                                    void* stream) {
  KMOE_REQUIRE(w1 && w2 && w3 && w13_packed && w13_scale && w3_packed && w3_scale, KMOE_ERR_NULL,
               "kmoe_pack_weights_mx: null buffer");
  KMOE_REQUIRE(is_float(w_dtype), KMOE_ERR_DTYPE, "kmoe_pack_weights_mx: dtype %d", w_dtype);
  KMOE_REQUIRE(packed_ok(E, d, F), KMOE_ERR_SHAPE,
               "kmoe_pack_weights_mx: E=%d (1..%d), d=%d (a multiple of 64), F=%d", E, KMOE_MAX_EXPERTS, d, F);
  hipStream_t s = kmoe::as_stream(stream);
  const int Fp = round_up(F, 128), dp = round_up(d, 256);
  auto one = [&](const void* w, int K, int N, int Np, bool gate_up, int half, int tiles, void* q, uint8_t* sc) {
    const bool f32 = w_dtype == KMOE_DTYPE_F32;
    const int C = four_columns(w, f32, N) ? 4 : 1;
    const dim3 grid(grid_of((int64_t)E * (round_up(K, STEP) / BLOCK) * (Np / C), 256));
    uint8_t* qp = static_cast<uint8_t*>(q);
    if (f32 && C == 4)
      hipLaunchKernelGGL((pack_mx_kernel<true, 4>), grid, dim3(256), 0, s, w, E, K, N, Np, gate_up, half, tiles, qp, sc);
    else if (f32)
      hipLaunchKernelGGL((pack_mx_kernel<true, 1>), grid, dim3(256), 0, s, w, E, K, N, Np, gate_up, half, tiles, qp, sc);
    else if (C == 4)
      hipLaunchKernelGGL((pack_mx_kernel<false, 4>), grid, dim3(256), 0, s, w, E, K, N, Np, gate_up, half, tiles, qp, sc);
    else
      hipLaunchKernelGGL((pack_mx_kernel<false, 1>), grid, dim3(256), 0, s, w, E, K, N, Np, gate_up, half, tiles, qp, sc);
  };
  one(w1, d, F, Fp, true, 0, Fp / 128, w13_packed, w13_scale);
  one(w2, d, F, Fp, true, 1, Fp / 128, w13_packed, w13_scale);
  one(w3, F, d, dp, false, 0, dp / 256, w3_packed, w3_scale);
  return kmoe::check_launch("kmoe_pack_weights_mx");
}
