// Grouped expert products over microscaled rows: launch choice and C entry points.  The
// kernels are in kmoe_mx_gemm.h.
#include <algorithm>

#include "kmoe_mx_gemm.h"

using namespace kmoe_mx;

namespace {

// Rows of a tile for max_rows rows over E experts.
int tile_rows(int64_t max_rows, int E) {
  const int64_t per = max_rows / E;
  return per > 64 ? 128 : 64;
}

// Whether a product runs on the small-row kernel (kmoe_mx_gemm_small.hip): where its grid is at
// most three workgroups per CU, as latency then counts, at few rows per expert.  Kernel times
// in us, small-row kernel / 64-row tiles, top-2 of 16 experts, d 2048, F 2816, w4a8: 1 token
// (176 workgroups in gate/up, 128 in down) 6.1 / 11.2 and 5.2 / 12.7; 4 tokens (704, 512) 9.8 /
// 11.9 and 7.5 / 12.7; 8 tokens (1408, 1024) 19.5 / 12.8 and 10.4 / 12.7; 48 tokens (1672,
// 1216) 28 / 20 and 15.7 / 13.5; 32 rows of 64 experts, d 1024, F 704 (792, 1056) 12.5 / 8.1
// and 7.5 / 6.3: each workgroup looks its slot up and reduces, which the tiles do once for
// eight times the weights.
bool small_product(bool gate_up, int64_t max_rows, int E, int b_tiles) {
  const int64_t slots = max_rows / SMALL_ROWS + std::min<int64_t>(max_rows, E);
  return max_rows <= 32 * (int64_t)E && slots * b_tiles * (gate_up ? 4 : 8) <= 3 * kmoe::cu_count();
}

int check(const char* who, const void* a, const uint8_t* a_scale, int fmt, const int32_t* offsets, int E, int d, int F,
          int64_t max_rows, const void* w, const uint8_t* ws, int64_t a_rows, int K) {
  KMOE_REQUIRE(a && a_scale && offsets && w && ws, KMOE_ERR_NULL, "%s: null buffer", who);
  KMOE_REQUIRE(fmt == KMOE_DTYPE_FP8_E4M3 || fmt == KMOE_DTYPE_FP4_E2M1, KMOE_ERR_DTYPE,
               "%s: element type %d is neither e4m3 nor e2m1", who, fmt);
  KMOE_REQUIRE(E >= 1 && E <= KMOE_MAX_EXPERTS, KMOE_ERR_SHAPE, "%s: E=%d out of range", who, E);
  KMOE_REQUIRE(d > 0 && d % 64 == 0 && F > 0, KMOE_ERR_SHAPE, "%s: d=%d must be a positive multiple of 64, F=%d > 0", who,
               d, F);
  KMOE_REQUIRE(max_rows >= 0 && max_rows < (int64_t)1 << 31, KMOE_ERR_SHAPE, "%s: max_rows out of range", who);
  // loads address 2 GiB from the first row of a gathered matrix, of a tile and of a weight tile
  const int64_t lda = row_bytes(fmt == KMOE_DTYPE_FP4_E2M1, K);
  KMOE_REQUIRE((a_rows + 1) * lda < (int64_t)1 << 31 && 257 * lda < (int64_t)1 << 31 &&
                   (int64_t)round_up(K, STEP) * 128 < (int64_t)1 << 31,
               KMOE_ERR_SHAPE, "%s: operand too large for 32-bit offsets (%lld rows, K=%d)", who, (long long)a_rows, K);
  // a launch takes 2^24 workgroups of 256, 2^23 of 512
  KMOE_REQUIRE((max_rows / SMALL_ROWS + E) * (int64_t)std::max(round_up(F, 128) / 32, round_up(d, 256) / 32) < 1 << 23,
               KMOE_ERR_SHAPE, "%s: grid too large", who);
  return KMOE_OK;
}

}  // namespace

extern "C" int kmoe_gemm_gate_up_mx(const void* xq, const uint8_t* x_scale, int fmt, int64_t n_x_rows,
                                    const int32_t* row_token, const int32_t* offsets, int E, int d, int F,
                                    int64_t max_rows, const void* w13_packed, const uint8_t* w13_scale, void* hq,
                                    uint8_t* h_scale, void* gu, void* stream) {
  const int rc = check("kmoe_gemm_gate_up_mx", xq, x_scale, fmt, offsets, E, d, F, max_rows, w13_packed, w13_scale,
                       row_token ? n_x_rows : 0, d);
  if (rc) return rc;
  KMOE_REQUIRE(hq && h_scale, KMOE_ERR_NULL, "kmoe_gemm_gate_up_mx: null output");
  KMOE_REQUIRE(!row_token || n_x_rows >= 1, KMOE_ERR_SHAPE, "kmoe_gemm_gate_up_mx: n_x_rows=%lld must be >= 1",
               (long long)n_x_rows);
  if (max_rows == 0) return KMOE_OK;
  const int Fp = round_up(F, 128);
  MxLaunch l{};
  l.g.a = static_cast<const uint8_t*>(xq);
  l.g.a_scale = x_scale;
  l.g.a_rows = n_x_rows;
  l.g.row_token = row_token;
  l.g.offsets = offsets;
  l.g.E = E;
  l.g.k_steps = round_up(d, STEP) / STEP;
  l.g.b = static_cast<const uint8_t*>(w13_packed);
  l.g.b_scale = w13_scale;
  l.g.b_tiles = Fp / 128;
  l.g.q = static_cast<uint8_t*>(hq);
  l.g.q_scale = h_scale;
  l.g.gu = static_cast<uint16_t*>(gu);
  l.g.ldc = Fp;
  l.max_rows = max_rows;
  l.s = kmoe::as_stream(stream);
  if (small_product(true, max_rows, E, l.g.b_tiles))
    launch_mx_small(l, true, fmt == KMOE_DTYPE_FP4_E2M1);
  else
    launch_mx_gate_up(l, fmt == KMOE_DTYPE_FP4_E2M1, tile_rows(max_rows, E));
  return kmoe::check_launch("kmoe_gemm_gate_up_mx");
}

extern "C" int kmoe_gemm_down_mx(const void* hq, const uint8_t* h_scale, int fmt, const int32_t* offsets, int E, int d,
                                 int F, int64_t max_rows, const void* w3_packed, const uint8_t* w3_scale, void* y,
                                 void* stream) {
  const int rc = check("kmoe_gemm_down_mx", hq, h_scale, fmt, offsets, E, d, F, max_rows, w3_packed, w3_scale, 0, F);
  if (rc) return rc;
  KMOE_REQUIRE(y, KMOE_ERR_NULL, "kmoe_gemm_down_mx: null output");
  if (max_rows == 0) return KMOE_OK;
  MxLaunch l{};
  l.g.a = static_cast<const uint8_t*>(hq);
  l.g.a_scale = h_scale;
  l.g.a_rows = max_rows;
  l.g.offsets = offsets;
  l.g.E = E;
  l.g.k_steps = round_up(F, STEP) / STEP;
  l.g.b = static_cast<const uint8_t*>(w3_packed);
  l.g.b_scale = w3_scale;
  l.g.b_tiles = round_up(d, 256) / 256;
  l.g.c = static_cast<uint16_t*>(y);
  l.g.ldc = d;
  l.g.n_valid = d;
  l.max_rows = max_rows;
  l.s = kmoe::as_stream(stream);
  if (small_product(false, max_rows, E, l.g.b_tiles))
    launch_mx_small(l, false, fmt == KMOE_DTYPE_FP4_E2M1);
  else
    launch_mx_down(l, fmt == KMOE_DTYPE_FP4_E2M1, tile_rows(max_rows, E));
  return kmoe::check_launch("kmoe_gemm_down_mx");
}
