// Grouped expert products over microscaled rows: launch choice and C entry points.  The
// kernels are in kmoe_mx_gemm.h.
#include <algorithm>

#include "kmoe_mx_gemm.h"

using namespace kmoe_mx;

namespace {

// Tile of a product of max_rows rows over E experts, by the number of 64 x 256 tiles that they
// come to where rows spread over the experts.  Up to 1.5 of those a CU, half as wide tiles use
// the idle CUs; from there on the width halves the reads of rows.  128 rows halve the reads of
// weights: with e2m1 rows where the experts have more than 64 and the tiles fill the CUs; with
// e4m3 rows, of which two workgroups fit a CU with two LDS stages only, from 5 tiles a CU.  us
// for 64x128 / 64x256 / 128x256, weights from HBM, (tiles a CU): top-2 of 16, d 2048, F 2816,
// e4m3: down, 48 tokens (0.5) 13.8 / 15.6 / 27; 777 (1) 22.5 / 23.5 / 28; 2042 (2.2) 36 / 35 /
// 37; gate/up, 48 (1.4) 22.6 / 22.3 / 30; 1024 (3.4) 43 / 39 / 48; 2042 (6.2) 63 / 58 / 58; 4096
// (12) 115 / 97 / 99; e2m1: down, 500 (0.8) 17.4 / 15.3 / 17.5; 777 (1) 21.5 / 22 / 18; 2042 33 /
// 31 / 32; gate/up, 777 (2.8) 34 / 32 / 27; 2042 55 / 51 / 45.  Top-6 of 64, d 1024, F 704,
// gate/up: e4m3, 400 (1.6) 17.6 / 15.3 / 19.6; 2000 (5.1) 34 / 31 / 31; e2m1, 400 15.5 / 14.7 /
// 17.1; 1000 (93 rows an expert, 2.9) 19.1 / 19.2 / 18.8.  The 1.5 is e4m3's: the e2m1 product of
// 500 tokens (0.8) loses 12 % by it.
MxTileSize tile_size(bool fp4, int64_t max_rows, int E, int b_tiles) {
  const int64_t used = std::min<int64_t>(max_rows, E), tiles = std::max(used, max_rows / 64 + used / 2) * b_tiles;
  const int64_t cu = kmoe::cu_count();
  if (fp4 ? max_rows > 64 * (int64_t)E && tiles >= cu : tiles > 5 * cu) return MxTileSize::R128xC256;
  return 2 * tiles <= 3 * cu ? MxTileSize::R64xC128 : MxTileSize::R64xC256;
}

// Whether a product runs on the small-row kernel (kmoe_mx_gemm_small.hip): where its grid is at
// most two workgroups per CU, as latency then counts, at few rows per expert.  us, small-row
// kernel / 64 x 128 tiles, e4m3, weights from HBM (workgroups): top-2 of 16 experts, d 2048, F
// 2816, down, 1 token (128) 4.9 / 9.8, 4 (512) 8.0 / 10.0, 16 (1088) 14.9 / 13.3; gate/up, 1
// (176) 6.5 / 9.0, 2 (352) 9.7 / 9.1, 4 (704) 14.1 / 12.6, 48 (1672) 31 / 22; top-2 of 8, d 4096,
// F 1408, gate/up, 4 (352) 9.5 / 18.3, 48 (484) 18.0 / 20.1, 100 (616) 23.5 / 20.1; of the first shape 2 tokens
// lose 6 % by the limit: each
// workgroup looks its slot up and reduces, which the tiles do once for four times the weights.
bool small_product(bool gate_up, int64_t max_rows, int E, int b_tiles) {
  const int64_t slots = max_rows / SMALL_ROWS + std::min<int64_t>(max_rows, E);
  return max_rows <= 32 * (int64_t)E && slots * b_tiles * (gate_up ? 4 : 8) <= 2 * kmoe::cu_count();
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
  return KMOE_OK;
}

// Picks a product's kernel and launches it, if its grid is one that a launch takes (fewer than 2^24 workgroups of
// 256; the small-row kernel's is a few per CU).
int launch(const char* who, const MxLaunch& l, bool gate_up, bool fp4) {
  if (small_product(gate_up, l.max_rows, l.g.E, l.g.b_tiles)) {
    launch_mx_small(l, gate_up, fp4);
    return kmoe::check_launch(who);
  }
  const MxTileSize t = tile_size(fp4, l.max_rows, l.g.E, l.g.b_tiles);
  const int rows = t == MxTileSize::R128xC256 ? 128 : 64, split = t == MxTileSize::R64xC128 ? 2 : 1;
  KMOE_REQUIRE(mx_workgroups(l.max_rows, l.g.E, l.g.b_tiles, rows, split) < 1 << 24, KMOE_ERR_SHAPE, "%s: grid too large",
               who);
  if (gate_up)
    launch_mx_gate_up(l, fp4, t);
  else
    launch_mx_down(l, fp4, t);
  return kmoe::check_launch(who);
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
  return launch("kmoe_gemm_gate_up_mx", l, true, fmt == KMOE_DTYPE_FP4_E2M1);
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
  return launch("kmoe_gemm_down_mx", l, false, fmt == KMOE_DTYPE_FP4_E2M1);
}
