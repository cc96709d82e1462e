// Entry points of the dense products (kmoe_dense.h): host checks and the choice of a tile.
#include <initializer_list>

#include "kmoe_dense_launch.h"

using namespace kmoe_dense;

namespace {

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace

#define KMOE_DENSE_SIZES(who, M, N, K)                                                                                   \
  KMOE_REQUIRE((M) >= 0 && (N) > 0 && (K) > 0 && (N) % 8 == 0 && (K) % 8 == 0 && (M) < ((int64_t)1 << 31), KMOE_ERR_SHAPE, \
               who ": %lld rows of %d and %d values (positive multiples of 8)", (long long)(M), (int)(K), (int)(N))
#define KMOE_DENSE_ALIGNED(who, ...)                                            \
  for (const void* p_ : std::initializer_list<const void*>{__VA_ARGS__})                                        \
  KMOE_REQUIRE(aligned(p_), KMOE_ERR_SHAPE, who ": buffers are aligned to 16 bytes")
#define KMOE_DENSE_LOST(who, lost, T)                                                                           \
  KMOE_REQUIRE(!(lost) || (T) <= LOST_ROWS, KMOE_ERR_SHAPE, who ": %lld rows with what they lost (at most %d)", \
               (long long)(T), LOST_ROWS)

extern "C" size_t kmoe_dense_saved_bytes(int64_t T, int F) {
  return T <= 0 || F <= 0 ? 0 : (size_t)kmoe::ceil_div<int64_t>(T, 16) * kmoe::ceil_div(F, 16) * SAVED_BLOCK;
}

extern "C" int kmoe_dense_gate_up(const void* x, int64_t T, int d, const void* w_gate, const void* w_up, int F, int act,
                                  void* h, int lost, void* saved, void* stream) {
  KMOE_DENSE_SIZES("kmoe_dense_gate_up", T, F, d);
  KMOE_REQUIRE(act >= KMOE_ACT_SILU && act <= KMOE_ACT_RELU, KMOE_ERR_UNSUPPORTED, "kmoe_dense_gate_up: activation %d", act);
  if (T == 0) return KMOE_OK;
  KMOE_REQUIRE(x && w_gate && w_up && h, KMOE_ERR_NULL, "kmoe_dense_gate_up: null buffer");
  KMOE_DENSE_ALIGNED("kmoe_dense_gate_up", x, w_gate, w_up, h, saved);
  Args g{};
  g.a[0] = static_cast<const uint16_t*>(x);
  g.b[0] = static_cast<const uint16_t*>(w_gate), g.b[1] = static_cast<const uint16_t*>(w_up);
  g.K = d, g.lda = d, g.ldb = d, g.M = T, g.N = F, g.ldc = F, g.c = h, g.act = act;
  g.saved = static_cast<uint8_t*>(saved);
  KMOE_DENSE_LOST("kmoe_dense_gate_up", lost, T);
  g.lost = lost ? T * F : 0;
  return launch_gated(g, kmoe::as_stream(stream));
}

extern "C" int kmoe_dense_linear(const void* x, int lost, int64_t T, int K, const void* w, int N, void* y,
                                 void* stream) {
  KMOE_DENSE_SIZES("kmoe_dense_linear", T, N, K);
  if (T == 0) return KMOE_OK;
  KMOE_REQUIRE(x && w && y, KMOE_ERR_NULL, "kmoe_dense_linear: null buffer");
  KMOE_DENSE_ALIGNED("kmoe_dense_linear", x, w, y);
  Args g{};
  g.a[0] = static_cast<const uint16_t*>(x), g.b[0] = static_cast<const uint16_t*>(w);
  g.K = K, g.lda = K, g.ldb = K, g.M = T, g.N = N, g.ldc = N, g.c = y;
  KMOE_DENSE_LOST("kmoe_dense_linear", lost, T);
  g.fold = lost ? T * K : 0;
  return launch_linear(g, kmoe::as_stream(stream));
}

extern "C" int kmoe_dense_dh(const void* dy, int64_t T, int d, const void* w_down, int F, const void* saved, void* dgate,
                             void* dup, int lost, void* stream) {
  KMOE_DENSE_SIZES("kmoe_dense_dh", T, F, d);
  if (T == 0) return KMOE_OK;
  KMOE_REQUIRE(dy && w_down && saved && dgate && dup, KMOE_ERR_NULL, "kmoe_dense_dh: null buffer");
  KMOE_DENSE_ALIGNED("kmoe_dense_dh", dy, w_down, saved, dgate, dup);
  Args g{};
  g.a[0] = static_cast<const uint16_t*>(dy), g.b[0] = static_cast<const uint16_t*>(w_down);
  g.K = d, g.lda = d, g.ldb = F, g.M = T, g.N = F, g.ldc = F, g.c = dgate;
  g.c2 = static_cast<uint16_t*>(dup);
  g.saved = static_cast<uint8_t*>(const_cast<void*>(saved));
  KMOE_DENSE_LOST("kmoe_dense_dh", lost, T);
  g.lost = lost ? T * F : 0;
  return launch_dh(g, kmoe::as_stream(stream));
}

extern "C" int kmoe_dense_dx(const void* dy, const void* dy2, int lost, int64_t T, int N, const void* w, const void* w2, int K,
                             void* dx, void* stream) {
  KMOE_DENSE_SIZES("kmoe_dense_dx", T, N, K);
  if (T == 0) return KMOE_OK;
  KMOE_REQUIRE(dy && w && dx && !dy2 == !w2, KMOE_ERR_NULL, "kmoe_dense_dx: null buffer");
  KMOE_DENSE_ALIGNED("kmoe_dense_dx", dy, dy2, w, w2, dx);
  Args g{};
  g.a[0] = static_cast<const uint16_t*>(dy), g.b[0] = static_cast<const uint16_t*>(w);
  g.a[1] = static_cast<const uint16_t*>(dy2), g.b[1] = static_cast<const uint16_t*>(w2);
  g.K = N, g.lda = N, g.ldb = K, g.M = T, g.N = K, g.ldc = K, g.c = dx;
  KMOE_DENSE_LOST("kmoe_dense_dx", lost, T);
  g.fold = lost ? T * N : 0;
  hipStream_t s = kmoe::as_stream(stream);
  return dy2 ? launch_dx_two(g, s) : launch_dx(g, s);
}

extern "C" int kmoe_dense_wgrad(const void* a, const void* b, const void* a2, const void* b2, int64_t T, int M, int N,
                                void* c, int c_dtype, void* stream) {
  // (the rows are the product's K: its steps of up to 64 are counted in 32 bits)
  KMOE_REQUIRE(T >= 0 && T < ((int64_t)1 << 31) - 63 && M > 0 && N > 0 && M % 8 == 0 && N % 8 == 0, KMOE_ERR_SHAPE,
               "kmoe_dense_wgrad: %lld rows (below 2^31 - 63) of %d and %d values (positive multiples of 8)", (long long)T, M, N);
  KMOE_REQUIRE(c_dtype == KMOE_DTYPE_BF16 || c_dtype == KMOE_DTYPE_F32, KMOE_ERR_DTYPE, "kmoe_dense_wgrad: dtype %d", c_dtype);
  KMOE_REQUIRE(((a && b) || T == 0) && c && !a2 == !b2, KMOE_ERR_NULL, "kmoe_dense_wgrad: null buffer");
  KMOE_DENSE_ALIGNED("kmoe_dense_wgrad", a, b, a2, b2, c);
  Args g{};
  g.a[0] = static_cast<const uint16_t*>(a), g.b[0] = static_cast<const uint16_t*>(b);
  g.a[1] = static_cast<const uint16_t*>(a2), g.b[1] = static_cast<const uint16_t*>(b2);
  g.K = (int)T, g.lda = M, g.ldb = N, g.M = M, g.N = N, g.ldc = N, g.c = c;
  g.c_f32 = c_dtype == KMOE_DTYPE_F32;
  hipStream_t s = kmoe::as_stream(stream);
  return a2 && T > 0 ? launch_wgrad_two(g, s) : launch_wgrad(g, s);
}
