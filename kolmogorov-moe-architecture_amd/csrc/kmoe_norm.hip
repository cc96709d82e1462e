// RMSNorm forward and backward at the MoE block's boundary, for the training path.
//
// RMSNorm (moe_arch/model/embeddings.py:167-195):  n = g * x * r,  r = 1/sqrt(mean(x^2) + eps)
// Backward, per row (d columns):
//   dx_c = r g_c dn_c - (r^3 / d) x_c sum_c' g_c' dn_c' x_c'   (+ dres_c, the residual's gradient)
//   dg_c = sum_t dn_tc x_tc r_t
// Both kernels hold one row per wave in registers (lane l holds the 8-element vectors
// l, l + 64, ... of the row), so each row is read once; HBM-bound.  The training
// forward materialises n (bf16): the backward's weight gradients need the normalised
// rows, which the inference path's fold of g into the weights never writes.
#include <type_traits>

#include "kmoe_mx.h"

namespace {

// Rows in flight per workgroup, and the most row segments of the backward (each writes a
// d-float partial of dg that a second kernel reduces).  Measured at T = 16384, d = 2048:
// 4 waves / 1024 segments 58 us, 4 / 512 52, 8 / 512 54, 8 / 256 50.5, 4 / 4096 121
// (the partial sums' reduction dominates with many segments).
constexpr int NORM_WAVES = 8;
constexpr int NORM_MAX_SEGS = 256;
constexpr int NORM_FWD_WAVES = 4;  // forward: one row per wave, 4 per workgroup (8: 32 -> 37 us)

// 8 consecutive elements (bf16 or f32) as floats
template <bool F32>
__device__ __forceinline__ void load8(const void* __restrict__ base, int64_t elem, float (&v)[8]) {
  if constexpr (F32) {
    const f32x4_t* p = reinterpret_cast<const f32x4_t*>(static_cast<const float*>(base) + elem);
    const f32x4_t a = p[0], b = p[1];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      v[q] = a[q];
      v[4 + q] = b[q];
    }
  } else {
    const i32x4_t a = *reinterpret_cast<const i32x4_t*>(static_cast<const uint16_t*>(base) + elem);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      v[2 * q] = __uint_as_float(((uint32_t)a[q]) << 16);
      v[2 * q + 1] = __uint_as_float(((uint32_t)a[q]) & 0xffff0000u);
    }
  }
}

template <bool F32>
__device__ __forceinline__ void store8(void* __restrict__ base, int64_t elem, const float (&v)[8]) {
  if constexpr (F32) {
    f32x4_t a, b;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      a[q] = v[q];
      b[q] = v[4 + q];
    }
    f32x4_t* p = reinterpret_cast<f32x4_t*>(static_cast<float*>(base) + elem);
    p[0] = a;
    p[1] = b;
  } else {
    i32x4_t a;
#pragma unroll
    for (int q = 0; q < 4; ++q) a[q] = (int)((uint32_t)f32_to_bf16(v[2 * q]) | ((uint32_t)f32_to_bf16(v[2 * q + 1]) << 16));
    *reinterpret_cast<i32x4_t*>(static_cast<uint16_t*>(base) + elem) = a;
  }
}

__device__ __forceinline__ void load8_any(const void* __restrict__ base, bool f32, int64_t elem, float (&v)[8]) {
  if (f32)
    load8<true>(base, elem, v);
  else
    load8<false>(base, elem, v);
}

// n[t] = bf16(g * x[t] * r_t), rrms[t] = r_t.  One wave per row.  With w_mod, also
// mod_logits[t] = n[t] . w_mod over the rounded n, in the lane / vector / wave-sum order
// of the MoD selection's own logits kernel (so the selection is the same as from n).
template <int NV, bool XF32>
__global__ __launch_bounds__(64 * NORM_FWD_WAVES) void rmsnorm_kernel(const void* __restrict__ x,
                                                                  const void* __restrict__ g, bool g_f32, float eps,
                                                                  int64_t T, int d, uint16_t* __restrict__ n,
                                                                  float* __restrict__ rrms,
                                                                  const uint16_t* __restrict__ w_mod,
                                                                  float* __restrict__ mod_logits) {
  const int lane = threadIdx.x & 63;
  const int64_t t = (int64_t)blockIdx.x * NORM_FWD_WAVES + (threadIdx.x >> 6);
  if (t >= T) return;
  const int nvec = d / 8;
  float xv[NV][8];
  float ss = 0.0f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = lane + 64 * i;
    if (v < nvec) {
      load8<XF32>(x, t * d + (int64_t)v * 8, xv[i]);
#pragma unroll
      for (int q = 0; q < 8; ++q) ss = fmaf(xv[i][q], xv[i][q], ss);
    }
  }
  ss = wave_sum(ss);
  const float r = 1.0f / sqrtf(ss / (float)d + eps);
  float ml = 0.0f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = lane + 64 * i;
    if (v < nvec) {
      float gv[8], o[8];
      load8_any(g, g_f32, (int64_t)v * 8, gv);
#pragma unroll
      for (int q = 0; q < 8; ++q) o[q] = gv[q] * (xv[i][q] * r);
      store8<false>(n, t * d + (int64_t)v * 8, o);
      if (w_mod) {
        float wv[8];
        load8<false>(w_mod, (int64_t)v * 8, wv);
#pragma unroll
        for (int q = 0; q < 8; ++q) ml = fmaf(bf16_to_f32(f32_to_bf16(o[q])), wv[q], ml);
      }
    }
  }
  if (w_mod) {
    ml = wave_sum(ml);
    if (lane == 0) mod_logits[t] = ml;
  }
  if (lane == 0) rrms[t] = r;
}

// One row's inputs as loaded (bf16: one 16-byte vector per 8 elements, f32: two).
template <bool F32>
struct Raw8 {
  i32x4_t v[F32 ? 2 : 1];
};
template <bool F32>
__device__ __forceinline__ void load_raw(const void* __restrict__ base, int64_t elem, Raw8<F32>& r) {
  const i32x4_t* p = reinterpret_cast<const i32x4_t*>(static_cast<const uint8_t*>(base) + elem * (F32 ? 4 : 2));
  r.v[0] = p[0];
  if constexpr (F32) r.v[1] = p[1];
}
template <bool F32>
__device__ __forceinline__ void unpack_raw(const Raw8<F32>& r, float (&v)[8]) {
  if constexpr (F32) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      v[q] = __int_as_float(r.v[0][q]);
      v[4 + q] = __int_as_float(r.v[1][q]);
    }
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      v[2 * q] = __uint_as_float(((uint32_t)r.v[0][q]) << 16);
      v[2 * q + 1] = __uint_as_float(((uint32_t)r.v[0][q]) & 0xffff0000u);
    }
  }
}

// h = x + delta rounded to x's type (without delta h is x, not written), n = bf16(g * (h r)), r =
// 1/sqrt(mean(h^2) + eps), all from the rounded h (what the backward and the next block read),
// and n's microscaled rows (Q 1: e4m3, 2: e2m1; 0: none).  The rows are those of the bf16 n, so
// the experts' products see the values that the router sees, and the codes do not depend on the
// norm being fused.  Sums as in rmsnorm_kernel, so n is that of a torch addition followed by
// kmoe_rmsnorm, bit for bit.  One wave per row.  Memory bounds it, at few rows its latency: a
// row's loads (up to d 2048 the weight's too) go out before the first is waited for.  bf16 with
// e4m3 rows, d 2048: 16384 rows 56 us, 5.4 TB/s (each vector waited for on its own 65), 48 rows 7.4
// (8.7), one wave's walk over a whole row.  Without codes, d 4096 / 8192: bf16 4.4 / 2.8 TB/s, f32 5.7 / 4.2.
template <int NV, bool XF32, int Q>
__global__ __launch_bounds__(64 * NORM_FWD_WAVES) void add_rmsnorm_kernel(
    const void* __restrict__ x, const void* __restrict__ delta, bool delta_f32, const void* __restrict__ g, bool g_f32,
    float eps, int64_t T, int d, void* __restrict__ h, uint16_t* __restrict__ n, float* __restrict__ rrms,
    uint8_t* __restrict__ q, uint8_t* __restrict__ scale) {
  const int lane = threadIdx.x & 63;
  const int64_t t = (int64_t)blockIdx.x * NORM_FWD_WAVES + (threadIdx.x >> 6);
  if (t >= T) return;
  const int nvec = d / 8;
  constexpr bool EARLY_G = NV <= 4;
  auto at = [&](int i) { return (int64_t)min(lane + 64 * i, nvec - 1) * 8; };  // lanes past the row read its end
  Raw8<XF32> xr[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) load_raw<XF32>(x, t * d + at(i), xr[i]);
  Raw8<true> gr[EARLY_G ? NV : 1];
  auto early_g = [&]() {
    if constexpr (EARLY_G) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const i32x4_t* const p = reinterpret_cast<const i32x4_t*>(static_cast<const uint8_t*>(g) + at(i) * (g_f32 ? 4 : 2));
        gr[i].v[0] = p[0];
        gr[i].v[1] = p[g_f32 ? 1 : 0];
      }
    }
  };
  float hv[NV][8];
  auto add = [&](auto f32_tag) {
    constexpr bool F32 = decltype(f32_tag)::value;
    Raw8<F32> dr[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) load_raw<F32>(delta, t * d + at(i), dr[i]);
    early_g();
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float dv[8];
      unpack_raw<XF32>(xr[i], hv[i]);
      unpack_raw<F32>(dr[i], dv);
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        hv[i][c] += dv[c];
        if (!XF32) hv[i][c] = bf16_to_f32(f32_to_bf16(hv[i][c]));
      }
      if (lane + 64 * i < nvec) store8<XF32>(h, t * d + at(i), hv[i]);
    }
  };
  if (!delta) {
    early_g();
#pragma unroll
    for (int i = 0; i < NV; ++i) unpack_raw<XF32>(xr[i], hv[i]);
  } else if (delta_f32) {
    add(std::true_type{});
  } else {
    add(std::false_type{});
  }
  float ss = 0.0f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (lane + 64 * i < nvec) {
#pragma unroll
      for (int c = 0; c < 8; ++c) ss = fmaf(hv[i][c], hv[i][c], ss);
    }
  ss = wave_sum(ss);
  const float r = 1.0f / sqrtf(ss / (float)d + eps);
  if (lane == 0) rrms[t] = r;
  const int qvec = Q ? kmoe_mx::round_up(d, kmoe_mx::STEP) / 8 : nvec;  // with the padding of a coded row
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = lane + 64 * i;
    if (v < qvec) {  // d is a multiple of 32 with Q: the four lanes of a block agree
      float o[8] = {};
      if (v < nvec) {
        float gv[8];
        if constexpr (!EARLY_G) {
          load8_any(g, g_f32, (int64_t)v * 8, gv);
        } else if (g_f32) {
          unpack_raw<true>(gr[i], gv);
        } else {
          unpack_raw<false>(Raw8<false>{{gr[i].v[0]}}, gv);
        }
#pragma unroll
        for (int c = 0; c < 8; ++c) o[c] = bf16_to_f32(f32_to_bf16(gv[c] * (hv[i][c] * r)));
        store8<false>(n, t * d + (int64_t)v * 8, o);
      }
      if constexpr (Q != 0) {
        uint32_t code;
        const kmoe_mx::Codes<Q == 2, 8> w = kmoe_mx::encode_quad<Q == 2>(o, code);
        if constexpr (Q == 2)
          *reinterpret_cast<uint32_t*>(q + t * (qvec * 4) + v * 4) = w.w[0];
        else
          *reinterpret_cast<i32x2_t*>(q + t * (qvec * 8) + v * 8) = i32x2_t{(int)w.w[0], (int)w.w[1]};
        if ((v & 3) == 0) scale[t * kmoe_mx::scale_bytes(d) + v / 4] = (uint8_t)code;
      }
    }
  }
}

template <int NV, bool XF32>
struct NormRow {
  Raw8<XF32> x[NV], res[NV];
  Raw8<false> dn[NV];
  float r;
};

// dx (dtype of x; with dx16 also rounded to bf16) and the per-segment partial sums of dg.  Workgroup = NORM_WAVES waves
// over the rows [seg * seg_rows, ...) of its segment, wave w taking every NORM_WAVES-th
// row (its x, dn and dres loads issued together); the waves' dg sums are then added in
// wave order through LDS and written as partial[seg][:] (reduced over segments afterwards
// in a fixed order).  HBM bounds it up to d 2048: bf16 / f32 rows with dres 4.7 / 5.6 TB/s.  Wider rows do
// not fit a lane's 256 registers: NV 8 spills 73 / 192 of them (d 4096: 2.5 / 2.8 TB/s), NV 16 793 / 919
// (d 8192: 0.7 / 1.2 TB/s).
template <int NV, bool XF32>
__global__ __launch_bounds__(64 * NORM_WAVES) void rmsnorm_bwd_kernel(
    const uint16_t* __restrict__ dn, const void* __restrict__ x, const void* __restrict__ g, bool g_f32,
    const float* __restrict__ rrms, const void* __restrict__ dres, int64_t T, int d, int64_t seg_rows,
    void* __restrict__ dx, uint16_t* __restrict__ dx16, float* __restrict__ partial) {
  __shared__ float red[NORM_WAVES][512];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int nvec = d / 8;
  float gv[NV][8], acc[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = lane + 64 * i;
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      gv[i][q] = 0.0f;
      acc[i][q] = 0.0f;
    }
    if (v < nvec) load8_any(g, g_f32, (int64_t)v * 8, gv[i]);
  }
  const int64_t t0 = (int64_t)blockIdx.x * seg_rows;
  const int64_t t1 = t0 + seg_rows < T ? t0 + seg_rows : T;
  const float inv_d = 1.0f / (float)d;
  auto load_row = [&](int64_t t, NormRow<NV, XF32>& R) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = lane + 64 * i;
      if (v < nvec) {
        load_raw<XF32>(x, t * d + (int64_t)v * 8, R.x[i]);
        load_raw<false>(dn, t * d + (int64_t)v * 8, R.dn[i]);
        if (dres) load_raw<XF32>(dres, t * d + (int64_t)v * 8, R.res[i]);
      }
    }
    R.r = rrms[t];
  };
  auto process = [&](int64_t t, const NormRow<NV, XF32>& R) {
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = lane + 64 * i;
      if (v < nvec) {
        float xv[8], dv[8];
        unpack_raw<XF32>(R.x[i], xv);
        unpack_raw<false>(R.dn[i], dv);
#pragma unroll
        for (int q = 0; q < 8; ++q) s = fmaf(gv[i][q] * dv[q], xv[q], s);
      }
    }
    s = wave_sum(s);
    const float r = R.r;
    const float c = r * r * r * s * inv_d;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = lane + 64 * i;
      if (v < nvec) {
        float xv[8], dv[8], rv[8], o[8];
        unpack_raw<XF32>(R.x[i], xv);
        unpack_raw<false>(R.dn[i], dv);
        if (dres) {
          unpack_raw<XF32>(R.res[i], rv);
        } else {
#pragma unroll
          for (int q = 0; q < 8; ++q) rv[q] = 0.0f;
        }
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          o[q] = rv[q] + (r * gv[i][q] * dv[q] - c * xv[q]);
          acc[i][q] = fmaf(dv[q] * xv[q], r, acc[i][q]);
        }
        store8<XF32>(dx, t * d + (int64_t)v * 8, o);
        if (XF32 && dx16) store8<false>(dx16, t * d + (int64_t)v * 8, o);
      }
    }
  };
  // one row at a time: a second row in flight (prefetch) needs 256 VGPRs at d = 2048 and
  // the lower occupancy made the kernel slower (75 vs 58 us at T = 16384, d = 2048)
  NormRow<NV, XF32> ra;
  for (int64_t t = t0 + w; t < t1; t += NORM_WAVES) {
    load_row(t, ra);
    process(t, ra);
  }
  // dg: per 512-column chunk, the waves' sums added in wave order
  float* out = partial + (int64_t)blockIdx.x * d;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
#pragma unroll
    for (int q = 0; q < 8; ++q) red[w][lane * 8 + q] = acc[i][q];
    __syncthreads();
    for (int c = threadIdx.x; c < 512; c += 64 * NORM_WAVES) {
      const int col = i * 512 + c;
      if (col < d) {
        float sum = red[0][c];
#pragma unroll
        for (int q = 1; q < NORM_WAVES; ++q) sum += red[q][c];
        out[col] = sum;
      }
    }
    __syncthreads();
  }
}

int64_t norm_seg_rows(int64_t T) {
  int64_t rows = kmoe::ceil_div<int64_t>(T, NORM_MAX_SEGS);
  rows = kmoe::ceil_div<int64_t>(rows, NORM_WAVES) * NORM_WAVES;
  return rows < NORM_WAVES ? NORM_WAVES : rows;
}

template <bool XF32>
int launch_norm(const void* x, const void* g, bool g_f32, float eps, int64_t T, int d, uint16_t* n, float* rrms,
                const uint16_t* w_mod, float* mod_logits, hipStream_t s) {
  const dim3 grid((unsigned)kmoe::ceil_div<int64_t>(T, NORM_FWD_WAVES)), block(64 * NORM_FWD_WAVES);
  const int nv = kmoe::ceil_div(d / 8, 64);
#define KMOE_NORM_CASE(NVV)                                                                                   \
  if (nv <= NVV) {                                                                                            \
    hipLaunchKernelGGL((rmsnorm_kernel<NVV, XF32>), grid, block, 0, s, x, g, g_f32, eps, T, d, n, rrms,    \
                       w_mod, mod_logits);                                                                  \
    return KMOE_OK;                                                                                           \
  }
  KMOE_NORM_CASE(1)
  KMOE_NORM_CASE(2)
  KMOE_NORM_CASE(4)
  KMOE_NORM_CASE(8)
  KMOE_NORM_CASE(16)
#undef KMOE_NORM_CASE
  return KMOE_ERR_UNSUPPORTED;
}

template <bool XF32>
int launch_norm_bwd(const uint16_t* dn, const void* x, const void* g, bool g_f32, const float* rrms, const void* dres,
                    int64_t T, int d, int64_t seg_rows, void* dx, uint16_t* dx16, float* partial, hipStream_t s) {
  const dim3 grid((unsigned)kmoe::ceil_div<int64_t>(T, seg_rows)), block(64 * NORM_WAVES);
  const int nv = kmoe::ceil_div(d / 8, 64);
#define KMOE_NORM_CASE(NVV)                                                                              \
  if (nv <= NVV) {                                                                                       \
    hipLaunchKernelGGL((rmsnorm_bwd_kernel<NVV, XF32>), grid, block, 0, s, dn, x, g, g_f32, rrms, dres, T, \
                       d, seg_rows, dx, dx16, partial);                                                  \
    return KMOE_OK;                                                                                      \
  }
  KMOE_NORM_CASE(1)
  KMOE_NORM_CASE(2)
  KMOE_NORM_CASE(4)
  KMOE_NORM_CASE(8)
  KMOE_NORM_CASE(16)
#undef KMOE_NORM_CASE
  return KMOE_ERR_UNSUPPORTED;
}

__global__ void zero_words_kernel(uint16_t* __restrict__ p, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) p[i] = 0;
}

template <bool XF32, int Q>
int launch_add_norm(const void* x, const void* delta, bool delta_f32, const void* g, bool g_f32, float eps, int64_t T, int d,
                    void* h, uint16_t* n, float* rrms, uint8_t* q, uint8_t* scale, hipStream_t s) {
  const dim3 grid((unsigned)kmoe::ceil_div<int64_t>(T, NORM_FWD_WAVES)), block(64 * NORM_FWD_WAVES);
  const int nv = kmoe::ceil_div((Q ? kmoe_mx::round_up(d, kmoe_mx::STEP) : d) / 8, 64);
#define KMOE_NORM_CASE(NVV)                                                                                          \
  if (nv <= NVV) {                                                                                                   \
    hipLaunchKernelGGL((add_rmsnorm_kernel<NVV, XF32, Q>), grid, block, 0, s, x, delta, delta_f32, g, g_f32, eps, T, \
                       d, h, n, rrms, q, scale);                                                                     \
    return KMOE_OK;                                                                                                  \
  }
  KMOE_NORM_CASE(1)
  KMOE_NORM_CASE(2)
  KMOE_NORM_CASE(4)
  KMOE_NORM_CASE(8)
  KMOE_NORM_CASE(16)
#undef KMOE_NORM_CASE
  return KMOE_ERR_UNSUPPORTED;
}

bool is_float_dtype(int dt) { return dt == KMOE_DTYPE_BF16 || dt == KMOE_DTYPE_F32; }

}  // namespace

extern "C" int kmoe_rmsnorm(const void* x, int x_dtype, const void* weight, int w_dtype, float eps, int64_t T, int d,
                            void* n, float* rrms, const void* w_mod, float* mod_logits, void* stream) {
  KMOE_REQUIRE(weight && (T == 0 || (x && n && rrms)), KMOE_ERR_NULL, "kmoe_rmsnorm: null buffer");
  KMOE_REQUIRE(!w_mod == !mod_logits, KMOE_ERR_NULL, "kmoe_rmsnorm: w_mod and mod_logits go together");
  KMOE_REQUIRE(is_float_dtype(x_dtype) && is_float_dtype(w_dtype), KMOE_ERR_DTYPE, "kmoe_rmsnorm: dtypes %d/%d",
               x_dtype, w_dtype);
  KMOE_REQUIRE(T >= 0 && d > 0 && d % 8 == 0, KMOE_ERR_SHAPE, "kmoe_rmsnorm: d=%d must be a positive multiple of 8",
               d);
  KMOE_REQUIRE(d <= 8192, KMOE_ERR_UNSUPPORTED, "kmoe_rmsnorm: d=%d > 8192", d);
  KMOE_REQUIRE(eps >= 0.0f, KMOE_ERR_SHAPE, "kmoe_rmsnorm: eps must be >= 0");
  if (T == 0) return KMOE_OK;
  hipStream_t s = kmoe::as_stream(stream);
  const bool g_f32 = w_dtype == KMOE_DTYPE_F32;
  const uint16_t* wm = static_cast<const uint16_t*>(w_mod);
  const int rc =
      x_dtype == KMOE_DTYPE_F32
          ? launch_norm<true>(x, weight, g_f32, eps, T, d, static_cast<uint16_t*>(n), rrms, wm, mod_logits, s)
          : launch_norm<false>(x, weight, g_f32, eps, T, d, static_cast<uint16_t*>(n), rrms, wm, mod_logits, s);
  if (rc != KMOE_OK) return rc;
  return kmoe::check_launch("kmoe_rmsnorm");
}

extern "C" int kmoe_add_rmsnorm(const void* x, int x_dtype, const void* delta, int delta_dtype, const void* weight,
                                int w_dtype, float eps, int64_t T, int d, void* h, void* n, float* rrms, int fmt, void* q,
                                uint8_t* scale, void* stream) {
  KMOE_REQUIRE(weight && (T == 0 || (x && n && rrms && (!delta || h))), KMOE_ERR_NULL, "kmoe_add_rmsnorm: null buffer");
  KMOE_REQUIRE(is_float_dtype(x_dtype) && is_float_dtype(delta_dtype) && is_float_dtype(w_dtype), KMOE_ERR_DTYPE,
               "kmoe_add_rmsnorm: dtypes %d/%d/%d", x_dtype, delta_dtype, w_dtype);
  const bool coded = fmt == KMOE_DTYPE_FP8_E4M3 || fmt == KMOE_DTYPE_FP4_E2M1;
  KMOE_REQUIRE(coded || fmt == KMOE_DTYPE_BF16, KMOE_ERR_DTYPE, "kmoe_add_rmsnorm: element type %d of the coded rows", fmt);
  KMOE_REQUIRE(!coded || T == 0 || (q && scale), KMOE_ERR_NULL, "kmoe_add_rmsnorm: coded rows need q and scale");
  KMOE_REQUIRE(T >= 0 && T < (int64_t)1 << 31 && d > 0 && d % 8 == 0 && (!coded || d % kmoe_mx::BLOCK == 0), KMOE_ERR_SHAPE,
               "kmoe_add_rmsnorm: d=%d must be a positive multiple of %d", d, coded ? kmoe_mx::BLOCK : 8);
  KMOE_REQUIRE(d <= 8192, KMOE_ERR_UNSUPPORTED, "kmoe_add_rmsnorm: d=%d > 8192", d);
  KMOE_REQUIRE(eps >= 0.0f, KMOE_ERR_SHAPE, "kmoe_add_rmsnorm: eps must be >= 0");
  if (T == 0) return KMOE_OK;
  hipStream_t s = kmoe::as_stream(stream);
  const bool g_f32 = w_dtype == KMOE_DTYPE_F32, d_f32 = delta_dtype == KMOE_DTYPE_F32;
  uint16_t* np = static_cast<uint16_t*>(n);
  uint8_t* qp = static_cast<uint8_t*>(q);
  auto with = [&](auto xf32, auto qt) {
    return launch_add_norm<decltype(xf32)::value, decltype(qt)::value>(x, delta, d_f32, weight, g_f32, eps, T, d, h, np, rrms,
                                                                       qp, scale, s);
  };
  auto by_x = [&](auto qt) {
    return x_dtype == KMOE_DTYPE_F32 ? with(std::true_type{}, qt) : with(std::false_type{}, qt);
  };
  const int rc = !coded                       ? by_x(std::integral_constant<int, 0>{})
                 : fmt == KMOE_DTYPE_FP8_E4M3 ? by_x(std::integral_constant<int, 1>{})
                                              : by_x(std::integral_constant<int, 2>{});
  if (rc != KMOE_OK) return rc;
  return kmoe::check_launch("kmoe_add_rmsnorm");
}

extern "C" size_t kmoe_rmsnorm_bwd_workspace_bytes(int64_t T, int d) {
  if (T <= 0 || d <= 0) return 0;
  return (size_t)kmoe::ceil_div<int64_t>(T, norm_seg_rows(T)) * (size_t)d * sizeof(float);
}

static int norm_bwd(const char* who, const void* dn, const void* x, int x_dtype, const void* weight, int w_dtype,
                    const float* rrms, const void* dres, int64_t T, int d, void* dx, void* dx16, void* dweight, int dw_dtype,
                    void* workspace, size_t workspace_bytes, void* stream) {
  // with no rows only the weight gradient (zeros) is written
  KMOE_REQUIRE(weight && dweight && (T == 0 || (dn && x && rrms && dx)), KMOE_ERR_NULL,
               "%s: null buffer", who);
  KMOE_REQUIRE(is_float_dtype(x_dtype) && is_float_dtype(w_dtype) && is_float_dtype(dw_dtype), KMOE_ERR_DTYPE,
               "%s: dtypes %d/%d/%d", who, x_dtype, w_dtype, dw_dtype);
  KMOE_REQUIRE(T >= 0 && d > 0 && d % 8 == 0, KMOE_ERR_SHAPE,
               "%s: d=%d must be a positive multiple of 8", who, d);
  KMOE_REQUIRE(d <= 8192, KMOE_ERR_UNSUPPORTED, "%s: d=%d > 8192", who, d);
  hipStream_t s = kmoe::as_stream(stream);
  if (T == 0) {  // no rows: dg = 0 (a fill kernel, so the call stays capturable)
    hipLaunchKernelGGL(zero_words_kernel, dim3((unsigned)kmoe::ceil_div(d, 256)), dim3(256), 0, s,
                       static_cast<uint16_t*>(dweight), (int64_t)d * (dw_dtype == KMOE_DTYPE_F32 ? 2 : 1));
    return kmoe::check_launch(who);
  }
  const size_t need = kmoe_rmsnorm_bwd_workspace_bytes(T, d);
  KMOE_REQUIRE(workspace && workspace_bytes >= need, KMOE_ERR_WORKSPACE,
               "%s: workspace %zu < %zu bytes", who, workspace_bytes, need);
  const int64_t seg_rows = norm_seg_rows(T);
  const int64_t nseg = kmoe::ceil_div<int64_t>(T, seg_rows);
  float* partial = static_cast<float*>(workspace);
  const bool g_f32 = w_dtype == KMOE_DTYPE_F32;
  const uint16_t* dnp = static_cast<const uint16_t*>(dn);
  const int rc = x_dtype == KMOE_DTYPE_F32
                     ? launch_norm_bwd<true>(dnp, x, weight, g_f32, rrms, dres, T, d, seg_rows, dx,
                                             static_cast<uint16_t*>(dx16), partial, s)
                     : launch_norm_bwd<false>(dnp, x, weight, g_f32, rrms, dres, T, d, seg_rows, dx,
                                             static_cast<uint16_t*>(dx16), partial, s);
  if (rc != KMOE_OK) return rc;
  const int rc2 = kmoe::check_launch(who);
  if (rc2 != KMOE_OK) return rc2;
  return kmoe_reduce_f32(partial, nseg, d, dweight, dw_dtype, stream);
}

extern "C" int kmoe_rmsnorm_bwd(const void* dn, const void* x, int x_dtype, const void* weight, int w_dtype,
                                const float* rrms, const void* dres, int64_t T, int d, void* dx, void* dweight,
                                int dw_dtype, void* workspace, size_t workspace_bytes, void* stream) {
  return norm_bwd("kmoe_rmsnorm_bwd", dn, x, x_dtype, weight, w_dtype, rrms, dres, T, d, dx, nullptr, dweight, dw_dtype,
                  workspace, workspace_bytes, stream);
}

extern "C" int kmoe_add_rmsnorm_bwd(const void* dn, const void* h, int h_dtype, const void* weight, int w_dtype,
                                    const float* rrms, const void* dh, int64_t T, int d, void* dx, void* dx_bf16,
                                    void* dweight, int dw_dtype, void* workspace, size_t workspace_bytes, void* stream) {
  KMOE_REQUIRE(!dx_bf16 || h_dtype == KMOE_DTYPE_F32, KMOE_ERR_DTYPE,
               "kmoe_add_rmsnorm_bwd: dx_bf16 is the rounding of an f32 gradient");
  return norm_bwd("kmoe_add_rmsnorm_bwd", dn, h, h_dtype, weight, w_dtype, rrms, dh, T, d, dx, dx_bf16, dweight, dw_dtype,
                  workspace, workspace_bytes, stream);
}
