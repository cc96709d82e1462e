// AdamW over many tensors in one launch, states in 32 or in 8 bits.
//
//   m' = b1 m + (1 - b1) g,   v' = b2 v + (1 - b2) g^2
//   p' = p - lr wd p - lr / (1 - b1^t) m' / (sqrt(v' / (1 - b2^t)) + eps)
//
// The step counts t live on the device, one per tensor, so a captured step counts its replays;
// the last workgroup of a tensor moves its count on, which costs no launch.
//
// States in 8 bits, in blocks of 256 values with a scale in f32 each:
//   m       e4m3 codes, scale = largest |m| / 448
//   sqrt v  (what the update divides by) unsigned codes of 4 exponent and 4 mantissa bits,
//           (16 + f) 2^(e - 19) for e > 0 and f 2^-18 for e = 0, scale = largest / 1.9375; the
//           sign that a second moment has no use for buys a mantissa bit over e4m3 (half step
//           2^-5 against 2^-4), the root halves the exponents that have to be spanned.
//           What is positive is never rounded to zero: the update divides by it.
// The update takes the moments before they are rounded.  A block with a value that is not finite
// gets the scale NaN: the error shows at its next use.
//
// Bound by memory: a bf16 weight moves 22 bytes with states in 32 bits (2 + 2 + 2 and 4 x 4),
// 10.03 with states in 8.  A lane takes 8 consecutive values, the widest loads of every type.
// m', v' and the codes are computed without contraction, so they are those of the same
// formulas in separate f32 operations, bit for bit; square roots are IEEE for that reason too.
#include "kmoe_common.h"

namespace {

constexpr int ROW = KMOE_ADAMW_FIELDS;      // int64 fields of a tensor in the table
constexpr int THREADS = 256;
constexpr int VALS = 8;                     // values of a lane
constexpr int STEP_VALS = THREADS * VALS;   // values of a workgroup and iteration
constexpr int ITERS = KMOE_ADAMW_CHUNK / STEP_VALS;
constexpr int MAX_GRADS = 256;              // tensors of a launch: their gradients' addresses are arguments
constexpr int QBLOCK = KMOE_ADAMW_BLOCK;    // values that share a scale: 32 lanes
static_assert(QBLOCK == 32 * VALS && KMOE_ADAMW_CHUNK % STEP_VALS == 0, "layout");

struct Grads {
  const void* g[MAX_GRADS];
};

struct Hyper {
  float lr, b1, b2, omb1, omb2, eps, wd;  // omb: 1 - b, rounded from 64 bits
  double b1d, b2d;
  const float* lr_dev;  // when set: the learning rate
};

// Addresses from the table are global ones: without the address space the compiler makes flat
// accesses of them.
#define KMOE_GLOBAL __attribute__((address_space(1)))
template <typename T>
__device__ __forceinline__ KMOE_GLOBAL T* global_ptr(int64_t a) {
  return (KMOE_GLOBAL T*)(uintptr_t)a;
}

// 8 values from or to memory: WIDE with 16-byte accesses, else the first n one by one
template <bool WIDE>
__device__ __forceinline__ void load8(const KMOE_GLOBAL float* p, int n, float* o) {
  if constexpr (WIDE) {
    const f32x4_t a = ((const KMOE_GLOBAL f32x4_t*)p)[0], b = ((const KMOE_GLOBAL f32x4_t*)p)[1];
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = a[i], o[4 + i] = b[i];
  } else {
#pragma unroll
    for (int i = 0; i < VALS; ++i) o[i] = i < n ? p[i] : 0.0f;
  }
}
template <bool WIDE>
__device__ __forceinline__ void load8(const KMOE_GLOBAL uint16_t* p, int n, float* o) {
  if constexpr (WIDE) {
    const i32x4_t a = *(const KMOE_GLOBAL i32x4_t*)p;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      o[2 * i] = __uint_as_float((uint32_t)a[i] << 16);
      o[2 * i + 1] = __uint_as_float((uint32_t)a[i] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < VALS; ++i) o[i] = i < n ? bf16_to_f32(p[i]) : 0.0f;
  }
}
template <bool WIDE>
__device__ __forceinline__ void store8(KMOE_GLOBAL float* p, int n, const float* v) {
  if constexpr (WIDE) {
    ((KMOE_GLOBAL f32x4_t*)p)[0] = f32x4_t{v[0], v[1], v[2], v[3]};
    ((KMOE_GLOBAL f32x4_t*)p)[1] = f32x4_t{v[4], v[5], v[6], v[7]};
  } else {
#pragma unroll
    for (int i = 0; i < VALS; ++i)
      if (i < n) p[i] = v[i];
  }
}
template <bool WIDE>
__device__ __forceinline__ void store8(KMOE_GLOBAL uint16_t* p, int n, const float* v) {
  if constexpr (WIDE) {
    i32x4_t a;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      a[i] = (int)__builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{v[2 * i], v[2 * i + 1]}, bf16x2_t));
    *(KMOE_GLOBAL i32x4_t*)p = a;
  } else {
#pragma unroll
    for (int i = 0; i < VALS; ++i)
      if (i < n) p[i] = f32_to_bf16(v[i]);
  }
}
template <bool WIDE>
__device__ __forceinline__ i32x2_t load8c(const KMOE_GLOBAL uint8_t* p, int n) {
  if constexpr (WIDE) return *(const KMOE_GLOBAL i32x2_t*)p;
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < VALS; ++i)
    if (i < n) w[i >> 2] |= (uint32_t)p[i] << (8 * (i & 3));
  return i32x2_t{(int)w[0], (int)w[1]};
}
template <bool WIDE>
__device__ __forceinline__ void store8c(KMOE_GLOBAL uint8_t* p, int n, i32x2_t v) {
  if constexpr (WIDE) {
    *(KMOE_GLOBAL i32x2_t*)p = v;
  } else {
#pragma unroll
    for (int i = 0; i < VALS; ++i)
      if (i < n) p[i] = (uint8_t)((uint32_t)v[i >> 2] >> (8 * (i & 3)));
  }
}

// Largest of the 32 lanes that share a scale.
__device__ __forceinline__ float max32(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
  return v;
}

// The numbers of the unsigned codes.
__device__ __forceinline__ float root_value(uint32_t c) {
  // the byte is the exponent and the top of the mantissa of 2^-112 times the number (subnormals
  // too), 2^112 = 2^(127 - 15): one product gives either
  return __uint_as_float(c << 19) * 0x1p112f;
}
// The code of q in [0, 1.9375]: to nearest, ties to even.
__device__ __forceinline__ uint32_t root_code(float q) {
  if (q < 0x1p-14f) return (uint32_t)__builtin_rintf(q * 0x1p18f);  // 16 is 2^-14
  const uint32_t u = __float_as_uint(q);
  return ((u + 0x3ffffu + ((u >> 19) & 1u)) >> 19) - (uint32_t)((127 - 15) << 4);
}

// b^t by squares, in 64 bits: 1 - b^t keeps its digits where b^t is near 1.
__device__ __forceinline__ double ipow(double b, uint32_t t) {
  double r = 1.0;
  for (; t; t >>= 1, b *= b)
    if (t & 1u) r *= b;
  return r;
}

// The moments that 8 codes of each stand for.
__device__ __forceinline__ void decode8(i32x2_t cm, i32x2_t cv, float sm, float sv, float* mv, float* root) {
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const f32x2_t lo = __builtin_amdgcn_cvt_pk_f32_fp8(cm[w], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(cm[w], true);
    const float c[4] = {lo[0], lo[1], hi[0], hi[1]};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      mv[4 * w + i] = c[i] * sm;
      root[4 * w + i] = root_value(((uint32_t)cv[w] >> (8 * i)) & 255u) * sv;
    }
  }
}

// One tensor's places and the step's factors.
template <typename PT>
struct Tensor {
  KMOE_GLOBAL PT* p;
  const KMOE_GLOBAL PT* g;
  KMOE_GLOBAL float *master, *mf, *vf, *ms, *vs;
  KMOE_GLOBAL uint8_t *mc, *vc;
  float step_size, inv_c2, keep;
};

// Values [at, at + 8) of a tensor (FAST: all there and aligned; else the first nv).
template <typename PT, int BITS, bool MASTER, bool FAST>
__device__ __forceinline__ void update8(const Tensor<PT>& t, const Hyper& hp, int64_t at, int nv) {
#pragma clang fp contract(off)
  float pv[VALS], gv[VALS], mv[VALS], vv[VALS], rv[VALS];
  const int64_t qb = at / QBLOCK;
  load8<FAST>(t.g + at, nv, gv);
  if constexpr (MASTER)
    load8<FAST>(t.master + at, nv, pv);
  else
    load8<FAST>(t.p + at, nv, pv);
  if constexpr (BITS == 32) {
    load8<FAST>(t.mf + at, nv, mv);
    load8<FAST>(t.vf + at, nv, vv);
  } else {
    const i32x2_t cm = load8c<FAST>(t.mc + at, nv), cv = load8c<FAST>(t.vc + at, nv);
    const float sm = FAST || nv > 0 ? t.ms[qb] : 0.0f, sv = FAST || nv > 0 ? t.vs[qb] : 0.0f;
    decode8(cm, cv, sm, sv, mv, vv);
#pragma unroll
    for (int i = 0; i < VALS; ++i) vv[i] = vv[i] * vv[i];
  }
#pragma unroll
  for (int i = 0; i < VALS; ++i) {
    mv[i] = hp.b1 * mv[i] + hp.omb1 * gv[i];
    vv[i] = hp.b2 * vv[i] + (hp.omb2 * gv[i]) * gv[i];
    rv[i] = sqrtf(vv[i]);
    // (the hardware reciprocal: its last bit is far below a weight's)
    const float upd = t.step_size * mv[i] * __builtin_amdgcn_rcpf(rv[i] * t.inv_c2 + hp.eps);
    pv[i] = pv[i] * t.keep - upd;
  }
  store8<FAST>(t.p + at, nv, pv);
  if constexpr (MASTER) store8<FAST>(t.master + at, nv, pv);
  if constexpr (BITS == 32) {
    store8<FAST>(t.mf + at, nv, mv);
    store8<FAST>(t.vf + at, nv, vv);
  } else {
    float am = 0.0f, av = 0.0f, bad = 0.0f;
#pragma unroll
    for (int i = 0; i < VALS; ++i) {
      // values past the end are zeros of zeros: they do not raise the largest and are not stored
      am = fmaxf(am, fabsf(mv[i]));
      av = fmaxf(av, rv[i]);
      bad = fmaxf(bad, fabsf(mv[i]) < __builtin_inff() && rv[i] < __builtin_inff() ? 0.0f : 1.0f);
    }
    am = max32(am), av = max32(av), bad = max32(bad);
    // (a largest |m| below 2^-91 counts as zero, and the reciprocal stays finite)
    float sm = am * (1.0f / 448.0f), sv = av * (1.0f / 1.9375f);
    const float im = sm >= 0x1p-100f ? 1.0f / sm : 0.0f, iv = sv > 0.0f ? 1.0f / sv : 0.0f;
    if (sm < 0x1p-100f) sm = 0.0f;
    if (bad > 0.0f) sm = sv = __builtin_nanf("");
    i32x2_t cm, cv;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      cm[w] = (int)e4m3x4(mv[4 * w] * im, mv[4 * w + 1] * im, mv[4 * w + 2] * im, mv[4 * w + 3] * im);
      uint32_t u = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float q = fminf(rv[4 * w + i] * iv, 1.9375f);
        uint32_t c = root_code(q);
        if (c == 0 && rv[4 * w + i] > 0.0f) c = 1;
        u |= c << (8 * i);
      }
      cv[w] = (int)u;
    }
    store8c<FAST>(t.mc + at, nv, cm);
    store8c<FAST>(t.vc + at, nv, cv);
    if ((threadIdx.x & 31) == 0 && (FAST || nv > 0)) {
      t.ms[qb] = sm;
      t.vs[qb] = sv;
    }
  }
}

template <typename PT, int BITS, bool MASTER>
__global__ __launch_bounds__(THREADS) void adamw_kernel(const int64_t* __restrict__ table,
                                                        const int32_t* __restrict__ chunk_tensor,
                                                        const int32_t* __restrict__ chunk_base, int t0, int c0,
                                                        int32_t* __restrict__ tickets, Grads grads, Hyper hp) {
  const int chunk = c0 + blockIdx.x;
  const int ti = __builtin_amdgcn_readfirstlane(chunk_tensor[chunk]);
  const int64_t g = (int64_t)(uintptr_t)grads.g[ti - t0];
  if (g == 0) return;  // no gradient: neither the tensor nor its count moves
  const int64_t* const row = table + (int64_t)ti * ROW;
  Tensor<PT> t;
  t.p = global_ptr<PT>(row[0]);
  t.g = global_ptr<const PT>(g);
  t.mf = global_ptr<float>(row[1]), t.vf = global_ptr<float>(row[2]);
  t.mc = global_ptr<uint8_t>(row[1]), t.vc = global_ptr<uint8_t>(row[2]);
  t.ms = global_ptr<float>(row[3]), t.vs = global_ptr<float>(row[4]);
  t.master = global_ptr<float>(row[5]);
  KMOE_GLOBAL int32_t* const step = global_ptr<int32_t>(row[6]);
  const int64_t n = row[7];
  const int first = chunk_base[ti], n_chunks = chunk_base[ti + 1] - first;
  const int64_t start = (int64_t)(chunk - first) * KMOE_ADAMW_CHUNK;

  const uint32_t count = (uint32_t)__builtin_amdgcn_readfirstlane(*step) + 1u;
  const float lr = hp.lr_dev ? *hp.lr_dev : hp.lr;
  t.step_size = (float)((double)lr / (1.0 - ipow(hp.b1d, count)));
  t.inv_c2 = (float)(1.0 / sqrt(1.0 - ipow(hp.b2d, count)));
  t.keep = (float)(1.0 - (double)lr * (double)hp.wd);

  if (((row[0] | g | row[1] | row[2] | row[5]) & 15) == 0 && start + KMOE_ADAMW_CHUNK <= n) {
#pragma unroll 2
    for (int it = 0; it < ITERS; ++it)
      update8<PT, BITS, MASTER, true>(t, hp, start + (int64_t)it * STEP_VALS + threadIdx.x * VALS, VALS);
  } else {
#pragma unroll 1
    for (int it = 0; it < ITERS; ++it) {
      // (a wave is past the end as a whole, or takes part in the reductions as a whole)
      const int64_t at = start + (int64_t)it * STEP_VALS + threadIdx.x * VALS, left = n - at;
      if (n - at + (threadIdx.x & 63) * VALS <= 0) break;
      update8<PT, BITS, MASTER, false>(t, hp, at, left >= VALS ? VALS : (left > 0 ? (int)left : 0));
    }
  }

  // The tensor's last workgroup counts the step: the others have read the count by then, it
  // went into what they computed.  No fence: nothing else passes between workgroups, and at
  // this scope a fence writes the L2 back (experts of one layer, 34000 workgroups: 3386 us with it).
  __syncthreads();
  if (threadIdx.x == 0) {
    if (__hip_atomic_fetch_add(&tickets[ti], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == n_chunks - 1) {
      *step = (int32_t)count;
      tickets[ti] = 0;
    }
  }
}

// The values that 8-bit states stand for: the first moment and the root of the second.
template <typename OT>
__global__ __launch_bounds__(THREADS) void adamw_values_kernel(const uint8_t* __restrict__ mc, const float* __restrict__ ms,
                                                               const uint8_t* __restrict__ vc, const float* __restrict__ vs,
                                                               int64_t n, bool wide, OT* __restrict__ m,
                                                               OT* __restrict__ root) {
  const int64_t at = ((int64_t)blockIdx.x * THREADS + threadIdx.x) * VALS;
  if (at >= n) return;
  const int nv = n - at < VALS ? (int)(n - at) : VALS;
  const float sm = ms[at / QBLOCK], sv = vs[at / QBLOCK];
  const auto *gm = (const KMOE_GLOBAL uint8_t*)(mc + at), *gv = (const KMOE_GLOBAL uint8_t*)(vc + at);
  float a[VALS], b[VALS];
  if (wide && nv == VALS) {
    decode8(load8c<true>(gm, nv), load8c<true>(gv, nv), sm, sv, a, b);
    store8<true>((KMOE_GLOBAL OT*)(m + at), nv, a);
    store8<true>((KMOE_GLOBAL OT*)(root + at), nv, b);
  } else {
    decode8(load8c<false>(gm, nv), load8c<false>(gv, nv), sm, sv, a, b);
    store8<false>((KMOE_GLOBAL OT*)(m + at), nv, a);
    store8<false>((KMOE_GLOBAL OT*)(root + at), nv, b);
  }
}

template <typename PT, int BITS, bool MASTER>
void launch(const int64_t* table, const int32_t* ct, const int32_t* cb, int t0, int c0, int c1, int32_t* tickets,
            const Grads& gr, const Hyper& hp, hipStream_t s) {
  hipLaunchKernelGGL((adamw_kernel<PT, BITS, MASTER>), dim3((unsigned)(c1 - c0)), dim3(THREADS), 0, s, table, ct, cb, t0,
                     c0, tickets, gr, hp);
}

}  // namespace

extern "C" int kmoe_adamw(const int64_t* table, const int32_t* chunk_tensor, const int32_t* chunk_base,
                          const int32_t* chunk_base_host, int n_tensors, const void* const* grads, int dtype, int bits,
                          int has_master, float lr, const float* lr_dev, double beta1, double beta2, float eps, float wd,
                          int32_t* tickets, void* stream) {
  KMOE_REQUIRE(n_tensors >= 0, KMOE_ERR_SHAPE, "kmoe_adamw: n_tensors=%d", n_tensors);
  if (n_tensors == 0) return KMOE_OK;
  KMOE_REQUIRE(table && chunk_tensor && chunk_base && chunk_base_host && grads && tickets, KMOE_ERR_NULL,
               "kmoe_adamw: null buffer");
  KMOE_REQUIRE(dtype == KMOE_DTYPE_BF16 || dtype == KMOE_DTYPE_F32, KMOE_ERR_DTYPE, "kmoe_adamw: dtype %d", dtype);
  KMOE_REQUIRE(bits == 32 || bits == 8, KMOE_ERR_UNSUPPORTED, "kmoe_adamw: states of %d bits (32 or 8)", bits);
  KMOE_REQUIRE(!has_master || dtype == KMOE_DTYPE_BF16, KMOE_ERR_UNSUPPORTED, "kmoe_adamw: f32 weights have no f32 copy");
  KMOE_REQUIRE(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0 && eps >= 0.0f && wd >= 0.0f, KMOE_ERR_SHAPE,
               "kmoe_adamw: betas (%g, %g) in [0, 1), eps %g and weight decay %g not negative", beta1, beta2, eps, wd);
  for (int t = 0; t < n_tensors; ++t)
    KMOE_REQUIRE(chunk_base_host[t] >= 0 && chunk_base_host[t + 1] >= chunk_base_host[t], KMOE_ERR_SHAPE,
                 "kmoe_adamw: chunk_base_host falls at tensor %d", t);
  Hyper hp{lr, (float)beta1, (float)beta2, (float)(1.0 - beta1), (float)(1.0 - beta2), eps, wd, beta1, beta2, lr_dev};
  hipStream_t s = kmoe::as_stream(stream);
  for (int t0 = 0; t0 < n_tensors; t0 += MAX_GRADS) {
    const int t1 = t0 + MAX_GRADS < n_tensors ? t0 + MAX_GRADS : n_tensors;
    Grads gr{};
    bool any = false;
    for (int t = t0; t < t1; ++t) any |= (gr.g[t - t0] = grads[t]) != nullptr;
    const int c0 = chunk_base_host[t0], c1 = chunk_base_host[t1];
    if (!any || c1 == c0) continue;
    // (a launch has fewer than 2^32 threads)
    KMOE_REQUIRE(c1 - c0 < 1 << 24, KMOE_ERR_SHAPE, "kmoe_adamw: %d workgroups of %d values in a launch (below 2^24)", c1 - c0,
                 KMOE_ADAMW_CHUNK);
#define KMOE_ADAMW_CASE(PT, B, M) launch<PT, B, M>(table, chunk_tensor, chunk_base, t0, c0, c1, tickets, gr, hp, s)
    if (dtype == KMOE_DTYPE_F32)
      bits == 32 ? KMOE_ADAMW_CASE(float, 32, false) : KMOE_ADAMW_CASE(float, 8, false);
    else if (has_master)
      bits == 32 ? KMOE_ADAMW_CASE(uint16_t, 32, true) : KMOE_ADAMW_CASE(uint16_t, 8, true);
    else
      bits == 32 ? KMOE_ADAMW_CASE(uint16_t, 32, false) : KMOE_ADAMW_CASE(uint16_t, 8, false);
#undef KMOE_ADAMW_CASE
    const int rc = kmoe::check_launch("kmoe_adamw");
    if (rc != KMOE_OK) return rc;
  }
  return KMOE_OK;
}

extern "C" int kmoe_adamw_values(const void* m_codes, const float* m_scale, const void* v_codes, const float* v_scale,
                                 int64_t n, int dtype, void* m, void* root, void* stream) {
  KMOE_REQUIRE(n >= 0, KMOE_ERR_SHAPE, "kmoe_adamw_values: n=%lld", (long long)n);
  KMOE_REQUIRE(dtype == KMOE_DTYPE_BF16 || dtype == KMOE_DTYPE_F32, KMOE_ERR_DTYPE, "kmoe_adamw_values: dtype %d", dtype);
  if (n == 0) return KMOE_OK;
  KMOE_REQUIRE(m_codes && m_scale && v_codes && v_scale && m && root, KMOE_ERR_NULL, "kmoe_adamw_values: null buffer");
  const int64_t blocks = kmoe::ceil_div<int64_t>(n, STEP_VALS);
  KMOE_REQUIRE(blocks < (int64_t)1 << 24, KMOE_ERR_SHAPE, "kmoe_adamw_values: %lld values", (long long)n);
  const bool wide = ((reinterpret_cast<uintptr_t>(m_codes) | reinterpret_cast<uintptr_t>(v_codes) |
                      reinterpret_cast<uintptr_t>(m) | reinterpret_cast<uintptr_t>(root)) & 15) == 0;
  const auto *mc = static_cast<const uint8_t*>(m_codes), *vc = static_cast<const uint8_t*>(v_codes);
  hipStream_t s = kmoe::as_stream(stream);
  if (dtype == KMOE_DTYPE_F32)
    hipLaunchKernelGGL(adamw_values_kernel<float>, dim3((unsigned)blocks), dim3(THREADS), 0, s, mc, m_scale, vc, v_scale, n,
                       wide, static_cast<float*>(m), static_cast<float*>(root));
  else
    hipLaunchKernelGGL(adamw_values_kernel<uint16_t>, dim3((unsigned)blocks), dim3(THREADS), 0, s, mc, m_scale, vc, v_scale,
                       n, wide, static_cast<uint16_t*>(m), static_cast<uint16_t*>(root));
  return kmoe::check_launch("kmoe_adamw_values");
}
