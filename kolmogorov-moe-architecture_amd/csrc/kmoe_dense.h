// Dense products on MFMA with operands as torch holds them, no packed copies: the gated
// feed-forward block, its backward, and adapted projections.
//
//   C[m, n] = sum_k A[m, k] B[n, k]     bf16 operands, f32 sums
//
// Each operand is either K-contiguous (its rows are the product's rows: x, h, a Linear weight in
// the forward) or K-strided (its rows run along K: a Linear weight in the backward, the rows of
// both operands of a weight gradient).
//
// A workgroup of 8 waves owns a BM x BN tile; waves form 2 (rows) x 4 (columns).  The tile is
// split into halves along both sides and a wave holds the same place of each of the four
// quadrants, so that the two column halves may come from two matrices: the gate and up rows of
// the same f, whose values then meet in one lane.  K advances 64 per step; a step's 16-byte
// pieces go from memory to LDS without passing registers, each lane picking the piece that belongs
// where the hardware puts it, so the swizzle costs nothing.  NST stages, loads NST - 1 steps ahead,
// one barrier a step.
//   K-contiguous tiles: rows of 128 bytes, 16-byte chunks XOR-ed by (row / 2) % 8; a fragment is
//   one ds_read_b128.
//   K-strided tiles: 64 rows of the tile's columns, 32-byte slots XOR-ed by bits 0, 1 and 3 of the
//   row; a fragment is two ds_read_b64_tr_b16 (in each 16-lane group, lane i receives element
//   i % 4 of the 8-byte chunks addressed by lanes 4 p + i / 4), whose 16 rows spread over all
//   banks twice, the least for 512 bytes.
// The MFMAs take the B fragment first, so a lane holds four consecutive columns of one row.
// Rows and columns past the end read the last row's or zeros and are not stored; K past the end
// reads zeros in both operands (a NaN next to a row's end must not meet a zero).
#pragma once

#include <type_traits>

#include "kmoe_common.h"

namespace kmoe_dense {

constexpr int THREADS = 512;
constexpr int BK = 64;      // K per step
constexpr int KROWB = 128;  // bytes of a K-contiguous tile row

// 16 zero bytes that lanes without data load
__device__ __attribute__((aligned(16))) const uint32_t kZeros[4] = {0, 0, 0, 0};

// Low-rank adapters on top of a product: row m gets v[m] . b[ids[m]]^T, v (M, r) bf16 with the scale
// in it, b (n, N, r); an id outside [0, n) is no adapter.  GATED: [1] are the up half's.
struct Adapt {
  const int32_t* ids;
  const uint16_t* v[2];
  const uint16_t* b[2];
  int n, r;
};

struct Args {
  // the product's parts along K: A and B of each (GATED: one part, b[0] and b[1] the two halves)
  const uint16_t* a[2];
  const uint16_t* b[2];
  int parts;
  int K;              // of each part, a multiple of 8
  int64_t lda, ldb;   // elements
  int64_t M;
  int N;              // columns (GATED: of each half)
  int64_t ldc;
  void* c;            // bf16, or f32 with c_f32
  int c_f32;
  int act;            // GATED
  uint16_t* p;        // GATED: up act'(gate), and q: act(gate), for the backward (nullable); DH: the same, read
  uint16_t* q;
  uint16_t* c2;       // DH: the up half's gradient
  Adapt ad;
};

enum { EPI_PLAIN = 0, EPI_GATED = 1, EPI_DH = 2 };

typedef short tr4_t __attribute__((ext_vector_type(4)));

template <int ROWB>
__device__ __forceinline__ int strided_swz(int r) {
  return ROWB >= 256 ? ((r & 3) | (((r >> 3) & 1) << 2)) : (((r >> 1) & 1) | (((r >> 3) & 1) << 1));
}

// Activation and its derivative at g.
__device__ __forceinline__ void act_f32(int act, float g, float& a, float& da) {
  switch (act) {
    case KMOE_ACT_SILU: {
      const float s = __builtin_amdgcn_rcpf(1.0f + __expf(-g));
      a = g * s;
      da = s * (1.0f + g * (1.0f - s));
      break;
    }
    case KMOE_ACT_GELU: {
      const float c = 0.5f * (1.0f + erff(g * 0.70710678f));
      a = g * c;
      da = c + g * __expf(-0.5f * g * g) * 0.39894228f;
      break;
    }
    case KMOE_ACT_GELU_TANH: {
      const float g2 = g * g, in = 0.79788456f * g * (1.0f + 0.044715f * g2);
      // tanh(z) = 1 - 2 / (1 + e^(2z)): 1 and -1 at its ends
      const float t = 1.0f - 2.0f * __builtin_amdgcn_rcpf(1.0f + __expf(2.0f * in));
      a = 0.5f * g * (1.0f + t);
      da = 0.5f * (1.0f + t) + 0.5f * g * (1.0f - t * t) * 0.79788456f * (1.0f + 0.134145f * g2);
      break;
    }
    default:
      a = g > 0.0f ? g : 0.0f;
      da = g > 0.0f ? 1.0f : 0.0f;
  }
}

__device__ __forceinline__ i32x2_t pack4(float a, float b, float c, float d) {
  const uint32_t lo = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{a, b}, bf16x2_t));
  const uint32_t hi = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{c, d}, bf16x2_t));
  return i32x2_t{(int)lo, (int)hi};
}
__device__ __forceinline__ void unpack4(i32x2_t v, float* o) {
  o[0] = __uint_as_float((uint32_t)v[0] << 16), o[1] = __uint_as_float((uint32_t)v[0] & 0xffff0000u);
  o[2] = __uint_as_float((uint32_t)v[1] << 16), o[3] = __uint_as_float((uint32_t)v[1] & 0xffff0000u);
}

// Workgroup -> tile: ids go round-robin over the 8 XCDs, so each XCD gets a run of consecutive
// tiles, and tiles run down groups of 8 row tiles before the next column tile: a run shares its
// weight columns and its rows in that XCD's L2.
__device__ __forceinline__ void tile_of(int id, int n_mt, int n_nt, int& mt, int& nt) {
  const int n = n_mt * n_nt, per = (n + 7) / 8, full = n - (per - 1) * 8;  // XCDs with `per` tiles
  const int x = id & 7, i = id >> 3;
  const int t = n < 8 ? id : (x < full ? x * per : full * per + (x - full) * (per - 1)) + i;
  constexpr int G = 8;
  const int g = t / (G * n_nt), r = t - g * G * n_nt, gm = n_mt - g * G < G ? n_mt - g * G : G;
  nt = r / gm;
  mt = g * G + (r - nt * gm);
}

// Loads of one operand's stage tile (R rows or columns of the product).
template <int R, bool STRIDED, bool SPLIT>
struct Loader {
  static constexpr int BYTES = R * KROWB;      // of a stage tile, either layout
  static constexpr int NB = BYTES / 1024 / 8;  // 1 KiB pieces of a wave
  static constexpr int ROWB = STRIDED ? R * 2 : KROWB;
  static constexpr int BROWS = 1024 / ROWB;    // tile rows of a piece
  const uint16_t* src[NB];
  int kpos[NB];   // first K of this lane's chunk (row, for strided tiles)
  bool in[NB];    // strided: the chunk's columns exist

  // Rows (columns) [r0, r0 + R) of an operand with `rows` of them; SPLIT: the second half of the
  // tile is the same rows of another matrix.
  __device__ __forceinline__ void init(const uint16_t* base, const uint16_t* base2, int64_t ld, int64_t r0, int64_t rows,
                                       int wave, int lane) {
#pragma unroll
    for (int q = 0; q < NB; ++q) {
      const int blk = wave + 8 * q;
      if constexpr (!STRIDED) {
        const int row = blk * BROWS + (lane >> 3), chunk = (lane & 7) ^ ((row >> 1) & 7);
        const bool second = SPLIT && row >= R / 2;
        int64_t g = r0 + (second ? row - R / 2 : row);
        g = g < rows ? g : rows - 1;
        src[q] = (second ? base2 : base) + g * ld + chunk * 8;
        kpos[q] = chunk * 8;
        in[q] = true;
      } else {
        constexpr int CPR = ROWB / 16;
        const int row = blk * BROWS + lane / CPR, chunk = (lane % CPR) ^ (strided_swz<ROWB>(row) << 1);
        in[q] = r0 + chunk * 8 < rows;
        src[q] = base + (int64_t)row * ld + (in[q] ? r0 + chunk * 8 : 0);
        kpos[q] = row;
      }
    }
  }
  // the next part's matrix, from K = 0
  __device__ __forceinline__ void rebase(int64_t delta) {
#pragma unroll
    for (int q = 0; q < NB; ++q) src[q] += delta;
  }
  // K-step with `left` of K to go into the stage tile at lds; moves on to the next step
  __device__ __forceinline__ void load(int left, int64_t step, KMOE_LDS uint8_t* lds, int wave) {
#pragma unroll
    for (int q = 0; q < NB; ++q) {
      const uint16_t* s = src[q];
      if ((STRIDED && !in[q]) || (left < BK && kpos[q] >= left)) s = reinterpret_cast<const uint16_t*>(kZeros);
      dma16_to_lds(s, lds + (wave + 8 * q) * 1024);
      src[q] += step;
    }
  }
};

// Fragment of 16 rows (columns) at tile row `r`, K-substep i.
template <int R, bool STRIDED>
__device__ __forceinline__ bf16x8_t frag(const uint8_t* l, int r, int i, int lane) {
  if constexpr (!STRIDED) {
    const int row = r + (lane & 15), chunk = 4 * i + (lane >> 4);
    return *reinterpret_cast<const bf16x8_t*>(l + row * KROWB + ((chunk ^ ((row >> 1) & 7)) << 4));
  } else {
    constexpr int ROWB = R * 2;
    const int i16 = lane & 15, row = 32 * i + 8 * (lane >> 4) + (i16 >> 2), col = r + 4 * (i16 & 3);
    const uint8_t* p = l + row * ROWB + (((col >> 3) ^ (strided_swz<ROWB>(row) << 1)) << 4) + (col & 4) * 2;
    const tr4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((KMOE_LDS tr4_t*)p);
    const tr4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((KMOE_LDS tr4_t*)(p + 4 * ROWB));
    return __builtin_bit_cast(bf16x8_t, (short __attribute__((ext_vector_type(8)))){lo[0], lo[1], lo[2], lo[3], hi[0], hi[1],
                                                                                   hi[2], hi[3]});
  }
}

// Distinct adapters of the tile's rows: list[0 .. *count), in no order (a row has one adapter, so the
// order does not reach the results).  sid: the rows' ids, -1 without one.
template <int BM>
__device__ __forceinline__ void list_adapters(const Adapt& ad, int64_t m0, int64_t M, int tid, int* sid, int* list,
                                              int* count) {
  int id = -1;
  if (tid < BM) {
    if (m0 + tid < M) id = ad.ids[m0 + tid];
    if ((unsigned)id >= (unsigned)ad.n) id = -1;
    sid[tid] = id;
  }
  if (tid == 0) *count = 0;
  __syncthreads();
  if (tid < BM && id >= 0 && !(tid > 0 && sid[tid - 1] == id)) {
    bool first = true;
    for (int t = 0; t + 1 < tid && first; ++t) first = sid[t] != id;
    if (first) list[atomicAdd(count, 1)] = id;
  }
  __syncthreads();
}

template <int BM, int BN, bool SA, bool SB, int EPI, int NST, bool ADAPT = false>
__global__ __launch_bounds__(THREADS, 2) void dense_kernel(Args g, int n_mt, int n_nt) {
  constexpr bool GATED = EPI == EPI_GATED;
  static_assert(!GATED || !SB, "gate and up rows are K-contiguous");
  constexpr int QA = BM / 64, QB = BN / 128;  // 16 x 16 blocks of a wave and quadrant
  using LoadA = Loader<BM, SA, false>;
  using LoadB = Loader<BN, SB, GATED>;
  constexpr int STAGE = LoadA::BYTES + LoadB::BYTES;
  constexpr int NL = LoadA::NB + LoadB::NB;  // loads of a wave and step
  __shared__ __attribute__((aligned(1024))) uint8_t lds[NST * STAGE];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave >> 2, wn = wave & 3;
  int mt, nt;
  tile_of(blockIdx.x, n_mt, n_nt, mt, nt);
  const int64_t m0 = (int64_t)mt * BM;
  const int n0 = nt * (GATED ? BN / 2 : BN);

  LoadA la;
  LoadB lb;
  la.init(g.a[0], nullptr, g.lda, m0, g.M, wave, lane);
  lb.init(g.b[0], g.b[1], g.ldb, n0, g.N, wave, lane);
  const int per = (g.K + BK - 1) / BK, nk = per * g.parts;
  const int64_t step_a = SA ? (int64_t)BK * g.lda : BK, step_b = SB ? (int64_t)BK * g.ldb : BK;
  KMOE_LDS uint8_t* const ldsp = (KMOE_LDS uint8_t*)lds;
  int issued = 0, pos = 0;  // steps asked for; the next one's place in its part
  auto issue = [&]() {
    const int st = issued % NST;
    la.load(g.K - pos * BK, step_a, ldsp + st * STAGE, wave);
    lb.load(g.K - pos * BK, step_b, ldsp + st * STAGE + LoadA::BYTES, wave);
    ++issued;
    if (++pos == per && !GATED && issued < nk) {
      pos = 0;
      la.rebase((g.a[1] - g.a[0]) - per * step_a);
      lb.rebase((g.b[1] - g.b[0]) - per * step_b);
    }
  };

  f32x4_t acc[2][2][QA][QB];
#pragma unroll
  for (int x = 0; x < 2; ++x)
#pragma unroll
    for (int y = 0; y < 2; ++y)
#pragma unroll
      for (int i = 0; i < QA; ++i)
#pragma unroll
        for (int j = 0; j < QB; ++j) acc[x][y][i][j] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};

  for (int s = 0; s < NST - 1 && s < nk; ++s) issue();
  __shared__ int sid[ADAPT ? BM : 1], list[ADAPT ? BM : 1], n_list;
  if constexpr (ADAPT) list_adapters<BM>(g.ad, m0, g.M, tid, sid, list, &n_list);
  for (int kt = 0; kt < nk; ++kt) {
    // step kt has landed when at most the loads of the steps behind it are in flight; past the
    // barrier every wave's part of it has, and every wave is done with step kt - 1
    if (issued - kt - 1 >= NST - 2 && NST > 2)
      wait_vmcnt<(NST - 2) * NL>();
    else
      wait_vmcnt<0>();
    wait_lgkmcnt0();
    barrier_nofence();
    if (issued < nk) issue();
    const uint8_t* const pa = lds + (kt % NST) * STAGE;
    const uint8_t* const pb = pa + LoadA::BYTES;
    bf16x8_t fa[2][QA][2], fb[2][QB][2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
#pragma unroll
      for (int i = 0; i < QA; ++i)
#pragma unroll
        for (int s = 0; s < 2; ++s) fa[x][i][s] = frag<BM, SA>(pa, x * (BM / 2) + wm * (BM / 4) + i * 16, s, lane);
#pragma unroll
      for (int j = 0; j < QB; ++j)
#pragma unroll
        for (int s = 0; s < 2; ++s) fb[x][j][s] = frag<BN, SB>(pb, x * (BN / 2) + wn * (BN / 8) + j * 16, s, lane);
    }
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int yy = 0; yy < 2; ++yy) {
        const int y = x ? 1 - yy : yy;
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int i = 0; i < QA; ++i)
#pragma unroll
            for (int j = 0; j < QB; ++j)
              acc[x][y][i][j] =
                  __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[y][j][s], fa[x][i][s], acc[x][y][i][j], 0, 0, 0);
      }
  }

  const int l16 = lane & 15, lq = lane >> 4;
  if constexpr (ADAPT) {
    // Each adapter of the tile: its product with the rows that have it, 32 ranks at a time.  A
    // wave computes it for whole blocks of 16 rows and adds it, by selection, to the rows that have
    // the adapter: a sum over masked operands would carry a NaN or an infinity of one request's
    // adapter into the others' rows.
    for (int a = 0; a < n_list; ++a) {
      const int id = __builtin_amdgcn_readfirstlane(list[a]);
      for (int s = 0; s < g.ad.r; s += 32) {
        const int k = s + 8 * lq;
        const bool in = k < g.ad.r;
        bf16x8_t fb[2][QB];
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
          for (int j = 0; j < QB; ++j) {
            const int n = n0 + (GATED ? 0 : y * (BN / 2)) + wn * (BN / 8) + j * 16 + l16;
            const uint16_t* b = g.ad.b[GATED ? y : 0];
            fb[y][j] = bf16x8_t{};
            if (in && n < g.N && b)
              fb[y][j] = *reinterpret_cast<const bf16x8_t*>(b + ((int64_t)id * g.N + n) * g.ad.r + k);
          }
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int i = 0; i < QA; ++i) {
            const int tr = x * (BM / 2) + wm * (BM / 4) + i * 16 + l16;
            const bool mine = sid[tr] == id;
            if (!__any(mine)) continue;
            bf16x8_t fv[2];
#pragma unroll
            for (int y = 0; y < (GATED ? 2 : 1); ++y) {
              const uint16_t* v = g.ad.v[y];
              fv[y] = bf16x8_t{};
              if (in && mine && v) fv[y] = *reinterpret_cast<const bf16x8_t*>(v + (m0 + tr) * g.ad.r + k);
            }
#pragma unroll
            for (int y = 0; y < 2; ++y)
#pragma unroll
              for (int j = 0; j < QB; ++j) {
                const f32x4_t d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[y][j], fv[GATED ? y : 0],
                                                                         f32x4_t{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0);
#pragma unroll
                for (int t = 0; t < 4; ++t) acc[x][y][i][j][t] += mine ? d[t] : 0.0f;
              }
          }
      }
    }
  }
  // ---- epilogue: acc[x][y][i][j][t] is row m, column n + t
#pragma unroll
  for (int x = 0; x < 2; ++x)
#pragma unroll
    for (int i = 0; i < QA; ++i) {
      const int64_t m = m0 + x * (BM / 2) + wm * (BM / 4) + i * 16 + l16;
      if (m >= g.M) continue;
      if constexpr (GATED) {
#pragma unroll
        for (int j = 0; j < QB; ++j) {
          const int n = n0 + wn * (BN / 8) + j * 16 + 4 * lq;
          if (n >= g.N) continue;
          float h[4], p[4], q[4];
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            float a, da;
            const float up = acc[x][1][i][j][t];
            act_f32(g.act, acc[x][0][i][j][t], a, da);
            h[t] = a * up, p[t] = da * up, q[t] = a;
          }
          const int64_t at = m * g.ldc + n;
          *reinterpret_cast<i32x2_t*>(static_cast<uint16_t*>(g.c) + at) = pack4(h[0], h[1], h[2], h[3]);
          if (g.p) {
            *reinterpret_cast<i32x2_t*>(g.p + at) = pack4(p[0], p[1], p[2], p[3]);
            *reinterpret_cast<i32x2_t*>(g.q + at) = pack4(q[0], q[1], q[2], q[3]);
          }
        }
      } else {
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
          for (int j = 0; j < QB; ++j) {
            const int n = n0 + y * (BN / 2) + wn * (BN / 8) + j * 16 + 4 * lq;
            if (n >= g.N) continue;
            const f32x4_t v = acc[x][y][i][j];
            const int64_t at = m * g.ldc + n;
            if constexpr (EPI == EPI_DH) {
              float p[4], q[4];
              unpack4(*reinterpret_cast<const i32x2_t*>(g.p + at), p);
              unpack4(*reinterpret_cast<const i32x2_t*>(g.q + at), q);
              *reinterpret_cast<i32x2_t*>(static_cast<uint16_t*>(g.c) + at) =
                  pack4(v[0] * p[0], v[1] * p[1], v[2] * p[2], v[3] * p[3]);
              *reinterpret_cast<i32x2_t*>(g.c2 + at) = pack4(v[0] * q[0], v[1] * q[1], v[2] * q[2], v[3] * q[3]);
            } else if (g.c_f32) {
              *reinterpret_cast<f32x4_t*>(static_cast<float*>(g.c) + at) = v;
            } else {
              *reinterpret_cast<i32x2_t*>(static_cast<uint16_t*>(g.c) + at) = pack4(v[0], v[1], v[2], v[3]);
            }
          }
      }
    }
}

}  // namespace kmoe_dense
