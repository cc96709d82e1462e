// Dense products on MFMA with operands as torch holds them, no packed copies: the gated
// feed-forward block, its backward, and adapted projections.
//
//   C[m, n] = sum_k A[m, k] B[n, k]     bf16 operands, f32 sums
//
// Each operand is either K-contiguous (its rows are the product's rows: x, h, a Linear weight in
// the forward) or K-strided (its rows run along K: a Linear weight in the backward, the rows of
// both operands of a weight gradient).
//
// A workgroup of four waves, one on a SIMD, owns a BM x BN tile.  The tile is split into halves along
// both sides and a wave of the 2 x 2 holds the same place of each of the four quadrants, so that
// the two column halves may come from two matrices: the gate and up rows of the same f, whose
// values then meet in one lane.  Four waves and not more: LDS moves 128 bytes a cycle, every fragment
// has to feed as many MFMAs as a wave can hold (256 x 256 with eight waves of 128 x 64: reads and
// loads took longer than the MFMAs, 16384 rows, d 2048, F 5632, down 352 us; the MFMAs alone 189).
// Measured on normal numbers, 60 ms back to back: gate and up 563 us (1.34 PFLOP/s; a library product of
// the shape 527), down 259 (243), dx 578 (567), weight gradients 311 each (349); in the first
// milliseconds after a pause all take some 20% longer.  Bound by the chip's power on such data.
// K advances 32 or 64 (32 KS) per step.  A step's 16-byte pieces go from memory to LDS without passing registers,
// each lane picking the piece that belongs where the hardware puts it, so the swizzle costs nothing:
//   K-contiguous tiles: rows of 64 KS bytes, 16-byte chunks XOR-ed by (row / 2) modulo their number;
//   a fragment is one ds_read_b128.
//   K-strided tiles: 32 KS rows of the tile's columns (192 lie as 256), 32-byte slots XOR-ed by bits 0, 1 and 3 of the
//   row; a fragment is two ds_read_b64_tr_b16 (in each 16-lane group, lane i receives element
//   i % 4 of the 8-byte chunks addressed by lanes 4 p + i / 4), whose 16 rows spread over all
//   banks twice, the least for 512 bytes.
// The MFMAs of 32 of K (16x16x32, the B fragment first: a lane holds four consecutive columns of a
// row) are issued in program order, with the reads of the next 32's fragments, into another set of
// registers, between them, and in a step's last 32 the loads of the step STAGES on.  These go
// into the step's own stage: every wave has all of its fragments, as it passed the barrier before
// its last 32, the step's only one.  A load has STAGES - 1 steps to land.  Past the last step zeros
// are loaded, so that the counts of loads in flight stay the same.
// Rows, columns and K past the end read as zeros (K's in both operands: a NaN next to a row's end must
// not meet a zero); what they give is not stored.
#pragma once

#include <type_traits>

#include "kmoe_common.h"

namespace kmoe_dense {

constexpr int THREADS = 256;
constexpr int LOST_ROWS = KMOE_DENSE_LOST_ROWS;  // half a tile of 64
static_assert(LOST_ROWS == 32, "half a tile of 64 rows");

// Low-rank adapters on top of a product: row m gets v[m] . b[ids[m]]^T, v (2, M, r) bf16 with the scale
// in it and then what it lost by its rounding, b (n, N, r); an id outside [0, n) is no adapter.  GATED:
// [1] are the up half's.
struct Adapt {
  const int32_t* ids;
  const uint16_t* v[2];
  const uint16_t* b[2];
  int n, r;
};

struct Args {
  // A and B, and of a product in two parts along K the second ones (GATED: b[0] and b[1] are the halves)
  const uint16_t* a[2];
  const uint16_t* b[2];
  int K;              // of each part, a multiple of 8
  int k_run;          // of a run of K (a multiple of 64), one for each y of the grid; 0: K
  int64_t lda, ldb;   // elements
  int64_t M;
  int N;              // columns (GATED: of each half)
  int64_t ldc;
  void* c;            // bf16, or f32 with c_f32
  int c_f32;          // (with runs of K: 1, their sums one after the other, M ldc apart)
  int act;            // GATED
  uint8_t* saved;     // GATED: up act'(gate) and act(gate) for the backward (nullable); DH: the same, read
  uint16_t* c2;       // DH: the up half's gradient
  int64_t lost;       // GATED, DH: elements from a value of c (c2) to what it lost by its rounding; 0: not kept
  int64_t fold;       // of M <= 32 rows (tiles of 64 rows): elements from A to what it lost; 0: nothing
  Adapt ad;
};

// EPI_TWO: as EPI_PLAIN, of a product in two parts along K
enum { EPI_PLAIN = 0, EPI_GATED = 1, EPI_DH = 2, EPI_TWO = 3 };

template <int I0, int N, class Fn>
__device__ __forceinline__ void static_for(Fn&& f) {
  if constexpr (I0 < N) {
    f(std::integral_constant<int, I0>{});
    static_for<I0 + 1, N>(f);
  }
}

// 16 bytes at a uniform address plus a 32-bit offset, zeros without an access where the offset has
// bit 31: no branch around the load, so that later ones need not wait for it.
constexpr uint32_t NOWHERE = 0x80000000u;
__device__ __forceinline__ bf16x8_t load16(const void* base, uint32_t off) {
  return __builtin_bit_cast(bf16x8_t, __builtin_amdgcn_raw_buffer_load_b128(
                                          __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, 0x7fffffff, 0x00020000),
                                          off, 0, 0));
}

typedef short tr4_t __attribute__((ext_vector_type(4)));

// What the 32-byte slots of a K-strided tile's row r are XOR-ed by.
template <int ROWB>
__device__ __forceinline__ int strided_swz(int r) {
  return ROWB >= 256 ? ((r & 3) | (((r >> 3) & 1) << 2)) : (((r >> 1) & 1) | (((r >> 3) & 1) << 1));
}

// Activation and its derivative at g.
template <int ACT>
__device__ __forceinline__ void act_at(float g, float& a, float& da) {
  if constexpr (ACT == KMOE_ACT_SILU) {
    const float s = __builtin_amdgcn_rcpf(1.0f + __expf(-g));
    a = g * s;
    da = s * (1.0f + g * (1.0f - s));
  } else if constexpr (ACT == KMOE_ACT_GELU) {
    const float c = 0.5f * (1.0f + erff(g * 0.70710678f));
    a = g * c;
    da = c + g * __expf(-0.5f * g * g) * 0.39894228f;
  } else if constexpr (ACT == KMOE_ACT_GELU_TANH) {
    const float g2 = g * g, in = 0.79788456f * g * (1.0f + 0.044715f * g2);
    // tanh(z) = 1 - 2 / (1 + e^(2z)): 1 and -1 at its ends
    const float t = 1.0f - 2.0f * __builtin_amdgcn_rcpf(1.0f + __expf(2.0f * in));
    a = 0.5f * g * (1.0f + t);
    // (where tanh is 1 or -1 its slope is 0, also against a square past f32's range)
    const float slope = 1.0f - t * t;
    da = 0.5f * (1.0f + t) + (slope == 0.0f ? 0.0f : 0.5f * g * slope * 0.79788456f * (1.0f + 0.134145f * g2));
  } else {
    a = g <= 0.0f ? 0.0f : g;  // (a NaN stays one)
    da = g <= 0.0f ? 0.0f : 1.0f;
  }
}
// f(tag of the activation): the choice is made once, not at every value.
template <class Fn>
__device__ __forceinline__ void with_act(int act, Fn&& f) {
  switch (act) {
    case KMOE_ACT_SILU: f(std::integral_constant<int, KMOE_ACT_SILU>{}); break;
    case KMOE_ACT_GELU: f(std::integral_constant<int, KMOE_ACT_GELU>{}); break;
    case KMOE_ACT_GELU_TANH: f(std::integral_constant<int, KMOE_ACT_GELU_TANH>{}); break;
    default: f(std::integral_constant<int, KMOE_ACT_RELU>{});
  }
}

__device__ __forceinline__ i32x2_t pack4(float a, float b, float c, float d) {
  const uint32_t lo = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{a, b}, bf16x2_t));
  const uint32_t hi = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{c, d}, bf16x2_t));
  return i32x2_t{(int)lo, (int)hi};
}
// What four values lost by their rounding to w.  Of up to 32 rows the products take that too, at the
// cost of rows that a tile has anyway: there a rounding is seen in few results, and does not average
// out.
__device__ __forceinline__ void store_lost(uint16_t* to, const float* v, i32x2_t w) {
  float r[4];
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const uint32_t u = (uint32_t)w[t / 2];
    r[t] = v[t] - __uint_as_float(t % 2 ? u & 0xffff0000u : u << 16);
    if (!(r[t] - r[t] == 0.0f)) r[t] = 0.0f;  // (of an infinity nothing)
  }
  *reinterpret_cast<i32x2_t*>(to) = pack4(r[0], r[1], r[2], r[3]);
}
// A product's result with what its operand lost by the rounding.  An infinity of the other operand has made
// its infinity of the operand itself; what that lost would make a second one of any sign, or a NaN.
__device__ __forceinline__ float with_lost(float v, float lost) { return v - v == 0.0f ? v + lost : v; }
// What the backward multiplies by, up act'(gate) and act(gate), is held in 24 bits, the top of its f32
// rounded to the nearest, ties to even (cut, it would lose up to twice as much, always towards zero;
// 2042 rows, forward and backward 427.7 us, cut 426.6): in bf16 its rounding would add to those of the
// products' operands and results, a third of one size (gradients of the weights and of x: 1.73
// roundings off, so 1.41).  It lies as the MFMAs leave it, by 16 x 16 blocks, a lane's four values
// in 12 bytes: in one access of 768 bytes a wave.
constexpr int SAVED_BLOCK = 2 * 768;  // bytes of a block: both values
struct Three {  // (12 bytes: a vector of three would be stored as four)
  uint32_t a, b, c;
};
__device__ __forceinline__ uint8_t* saved_block(uint8_t* p, int N, int64_t m, int n) {
  return p + ((m >> 4) * ((N + 15) >> 4) + (n >> 4)) * SAVED_BLOCK;
}
__device__ __forceinline__ void store24(uint8_t* block, int lane, const float* v) {
  uint32_t u[4];
#pragma unroll
  // (a NaN is a bf16 number's or an operation's own: its low bits are zeros and do not carry)
  for (int t = 0; t < 4; ++t) {
    u[t] = __float_as_uint(v[t]);
    u[t] += 0x7fu + ((u[t] >> 8) & 1u);
  }
  *reinterpret_cast<Three*>(block + lane * 12) = {(u[0] >> 8) | (u[1] << 16 & 0xff000000u),
                                                  (u[1] >> 16) | (u[2] << 8 & 0xffff0000u),
                                                  (u[2] >> 24) | (u[3] & 0xffffff00u)};
}
__device__ __forceinline__ void load24(const uint8_t* block, int lane, float* v) {
  const Three w = *reinterpret_cast<const Three*>(block + lane * 12);
  v[0] = __uint_as_float(w.a << 8);
  v[1] = __uint_as_float((w.a >> 24 << 8) | (w.b << 16));
  v[2] = __uint_as_float((w.b >> 16 << 8) | (w.c << 24));
  v[3] = __uint_as_float(w.c & 0xffffff00u);
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

// Distinct adapters of the tile's rows: list[0 .. *count), in no order (a row has one adapter, so the
// order does not reach the results).  sid: the rows' ids, of which those that are no adapter's become
// -1.  A wave takes 64 rows, one adapter after the other, and leaves out those of the waves before it.
template <int BM>
__device__ __forceinline__ void list_adapters(int n_adapters, int rows, int tid, int* sid, int* list, int* count) {
  int id = -1;
  if (tid < BM) {
    if (tid < rows) id = sid[tid];
    if ((unsigned)id >= (unsigned)n_adapters) id = -1;
    sid[tid] = id;
  }
  if (tid == 0) *count = 0;
  wait_lgkmcnt0();
  barrier_nofence();
  if (tid < BM) {
    const int wave = tid >> 6, lane = tid & 63;
    int before[BM / 64];
#pragma unroll
    for (int w = 0; w < BM / 64; ++w) before[w] = w < wave ? sid[w * 64 + lane] : -1;
    int mine = -1, n = 0;  // this wave's n-th adapter is held by lane n
    for (uint64_t todo = __ballot(id >= 0); todo;) {
      const int cur = __builtin_amdgcn_readlane(id, __builtin_ctzll(todo));
      todo &= ~__ballot(id == cur);
      bool known = false;
#pragma unroll
      for (int w = 0; w + 1 < BM / 64; ++w) known |= before[w] == cur;
      if (__ballot(known)) continue;
      if (lane == n) mine = cur;
      ++n;
    }
    int at = 0;
    if (lane == 0 && n) at = atomicAdd(count, n);
    at = __builtin_amdgcn_readfirstlane(at);
    if (lane < n) list[at + lane] = mine;
  }
  wait_lgkmcnt0();
  barrier_nofence();
}

// The adapters' outer products of a tile.  A turn is an MFMA's 32 of K: 32 ranks of an adapter of the tile's
// list, or two adapters of 16, or four of 8, each with the rows' inner products where they have it
// and zeros where not, so the sums go on in their registers.  A zero times an infinity or a NaN of
// another request's adapter would be a NaN: a turn with such factors is computed one adapter at a
// time and kept, by selection, for the rows that have it.  Bound by the latency of the factors' reads:
// those of the next C turns run during these.  What the inner products lost by their rounding takes
// part too where it costs little (tiles of 64 rows) and where such an error, which reaches a whole
// row, adds to those of the hidden values' rounding (GATED; the block's result was 1.7 times as far
// off as with one rounding, now 1.4).
// (48 rows, F 5632, gate and up: 10.7 us, with 16 adapters of rank 16 in turn 18.6; read and selected turn
// by turn they took 25 us more).
template <int BM, int BN, bool GATED>
struct Outer {
  static constexpr int QA = BM / 64, QB = BN / 64, H = GATED ? 2 : 1, C = QB == 1 ? 8 : 1;
  static constexpr int HELD = QA == 1 ? 2 : 1, PASSES = GATED && QA > 1 ? 2 : 1;  // both at once where registers are
  const Adapt& ad;
  const int *sid, *list;
  int n_list;
  int64_t m0;
  int n0, N, wm, wn, lane;
  int per;       // adapters of a turn
  int slot, k0;  // this lane's adapter of them, and its first rank
  int turns;     // of 32 ranks
  int own[2 * QA];
  bf16x8_t fv[H][HELD][2 * QA];
  int64_t behind;  // from an inner product to what it lost
  bf16x8_t next[C][2 * QB];
  int next_id[C];

  __device__ __forceinline__ Outer(const Adapt& ad, const int* sid, const int* list, int n_list, int64_t m0, int64_t M, int n0,
                                   int N, int wm, int wn, int lane)
      : ad(ad), sid(sid), list(list), n_list(n_list), m0(m0), n0(n0), N(N), wm(wm), wn(wn), lane(lane), behind(M * ad.r) {
    const int lq = lane >> 4;
    per = ad.r <= 8 ? 4 : ad.r <= 16 ? 2 : 1;
    slot = per == 4 ? lq : per == 2 ? lq >> 1 : 0;
    k0 = per == 4 ? 0 : per == 2 ? (lq & 1) * 8 : lq * 8;
    turns = (n_list + per - 1) / per;
#pragma unroll
    for (int b = 0; b < 2 * QA; ++b) own[b] = sid[row(b)];
  }
  __device__ __forceinline__ int row(int blk) const {  // of the tile
    return (blk / QA) * (BM / 2) + wm * (BM / 4) + (blk % QA) * 16 + (lane & 15);
  }
  // the factors of turns t .. t + C - 1 from rank s on.  Every address is some adapter's: a lane without
  // one, or past the ranks, meets zeros of the rows, and columns past the end are not stored.
  __device__ __forceinline__ void load(int s, int t) {
    const int k = s + k0 < ad.r ? s + k0 : 0;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      if (t + c >= turns) break;
      const int a = (t + c) * per + slot;
      const int id = list[a < n_list ? a : 0];
      next_id[c] = a < n_list ? id : -2;
#pragma unroll
      for (int yj = 0; yj < 2 * QB; ++yj) {
        const int n = n0 + (GATED ? 0 : yj / QB * (BN / 2)) + wn * (BN / 4) + yj % QB * 16 + (lane & 15);
        const uint16_t* const b = GATED && yj >= QB ? ad.b[1] : ad.b[0];
        next[c][yj] = bf16x8_t{};
        if (b) next[c][yj] = *reinterpret_cast<const bf16x8_t*>(b + ((int64_t)id * N + (n < N ? n : N - 1)) * ad.r + k);
      }
    }
  }
  __device__ __forceinline__ void load_rows(int pass, int s) {
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
      for (int p = 0; p < HELD; ++p)
#pragma unroll
        for (int b = 0; b < 2 * QA; ++b) {
          fv[h][p][b] = bf16x8_t{};
          if (s + k0 < ad.r && own[b] >= 0 && ad.b[h])
            fv[h][p][b] = *reinterpret_cast<const bf16x8_t*>(ad.v[h] + (m0 + row(b)) * ad.r + s + k0 + (pass + p) * behind);
        }
  }
  __device__ __forceinline__ void add(f32x4_t (&acc)[2][2][QA][QB]) {
    load(0, 0);
#pragma unroll 1
    for (int pass = 0, s = 0; pass < PASSES; s + 32 < ad.r ? s += 32 : (s = 0, ++pass)) {
      load_rows(pass, s);
#pragma unroll 1
      for (int t = 0; t < turns; t += C) {
        bf16x8_t fb[C][2 * QB];
        int id[C];
#pragma unroll
        for (int c = 0; c < C; ++c) {
          id[c] = next_id[c];
#pragma unroll
          for (int yj = 0; yj < 2 * QB; ++yj) fb[c][yj] = next[c][yj];
        }
        if (t + C < turns)
          load(s, t + C);
        else if (s + 32 < ad.r || pass + 1 < PASSES)
          load(s + 32 < ad.r ? s + 32 : 0, 0);
        uint32_t splits = 0;
        static_for<0, C>([&](auto ct) {
          constexpr int c = decltype(ct)::value;
          if (C == 1 || t + c < turns) {
            uint32_t odd = 0;  // a half with all exponent bits, where adding one to them reaches the sign
#pragma unroll
            for (int yj = 0; yj < 2 * QB; ++yj) {
              const i32x4_t w = __builtin_bit_cast(i32x4_t, fb[c][yj]);
#pragma unroll
              for (int q = 0; q < 4; ++q) odd |= ((uint32_t)w[q] & 0x7f807f80u) + 0x00800080u;
            }
            const bool split = __ballot((odd & 0x80008000u) != 0) != 0;
            static_for<0, 2 * QA>([&](auto bt) {
              constexpr int blk = decltype(bt)::value;
              const bool mine = own[blk] == id[c] && !split;
              const bf16x8_t zero = {};
#pragma unroll
              for (int p = 0; p < HELD; ++p) {
                bf16x8_t v[H];
#pragma unroll
                for (int h = 0; h < H; ++h) v[h] = mine ? fv[h][p][blk] : zero;
#pragma unroll
                for (int yj = 0; yj < 2 * QB; ++yj) {
                  f32x4_t& a = acc[blk / QA][yj / QB][blk % QA][yj % QB];
                  a = __builtin_amdgcn_mfma_f32_16x16x32_bf16(split ? zero : fb[c][yj], v[GATED ? yj / QB : 0], a, 0, 0, 0);
                }
              }
              __builtin_amdgcn_sched_barrier(0);
            });
            hold(acc);
            splits |= split ? 1u << c : 0u;
          }
        });
        // (a row has terms in one turn only, so those taken apart may come last, in one copy of the code)
        for (; splits; splits &= splits - 1) {
          const int at = __builtin_ctz(splits);
          bf16x8_t f[2 * QB];
          int who = 0;
          static_for<0, C>([&](auto ct) {
            constexpr int c = decltype(ct)::value;
            if (at == c) {
#pragma unroll
              for (int yj = 0; yj < 2 * QB; ++yj) f[yj] = fb[c][yj];
              who = id[c];
            }
          });
          apart(acc, f, who, s, pass);
          hold(acc);
        }
      }
    }
  }
  // (after each branch the sums are back in their accumulation registers)
  __device__ __forceinline__ static void hold(f32x4_t (&acc)[2][2][QA][QB]) {
#pragma unroll
    for (int i = 0; i < 4 * QA * QB; ++i) asm volatile("" : "+a"(acc[i / (2 * QA * QB)][i / (QA * QB) % 2][i / QB % QA][i % QB]));
    __builtin_amdgcn_sched_barrier(0);
  }
  // a turn's products, one adapter at a time.  A lane past the ranks holds some rank's factor again, which
  // must not meet its zeros; and what the inner products lost meets the finite factors only: an infinity
  // has what it makes of the inner product itself.
  __device__ __forceinline__ void apart(f32x4_t (&acc)[2][2][QA][QB], bf16x8_t (&fb)[2 * QB], int id, int s, int pass) {
    const bf16x8_t zero = {};
#pragma unroll
    for (int yj = 0; yj < 2 * QB; ++yj) fb[yj] = s + k0 < ad.r ? fb[yj] : zero;
#pragma unroll 1
    for (int i = 0; i < HELD * per; ++i) {  // (one body for both parts: the instruction cache holds more of the turns)
      const int p = HELD > 1 && i >= per ? i - per : i;
      const bool lost = HELD > 1 ? i >= per : pass > 0;
      if (p == 0 && lost) {
#pragma unroll
        for (int yj = 0; yj < 2 * QB; ++yj) fb[yj] = finite(fb[yj]);
      }
      const int cur = __builtin_amdgcn_readlane(id, per == 4 ? p * 16 : p * 32);
      static_for<0, 2 * QA>([&](auto bt) {
        constexpr int blk = decltype(bt)::value;
        static_for<0, 2 * QB>([&](auto yt) {
          constexpr int yj = decltype(yt)::value, h = GATED ? yj / QB : 0;
          // (from the sums on, as the others: a row's result does not depend on whom it is computed with)
          f32x4_t& a = acc[blk / QA][yj / QB][blk % QA][yj % QB];
          const bf16x8_t v = HELD > 1 && lost ? fv[h][HELD - 1][blk] : fv[h][0][blk];
          const f32x4_t d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              slot == p ? fb[yj] : zero, slot == p && own[blk] == cur ? v : zero, a, 0, 0, 0);
#pragma unroll
          for (int c = 0; c < 4; ++c) a[c] = own[blk] == cur ? d[c] : a[c];
          asm volatile("" : "+a"(a));
        });
      });
    }
  }
  // f with zeros for infinities and NaN
  __device__ __forceinline__ static bf16x8_t finite(bf16x8_t f) {
    i32x4_t w = __builtin_bit_cast(i32x4_t, f);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const uint32_t u = (uint32_t)w[q];
      const uint32_t lo = (u & 0x7f80u) == 0x7f80u ? 0u : u & 0xffffu;
      w[q] = (int)((u & 0x7f800000u) == 0x7f800000u ? lo : lo | (u & 0xffff0000u));
    }
    return __builtin_bit_cast(bf16x8_t, w);
  }
};

// Epilogue of a tile: acc[x][y][i][j][t] is row m0 + x BM / 2 + wm BM / 4 + 16 i + l % 16, column
// n0 + y BN / 2 + wn BN / 4 + 16 j + 4 (l / 16) + t.
template <int BM, int BN, int EPI>
__device__ __forceinline__ void finish(const Args& g, const f32x4_t (&acc)[2][2][BM / 64][BN / 64], int64_t m0, int n0, int wm,
                                       int wn, int lane) {
  constexpr bool GATED = EPI == EPI_GATED;
  constexpr int QA = BM / 64, QB = BN / 64, WC = BN / 4;
  const int l16 = lane & 15, lq = lane >> 4;
  auto rows = [&](auto&& f) {  // f(x, i, m) for this lane's rows
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int i = 0; i < QA; ++i) {
        const int64_t m = m0 + x * (BM / 2) + wm * (BM / 4) + i * 16;
        if (m < g.M) f(x, i, m + l16);
      }
  };
  if constexpr (GATED) {
    with_act(g.act, [&](auto tag) {
      rows([&](int x, int i, int64_t m) {
#pragma unroll
        for (int j = 0; j < QB; ++j) {
          const int n16 = n0 + wn * WC + j * 16, n = n16 + 4 * lq;
          if (n16 >= g.N) continue;
          float h[4], p[4], q[4];
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            float a, da;
            const float up = acc[x][1][i][j][t];
            act_at<decltype(tag)::value>(acc[x][0][i][j][t], a, da);
            h[t] = a * up, p[t] = da * up, q[t] = a;
          }
          if (m < g.M && n < g.N) {
            const i32x2_t w = pack4(h[0], h[1], h[2], h[3]);
            *reinterpret_cast<i32x2_t*>(static_cast<uint16_t*>(g.c) + m * g.ldc + n) = w;
            if (g.lost) store_lost(static_cast<uint16_t*>(g.c) + g.lost + m * g.ldc + n, h, w);
          }
          if (g.saved) {  // (whole blocks: the buffer has them)
            uint8_t* const block = saved_block(g.saved, g.N, m, n16);
            store24(block, lane, p);
            store24(block + SAVED_BLOCK / 2, lane, q);
          }
        }
      });
    });
  } else {
    rows([&](int x, int i, int64_t m) {
#pragma unroll
      for (int y = 0; y < 2; ++y)
#pragma unroll
        for (int j = 0; j < QB; ++j) {
          const int n16 = n0 + y * (BN / 2) + wn * WC + j * 16, n = n16 + 4 * lq;
          if (n16 >= g.N) continue;
          const f32x4_t v = acc[x][y][i][j];
          const int64_t at = m * g.ldc + n;
          if constexpr (EPI == EPI_DH) {
            float p[4], q[4];
            const uint8_t* const block = saved_block(g.saved, g.N, m, n16);
            load24(block, lane, p);
            load24(block + SAVED_BLOCK / 2, lane, q);
            if (m < g.M && n < g.N) {
#pragma unroll
              for (int t = 0; t < 4; ++t) p[t] *= v[t], q[t] *= v[t];
              const i32x2_t dg = pack4(p[0], p[1], p[2], p[3]), du = pack4(q[0], q[1], q[2], q[3]);
              uint16_t* const c = static_cast<uint16_t*>(g.c);
              *reinterpret_cast<i32x2_t*>(c + at) = dg;
              *reinterpret_cast<i32x2_t*>(g.c2 + at) = du;
              if (g.lost) store_lost(c + g.lost + at, p, dg), store_lost(g.c2 + g.lost + at, q, du);
            }
          } else if (m < g.M && n < g.N) {
            if (g.c_f32)
              *reinterpret_cast<f32x4_t*>(static_cast<float*>(g.c) + at) = v;
            else
              *reinterpret_cast<i32x2_t*>(static_cast<uint16_t*>(g.c) + at) = pack4(v[0], v[1], v[2], v[3]);
          }
        }
    });
  }
}

// ---------------------------------------------------------------- the tile kernel
template <int R, bool STRIDED, int KS>
struct Loads {  // of one operand's stage tile (R rows or columns, 32 KS of K): this lane's pieces
  static constexpr int P = STRIDED && R == 192 ? 256 : R;  // (rows of 384 bytes take 512: the swizzle is for powers of two)
  static constexpr int BYTES = P * 64 * KS;  // of the stage tile, either layout
  static constexpr int N = BYTES / 4096;     // 1 KiB pieces of a wave
  static constexpr int CPR = STRIDED ? P / 8 : 4 * KS;  // 16-byte chunks of a row
  uint32_t off[N];  // bytes from the first row (column) of the tile, or for split of its half
  int kpos;         // first K of the first piece's chunk

  // rows: how many of the tile's R exist (what is past them reads as zeros, for nothing: a tile of few
  // rows costs the other operand's bytes); split: its halves are the same R / 2 rows of two matrices;
  // fold: the second half is the same rows, that many elements behind
  __device__ __forceinline__ void init(int64_t ld, int64_t rows, bool split, int64_t fold, int wave, int lane) {
#pragma unroll
    for (int q = 0; q < N; ++q) {
      const int row = (wave + 4 * q) * (64 / CPR) + lane / CPR;
      if constexpr (!STRIDED) {
        // (rows of a lane's pieces are multiples of 32 apart: the same chunk of K)
        const int chunk = (lane % CPR) ^ ((row >> 1) & (CPR - 1));
        const int r = split || fold ? row % (R / 2) : row;
        off[q] = r < rows ? (uint32_t)((r * ld + (row >= R / 2 ? fold : 0)) * 2) + chunk * 16 : NOWHERE;
        if (q == 0) kpos = chunk * 8;
      } else {
        const int chunk = (lane % CPR) ^ (strided_swz<2 * P>(row) << 1);
        off[q] = chunk * 8 < (rows < R ? rows : R) ? (uint32_t)(row * ld * 2) + chunk * 16 : NOWHERE;
        if (q == 0) kpos = row;
      }
    }
  }
  // with `left` of K to go, what is past its end reads as zeros
  __device__ __forceinline__ void cut(int left) {
#pragma unroll
    for (int q = 0; q < N; ++q)
      if (kpos + (STRIDED ? 4 * q * (64 / CPR) : 0) >= left) off[q] |= NOWHERE;
  }
};

// Direct global -> LDS load of 16 bytes a lane (see dma16_to_lds) at a uniform address plus a 32-bit
// offset, in two parts with an MFMA between them: M0, the LDS address, needs a cycle before its
// use, and the wave's SIMD issues nothing else meanwhile.  Nothing else in the loop writes M0.
// A buffer load, whose window of 2 GiB turns larger offsets into zeros without an access.
__device__ __forceinline__ void dma16_where(KMOE_LDS void* lds) {
  const uint32_t la = (uint32_t)(uintptr_t)lds;
  asm volatile("s_mov_b32 m0, %0" ::"s"(__builtin_amdgcn_readfirstlane(la)) : "m0");
}
__device__ __forceinline__ void dma16_at(const void* base, uint32_t off) {
  const uint64_t b = reinterpret_cast<uint64_t>(base);
  const i32x4_t window = {(int)(uint32_t)b, (int)(uint32_t)(b >> 32), 0x7fffffff, 0x00020000};
  asm volatile("buffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(off), "s"(window));
}
__device__ __forceinline__ void dma4_at(const void* base, uint32_t off) {
  const uint64_t b = reinterpret_cast<uint64_t>(base);
  const i32x4_t window = {(int)(uint32_t)b, (int)(uint32_t)(b >> 32), 0x7fffffff, 0x00020000};
  asm volatile("buffer_load_dword %0, %1, 0 offen lds" ::"v"(off), "s"(window));
}

// Where a lane reads a wave's fragments of an R-row stage tile: the wave's 16-row blocks are
// r = half R / 2 + w R / 4 + 16 i, Q = R / 64 of them in a half.
template <int R, bool STRIDED, int KS>
struct Frags {
  static constexpr int Q = R / 64;
  static constexpr int P = Loads<R, STRIDED, KS>::P;
  // K-contiguous: the swizzle repeats every 16 rows, a block only adds to the address.  Strided: a
  // block's number is XOR-ed into bits from 5 on, which for the halves of 256 columns is an addition.
  static constexpr int PLACES = !STRIDED ? 1 : R == 256 ? Q : 2 * Q;
  uint32_t place[PLACES];

  __device__ __forceinline__ void init(int w, int lane) {
    if constexpr (!STRIDED) {
      const int row = w * (R / 4) + (lane & 15);
      place[0] = row * 64 * KS + (((lane >> 4) ^ ((row >> 1) & (4 * KS - 1))) << 4);
    } else {
      const int i16 = lane & 15, row = 8 * (lane >> 4) + (i16 >> 2);
#pragma unroll
      for (int i = 0; i < PLACES; ++i) {
        const int block = (i / Q) * (R / 32) + w * Q + i % Q;
        place[i] = row * 2 * P + ((block ^ strided_swz<2 * P>(row)) << 5) + (i16 & 3) * 8;
      }
    }
  }
  // block b (b / Q the half) of K from 32 ks on, of a stage tile.  (One addition for a tile and place: the
  // rest goes into the instructions' offsets.)
  __device__ __forceinline__ bf16x8_t read(const KMOE_LDS uint8_t* tile, int b, int ks) const {
    if constexpr (!STRIDED) {
      // (the second 32 of K are chunks 4 .. 7: bit 6 of the place, whatever the swizzle makes of it)
      const KMOE_LDS uint8_t* at = tile + (ks ? place[0] ^ 64u : place[0]);
      return *(const KMOE_LDS bf16x8_t*)(at + ((b / Q) * (R / 2) + (b % Q) * 16) * 64 * KS);
    } else {
      const KMOE_LDS uint8_t* at = tile + (R == 256 ? place[b % Q] : place[b]);
      const int c = (R == 256 ? (b / Q) * 256 : 0) + ks * 64 * P;
      const tr4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((KMOE_LDS tr4_t*)(at + c));
      const tr4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((KMOE_LDS tr4_t*)(at + c + 8 * P));
      return __builtin_bit_cast(bf16x8_t, (short __attribute__((ext_vector_type(8)))){lo[0], lo[1], lo[2], lo[3], hi[0],
                                                                                     hi[1], hi[2], hi[3]});
    }
  }
};

// Waves of a SIMD that the tile leaves room for.
template <int BM, int BN, int KS, int STAGES>
constexpr int side_by_side = (BM * BN > 128 * 256 || (BM + BN) * 64 * KS * STAGES > 78 * 1024) ? 1 : 2;

template <int BM, int BN, int KS, int STAGES, bool SA, bool SB, int EPI, bool ADAPT>
__global__ __launch_bounds__(THREADS, (side_by_side<BM, BN, KS, STAGES>)) __attribute__((
    amdgpu_waves_per_eu(side_by_side<BM, BN, KS, STAGES>, side_by_side<BM, BN, KS, STAGES>))) void dense_kernel(Args g, int n_mt,
                                                                                                       int n_nt) {
  constexpr bool GATED = EPI == EPI_GATED;
  static_assert(!GATED || !SB, "gate and up rows are K-contiguous");
  static_assert(KS == 1 || KS == 2, "K per step");
  constexpr int PARTS = EPI == EPI_TWO ? 2 : 1;
  constexpr int SK = 32 * KS;
  using LoadA = Loads<BM, SA, KS>;
  using LoadB = Loads<BN, SB, KS>;
  static_assert(!GATED || LoadB::N % 2 == 0, "a wave's loads are of one half");
  constexpr int QA = BM / 64, QB = BN / 64;          // 16 x 16 blocks of a wave in a half
  constexpr int TILE = LoadA::BYTES, STAGE = TILE + LoadB::BYTES;
  constexpr int NP = LoadA::N + LoadB::N;            // loads of a wave and step
  constexpr int NR = 2 * (QA + QB), NM = 4 * QA * QB;  // fragments and MFMAs of a wave and 32 of K
  __shared__ __attribute__((aligned(1024))) uint8_t lds[STAGES * STAGE];
  __shared__ __attribute__((aligned(256))) int sid[ADAPT ? BM : 1];
  __shared__ int list[ADAPT ? BM : 1], n_list;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave >> 1, wn = wave & 1;
  int mt, nt;
  tile_of(blockIdx.x, n_mt, n_nt, mt, nt);
  const int64_t m0 = (int64_t)mt * BM;
  const int n0 = nt * (GATED ? BN / 2 : BN);
  KMOE_LDS uint8_t* const ldsp = (KMOE_LDS uint8_t*)lds;

  // where the step to load lies, and how much of K is left from it on
  const int64_t row_a = SA ? 1 : g.lda, row_b = SB ? 1 : g.ldb;
  const int64_t step_a = SA ? (int64_t)SK * g.lda : SK, step_b = SB ? (int64_t)SK * g.ldb : SK;
  const int64_t fold = BM == 64 && !SA && !GATED ? g.fold : 0;
  LoadA la;
  LoadB lb;
  la.init(g.lda, g.M - m0, false, fold, wave, lane);
  lb.init(g.ldb, g.N - n0, GATED, 0, wave, lane);
  const uint16_t* pa = g.a[0] + m0 * row_a;
  const uint16_t* pb = g.b[0] + n0 * row_b;
  const int64_t second = GATED ? g.b[1] - g.b[0] : 0;  // from the gate's to the up projection's rows
  int left = g.K, part = 1, to = 0;
  if (g.k_run) {
    const int k0 = blockIdx.y * g.k_run;
    left = g.K - k0 < g.k_run ? g.K - k0 : g.k_run;
    pa += SA ? k0 * g.lda : k0, pb += SB ? k0 * g.ldb : k0;
    g.c = static_cast<float*>(g.c) + blockIdx.y * g.M * g.ldc;
    if (blockIdx.y) g.ad.n = 0;  // (adapters: the first run's)
  }
  // piece q of the step to load, A's before B's
  auto place_piece = [&](int q) {
    return ldsp + to * STAGE + (q < LoadA::N ? wave + 4 * q : TILE / 1024 + wave + 4 * (q - LoadA::N)) * 1024;
  };
  auto load_piece = [&](int q) {
    const int c = q < LoadA::N ? q : q - LoadA::N;
    // (the second half of B's pieces are the second half of its rows)
    if (q < LoadA::N)
      dma16_at(pa, la.off[c]);
    else
      dma16_at(pb + (GATED && c >= LoadB::N / 2 ? second : 0), lb.off[c]);
  };
  auto next_step = [&]() {
    left -= SK, to = to + 1 == STAGES ? 0 : to + 1;
    pa += step_a, pb += step_b;
    if (left < SK) {  // the last step of a part and those past it
      if (PARTS == 2 && left <= 0 && part == 1) {
        left = g.K, part = 2;
        pa = g.a[1] + m0 * row_a;
        pb = g.b[1] + n0 * row_b;
        la.init(g.lda, g.M - m0, false, fold, wave, lane);
        lb.init(g.ldb, g.N - n0, GATED, 0, wave, lane);
      }
      if (left < SK) la.cut(left), lb.cut(left);
    }
  };
  const int nk = (left + SK - 1) / SK * PARTS;
  if (left < SK) la.cut(left), lb.cut(left);

  f32x4_t acc[2][2][QA][QB];
#pragma unroll
  for (int x = 0; x < 2; ++x)
#pragma unroll
    for (int y = 0; y < 2; ++y)
#pragma unroll
      for (int i = 0; i < QA; ++i)
#pragma unroll
        for (int j = 0; j < QB; ++j) acc[x][y][i][j] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  bf16x8_t fa[2][2 * QA], fb[2][2 * QB];
  Frags<BM, SA, KS> ra;
  Frags<BN, SB, KS> rb;
  ra.init(wm, lane);
  rb.init(wn, lane);
  // fragment r of 32 of a stage's K, B's before A's
  auto read_frag = [&](int set, int r, const KMOE_LDS uint8_t* st, int ks) {
    if (r < 2 * QB)
      fb[set][r] = rb.read(st + TILE, r, ks);
    else
      fa[set][r - 2 * QB] = ra.read(st, r - 2 * QB, ks);
  };

  if constexpr (ADAPT) {  // (ids past the tile's rows: zeros, which list_adapters does not look at)
    if (wave < BM / 64) {
      const int64_t m = m0 + tid;
      dma16_where((KMOE_LDS uint8_t*)sid + wave * 256);
      asm volatile("s_nop 1");
      dma4_at(g.ad.ids + m0, m < g.M ? (uint32_t)tid * 4 : NOWHERE);
    }
  }
#pragma unroll 1
  for (int s = 0; s < STAGES; ++s) {
#pragma unroll
    for (int q = 0; q < NP; ++q) {
      dma16_where(place_piece(q));
      asm volatile("s_nop 1");
      load_piece(q);
    }
    next_step();
  }
  if constexpr (ADAPT) {
    // (the ids have landed before the first step's operands)
    wait_vmcnt<STAGES * NP>();
    barrier_nofence();
    list_adapters<BM>(g.ad.n, g.M - m0 < BM ? (int)(g.M - m0) : BM, tid, sid, list, &n_list);
  }
  wait_vmcnt<(STAGES - 1) * NP>();
  barrier_nofence();
#pragma unroll
  for (int r = 0; r < NR; ++r) read_frag(0, r, ldsp, 0);
  constexpr int RS = NM >= 3 * NR + 8 ? 3 : NM >= 2 * NR ? 2 : 1;  // MFMAs from read to read: the last has time to land
  constexpr int PS = NM / NP;                                      // and from load to load
  static_assert(RS * (NR - 1) < NM && NP <= NM, "reads and loads find their places");
  int at = 0;  // where the step's stage begins
  // 32 of K of a step: its fragments are in set SET, those of the next 32 are read into the other;
  // LAST of a step: from the next stage, which has landed past the barrier, and the step STAGES on is
  // loaded into this one, of which every wave then has all fragments.
  auto sub = [&](auto ks_tag, auto set_tag) {
    constexpr int ks = decltype(ks_tag)::value, SET = decltype(set_tag)::value;
    constexpr bool LAST = ks == KS - 1;
    if constexpr (LAST) {
      wait_lgkmcnt0();
      wait_vmcnt<(STAGES - 2) * NP>();
      barrier_nofence();
      __builtin_amdgcn_sched_barrier(0);
      at = at == (STAGES - 1) * STAGE ? 0 : at + STAGE;
    }
    static_for<0, NM>([&](auto gt) {
      constexpr int G = decltype(gt)::value, a = G / (2 * QB), b = G % (2 * QB);
      f32x4_t& c = acc[a / QA][b / QB][a % QA][b % QB];
      c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[SET][b], fa[SET][a], c, 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
      constexpr bool reads = G % RS == 0 && G / RS < NR;
      constexpr bool points = LAST && G % PS == 0 && G / PS < NP;
      constexpr bool loads = LAST && G % PS == (PS > 1) && G / PS < NP;
      if constexpr (reads) read_frag(SET ^ 1, G / RS, ldsp + at, LAST ? 0 : ks + 1);
      if constexpr (points) dma16_where(place_piece(G / PS));
      if constexpr (points && loads) asm volatile("s_nop 1");  // (no MFMA between the two)
      if constexpr (loads) load_piece(G / PS);
      if constexpr (reads || points || loads) __builtin_amdgcn_sched_barrier(0);
    });
    if constexpr (LAST) next_step();
  };
  using Zero = std::integral_constant<int, 0>;
  using One = std::integral_constant<int, 1>;
  // (two times 32 of K, two steps or one of 64: the fragments' sets take turns.  An odd last step of 32
  // is followed by one of zeros.)
  // The accumulators stay in accumulation registers over the loop: left to itself the compiler keeps some
  // in others and copies them there and back in every step.
  auto hold = [&]() {
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int y = 0; y < 2; ++y)
#pragma unroll
        for (int i = 0; i < QA; ++i)
#pragma unroll
          for (int j = 0; j < QB; ++j) asm volatile("" : "+a"(acc[x][y][i][j]));
  };
  hold();
  int n = 0;
#pragma unroll 1
  do {
    sub(Zero{}, Zero{});
    sub(std::integral_constant<int, KS - 1>{}, One{});
  } while ((n += 2) < nk * KS);
  hold();
  wait_vmcnt<0>();  // (the zeros past the end are on their way into this workgroup's LDS)
  if constexpr (BM == 64 && !SA && !GATED) {
    if (fold) {  // (both halves' rows lie in one lane; the second half's are past M)
#pragma unroll
      for (int y = 0; y < 2; ++y)
#pragma unroll
        for (int j = 0; j < QB; ++j)
#pragma unroll
          for (int c = 0; c < 4; ++c) acc[0][y][0][j][c] = with_lost(acc[0][y][0][j][c], acc[1][y][0][j][c]);
      hold();
    }
  }
  if constexpr (ADAPT) {
    if (n_list) {
      Outer<BM, BN, GATED> outer(g.ad, sid, list, n_list, m0, g.M, n0, g.N, wm, wn, lane);
      outer.add(acc);
    }
    hold();
  }
  finish<BM, BN, EPI>(g, acc, m0, n0, wm, wn, lane);
}

}  // namespace kmoe_dense
