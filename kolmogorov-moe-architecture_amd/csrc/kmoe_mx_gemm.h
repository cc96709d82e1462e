// Grouped expert products over microscaled rows and 4-bit weights: the tile kernel.
//   gate_up:  h[r, f] = silu(x[r] . w1[e][:, f]) * (x[r] . w2[e][:, f]), quantised to the
//             rows' own format in the epilogue
//   down:     y[r, n] = h[r] . w3[e][:, n], bf16
// for the rows r of expert e, [offsets[e], offsets[e+1]).  x and h are e4m3 (w4a8) or e2m1
// (w4a4) rows with one scale per 32 values, the weights are packed e2m1 (kmoe_mx.h).
//
// v_mfma_scale_f32_32x32x64_f8f6f4 takes both operands' codes and their scale bytes, so a
// block's scales cost no arithmetic.  Operand layout (lane l, row l % 32, half h = l / 32):
// e2m1 holds K 32 h .. + 31; e4m3 holds K 16 h .. + 15 and 32 + 16 h .. + 15; the scale byte
// of lane half h is that of K 32 h .. + 31 in both.  Weights are the first operand, so a
// lane's results are four consecutive output columns 8 c + 4 h .. of one row, c = 0 .. 3: a
// 32-column MX block of h is the 16 results of a lane and of its partner half.
//
// A workgroup of 2 x 2 waves owns 64 MI rows x 64 NJ weight rows, a wave 32 MI x 32 NJ.
// Both operands go global -> LDS directly, 128 of K per step, three stages; the K loop has
// one barrier per step, placed where every wave has the step's last fragments in registers.
#pragma once

#include <type_traits>

#include "kmoe_mx.h"

namespace kmoe_mx {

constexpr int GEMM_THREADS = 256;
constexpr int NST = 3;  // LDS stages

struct MxGemmArgs {
  const uint8_t* a;        // activation rows
  const uint8_t* a_scale;
  int64_t a_rows;          // rows of a (gathered) or max_rows
  const int32_t* row_token;  // gate_up: permuted row r is a's row row_token[r] (nullable; -1: zeros)
  const int32_t* offsets;
  int E;
  int k_steps;             // K / 128, padded
  const uint8_t* b;        // packed weights and scales
  const uint8_t* b_scale;
  int b_tiles;             // 256-row weight tiles of an expert
  uint8_t* q;              // gate_up: h's codes, scales, and (training) gate / up values
  uint8_t* q_scale;
  uint16_t* gu;
  uint16_t* c;             // down: output
  int64_t ldc;             // gate_up: padded columns of h; down: columns of c
  int n_valid;             // down: columns to store
  int n_ct;                // column tiles of 64 NJ weight rows
};

__device__ __forceinline__ i32x4_t buffer_of(const void* base, int64_t bytes) {
  const uint64_t p = (uint64_t)(uintptr_t)base;
  const int64_t n = bytes < 0 ? 0 : (bytes > 0x7fffffffll ? 0x7fffffffll : bytes);
  return i32x4_t{__builtin_amdgcn_readfirstlane((int)(uint32_t)p), __builtin_amdgcn_readfirstlane((int)(uint32_t)(p >> 32)),
                 __builtin_amdgcn_readfirstlane((int)n), 0x00020000};
}
// 16 (4) bytes per lane from buffer offset voff + soff to LDS, lane l at lds + 16 l (4 l); an
// offset past the buffer's end reads as zeros.  Written as asm for the reason given at
// dma16_to_lds: the caller orders these loads with wait_vmcnt and a barrier.
__device__ __forceinline__ void buffer_to_lds16(const i32x4_t& rsrc, uint32_t voff, uint32_t soff, uint32_t lds) {
  asm volatile("s_nop 1\n\tbuffer_load_dwordx4 %0, %1, %2 offen lds" ::"v"(voff), "s"(rsrc), "s"(soff), "{m0}"(lds));
}
__device__ __forceinline__ void buffer_to_lds4(const i32x4_t& rsrc, uint32_t voff, uint32_t soff, uint32_t lds) {
  asm volatile("s_nop 1\n\tbuffer_load_dword %0, %1, %2 offen lds" ::"v"(voff), "s"(rsrc), "s"(soff), "{m0}"(lds));
}

// Byte offset of 16-byte chunk `c` of LDS row `row`: rows of 128 bytes (e4m3) or 64 (e2m1),
// chunks XOR-ed so that the 16 rows of a read pass fall on distinct banks.
template <bool FP4>
__device__ __forceinline__ int a_lds(int row, int c) {
  return FP4 ? row * 64 + ((c ^ ((row >> 2) & 3)) << 4) : row * 128 + ((c ^ ((row >> 1) & 7)) << 4);
}

// Slot `slot` of `rows`-row slots numbered expert by expert: its expert and row range; n_slots
// is the number of slots of all experts.  Every wave of a workgroup calls it.
struct SlotScan {
  int lo, hi, incl;  // this lane's expert: rows, and slots up to and including it
  int n_slots;
};
template <int ROWS>
__device__ __forceinline__ SlotScan scan_slots(const int32_t* __restrict__ offsets, int E) {
  const int lane = threadIdx.x & 63;
  SlotScan s{0, 0, 0, 0};
  if (lane < E) {
    s.lo = offsets[lane];
    s.hi = offsets[lane + 1];
  }
  s.incl = (s.hi - s.lo + ROWS - 1) / ROWS;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int u = __shfl_up(s.incl, o, 64);
    if (lane >= o) s.incl += u;
  }
  s.n_slots = __builtin_amdgcn_readlane(s.incl, 63);
  return s;
}
template <int ROWS>
__device__ __forceinline__ void slot_rows(const SlotScan& s, int slot, int& e, int& m0, int& m_end) {
  e = __builtin_ctzll(__ballot(slot < s.incl));  // slot < n_slots: some lane holds it
  const int before = e > 0 ? __builtin_amdgcn_readlane(s.incl, e - 1) : 0;
  m0 = __builtin_amdgcn_readlane(s.lo, e) + (slot - before) * ROWS;
  m_end = __builtin_amdgcn_readlane(s.hi, e);
}

// Four values as bf16.
__device__ __forceinline__ i32x2_t pack4_bf16(float a, float b, float c, float d) {
  const uint32_t lo = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{a, b}, bf16x2_t));
  const uint32_t hi = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{c, d}, bf16x2_t));
  return i32x2_t{(int)lo, (int)hi};
}
// The low half of the wave gets (its x, its partner's x), the high half (its partner's y, its y).
__device__ __forceinline__ void swap_halves(uint32_t x, uint32_t y, uint32_t& first, uint32_t& second) {
  const auto r = __builtin_amdgcn_permlane32_swap(x, y, false, false);
  first = r[0];
  second = r[1];
}
// Eight consecutive bf16 columns from the runs c (x) and c + 1 (y): run c + half.
__device__ __forceinline__ i32x4_t merge_runs(i32x2_t x, i32x2_t y) {
  uint32_t a0, a1, b0, b1;
  swap_halves((uint32_t)x[0], (uint32_t)y[0], a0, a1);
  swap_halves((uint32_t)x[1], (uint32_t)y[1], b0, b1);
  return i32x4_t{(int)a0, (int)b0, (int)a1, (int)b1};
}

// Stores a row's 32 values, 16 a lane (v[4 c + t]: column 8 c + 4 half + t), as an MX block.
// q: the block's codes, scale: its byte; nothing is stored where !on.  All lanes take part.
template <bool FP4>
__device__ __forceinline__ void store_block(const float (&v)[16], int half, bool on, uint8_t* q, uint8_t* scale) {
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < 16; ++i) m = amax_nan(m, v[i]);
  uint32_t o0, o1;
  swap_halves(__float_as_uint(m), __float_as_uint(m), o0, o1);  // (own or partner's, the other)
  m = fmaxf(__uint_as_float(o0), __uint_as_float(o1));
  const uint32_t code = scale_code<FP4>(m);
  const Codes<FP4, 16> d = encode<FP4, 16>(v, code);
  if constexpr (FP4) {
    // d.w[p]: runs 2 p (low 16 bits) and 2 p + 1
    uint32_t a, b;
    swap_halves(d.w[0], d.w[1], a, b);
    if (on) *reinterpret_cast<i32x2_t*>(q + 8 * half) = i32x2_t{(int)((a & 0xffffu) | (b << 16)), (int)((a >> 16) | (b & 0xffff0000u))};
  } else {
    uint32_t a0, a1, b0, b1;
    swap_halves(d.w[0], d.w[2], a0, a1);
    swap_halves(d.w[1], d.w[3], b0, b1);
    if (on) *reinterpret_cast<i32x4_t*>(q + 16 * half) = i32x4_t{(int)a0, (int)a1, (int)b0, (int)b1};
  }
  if (on && half == 0) *scale = (uint8_t)code;
}

template <bool GATE_UP, bool FP4, int MI, int NJ, bool SAVE_GU>
struct MxTile {
  static constexpr int BM = 64 * MI;
  static constexpr int AB = BM * (FP4 ? 64 : 128), BB = NJ * 4096, AS = BM * 4, BS = NJ * 256;
  static constexpr int STAGE = AB + BB + AS + BS;
  static constexpr int NA = AB / 4096, NB = NJ, NL = NA + NB + 2;  // loads per wave and step
  static_assert(NST * STAGE <= 160 * 1024, "LDS");
};

template <bool GATE_UP, bool FP4, int MI, int NJ, bool SAVE_GU>
__global__ __launch_bounds__(GEMM_THREADS, 1) void mx_gemm_kernel(MxGemmArgs g) {
  using T = MxTile<GATE_UP, FP4, MI, NJ, SAVE_GU>;
  static_assert(!SAVE_GU || GATE_UP, "gate / up values are the first product's");
  __shared__ __attribute__((aligned(1024))) uint8_t lds[NST * T::STAGE];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lr = lane & 31, lh = lane >> 5;
  const int wm = wave >> 1, wn = wave & 1;

  // tile: each XCD (workgroups go round over the 8) takes a contiguous range of the tiles, in
  // which four slots share a column tile's weights in its L2
  const SlotScan st = scan_slots<T::BM>(g.offsets, g.E);
  const int n_all = st.n_slots * g.n_ct;
  const int chunk = (n_all + 7) / 8, at = blockIdx.x >> 3;
  const int t = (blockIdx.x & 7) * chunk + at;
  if (at >= chunk || t >= n_all) return;
  int slot, ct;
  {
    const int full = (st.n_slots >> 2) * 4 * g.n_ct;
    if (t < full) {
      const int grp = t / (4 * g.n_ct), r = t - grp * 4 * g.n_ct;
      ct = r >> 2;
      slot = grp * 4 + (r & 3);
    } else {
      const int rem = st.n_slots & 3, u = t - full;
      ct = u / rem;
      slot = (st.n_slots & ~3) + (u - ct * rem);
    }
  }
  int e, m0, m_end;
  slot_rows<T::BM>(st, slot, e, m0, m_end);
  const int rows = m_end - m0;

  // operand windows and per-lane offsets of a step's loads
  const int64_t lda = (int64_t)g.k_steps * (FP4 ? 64 : 128), lds_a = (int64_t)g.k_steps * 4;
  const bool gather = GATE_UP && g.row_token;
  const i32x4_t ar = gather ? buffer_of(g.a, g.a_rows * lda) : buffer_of(g.a + m0 * lda, rows * lda);
  const i32x4_t sr = gather ? buffer_of(g.a_scale, g.a_rows * lds_a) : buffer_of(g.a_scale + m0 * lds_a, rows * lds_a);
  constexpr int SPLIT = 4 / NJ;  // column tiles of a weight tile
  const int64_t bt = ((int64_t)e * g.b_tiles + ct / SPLIT) * g.k_steps;
  const i32x4_t br = buffer_of(g.b + bt * TILE_STEP + (ct % SPLIT) * T::BB, (int64_t)g.k_steps * TILE_STEP - (ct % SPLIT) * T::BB);
  const i32x4_t tr = buffer_of(g.b_scale + bt * SCALE_STEP + (ct % SPLIT) * T::BS, (int64_t)g.k_steps * SCALE_STEP - (ct % SPLIT) * T::BS);
  constexpr uint32_t NONE = 0x80000000u;  // an offset past every window
  auto source_row = [&](int r) -> uint32_t {  // row of `a` (or of the slot) that tile row r is; NONE without one
    if (r >= rows) return NONE;
    if (!gather) return (uint32_t)r;
    const int src = g.row_token[m0 + r];
    return src < 0 ? NONE : (uint32_t)src;
  };
  constexpr int CPR = FP4 ? 4 : 8, RPB = 64 / CPR;  // 16-byte chunks per row, rows per 1 KiB load
  uint32_t aoff[T::NA];
#pragma unroll
  for (int q = 0; q < T::NA; ++q) {
    const int r = (wave * T::NA + q) * RPB + lane / CPR;
    // LDS position lane % CPR of the row holds chunk (lane % CPR) ^ swizzle
    const uint32_t chunk16 = (uint32_t)((lane % CPR) ^ (FP4 ? (r >> 2) & 3 : (r >> 1) & 7)) << 4;
    const uint32_t src = source_row(r);
    aoff[q] = src == NONE ? NONE : src * (uint32_t)lda + chunk16;
  }
  const uint32_t ssrc = source_row((wave % MI) * 64 + lane);
  const uint32_t soff = ssrc == NONE ? NONE : ssrc * (uint32_t)lds_a;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(KMOE_LDS uint8_t*)lds;

  auto load_step = [&](int kt) {
    const uint32_t base = lds0 + (uint32_t)(kt % NST) * T::STAGE;
    const int k = __builtin_amdgcn_readfirstlane(kt);
#pragma unroll
    for (int q = 0; q < T::NA; ++q)
      buffer_to_lds16(ar, aoff[q], k * (FP4 ? 64 : 128), __builtin_amdgcn_readfirstlane(base + (wave * T::NA + q) * 1024));
#pragma unroll
    for (int q = 0; q < T::NB; ++q)
      buffer_to_lds16(br, (wave * T::NB + q) * 1024 + lane * 16, k * TILE_STEP,
                      __builtin_amdgcn_readfirstlane(base + T::AB + (wave * T::NB + q) * 1024));
    // scales: 64 rows (128-byte halves of the column blocks) a load; with fewer loads than
    // waves two waves write the same values
    buffer_to_lds4(sr, soff, k * 4, __builtin_amdgcn_readfirstlane(base + T::AB + T::BB + (wave % MI) * 256));
    buffer_to_lds4(tr, (wave % NJ) * 256 + lane * 4, k * SCALE_STEP,
                   __builtin_amdgcn_readfirstlane(base + T::AB + T::BB + T::AS + (wave % NJ) * 256));
  };

  f32x16_t acc[MI][NJ];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;

  i32x8_t fa[2][MI];
  i32x4_t fb[2][NJ];
  int sa[2][MI], sb[2][NJ];  // scales of a step (both substeps), double buffered
  auto read_sub = [&](int kt, int i, int set) {
    const uint8_t* const st = lds + (kt % NST) * T::STAGE;
#pragma unroll
    for (int mi = 0; mi < MI; ++mi) {
      const int r = wm * 32 * MI + mi * 32 + lr;
      if constexpr (FP4) {
        const i32x4_t v = *reinterpret_cast<const i32x4_t*>(st + a_lds<true>(r, 2 * i + lh));
        fa[set][mi] = i32x8_t{v[0], v[1], v[2], v[3], 0, 0, 0, 0};
      } else {
        const i32x4_t v = *reinterpret_cast<const i32x4_t*>(st + a_lds<false>(r, 4 * i + lh));
        const i32x4_t u = *reinterpret_cast<const i32x4_t*>(st + a_lds<false>(r, 4 * i + 2 + lh));
        fa[set][mi] = i32x8_t{v[0], v[1], v[2], v[3], u[0], u[1], u[2], u[3]};
      }
    }
#pragma unroll
    for (int j = 0; j < NJ; ++j)
      fb[set][j] = *reinterpret_cast<const i32x4_t*>(st + T::AB + (wn * NJ + j) * 2048 + i * 1024 + lane * 16);
  };
  auto read_scales = [&](int kt, int set) {
    const uint8_t* const sp = lds + (kt % NST) * T::STAGE + T::AB + T::BB;
#pragma unroll
    for (int mi = 0; mi < MI; ++mi)
      sa[set][mi] = (int)(*reinterpret_cast<const uint32_t*>(sp + (wm * 32 * MI + mi * 32 + lr) * 4) >> (8 * lh));
#pragma unroll
    for (int j = 0; j < NJ; ++j)
      sb[set][j] = *reinterpret_cast<const uint16_t*>(sp + T::AS + (wn * NJ + j) * 128 + lane * 2);
  };
  auto mma = [&](auto i_tag, int set) {
    constexpr int i = decltype(i_tag)::value;
#pragma unroll
    for (int mi = 0; mi < MI; ++mi)
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const i32x4_t b = fb[i][j];
        acc[mi][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(i32x8_t{b[0], b[1], b[2], b[3], 0, 0, 0, 0}, fa[i][mi],
                                                                      acc[mi][j], 4, FP4 ? 4 : 0, i, sb[set][j], 2 * i,
                                                                      sa[set][mi]);
      }
  };

  const int nk = g.k_steps;
#pragma unroll
  for (int s = 0; s < NST; ++s)
    if (s < nk) load_step(s);
  if (nk >= 3)
    wait_vmcnt<2 * T::NL>();
  else if (nk == 2)
    wait_vmcnt<T::NL>();
  else
    wait_vmcnt<0>();
  barrier_nofence();
  read_sub(0, 0, 0);
  read_scales(0, 0);
  // Step kt: its first half is in registers.  Its second half is read under the first half's
  // products; then every wave is done with the step's stage, so the barrier that publishes
  // step kt + 1 also frees it for step kt + 3.
  auto step = [&](int kt, auto par_tag) {
    constexpr int par = decltype(par_tag)::value;  // set of the step's scales
    read_sub(kt, 1, 1);
    mma(std::integral_constant<int, 0>{}, par);
    if (kt + 1 < nk) {
      wait_lgkmcnt0();
      if (kt + 2 < nk)
        wait_vmcnt<T::NL>();
      else
        wait_vmcnt<0>();
      barrier_nofence();
      if (kt + 3 < nk) load_step(kt + 3);
      read_sub(kt + 1, 0, 0);
      read_scales(kt + 1, par ^ 1);
    }
    mma(std::integral_constant<int, 1>{}, par);
  };
  int kt = 0;
#pragma unroll 1
  for (; kt + 1 < nk; kt += 2) {
    step(kt, std::integral_constant<int, 0>{});
    step(kt + 1, std::integral_constant<int, 1>{});
  }
  if (kt < nk) step(kt, std::integral_constant<int, 0>{});

  // ---- epilogue: lane's row of block mi, columns 8 c + 4 lh + t of block j
#pragma unroll
  for (int mi = 0; mi < MI; ++mi) {
    const int r = wm * 32 * MI + mi * 32 + lr;
    const bool on = r < rows;
    const int64_t row = m0 + r;
    if constexpr (GATE_UP) {
#pragma unroll
      for (int p = 0; p < NJ / 2; ++p) {
        const int f0 = (ct * 2 * NJ + wn * NJ) * 16 + p * 32;  // first of the block's 32 columns
        float h[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) h[i] = silu_fast_f32(acc[mi][2 * p][i]) * acc[mi][2 * p + 1][i];
        store_block<FP4>(h, lh, on, g.q + row * (g.ldc / (FP4 ? 2 : 1)) + f0 / (FP4 ? 2 : 1),
                         g.q_scale + row * (g.ldc / BLOCK) + f0 / BLOCK);
        if constexpr (SAVE_GU) {
          uint16_t* const gp = g.gu + row * 2 * g.ldc + (f0 >> 7) * 256 + (f0 & 127) + 8 * lh;
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int c = 0; c < 4; c += 2) {
              const f32x16_t& a = acc[mi][2 * p + u];
              const i32x4_t v = merge_runs(pack4_bf16(a[4 * c], a[4 * c + 1], a[4 * c + 2], a[4 * c + 3]),
                                           pack4_bf16(a[4 * c + 4], a[4 * c + 5], a[4 * c + 6], a[4 * c + 7]));
              if (on) *reinterpret_cast<i32x4_t*>(gp + u * 128 + 8 * c) = v;
            }
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int c = 0; c < 4; c += 2) {
          const f32x16_t& a = acc[mi][j];
          const i32x4_t v = merge_runs(pack4_bf16(a[4 * c], a[4 * c + 1], a[4 * c + 2], a[4 * c + 3]),
                                       pack4_bf16(a[4 * c + 4], a[4 * c + 5], a[4 * c + 6], a[4 * c + 7]));
          const int col = (ct * 2 * NJ + wn * NJ + j) * 32 + 8 * (c + lh);
          if (on && col < g.n_valid) *reinterpret_cast<i32x4_t*>(g.c + row * g.ldc + col) = v;
        }
    }
  }
}

// One product to launch; the variants are compiled in separate files.
struct MxLaunch {
  MxGemmArgs g;
  int64_t max_rows;
  hipStream_t s;
};
template <bool GATE_UP, bool FP4, int MI, int NJ, bool SAVE_GU = false>
void launch_mx_tile(MxLaunch l) {
  using T = MxTile<GATE_UP, FP4, MI, NJ, SAVE_GU>;
  l.g.n_ct = l.g.b_tiles * (4 / NJ);
  const int64_t slots = l.max_rows / T::BM + (l.max_rows < l.g.E ? l.max_rows : l.g.E);
  const int64_t blocks = (slots * l.g.n_ct + 7) / 8 * 8;
  hipLaunchKernelGGL((mx_gemm_kernel<GATE_UP, FP4, MI, NJ, SAVE_GU>), dim3((unsigned)blocks), dim3(GEMM_THREADS), 0, l.s, l.g);
}
void launch_mx_gate_up(const MxLaunch& l, bool fp4, int mi);  // with l.g.gu: saving the gate / up values
void launch_mx_down(const MxLaunch& l, bool fp4, int mi);

}  // namespace kmoe_mx
