// Grouped products over microscaled rows for few rows per expert (decode steps, short
// prompts), where the time is that of streaming the 4-bit weights once.
//
// A workgroup owns one slot of 32 rows of an expert and 32 output columns (gate/up: the 32
// gate and the 32 up rows of the same columns); its eight waves split K, each loading its
// weights and rows straight into MFMA operand registers, and their sums meet in LDS in wave
// order.  v_mfma_scale_f32_16x16x128_f8f6f4, weights first: lane l holds weight row l % 16 at
// K 32 q .. + 31 (q = l / 16), which the packed order has as 16 bytes; an activation row's K
// 16 q .. and 64 + 16 q .. (e4m3) or 32 q .. (e2m1); the scale byte is that of K 32 q ..
// The result lane holds output columns 4 q .. + 3 of row l % 16.
//
// With a row or two an expert there are too few column tiles to fill the CUs and the time is one
// wave's chain of K steps, so K is split: one token, top-2 of 16 experts, d 2048, F 2816, weights
// from HBM, gate/up 6.5 us and down 4.9 (64 x 128 tiles 9.0 and 9.8).  When it stops paying is
// said at its launch rule.
#include <type_traits>

#include "kmoe_mx_gemm.h"

namespace kmoe_mx {
namespace {

constexpr int WAVES = 8;
constexpr int DEPTH = 2;  // steps of a wave in flight

__device__ __forceinline__ i32x4_t load16(__amdgpu_buffer_rsrc_t r, uint32_t off, int soff) {
  return __builtin_bit_cast(i32x4_t, __builtin_amdgcn_raw_buffer_load_b128(r, off, soff, 0));
}
__device__ __forceinline__ __amdgpu_buffer_rsrc_t window(const void* base, int64_t bytes) {
  const int n = bytes < 0 ? 0 : (bytes > 0x7fffffffll ? 0x7fffffff : (int)bytes);
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0, n, 0x00020000);
}

template <bool GATE_UP, bool FP4>
__global__ __launch_bounds__(64 * WAVES) void mx_small_kernel(MxGemmArgs g) {
  constexpr int NB = GATE_UP ? 4 : 2;  // 16-row weight blocks: (gate, up) x two halves of 32 columns
  __shared__ f32x4_t red[WAVES][2 * NB][64];
  const SlotScan st = scan_slots<SMALL_ROWS>(g.offsets, g.E);
  const int slot = blockIdx.x / g.n_ct, ct = blockIdx.x - slot * g.n_ct;
  if (slot >= st.n_slots) return;
  int e, m0, m_end;
  slot_rows<SMALL_ROWS>(st, slot, e, m0, m_end);
  const int lane = threadIdx.x & 63, r16 = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int rows = min(m_end - m0, SMALL_ROWS);
  const int nk = g.k_steps, s0 = wave * nk / WAVES, s1 = (wave + 1) * nk / WAVES;

  // weights: 32-row block pair (gate/up) or block of this column block
  constexpr int PER_TILE = GATE_UP ? 4 : 8;  // column blocks of a weight tile
  const int64_t tile = ((int64_t)e * g.b_tiles + ct / PER_TILE) * nk;
  const uint8_t* const wq = g.b + tile * TILE_STEP + (ct % PER_TILE) * (GATE_UP ? 4096 : 2048);
  const uint8_t* const ws = g.b_scale + tile * SCALE_STEP + (ct % PER_TILE) * NB;
  const uint32_t woff = (q >> 1) * 1024 + ((q & 1) * 32 + r16) * 16;   // + 256 for the other 16 rows, + 2048 for up
  const uint32_t soff = lane * 16;
  const int64_t lda = (int64_t)nk * (FP4 ? 64 : 128), lds_a = (int64_t)((nk + 3) / 4) * 16;
  const bool gather = GATE_UP && g.row_token;
  const uint8_t* const abase = gather ? g.a : g.a + m0 * lda;
  const uint8_t* const sbase = gather ? g.a_scale : g.a_scale + m0 * lds_a;
  const int64_t a_rows = gather ? g.a_rows : rows;  // rows past these read as zeros

  f32x4_t acc[2][NB];
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int b = 0; b < NB; ++b) acc[m][b] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};

  auto run = [&](auto mb_tag) {
    constexpr int MB = decltype(mb_tag)::value;  // 16-row blocks with rows
    constexpr int PA = FP4 ? 1 : 2;
    i32x4_t w[DEPTH][NB], a[DEPTH][MB][PA];
    int sw[DEPTH], sa[DEPTH][MB];
    // step s into ring entry u; steps past the wave's range read nothing (empty windows)
    auto load_w = [&](int u, int s) {
      const __amdgpu_buffer_rsrc_t rw = window(wq, s < s1 ? 0x7fffffff : 0), rs = window(ws, s < s1 ? 0x7fffffff : 0);
#pragma unroll
      for (int b = 0; b < NB; ++b) w[u][b] = load16(rw, woff + (b & 1) * 256 + (b >> 1) * 2048, s * TILE_STEP);
      sw[u] = GATE_UP ? (int)__builtin_amdgcn_raw_buffer_load_b32(rs, soff, s * SCALE_STEP, 0)
                      : (int)__builtin_amdgcn_raw_buffer_load_b16(rs, soff, s * SCALE_STEP, 0);
    };
    uint32_t aoff[MB], asoff[MB];
    auto load_a = [&](int u, int s) {
      const __amdgpu_buffer_rsrc_t ra = window(abase, s < s1 ? a_rows * lda : 0), rs = window(sbase, s < s1 ? a_rows * lds_a : 0);
#pragma unroll
      for (int m = 0; m < MB; ++m) {
#pragma unroll
        for (int p = 0; p < PA; ++p) a[u][m][p] = load16(ra, aoff[m] + 64u * p, s * (FP4 ? 64 : 128));
        sa[u][m] = __builtin_amdgcn_raw_buffer_load_b8(rs, asoff[m], s * 4, 0);
      }
    };
    // the weights first: their addresses do not wait for the row lookup
#pragma unroll
    for (int u = 0; u < DEPTH; ++u) load_w(u, s0 + u);
#pragma unroll
    for (int m = 0; m < MB; ++m) {
      const int r = m * 16 + r16;
      const uint32_t src = r < rows ? (gather ? (uint32_t)g.row_token[m0 + r] : (uint32_t)r) : ~0u;
      // (a missing row's offset is past every window; that of a row past the end could wrap into it)
      const bool on = src < (uint32_t)a_rows;
      aoff[m] = on ? src * (uint32_t)lda + q * 16u : 0x80000000u;
      asoff[m] = on ? src * (uint32_t)lds_a + q : 0x80000000u;
    }
#pragma unroll
    for (int u = 0; u < DEPTH; ++u) load_a(u, s0 + u);
    for (int s = s0; s < s1; s += DEPTH) {
#pragma unroll
      for (int u = 0; u < DEPTH; ++u) {
        // entries past the range hold zeros (codes and scales)
#pragma unroll
        for (int m = 0; m < MB; ++m)
          static_for<0, NB>([&](auto b) {
            const i32x4_t wv = w[u][b], a0 = a[u][m][0], a1 = FP4 ? i32x4_t{0, 0, 0, 0} : a[u][m][PA - 1];
            acc[m][b] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                i32x8_t{wv[0], wv[1], wv[2], wv[3], 0, 0, 0, 0}, i32x8_t{a0[0], a0[1], a0[2], a0[3], a1[0], a1[1], a1[2], a1[3]},
                acc[m][b], 4, FP4 ? 4 : 0, decltype(b)::value, sw[u], 0, sa[u][m]);
          });
        load_w(u, s + u + DEPTH);
        load_a(u, s + u + DEPTH);
      }
    }
#pragma unroll
    for (int m = 0; m < MB; ++m)
#pragma unroll
      for (int b = 0; b < NB; ++b) red[wave][m * NB + b][lane] = acc[m][b];
  };
  const int nb = rows > 16 ? 2 : 1;
  if (nb == 2)
    run(std::integral_constant<int, 2>{});
  else
    run(std::integral_constant<int, 1>{});
  __syncthreads();
  auto total = [&](int i) {
    f32x4_t t = red[0][i][lane];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) t += red[w][i][lane];
    return t;
  };
  if constexpr (GATE_UP) {
    if (wave >= nb) return;
    const int r = wave * 16 + r16;
    const bool on = r < rows;
    const int64_t row = m0 + r;
    float h[2][4], gv[2][4], uv[2][4];
    uint32_t m = 0;
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const f32x4_t gt = total(wave * NB + hf), up = total(wave * NB + 2 + hf);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        gv[hf][c] = gt[c];
        uv[hf][c] = up[c];
        h[hf][c] = silu_fast_f32(gt[c]) * up[c];
        m = amax_bits(m, h[hf][c]);
      }
    }
    // the block's 32 columns are 8 values in each of the row's four lanes
    m = max(m, (uint32_t)__shfl_xor((int)m, 16, 64));
    m = max(m, (uint32_t)__shfl_xor((int)m, 32, 64));
    const uint32_t code = scale_code<FP4>(m);
    const float v[8] = {h[0][0], h[0][1], h[0][2], h[0][3], h[1][0], h[1][1], h[1][2], h[1][3]};
    const Codes<FP4, 8> d = encode<FP4, 8>(v, code);
    if (!on) return;
    const int f0 = ct * 32;
    uint8_t* const out = g.q + row * (g.ldc / (FP4 ? 2 : 1)) + f0 / (FP4 ? 2 : 1);
    if constexpr (FP4) {
      *reinterpret_cast<uint16_t*>(out + 2 * q) = (uint16_t)d.w[0];
      *reinterpret_cast<uint16_t*>(out + 8 + 2 * q) = (uint16_t)(d.w[0] >> 16);
    } else {
      *reinterpret_cast<uint32_t*>(out + 4 * q) = d.w[0];
      *reinterpret_cast<uint32_t*>(out + 16 + 4 * q) = d.w[1];
    }
    if (q == 0) g.q_scale[row * scale_bytes((int)g.ldc) + f0 / BLOCK] = (uint8_t)code;
    if (g.gu) {
      uint16_t* const gp = g.gu + row * 2 * g.ldc + (f0 >> 7) * 256 + (f0 & 127) + 4 * q;
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        *reinterpret_cast<i32x2_t*>(gp + 16 * hf) = pack4_bf16(gv[hf][0], gv[hf][1], gv[hf][2], gv[hf][3]);
        *reinterpret_cast<i32x2_t*>(gp + 128 + 16 * hf) = pack4_bf16(uv[hf][0], uv[hf][1], uv[hf][2], uv[hf][3]);
      }
    }
  } else {
    if (wave >= NB * nb) return;
    const int r = (wave / NB) * 16 + r16, col = ct * 32 + (wave % NB) * 16 + 4 * q;
    if (r < rows && col < g.n_valid) {
      const f32x4_t t = total(wave);
      *reinterpret_cast<i32x2_t*>(g.c + (int64_t)(m0 + r) * g.ldc + col) = pack4_bf16(t[0], t[1], t[2], t[3]);
    }
  }
}

template <bool GATE_UP, bool FP4>
void launch(MxLaunch l) {
  l.g.n_ct = l.g.b_tiles * (GATE_UP ? 4 : 8);
  const int64_t slots = l.max_rows / SMALL_ROWS + (l.max_rows < l.g.E ? l.max_rows : l.g.E);
  hipLaunchKernelGGL((mx_small_kernel<GATE_UP, FP4>), dim3((unsigned)(slots * l.g.n_ct)), dim3(64 * WAVES), 0, l.s, l.g);
}

}  // namespace

void launch_mx_small(const MxLaunch& l, bool gate_up, bool fp4) {
  if (gate_up)
    fp4 ? launch<true, true>(l) : launch<true, false>(l);
  else
    fp4 ? launch<false, true>(l) : launch<false, false>(l);
}

}  // namespace kmoe_mx
