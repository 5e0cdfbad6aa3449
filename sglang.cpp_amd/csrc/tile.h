// Many tokens: tiles of weight rows x tokens whose operands go through LDS.
//
// WR x WC waves of 32 AT weight rows x 32 BT tokens each. 64 inputs of the tile's rows are a
// stage; two stages are in LDS. A stage is loaded as four pieces, in the order they are
// needed: the first halves of every wave's weight rows and of its tokens, the second half
// of the tokens, the second half of the rows. A piece's place is free as soon as its
// operands are in registers, a phase later the piece two stages ahead is on its way into
// it: loads have between one and two stages' products to arrive and no register holds them.
//
// A stage is four phases of AT BT 2 matrix instructions: rows 0 x tokens 0, rows 0 x tokens
// 1, rows 1 x tokens 1, rows 1 x tokens 0, each behind the reads of what it needs anew.
// With eight waves, two on a SIMD, waves 4-7 run half a phase behind waves 0-3: one reads
// while the other one multiplies.
#pragma once

#include "stream.h"

namespace sgl {
namespace gemm {

constexpr int kXcds = 8;  // chiplets, each with an L2 of its own, take workgroups in turn

template <int WR, int WC, int AT, int BT>
struct TileShape {
  static constexpr int kWaves = WR * WC;
  static constexpr int kM = WR * AT * 32, kN = WC * BT * 32;        // weight rows, tokens
  static constexpr int kPieceA = WR * AT * 16, kPieceB = WC * BT * 16;  // rows of a piece
  static constexpr int kLoadA = kPieceA / 8 / kWaves, kLoadB = kPieceB / 8 / kWaves;
  static constexpr int kOffA0 = 0, kOffB0 = kPieceA * 128, kOffB1 = kOffB0 + kPieceB * 128,
                       kOffA1 = kOffB1 + kPieceB * 128, kStage = kOffA1 + kPieceA * 128;
  static constexpr int kBytes = 2 * kStage;
};

template <int OFF, int N>
__device__ __forceinline__ void read_tiles(uint32_t at, u32x4_t (&f)[2][N]) {
  static_for<0, N>([&](auto i) {
    f[0][i.value] = lds_read<OFF + i.value * 2048>(at);
    f[1][i.value] = lds_read<OFF + i.value * 2048>(at ^ 64);
  });
}
template <int N>
__device__ __forceinline__ void wait_tiles(u32x4_t (&f)[2][N]) {
  static_for<0, N>([&](auto i) { lds_wait(f[0][i.value], f[1][i.value]); });
}

template <int DT, int AT, int BT>
__device__ __forceinline__ void multiply(const u32x4_t (&a)[2][AT], const u32x4_t (&b)[2][BT],
                                         f32x4_t (&acc)[AT][BT]) {
  __builtin_amdgcn_s_setprio(1);
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int i = 0; i < AT; ++i)
#pragma unroll
      for (int j = 0; j < BT; ++j) acc[i][j] = mfma16<DT>(a[h][i], b[h][j], acc[i][j]);
  __builtin_amdgcn_s_setprio(0);
}

// A barrier that no memory operation and no matrix instruction moves across; the waits in
// front of it are explicit.
__device__ __forceinline__ void phase_barrier() {
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
}

template <int DT, int MODE, bool GATED, int WR, int WC, int AT, int BT>
__global__ __launch_bounds__(64 * WR * WC, 2) void tile_kernel(const Args a) {
  using S = TileShape<WR, WC, AT, BT>;
  constexpr int LA = S::kLoadA, LB = S::kLoadB;
  constexpr bool kPhased = S::kWaves == 8;
  static_assert(LA == 2 && LB == 2, "a wave's loads of gate or up rows");
  __shared__ __attribute__((aligned(1024))) char lds[S::kBytes];
  // Consecutive workgroups go to the chiplets in turn: each chiplet has a run of tiles,
  // eight tiles of weights by all tiles of tokens after another, so that those it works on
  // at a time share rows of both.
  const int total = gridDim.x, xcd = blockIdx.x % kXcds;
  const int at = xcd * (total / kXcds) + min(xcd, total % kXcds) + static_cast<int>(blockIdx.x) / kXcds;
  const int tiles_t = total / a.tiles_n, band = at / (8 * tiles_t), in_band = at - band * 8 * tiles_t;
  const int wide = min(8, a.tiles_n - 8 * band);
  const int tn = 8 * band + in_band % wide, tt = in_band / wide;
  const Part p = part_of<MODE>(a, tt, S::kN);
  if (p.rows <= 0) return;
  const int n0 = tn * (GATED ? S::kM / 2 : S::kM);
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wr = wave % WR, wc = wave / WR;

  // This wave's loads: rows 8 q .. + 7 of a piece, q = wave LA + u. Lane offsets in bytes.
  uint32_t wo[2][LA], xo[2][LB];
  const bool up = GATED && (wave * LA / 2) % 2 == 1;
  const int first_n = min(n0, a.n - 1);
  const uint16_t* wbase = a.w + p.expert * a.w_se + ((up ? static_cast<int64_t>(a.n) : 0) + first_n) * a.w_st;
  const uint16_t* xbase = a.x + (MODE == kGateUp ? 0 : static_cast<int64_t>(p.first) * a.x_st);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
#pragma unroll
    for (int u = 0; u < LA; ++u) {
      const int q = wave * LA + u, r = 8 * q + (lane >> 3);
      const int row = r / (AT * 16) * (AT * 32) + h * (AT * 16) + r % (AT * 16);  // of the tile
      const int n = GATED ? (row >> 5) * 16 + (row & 15) : row;
      const int c = ((lane & 7) ^ ((4 * q + (lane >> 4)) & 7)) * 8;
      wo[h][u] = 2u * (static_cast<uint32_t>(min(n, a.n - 1 - first_n)) * static_cast<uint32_t>(a.w_st) + c);
    }
#pragma unroll
    for (int u = 0; u < LB; ++u) {
      const int q = wave * LB + u, r = 8 * q + (lane >> 3);
      const int row = min(r / (BT * 16) * (BT * 32) + h * (BT * 16) + r % (BT * 16), p.rows - 1);
      const int c = ((lane & 7) ^ ((4 * q + (lane >> 4)) & 7)) * 8;
      const uint32_t src = MODE == kGateUp ? a.order[p.first + row] / a.top_k : row;
      xo[h][u] = 2u * (src * static_cast<uint32_t>(a.x_st) + c);
    }
  }
  const auto wr_src = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(wbase), 0, kNowhere, 0x00027000);
  const auto xr_src = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(xbase), 0, kNowhere, 0x00027000);
  // Stage s is inputs 64 s .. + 63; where k is not a whole number of stages, the part of one
  // comes first (the order of the sum is free) and the others follow from input 0 on.
  const int tail = a.k % 64, stages = a.k / 64 + (tail ? 1 : 0);
  auto fetch_a = [&](int s, auto h, int slot) {
    const int k_at = __builtin_amdgcn_readfirstlane((s - (tail ? 1 : 0)) * 128);
#pragma unroll
    for (int u = 0; u < LA; ++u)
      stage16<false>(wr_src,
                     lds + slot * S::kStage + (h.value ? S::kOffA1 : S::kOffA0) + (wave * LA + u) * 1024,
                     wo[h.value][u], k_at);
  };
  auto fetch_b = [&](int s, auto h, int slot) {
    const int k_at = __builtin_amdgcn_readfirstlane((s - (tail ? 1 : 0)) * 128);
#pragma unroll
    for (int u = 0; u < LB; ++u)
      stage16<false>(xr_src,
                     lds + slot * S::kStage + (h.value ? S::kOffB1 : S::kOffB0) + (wave * LB + u) * 1024,
                     xo[h.value][u], k_at);
  };
  const std::integral_constant<int, 0> i0;
  const std::integral_constant<int, 1> i1;
  if (tail) {
    const int k_at = a.k - tail;
    auto part = [&](const __amdgpu_buffer_rsrc_t& src, uint32_t off, int q, int place) {
      const int c = ((lane & 7) ^ ((4 * q + (lane >> 4)) & 7)) * 8;
      const u32x4_t v = __builtin_amdgcn_raw_buffer_load_b128(src, c < tail ? off : kNowhere, 2 * k_at, 0);
      stg128(lds + place + q * 1024 + lane * 16, v);
    };
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int u = 0; u < LA; ++u) part(wr_src, wo[h][u], wave * LA + u, h ? S::kOffA1 : S::kOffA0);
#pragma unroll
      for (int u = 0; u < LB; ++u) part(xr_src, xo[h][u], wave * LB + u, h ? S::kOffB1 : S::kOffB0);
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" : : : "memory");
  } else {
    fetch_a(0, i0, 0), fetch_b(0, i0, 0), fetch_b(0, i1, 0), fetch_a(0, i1, 0);
  }
  if (stages > 1) {
    fetch_a(1, i0, 1), fetch_b(1, i0, 1), fetch_b(1, i1, 1), fetch_a(1, i1, 1);
    vm_wait<3 * LA + 3 * LB>();
  } else {
    vm_wait<0>();
  }
  phase_barrier();
  if (kPhased && wave >= 4) phase_barrier();

  const int r = lane & 15;
  const uint32_t base = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(
                            (__attribute__((address_space(3))) char*)lds)) +
                        r * 128 + (((lane >> 4) ^ (r >> 1)) & 7) * 16;
  const uint32_t base_a = base + wr * AT * 2048, base_b = base + wc * BT * 2048;
  f32x4_t acc[2][2][AT][BT] = {};
  u32x4_t fa[2][AT], fb0[2][BT], fb1[2][BT];
  for (int s = 0; s < stages; ++s) {
    const int slot = s & 1;
    const uint32_t at_a = base_a + slot * S::kStage, at_b = base_b + slot * S::kStage;
    const bool more = s + 2 < stages;
    // Rows 0 x tokens 0.
    read_tiles<S::kOffB0>(at_b, fb0);
    read_tiles<S::kOffA0>(at_a, fa);
    if (more) vm_wait<3 * LA + 2 * LB>();  // tokens 1 of this stage
    else vm_wait<0>();
    wait_tiles(fb0), wait_tiles(fa);
    phase_barrier();
    multiply<DT>(fa, fb0, acc[0][0]);
    if constexpr (kPhased) phase_barrier();
    // Rows 0 x tokens 1.
    read_tiles<S::kOffB1>(at_b, fb1);
    if (more) {
      fetch_a(s + 2, i0, slot), fetch_b(s + 2, i0, slot);
      vm_wait<3 * LA + 3 * LB>();  // rows 1 of this stage
    }
    wait_tiles(fb1);
    phase_barrier();
    multiply<DT>(fa, fb1, acc[0][1]);
    if constexpr (kPhased) phase_barrier();
    // Rows 1 x tokens 1.
    read_tiles<S::kOffA1>(at_a, fa);
    if (more) fetch_b(s + 2, i1, slot);
    wait_tiles(fa);
    phase_barrier();
    multiply<DT>(fa, fb1, acc[1][1]);
    if constexpr (kPhased) phase_barrier();
    // Rows 1 x tokens 0.
    if (more) {
      fetch_a(s + 2, i1, slot);
      vm_wait<3 * LA + 3 * LB>();  // rows 0 and tokens 0 of the next stage
    }
    phase_barrier();
    multiply<DT>(fa, fb0, acc[1][0]);
    if constexpr (kPhased) phase_barrier();
  }
  if (kPhased && wave < 4) phase_barrier();

#pragma unroll
  for (int hb = 0; hb < 2; ++hb)
#pragma unroll
    for (int j = 0; j < BT; ++j) {
      const int t = wc * BT * 32 + hb * BT * 16 + j * 16 + (lane & 15);
      if (t >= p.rows) continue;
      float scale;
      const int64_t row = target_row<MODE>(a, p.first + t, scale);
#pragma unroll
      for (int ha = 0; ha < 2; ++ha) {
        const int n = n0 + (wr * AT * 32 + ha * AT * 16) / (GATED ? 2 : 1) + 4 * (lane >> 4);
        if constexpr (GATED) {
#pragma unroll
          for (int i = 0; i < AT; i += 2)
            finish4<DT, MODE, true>(a, n + i * 8, row, scale, acc[ha][hb][i][j], acc[ha][hb][i + 1][j]);
        } else {
#pragma unroll
          for (int i = 0; i < AT; ++i)
            finish4<DT, MODE, false>(a, n + i * 16, row, scale, acc[ha][hb][i][j], acc[ha][hb][i][j]);
        }
      }
    }
}

template <int DT, int MODE, bool GATED, int WR, int WC, int AT, int BT>
int launch_tile(Args a, int64_t tiles_t, hipStream_t s) {
  using S = TileShape<WR, WC, AT, BT>;
  constexpr int out = GATED ? S::kM / 2 : S::kM;
  a.tiles_n = static_cast<int32_t>((static_cast<int64_t>(a.n) + out - 1) / out);
  const int64_t grid = grid_of(a.tiles_n, tiles_t);
  if (grid < 0) return SGL_ERR_UNSUPPORTED;
  hipLaunchKernelGGL((tile_kernel<DT, MODE, GATED, WR, WC, AT, BT>), dim3(static_cast<uint32_t>(grid)),
                     dim3(64 * S::kWaves), 0, s, a);
  return launch_status();
}

}  // namespace gemm
}  // namespace sgl
