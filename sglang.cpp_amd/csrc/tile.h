// Many tokens: tiles of weight rows x tokens whose operands go through LDS.
//
// WR x WC waves of 32 AT weight rows x 32 BT tokens each. 64 inputs of the tile's rows are a
// stage; D stages are in LDS. A stage is loaded as four pieces, in the order they are
// needed: the first halves of every wave's weight rows and of its tokens, the second half
// of the tokens, the second half of the rows. A piece's place is free as soon as its
// operands are in registers, a phase later the piece D stages ahead is on its way into
// it: loads have between D - 1 and D stages' products to arrive and no register holds them.
//
// Eight waves (256 x 256 tiles, one workgroup a CU): a stage is four phases of AT BT 2 matrix
// instructions: rows 0 x tokens 0, rows 0 x tokens 1, rows 1 x tokens 1, rows 1 x tokens 0,
// each behind the reads of what it needs anew. Waves 4-7, the second one of each SIMD, run half
// a phase behind waves 0-3: one reads while the other one multiplies. Four waves (smaller tiles,
// two workgroups a CU): the operands of the next stage are read between the products of
// this one. 8,192 x 24,576 x 4,096: 1,340 to 1,380 TFLOP/s, bound by the matrix instructions and the clock that
// they leave (1,830 alone on random operands).
#pragma once

#include "stream.h"

namespace sgl {
namespace gemm {

constexpr int kXcds = 8;  // chiplets, each with an L2 of its own, take workgroups in turn

template <int WR, int WC, int AT, int BT, int D>
struct TileShape {
  static constexpr int kWaves = WR * WC;
  static constexpr int kM = WR * AT * 32, kN = WC * BT * 32;        // weight rows, tokens
  static constexpr int kPieceA = WR * AT * 16, kPieceB = WC * BT * 16;  // rows of a piece
  static constexpr int kLoadA = kPieceA / 8 / kWaves, kLoadB = kPieceB / 8 / kWaves;
  static constexpr int kOffA0 = 0, kOffB0 = kPieceA * 128, kOffB1 = kOffB0 + kPieceB * 128,
                       kOffA1 = kOffB1 + kPieceB * 128, kStage = kOffA1 + kPieceA * 128;
  static constexpr int kBytes = D * kStage, kLoads = 2 * kLoadA + 2 * kLoadB;
};

// LDS operations of a wave are in order; this keeps the compiler from changing it.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

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

// The operands of a whole stage and their products, for waves that have their SIMD's matrix
// unit to themselves: [half of 64 inputs][half of the rows or tokens][tile].
template <int AT, int BT>
struct Operands {
  u32x4_t a[2][2][AT], b[2][2][BT];

  // Reads the stage in `slot`; between the reads, part(i) for i = 0 .. 4 (AT + BT) - 1.
  template <typename S, int D, typename F>
  __device__ __forceinline__ void read(uint32_t base_a, uint32_t base_b, int slot, F&& part) {
    const uint32_t at_a[2] = {base_a + slot * S::kStage, (base_a + slot * S::kStage) ^ 64};
    const uint32_t at_b[2] = {base_b + slot * S::kStage, (base_b + slot * S::kStage) ^ 64};
    static_for<0, 4 * (AT + BT)>([&](auto i) {
      constexpr int k = i.value / (2 * (AT + BT)), r = i.value % (2 * (AT + BT));
      if constexpr (r < 2 * AT)
        a[k][r / AT][r % AT] = lds_read<(r / AT ? S::kOffA1 : S::kOffA0) + r % AT * 2048>(at_a[k]);
      else
        b[k][(r - 2 * AT) / BT][(r - 2 * AT) % BT] =
            lds_read<((r - 2 * AT) / BT ? S::kOffB1 : S::kOffB0) + (r - 2 * AT) % BT * 2048>(at_b[k]);
      part(i);
      __builtin_amdgcn_sched_barrier(0);
    });
  }

  __device__ __forceinline__ void wait() {
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int i = 0; i < AT; ++i) lds_wait(a[k][h][i]);
#pragma unroll
        for (int j = 0; j < BT; ++j) lds_wait(b[k][h][j]);
      }
  }

  // The I-th of 4 (AT + BT) shares of the products.
  template <int DT, typename I>
  __device__ __forceinline__ void multiply(I, f32x4_t (&acc)[2][2][AT][BT]) const {
    constexpr int kAll = 8 * AT * BT, kParts = 4 * (AT + BT);
    static_for<I::value * kAll / kParts, (I::value + 1) * kAll / kParts>([&](auto n) {
      constexpr int k = n.value / (4 * AT * BT), m = n.value % (4 * AT * BT);
      constexpr int ha = m / (2 * AT * BT), i = m / (2 * BT) % AT, hb = m / BT % 2, j = m % BT;
      acc[ha][hb][i][j] = mfma16<DT>(a[k][ha][i], b[k][hb][j], acc[ha][hb][i][j]);
    });
  }
};

// Waits until at most `left` whole stages and kMore loads are in flight, left < D.
template <int D, int kLoads, int kMore>
__device__ __forceinline__ void stages_wait(int left) {
  static_for<0, D>([&](auto i) {
    if (left == i.value) vm_wait<i.value * kLoads + kMore>();
  });
}

// A barrier that no memory operation and no matrix instruction moves across; the waits in
// front of it are explicit.
__device__ __forceinline__ void phase_barrier() {
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
}

// The tile of a workgroup. Consecutive workgroups go to the chiplets in turn: each chiplet
// has a run of tiles, eight tiles of weights by all tiles of tokens after another, so that
// those it works on at a time share rows of both.
struct Tile {
  int n, t;
};
__device__ __forceinline__ Tile tile_of(int block, int total, int tiles_n) {
  const int xcd = block % kXcds;
  const int at = xcd * (total / kXcds) + min(xcd, total % kXcds) + block / kXcds;
  const int tiles_t = total / tiles_n, band = at / (8 * tiles_t), in_band = at - band * 8 * tiles_t;
  const int wide = min(8, tiles_n - 8 * band);
  return {8 * band + in_band % wide, in_band / wide};
}

// What follows a wave's sums, by way of its own part of LDS, half of its tokens at a time:
// the matrix instruction leaves four outputs of a token to a lane, stores of which would
// touch 32 bytes of each of 16 rows (8 slots of 8,192 tokens x 2,048 outputs: half of the
// kernel's time); from LDS every 16 lanes (8, 4) store a token's whole run of outputs.
// Rows of outputs are in pieces of four, piece c of token t at place c ^ t (mod 16) or c ^
// (t / 2) (mod 8), so that 16 tokens' pieces are spread over all banks. kDown: lane l has the
// slot and weight of the wave's token l.
template <int DT, int MODE, bool GATED, int WR, int WC, int AT, int BT>
__device__ __forceinline__ void finish_wave(const Args& a, const Part& p, int n0, int wr, int wc, char* lds,
                                            int32_t slot, float weight, const f32x4_t (&acc)[2][2][AT][BT]) {
  constexpr int kOut = GATED ? AT * 16 : AT * 32, kPieces = kOut / 4;  // of a wave
  constexpr int kTokens = BT * 16, kLanes = kOut / 8, kRows = 64 / kLanes;
  constexpr int kSteps = kTokens / kRows;
  const int lane = threadIdx.x & 63;
  f32x4_t* stage = reinterpret_cast<f32x4_t*>(lds) + (wc * WR + wr) * (kTokens * kPieces);
  const auto place = [&](int t, int c) {
    return t * kPieces + (kPieces >= 16 ? c ^ (t & 15) : c ^ ((t >> 1) & 7));
  };
  const int first_n = n0 + wr * kOut;
  static_for<0, 2>([&](auto hb) {
    const int t0 = (wc * 2 + hb.value) * kTokens, mine = lane / kLanes;
    int64_t row[kSteps];
    float scale[kSteps];
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      row[s] = p.first + t0 + s * kRows + mine, scale[s] = 1.f;
      if constexpr (MODE == kDown) {
        const int from = hb.value * kTokens + s * kRows + mine;
        row[s] = __shfl(slot, from, kWave), scale[s] = __shfl(weight, from, kWave);
      }
    }
#pragma unroll
    for (int j = 0; j < BT; ++j)
#pragma unroll
      for (int ha = 0; ha < 2; ++ha)
#pragma unroll
        for (int i = 0; i < AT; i += GATED ? 2 : 1) {
          const int n = (ha * AT + i) * (GATED ? 8 : 16) + 4 * (lane >> 4);  // of the wave's
          const f32x4_t& u = acc[ha][hb.value][GATED ? i + 1 : i][j];
          stage[place(j * 16 + (lane & 15), n / 4)] =
              activated4<DT, MODE, GATED>(a, first_n + n, acc[ha][hb.value][i][j], u);
        }
    wave_sync();
    const int c = 2 * (lane % kLanes);
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int t = s * kRows + mine;
      const f32x4_t lo = stage[place(t, c)], hi = stage[place(t, c + 1)];
      float y[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      if (t0 + t < p.rows) store8<DT, MODE>(a, first_n + 4 * c, row[s], scale[s], y);
    }
    wave_sync();
  });
}

// Place of a lane's four sums: part, tile, quarter, piece of it; whole waves store whole lines.
template <int WR, int WC, int AT, int BT>
__device__ __forceinline__ f32x4_t* part_at(const Args& a, int tiles, int split, int tile, int quarter) {
  constexpr int kThreads = 64 * WR * WC;
  return reinterpret_cast<f32x4_t*>(a.part) +
         ((static_cast<int64_t>(split) * tiles + tile) * 4 + quarter) * (AT * BT * kThreads) + threadIdx.x;
}

template <int DT, int MODE, bool GATED, int WR, int WC, int AT, int BT, int D>
__global__ __launch_bounds__(64 * WR * WC, 2) void tile_kernel(const Args a) {
  using S = TileShape<WR, WC, AT, BT, D>;
  constexpr int LA = S::kLoadA, LB = S::kLoadB;
  constexpr bool kPhased = S::kWaves == 8;
  static_assert(LA <= 2, "a wave's loads are of gate rows or of up rows");
  __shared__ __attribute__((aligned(1024))) char lds[S::kBytes];
  // Parts of k: all tiles of the first one, then of the next.
  const int total = a.tiles;
  const int split = group_index() / static_cast<uint32_t>(total);
  if (split >= a.splits) return;
  const int block = static_cast<int>(group_index()) - split * total;
  const Tile tile = tile_of(block, total, a.tiles_n);
  const int tn = tile.n, tt = tile.t;
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
      const int c = staged_input(lane, q);
      wo[h][u] = 2u * (static_cast<uint32_t>(min(n, a.n - 1 - first_n)) * static_cast<uint32_t>(a.w_st) + c);
    }
#pragma unroll
    for (int u = 0; u < LB; ++u) {
      const int q = wave * LB + u, r = 8 * q + (lane >> 3);
      const int row = min(r / (BT * 16) * (BT * 32) + h * (BT * 16) + r % (BT * 16), p.rows - 1);
      const int c = staged_input(lane, q);
      const uint32_t src = MODE == kGateUp ? a.order[p.first + row] / a.top_k : row;
      xo[h][u] = 2u * (src * static_cast<uint32_t>(a.x_st) + c);
    }
  }
  const auto wr_src = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(wbase), 0, kNowhere, 0x00027000);
  const auto xr_src = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(xbase), 0, kNowhere, 0x00027000);
  // Stage s is inputs 64 s .. + 63; where k is not a whole number of stages, the part of one
  // comes first (the order of the sum is free) and the others follow from input 0 on.
  const int k_tail = a.k % 64, all = a.k / 64 + (k_tail ? 1 : 0);
  const int begin = static_cast<int>(static_cast<int64_t>(all) * split / a.splits);
  const int stages = static_cast<int>(static_cast<int64_t>(all) * (split + 1) / a.splits) - begin;
  const int tail = begin == 0 ? k_tail : 0, shift = begin - (k_tail ? 1 : 0);
  auto fetch_a = [&](int s, auto h, int slot) {
    const int k_at = __builtin_amdgcn_readfirstlane((s + shift) * 128);
#pragma unroll
    for (int u = 0; u < LA; ++u)
      stage16<false>(wr_src,
                     lds + slot * S::kStage + (h.value ? S::kOffA1 : S::kOffA0) + (wave * LA + u) * 1024,
                     wo[h.value][u], k_at);
  };
  auto fetch_b = [&](int s, auto h, int slot) {
    const int k_at = __builtin_amdgcn_readfirstlane((s + shift) * 128);
#pragma unroll
    for (int u = 0; u < LB; ++u)
      stage16<false>(xr_src,
                     lds + slot * S::kStage + (h.value ? S::kOffB1 : S::kOffB0) + (wave * LB + u) * 1024,
                     xo[h.value][u], k_at);
  };
  const std::integral_constant<int, 0> i0;
  const std::integral_constant<int, 1> i1;
  int32_t slot_of = 0;
  if constexpr (MODE == kDown) slot_of = a.order[p.first + min(wc * BT * 32 + lane % (BT * 32), p.rows - 1)];
  if (tail) {
    const int k_at = a.k - tail;
    auto part = [&](const __amdgpu_buffer_rsrc_t& src, uint32_t off, int q, int place) {
      const int c = staged_input(lane, q);
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
  for (int d = 1; d < D; ++d)
    if (d < stages) fetch_a(d, i0, d), fetch_b(d, i0, d), fetch_b(d, i1, d), fetch_a(d, i1, d);
  if (kPhased) stages_wait<D, S::kLoads, LA + LB>(min(stages, D) - 1);
  else stages_wait<D, S::kLoads, 0>(min(stages, D) - 1);
  phase_barrier();
  if (kPhased && wave >= 4) phase_barrier();

  float weight_of = 0.f;  // on its way while the products are summed
  if constexpr (MODE == kDown) weight_of = a.scale[slot_of];
  const int r = lane & 15;
  const uint32_t base = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(
                            (__attribute__((address_space(3))) char*)lds)) +
                        r * 128 + (((lane >> 4) ^ (r >> 1)) & 7) * 16;
  const uint32_t base_a = base + wr * AT * 2048, base_b = base + wc * BT * 2048;
  f32x4_t acc[2][2][AT][BT] = {};
  const bool idle = wc * BT * 32 >= p.rows;  // no token of this wave's: it only loads and waits
  const std::true_type steady;
  const std::false_type ending;
  int slot = 0, s = 0;
  if constexpr (kPhased) {
    u32x4_t fa[2][AT], fb0[2][BT], fb1[2][BT];
    // steady: stage s + D exists, so that what is in flight is known.
    auto stage = [&](auto more) {
      const uint32_t at_a = base_a + slot * S::kStage, at_b = base_b + slot * S::kStage;
      const int left = min(stages - 1 - s, D - 1);  // stages on their way behind this one
      // Rows 0 x tokens 0.
      read_tiles<S::kOffB0>(at_b, fb0);
      read_tiles<S::kOffA0>(at_a, fa);
      if constexpr (more.value) vm_wait<(D - 1) * S::kLoads + LA>();  // tokens 1 of this stage
      else stages_wait<D, S::kLoads, LA>(left);
      wait_tiles(fb0), wait_tiles(fa);
      phase_barrier();
      if (!idle) multiply<DT>(fa, fb0, acc[0][0]);
      phase_barrier();
      // Rows 0 x tokens 1.
      read_tiles<S::kOffB1>(at_b, fb1);
      if constexpr (more.value) {
        fetch_a(s + D, i0, slot), fetch_b(s + D, i0, slot);
        vm_wait<(D - 1) * S::kLoads + LA + LB>();  // rows 1 of this stage
      } else {
        stages_wait<D, S::kLoads, 0>(left);
      }
      wait_tiles(fb1);
      phase_barrier();
      if (!idle) multiply<DT>(fa, fb1, acc[0][1]);
      phase_barrier();
      // Rows 1 x tokens 1.
      read_tiles<S::kOffA1>(at_a, fa);
      if constexpr (more.value) fetch_b(s + D, i1, slot);
      wait_tiles(fa);
      phase_barrier();
      if (!idle) multiply<DT>(fa, fb1, acc[1][1]);
      phase_barrier();
      // Rows 1 x tokens 0.
      if constexpr (more.value) {
        fetch_a(s + D, i1, slot);
        vm_wait<(D - 1) * S::kLoads + LA + LB>();  // rows 0 and tokens 0 of the next stage
      } else if (left > 0) {
        stages_wait<D, S::kLoads, LA + LB>(left - 1);
      }
      phase_barrier();
      if (!idle) multiply<DT>(fa, fb0, acc[1][0]);
      phase_barrier();
      slot = slot + 1 == D ? 0 : slot + 1;
      ++s;
    };
    while (s + D < stages) stage(steady);
    while (s < stages) stage(ending);
    if (wave < 4) phase_barrier();
  } else {
    Operands<AT, BT> f[2];
    f[0].template read<S, D>(base_a, base_b, 0, [](auto) {});
    f[0].wait();
    // One stage: the operands of the next one are read between its products.
    auto stage = [&](auto more, Operands<AT, BT>& now, Operands<AT, BT>& next) {
      if constexpr (more.value) vm_wait<(D - 2) * S::kLoads>();
      else if (s + 1 < stages) stages_wait<D - 1, S::kLoads, 0>(min(stages - 2 - s, D - 2));
      phase_barrier();  // the next stage is there, and every wave has this one in registers
      if (more.value || s + D < stages)
        fetch_a(s + D, i0, slot), fetch_b(s + D, i0, slot), fetch_b(s + D, i1, slot), fetch_a(s + D, i1, slot);
      slot = slot + 1 == D ? 0 : slot + 1;
      // Behind the last stage the reads find what was there and nobody takes it.
      next.template read<S, D>(base_a, base_b, slot, [&](auto i) { now.template multiply<DT>(i, acc); });
      next.wait();
      ++s;
    };
    while (s + D + 1 < stages) stage(steady, f[0], f[1]), stage(steady, f[1], f[0]);
    for (;;) {
      stage(ending, f[0], f[1]);
      if (s == stages) break;
      stage(ending, f[1], f[0]);
      if (s == stages) break;
    }
  }

  if (MODE == kLinear && a.splits > 1) {
    static_for<0, 4>([&](auto q) {
      constexpr int ha = q.value / 2, hb = q.value % 2;
      f32x4_t* out = part_at<WR, WC, AT, BT>(a, total, split, block, q.value);
#pragma unroll
      for (int i = 0; i < AT; ++i)
#pragma unroll
        for (int j = 0; j < BT; ++j) out[(i * BT + j) * 64 * S::kWaves] = acc[ha][hb][i][j];
    });
    return;
  }
  phase_barrier();  // every wave is done with the operands
  finish_wave<DT, MODE, GATED, WR, WC, AT, BT>(a, p, n0, wr, wc, lds, slot_of, weight_of, acc);
}

// The sum of a tile's parts, in their order, and what follows it: a workgroup for each piece
// of a quarter of the waves' sums, so that every part's loads are in flight at once.
constexpr int kMostSplits = 8;

template <int DT, bool GATED, int WR, int WC, int AT, int BT>
__global__ __launch_bounds__(64 * WR * WC) void fold_kernel(const Args a) {
  using S = TileShape<WR, WC, AT, BT, 2>;
  constexpr int kPair = GATED ? 2 : 1, kPieces = AT / kPair * BT;
  const int total = gridDim.x, block = blockIdx.x, quarter = blockIdx.y / kPieces, piece = blockIdx.y % kPieces;
  const int i = piece / BT * kPair, j = piece % BT;
  const Tile tile = tile_of(block, total, a.tiles_n);
  const Part p = part_of<kLinear>(a, tile.t, S::kN);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  f32x4_t v[kMostSplits][kPair];
#pragma unroll
  for (int split = 0; split < kMostSplits; ++split) {
    if (split >= a.splits) break;
    const f32x4_t* in = part_at<WR, WC, AT, BT>(a, total, split, block, quarter);
#pragma unroll
    for (int e = 0; e < kPair; ++e)
      v[split][e] = __builtin_nontemporal_load(&in[((i + e) * BT + j) * 64 * S::kWaves]);
  }
  f32x4_t g = {0.f, 0.f, 0.f, 0.f}, u = g;
#pragma unroll
  for (int split = 0; split < kMostSplits; ++split) {
    if (split >= a.splits) break;
    g += v[split][0];
    if constexpr (GATED) u += v[split][1];
  }
  const int wr = wave % WR, wc = wave / WR, ha = quarter / 2, hb = quarter % 2;
  const int t = ((wc * 2 + hb) * BT + j) * 16 + (lane & 15);
  if (t >= p.rows) return;
  const int n0 = tile.n * (S::kM / kPair) + ((wr * 2 + ha) * AT + i) * 16 / kPair + 4 * (lane >> 4);
  finish4<DT, kLinear, GATED>(a, n0, p.first + t, 1.f, g, u);
}

template <int DT, int MODE, bool GATED, int WR, int WC, int AT, int BT, int D>
int launch_tile(Args a, int64_t tiles_t, hipStream_t s) {
  using S = TileShape<WR, WC, AT, BT, D>;
  constexpr int out = GATED ? S::kM / 2 : S::kM;
  a.tiles_n = static_cast<int32_t>((static_cast<int64_t>(a.n) + out - 1) / out);
  const int64_t tiles = all_tiles(a.tiles_n, tiles_t);
  if (tiles < 0) return SGL_ERR_UNSUPPORTED;
  a.tiles = static_cast<int32_t>(tiles);
  if (a.splits < 1) a.splits = 1;
  hipLaunchKernelGGL((tile_kernel<DT, MODE, GATED, WR, WC, AT, BT, D>), rows_of(tiles * a.splits),
                     dim3(64 * S::kWaves), 0, s, a);
  if constexpr (MODE == kLinear) {
    if (a.splits > 1) {
      const int st = launch_status();
      if (st != SGL_OK) return st;
      hipLaunchKernelGGL((fold_kernel<DT, GATED, WR, WC, AT, BT>), dim3(a.tiles, 4 * BT * (GATED ? AT / 2 : AT)),
                         dim3(64 * S::kWaves), 0, s, a);
    }
  }
  return launch_status();
}

}  // namespace gemm
}  // namespace sgl
