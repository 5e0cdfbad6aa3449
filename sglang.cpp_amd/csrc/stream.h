// Few tokens: every weight is read once and everything else is kept out of its way.
//
// A workgroup has MT tiles of 16 weight rows, its waves share out the inputs (k) in units of
// 64 (128 bytes of a row, a cache line) and fold their sums through LDS at the end. One
// instruction multiplies 16 rows by 16 columns (tokens) over 32 inputs. Its operands have
// neighbouring lanes in different rows: loaded straight into registers, every lane's 16
// bytes are an access of their own (24 tokens through 84 experts of 2 x 768 x 2,048: 129 us
// where this takes 85). So each wave brings whole pieces of rows into a ring of its own in
// LDS, which holds no registers and needs no barrier, and reads the operands from there.
#pragma once

#include "gemm.h"

namespace sgl {
namespace gemm {

// Slots of one expert, found by every workgroup of a launch for itself: a few hundred
// choices are read faster than another launch would sort them.
constexpr int kMostSlots = 1024;
// Strides whose 16 weight rows, 64 rows of x or 1,024 rows of h stay below 2^31 bytes.
constexpr int64_t kMostStride = 1 << 20;

struct StreamArgs {
  Args g;
  const int32_t* experts;  // choices [slots] (experts only)
  int32_t slots, num_experts, by_slot;  // by_slot: grid.y is a slot, not an expert
};

// The workgroup's expert and the slots that chose it, 0 where another workgroup has them or
// there are none. Every wave looks for itself and writes the same list, so none waits.
__device__ __forceinline__ int find_slots(const StreamArgs& s, int32_t* list, int& expert) {
  const int lane = threadIdx.x & 63;
  constexpr int kAhead = 4;  // loads in flight: 256 choices
  int32_t e[kAhead];
  auto load = [&](int i0) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int i = i0 + 64 * u + lane;
      e[u] = i < s.slots ? s.experts[i] : -1;
    }
  };
  load(0);
  expert = s.by_slot ? s.experts[blockIdx.y] : static_cast<int>(blockIdx.y);
  expert = __builtin_amdgcn_readfirstlane(expert);
  if (expert < 0 || expert >= s.num_experts) return 0;
  int count = 0;
  for (int i0 = 0;;) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const uint64_t hits = __ballot(e[u] == expert);
      if (hits == 0) continue;
      const int at = i0 + 64 * u;
      if (count == 0 && s.by_slot && at + __builtin_ctzll(hits) < static_cast<int>(blockIdx.y)) return 0;
      if (e[u] == expert) list[count + __popcll(hits & ((1ull << lane) - 1))] = at + lane;
      count += __popcll(hits);
    }
    i0 += 64 * kAhead;
    if (i0 >= s.slots) break;
    load(i0);
  }
  return count;
}

// Where a wave reads: a uniform row (a buffer resource in scalar registers) and each lane's
// bytes from it, so that a load takes a lane offset and a scalar one and no address
// arithmetic. Offsets below 2^31 are in range, kNowhere is not and loads zero.
struct Rows {
  __amdgpu_buffer_rsrc_t base;
  uint32_t lane;
};
constexpr uint32_t kNowhere = 0x80000000u;

__device__ __forceinline__ Rows rows_at(const uint16_t* base, uint32_t elements) {
  return {__builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(base), 0, kNowhere, 0x00027000),
          2u * elements};
}
template <bool NT>
__device__ __forceinline__ u32x4_t stream_load(const Rows& r, int at, bool in = true) {
  return __builtin_amdgcn_raw_buffer_load_b128(r.base, in ? r.lane : kNowhere, 2 * at, NT ? 2 : 0);
}

// Rows of tile i (the gate rows of its outputs, then their up rows), lane's row r; rows past
// the last output are computed from it and dropped.
template <bool GATED, int R>
__device__ __forceinline__ Rows weight_rows(const Args& a, int expert, int n0, int i, int r, int koff) {
  const int n = min(n0 + (GATED ? i / 2 : i) * R, a.n - 1);
  const int64_t row = (GATED && (i & 1) ? static_cast<int64_t>(a.n) : 0) + n;
  return rows_at(a.w + expert * a.w_se + row * a.w_st,
                 static_cast<uint32_t>(min(r, a.n - 1 - n)) * static_cast<uint32_t>(a.w_st) + koff);
}

// First input of a lane's 16 bytes in a unit of 32 P.
template <int P>
__device__ __forceinline__ int lane_input(int lane) {
  return ((lane >> 4) * P + (lane & 15) % P) * 8;
}

// The inputs from `at` on, fewer than a unit; what is behind the last one is zero.
template <int DT, int P, int MT, int NT>
__device__ __forceinline__ void stream_tail(const Rows (&w)[MT], const Rows (&x)[NT], int k, int at,
                                            f32x4_t (&acc)[MT][NT]) {
  for (; at < k; at += 32 * P) {
    const bool in = at + lane_input<P>(threadIdx.x & 63) < k;
    u32x4_t fw[MT], fx[NT];
#pragma unroll
    for (int i = 0; i < MT; ++i) fw[i] = stream_load<true>(w[i], at, in);
#pragma unroll
    for (int j = 0; j < NT; ++j) fx[j] = stream_load<false>(x[j], at, in);
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) acc[i][j] = mfma16<DT>(fw[i], fx[j], acc[i][j]);
  }
}

// acc[i][j] += the products of the units first, first + stride .. of 32 P inputs. Loads go
// round a ring of kRing instructions' operands, so that what is in flight never runs dry
// between batches. turn: the first unit of a workgroup.
template <int DT, int P, int MT, int NT>
__device__ __forceinline__ void stream_units(const Rows (&w)[MT], const Rows (&x)[NT], int k,
                                             int first, int stride, int turn,
                                             f32x4_t (&acc)[MT][NT]) {
  constexpr int kUnit = 32 * P;
  constexpr int kRing = 20 / (MT + NT);
  const int whole = k / kUnit;  // units without a tail
  u32x4_t fw[kRing][MT], fx[kRing][NT];
  auto load = [&](int d, int at) {
#pragma unroll
    for (int i = 0; i < MT; ++i) fw[d][i] = stream_load<true>(w[i], at);
#pragma unroll
    for (int j = 0; j < NT; ++j) fx[d][j] = stream_load<false>(x[j], at);
  };
  auto multiply = [&](int d) {
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) acc[i][j] = mfma16<DT>(fw[d][i], fx[d][j], acc[i][j]);
  };
  turn = whole > 0 ? turn % whole : 0;
  const int n = first < whole ? (whole - first - 1) / stride + 1 : 0;  // its units
  auto place = [&](int q) {
    const int u = first + q * stride + turn;
    return (u < whole ? u : u - whole) * kUnit;
  };
#pragma unroll
  for (int d = 0; d < kRing; ++d)
    if (d < n) load(d, place(d));
  int q = 0;
  for (; q + 2 * kRing <= n; q += kRing) {
#pragma unroll
    for (int d = 0; d < kRing; ++d) {
      multiply(d);
      __builtin_amdgcn_sched_barrier(0);  // a load goes where its operand just was
      load(d, place(q + kRing + d));
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  for (; q < n; q += kRing) {
#pragma unroll
    for (int d = 0; d < kRing; ++d) {
      if (q + d < n) multiply(d);
      __builtin_amdgcn_sched_barrier(0);
      if (q + d + kRing < n) load(d, place(q + kRing + d));
    }
  }
  if (whole * kUnit < k && whole % stride == first)  // the last unit is a part of one
    stream_tail<DT, P, MT, NT>(w, x, k, whole * kUnit, acc);
}

// The ring's tiles: 16 rows x 64 inputs, row r's 16-byte piece c at place c ^ ((r >> 1) &
// 7) of its 128 bytes, so that the 16 rows' reads of one piece are spread over all banks.
constexpr int kPiece = 64;           // inputs of a unit
constexpr int kTileBytes = 2048;     // 16 rows of one

// Lane offsets of a tile's two loads of 8 rows: lane i has row 8 h + i / 8 and the piece that
// belongs at place i % 8.
struct Staged {
  __amdgpu_buffer_rsrc_t base;
  uint32_t lane[2];
};
__device__ __forceinline__ int staged_input(int lane, int h) {
  return ((lane & 7) ^ ((4 * h + (lane >> 4)) & 7)) * 8;
}

// 16 bytes a lane into LDS, lane i's at `place` + 16 i; NT: read once. (Only the device pass
// knows loads of 16 bytes.)
template <bool NT>
__device__ __forceinline__ void stage16(const __amdgpu_buffer_rsrc_t& base, char* place, uint32_t lane,
                                        int at) {
#ifdef __HIP_DEVICE_COMPILE__
  __builtin_amdgcn_raw_ptr_buffer_load_lds(base, (__attribute__((address_space(3))) void*)place, 16, lane,
                                           at, 0, NT ? 2 : 0);
#endif
}

template <int N>
__device__ __forceinline__ void vm_wait() {
  asm volatile("s_waitcnt vmcnt(%0)" : : "i"(N) : "memory");
}

template <int OFF>
__device__ __forceinline__ u32x4_t lds_read(uint32_t addr) {
  u32x4_t v;
  asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(v) : "v"(addr), "i"(OFF));
  return v;
}

// The operands have arrived (the reads are in order: the first wait is the only one).
__device__ __forceinline__ void lds_wait(u32x4_t& a, u32x4_t& b) {
  asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(a), "+v"(b) : : "memory");
}

__device__ __forceinline__ void lds_wait(u32x4_t& a) {
  asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(a) : : "memory");
}

// Waits until at most `left` units of kEach loads are in flight, left < kMost.
template <int kMost, int kEach>
__device__ __forceinline__ void units_wait(int left) {
  static_for<0, kMost>([&](auto i) {
    if (left == i.value) vm_wait<i.value * kEach>();
  });
}

template <int DT, int MT, int NT, int D>
__device__ __forceinline__ void staged_units(const Staged (&t)[MT + NT], char* ring, int k, int first,
                                             int stride, int turn, f32x4_t (&acc)[MT][NT]) {
  constexpr int kTiles = MT + NT, kSlot = kTiles * kTileBytes, kLoads = 2 * kTiles;
  const int whole = k / kPiece;
  turn = whole > 0 ? turn % whole : 0;
  const int n = first < whole ? (whole - first - 1) / stride + 1 : 0;
  const int lane = threadIdx.x & 63;
  auto fetch = [&](int q, int slot) {
    const int u = first + q * stride + turn;
    const int at = (u < whole ? u : u - whole) * kPiece * 2;
    static_for<0, kTiles>([&](auto i) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        stage16<(i.value < MT)>(t[i.value].base, ring + slot * kSlot + i.value * kTileBytes + h * 1024,
                                t[i.value].lane[h], at);
    });
  };
  // Place of this lane's operand: row l % 16, piece l / 16 (and 4 further for the second half).
  const int r = lane & 15;
  const uint32_t at0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(
                           (__attribute__((address_space(3))) char*)ring)) +
                       r * 128 + (((lane >> 4) ^ (r >> 1)) & 7) * 16;
  for (int d = 0; d < D; ++d)
    if (d < n) fetch(d, d);
  int slot = 0;
  for (int q = 0; q < n; ++q) {
    units_wait<D, kLoads>(min(n - 1 - q, D - 1));
    u32x4_t f[2][kTiles];
    const uint32_t at = at0 + slot * kSlot, at1 = at ^ 64;
    static_for<0, kTiles>([&](auto i) {
      f[0][i.value] = lds_read<i.value * kTileBytes>(at);
      f[1][i.value] = lds_read<i.value * kTileBytes>(at1);
    });
    static_for<0, kTiles>([&](auto i) { lds_wait(f[0][i.value], f[1][i.value]); });
    if (q + D < n) fetch(q + D, slot);
    slot = slot + 1 == D ? 0 : slot + 1;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = mfma16<DT>(f[h][i], f[h][MT + j], acc[i][j]);
  }
}

// Units of a ring: 16 to 20 KB a wave, 8 waves a CU.
constexpr int stream_depth(int mt, int nt) { return mt + nt <= 2 ? 4 : mt + nt <= 3 ? 3 : 2; }

// The waves' sums, each wave's own in LDS: outputs 4 q .. + 3 of (tile i, column tile j),
// column c.
template <int MT, int NT, int NW>
__device__ __forceinline__ f32x4_t folded(const f32x4_t* red, int i, int j, int q, int c) {
  f32x4_t sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int w = 0; w < NW; ++w) sum += red[((w * MT + i) * NT + j) * 64 + q * 16 + c];
  return sum;
}

template <int DT, int MODE, bool GATED, int MT, int NT, int NW>
__global__ __launch_bounds__(64 * NW, 2) void stream_kernel(const StreamArgs s) {
  static_assert(!GATED || MT % 2 == 0, "gate and up rows");
  constexpr int kDepth = stream_depth(MT, NT);
  constexpr int kOut = (GATED ? MT / 2 : MT) * 16;  // outputs of a workgroup
  // The rings and, behind the last unit, the waves' sums.
  __shared__ f32x4_t red[NW * kDepth * (MT + NT) * kTileBytes / 16];
  __shared__ int32_t list[MODE == kLinear ? 1 : kMostSlots];
  const Args& a = s.g;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // kLinear: rows of workgroups; experts have one of the grid's rows each.
  const uint32_t group = MODE == kLinear ? group_index() : blockIdx.x;
  if (group * kOut >= static_cast<uint32_t>(a.n)) return;
  const int n0 = static_cast<int>(group) * kOut;
  int expert = 0, count = a.tokens;
  if constexpr (MODE != kLinear) {
    count = find_slots(s, list, expert);
    if (count == 0) return;
  }
  // Row of x of column c; columns past the last are computed from it and dropped.
  auto source = [&](int c) -> uint32_t {
    c = min(c, count - 1);
    return MODE == kGateUp ? list[c] / a.top_k : MODE == kDown ? list[c] : c;
  };
  const uint32_t x_st = static_cast<uint32_t>(a.x_st);
  const int whole = a.k / kPiece;
  for (int first = 0; first < count; first += 16 * NT) {
    Staged t[MT + NT];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = 8 * h + (lane >> 3), at = staged_input(lane, h);
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const Rows row = weight_rows<GATED, 16>(a, expert, n0, i, r, at);
        t[i].base = row.base, t[i].lane[h] = row.lane;
      }
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const Rows row = rows_at(a.x, source(first + j * 16 + r) * x_st + at);
        t[MT + j].base = row.base, t[MT + j].lane[h] = row.lane;
      }
    }
    if (MODE != kLinear && first > 0) __syncthreads();  // the sums in the rings were read
    char* ring = reinterpret_cast<char*>(red) + wave * (kDepth * (MT + NT) * kTileBytes);
    f32x4_t acc[MT][NT] = {};
    staged_units<DT, MT, NT, kDepth>(t, ring, a.k, wave, NW, 5 * blockIdx.x + 11 * expert, acc);
    if (whole * kPiece < a.k && whole % NW == wave) {  // the last unit is a part of one
      const int r = lane & 15, in = lane_input<1>(lane);
      Rows w[MT], x[NT];
#pragma unroll
      for (int i = 0; i < MT; ++i) w[i] = weight_rows<GATED, 16>(a, expert, n0, i, r, in);
#pragma unroll
      for (int j = 0; j < NT; ++j) x[j] = rows_at(a.x, source(first + j * 16 + r) * x_st + in);
      stream_tail<DT, 1, MT, NT>(w, x, a.k, whole * kPiece, acc);
    }
    __syncthreads();  // every wave is done with its ring
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) red[((wave * MT + i) * NT + j) * 64 + lane] = acc[i][j];
    __syncthreads();
    constexpr int kUnits = kOut * 4 * NT;
    for (int unit = tid; unit < kUnits; unit += 64 * NW) {
      const int c = unit % 16, q = unit / 16 % 4, j = unit / 64 % NT, i = unit / 64 / NT;
      const int col = first + j * 16 + c;
      if (col >= count) continue;
      const int n = n0 + i * 16 + 4 * q;
      float scale = 1.f;
      int64_t row = col;
      if constexpr (MODE != kLinear) row = list[col];
      if constexpr (MODE == kDown) scale = a.scale[row];
      if constexpr (GATED) {
        finish4<DT, MODE, true>(a, n, row, scale, folded<MT, NT, NW>(red, 2 * i, j, q, c),
                                folded<MT, NT, NW>(red, 2 * i + 1, j, q, c));
      } else {
        const f32x4_t y = folded<MT, NT, NW>(red, i, j, q, c);
        finish4<DT, MODE, false>(a, n, row, scale, y, y);
      }
    }
  }
}

// The down projections of at most four tokens with their weighted sum: the waves share out
// (expert, part of its inputs), each adds its weighted sums, and the fold is the token's
// output, 4 MT of them a workgroup.
//
// The instruction's rows and columns stand for 4 rows and tokens times 4 parts of 128 inputs:
// row and column blocks of the same part meet on the diagonal, whose blocks are summed, and
// what is off it is dropped. Neighbouring lanes then hold neighbouring inputs of a row, so
// operands come straight into registers, and a workgroup has few outputs, so that all CUs
// have one (hidden 2,048: 256 workgroups of 8).
constexpr int kFewTokens = 4;
constexpr int kFewSlots = 128;

template <int DT, int MT, int NW>
__global__ __launch_bounds__(64 * NW) void down_few_kernel(const StreamArgs s, const uint16_t* res,
                                                           int64_t r_st) {
  constexpr int P = 4, R = 4, NT = 1;
  __shared__ f32x4_t red[NW * MT * 64];
  __shared__ int32_t chosen[kFewSlots];
  __shared__ float weight_of[kFewSlots];
  __shared__ int32_t first_of[kFewSlots];  // first slot of each chosen expert, in order
  __shared__ int32_t num;
  const Args& a = s.g;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n0 = static_cast<int>(blockIdx.x) * MT * R;
  if (tid < s.slots) {
    chosen[tid] = s.experts[tid];
    weight_of[tid] = a.scale[tid];
  }
  __syncthreads();
  if (wave == 0) {
    int count = 0;
    for (int i0 = 0; i0 < s.slots; i0 += 64) {
      const int i = i0 + lane;
      const int e = i < s.slots ? chosen[i] : -1;
      bool fresh = e >= 0 && e < s.num_experts;
      for (int o = 0; o < min(i0 + 64, s.slots); ++o) fresh = fresh && !(o < i && chosen[o] == e);
      const uint64_t hits = __ballot(fresh);
      if (fresh) first_of[count + __popcll(hits & ((1ull << lane) - 1))] = i;
      count += __popcll(hits);
    }
    if (lane == 0) num = count;
  }
  __syncthreads();
  const int experts = num;
  const int c = (lane & 15) / P, in = lane_input<P>(lane);
  // Fewer experts than waves: each is shared by as many waves as there are for it.
  const int parts = experts > 0 ? max(1, NW / experts) : 1;
  f32x4_t total[MT] = {};
  for (int unit = wave; unit < experts * parts; unit += NW) {
    const int slot0 = first_of[unit / parts];
    const int e = __builtin_amdgcn_readfirstlane(chosen[slot0]);
    // Slots of this lane's token that chose e: usually one or none.
    bool mine = false;
    int slot = slot0;
    float weight = 0.f;
    Rows w[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) w[i] = weight_rows<false, R>(a, e, n0, i, c, in);
    if (c < s.g.tokens)
      for (int j = 0; j < a.top_k; ++j)
        if (chosen[c * a.top_k + j] == e) {
          // The same rows of h, so the weights add.
          if (!mine) slot = c * a.top_k + j;
          mine = true;
          weight += weight_of[c * a.top_k + j];
        }
    const Rows x[1] = {rows_at(a.x, static_cast<uint32_t>(slot) * static_cast<uint32_t>(a.x_st) + in)};
    f32x4_t acc[MT][1] = {};
    stream_units<DT, P, MT, NT>(w, x, a.k, unit % parts, parts, 5 * blockIdx.x + 11 * e, acc);
    // A token that did not choose e has another token's products: dropped, not weighted.
#pragma unroll
    for (int i = 0; i < MT; ++i)
      if (mine) total[i] += acc[i][0] * weight;
  }
#pragma unroll
  for (int i = 0; i < MT; ++i) red[(wave * MT + i) * 64 + lane] = total[i];
  __syncthreads();
  if (tid < MT * R) {
    const int col = tid % R, i = tid / R;
    if (col < s.g.tokens) {
      Args o = a;
      o.res = res, o.r_st = r_st, o.act = SGL_ACT_NONE;
      // Row r and column c of part p are the instruction's row 4 r + p and column 4 c + p.
      f32x4_t y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 2
      for (int w = 0; w < NW; ++w)
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int p = 0; p < P; ++p)
            y[r] += reinterpret_cast<const float*>(&red[(w * MT + i) * 64 + r * 16 + col * P + p])[p];
      finish4<DT, kLinear, false>(o, n0 + i * R, col, 1.f, y, y);
    }
  }
}

template <int DT, int MODE, bool GATED, int MT, int NT, int NW>
void launch_stream_as(const StreamArgs& s, int rows, hipStream_t st) {
  constexpr int kOut = (GATED ? MT / 2 : MT) * 16;
  const int64_t groups = (static_cast<int64_t>(s.g.n) + kOut - 1) / kOut;
  const dim3 grid = MODE == kLinear ? rows_of(groups) : dim3(static_cast<uint32_t>(groups), rows);
  hipLaunchKernelGGL((stream_kernel<DT, MODE, GATED, MT, NT, NW>), grid, dim3(64 * NW), 0, st, s);
}

// Weight tiles of a workgroup: one where that leaves every CU at most one workgroup (4,096
// outputs of one token 7.6 us, with two tiles 8.9; 6,144: 12.3 and 10.3), two otherwise.
inline int stream_tiles(bool gated, int64_t n, int rows) {
  return gated || (n + 15) / 16 * rows > kCus ? 2 : 1;
}

// Tokens of a call that these kernels take at most: the rings of a workgroup's waves fill
// the LDS.
inline int stream_tokens(bool gated, int64_t n) { return stream_tiles(gated, n, 1) == 2 ? 48 : 64; }

// A projection of up to stream_tokens: eight waves a workgroup, four where CUs have two
// workgroups (24,576 rows: 33.5 us, 36.1 with eight).
template <int DT, bool GATED, int NT>
void launch_stream_at(const StreamArgs& s, hipStream_t st) {
  constexpr int kTwo = GATED ? 16 : 32;
  if constexpr (!GATED) {
    if (stream_tiles(false, s.g.n, 1) == 1) return launch_stream_as<DT, kLinear, GATED, 1, NT, 8>(s, 1, st);
  }
  if constexpr (NT <= 2) {
    if ((s.g.n + kTwo - 1) / kTwo <= kCus) return launch_stream_as<DT, kLinear, GATED, 2, NT, 8>(s, 1, st);
  }
  if constexpr (NT <= 3) launch_stream_as<DT, kLinear, GATED, 2, NT, 4>(s, 1, st);
}
template <int DT, bool GATED>
int launch_stream(const StreamArgs& s, hipStream_t st) {
  if (s.g.tokens <= 16) launch_stream_at<DT, GATED, 1>(s, st);
  else if (s.g.tokens <= 32) launch_stream_at<DT, GATED, 2>(s, st);
  else if (s.g.tokens <= 48) launch_stream_at<DT, GATED, 3>(s, st);
  else if constexpr (!GATED) launch_stream_at<DT, GATED, 4>(s, st);
  return launch_status();
}

// A projection of the experts, `rows` of them or slots: workgroups of two waves, several of
// which a CU holds while others look for their slots (64 tokens x 8 of 128 experts of 2,048 x
// 768: 68 us, 82 with four waves).
template <int DT, int MODE, bool GATED>
int launch_experts(const StreamArgs& s, int rows, hipStream_t st) {
  launch_stream_as<DT, MODE, GATED, 2, 1, 2>(s, rows, st);
  return launch_status();
}

}  // namespace gemm
}  // namespace sgl
