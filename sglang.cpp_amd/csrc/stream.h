// Few tokens: every weight is read once, straight into the registers of the matrix
// instruction that takes it, and everything else is kept out of its way.
//
// A workgroup has MT tiles of weight rows, its waves share out the inputs (k) in steps and
// fold their sums through LDS at the end. One instruction multiplies 16 rows by 16
// columns over 32 inputs. Where there are at most 16 / P tokens (P = 2, 4), rows and
// columns stand for 16 / P rows and tokens times P parts of 32 P inputs instead: row and
// column blocks of the same part meet on the diagonal, whose P blocks are summed, and
// what is off it is dropped. A load then covers 64 P contiguous bytes of a row instead of
// 64 and a tile fewer rows, so that short launches spread over more workgroups; the
// wasted products cost nothing where the weights' bytes are what bounds the kernel.
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

// acc[i][j] += the products of the units first, first + stride ..: a unit is 32 P inputs, but
// 64 at least (128 bytes of a row, a whole cache line). Loads go round a ring of kRing
// instructions' operands, so that what is in flight never runs dry between batches.
template <int DT, int P, int MT, int NT>
__device__ __forceinline__ void stream_units(const Rows (&w)[MT], const Rows (&x)[NT], int k,
                                             int first, int stride, int turn,
                                             f32x4_t (&acc)[MT][NT]) {
  constexpr int kStep = 32 * P, kSub = P == 1 ? 2 : 1, kUnit = kStep * kSub;
  constexpr int kRing = (20 / (MT + NT)) / kSub < 1 ? kSub : (20 / (MT + NT)) / kSub * kSub;
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
  const int n = first < whole ? ((whole - first - 1) / stride + 1) * kSub : 0;  // its steps
  auto place = [&](int q) {
    int u = first + q / kSub * stride + turn;
    u = u < whole ? u : u - whole;
    return u * kUnit + (q % kSub) * kStep;
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
  if (whole * kUnit < k && whole % stride == first) {  // the last unit is a part of one
    const int m = threadIdx.x & 15, koff = ((m / (16 / P)) * 4 + ((threadIdx.x & 63) >> 4)) * 8;
#pragma unroll
    for (int d = 0; d < kSub; ++d) {
      const int at = whole * kUnit + d * kStep;
      if (at >= k) break;
      const bool in = at + koff < k;
#pragma unroll
      for (int i = 0; i < MT; ++i) fw[0][i] = stream_load<true>(w[i], at, in);
#pragma unroll
      for (int j = 0; j < NT; ++j) fx[0][j] = stream_load<false>(x[j], at, in);
      multiply(0);
    }
  }
}

// The waves' sums, each wave's own in LDS: the sum of unit (tile i, column tile j, quad q
// of rows, column c) over waves and parts.
template <int P, int MT, int NT, int NW>
__device__ __forceinline__ f32x4_t folded(const f32x4_t* red, int i, int j, int q, int c) {
  constexpr int R = 16 / P;
  f32x4_t sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int w = 0; w < NW; ++w)
#pragma unroll
    for (int p = 0; p < P; ++p)
      sum += red[((w * MT + i) * NT + j) * 64 + (p * (R / 4) + q) * 16 + p * R + c];
  return sum;
}

template <int DT, int MODE, bool GATED, int P, int MT, int NT, int NW>
__global__ __launch_bounds__(64 * NW, 4) void stream_kernel(const StreamArgs s) {
  static_assert((P == 1 || NT == 1) && (!GATED || MT % 2 == 0), "tiles");
  constexpr int R = 16 / P;                        // rows of a tile, columns of a column tile
  constexpr int kOut = (GATED ? MT / 2 : MT) * R;  // outputs of a workgroup
  __shared__ f32x4_t red[NW * MT * NT * 64];
  __shared__ int32_t list[MODE == kLinear ? 1 : kMostSlots];
  const Args& a = s.g;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n0 = static_cast<int>(blockIdx.x) * kOut;
  int expert = 0, count = a.tokens;
  if constexpr (MODE != kLinear) {
    count = find_slots(s, list, expert);
    if (count == 0) return;
  }
  const int m = lane & 15, koff = ((m / R) * 4 + (lane >> 4)) * 8;
  Rows w[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) w[i] = weight_rows<GATED, R>(a, expert, n0, i, m % R, koff);
  for (int first = 0; first < count; first += R * NT) {
    Rows x[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      // Columns past the last are computed from it and dropped.
      const int c = min(first + j * 16 + m % R, count - 1);
      uint32_t row = c;
      if constexpr (MODE == kGateUp) row = list[c] / a.top_k;
      if constexpr (MODE == kDown) row = list[c];
      x[j] = rows_at(a.x, row * static_cast<uint32_t>(a.x_st) + koff);
    }
    f32x4_t acc[MT][NT] = {};
    stream_units<DT, P, MT, NT>(w, x, a.k, wave, NW, 5 * blockIdx.x + 11 * expert, acc);
    if (MODE != kLinear && first > 0) __syncthreads();
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) red[((wave * MT + i) * NT + j) * 64 + lane] = acc[i][j];
    __syncthreads();
    constexpr int kUnits = kOut / 4 * R * NT;
    for (int unit = tid; unit < kUnits; unit += 64 * NW) {
      const int c = unit % R, q = unit / R % (R / 4), rest = unit / R / (R / 4);
      const int j = rest % NT, i = rest / NT;
      const int col = first + j * 16 + c;
      if (col >= count) continue;
      const int n = n0 + i * R + 4 * q;
      float scale = 1.f;
      int64_t row = col;
      if constexpr (MODE != kLinear) row = list[col];
      if constexpr (MODE == kDown) scale = a.scale[row];
      if constexpr (GATED)
        finish4<DT, MODE, true>(a, n, row, scale, folded<P, MT, NT, NW>(red, 2 * i, j, q, c),
                                folded<P, MT, NT, NW>(red, 2 * i + 1, j, q, c));
      else {
        const f32x4_t y = folded<P, MT, NT, NW>(red, i, j, q, c);
        finish4<DT, MODE, false>(a, n, row, scale, y, y);
      }
    }
  }
}

// The down projections of at most four tokens with their weighted sum: the waves share out
// (expert, part of its inputs), each adds its weighted sums, and the fold is the token's
// output. kOut = 4 MT outputs a workgroup.
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
  const int m = lane & 15, c = m % R, koff = ((m / R) * 4 + (lane >> 4)) * 8;
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
    for (int i = 0; i < MT; ++i) w[i] = weight_rows<false, R>(a, e, n0, i, c, koff);
    if (c < s.g.tokens)
      for (int j = 0; j < a.top_k; ++j)
        if (chosen[c * a.top_k + j] == e) {
          // The same rows of h, so the weights add.
          if (!mine) slot = c * a.top_k + j;
          mine = true;
          weight += weight_of[c * a.top_k + j];
        }
    const Rows x[1] = {rows_at(a.x, static_cast<uint32_t>(slot) * static_cast<uint32_t>(a.x_st) + koff)};
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
      const f32x4_t y = folded<P, MT, 1, NW>(red, i, 0, 0, col);
      finish4<DT, kLinear, false>(o, n0 + i * R, col, 1.f, y, y);
    }
  }
}

template <int DT, int MODE, bool GATED, int P, int MT, int NT, int NW>
void launch_stream_as(const StreamArgs& s, int rows, hipStream_t st) {
  constexpr int kOut = (GATED ? MT / 2 : MT) * 16 / P;
  const dim3 grid((s.g.n + kOut - 1) / kOut, rows);
  hipLaunchKernelGGL((stream_kernel<DT, MODE, GATED, P, MT, NT, NW>), grid, dim3(64 * NW), 0, st, s);
}

// MT tiles a workgroup where that leaves a workgroup for every CU, a half otherwise; as many
// waves as fill the CUs with 16 each.
template <int DT, int MODE, bool GATED, int P, int MT, int NT>
void launch_stream_at(const StreamArgs& s, int rows, hipStream_t st) {
  constexpr int kOut = (GATED ? MT / 2 : MT) * 16 / P;
  constexpr int kLess = GATED && MT == 2 ? 2 : MT > 1 ? MT / 2 : 1;
  const int64_t groups = static_cast<int64_t>((s.g.n + kOut - 1) / kOut) * rows;
  if (groups >= 1024) launch_stream_as<DT, MODE, GATED, P, MT, NT, 4>(s, rows, st);
  else if (groups >= 256) launch_stream_as<DT, MODE, GATED, P, MT, NT, 8>(s, rows, st);
  else launch_stream_as<DT, MODE, GATED, P, kLess, NT, 8>(s, rows, st);
}

// columns: tokens of the call, or the most places an expert is expected to have. rows:
// the grid's second extent.
template <int DT, int MODE, bool GATED>
int launch_stream(const StreamArgs& s, int columns, int rows, hipStream_t st) {
  constexpr int kWide = GATED ? 2 : 1;
  if (columns <= 4) launch_stream_at<DT, MODE, GATED, 4, 4, 1>(s, rows, st);
  else if (columns <= 8) launch_stream_at<DT, MODE, GATED, 2, 4, 1>(s, rows, st);
  else if (columns <= 16) launch_stream_at<DT, MODE, GATED, 1, 4, 1>(s, rows, st);
  else if (columns <= 32) launch_stream_at<DT, MODE, GATED, 1, 2, 2>(s, rows, st);
  else if (columns <= 48) launch_stream_at<DT, MODE, GATED, 1, 2, 3>(s, rows, st);
  else launch_stream_at<DT, MODE, GATED, 1, 2, 4>(s, rows, st);
  return launch_status();
}

}  // namespace gemm
}  // namespace sgl
