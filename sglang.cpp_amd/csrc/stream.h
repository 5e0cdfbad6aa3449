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

struct StreamArgs {
  Args g;
  const int32_t* experts;  // choices [slots] (experts only)
  int32_t slots, num_experts, by_slot;  // by_slot: grid.y is a slot, not an expert
};

// The workgroup's expert and the slots that chose it, -1 where another workgroup has
// them or there are none.
template <int NW>
__device__ __forceinline__ int find_slots(const StreamArgs& s, int32_t* list, int32_t* shared,
                                          int& expert) {
  const int tid = threadIdx.x, lane = tid & 63;
  if (tid < 2) shared[tid] = 0;
  expert = s.by_slot ? s.experts[blockIdx.y] : static_cast<int>(blockIdx.y);
  __syncthreads();
  if (expert < 0 || expert >= s.num_experts) return -1;
  for (int i0 = 0; i0 < s.slots; i0 += 64 * NW) {
    const int i = i0 + tid;
    const bool hit = i < s.slots && s.experts[i] == expert;
    const uint64_t hits = __ballot(hit);
    if (hits) {
      int at = 0;
      if (lane == 0) at = atomicAdd(&shared[0], __popcll(hits));
      at = __builtin_amdgcn_readfirstlane(at) + __popcll(hits & ((1ull << lane) - 1));
      if (hit) list[at] = i;
      if (s.by_slot && hit && i < static_cast<int>(blockIdx.y)) shared[1] = 1;
    }
  }
  __syncthreads();
  return shared[1] ? -1 : shared[0];
}

// Weight row of row r of tile i (the gate rows of its outputs, then their up rows).
template <bool GATED, int R>
__device__ __forceinline__ int64_t stream_row(const Args& a, int n0, int i, int r) {
  const int n = n0 + (GATED ? i / 2 : i) * R + r;
  const int64_t row = n < a.n ? n : a.n - 1;  // rows past the end are computed and dropped
  return GATED && (i & 1) ? a.n + row : row;
}

// acc[i][j] += the products of the steps first, first + stride .. below `steps`.
template <int DT, int P, int MT, int NT>
__device__ __forceinline__ void stream_steps(const uint16_t* const (&w)[MT],
                                             const uint16_t* const (&x)[NT], int k, int first,
                                             int stride, int steps, f32x4_t (&acc)[MT][NT]) {
  constexpr int kWidth = 32 * P;
  constexpr int kBatch = 20 / (MT + NT) < 1 ? 1 : 20 / (MT + NT);  // loads in flight: 20 at most
  const int whole = k / kWidth;  // steps without a tail
  int s = first;
  for (; s + (kBatch - 1) * stride < whole; s += kBatch * stride) {
    u32x4_t fw[kBatch][MT], fx[kBatch][NT];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int64_t at = static_cast<int64_t>(s + u * stride) * kWidth;
#pragma unroll
      for (int i = 0; i < MT; ++i) fw[u][i] = ldg128_nt<true>(w[i] + at);
#pragma unroll
      for (int j = 0; j < NT; ++j) fx[u][j] = ldg128(x[j] + at);
    }
#pragma unroll
    for (int u = 0; u < kBatch; ++u)
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = mfma16<DT>(fw[u][i], fx[u][j], acc[i][j]);
  }
  if (s >= steps) return;
  u32x4_t fw[kBatch][MT], fx[kBatch][NT];
  const u32x4_t zero = {0, 0, 0, 0};
  const int m = threadIdx.x & 15, koff = ((m / (16 / P)) * 4 + ((threadIdx.x & 63) >> 4)) * 8;
#pragma unroll
  for (int u = 0; u < kBatch; ++u) {
    const int64_t at = static_cast<int64_t>(s + u * stride) * kWidth;
    const bool in = at + koff < k;
#pragma unroll
    for (int i = 0; i < MT; ++i) fw[u][i] = in ? ldg128_nt<true>(w[i] + at) : zero;
#pragma unroll
    for (int j = 0; j < NT; ++j) fx[u][j] = in ? ldg128(x[j] + at) : zero;
  }
#pragma unroll
  for (int u = 0; u < kBatch; ++u) {
    if (s + u * stride >= steps) break;
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) acc[i][j] = mfma16<DT>(fw[u][i], fx[u][j], acc[i][j]);
  }
}

// The waves' sums, each wave's own in LDS: the sum of unit (tile i, column tile j, quad q
// of rows, column c) over waves and parts.
template <int P, int MT, int NT, int NW>
__device__ __forceinline__ f32x4_t folded(const f32x4_t* red, int i, int j, int q, int c) {
  constexpr int R = 16 / P;
  f32x4_t sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
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
  __shared__ int32_t shared[2];
  const Args& a = s.g;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n0 = static_cast<int>(blockIdx.x) * kOut;
  int expert = 0, count = a.tokens;
  if constexpr (MODE != kLinear) {
    count = find_slots<NW>(s, list, shared, expert);
    if (count <= 0) return;
  }
  const int m = lane & 15, koff = ((m / R) * 4 + (lane >> 4)) * 8;
  const uint16_t* w[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
    w[i] = a.w + expert * a.w_se + stream_row<GATED, R>(a, n0, i, m % R) * a.w_st + koff;
  const int steps = (a.k + 32 * P - 1) / (32 * P);
  for (int first = 0; first < count; first += R * NT) {
    const uint16_t* x[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      // Columns past the last are computed from it and dropped.
      const int c = min(first + j * 16 + m % R, count - 1);
      int64_t row = c;
      if constexpr (MODE == kGateUp) row = list[c] / a.top_k;
      if constexpr (MODE == kDown) row = list[c];
      x[j] = a.x + row * a.x_st + koff;
    }
    f32x4_t acc[MT][NT] = {};
    stream_steps<DT, P, MT, NT>(w, x, a.k, wave, NW, steps, acc);
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
  const int steps = (a.k + 32 * P - 1) / (32 * P);
  // Fewer experts than waves: each is shared by as many waves as there are for it.
  const int parts = experts > 0 ? max(1, NW / experts) : 1;
  f32x4_t total[MT] = {};
  for (int unit = wave; unit < experts * parts; unit += NW) {
    const int slot0 = first_of[unit / parts];
    const int e = chosen[slot0];
    // Slots of this lane's token that chose e: usually one or none.
    bool mine = false;
    int slot = slot0;
    float weight = 0.f;
    const uint16_t* w[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
      w[i] = a.w + e * a.w_se + stream_row<false, R>(a, n0, i, c) * a.w_st + koff;
    if (c < s.g.tokens)
      for (int j = 0; j < a.top_k; ++j)
        if (chosen[c * a.top_k + j] == e) {
          // The same rows of h, so the weights add.
          if (!mine) slot = c * a.top_k + j;
          mine = true;
          weight += weight_of[c * a.top_k + j];
        }
    const uint16_t* x[1] = {a.x + static_cast<int64_t>(slot) * a.x_st + koff};
    f32x4_t acc[MT][1] = {};
    stream_steps<DT, P, MT, NT>(w, x, a.k, unit % parts, parts, steps, acc);
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

template <int DT, int MODE, bool GATED, int P, int MT, int NT>
void launch_stream_as(const StreamArgs& s, int rows, hipStream_t st) {
  constexpr int kOut = (GATED ? MT / 2 : MT) * 16 / P;
  const dim3 grid((s.g.n + kOut - 1) / kOut, rows);
  hipLaunchKernelGGL((stream_kernel<DT, MODE, GATED, P, MT, NT, 8>), grid, dim3(512), 0, st, s);
}

// columns: tokens of the call, or the most places an expert is expected to have. rows:
// the grid's second extent.
template <int DT, int MODE, bool GATED>
int launch_stream(const StreamArgs& s, int columns, int rows, hipStream_t st) {
  constexpr int kWide = GATED ? 2 : 1;
  if (columns <= 4) launch_stream_as<DT, MODE, GATED, 4, 4, 1>(s, rows, st);
  else if (columns <= 8) launch_stream_as<DT, MODE, GATED, 2, 2 * kWide, 1>(s, rows, st);
  else if (columns <= 16) launch_stream_as<DT, MODE, GATED, 1, kWide, 1>(s, rows, st);
  else if (columns <= 32) launch_stream_as<DT, MODE, GATED, 1, kWide, 2>(s, rows, st);
  else if (columns <= 48) launch_stream_as<DT, MODE, GATED, 1, kWide, 3>(s, rows, st);
  else launch_stream_as<DT, MODE, GATED, 1, kWide, 4>(s, rows, st);
  return launch_status();
}

}  // namespace gemm
}  // namespace sgl
