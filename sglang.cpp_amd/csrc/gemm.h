// Device code shared by the projections (linear.hip) and the experts (moe.hip):
// y[t, n] = sum_k x[t, k] w[n, k] and what follows it.
//
// The matrix instruction's rows are weight rows and its columns tokens, so a lane
// ends with four consecutive outputs of one token (one 8-byte store). Products of
// 16-bit values, sums, bias, activation, weighting and residual are fp32; the result
// is rounded once. Gate and up projections (GATED) are one matrix of 2 n rows: a tile
// alternates blocks of 16 gate rows with the 16 up rows of the same outputs, which so
// meet in one lane.
#pragma once

#include "common.h"

namespace sgl {
namespace gemm {

enum Mode : int {
  kLinear = 0,  // rows of x are the tokens
  kGateUp = 1,  // experts: sorted places read their token's row of x, written in order
  kDown = 2,    // experts: sorted places read in order, weighted, written to their slot
};

struct Args {
  const uint16_t* x;
  const uint16_t* w;
  const uint16_t* bias;  // kLinear
  const uint16_t* res;   // kLinear
  void* out;
  int64_t x_st, w_st, w_se, r_st, o_st;  // strides of a row (w_se: of an expert)
  int32_t tokens, n, k;
  int32_t act;      // SGL_ACT_*
  int32_t out_f32;  // out is fp32
  int32_t wide;     // outputs, bias and residual: 1 of four columns, 2 of eight in whole accesses
  int32_t tiles_n;  // tiles over the outputs
  int32_t tiles;    // tiles in all
  int32_t top_k;
  const int4* places;    // experts: {expert, first place, places, 0} of a tile of places
  const int32_t* order;  // experts: slot (token top_k + j) of each place
  const float* scale;    // kDown: weight of each slot
  float* part;           // sums of the parts of k, where a tile's is split
  int32_t splits;        // parts
};

// A dimension of a grid has fewer than 2^32 threads, and a launch with more is cut short without
// an error. Workgroups past a row of kRow are the next row's; the last row may reach past the
// last of them. Up to 2^31 of them, of up to 512 threads.
constexpr int kRowShift = 22;
constexpr int64_t kRow = 1 << kRowShift;

inline dim3 rows_of(int64_t groups) {
  return dim3(static_cast<uint32_t>(groups < kRow ? groups : kRow),
              static_cast<uint32_t>((groups + kRow - 1) / kRow));
}
__device__ __forceinline__ uint32_t group_index() { return blockIdx.y << kRowShift | blockIdx.x; }

typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));

// D += A B with 16 x 32 and 32 x 16 operands: lane l holds elements 8 (l / 16) .. + 7 of
// A's row l % 16 and of B's column l % 16, and rows 4 (l / 16) .. + 3 of D's column l % 16.
template <int DT>
__device__ __forceinline__ f32x4_t mfma16(const u32x4_t& a, const u32x4_t& b, const f32x4_t& c) {
  if constexpr (DT == SGL_DTYPE_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                   __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a),
                                                  __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}

// x sigmoid(z), z = x (SiLU) or 2 * 0.7978845608 (x + 0.044715 x^3) (tanh GELU, since
// (1 + tanh(u)) / 2 = sigmoid(2 u)), on the hardware exp2 and reciprocal. z log2(e) is rounded, so
// the relative error grows with |z|, to (1 + |z|) 2^-21 at most: a small part of a 16-bit output's
// rounding, all of an fp32 output's error. Below |x| 2^-126 the result is zero.
__device__ __forceinline__ float activate(int act, float x) {
  if (act == SGL_ACT_NONE) return x;
  float z = x;
  if (act == SGL_ACT_GELU || act == SGL_ACT_GELU_AND_MUL)
    z = 2.0f * 0.7978845608f * (x + 0.044715f * x * x * x);
  return x * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-z * 1.4426950408889634f));
}

// Eight elements of a row from element e on, zero from element k on; a row starts anywhere.
__device__ __forceinline__ u32x4_t load8(const uint16_t* row, int e, int k) {
  u32x4_t v = {0, 0, 0, 0};
  if (e + 8 <= k) {
    __builtin_memcpy(&v, row + e, 16);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (e + i < k) v[i / 2] |= static_cast<uint32_t>(row[e + i]) << (16 * (i & 1));
  }
  return v;
}

// Bias and activation of outputs n0 .. n0 + 3 (columns past the last are dropped later).
template <int DT, int MODE, bool GATED>
__device__ __forceinline__ f32x4_t activated4(const Args& a, int n0, f32x4_t g, f32x4_t u) {
  if constexpr (MODE == kLinear) {
    if (a.bias) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int n = min(n0 + i, a.n - 1);
        g[i] += to_f32<DT>(a.bias[n]);
        if constexpr (GATED) u[i] += to_f32<DT>(a.bias[static_cast<int64_t>(a.n) + n]);
      }
    }
  }
  if constexpr (MODE != kDown) {
#pragma unroll
    for (int i = 0; i < 4; ++i) g[i] = activate(a.act, g[i]);
  }
  if constexpr (GATED) g *= u;
  return g;
}

// Weight, residual and rounding of the activated outputs n0 .. n0 + 7 of one row.
template <int DT, int MODE>
__device__ __forceinline__ void store8(const Args& a, int n0, int64_t row, float scale, float (&y)[8]) {
  if (n0 >= a.n) return;
  if constexpr (MODE == kDown) {
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] *= scale;
  }
  const uint16_t* r = MODE == kLinear && a.res ? a.res + row * a.r_st + n0 : nullptr;
  if (a.wide == 2 && n0 + 8 <= a.n) {
    if (r) {
      float f[8];
      unpack8_t<DT>(ldg128(r), f);
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] += f[i];
    }
    if (a.out_f32) {
      float* o = static_cast<float*>(a.out) + row * a.o_st + n0;
      *reinterpret_cast<f32x4_t*>(o) = f32x4_t{y[0], y[1], y[2], y[3]};
      *reinterpret_cast<f32x4_t*>(o + 4) = f32x4_t{y[4], y[5], y[6], y[7]};
    } else {
      stg128(static_cast<uint16_t*>(a.out) + row * a.o_st + n0, pack8_t<DT>(y));
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (n0 + i >= a.n) break;
    const float v = r ? y[i] + to_f32<DT>(r[i]) : y[i];
    if (a.out_f32) static_cast<float*>(a.out)[row * a.o_st + n0 + i] = v;
    else static_cast<uint16_t*>(a.out)[row * a.o_st + n0 + i] = static_cast<uint16_t>(from_f32<DT>(v));
  }
}

// Outputs n0 .. n0 + 3 of one row: g (and, gated, u) from the accumulators.
template <int DT, int MODE, bool GATED>
__device__ __forceinline__ void finish4(const Args& a, int n0, int64_t row, float scale, f32x4_t g,
                                        f32x4_t u) {
  if (n0 >= a.n) return;
  if (a.wide && n0 + 4 <= a.n) {
    if constexpr (MODE == kLinear) {
      if (a.bias) {
        const u32x2_t b = *reinterpret_cast<const u32x2_t*>(a.bias + n0);
#pragma unroll
        for (int i = 0; i < 4; ++i) g[i] += to_f32<DT>((b[i / 2] >> (16 * (i & 1))) & 0xffffu);
        if constexpr (GATED) {
          const u32x2_t c = *reinterpret_cast<const u32x2_t*>(a.bias + a.n + n0);
#pragma unroll
          for (int i = 0; i < 4; ++i) u[i] += to_f32<DT>((c[i / 2] >> (16 * (i & 1))) & 0xffffu);
        }
      }
    }
    if constexpr (MODE != kDown) {
#pragma unroll
      for (int i = 0; i < 4; ++i) g[i] = activate(a.act, g[i]);
    }
    if constexpr (GATED) g *= u;
    if constexpr (MODE == kDown) g *= scale;
    if constexpr (MODE == kLinear) {
      if (a.res) {
        const u32x2_t r = *reinterpret_cast<const u32x2_t*>(a.res + row * a.r_st + n0);
#pragma unroll
        for (int i = 0; i < 4; ++i) g[i] += to_f32<DT>((r[i / 2] >> (16 * (i & 1))) & 0xffffu);
      }
    }
    if (a.out_f32) {
      *reinterpret_cast<f32x4_t*>(static_cast<float*>(a.out) + row * a.o_st + n0) = g;
    } else {
      const u32x2_t v = {pack2_t<DT>(g[0], g[1]), pack2_t<DT>(g[2], g[3])};
      *reinterpret_cast<u32x2_t*>(static_cast<uint16_t*>(a.out) + row * a.o_st + n0) = v;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int n = n0 + i;
    if (n >= a.n) break;
    float y = g[i];
    if constexpr (MODE == kLinear) {
      if (a.bias) y += to_f32<DT>(a.bias[n]);
    }
    if constexpr (MODE != kDown) y = activate(a.act, y);
    if constexpr (GATED) {
      float z = u[i];
      if constexpr (MODE == kLinear) {
        if (a.bias) z += to_f32<DT>(a.bias[static_cast<int64_t>(a.n) + n]);
      }
      y *= z;
    }
    if constexpr (MODE == kDown) y *= scale;
    if constexpr (MODE == kLinear) {
      if (a.res) y += to_f32<DT>(a.res[row * a.r_st + n]);
    }
    if (a.out_f32) static_cast<float*>(a.out)[row * a.o_st + n] = y;
    else static_cast<uint16_t*>(a.out)[row * a.o_st + n] = static_cast<uint16_t>(from_f32<DT>(y));
  }
}

// The part of a launch that a workgroup has: rows [first, first + rows) of the tokens, or
// of an expert's places.
struct Part {
  int expert, first, rows;
};

template <int MODE>
__device__ __forceinline__ Part part_of(const Args& a, int tile, int tile_rows) {
  if constexpr (MODE == kLinear) {
    const int first = tile * tile_rows;
    return {0, first, min(tile_rows, a.tokens - first)};
  } else {
    const int4 t = a.places[tile];
    return {t.x, t.y, t.z};
  }
}

// Row of x, row of the output and weight of place or token i.
template <int MODE>
__device__ __forceinline__ int64_t source_row(const Args& a, int i) {
  return MODE == kGateUp ? a.order[i] / a.top_k : i;
}
template <int MODE>
__device__ __forceinline__ int64_t target_row(const Args& a, int i, float& scale) {
  scale = 1.f;
  if constexpr (MODE == kDown) {
    const int slot = a.order[i];
    scale = a.scale[slot];
    return slot;
  }
  return i;
}

// Weight row of row r of a tile whose first output is n0, -1 past the last output.
template <bool GATED>
__device__ __forceinline__ int64_t weight_row(const Args& a, int n0, int r) {
  const int n = GATED ? n0 + (r >> 5) * 16 + (r & 15) : n0 + r;
  if (n >= a.n) return -1;
  return GATED && (r & 16) ? static_cast<int64_t>(a.n) + n : n;
}

// Any sizes, strides and alignment: tiles of 64 weight rows x 64 tokens, staged through
// registers and LDS, four waves of 32 x 32 outputs. Taken where rows are not whole 16 bytes
// or strides pass what the other kernels' 32-bit offsets reach (8,192 x 24,576 x 4,096: 4.3 ms,
// the other tiles 1.2).
constexpr int kAnyTile = 64;
constexpr int kAnyPitch = 40;  // 32 elements and 16 bytes: rows start on different banks

template <int DT, int MODE, bool GATED>
__global__ __launch_bounds__(256) void any_kernel(const Args a) {
  __shared__ uint16_t sw[kAnyTile * kAnyPitch], sx[kAnyTile * kAnyPitch];
  if (group_index() >= static_cast<uint32_t>(a.tiles)) return;
  const int tn = group_index() % a.tiles_n, tt = group_index() / a.tiles_n;
  const Part p = part_of<MODE>(a, tt, kAnyTile);
  if (p.rows <= 0) return;
  const int n0 = tn * (GATED ? kAnyTile / 2 : kAnyTile);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int r = tid >> 2, c = (tid & 3) * 8;
  const int64_t wr = weight_row<GATED>(a, n0, r);
  const uint16_t* wp = a.w + p.expert * a.w_se + (wr < 0 ? 0 : wr) * a.w_st;
  const bool has_x = r < p.rows;
  const uint16_t* xp = a.x + (has_x ? source_row<MODE>(a, p.first + r) : 0) * a.x_st;
  const u32x4_t zero = {0, 0, 0, 0};
  f32x4_t acc[2][2] = {};
  const int aw = (wave & 1) * 32 + (lane & 15), ax = (wave >> 1) * 32 + (lane & 15);
  const int ac = (lane >> 4) * 8;
  u32x4_t vw = wr < 0 ? zero : load8(wp, c, a.k);
  u32x4_t vx = has_x ? load8(xp, c, a.k) : zero;
  for (int k0 = 0; k0 < a.k; k0 += 32) {
    stg128(&sw[r * kAnyPitch + c], vw);
    stg128(&sx[r * kAnyPitch + c], vx);
    __syncthreads();
    if (k0 + 32 < a.k) {
      vw = wr < 0 ? zero : load8(wp, k0 + 32 + c, a.k);
      vx = has_x ? load8(xp, k0 + 32 + c, a.k) : zero;
    }
    u32x4_t fw[2], fx[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      fw[i] = ldg128(&sw[(aw + 16 * i) * kAnyPitch + ac]);
      fx[i] = ldg128(&sx[(ax + 16 * i) * kAnyPitch + ac]);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) acc[i][j] = mfma16<DT>(fw[i], fx[j], acc[i][j]);
    __syncthreads();
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int t = ax + 16 * j;
    if (t >= p.rows) continue;
    float scale;
    const int64_t row = target_row<MODE>(a, p.first + t, scale);
    const int q = 4 * (lane >> 4);
    if constexpr (GATED) {
      finish4<DT, MODE, true>(a, n0 + (wave & 1) * 16 + q, row, scale, acc[0][j], acc[1][j]);
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i)
        finish4<DT, MODE, false>(a, n0 + (wave & 1) * 32 + 16 * i + q, row, scale, acc[i][j],
                                 acc[i][j]);
    }
  }
}

// Few tokens of any layout: 16 outputs (GATED: and their 16 up rows) and 16 tokens a workgroup,
// whose waves share out units of 32 inputs and fold their sums. Operands come straight into
// registers, 64 bytes of a row by four lanes, kAhead units in flight a wave. Taken up to 16
// tokens, and above while there are at most three workgroups a CU, since each 16 tokens read
// the weights again (1 x 6,144 x 4,097: 30 us, tiles 90; 48 x 4,096 x 12,287, 768 workgroups:
// 224 and 284; 64 tokens: 298 and 290).
template <int DT, bool GATED, int NW>
__global__ __launch_bounds__(64 * NW) void any_few_kernel(const Args a) {
  constexpr int MT = GATED ? 2 : 1, kAhead = 4;
  __shared__ f32x4_t red[NW * MT * 64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n0 = 16 * static_cast<int>(blockIdx.x), t0 = 16 * static_cast<int>(blockIdx.y);
  const int r = lane & 15, c = 8 * (lane >> 4);
  // Rows past the last output or token are computed from it and dropped.
  const int64_t n = min(n0 + r, a.n - 1);
  const uint16_t* w[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) w[i] = a.w + (i * static_cast<int64_t>(a.n) + n) * a.w_st;
  const uint16_t* x = a.x + min(t0 + r, a.tokens - 1) * a.x_st;
  const int whole = a.k / 32;
  const int units = wave < whole ? (whole - wave - 1) / NW + 1 : 0;
  f32x4_t acc[MT] = {};
  u32x4_t fw[kAhead][MT], fx[kAhead];
  auto load = [&](int d, int q) {
    const int at = (wave + q * NW) * 32 + c;
#pragma unroll
    for (int i = 0; i < MT; ++i) __builtin_memcpy(&fw[d][i], w[i] + at, 16);
    __builtin_memcpy(&fx[d], x + at, 16);
  };
#pragma unroll
  for (int d = 0; d < kAhead; ++d)
    if (d < units) load(d, d);
  for (int q = 0; q < units; q += kAhead) {
#pragma unroll
    for (int d = 0; d < kAhead; ++d) {
      if (q + d >= units) break;
#pragma unroll
      for (int i = 0; i < MT; ++i) acc[i] = mfma16<DT>(fw[d][i], fx[d], acc[i]);
      if (q + d + kAhead < units) load(d, q + d + kAhead);
    }
  }
  if (whole * 32 < a.k && whole % NW == wave) {  // the last unit is a part of one
    const u32x4_t v = load8(x, whole * 32 + c, a.k);
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[i] = mfma16<DT>(load8(w[i], whole * 32 + c, a.k), v, acc[i]);
  }
#pragma unroll
  for (int i = 0; i < MT; ++i) red[(wave * MT + i) * 64 + lane] = acc[i];
  __syncthreads();
  if (wave > 0 || t0 + r >= a.tokens) return;
  f32x4_t sum[MT] = {};
  for (int v = 0; v < NW; ++v)
#pragma unroll
    for (int i = 0; i < MT; ++i) sum[i] += red[(v * MT + i) * 64 + lane];
  finish4<DT, kLinear, GATED>(a, n0 + 4 * (lane >> 4), t0 + r, 1.f, sum[0], sum[MT - 1]);
}

inline bool aligned(const void* p, int64_t stride, int64_t bytes, int64_t size) {
  return !p || (reinterpret_cast<uintptr_t>(p) % bytes == 0 && stride * size % bytes == 0);
}

// Tiles of a product, or -1 where a launch has no numbers for them.
inline int64_t all_tiles(int64_t tiles_n, int64_t tiles_t) {
  return tiles_t > 0 && tiles_n > 0x7fffffff / tiles_t ? -1 : tiles_n * tiles_t;
}

constexpr int kCus = 256;
constexpr int kFewWaves = 8;

inline bool takes_any_few(const Args& a) {
  const int64_t x = (static_cast<int64_t>(a.n) + 15) / 16, y = (static_cast<int64_t>(a.tokens) + 15) / 16;
  if (x > 0xffffffffll / (64 * kFewWaves)) return false;  // a grid has fewer than 2^32 threads
  return y == 1 || x * y <= 3 * kCus;
}

template <int DT, bool GATED>
int launch_any_few(const Args& a, hipStream_t s) {
  constexpr int kWaves = kFewWaves;
  const dim3 grid(static_cast<uint32_t>((static_cast<int64_t>(a.n) + 15) / 16), (a.tokens + 15) / 16);
  hipLaunchKernelGGL((any_few_kernel<DT, GATED, kWaves>), grid, dim3(64 * kWaves), 0, s, a);
  return launch_status();
}

template <int DT, int MODE, bool GATED>
int launch_any(Args a, int64_t tiles_t, hipStream_t s) {
  const int out = GATED ? kAnyTile / 2 : kAnyTile;
  a.tiles_n = static_cast<int32_t>((static_cast<int64_t>(a.n) + out - 1) / out);
  const int64_t tiles = all_tiles(a.tiles_n, tiles_t);
  if (tiles < 0) return SGL_ERR_UNSUPPORTED;
  a.tiles = static_cast<int32_t>(tiles);
  hipLaunchKernelGGL((any_kernel<DT, MODE, GATED>), rows_of(tiles), dim3(256), 0, s, a);
  return launch_status();
}

}  // namespace gemm
}  // namespace sgl
