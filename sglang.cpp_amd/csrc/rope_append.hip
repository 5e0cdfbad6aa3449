// Rotary tables scaled for long contexts, and the pass that rotates q and k
// and appends k and v to the paged pool.
//
// Table: cos[p, i] = m cos(p f_i), sin[p, i] = m sin(p f_i) for the rotary
// dimension R and i < R / 2, the frequencies f_i = base^(-2 i / R) changed by
// the scaling (see scaled_frequencies). The angle is p f_i in 64 bits: in 32 a
// position of 100,000 moves the first pairs by some thousandths of a radian.
//
// Rotation of the pair (a, b) of a head: a' = a c - b s, b' = b c + a s, with
// (a, b) = (x[i], x[i + R/2]) (half layout) or (x[2 i], x[2 i + 1])
// (interleaved), in fp32, rounded once; elements from R on pass through.
#include <math.h>

#include "common.h"
#include "norm_rope_row.h"

namespace sgl {
namespace {

constexpr int kMaxPairs = 256;

constexpr int kFewPairs = 64;

// Quarter turns per position of each pair: f_i 2 / pi. A launch copies its arguments, so
// few pairs have a small one (4,096 positions of 32 pairs 6.8 us a call with room for 256
// pairs, 6.4 with room for 64).
template <int P>
struct TurnArgs {
  double turns[P];
};

// cos and sin of x quarter turns, |x| < 2^31, x in 64 bits: the nearest whole
// number of quarter turns goes in 64 bits, the rest (at most half a quarter
// turn, so an angle up to pi / 4) into the Taylor series of sin to the 9th and
// cos to the 10th power (what they leave out is below 2e-9), in fp32.
__device__ __forceinline__ void cos_sin_turns(double x, float& c, float& s) {
  const double k = rint(x);
  const float y = static_cast<float>(x - k) * 1.57079632679489662f;
  const float z = y * y;
  float sy = fmaf(z, 2.7557319224e-6f, -1.9841269841e-4f);
  sy = fmaf(z, sy, 8.3333333333e-3f);
  sy = fmaf(z, sy, -1.6666666667e-1f);
  sy = fmaf(y * z, sy, y);
  float cy = fmaf(z, -2.7557319224e-7f, 2.4801587302e-5f);
  cy = fmaf(z, cy, -1.3888888889e-3f);
  cy = fmaf(z, cy, 4.1666666667e-2f);
  cy = fmaf(z, cy, -0.5f);
  cy = fmaf(z, cy, 1.0f);
  const uint32_t quarter = static_cast<uint32_t>(static_cast<int32_t>(k));
  // Quarters 0..3: (c, s), (-s, c), (-c, -s), (s, -c).
  const float cc = quarter & 1 ? sy : cy, ss = quarter & 1 ? cy : sy;
  c = __uint_as_float(__float_as_uint(cc) ^ (((quarter + 1) & 2) << 30));
  s = __uint_as_float(__float_as_uint(ss) ^ ((quarter & 2) << 30));
}

// A thread keeps the frequencies of N consecutive pairs and walks positions, so
// an entry costs one 64-bit product and the series. Bound by its stores: 131,072
// positions of 64 pairs (67 MB) 12.2 us, 5.5 TB/s (a fill of 1 GiB 6.85); a few thousand
// positions by the launch.
template <int N, int P>
__global__ void __launch_bounds__(256) rope_table_kernel(float* __restrict__ cos_cache,
                                                         float* __restrict__ sin_cache,
                                                         int64_t max_pos, int half, float m,
                                                         int rows, TurnArgs<P> t) {
  const int cols = half / N;  // threads of a position
  const int r = threadIdx.x / cols;
  const int col = threadIdx.x - r * cols;
  if (r >= rows) return;
  double turns[N];
#pragma unroll
  for (int i = 0; i < N; ++i) turns[i] = t.turns[col * N + i];
  const int64_t step = static_cast<int64_t>(gridDim.x) * rows;
  for (int64_t p = static_cast<int64_t>(blockIdx.x) * rows + r; p < max_pos; p += step) {
    float c[N], s[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      cos_sin_turns(static_cast<double>(p) * turns[i], c[i], s[i]);
      c[i] *= m;
      s[i] *= m;
    }
    const int64_t at = p * half + col * N;
    if constexpr (N == 4) {
      *reinterpret_cast<f32x4_t*>(cos_cache + at) = f32x4_t{c[0], c[1], c[2], c[3]};
      *reinterpret_cast<f32x4_t*>(sin_cache + at) = f32x4_t{s[0], s[1], s[2], s[3]};
    } else {
      cos_cache[at] = c[0];
      sin_cache[at] = s[0];
    }
  }
}

// --- rotate and append --------------------------------------------------------

struct AppendArgs {
  const uint16_t* q;
  int64_t q_st, q_sh;
  uint16_t* q_out;
  int64_t qo_st, qo_sh;
  const uint16_t* k;
  int64_t k_st, k_sh;
  const uint16_t* v;
  int64_t v_st, v_sh;
  uint16_t* k_cache;
  uint16_t* v_cache;
  int64_t kv_ss, kv_sh, num_slots;
  const float* cos;
  const float* sin;
  int64_t max_pos;
  const int32_t* positions;
  const void* out_loc;  // null: token t goes to slot t
  int64_t tokens;
  int hq, hk, hv;  // rows of a token: q heads, k heads, v heads (0 or hk)
  int d, rotary;
  bool wide_slots;  // out_loc is int64
};

__device__ __forceinline__ int64_t slot_of(const AppendArgs& a, int64_t t) {
  if (a.out_loc == nullptr) return t;
  return a.wide_slots ? static_cast<const int64_t*>(a.out_loc)[t]
                      : static_cast<const int32_t*>(a.out_loc)[t];
}

// Source and destination of row r of token t; dst is null where the token's slot
// is outside the pool (padding).
__device__ __forceinline__ void append_row(const AppendArgs& a, int64_t t, int r, int64_t slot,
                                           const uint16_t*& src, uint16_t*& dst) {
  if (r < a.hq) {
    src = a.q + t * a.q_st + r * a.q_sh;
    dst = a.q_out + t * a.qo_st + r * a.qo_sh;
    return;
  }
  const bool is_v = r >= a.hq + a.hk;
  const int h = r - a.hq - (is_v ? a.hk : 0);
  src = is_v ? a.v + t * a.v_st + h * a.v_sh : a.k + t * a.k_st + h * a.k_sh;
  dst = slot >= 0 && slot < a.num_slots
            ? (is_v ? a.v_cache : a.k_cache) + slot * a.kv_ss + h * a.kv_sh : nullptr;
}

// Any size and alignment: a thread takes one pair, or one element that passes
// through, in 2-byte accesses, and works out its token, row and pair with two divisions.
// 32q/8kv, us: 7 tokens 5 to 6; 2,047 and 16,384 tokens of head_dim 128 off the 16-byte grid
// 29 and 249 (1.6 TB/s), rotary 40 46 and 394, head_dim 80 with rotary 20 31 and 266,
// head_dim 72 with rotary 36 26 and 217 (1.0 TB/s). The chunks below take 10 and 67 for
// head_dim 128, 11 and 65 for head_dim 80, whole heads.
template <int DT, bool kInterleaved>
__global__ void __launch_bounds__(256) rope_append_elements_kernel(AppendArgs a) {
  const int half = a.rotary / 2;
  const int jobs = a.d - half;  // of a row
  const int per_token = (a.hq + a.hk + a.hv) * jobs;
  const int64_t all = a.tokens * per_token;
  for (int64_t at = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; at < all;
       at += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t t = at / per_token;
    const int rest = static_cast<int>(at - t * per_token);
    const int r = rest / jobs, j = rest - r * jobs;
    const uint16_t* src;
    uint16_t* dst;
    append_row(a, t, r, slot_of(a, t), src, dst);
    if (dst == nullptr) continue;
    const bool is_v = r >= a.hq + a.hk;
    if (j >= half) {
      dst[half + j] = src[half + j];
      continue;
    }
    const int e0 = kInterleaved ? 2 * j : j, e1 = kInterleaved ? 2 * j + 1 : j + half;
    const uint16_t x0 = src[e0], x1 = src[e1];
    if (is_v) {
      dst[e0] = x0;
      dst[e1] = x1;
      continue;
    }
    const int64_t p = a.positions[t];
    float c = NAN, s = NAN;  // a position outside the table is never rotated by a guess
    if (p >= 0 && p < a.max_pos) {
      c = a.cos[p * half + j];
      s = a.sin[p * half + j];
    }
    const float f0 = to_f32<DT>(x0), f1 = to_f32<DT>(x1);
    dst[e0] = static_cast<uint16_t>(from_f32<DT>(rope_one(f0, -f1, c, s)));
    dst[e1] = static_cast<uint16_t>(from_f32<DT>(rope_one(f1, f0, c, s)));
  }
}

// Rows in 16-byte chunks: a job takes two chunks of a row, so that a rotated pair
// of the half layout is in one thread (chunks j and j + R / 16) and nothing is
// exchanged; interleaved pairs and copied elements lie inside a chunk, and there the
// two are half a row apart, so that the lanes of a row read and write whole lines.
// The token is the same for a whole workgroup (scalar slot and position loads); its
// rows' jobs take blocks_per_token workgroups of a width that leaves few threads
// without a job. kTokens tokens a thread, their loads in flight together. Bound by
// the bytes of the rows, read once and written once: non-temporal. 32q/8kv, head_dim
// 128, us with two tokens a thread and with one: 2,047 tokens (50 MB, from and to the
// last-level cache) 9.8 and 10.6, 4,096 20.3 and 18.4, 16,384 (403 MB) 72 and 67.
constexpr int64_t kOneTokenBytes = 64ll << 20;  // rows read and written, from which a thread has one token

template <int DT>
__device__ __forceinline__ void rotate_half(u32x4_t& x, u32x4_t& y, const float* c, const float* s) {
  float a[8], b[8], u[8], v[8];
  unpack8_t<DT>(x, a);
  unpack8_t<DT>(y, b);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    u[i] = rope_one(a[i], -b[i], c[i], s[i]);
    v[i] = rope_one(b[i], a[i], c[i], s[i]);
  }
  x = pack8_t<DT>(u);
  y = pack8_t<DT>(v);
}

template <int DT>
__device__ __forceinline__ void rotate_pairs(u32x4_t& x, const f32x4_t& c, const f32x4_t& s) {
  float a[8], u[8];
  unpack8_t<DT>(x, a);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    u[2 * i] = rope_one(a[2 * i], -a[2 * i + 1], c[i], s[i]);
    u[2 * i + 1] = rope_one(a[2 * i + 1], a[2 * i], c[i], s[i]);
  }
  x = pack8_t<DT>(u);
}

// J: jobs of a row (head_dim / 16), 0: read from the arguments.
template <int DT, bool kInterleaved, int J, int kTokens>
__global__ void __launch_bounds__(512) rope_append_kernel(AppendArgs a, int blocks_per_token) {
  const int jobs = J ? J : a.d / 16;
  const uint32_t group = blockIdx.x / static_cast<uint32_t>(blocks_per_token);
  const int item = static_cast<int>(blockIdx.x - group * blocks_per_token) * blockDim.x + threadIdx.x;
  const int r = item / jobs, j = item - r * jobs;
  if (r >= a.hq + a.hk + a.hv) return;
  const bool is_v = r >= a.hq + a.hk;
  const int pairs = a.rotary / 16;  // half layout: jobs that rotate
  int c0, c1;                       // the job's chunks
  bool turn0, turn1;
  if (kInterleaved || is_v) {
    c0 = j, c1 = j + jobs;
    turn0 = !is_v && 8 * c0 < a.rotary, turn1 = !is_v && 8 * c1 < a.rotary;
  } else {
    turn0 = turn1 = j < pairs;
    c0 = turn0 ? j : 2 * pairs + (j - pairs);
    c1 = turn0 ? j + pairs : c0 + (jobs - pairs);
  }
  u32x4_t x[kTokens], y[kTokens];
  uint16_t* dst[kTokens];
  int64_t pos[kTokens];
#pragma unroll
  for (int k = 0; k < kTokens; ++k) {
    const int64_t t = min(static_cast<int64_t>(group) * kTokens + k, a.tokens - 1);
    const uint16_t* src;
    append_row(a, t, r, slot_of(a, t), src, dst[k]);
    if (static_cast<int64_t>(group) * kTokens + k >= a.tokens) dst[k] = nullptr;
    x[k] = ldg128_nt<true>(src + 8 * c0);
    y[k] = ldg128_nt<true>(src + 8 * c1);
    pos[k] = a.positions[t];
  }
  const int half = a.rotary / 2;
#pragma unroll
  for (int k = 0; k < kTokens; ++k) {
    if (dst[k] == nullptr) continue;
    const bool far = pos[k] < 0 || pos[k] >= a.max_pos;  // never rotated by a guess: NaN
    const float* cr = a.cos + (far ? 0 : pos[k]) * half;
    const float* sr = a.sin + (far ? 0 : pos[k]) * half;
    if (kInterleaved) {
      const f32x4_t nan = {NAN, NAN, NAN, NAN};
      if (turn0) {
        f32x4_t c = nan, s = nan;
        if (!far) {
          c = *reinterpret_cast<const f32x4_t*>(cr + 4 * c0);
          s = *reinterpret_cast<const f32x4_t*>(sr + 4 * c0);
        }
        rotate_pairs<DT>(x[k], c, s);
      }
      if (turn1) {
        f32x4_t c = nan, s = nan;
        if (!far) {
          c = *reinterpret_cast<const f32x4_t*>(cr + 4 * c1);
          s = *reinterpret_cast<const f32x4_t*>(sr + 4 * c1);
        }
        rotate_pairs<DT>(y[k], c, s);
      }
    } else if (turn0) {
      float c[8], s[8];
#pragma unroll
      for (int i = 0; i < 8; i += 4) {
        f32x4_t cv = {NAN, NAN, NAN, NAN}, sv = cv;
        if (!far) {
          cv = *reinterpret_cast<const f32x4_t*>(cr + 8 * j + i);
          sv = *reinterpret_cast<const f32x4_t*>(sr + 8 * j + i);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) c[i + e] = cv[e], s[i + e] = sv[e];
      }
      rotate_half<DT>(x[k], y[k], c, s);
    }
    stg128_nt<true>(dst[k] + 8 * c0, x[k]);
    stg128_nt<true>(dst[k] + 8 * c1, y[k]);
  }
}

template <int DT, bool kInterleaved, int kTokens>
void launch_chunks(const AppendArgs& a, hipStream_t s) {
  const int jobs = a.d / 16;
  const int64_t items = (static_cast<int64_t>(a.hq) + a.hk + a.hv) * jobs;
  // The workgroup width, in waves, that leaves the fewest threads without a job.
  int waves = 4;
  int64_t best = -1;
  for (int w = 8; w >= 2; --w) {
    const int64_t idle = (items + 64 * w - 1) / (64 * w) * (64 * w) - items;
    if (best < 0 || idle < best) best = idle, waves = w;
  }
  const int64_t per_token = (items + 64 * waves - 1) / (64 * waves);
  const dim3 grid(static_cast<uint32_t>((a.tokens + kTokens - 1) / kTokens * per_token));
  const dim3 block(64 * waves);
  const int bpt = static_cast<int>(per_token);
  switch (jobs) {
    case 4: hipLaunchKernelGGL((rope_append_kernel<DT, kInterleaved, 4, kTokens>), grid, block, 0, s, a, bpt); break;
    case 8: hipLaunchKernelGGL((rope_append_kernel<DT, kInterleaved, 8, kTokens>), grid, block, 0, s, a, bpt); break;
    default: hipLaunchKernelGGL((rope_append_kernel<DT, kInterleaved, 0, kTokens>), grid, block, 0, s, a, bpt);
  }
}

template <int P>
int launch_table(float* cos_cache, float* sin_cache, int64_t max_pos, int half, float m, const double* f, hipStream_t s) {
  TurnArgs<P> t{};
  for (int i = 0; i < half; ++i) t.turns[i] = f[i];
  const bool wide = half % 4 == 0 && aligned16(cos_cache) && aligned16(sin_cache);
  const int rows = 256 / (wide ? half / 4 : half);
  const int64_t blocks = (max_pos + rows - 1) / rows;
  const dim3 grid(static_cast<uint32_t>(blocks < 4096 ? blocks : 4096));
  if (wide)
    hipLaunchKernelGGL((rope_table_kernel<4, P>), grid, dim3(256), 0, s, cos_cache, sin_cache, max_pos, half, m, rows, t);
  else
    hipLaunchKernelGGL((rope_table_kernel<1, P>), grid, dim3(256), 0, s, cos_cache, sin_cache, max_pos, half, m, rows, t);
  return launch_status();
}

template <int DT>
void launch_chunks(const AppendArgs& a, bool interleaved, hipStream_t s) {
  const int64_t bytes = a.tokens * (static_cast<int64_t>(a.hq) + a.hk + a.hv) * a.d * 4;
  if (bytes >= kOneTokenBytes) {
    if (interleaved) launch_chunks<DT, true, 1>(a, s); else launch_chunks<DT, false, 1>(a, s);
  } else {
    if (interleaved) launch_chunks<DT, true, 2>(a, s); else launch_chunks<DT, false, 2>(a, s);
  }
}

inline int64_t blocks_for(int64_t jobs, int64_t per_block) { return (jobs + per_block - 1) / per_block; }

// f_i of each pair and the factor of cos and sin, from the scaling's published
// definition: positions divided by the factor (linear), the base raised so that
// the slowest pair does so and the fastest stays (ntk), or per pair a blend of
// both by how often it turns over the original context: by the pair's index
// between the two that turn beta_fast and beta_slow times (yarn, with its factor
// of cos and sin), or by the number of turns itself (bands).
int scaled_frequencies(int rotary, double base, const sgl_rope_scaling_t* sc, double* f, double& m) {
  const int half = rotary / 2;
  const int kind = sc ? sc->kind : SGL_ROPE_SCALING_NONE;
  m = 1.0;
  if (!(base > 0) || !isfinite(base)) return SGL_ERR_INVALID_ARG;
  for (int i = 0; i < half; ++i) f[i] = pow(base, -2.0 * i / rotary);
  if (kind == SGL_ROPE_SCALING_NONE) return SGL_OK;
  const double k = sc->factor;
  if (!(k > 0) || !isfinite(k)) return SGL_ERR_INVALID_ARG;
  const double length = sc->original_max_position;
  const double two_pi = 6.283185307179586476925;
  switch (kind) {
    case SGL_ROPE_SCALING_LINEAR:
      for (int i = 0; i < half; ++i) f[i] /= k;
      return SGL_OK;
    case SGL_ROPE_SCALING_NTK: {
      if (rotary <= 2) return SGL_ERR_INVALID_ARG;
      const double b = base * pow(k, rotary / (rotary - 2.0));
      for (int i = 0; i < half; ++i) f[i] = pow(b, -2.0 * i / rotary);
      return SGL_OK;
    }
    case SGL_ROPE_SCALING_YARN: {
      if (!(length > 0) || !(base > 1) || !(sc->beta_slow > 0) || !(sc->beta_fast >= sc->beta_slow) ||
          !isfinite(sc->beta_fast) || !(sc->attention_factor >= 0) || !isfinite(sc->attention_factor))
        return SGL_ERR_INVALID_ARG;
      auto pair_of = [&](double turns) {
        return rotary * log(length / (two_pi * turns)) / (2.0 * log(base));
      };
      const double low = fmax(floor(pair_of(sc->beta_fast)), 0.0);
      const double high = fmin(ceil(pair_of(sc->beta_slow)), rotary - 1.0);
      for (int i = 0; i < half; ++i) {
        const double keep = 1.0 - fmin(fmax((i - low) / fmax(high - low, 0.001), 0.0), 1.0);
        f[i] = f[i] / k * (1.0 - keep) + f[i] * keep;
      }
      m = sc->attention_factor > 0 ? sc->attention_factor : k > 1 ? 0.1 * log(k) + 1.0 : 1.0;
      return SGL_OK;
    }
    case SGL_ROPE_SCALING_BANDS:
      if (!(length > 0) || !(sc->low_freq_factor > 0) || !(sc->high_freq_factor > sc->low_freq_factor) ||
          !isfinite(sc->high_freq_factor))
        return SGL_ERR_INVALID_ARG;
      for (int i = 0; i < half; ++i) {
        const double turns = length * f[i] / two_pi;
        const double keep = fmin(fmax((turns - sc->low_freq_factor) /
                                          (sc->high_freq_factor - sc->low_freq_factor), 0.0), 1.0);
        f[i] = f[i] / k * (1.0 - keep) + f[i] * keep;
      }
      return SGL_OK;
    default:
      return SGL_ERR_UNSUPPORTED;
  }
}

}  // namespace
}  // namespace sgl

using namespace sgl;

extern "C" int sgl_rope_scaled_cache(float* cos_cache, float* sin_cache, int64_t max_pos,
                                     int rotary_dim, double base, const sgl_rope_scaling_t* scaling,
                                     void* stream) {
  if (max_pos < 0 || max_pos > 0x7fffffff || rotary_dim <= 0 || (rotary_dim & 1))
    return SGL_ERR_INVALID_ARG;
  const int half = rotary_dim / 2;
  if (half > kMaxPairs) return SGL_ERR_UNSUPPORTED;
  double f[kMaxPairs], m;
  const int st = scaled_frequencies(rotary_dim, base, scaling, f, m);
  if (st != SGL_OK) return st;
  if (max_pos == 0) return SGL_OK;
  if (!cos_cache || !sin_cache) return SGL_ERR_INVALID_ARG;
  for (int i = 0; i < half; ++i) {
    f[i] *= 0.636619772367581343076;  // 2 / pi
    // The whole quarter turns of the last position are counted in 31 bits.
    if (!(f[i] * static_cast<double>(max_pos) < 2147483647.0)) return SGL_ERR_UNSUPPORTED;
  }
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (half <= kFewPairs)
    return launch_table<kFewPairs>(cos_cache, sin_cache, max_pos, half, static_cast<float>(m), f, s);
  return launch_table<kMaxPairs>(cos_cache, sin_cache, max_pos, half, static_cast<float>(m), f, s);
}

extern "C" int sgl_rope_append(const sgl_rope_append_t* args, void* stream) {
  if (!args) return SGL_ERR_INVALID_ARG;
  const sgl_rope_append_t& x = *args;
  if (x.tokens < 0 || x.num_qo_heads < 0 || x.num_kv_heads < 0 || x.head_dim <= 0 ||
      x.num_slots < 0 || x.max_pos < 0)
    return SGL_ERR_INVALID_ARG;
  if (x.dtype != SGL_DTYPE_BF16 && x.dtype != SGL_DTYPE_F16) return SGL_ERR_UNSUPPORTED;
  if (x.out_loc && x.index_dtype != SGL_INDEX_I32 && x.index_dtype != SGL_INDEX_I64)
    return SGL_ERR_UNSUPPORTED;
  if (x.flags & ~SGL_ROPE_INTERLEAVED) return SGL_ERR_INVALID_ARG;
  if (x.rotary_dim <= 0 || (x.rotary_dim & 1) || x.rotary_dim > x.head_dim) return SGL_ERR_INVALID_ARG;
  if (x.head_dim > 1024 || x.num_qo_heads > 65536 || x.num_kv_heads > 65536)
    return SGL_ERR_UNSUPPORTED;
  if (x.tokens == 0 || x.num_qo_heads + x.num_kv_heads == 0) return SGL_OK;
  if ((x.v == nullptr) != (x.v_cache == nullptr)) return SGL_ERR_INVALID_ARG;
  if ((x.num_qo_heads && (!x.q || !x.q_out)) || (x.num_kv_heads && (!x.k || !x.k_cache)) || !x.cos ||
      !x.sin || !x.positions)
    return SGL_ERR_INVALID_ARG;
  // In place means the same rows at the same places.
  if (x.num_qo_heads && x.q == x.q_out && (x.q_stride_token != x.q_out_stride_token ||
                                           x.q_stride_head != x.q_out_stride_head))
    return SGL_ERR_INVALID_ARG;
  AppendArgs a{};
  a.q = static_cast<const uint16_t*>(x.q), a.q_st = x.q_stride_token, a.q_sh = x.q_stride_head;
  a.q_out = static_cast<uint16_t*>(x.q_out), a.qo_st = x.q_out_stride_token, a.qo_sh = x.q_out_stride_head;
  a.k = static_cast<const uint16_t*>(x.k), a.k_st = x.k_stride_token, a.k_sh = x.k_stride_head;
  a.v = static_cast<const uint16_t*>(x.v), a.v_st = x.v_stride_token, a.v_sh = x.v_stride_head;
  a.k_cache = static_cast<uint16_t*>(x.k_cache), a.v_cache = static_cast<uint16_t*>(x.v_cache);
  a.kv_ss = x.kv_stride_slot, a.kv_sh = x.kv_stride_head, a.num_slots = x.num_slots;
  a.cos = x.cos, a.sin = x.sin, a.max_pos = x.max_pos, a.positions = x.positions;
  a.out_loc = x.out_loc, a.wide_slots = x.index_dtype == SGL_INDEX_I64, a.tokens = x.tokens;
  a.hq = x.num_qo_heads, a.hk = x.num_kv_heads, a.hv = x.v ? x.num_kv_heads : 0;
  a.d = x.head_dim, a.rotary = x.rotary_dim;
  const bool il = (x.flags & SGL_ROPE_INTERLEAVED) != 0;
  const int64_t rows = static_cast<int64_t>(a.hq) + a.hk + a.hv;
  const int64_t per_token = rows * (a.d - a.rotary / 2);
  if (per_token > 0x7fffffff) return SGL_ERR_UNSUPPORTED;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  auto chunked = [](const void* p, int64_t st, int64_t sh) {
    return p == nullptr || (aligned16(p) && st % 8 == 0 && sh % 8 == 0);
  };
  // Whole chunks everywhere; the launch's threads (rows d / 16 a token and up to a
  // workgroup more) in 32 bits.
  if (a.d % 16 == 0 && a.rotary % 16 == 0 && chunked(a.q, a.q_st, a.q_sh) &&
      chunked(a.q_out, a.qo_st, a.qo_sh) && chunked(a.k, a.k_st, a.k_sh) &&
      chunked(a.v, a.v_st, a.v_sh) && chunked(a.k_cache, a.kv_ss, a.kv_sh) &&
      chunked(a.v_cache, a.kv_ss, a.kv_sh) && aligned16(a.cos) && aligned16(a.sin) &&
      a.tokens < 0xffffffffll / (rows * (a.d / 16) + 512)) {
    if (x.dtype == SGL_DTYPE_BF16) launch_chunks<SGL_DTYPE_BF16>(a, il, s);
    else launch_chunks<SGL_DTYPE_F16>(a, il, s);
    return launch_status();
  }
  const int64_t blocks = blocks_for(a.tokens * per_token, 256);
  const dim3 grid(static_cast<uint32_t>(blocks < 65536 ? blocks : 65536));
  if (x.dtype == SGL_DTYPE_BF16) {
    if (il) hipLaunchKernelGGL((rope_append_elements_kernel<SGL_DTYPE_BF16, true>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((rope_append_elements_kernel<SGL_DTYPE_BF16, false>), grid, dim3(256), 0, s, a);
  } else {
    if (il) hipLaunchKernelGGL((rope_append_elements_kernel<SGL_DTYPE_F16, true>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((rope_append_elements_kernel<SGL_DTYPE_F16, false>), grid, dim3(256), 0, s, a);
  }
  return launch_status();
}
