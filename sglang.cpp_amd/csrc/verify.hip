// Verification of drafted tokens (speculative sampling): request r's drafts
// x_i, i < n, each drawn from q_i, are accepted in order while
//   u_i q_i(x_i) < p_i(x_i)            (probability min(1, p / q)),
// p_i the target's probabilities after i drafts. The token that follows the
// accepted ones is drawn from w(j) = max(p_a(j) - q_a(j), 0) at the first
// rejected draft a, or from p_n when all were accepted: the first j whose running
// sum of w exceeds u * sum(w). The tokens are then distributed as the target's
// own draws. Drafts without probabilities are point masses: q_i(x_i) = 1.
//
// The product u q and the difference p - q of fp32 values and all sums are in
// 64 bits, where products are exact and the order of a sum moves the drawn
// token only for a u within about 1e-13 of a border.
//
// Two launches. verify_sums_kernel: a workgroup per (request, slice of the
// vocabulary) finds the request's first rejected draft by itself (a few
// dependent loads) and sums its slice of w and of p. verify_draw_kernel: a
// workgroup per request picks the slice the draw falls into from the slices'
// sums and walks that slice alone. Bound by reading one target row and, where a
// draft was rejected, one draft row per request: 48 requests of a vocabulary of 151,936
// (38 slices), some 23 of them with a rejected draft, 13.7 us in all, 43 MB, 3.1 TB/s (the
// first launch 10.5 us, 4.1 TB/s); one request 8.7 us, two launches and their chains of
// dependent loads.
#include "common.h"

namespace sgl {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kPer = 16;                    // elements of a thread
constexpr int kSlice = kThreads * kPer;     // elements of a slice
constexpr int kLines = kPer / 4;            // groups of 4 consecutive elements of a thread
// Slices of a launch up to which each is a workgroup, else runs of four: 1,824 slices (48
// requests of 151,936) 14.1 us one by one and 16.0 in runs, 9,728 (256 requests) 36.5 and
// 32.6.
constexpr int64_t kSingles = 4096;

struct VerifyArgs {
  const float* target;
  int64_t target_st;
  const float* draft;  // null: point masses
  int64_t draft_st;
  const int32_t* draft_tokens;
  const int32_t* indptr;
  const float* accept_u;
  const float* sample_u;
  int64_t num_drafts;
  int vocab, slices;
  int32_t* tokens;
  int32_t* accepted;
  double* sums;  // [batch, slices, 2]: of w and of p
};

struct Request {
  int64_t d0;   // first draft
  int n;        // drafts; -1: the offsets are not valid
  int a;        // accepted
};

// Accepted drafts of request r, the same in every thread of the calling wave.
__device__ __forceinline__ Request accepted_of(const VerifyArgs& v, int r, int lane) {
  Request q;
  const int64_t d0 = v.indptr[r], d1 = v.indptr[r + 1];
  q.d0 = d0;
  q.n = d0 >= 0 && d1 >= d0 && d1 <= v.num_drafts ? static_cast<int>(d1 - d0) : -1;
  q.a = q.n < 0 ? -1 : q.n;
  for (int i0 = 0; i0 < q.n; i0 += kWave) {
    const int i = i0 + lane;
    bool reject = false;
    if (i < q.n) {
      const int x = v.draft_tokens[d0 + i];
      reject = true;
      if (x >= 0 && x < v.vocab) {
        const double p = v.target[(d0 + i + r) * v.target_st + x];
        const double qx = v.draft ? static_cast<double>(v.draft[(d0 + i) * v.draft_st + x]) : 1.0;
        reject = !(static_cast<double>(v.accept_u[d0 + i]) * qx < p);
      }
    }
    const uint64_t m = __builtin_amdgcn_ballot_w64(reject);
    if (m != 0) {
      q.a = i0 + __builtin_ctzll(m);
      break;
    }
  }
  return q;
}

// The rows the draw of a request reads: p, and q where a draft was rejected.
struct Rows {
  const float* p;
  const float* q;  // null: none
  int point;       // the rejected draft as a point mass, or -1
};

__device__ __forceinline__ Rows rows_of(const VerifyArgs& v, const Request& q, int r) {
  Rows w;
  w.p = v.target + (q.d0 + q.a + r) * v.target_st;
  w.q = nullptr;
  w.point = -1;
  if (q.a < q.n) {
    if (v.draft) w.q = v.draft + (q.d0 + q.a) * v.draft_st;
    else w.point = v.draft_tokens[q.d0 + q.a];
  }
  return w;
}

// Four consecutive elements of a row, whose address is a multiple of 4 bytes.
typedef float f32x4_any_t __attribute__((ext_vector_type(4), aligned(4)));

// A thread's 16 elements of slice s: group g holds elements
// [1024 g + 4 t, ... + 4) of the slice, so a wave reads whole lines.
__device__ __forceinline__ void load_slice(const float* row, int s, int vocab, int t,
                                           float (&x)[kPer]) {
  const int e0 = s * kSlice + 4 * t;  // at most 2^24 and a few slices
  if ((s + 1) * kSlice <= vocab) {  // a whole slice
#pragma unroll
    for (int g = 0; g < kLines; ++g) {
      const f32x4_any_t v =
          __builtin_nontemporal_load(reinterpret_cast<const f32x4_any_t*>(row + e0 + g * 4 * kThreads));
#pragma unroll
      for (int i = 0; i < 4; ++i) x[4 * g + i] = v[i];
    }
    return;
  }
#pragma unroll
  for (int g = 0; g < kLines; ++g)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int e = e0 + g * 4 * kThreads + i;
      x[4 * g + i] = e < vocab ? row[e] : 0.f;
    }
}

// What an element weighs: its p, and its w.
__device__ __forceinline__ double positive(double x) { return x > 0 ? x : 0; }  // NaN weighs nothing

// Lane exchange inside the vector registers (a shuffle is an LDS round trip, twice for
// 64 bits): lanes that a shift brings nothing to, and rows outside the mask, get 0.
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_or_zero(double x) {
  const uint64_t w = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(w), CTRL, ROWS, 0xF, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(w >> 32), CTRL, ROWS, 0xF, false);
  return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}

// Sum over the lanes up to this one: shifts by 1, 2, 4 and 8 in each row of 16, then
// the last lane of a row to the next row, of the first half to the second.
__device__ __forceinline__ double wave_scan(double x) {
  x += dpp_or_zero<0x111, 0xF>(x);
  x += dpp_or_zero<0x112, 0xF>(x);
  x += dpp_or_zero<0x114, 0xF>(x);
  x += dpp_or_zero<0x118, 0xF>(x);
  x += dpp_or_zero<0x142, 0xA>(x);
  x += dpp_or_zero<0x143, 0xC>(x);
  return x;
}

// Lane `at`'s value (the same `at` in every lane).
__device__ __forceinline__ double lane_value(double x, int at) {
  const uint64_t w = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(w), at);
  const uint32_t hi = __builtin_amdgcn_readlane(static_cast<int>(w >> 32), at);
  return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}

// kRun consecutive slices a workgroup, the next one's loads in flight while one is
// summed: the dependent loads of accepted_of() come before 16 KB or before 64.
template <int kRun>
__global__ void __launch_bounds__(kThreads) verify_sums_kernel(VerifyArgs v) {
  __shared__ double part[kRun][2][kWaves];
  const int s0 = blockIdx.x * kRun, r = blockIdx.y;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const Request q = accepted_of(v, r, lane);
  if (s0 == 0) {
    // The accepted drafts, and -1 behind the place of the drawn token.
    for (int i = t; i < q.n; i += kThreads) {
      if (i < q.a) v.tokens[q.d0 + r + i] = v.draft_tokens[q.d0 + i];
      else v.tokens[q.d0 + r + i + 1] = -1;
    }
    if (t == 0) v.accepted[r] = q.a;
  }
  if (q.n < 0) return;
  const Rows w = rows_of(v, q, r);
  float p[2][kPer], d[2][kPer];
  load_slice(w.p, s0, v.vocab, t, p[0]);
  if (w.q) load_slice(w.q, s0, v.vocab, t, d[0]);
#pragma unroll
  for (int k = 0; k < kRun; ++k) {
    const int s = s0 + k, b = k & 1;
    if (k + 1 < kRun) {  // past the last slice: all zero, not read
      load_slice(w.p, s + 1, v.vocab, t, p[b ^ 1]);
      if (w.q) load_slice(w.q, s + 1, v.vocab, t, d[b ^ 1]);
    }
    double sp = 0, sw = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int e = s * kSlice + (i >> 2) * 4 * kThreads + 4 * t + (i & 3);
      sp += positive(p[b][i]);
      double x = p[b][i];
      if (w.q) x -= static_cast<double>(d[b][i]);
      if (e == w.point) x = 0;
      sw += positive(x);
    }
    sp = wave_scan(sp);
    sw = wave_scan(sw);
    if (lane == 63) part[k][0][wave] = sw, part[k][1][wave] = sp;
  }
  __syncthreads();
  if (t < 2 * kRun && s0 + t / 2 < v.slices) {
    double x = 0;
    for (int k = 0; k < kWaves; ++k) x += part[t / 2][t & 1][k];
    v.sums[(static_cast<int64_t>(r) * v.slices + s0) * 2 + t] = x;
  }
}

__global__ void __launch_bounds__(kThreads) verify_draw_kernel(VerifyArgs v) {
  __shared__ double part[kWaves];
  __shared__ int hit[kWaves], last[kWaves];
  const int r = blockIdx.x;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const double* sums = v.sums + static_cast<int64_t>(r) * v.slices * 2;
  Request q;
  q.a = v.accepted[r];
  q.d0 = v.indptr[r];
  q.n = static_cast<int>(v.indptr[r + 1] - q.d0);
  const double u = v.sample_u[r];
  // Every wave looks through the slices' sums, 64 at a time.
  double total = 0, total_p = 0;
  for (int k0 = 0; k0 < v.slices; k0 += kWave) {
    const int k = k0 + lane;
    total += lane_value(wave_scan(k < v.slices ? sums[2 * k] : 0), 63);
    total_p += lane_value(wave_scan(k < v.slices ? sums[2 * k + 1] : 0), 63);
  }
  if (q.a < 0) return;
  const bool residual = total > 0;  // p <= q everywhere: the draw is from p
  const int col = residual ? 0 : 1;
  if (!residual) total = total_p;
  int32_t* out = v.tokens + q.d0 + r + q.a;
  if (!(total > 0)) {
    if (t == 0) *out = v.vocab - 1;
    return;
  }
  const double goal = u * total;
  // The slice whose running sum passes the goal, or the last one with any weight,
  // should rounding leave none.
  double before = 0, base = 0;
  int s = 0;
  for (int k0 = 0; k0 < v.slices; k0 += kWave) {
    const int k = k0 + lane;
    const double x = k < v.slices ? sums[2 * k + col] : 0;
    const double incl = wave_scan(x);
    const uint64_t past = __builtin_amdgcn_ballot_w64(before + incl > goal && x > 0);
    const uint64_t any = __builtin_amdgcn_ballot_w64(x > 0);
    if (any == 0) continue;
    const int at = past ? __builtin_ctzll(past) : 63 - __builtin_clzll(any);
    s = k0 + at;
    base = before + lane_value(incl - x, at);
    if (past) break;
    before += lane_value(incl, 63);
  }
  // The slice in order: thread t has its elements [16 t, 16 t + 16).
  Rows w = rows_of(v, q, r);
  if (!residual) w.q = nullptr, w.point = -1;
  const int e0 = s * kSlice + kPer * t;
  double x[kPer];
  if (e0 + kPer <= v.vocab) {
    f32x4_any_t p[kLines], d[kLines];
#pragma unroll
    for (int g = 0; g < kLines; ++g) {
      p[g] = *reinterpret_cast<const f32x4_any_t*>(w.p + e0 + 4 * g);
      if (w.q) d[g] = *reinterpret_cast<const f32x4_any_t*>(w.q + e0 + 4 * g);
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      x[i] = p[i >> 2][i & 3];
      if (w.q) x[i] -= static_cast<double>(d[i >> 2][i & 3]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      x[i] = e0 + i < v.vocab ? w.p[e0 + i] : 0.f;
      if (w.q && e0 + i < v.vocab) x[i] -= static_cast<double>(w.q[e0 + i]);
    }
  }
  double sum = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    x[i] = e0 + i == w.point ? 0 : positive(x[i]);
    sum += x[i];
  }
  const double incl = wave_scan(sum);
  if (lane == 63) part[wave] = incl;
  __syncthreads();
  double run = base + (incl - sum);
  for (int k = 0; k < wave; ++k) run += part[k];
  int first = -1, final = -1;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    run += x[i];
    if (x[i] > 0) {
      final = e0 + i;
      if (first < 0 && run > goal) first = final;
    }
  }
  const uint64_t mf = __builtin_amdgcn_ballot_w64(first >= 0);
  const uint64_t ml = __builtin_amdgcn_ballot_w64(final >= 0);
  const int f = mf ? __builtin_amdgcn_readlane(first, __builtin_ctzll(mf)) : -1;
  const int l = ml ? __builtin_amdgcn_readlane(final, 63 - __builtin_clzll(ml)) : -1;
  if (lane == 0) hit[wave] = f, last[wave] = l;
  __syncthreads();
  if (t == 0) {
    int token = -1, end = v.vocab - 1;
    for (int k = 0; k < kWaves; ++k) {
      if (token < 0) token = hit[k];
      if (last[k] >= 0) end = last[k];
    }
    *out = token >= 0 ? token : end;
  }
}

inline int slices_of(int vocab) { return (vocab + kSlice - 1) / kSlice; }

}  // namespace
}  // namespace sgl

using namespace sgl;

extern "C" int64_t sgl_verify_workspace_bytes(int batch_size, int vocab) {
  if (batch_size <= 0 || vocab <= 0) return 0;
  return static_cast<int64_t>(batch_size) * slices_of(vocab) * 2 * 8;
}

extern "C" int sgl_verify_drafts(const sgl_verify_args_t* args, void* workspace,
                                 int64_t workspace_bytes, void* stream) {
  if (!args) return SGL_ERR_INVALID_ARG;
  const sgl_verify_args_t& x = *args;
  if (x.batch_size < 0 || x.num_drafts < 0 || x.vocab <= 0) return SGL_ERR_INVALID_ARG;
  if (x.batch_size == 0) return x.num_drafts == 0 ? SGL_OK : SGL_ERR_INVALID_ARG;
  if (!x.target_probs || !x.draft_indptr || !x.sample_uniform || !x.tokens || !x.accepted)
    return SGL_ERR_INVALID_ARG;
  if (x.num_drafts > 0 && (!x.draft_tokens || !x.accept_uniform)) return SGL_ERR_INVALID_ARG;
  if (x.target_stride_row < x.vocab || (x.draft_probs && x.draft_stride_row < x.vocab))
    return SGL_ERR_INVALID_ARG;
  if (x.batch_size > 65535 || x.num_drafts > 0x7fffffff - x.batch_size || x.vocab > (1 << 24))
    return SGL_ERR_UNSUPPORTED;
  if (!workspace || workspace_bytes < sgl_verify_workspace_bytes(x.batch_size, x.vocab))
    return SGL_ERR_CAPACITY;
  if (!aligned16(workspace)) return SGL_ERR_ALIGNMENT;
  VerifyArgs v{};
  v.target = x.target_probs, v.target_st = x.target_stride_row;
  v.draft = x.draft_probs, v.draft_st = x.draft_stride_row;
  v.draft_tokens = x.draft_tokens, v.indptr = x.draft_indptr;
  v.accept_u = x.accept_uniform, v.sample_u = x.sample_uniform;
  v.num_drafts = x.num_drafts, v.vocab = x.vocab, v.slices = slices_of(x.vocab);
  v.tokens = x.tokens, v.accepted = x.accepted;
  v.sums = static_cast<double*>(workspace);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (static_cast<int64_t>(v.slices) * x.batch_size <= kSingles)
    hipLaunchKernelGGL(verify_sums_kernel<1>, dim3(v.slices, x.batch_size), dim3(kThreads), 0, s, v);
  else
    hipLaunchKernelGGL(verify_sums_kernel<4>, dim3((v.slices + 3) / 4, x.batch_size), dim3(kThreads), 0, s, v);
  const int st = launch_status();
  if (st != SGL_OK) return st;
  hipLaunchKernelGGL(verify_draw_kernel, dim3(x.batch_size), dim3(kThreads), 0, s, v);
  return launch_status();
}
