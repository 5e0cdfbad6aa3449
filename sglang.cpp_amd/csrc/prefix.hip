// Attention of a batch that shares a prefix: row (token t, head) of request r is
//   o = softmax_j(q . k_j scale) . v_j  over the prefix's tokens, then the request's own,
// j <= i + kv_len - qo_len for its i-th query token. A softmax over a joined
// sequence folds from its parts: with each part's sum l, reference point m and
// output o (normalised), weights 2^(lse - max lse), lse = m + log2 l. So the prefix's
// K/V are walked once with the rows of every request as columns of one product,
// each request's own tokens with its rows alone, and a second launch folds.
//
// Units: the prefix (where the batch has at most 64 packed rows a kv head) and then
// the requests' own tokens form one stream, cut into units of equal length, one
// workgroup each; a wave has one kv head, so a workgroup reads whole token rows.
// A wave walks its piece 16 tokens a step on the matrix cores: S^T = K Q^T, then
// O^T += V^T P^T, whose operand P^T is S^T's accumulator layout, for up to four
// column blocks of 16 rows per K/V read. Both put the row on the lane's column, so
// the running maximum and sum are lane-local but for one exchange across four lane
// groups. K and V of the next step are in flight during a step.
#include <math.h>

#include "common.h"
#include "prefill_impl.h"

namespace sgl {
namespace {

constexpr int kD = 128;
constexpr int kStep = 16;                 // tokens a step
constexpr int kMinUnit = 16;              // shortest unit
constexpr int kQPitch = kD + 8;           // LDS row pitch (bf16) of the Q^T copy
constexpr float kRescaleSlack = 8.f;      // log2 units: p <= 256 between rescales
constexpr int kMaxTileRows = 64;

struct PrefixArgs {
  const uint16_t* q;
  int64_t q_st, q_sh;
  const uint16_t* kc;
  const uint16_t* vc;
  int64_t kv_ss, kv_sh;
  const int32_t* pidx;
  const int32_t* indices;
  const int32_t* kv_indptr;
  const int32_t* qo_indptr;
  int batch, tokens, hq, hkv, group;
  int prefix, tile_rows, tiles, units, max_qo;
  int shares, row_tiles;  // of the prefix's own launch: item = row tile, then kv head, then share
  float scale_log2;
  uint16_t* o;
  int64_t o_st, o_sh;
  // Partial outputs (fp32 [.., 128]) and log2-sum-exp. Prefix pieces: unit u's,
  // [u][kv head][packed row], or [share][kv head][packed row]. Own pieces: [token slot][q head], the piece a
  // request starts with at its rows' own tokens, the one running into unit u from
  // before it at tokens + u max_qo + i.
  float* p_o;
  float* p_lse;
  float* s_o;
  float* s_lse;
};

// The stream's places are below 2^30 (prefix) + 2^31 (the offsets are int32): 32 bits
// without a sign.
// Tokens of a unit, from the requests' lengths as they are now.
__device__ __forceinline__ uint32_t unit_tokens(const PrefixArgs& a, uint32_t all) {
  const uint32_t w = all / static_cast<uint32_t>(a.units) + 1;  // one more where it divides
  return max((w + kStep - 1) / kStep * kStep, static_cast<uint32_t>(kMinUnit));
}

__device__ __forceinline__ uint32_t own_tokens(const PrefixArgs& a) {
  return static_cast<uint32_t>(max(a.kv_indptr[a.batch] - max(a.kv_indptr[0], 0), 0));
}

struct Request {
  int q0, qo, kv0, kv;  // first query token, query tokens, first own index, own tokens
  bool ok;
};

__device__ __forceinline__ Request request_of(const PrefixArgs& a, int r) {
  Request x;
  x.q0 = a.qo_indptr[r];
  const int64_t q1 = a.qo_indptr[r + 1];
  x.kv0 = a.kv_indptr[r];
  const int64_t k1 = a.kv_indptr[r + 1];
  x.qo = static_cast<int>(q1 - x.q0);
  x.kv = static_cast<int>(k1 - x.kv0);
  // Rows and pieces of anything else have no place in the outputs and the workspace.
  x.ok = x.kv0 >= 0 && x.q0 >= max(a.qo_indptr[0], 0) && q1 >= x.q0 && q1 <= min(a.qo_indptr[a.batch], a.tokens) &&
         q1 - x.q0 <= a.max_qo && x.kv0 >= a.kv_indptr[0] && k1 >= x.kv0 && k1 <= a.kv_indptr[a.batch];
  return x;
}

__device__ __forceinline__ bf16x8_t as_bf16x8(const u32x4_t& v) {
  return __builtin_bit_cast(bf16x8_t, v);
}

__device__ __forceinline__ void wave_lds_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

__device__ __forceinline__ const char* slot_row(const char* base, int slot, uint32_t ss_bytes) {
  return base + static_cast<uint64_t>(static_cast<uint32_t>(slot)) * ss_bytes;
}

// A operand of O^T product nb: V^T[d = 8 n + nb][token 4 j + e], e < 4, from four rows.
template <int nb>
__device__ __forceinline__ bf16x4_t v_operand(const u32x4_t (&vr)[4]) {
  constexpr int w = nb / 2;
  constexpr uint32_t sel = (nb & 1) ? 0x07060302u : 0x05040100u;
  u32x2_t out;
  out[0] = __builtin_amdgcn_perm(vr[1][w], vr[0][w], sel);
  out[1] = __builtin_amdgcn_perm(vr[3][w], vr[2][w], sel);
  return __builtin_bit_cast(bf16x4_t, out);
}

// One wave: kv head h over the len tokens of slots idx[0, len), for the packed
// rows [row0, row_end) (at most 16 RB; row p: token tok0 + p / G, head h G + p % G).
// Row of token i sees the tokens below sees0 + i (all of them: sees0 >= len).
// Its output and lse go to row out0 + (p - row0) of o/lse, or, with by_token, to
// row (out0 + i) hq + head. lq: the wave's Q copy, 16 RB rows.
// Lane (n, j), n = lane % 16: token n (K), chunk n of tokens 4 j + e (V), row n
// (S, O).
template <int RB>
__device__ __forceinline__ void walk(const PrefixArgs& a, uint16_t* lq, const int32_t* idx, int len,
                                     int h, int tok0, int row0, int row_end, int sees0, float* o,
                                     float* lse, int64_t out0, bool by_token, int lane) {
  const int n = lane & 15, j = lane >> 4;
  const int G = a.group;
  const uint32_t ss_bytes = static_cast<uint32_t>(a.kv_ss * 2);
  const char* klane = reinterpret_cast<const char*>(a.kc + h * a.kv_sh + 8 * j);
  const char* vlane = reinterpret_cast<const char*>(a.vc + h * a.kv_sh + 8 * n);

  auto load_k = [&](int slot, u32x4_t (&kr)[4]) {
    const char* row = slot_row(klane, slot, ss_bytes);
#pragma unroll
    for (int s = 0; s < 4; ++s) kr[s] = ldg128(row + 64 * s);
  };
  auto load_v = [&](int slot, u32x4_t (&vr)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      vr[e] = ldg128_nt<true>(slot_row(vlane, __shfl(slot, 4 * j + e, kWave), ss_bytes));
  };

  // Token i and head of packed row p = row0 + x, x < 64: i0 + (rem + x) / G, the
  // division (of a number below 128 by G <= 64) as a product.
  const int i0 = row0 / G, rem = row0 - i0 * G;
  const uint32_t inv_g = (65536u + G - 1) / G;
  auto token_of = [&](int x, int& head) {
    const int y = rem + x;
    const int d = static_cast<int>(static_cast<uint32_t>(y) * inv_g >> 16);
    head = h * G + (y - d * G);
    return i0 + d;
  };
  const int nrows = row_end - row0;

  const int slot = idx[min(n, len - 1)];
  int slot_next = idx[min(kStep + n, len - 1)];
  // Q rows, four of a block at a time (chunk n); rows past the last one read it again
  // and are cleared, so that every load is in flight at once.
  u32x4_t qv[4 * RB];
#pragma unroll
  for (int u = 0; u < 4 * RB; ++u) {
    int head;
    const int i = token_of(min(4 * u + j, nrows - 1), head);
    qv[u] = ldg128(a.q + (tok0 + i) * a.q_st + head * a.q_sh + 8 * n);
  }
  u32x4_t kr[4], vr[4];
  load_k(slot, kr);
  load_v(slot, vr);
#pragma unroll
  for (int u = 0; u < 4 * RB; ++u)
    *reinterpret_cast<u32x4_t*>(lq + (4 * u + j) * kQPitch + 8 * n) =
        4 * u + j < nrows ? qv[u] : u32x4_t{0, 0, 0, 0};
  wave_lds_sync();
  int sees[RB];
  float m[RB], l[RB];
  f32x4_t acc[RB][8];
#pragma unroll
  for (int b = 0; b < RB; ++b) {
    int head;
    const int i = token_of(16 * b + n, head);
    sees[b] = 16 * b + n < nrows ? min(sees0 + i, len) : 0;
    m[b] = -INFINITY;
    l[b] = 0.f;
#pragma unroll
    for (int nb = 0; nb < 8; ++nb) acc[b][nb] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }

  for (int t = 0; t < len; t += kStep) {
    // The workgroup's waves (its kv heads) keep in step: together they read
    // whole token rows.
    __builtin_amdgcn_s_barrier();
    const int slot_after = idx[min(t + 2 * kStep + n, len - 1)];
    f32x4_t sacc[RB];
#pragma unroll
    for (int b = 0; b < RB; ++b) {
      sacc[b] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const bf16x8_t qop =
            *reinterpret_cast<const bf16x8_t*>(lq + (16 * b + n) * kQPitch + 32 * s + 8 * j);
        sacc[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(kr[s]), qop, sacc[b], 0, 0, 0);
      }
    }
    load_k(slot_next, kr);
    bf16x4_t pop[RB];
#pragma unroll
    for (int b = 0; b < RB; ++b) {
      float sc[4];
      float mt = -INFINITY;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        sc[i] = t + 4 * j + i < sees[b] ? sacc[b][i] : -INFINITY;
        mt = fmaxf(mt, sc[i]);
      }
      // The reference point moves only where a row's maximum exceeds it by
      // more than kRescaleSlack; p and l always use the same one, so the result
      // is exact and most steps leave O as it is.
      mt = max_xor32(max_xor16(mt)) * a.scale_log2;
      const bool move = mt > m[b] + kRescaleSlack;
      if (__builtin_amdgcn_ballot_w64(move) != 0) {
        const float mn = move ? mt : m[b];
        const float alpha = move ? __builtin_amdgcn_exp2f(m[b] - mn) : 1.f;
        l[b] *= alpha;
        m[b] = mn;
#pragma unroll
        for (int nb = 0; nb < 8; ++nb) acc[b][nb] *= alpha;
      }
      const float neg_m = m[b] == -INFINITY ? 0.f : -m[b];  // nothing seen yet
      float p[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) p[i] = __builtin_amdgcn_exp2f(fmaf(sc[i], a.scale_log2, neg_m));
      l[b] += (p[0] + p[1]) + (p[2] + p[3]);
      // P in bf16, the product's operand type: a weight is off by at most 2^-9 of
      // itself, below what rounding the output to bf16 takes.
      const u32x2_t pw = {pack_bf16x2(p[0], p[1]), pack_bf16x2(p[2], p[3])};
      pop[b] = __builtin_bit_cast(bf16x4_t, pw);
    }
    static_for<0, 8>([&](auto NB) {
      constexpr int nb = decltype(NB)::value;
      const bf16x4_t vop = v_operand<nb>(vr);
#pragma unroll
      for (int b = 0; b < RB; ++b)
        acc[b][nb] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(vop, pop[b], acc[b][nb], 0, 0, 0);
    });
    load_v(slot_next, vr);
    slot_next = slot_after;
  }
#pragma unroll
  for (int b = 0; b < RB; ++b) {
    const float sum = sum_xor32(sum_xor16(l[b]));
    if (16 * b + n >= nrows) continue;
    int head;
    const int i = token_of(16 * b + n, head);
    const int64_t row = by_token ? (out0 + i) * a.hq + head : out0 + 16 * b + n;
    const float inv = sum == 0.f ? 0.f : 1.0f / sum;  // a NaN sum stays one
    // acc[nb][c] holds d = 32 j + 8 c + nb.
    float* op = o + row * kD + 32 * j;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      f32x4_t lo, hi;
#pragma unroll
      for (int nb = 0; nb < 4; ++nb) lo[nb] = acc[b][nb][c] * inv, hi[nb] = acc[b][nb + 4][c] * inv;
      *reinterpret_cast<f32x4_t*>(op + 8 * c) = lo;
      *reinterpret_cast<f32x4_t*>(op + 8 * c + 4) = hi;
    }
    if (j == 0) lse[row] = sum == 0.f ? -INFINITY : m[b] + log2f(sum);
  }
}

// The walk with as many column blocks as the rows need.
template <int RB>
__device__ __forceinline__ void walk_rows(const PrefixArgs& a, uint16_t* lq, const int32_t* idx, int len,
                                          int h, int tok0, int row0, int row_end, int sees0, float* o,
                                          float* lse, int64_t out0, bool by_token, int lane) {
  if constexpr (RB > 1) {
    if (row_end - row0 <= 8 * RB) {
      walk_rows<RB / 2>(a, lq, idx, len, h, tok0, row0, row_end, sees0, o, lse, out0, by_token, lane);
      return;
    }
  }
  walk<RB>(a, lq, idx, len, h, tok0, row0, row_end, sees0, o, lse, out0, by_token, lane);
}

template <int RB>
__global__ void __launch_bounds__(512) prefix_units_kernel(PrefixArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint16_t lds_q[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int h = blockIdx.y * (blockDim.x >> 6) + wave;
  const uint32_t u = blockIdx.x;
  uint16_t* lq = lds_q + wave * 16 * RB * kQPitch;
  const uint32_t shared = a.tiles > 0 ? a.prefix : 0;
  const uint32_t all = shared + own_tokens(a);
  const uint32_t W = unit_tokens(a, all);
  if (static_cast<uint64_t>(u) * W >= all) return;
  const uint32_t t0 = u * W, t1 = min(all, t0 + W);
  // The shared prefix's part.
  if (t0 < shared) {
    const int first = max(a.qo_indptr[0], 0);
    const int last = min(a.qo_indptr[a.batch], a.tokens);
    const int rows = min(max(last - first, 0) * a.group, a.tile_rows);
    const int len = static_cast<int>(min(t1, shared) - t0);
    if (rows > 0)
      walk_rows<RB>(a, lq, a.pidx + t0, len, h, first, 0, rows, len, a.p_o, a.p_lse,
                    (static_cast<int64_t>(u) * a.hkv + h) * a.tile_rows, false, lane);
  }
  if (t1 <= shared) return;
  // The requests' own tokens [b0, b1) of the joined list.
  const int kv_first = max(a.kv_indptr[0], 0);
  const uint32_t b0 = max(t0, shared) - shared, b1 = t1 - shared;
  int r = 0;  // requests that end at or before b0, 64 at a time
  for (int at = 0; at < a.batch; at += kWave) {
    const int e = at + lane;
    const bool before = e < a.batch && a.kv_indptr[e + 1] - kv_first <= static_cast<int64_t>(b0);
    const uint64_t mask = __builtin_amdgcn_ballot_w64(before);
    r += __builtin_popcountll(mask);
    if (mask != ~0ull) break;
  }
  for (; r < a.batch; ++r) {
    const Request x = request_of(a, r);
    const int64_t rb = static_cast<int64_t>(x.kv0) - kv_first;
    if (rb >= b1) break;
    if (!x.ok || x.qo == 0 || x.kv == 0) continue;
    const int s0 = static_cast<int>(max(b0 - rb, int64_t{0}));
    const int s1 = static_cast<int>(min(b1 - rb, static_cast<int64_t>(x.kv)));
    if (s1 <= s0) continue;
    const int64_t out0 = s0 == 0 ? x.q0 : a.tokens + static_cast<int64_t>(u) * a.max_qo;
    for (int row0 = 0; row0 < x.qo * a.group; row0 += 16 * RB)
      walk_rows<RB>(a, lq, a.indices + x.kv0 + s0, s1 - s0, h, x.q0, row0,
                    min(x.qo * a.group, row0 + 16 * RB), max(x.kv - x.qo + 1 - s0, -x.qo), a.s_o,
                    a.s_lse, out0, true, lane);
  }
}

// The prefix for many rows: W waves with 32 packed rows each share the 64-token K/V
// tiles that they gather into LDS (two buffers, K one tile ahead of V), and tile t + 1's
// scores are on the matrix cores while tile t's become weights; the prefill kernel's
// tile steps without a causal bound. Item: (row tile, kv head, share of the prefix's
// tiles). Bound by the matrix cores: 4 x 64 x 128 flops a row and tile.
template <int W>
__device__ __forceinline__ void prefix_item(const PrefixArgs& a, char* lds_raw, int item) {
  using namespace pf;
  const int per_tile = a.hkv * a.shares;
  const int rt = item / per_tile;
  const int hs = item - rt * per_tile;
  const int h = hs % a.hkv, share = hs / a.hkv;
  const int first = max(a.qo_indptr[0], 0);
  const int last = min(a.qo_indptr[a.batch], a.tokens);
  const int rows = max(last - first, 0) * a.group;
  const int row0 = rt * 32 * W;
  if (row0 >= rows) return;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tid = threadIdx.x;
  const int c = lane & 31, hl = lane >> 5;
  const int prow = row0 + 32 * wave + c;
  const bool row_ok = prow < rows;
  const bool works = row0 + 32 * wave < rows;  // the others only gather
  const int safe = row_ok ? prow : row0;
  const int qtok = safe / a.group;
  const int qhead = h * a.group + (safe - qtok * a.group);
  const int nt = (a.prefix + kBN - 1) / kBN;
  const int per = (nt + a.shares - 1) / a.shares;
  const int tb = share * per, te = min(nt, tb + per);
  if (tb >= te) return;
  const int kv_len = a.prefix;

  Tile* tiles = reinterpret_cast<Tile*>(lds_raw);
  const uint16_t* kbase = a.kc + h * a.kv_sh;
  const uint16_t* vbase = a.vc + h * a.kv_sh;
  const uint32_t ss_bytes = static_cast<uint32_t>(a.kv_ss * 2);
  const int lch0 = (lane & 15) ^ swz(4 * wave + (lane >> 4));
  const int lch1 = (lane & 15) ^ swz((4 * wave + (lane >> 4) + 8) & 15);
  const char* const klane[2] = {reinterpret_cast<const char*>(kbase) + lch0 * 16,
                                reinterpret_cast<const char*>(kbase) + lch1 * 16};
  const char* const vlane[2] = {reinterpret_cast<const char*>(vbase) + lch0 * 16,
                                reinterpret_cast<const char*>(vbase) + lch1 * 16};
  LaneAddr la;
  {
    const uint32_t base = lds_addr(tiles);
    const int sw = swz(c);
#pragma unroll
    for (int s = 0; s < 8; ++s) la.k[s] = base + c * pf::kD * 2 + ((2 * s + hl) ^ sw) * 16;
    const int vrow = 4 * (lane >> 5) + ((lane & 15) >> 2);
    const int g = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
      for (int hi = 0; hi < 2; ++hi) {
        const int row = vrow + 8 * hi;
        la.v[2 * db + hi] = base + kVOffset + row * pf::kD * 2 + ((4 * db + g) ^ swz(row)) * 16 + 8 * (lane & 1);
      }
  }
  PrefillArgs pa{};
  pa.scale_log2 = a.scale_log2;
  RowState rs;
#pragma unroll
  for (int db = 0; db < 4; ++db)
#pragma unroll
    for (int v = 0; v < 16; ++v) rs.acc[db][v] = 0.f;
  rs.m = -INFINITY;
  rs.l = 0.f;

  int32_t sl_k[16 / W], sl_v[16 / W];
  load_slots<W>(a.pidx, tb * kBN, kv_len, tid, sl_k);
  load_slots<W>(a.pidx, (tb + 1) * kBN, kv_len, tid, sl_v);
  wait_gathers();
  issue_half<W>(klane, ss_bytes, sl_k, tiles[0].k, wave);
  issue_half<W>(vlane, ss_bytes, sl_k, tiles[0].v, wave);
  if (tb + 1 < te) issue_half<W>(klane, ss_bytes, sl_v, tiles[1].k, wave);
  load_slots<W>(a.pidx, (tb + 2) * kBN, kv_len, tid, sl_k);
  bf16x8_t qop[8];
  {
    const uint16_t* qp = a.q + static_cast<int64_t>(first + qtok) * a.q_st + static_cast<int64_t>(qhead) * a.q_sh;
    u32x4_t qv[8];
#pragma unroll
    for (int s = 0; s < 8; ++s) qv[s] = ldg128(qp + 16 * s + 8 * hl);
#pragma unroll
    for (int s = 0; s < 8; ++s) qop[s] = pf::as_bf16x8(row_ok ? qv[s] : u32x4_t{0, 0, 0, 0});
  }
  wait_gathers();
  __syncthreads();
  f32x16_t s_a[2], s_b[2];
  bf16x8_t pop[4];
  qk_tile<0>(la, qop, s_a);
  __syncthreads();  // every wave has read K(0) before K(2) overwrites it
  auto step = [&](auto B, int t, f32x16_t(&s_cur)[2], f32x16_t(&s_next)[2]) {
    constexpr int buf = decltype(B)::value;  // (t - tb) % 2
    if (t + 2 < te) issue_half<W>(klane, ss_bytes, sl_k, tiles[buf].k, wave);
    if (t + 1 < te) issue_half<W>(vlane, ss_bytes, sl_v, tiles[buf ^ 1].v, wave);
#pragma unroll
    for (int u = 0; u < 16 / W; ++u) sl_v[u] = sl_k[u];
    load_slots<W>(a.pidx, (t + 3) * kBN, kv_len, tid, sl_k);
    if (works) {
      u32x4_t kb[16];
      qk_tile_prefetch<buf ^ 1>(la, kb);
      softmax_head(pa, s_cur, rs, t * kBN, kv_len, kv_len - 1, kv_len, hl);
      lgkm_wait<0>(kb[kKAhead - 1]);
      u32x2_t vr[4][8];
      qk_tile_run<buf ^ 1>(la, qop, s_next, kb);  // S(t + 1); unused after the last tile
      softmax_exp_half<0>(pa, s_cur, rs, pop);
      pv_reads<buf, 0>(la, vr[0]);
      pv_steps<buf, 0, 2>(la, pop, vr, rs);
      softmax_exp_half<1>(pa, s_cur, rs, pop);
      pv_steps<buf, 2, 4>(la, pop, vr, rs);
    }
    wait_gathers();
    __syncthreads();
  };
  for (int t = tb; t < te; t += 2) {
    step(std::integral_constant<int, 0>{}, t, s_a, s_b);
    if (t + 1 >= te) break;
    step(std::integral_constant<int, 1>{}, t + 1, s_b, s_a);
  }
  const float l = sum_xor32(rs.l);
  if (!row_ok) return;
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  const int64_t row = (static_cast<int64_t>(share) * a.hkv + h) * (static_cast<int64_t>(a.tokens) * a.group) + prow;
  float* op = a.p_o + row * sgl::kD;
#pragma unroll
  for (int db = 0; db < 4; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<f32x4_t*>(op + 32 * db + 8 * g + 4 * hl) =
          f32x4_t{rs.acc[db][4 * g] * inv, rs.acc[db][4 * g + 1] * inv, rs.acc[db][4 * g + 2] * inv,
                  rs.acc[db][4 * g + 3] * inv};
  if (hl == 0) a.p_lse[row] = l == 0.f ? -INFINITY : rs.m + log2f(l);
}

template <int W>
__global__ void __launch_bounds__(64 * W, 8 / W) prefix_rows_kernel(PrefixArgs a) {
  __shared__ __attribute__((aligned(16))) char lds_raw[2 * pf::kTileBytes];
  prefix_item<W>(a, lds_raw, blockIdx.x);
}

// Sum over the 32 lanes of a half wave, the same in each.
__device__ __forceinline__ float half_sum(float x) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) x += __shfl_xor(x, off, kWave);
  return x;
}

// The row again, token by token over those it sees, by 32 lanes (4 values each):
// for rows that do not see the whole prefix, and for those whose products brought in
// a V value that is not finite from a token they do not see (0 x inf).
__device__ __forceinline__ f32x4_t plain_row(const PrefixArgs& a, const Request& x, int tok, int head,
                                             int64_t sees, int c) {
  const int h = head / a.group;
  const u32x2_t qw = *reinterpret_cast<const u32x2_t*>(a.q + tok * a.q_st + head * a.q_sh + 4 * c);
  const float q[4] = {bf16_lo(qw[0]), bf16_hi(qw[0]), bf16_lo(qw[1]), bf16_hi(qw[1])};
  float m = -INFINITY, l = 0.f;
  f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
  for (int64_t t = 0; t < sees; ++t) {
    const int64_t slot = static_cast<uint32_t>(t < a.prefix ? a.pidx[t] : a.indices[x.kv0 + (t - a.prefix)]);
    const u32x2_t kw = *reinterpret_cast<const u32x2_t*>(a.kc + slot * a.kv_ss + h * a.kv_sh + 4 * c);
    const u32x2_t vw = *reinterpret_cast<const u32x2_t*>(a.vc + slot * a.kv_ss + h * a.kv_sh + 4 * c);
    float s = q[0] * bf16_lo(kw[0]) + q[1] * bf16_hi(kw[0]) + q[2] * bf16_lo(kw[1]) + q[3] * bf16_hi(kw[1]);
    s = half_sum(s) * a.scale_log2;
    const float mn = fmaxf(m, s);
    const float alpha = m == -INFINITY ? 0.f : exp2f(m - mn);
    const float p = s == -INFINITY ? 0.f : exp2f(s - mn);  // NaN stays NaN
    l = l * alpha + p;
    const f32x4_t v = {bf16_lo(vw[0]), bf16_hi(vw[0]), bf16_lo(vw[1]), bf16_hi(vw[1])};
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = acc[i] * alpha + p * v[i];
    m = mn;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  return acc * inv;
}

// Folds the pieces of each row: kSets groups of 32 lanes take them in turn, four
// pieces' loads in flight, and are folded through LDS; 8 / kSets heads of one token a
// workgroup.
template <int kSets>
__global__ void __launch_bounds__(256) prefix_fold_kernel(PrefixArgs a, int head_groups) {
  constexpr int kRows = 8 / kSets;
  __shared__ int before[4];
  __shared__ float xch[6][8][32];
  const int t = blockIdx.x / static_cast<uint32_t>(head_groups);
  const int lane = threadIdx.x & 63;
  // The token's request: those that end at or before it are counted.
  int n = 0;
  for (int e = threadIdx.x; e < a.batch; e += 256) n += a.qo_indptr[e + 1] <= t;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) n += __shfl_xor(n, off, kWave);
  if (lane == 0) before[threadIdx.x >> 6] = n;
  __syncthreads();
  const int r = before[0] + before[1] + before[2] + before[3];
  if (r >= a.batch || t < a.qo_indptr[0]) return;  // no request's row: left as it was
  const Request x = request_of(a, r);
  const int first = max(a.qo_indptr[0], 0);
  const int P = a.prefix;
  const uint32_t shared = a.tiles > 0 ? P : 0;
  const uint32_t W = unit_tokens(a, shared + own_tokens(a));
  const int c = threadIdx.x & 31, group = threadIdx.x >> 5;
  const int set = group % kSets;
  const int head = (blockIdx.x - t * head_groups) * kRows + group / kSets;
  const bool head_ok = head < a.hq;
  const int hh = head_ok ? head : a.hq - 1;
  const int h = hh / a.group;
  const int i = t - x.q0;
  const int64_t sees = static_cast<int64_t>(P) + x.kv - x.qo + i + 1;  // tokens this row sees, prefix first
  float m = -INFINITY, l = 0.f;
  f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
  const bool folded = x.ok && sees >= P;
  if (folded) {
    // Prefix pieces [0, np) at p0 + k p_step, then the request's own.
    int np = 0, ns = 0;
    int64_t p0 = 0, s1 = 0;
    int64_t p_step = static_cast<int64_t>(a.hkv) * a.tile_rows;
    const int prow = (t - first) * a.group + hh - h * a.group;
    if (P > 0 && a.shares > 0) {
      np = a.shares;
      p_step = static_cast<int64_t>(a.hkv) * a.tokens * a.group;
      p0 = static_cast<int64_t>(h) * a.tokens * a.group + prow;
    } else if (P > 0) {
      np = static_cast<int>((P - 1) / W) + 1;
      p0 = static_cast<int64_t>(h) * a.tile_rows + prow;
    }
    if (x.kv > 0) {
      const uint32_t own0 = shared + (x.kv0 - max(a.kv_indptr[0], 0)), u0 = own0 / W;
      ns = static_cast<int>((own0 + x.kv - 1) / W - u0) + 1;
      s1 = (a.tokens + static_cast<int64_t>(u0) * a.max_qo + i) * a.hq + hh;
    }
    const int64_t s0 = static_cast<int64_t>(t) * a.hq + hh, s_step = static_cast<int64_t>(a.max_qo) * a.hq;
    for (int k0 = set; k0 < np + ns; k0 += 4 * kSets) {
      f32x4_t v[4];
      float lse[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int k = min(k0 + e * kSets, np + ns - 1);
        const int64_t row = k < np ? p0 + k * p_step : k == np ? s0 : s1 + (k - np) * s_step;
        v[e] = *reinterpret_cast<const f32x4_t*>((k < np ? a.p_o : a.s_o) + row * kD + 4 * c);
        lse[e] = (k < np ? a.p_lse : a.s_lse)[row];
        if (k0 + e * kSets >= np + ns) lse[e] = -INFINITY;
      }
      float mn = m;
#pragma unroll
      for (int e = 0; e < 4; ++e) mn = fmaxf(mn, lse[e]);
      const float alpha = m == -INFINITY ? 0.f : exp2f(m - mn);
      l *= alpha;
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[k] *= alpha;
      m = mn;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (lse[e] == -INFINITY) continue;  // nothing seen there: its values do not count
        const float w = exp2f(lse[e] - mn);
        l += w;
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[k] += v[e][k] * w;
      }
    }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) xch[k][group][c] = acc[k];
  xch[4][group][c] = m;
  xch[5][group][c] = l;
  __syncthreads();
  if (set != 0 || !head_ok) return;
  if (!x.ok) {
    acc = f32x4_t{NAN, NAN, NAN, NAN};
  } else if (!folded) {
    acc = plain_row(a, x, t, head, sees, c);
  } else {
#pragma unroll
    for (int e = 1; e < kSets; ++e) m = fmaxf(m, xch[4][group + e][c]);
    l = 0.f;
    acc = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < kSets; ++e) {
      const float me = xch[4][group + e][c], le = xch[5][group + e][c];
      if (le == 0.f) continue;  // no piece with a weight
      const float w = exp2f(me - m);
      l += le * w;
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[k] += xch[k][group + e][c] * w;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int k = 0; k < 4; ++k) acc[k] *= inv;
    // Tokens of the request behind this row's last one may have brought in
    // values that are not finite.
    bool bad = false;
#pragma unroll
    for (int k = 0; k < 4; ++k) bad = bad || !(fabsf(acc[k]) < INFINITY);
    const uint64_t any = __builtin_amdgcn_ballot_w64(bad);
    if (i + 1 < x.qo && ((any >> (lane & 32)) & 0xffffffffull) != 0)
      acc = plain_row(a, x, t, head, sees, c);
  }
  *reinterpret_cast<u32x2_t*>(a.o + t * a.o_st + head * a.o_sh + 4 * c) =
      u32x2_t{pack_bf16x2(acc[0], acc[1]), pack_bf16x2(acc[2], acc[3])};
}

int device_cus() {
  int dev = 0, cus = 0;
  if (hipGetDevice(&dev) == hipSuccess &&
      hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) == hipSuccess && cus > 0)
    return cus;
  return 256;
}

// kv heads of a workgroup: the largest divisor of theirs up to 8.
int heads_per_group(int hkv) {
  for (int n = 8; n > 1; --n)
    if (hkv % n == 0) return n;
  return 1;
}

struct Layout {
  int64_t p_o, p_lse, s_o, s_lse, total;
};

Layout workspace_layout(const sgl_prefix_plan_t& p) {
  auto align = [](int64_t x) { return (x + 255) / 256 * 256; };
  const int64_t prefix_rows = p.num_tiles > 0
      ? static_cast<int64_t>(p.num_units) * p.num_kv_heads * p.tile_rows
      : static_cast<int64_t>(p.num_shares) * p.max_tokens * p.num_qo_heads;
  const int64_t own_rows =
      (p.max_tokens + static_cast<int64_t>(p.num_units) * p.max_qo_len) * p.num_qo_heads;
  Layout l;
  l.p_o = 0;
  l.p_lse = l.p_o + align(prefix_rows * kD * 4);
  l.s_o = l.p_lse + align(prefix_rows * 4);
  l.s_lse = l.s_o + align(own_rows * kD * 4);
  l.total = l.s_lse + align(own_rows * 4);
  return l;
}

}  // namespace
}  // namespace sgl

using namespace sgl;

extern "C" int sgl_prefix_plan(int prefix_len, int batch_size, int max_tokens, int max_qo_len,
                               int num_qo_heads, int num_kv_heads, int head_dim,
                               sgl_prefix_plan_t* plan) {
  if (!plan || prefix_len < 0 || batch_size < 0 || max_tokens < 0 || max_qo_len < 0 ||
      num_qo_heads <= 0 || num_kv_heads <= 0 || num_qo_heads % num_kv_heads != 0)
    return SGL_ERR_INVALID_ARG;
  const int group = num_qo_heads / num_kv_heads;
  if (head_dim != kD || group > kMaxTileRows || max_qo_len > SGL_PREFIX_MAX_QO ||
      num_kv_heads > 65535)
    return SGL_ERR_UNSUPPORTED;
  // Packed rows and their tiles are counted in 32 bits.
  if (static_cast<int64_t>(max_tokens) * group > (1 << 30) || prefix_len > (1 << 30))
    return SGL_ERR_UNSUPPORTED;
  *plan = sgl_prefix_plan_t{};
  plan->prefix_len = prefix_len;
  plan->batch_size = batch_size;
  plan->max_tokens = max_tokens;
  plan->max_qo_len = max_qo_len;
  plan->num_qo_heads = num_qo_heads;
  plan->num_kv_heads = num_kv_heads;
  plan->head_dim = head_dim;
  const int64_t units = static_cast<int64_t>(device_cus()) * 8 / num_kv_heads;
  plan->num_units = static_cast<int32_t>(units < 1 ? 1 : units);
  const int64_t rows = static_cast<int64_t>(max_tokens) * group;
  if (prefix_len > 0 && rows > 0) {
    if (rows <= kMaxTileRows) {  // the units walk the prefix
      plan->tile_rows = static_cast<int32_t>((rows + 15) / 16 * 16);
      plan->num_tiles = 1;
    } else {
      // A launch of its own: the shares whose items, all rounds together, walk the
      // fewest tiles one after the other (two for an item's start and its states).
      plan->tile_rows = rows <= 128 ? 128 : 256;
      const int64_t slots = device_cus() * (256 / plan->tile_rows);
      const int64_t per_share = (rows + plan->tile_rows - 1) / plan->tile_rows * num_kv_heads;
      const int64_t nt = (prefix_len + pf::kBN - 1) / pf::kBN;
      int64_t best = 0, shares = 1;
      for (int64_t n = 1; n <= nt && (n == 1 || (n - 1) * per_share < 4 * slots); ++n) {
        const int64_t per = (nt + n - 1) / n, used = (nt + per - 1) / per;
        if (used != n) continue;
        const int64_t cost = (n * per_share + slots - 1) / slots * (per + 2);
        if (best == 0 || cost < best) best = cost, shares = n;
      }
      plan->num_shares = static_cast<int32_t>(shares);
    }
  }
  plan->workspace_bytes = workspace_layout(*plan).total;
  return SGL_OK;
}

extern "C" int sgl_prefix_attention(const sgl_prefix_plan_t* plan, const void* q,
                                    int64_t q_stride_token, int64_t q_stride_head,
                                    const void* k_cache, const void* v_cache,
                                    int64_t kv_stride_slot, int64_t kv_stride_head,
                                    const int32_t* prefix_indices, const int32_t* indices,
                                    const int32_t* kv_indptr, const int32_t* qo_indptr,
                                    int batch_size, int max_tokens, int num_qo_heads,
                                    int num_kv_heads, int head_dim, float sm_scale, void* o,
                                    int64_t o_stride_token, int64_t o_stride_head, void* workspace,
                                    int64_t workspace_bytes, void* stream) {
  if (!plan || batch_size < 0 || max_tokens < 0) return SGL_ERR_INVALID_ARG;
  if (num_qo_heads != plan->num_qo_heads || num_kv_heads != plan->num_kv_heads ||
      head_dim != plan->head_dim)
    return SGL_ERR_INVALID_ARG;
  // A plan as sgl_prefix_plan makes it.
  sgl_prefix_plan_t p;
  int st = sgl_prefix_plan(plan->prefix_len, plan->batch_size, plan->max_tokens, plan->max_qo_len,
                           num_qo_heads, num_kv_heads, head_dim, &p);
  if (st != SGL_OK) return st;
  p.num_units = plan->num_units;
  if (p.num_units <= 0 || p.num_units > (1 << 20) || plan->tile_rows != p.tile_rows ||
      plan->num_tiles != p.num_tiles || plan->num_shares != p.num_shares)
    return SGL_ERR_INVALID_ARG;
  if (batch_size > p.batch_size || max_tokens > p.max_tokens) return SGL_ERR_CAPACITY;
  if (batch_size == 0 || max_tokens == 0) return SGL_OK;
  if (!q || !k_cache || !v_cache || !kv_indptr || !qo_indptr || !o ||
      (p.prefix_len > 0 && !prefix_indices))
    return SGL_ERR_INVALID_ARG;
  // Slot addresses use 32-bit byte strides.
  if (kv_stride_slot <= 0 || kv_stride_slot > 0x3fffffff) return SGL_ERR_UNSUPPORTED;
  if (q_stride_head % 8 || q_stride_token % 8 || kv_stride_slot % 8 || kv_stride_head % 8 ||
      o_stride_token % 8 || o_stride_head % 8 || !aligned16(q) || !aligned16(k_cache) ||
      !aligned16(v_cache) || !aligned16(o) || !aligned16(workspace))
    return SGL_ERR_ALIGNMENT;
  const Layout l = workspace_layout(p);
  if (!workspace || workspace_bytes < l.total) return SGL_ERR_CAPACITY;
  char* ws = static_cast<char*>(workspace);
  PrefixArgs a{};
  a.q = static_cast<const uint16_t*>(q), a.q_st = q_stride_token, a.q_sh = q_stride_head;
  a.kc = static_cast<const uint16_t*>(k_cache), a.vc = static_cast<const uint16_t*>(v_cache);
  a.kv_ss = kv_stride_slot, a.kv_sh = kv_stride_head;
  a.pidx = prefix_indices, a.indices = indices, a.kv_indptr = kv_indptr, a.qo_indptr = qo_indptr;
  a.batch = batch_size, a.tokens = max_tokens;
  a.hq = num_qo_heads, a.hkv = num_kv_heads, a.group = num_qo_heads / num_kv_heads;
  a.prefix = p.prefix_len, a.tile_rows = p.tile_rows, a.units = p.num_units, a.max_qo = p.max_qo_len;
  a.scale_log2 = sm_scale * 1.4426950408889634f;
  a.o = static_cast<uint16_t*>(o), a.o_st = o_stride_token, a.o_sh = o_stride_head;
  a.p_o = reinterpret_cast<float*>(ws + l.p_o), a.p_lse = reinterpret_cast<float*>(ws + l.p_lse);
  a.s_o = reinterpret_cast<float*>(ws + l.s_o), a.s_lse = reinterpret_cast<float*>(ws + l.s_lse);
  const int64_t rows = static_cast<int64_t>(max_tokens) * a.group;
  a.tiles = p.num_tiles;
  a.shares = p.num_shares;
  a.row_tiles = a.shares > 0 ? static_cast<int>((rows + p.tile_rows - 1) / p.tile_rows) : 0;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const int64_t items = static_cast<int64_t>(a.row_tiles) * num_kv_heads * a.shares;
  if (items > 0x7fffffff) return SGL_ERR_UNSUPPORTED;
  // The fold's grid is at most a workgroup per row.
  if (static_cast<int64_t>(max_tokens) * num_qo_heads > 0x7fffffff) return SGL_ERR_UNSUPPORTED;
  const int waves = heads_per_group(num_kv_heads);
  const dim3 grid(p.num_units, num_kv_heads / waves), block(64 * waves);
  if (items > 0) {
    const dim3 own(static_cast<uint32_t>(items));
    if (p.tile_rows == 128) hipLaunchKernelGGL(prefix_rows_kernel<4>, own, dim3(256), 0, s, a);
    else hipLaunchKernelGGL(prefix_rows_kernel<8>, own, dim3(512), 0, s, a);
    st = launch_status();
    if (st != SGL_OK) return st;
  }
  const int own_rows = p.max_qo_len * a.group;
  const int need = a.tiles > 0 && own_rows < a.tile_rows ? a.tile_rows : own_rows;
  const int rb = need <= 16 ? 1 : need <= 32 ? 2 : 4;
  const size_t lds = static_cast<size_t>(waves) * 16 * rb * kQPitch * 2;
  if (rb == 1) hipLaunchKernelGGL(prefix_units_kernel<1>, grid, block, lds, s, a);
  else if (rb == 2) hipLaunchKernelGGL(prefix_units_kernel<2>, grid, block, lds, s, a);
  else hipLaunchKernelGGL(prefix_units_kernel<4>, grid, block, lds, s, a);
  st = launch_status();
  if (st != SGL_OK) return st;
  // Many pieces a row: a workgroup for each. Few: two groups of lanes a row.
  const int64_t pieces = a.tiles > 0 ? p.num_units : a.shares + 1;
  const int rows_per = pieces > 16 ? 1 : 4;
  const int head_groups = (num_qo_heads + rows_per - 1) / rows_per;
  const dim3 fold(static_cast<uint32_t>(max_tokens) * head_groups);
  if (rows_per == 1) hipLaunchKernelGGL(prefix_fold_kernel<8>, fold, dim3(256), 0, s, a, head_groups);
  else hipLaunchKernelGGL(prefix_fold_kernel<2>, fold, dim3(256), 0, s, a, head_groups);
  return launch_status();
}
