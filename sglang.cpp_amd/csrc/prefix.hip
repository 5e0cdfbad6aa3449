// Attention of a batch that shares a prefix: row (token t, head) of request r is
//   o = softmax_j(q . k_j scale) . v_j  over the prefix's tokens, then the request's own,
// j <= i + kv_len - qo_len for its i-th query token. A softmax over a joined
// sequence folds from its parts: with each part's sum l, reference point m and
// output o (normalised), weights 2^(lse - max lse), lse = m + log2 l. So the prefix's
// K/V are walked once with the rows of every request as columns of one product,
// each request's own tokens with its rows alone, and a second launch folds.
//
// Two ways over tokens in one launch (split_of). Tiles: the prefix, 64 tokens at a time
// through LDS, for up to 128 packed rows of a kv head. Units: the requests' own tokens
// form one stream, cut into units of equal length, one workgroup each as a rule; a wave
// has one kv head, so a workgroup reads whole token rows. A wave walks its piece 16
// tokens a step on the matrix cores: S^T = K Q^T, then O^T += V^T P^T, whose operand P^T
// is S^T's accumulator layout, for one or two column blocks of 16 rows per K/V read. Both
// put the row on the lane's column, so the running maximum and sum are lane-local but for
// one exchange across four lane groups. K and V of the next steps are in flight during one.
//
// The units could walk the prefix too where rows are few (32 at most, 16 tokens a step in
// registers, no LDS): 32q/8kv, 64 own tokens, 8 requests behind 1,024 / 4,096 / 16,384 /
// 65,536 tokens took 15.9 / 24.4 / 32.0 / 59.6 us so, 12.8 / 14.4 / 22.8 / 53.9 with tiles;
// one request 11.8 / 15.9 / 23.4 / 50.2, with tiles 12.1 / 13.0 / 21.8 / 51.4.
#include <math.h>

#include <algorithm>

#include "common.h"
#include "prefill_impl.h"

namespace sgl {
namespace {

constexpr int kD = 128;
constexpr int kStep = 16;                 // tokens a step
constexpr float kRescaleSlack = 8.f;      // log2 units: p <= 256 between rescales
// Workgroups of the fold up to which a lane group has one row. 512 and 4,096: 256 tokens of
// 32 heads 127 and 127 us in all (124 so), 384 of 32 44.6 and 41.4 (42.5), 32 of 32 23.8
// and 22.6 (22.6).
constexpr int kFoldGroups = 1024;
constexpr int kWaves = 4;                 // waves of a workgroup, two workgroups per CU
constexpr int kWaveLds = 8192;            // a wave's LDS for its output rows on their way to memory

// What the fold needs of a launch's Split.
struct alignas(16) FoldSplit {
  int first, rows, shares, W;
};

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
  uint32_t inv_group;    // 2^16 / group, rounded up
  int prefix, max_qo;
  int blocks;            // workgroups of the launch
  int heads, side, rest; // kv heads of a unit, units side by side in a workgroup, head groups
  float scale_log2;
  uint16_t* o;
  int64_t o_st, o_sh;
  // Partial outputs (fp32 [.., 128]) and log2-sum-exp. Prefix: [piece of the
  // item][kv head][packed row]. Own tokens: [token slot][q head],
  // the piece a request starts with at its rows' own tokens, the one running into unit
  // u from before it at tokens + u max_qo + i.
  float* p_o;
  float* p_lse;
  float* s_o;
  float* s_lse;
  FoldSplit* split;
};

// How a launch is shared out, from the lengths as they are now (so a captured launch
// follows them): every workgroup works it out alike, by the same instructions, and one leaves the
// fold what it needs of it.
// Workgroups [0, tile_blocks) walk the prefix's 64-token tiles, `run` of them for one row
// tile and kv head at a time: each row tile's tiles are cut into `shares` runs, all row
// tiles alike and taken run by run, so that the `wide` workgroups of a head, on the same
// XCD where there are eight heads, read the same K/V at about the same time. The others'
// units walk the stream of `all` tokens, W a unit.
struct Split {
  int first, rows;          // first query token, packed rows of a kv head
  int row_tiles, row_step;  // row tiles and their rows (32 a wave, spread evenly)
  int tiles;                // 64-token tiles of the prefix
  int tile_blocks, wide, shares, run;
  uint32_t all, W;
  int units;
  int q_first, q_end, kv_first, kv_end;  // the batch's offsets
};

// What a tile takes on one workgroup, and a token of a kv head, ns. Half and twice of the
// first: 256 requests of 200 own tokens behind 16,384 tokens 121 and 121 us (123 so), 128
// of 2,000 behind 1,024 183 and 177 (183), 32 of 300 behind 4,096 26.5 and 27.9 (26.2).
constexpr uint32_t kTileNs = 1400;
constexpr uint32_t kTokenNs = 16;
// A request counts as this many tokens more in the units' stream: what begins and ends
// its walk, about 3.4 us. 0, 24, 48 and 96 measured: 64 requests of 5 own tokens
// 16.7, 11.2, 10.3, 11.2 us; 64 of 16 behind 1,024 tokens 25.2, 25.6, 22.7, 22.8; 256 of
// 200 behind 16,384 121 to 125 with any.
constexpr uint32_t kRequestTokens = 48;

// A loaded value that is the same in every lane, in a scalar register (the compiler
// keeps it in a vector one, as the kernel's stores might change the memory).
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// x / d for x < 2^21, d > 0: the distance of (x + 1/2) / d from a whole number is at least
// 1 / (2 d), the product with the reciprocal off by less than 2^-22 of itself. (The split
// of a launch took 3,500 cycles with whole-number divisions, 1,800 so.)
__device__ __forceinline__ int quotient(int x, int d) {
  return static_cast<int>((static_cast<float>(x) + 0.5f) * __builtin_amdgcn_rcpf(static_cast<float>(d)));
}

// Minimum over the wave: shifts by 1, 2, 4 and 8 in each row of 16, then the last lane of
// a row to the next row, of the first half to the second, whose last lane has it.
__device__ __forceinline__ float wave_min(float x) {
  const auto with = [](float x, int y) { return fminf(x, __builtin_bit_cast(float, y)); };
  const int inf = __builtin_bit_cast(int, INFINITY);
  x = with(x, __builtin_amdgcn_update_dpp(inf, __builtin_bit_cast(int, x), 0x111, 0xF, 0xF, false));
  x = with(x, __builtin_amdgcn_update_dpp(inf, __builtin_bit_cast(int, x), 0x112, 0xF, 0xF, false));
  x = with(x, __builtin_amdgcn_update_dpp(inf, __builtin_bit_cast(int, x), 0x114, 0xF, 0xF, false));
  x = with(x, __builtin_amdgcn_update_dpp(inf, __builtin_bit_cast(int, x), 0x118, 0xF, 0xF, false));
  x = with(x, __builtin_amdgcn_update_dpp(inf, __builtin_bit_cast(int, x), 0x142, 0xA, 0xF, false));
  x = with(x, __builtin_amdgcn_update_dpp(inf, __builtin_bit_cast(int, x), 0x143, 0xC, 0xF, false));
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), 63));
}

// Offsets of 63 requests from request `base` on, lane i those of request base + i and the
// end of the one before: in registers, so that neither finding a request nor the next one
// of a walk waits for memory.
struct Offsets {
  int base, q, k;
};

constexpr int kWindow = kWave - 1;

__device__ __forceinline__ Offsets offsets_from(const PrefixArgs& a, int base, int lane) {
  const int e = min(base + lane, a.batch);
  return Offsets{base, a.qo_indptr[e], a.kv_indptr[e]};
}

// `head`: the offsets from request 0 on.
__device__ __forceinline__ Split split_of(const PrefixArgs& a, const Offsets& head) {
  Split s;
  s.q_end = uniform(a.qo_indptr[a.batch]), s.kv_end = uniform(a.kv_indptr[a.batch]);
  s.q_first = uniform(head.q), s.kv_first = uniform(head.k);
  s.first = max(s.q_first, 0);
  s.rows = max(min(s.q_end, a.tokens) - s.first, 0) * a.group;
  s.all = static_cast<uint32_t>(max(s.kv_end - max(s.kv_first, 0), 0)) + a.batch * kRequestTokens;
  s.tiles = (a.prefix + pf::kBN - 1) / pf::kBN;
  s.row_tiles = s.row_step = s.tile_blocks = s.wide = s.shares = s.run = 0;
  if (s.rows > 0 && s.tiles > 0) {
    // 32 rows a wave, up to 4 waves a row tile, spread evenly.
    const int waves = (s.rows + 31) / 32;
    s.row_tiles = (waves + kWaves - 1) / kWaves;
    const int each = 1 + (waves > s.row_tiles) + (waves > 2 * s.row_tiles) + (waves > 3 * s.row_tiles);
    s.row_step = 32 * each;
    const float t = static_cast<float>(s.row_tiles) * s.tiles * kTileNs, own = static_cast<float>(s.all) * kTokenNs;
    const int share = static_cast<int>(a.blocks * t * __builtin_amdgcn_rcpf(t + own) + 0.5f);
    // A second workgroup of tiles on a CU brings nothing (1.4 us a tile alone, 2.7 for
    // each of two).
    s.tile_blocks = max(1, min(share, a.blocks / 2));
    // An eighth more than its share: within 1% of none in most batches. us with none, an
    // eighth and a quarter: 160 requests of 20 own tokens behind 16,384 64.5, 63.6, 65.2; 64 of
    // 16 behind 1,024 14.4, 14.4, 16.5; 32 of 300 behind 4,096 22.2, 23.0, 23.1.
    s.wide = max(1, quotient(s.tile_blocks, a.hkv));
    s.wide = max(1, min(s.wide + s.wide / 8, quotient(a.blocks / 2, a.hkv)));
    // The number of runs. Many workgroups a row tile: one each. Else candidates, one a lane:
    // the tiles of the rounds that they take, what begins and ends a run (six tiles' time),
    // and a 43rd of a tile for the partial rows of a run and row tile, written and folded.
    // The workspace has room for two runs a row tile, or for as many as there are
    // workgroups. 640 requests of 20 own tokens behind 16,384, 32q/8kv (20 row tiles for 32
    // workgroups): one run each 319 us, three in two rounds 235. The constants hardly matter.
    // us with 3, 6 and 12 tiles: 160 of 20 behind 16,384 64.2, 63.6, 63.4; 96 of 100 behind
    // 4,096, 32q/4kv, 25.2, 25.4, 25.9. With a 21st, 43rd and 86th: 640 of 20 behind 2,048
    // 53.9, 53.7, 56.4. With candidates below 4, 8, 16 and 64 workgroups a row tile: 96 of 100
    // 25.5, 25.4, 24.3, 24.2; 4 requests of 40 behind 1,500, 16q/8kv, 11.2, 11.1, 11.2, 11.9.
    int take = min(quotient(s.wide, s.row_tiles), s.tiles);
    float k = 1.f;
    if (s.wide < 8 * s.row_tiles) {
      const int n = 1 + static_cast<int>(threadIdx.x & 63);
      const float items = static_cast<float>(n) * s.row_tiles;
      const float rounds = ceilf((items - 0.5f) * __builtin_amdgcn_rcpf(s.wide));
      const float cost = rounds * (ceilf((s.tiles - 0.5f) * __builtin_amdgcn_rcpf(n)) + 6.f) + items * a.hkv * (1.f / 43.f);
      const bool fits = n <= s.tiles && (n <= 2 || (items - 2.f * s.row_tiles) * a.hkv <= a.blocks);
      const float best = wave_min(fits ? cost : INFINITY);
      take = __builtin_ctzll(__builtin_amdgcn_ballot_w64(fits && cost == best));
      k = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, rounds), take));
      ++take;
    }
    // At least tiles / take (up to 2^23 of them: off by less than two), and the runs that are.
    int run = static_cast<int>(s.tiles * __builtin_amdgcn_rcpf(take));
    run += run * take < s.tiles;
    run += run * take < s.tiles;
    int shares = static_cast<int>(s.tiles * __builtin_amdgcn_rcpf(run));
    shares += shares * run < s.tiles;
    shares += shares * run < s.tiles;
    shares -= (shares - 1) * run >= s.tiles;
    s.run = uniform(run), s.shares = uniform(shares);
    const int all = s.shares * s.row_tiles;
    s.wide = uniform(min(min(s.wide, all), static_cast<int>(all * __builtin_amdgcn_rcpf(k)) + 1));
    s.tile_blocks = min(s.wide * a.hkv, a.blocks / 2);
  }
  s.units = max(1, quotient((a.blocks - s.tile_blocks) * a.side, a.rest));
  // At least all / units: the product is off by less than 2^-20 of itself.
  uint32_t w = static_cast<uint32_t>(s.all * __builtin_amdgcn_rcpf(s.units));
  w += (w >> 20) + 1;
  s.W = (w + kStep - 1) / kStep * kStep;
  // Quotients come from the vector unit.
  s.W = uniform(s.W), s.units = uniform(s.units);
  return s;
}

struct Request {
  int q0, qo, kv0, kv;  // first query token, query tokens, first own index, own tokens
  bool ok;
};

// From its own offsets and the batch's.
__device__ __forceinline__ Request request_from(const PrefixArgs& a, int q0, int64_t q1, int kv0, int64_t k1,
                                                int q_first, int q_end, int kv_first, int kv_end) {
  Request x;
  x.q0 = q0, x.kv0 = kv0;
  x.qo = static_cast<int>(q1 - q0);
  x.kv = static_cast<int>(k1 - kv0);
  // Rows and pieces of anything else have no place in the outputs and the workspace.
  x.ok = q0 >= max(q_first, 0) && q1 >= q0 && q1 <= min(q_end, a.tokens) && q1 - q0 <= a.max_qo &&
         kv0 >= max(kv_first, 0) && k1 >= kv0 && k1 <= kv_end;
  return x;
}

__device__ __forceinline__ bf16x8_t as_bf16x8(const u32x4_t& v) {
  return __builtin_bit_cast(bf16x8_t, v);
}

// Orders LDS traffic between the lanes of one wave (it runs in order; this only keeps
// the compiler from moving it).
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

// A piece: the len tokens of slots idx[0, len) for the packed rows [row0, row0 + rows)
// (row p: token tok0 + p / G, head h G + p % G of kv head h). A row of token i sees the
// tokens below sees0 + i. Its output and lse go to row (out0 + i) hq + head.
struct Piece {
  const int32_t* idx;
  int len;
  int tok0, row0, rows, sees0;
  int64_t out0;
};

// One wave over a piece of at most 16 RB rows. Lane (n, j), n = lane % 16: token n (K),
// chunk n of tokens 4 j + e (V), row n of each block (Q, S, O). Q stays in registers.
template <int RB>
__device__ __forceinline__ void walk(const PrefixArgs& a, const Piece& w, char* xch, int h, int lane) {
  // Steps whose K/V rows are in flight: two where the registers hold them.
  constexpr int kDepth = RB == 1 ? 2 : 1;
  const int n = lane & 15, j = lane >> 4;
  const int G = a.group, len = uniform(w.len), rows = uniform(w.rows);
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
  // Slots of this lane's token, kDepth steps' for the first K/V rows, then two steps' for
  // the next ones.
  int slot0[kDepth], slot[2];
#pragma unroll
  for (int i = 0; i < kDepth; ++i) slot0[i] = w.idx[min(i * kStep + n, len - 1)];
#pragma unroll
  for (int i = 0; i < 2; ++i) slot[i] = w.idx[min((kDepth + i) * kStep + n, len - 1)];
  // Token and head of this lane's row of each block; rows past the last one read
  // its Q again and see nothing.
  const int i0 = uniform(quotient(w.row0, G)), rem = w.row0 - i0 * G;
  const uint32_t inv_g = a.inv_group;  // (rem + x) / G as a product, both below 128
  int tok[RB], head[RB], sees[RB];
  u32x4_t q[RB][4];
#pragma unroll
  for (int b = 0; b < RB; ++b) {
    const int x = min(16 * b + n, rows - 1) + rem;
    const int d = static_cast<int>(static_cast<uint32_t>(x) * inv_g >> 16);
    tok[b] = i0 + d;
    head[b] = h * G + (x - d * G);
    sees[b] = 16 * b + n < rows ? min(w.sees0 + tok[b], len) : 0;
    const uint16_t* qp = a.q + (w.tok0 + tok[b]) * a.q_st + head[b] * a.q_sh + 8 * j;
#pragma unroll
    for (int s = 0; s < 4; ++s) q[b][s] = ldg128(qp + 32 * s);
  }
  // K before V, as in the loop, whose waits count the loads in flight: the compiler
  // merges the two orders, and waited for V with K where they differed.
  u32x4_t kr[kDepth][4], vr[kDepth][4];
#pragma unroll
  for (int i = 0; i < kDepth; ++i) {
    __builtin_amdgcn_sched_barrier(0);
    load_k(slot0[i], kr[i]);
    __builtin_amdgcn_sched_barrier(0);
    load_v(slot0[i], vr[i]);
  }
  __builtin_amdgcn_sched_barrier(0);
  float m[RB], l[RB];
  f32x4_t acc[RB][8];
#pragma unroll
  for (int b = 0; b < RB; ++b) {
    m[b] = -INFINITY;
    l[b] = 0.f;
#pragma unroll
    for (int nb = 0; nb < 8; ++nb) acc[b][nb] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }

  auto step = [&](int t, int& slot, u32x4_t (&kr)[4], u32x4_t (&vr)[4]) {
    f32x4_t sacc[RB];
#pragma unroll
    for (int b = 0; b < RB; ++b) {
      sacc[b] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < 4; ++s)
        sacc[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(kr[s]), as_bf16x8(q[b][s]), sacc[b], 0, 0, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
    load_k(slot, kr);
    __builtin_amdgcn_sched_barrier(0);
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
      // P in bf16, the product's operand type: a weight is off by at most 2^-8 of
      // itself, as the rounding of the output.
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
    __builtin_amdgcn_sched_barrier(0);
    load_v(slot, vr);
    slot = w.idx[min(t + (kDepth + 2) * kStep + n, len - 1)];
    __builtin_amdgcn_sched_barrier(0);
  };
  // Pairs of steps and one alone: with a way out between the two of a pair the compiler
  // takes the next pair to follow the first directly and waits for every load.
  int t = 0;
#pragma unroll 1
  for (; t + kStep < len; t += 2 * kStep) {
    step(t, slot[0], kr[0], vr[0]);
    step(t + kStep, slot[1], kr[kDepth - 1], vr[kDepth - 1]);
  }
  if (t < len) step(t, slot[0], kr[0], vr[0]);
  // The block's output through LDS (16 rows of 32 16-byte chunks, chunk c of row n at
  // c ^ n: no bank conflicts either way), so that whole rows are stored: as they lie in
  // the accumulators a store would touch 64 lines for 1 KB (64 requests of 6 query and
  // 256 own tokens, 32q/4kv: 42.4 us so, 32.2 through LDS).
  f32x4_t* xr = reinterpret_cast<f32x4_t*>(xch);
#pragma unroll
  for (int b = 0; b < RB; ++b) {
    if (16 * b >= rows) break;
    const float sum = sum_xor32(sum_xor16(l[b]));
    const float inv = sum == 0.f ? 0.f : 1.0f / sum;  // a NaN sum stays one
    // acc[nb][c] holds d = 32 j + 8 c + nb.
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      f32x4_t lo, hi;
#pragma unroll
      for (int nb = 0; nb < 4; ++nb) lo[nb] = acc[b][nb][c] * inv, hi[nb] = acc[b][nb + 4][c] * inv;
      xr[32 * n + ((8 * j + 2 * c) ^ n)] = lo;
      xr[32 * n + ((8 * j + 2 * c + 1) ^ n)] = hi;
    }
    wave_lds_sync();
    if (j == 0 && 16 * b + n < rows)
      a.s_lse[(w.out0 + tok[b]) * a.hq + head[b]] = sum == 0.f ? -INFINITY : m[b] + log2f(sum);
    const int c = lane & 31;
#pragma unroll
    for (int it = 0; it < 8; ++it) {
      const int x = 2 * it + (lane >> 5), y = 16 * b + x + rem;
      if (16 * b + x >= rows) break;
      const int d = static_cast<int>(static_cast<uint32_t>(y) * inv_g >> 16);
      const int64_t row = (w.out0 + i0 + d) * a.hq + (h * G + y - d * G);
      __builtin_nontemporal_store(xr[32 * x + (c ^ x)], reinterpret_cast<f32x4_t*>(a.s_o + row * kD + 4 * c));
    }
    wave_lds_sync();
  }
}

// Unit u's pieces of the stream for kv head h: places below 2^31 (the offsets are int32)
// + 2^25 requests' kRequestTokens, 32 bits without a sign.
template <int RB>
__device__ __forceinline__ void unit_pieces(const PrefixArgs& a, const Split& s, const Offsets& head, char* xch,
                                            uint32_t u, int h, int lane) {
  if (static_cast<uint64_t>(u) * s.W >= s.all) return;
  // The places [b0, b1), from request r on: those that end at or before b0 are passed over.
  const uint32_t b0 = u * s.W, b1 = min(s.all, b0 + s.W);
  const int kv_first = max(s.kv_first, 0);
  Offsets at = head;
  int r = 0;
  while (true) {
    const int e = at.base + lane;  // this lane's offset is where request e - 1 ends
    const int64_t end = static_cast<int64_t>(at.k) - kv_first + static_cast<int64_t>(e) * kRequestTokens;
    const int passed = __builtin_popcountll(
        __builtin_amdgcn_ballot_w64(lane > 0 && e <= a.batch && end <= static_cast<int64_t>(b0)));
    r = at.base + passed;
    if (passed < kWindow || r >= a.batch) break;
    at = offsets_from(a, r, lane);
  }
  for (; r < a.batch; ++r) {
    if (r - at.base >= kWindow) at = offsets_from(a, r, lane);
    const int i = r - at.base;
    const auto lane_of = [](int x, int i) { return __builtin_amdgcn_readlane(x, i); };
    const Request x = request_from(a, lane_of(at.q, i), lane_of(at.q, i + 1), lane_of(at.k, i),
                                   lane_of(at.k, i + 1), s.q_first, s.q_end, s.kv_first, s.kv_end);
    // Its kRequestTokens places, then its tokens'.
    const int64_t rb = static_cast<int64_t>(x.kv0) - kv_first + static_cast<int64_t>(r) * kRequestTokens;
    if (rb >= b1) return;
    if (!x.ok) continue;
    const int64_t own = rb + kRequestTokens;
    const int s0 = static_cast<int>(max(b0 - own, int64_t{0}));
    Piece w;
    w.len = static_cast<int>(min(b1 - own, static_cast<int64_t>(x.kv))) - s0;
    if (w.len <= 0) continue;
    w.idx = a.indices + x.kv0 + s0;
    w.tok0 = x.q0;
    w.sees0 = max(x.kv - x.qo + 1 - s0, -x.qo);
    w.out0 = s0 == 0 ? x.q0 : a.tokens + static_cast<int64_t>(u) * a.max_qo;
    const int rows = x.qo * a.group;
    for (w.row0 = 0; w.row0 < rows; w.row0 += 16 * RB) {
      w.rows = min(rows - w.row0, 16 * RB);
      walk<RB>(a, w, xch, h, lane);
    }
  }
}

// The prefix: W waves with 32 packed rows each share the 64-token K/V
// tiles that they gather into LDS (two buffers, K one tile ahead of V), and tile t + 1's
// scores are on the matrix cores while tile t's become weights; the prefill kernel's
// tile steps without a causal bound, P in bf16 for the product with V as there and in the
// units. Tiles [tb, te) of the prefix for row tile rt of kv head h, the item's piece number
// `piece`. 4 x 64 x 128 flops a row and tile: 1.4 us a tile of 128 rows, 0.77 PFLOP/s on all
// CUs, the matrix cores busy in 41% of the cycles (the prefill's 256 rows a tile: 1.0).
__device__ __forceinline__ void prefix_tiles(const PrefixArgs& a, const Split& sp, char* lds_raw, int rt,
                                             int h, int tb, int te, int piece) {
  using namespace pf;
  constexpr int W = kWaves;
  const int rows = sp.rows, first = sp.first;
  const int row0 = rt * sp.row_step, row_end = min(rows, row0 + sp.row_step);
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tid = threadIdx.x;
  const int c = lane & 31, hl = lane >> 5;
  const int prow = row0 + 32 * wave + c;
  const bool row_ok = prow < row_end;
  const bool works = row0 + 32 * wave < row_end;  // the others only gather
  const int safe = row_ok ? prow : row0;
  const int qtok = safe / a.group;
  const int qhead = h * a.group + (safe - qtok * a.group);
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
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  const int64_t row_first = (static_cast<int64_t>(piece) * a.hkv + h) * rows + row0 + 32 * wave;
  if (row_ok && hl == 0) a.p_lse[row_first + c] = l == 0.f ? -INFINITY : rs.m + log2f(l);
  // Whole rows to memory through the wave's 8 KB of LDS (free behind the last step's
  // barrier), half a row (64 values, 16 chunks; chunk k of row c at k ^ c) at a time.
  f32x4_t* xr = reinterpret_cast<f32x4_t*>(lds_raw + wave * kWaveLds);
  // The lane's places are worked out here, not ahead of the tiles, where they would
  // take registers that the tiles need.
  int ln = lane;
  asm volatile("" : "+v"(ln));
  const int left = row_end - (row0 + 32 * wave);
#pragma unroll
  for (int half = 0; half < 2; ++half) {
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x16_t& x = rs.acc[2 * half + e];
        xr[16 * (ln & 31) + ((8 * e + 2 * g + (ln >> 5)) ^ (ln & 15))] =
            f32x4_t{x[4 * g] * inv, x[4 * g + 1] * inv, x[4 * g + 2] * inv, x[4 * g + 3] * inv};
      }
    wave_lds_sync();
#pragma unroll
    for (int it = 0; it < 8; ++it) {
      const int x = 4 * it + (ln >> 4), k = ln & 15;
      if (x < left)
        __builtin_nontemporal_store(
            xr[16 * x + (k ^ (x & 15))],
            reinterpret_cast<f32x4_t*>(a.p_o + (row_first + x) * sgl::kD + 64 * half + 4 * k));
    }
    wave_lds_sync();
  }
  __syncthreads();  // before the next item's tiles
}

// Two workgroups of four waves per CU: those that walk the prefix's tiles, bound by
// their products, lie beside the others' units, bound by memory. 256 requests of 528
// own tokens each behind 16,384, 32q/8kv: the prefix alone 103 us, the own tokens alone 89,
// together 152 (fold included; 621 MB of K/V, 87 us at a read's 7.1 TB/s, and 71 GFLOP,
// 60 us at a large product's 1.19 PFLOP/s).
template <int RB>
__global__ void __launch_bounds__(64 * kWaves, 2) prefix_attention_kernel(PrefixArgs a) {
  __shared__ __attribute__((aligned(16))) char smem[2 * pf::kTileBytes];
  static_assert(sizeof(smem) >= kWaves * kWaveLds, "the waves' output rows take the tiles' place");
  const int lane = threadIdx.x & 63;
  const Offsets head = offsets_from(a, 0, lane);
  const Split s = split_of(a, head);
  const int b = blockIdx.x;
  if (b == a.blocks - 1 && threadIdx.x == 0)
    *a.split = FoldSplit{s.first, s.rows, s.shares, static_cast<int>(s.W)};
  if (b < s.tile_blocks) {
    // Workgroup b has head b % hkv and every wide-th item of it, or, with more heads than
    // workgroups, every tile_blocks-th head and all of its items.
    const bool few = s.wide * a.hkv > s.tile_blocks;
    const int j0 = few ? 0 : uniform(quotient(b, a.hkv)), wide = few ? 1 : s.wide;
    const int first_run = uniform(quotient(j0, s.row_tiles));
    for (int h = b - j0 * a.hkv; h < a.hkv; h += few ? s.tile_blocks : a.hkv) {
      int piece = first_run, rt = j0 - first_run * s.row_tiles;
      while (piece < s.shares) {
        const int tb = piece * s.run;
        prefix_tiles(a, s, smem, rt, h, tb, min(s.tiles, tb + s.run), piece);
        for (rt += wide; rt >= s.row_tiles; rt -= s.row_tiles) ++piece;
      }
    }
    return;
  }
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = uniform(quotient(wave, a.heads));
  if (g >= a.side) return;
  const int n = a.blocks - s.tile_blocks;
  for (int v = (b - s.tile_blocks) * a.side + g; v < s.units * a.rest; v += n * a.side) {
    const int u = uniform(quotient(v, a.rest));
    unit_pieces<RB>(a, s, head, smem + wave * kWaveLds, u, (v - u * a.rest) * a.heads + wave - g * a.heads, lane);
  }
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
// No reuse between rows and no matrix cores: 12,288 rows of 6,000 tokens 4.9 ms (6.6 with
// one token's loads in flight), 4 requests of 8 query and 2 own tokens behind 16,384 6.4 ms.
__device__ __forceinline__ f32x4_t plain_row(const PrefixArgs& a, const Request& x, int tok, int head,
                                             int64_t sees, int c) {
  const int h = head / a.group;
  const u32x2_t qw = *reinterpret_cast<const u32x2_t*>(a.q + tok * a.q_st + head * a.q_sh + 4 * c);
  const float q[4] = {bf16_lo(qw[0]), bf16_hi(qw[0]), bf16_lo(qw[1]), bf16_hi(qw[1])};
  float m = -INFINITY, l = 0.f;
  f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
  constexpr int kAhead = 8;  // tokens whose loads are in flight together
  for (int64_t t0 = 0; t0 < sees; t0 += kAhead) {
    u32x2_t kw[kAhead], vw[kAhead];
#pragma unroll
    for (int e = 0; e < kAhead; ++e) {
      const int64_t t = min(t0 + e, sees - 1);
      const int64_t slot = static_cast<uint32_t>(t < a.prefix ? a.pidx[t] : a.indices[x.kv0 + (t - a.prefix)]);
      kw[e] = *reinterpret_cast<const u32x2_t*>(a.kc + slot * a.kv_ss + h * a.kv_sh + 4 * c);
      vw[e] = *reinterpret_cast<const u32x2_t*>(a.vc + slot * a.kv_ss + h * a.kv_sh + 4 * c);
    }
    float s[kAhead];
#pragma unroll
    for (int e = 0; e < kAhead; ++e) {
      s[e] = q[0] * bf16_lo(kw[e][0]) + q[1] * bf16_hi(kw[e][0]) + q[2] * bf16_lo(kw[e][1]) + q[3] * bf16_hi(kw[e][1]);
      s[e] = half_sum(s[e]) * a.scale_log2;
    }
#pragma unroll
    for (int e = 0; e < kAhead; ++e) {
      if (t0 + e >= sees) break;
      const float mn = fmaxf(m, s[e]);
      const float alpha = m == -INFINITY ? 0.f : exp2f(m - mn);
      const float p = s[e] == -INFINITY ? 0.f : exp2f(s[e] - mn);  // NaN stays NaN
      l = l * alpha + p;
      const f32x4_t v = {bf16_lo(vw[e][0]), bf16_hi(vw[e][0]), bf16_lo(vw[e][1]), bf16_hi(vw[e][1])};
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] = acc[i] * alpha + p * v[i];
      m = mn;
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  return acc * inv;
}

// Folds the pieces of each row: kSets groups of 32 lanes take them in turn and are
// folded through LDS; a workgroup has `iters` times 8 / kSets heads of one token. Bound by
// instructions and the chain of dependent loads (request, its offsets, its pieces), so
// what is a token's is worked out once for its heads, in scalar registers, with every
// load that does not wait for another sent first.
template <int kSets>
__global__ void __launch_bounds__(256) prefix_fold_kernel(PrefixArgs a, int head_groups, int iters) {
  constexpr int kRows = 8 / kSets, kLoads = kSets == 1 ? 4 : 8;
  __shared__ int found[4][5];
  __shared__ float xch[kSets > 1 ? 6 : 1][8][32];
  const int t = uniform(blockIdx.x / static_cast<uint32_t>(head_groups));
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // The token's request, by one lane each; the first where offsets that decrease give
  // it several.
  int r = -1;
  for (int at = 64 * wave; at < a.batch; at += 256) {
    const int e = min(at + lane, a.batch - 1);
    const int q0 = a.qo_indptr[e], q1 = a.qo_indptr[e + 1], k0 = a.kv_indptr[e], k1 = a.kv_indptr[e + 1];
    const uint64_t mask = __builtin_amdgcn_ballot_w64(at + lane < a.batch && q0 <= t && t < q1);
    if (mask == 0) continue;
    const int by = __builtin_ctzll(mask);
    r = at + by;
    if (lane == by) {
      found[wave][1] = q0, found[wave][2] = q1;
      found[wave][3] = k0, found[wave][4] = k1;
    }
    break;
  }
  FoldSplit sp = *a.split;
  const int q_first = a.qo_indptr[0], q_end = a.qo_indptr[a.batch];
  const int kv_first = uniform(a.kv_indptr[0]), kv_end = a.kv_indptr[a.batch];
  sp = FoldSplit{uniform(sp.first), uniform(sp.rows), uniform(sp.shares), uniform(sp.W)};
  if (lane == 0) found[wave][0] = r;
  __syncthreads();
  int from = 3;
#pragma unroll
  for (int k = 2; k >= 0; --k) from = found[k][0] >= 0 ? k : from;
  r = uniform(found[from][0]);
  if (r < 0) return;  // no request's row: left as it was
  const Request x = request_from(a, uniform(found[from][1]), uniform(found[from][2]), uniform(found[from][3]),
                                 uniform(found[from][4]), uniform(q_first), uniform(q_end), kv_first,
                                 uniform(kv_end));
  const int P = a.prefix, i = t - x.q0;
  const int64_t sees = static_cast<int64_t>(P) + x.kv - x.qo + i + 1;  // tokens this row sees, prefix first
  const bool folded = x.ok && sees >= P;
  // The request's own pieces: ns of them, the first at s0 + head, the k-th behind it at s1 + k s_step + head.
  int ns = 0;
  int64_t s1 = 0;
  if (x.kv > 0 && x.ok) {
    const uint32_t W = sp.W;
    const uint32_t own0 = (x.kv0 - max(kv_first, 0)) + (r + 1) * kRequestTokens;
    const uint32_t u0 = uniform(own0 / W);
    ns = uniform((own0 + x.kv - 1) / W) - u0 + 1;
    s1 = (a.tokens + static_cast<int64_t>(u0) * a.max_qo + i) * a.hq;
  }
  const int64_t s0 = static_cast<int64_t>(t) * a.hq, s_step = static_cast<int64_t>(a.max_qo) * a.hq;
  const int row_of_head = (t - sp.first) * a.group;
  const int c = threadIdx.x & 31, group = threadIdx.x >> 5, set = group % kSets;
  for (int it = 0; it < iters; ++it) {
    const int head = ((blockIdx.x - t * head_groups) * iters + it) * kRows + group / kSets;
    const int hh = min(head, a.hq - 1);
    const int h = hh / a.group;
    float m = -INFINITY, l = 0.f;
    f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
    if (folded) {
      // Prefix pieces: np of them, p_step rows apart.
      const int prow = row_of_head + hh - h * a.group;
      const int np = sp.shares;
      const int64_t p_step = static_cast<int64_t>(a.hkv) * sp.rows, p0 = static_cast<int64_t>(h) * sp.rows + prow;
      for (int k0 = set; k0 < np + ns; k0 += kLoads * kSets) {
        f32x4_t v[kLoads];
        float lse[kLoads];
#pragma unroll
        for (int e = 0; e < kLoads; ++e) {
          const int k = min(k0 + e * kSets, np + ns - 1);
          const int64_t row = k < np ? p0 + k * p_step : hh + (k == np ? s0 : s1 + (k - np) * s_step);
          v[e] = *reinterpret_cast<const f32x4_t*>((k < np ? a.p_o : a.s_o) + row * kD + 4 * c);
          lse[e] = (k < np ? a.p_lse : a.s_lse)[row];
          if (k0 + e * kSets >= np + ns) lse[e] = -INFINITY;
        }
        float mn = m;
#pragma unroll
        for (int e = 0; e < kLoads; ++e) mn = fmaxf(mn, lse[e]);
        const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
        l *= alpha;
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[k] *= alpha;
        m = mn;
#pragma unroll
        for (int e = 0; e < kLoads; ++e) {
          if (lse[e] == -INFINITY) continue;  // nothing seen there: its values do not count
          const float w = __builtin_amdgcn_exp2f(lse[e] - mn);
          l += w;
#pragma unroll
          for (int k = 0; k < 4; ++k) acc[k] += v[e][k] * w;
        }
      }
    }
    if constexpr (kSets > 1) {
      if (it > 0) __syncthreads();  // the last row's values have been read
#pragma unroll
      for (int k = 0; k < 4; ++k) xch[k][group][c] = acc[k];
      xch[4][group][c] = m;
      xch[5][group][c] = l;
      __syncthreads();
      if (set == 0) {
#pragma unroll
        for (int e = 1; e < kSets; ++e) m = fmaxf(m, xch[4][group + e][c]);
        l = 0.f;
        acc = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int e = 0; e < kSets; ++e) {
          const float me = xch[4][group + e][c], le = xch[5][group + e][c];
          if (le == 0.f) continue;  // no piece with a weight
          const float w = __builtin_amdgcn_exp2f(me - m);
          l += le * w;
#pragma unroll
          for (int k = 0; k < 4; ++k) acc[k] += xch[k][group + e][c] * w;
        }
      }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int k = 0; k < 4; ++k) acc[k] *= inv;
    if (!x.ok) acc = f32x4_t{NAN, NAN, NAN, NAN};
    // Tokens of the request behind this row's last one may have brought in values
    // that are not finite.
    bool bad = false;
#pragma unroll
    for (int k = 0; k < 4; ++k) bad = bad || !(fabsf(acc[k]) < INFINITY);
    const uint64_t any = __builtin_amdgcn_ballot_w64(bad);
    const bool again = x.ok && (!folded || (i + 1 < x.qo && ((any >> (lane & 32)) & 0xffffffffull) != 0));
    if (set == 0 && head < a.hq) {
      if (again) acc = plain_row(a, x, t, head, sees, c);
      *reinterpret_cast<u32x2_t*>(a.o + t * a.o_st + head * a.o_sh + 4 * c) =
          u32x2_t{pack_bf16x2(acc[0], acc[1]), pack_bf16x2(acc[2], acc[3])};
    }
  }
}

int device_cus() {
  int dev = 0, cus = 0;
  if (hipGetDevice(&dev) == hipSuccess &&
      hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) == hipSuccess && cus > 0)
    return cus;
  return 256;
}

// kv heads of a unit: the largest divisor of theirs up to a workgroup's waves.
int heads_per_group(int hkv) {
  for (int n = kWaves; n > 1; --n)
    if (hkv % n == 0) return n;
  return 1;
}

struct Layout {
  int64_t p_o, p_lse, s_o, s_lse, split, total;
};

Layout workspace_layout(const sgl_prefix_plan_t& p) {
  auto align = [](int64_t x) { return (x + 255) / 256 * 256; };
  const int64_t own_rows =
      (p.max_tokens + static_cast<int64_t>(p.max_units) * p.max_qo_len) * p.num_qo_heads;
  Layout l;
  l.p_o = 0;
  l.p_lse = l.p_o + align(p.prefix_rows * kD * 4);
  l.s_o = l.p_lse + align(p.prefix_rows * 4);
  l.s_lse = l.s_o + align(own_rows * kD * 4);
  l.split = l.s_lse + align(own_rows * 4);
  l.total = l.split + align(sizeof(FoldSplit));
  return l;
}

// What a plan's sizes may be; the device is asked for its CUs only behind this.
int check_sizes(int prefix_len, int batch_size, int max_tokens, int max_qo_len, int num_qo_heads,
                int num_kv_heads, int head_dim) {
  if (prefix_len < 0 || batch_size < 0 || max_tokens < 0 || max_qo_len < 0 || num_qo_heads <= 0 ||
      num_kv_heads <= 0 || num_qo_heads % num_kv_heads != 0)
    return SGL_ERR_INVALID_ARG;
  const int group = num_qo_heads / num_kv_heads;
  if (head_dim != kD || group > 64 || max_qo_len > SGL_PREFIX_MAX_QO ||
      num_kv_heads > 65535 || prefix_len > (1 << 29) || batch_size > (1 << 25))
    return SGL_ERR_UNSUPPORTED;
  // Packed rows are counted in 32 bits, and so are the threads of the fold's launch, a
  // workgroup of 256 a token from kFoldGroups tokens on.
  if (static_cast<int64_t>(max_tokens) * group > (1 << 30) || max_tokens >= 1 << 24 ||
      static_cast<int64_t>(max_tokens) * num_qo_heads > 0x7fffffff)
    return SGL_ERR_UNSUPPORTED;
  return SGL_OK;
}

// The plan for workgroups `blocks`; everything else follows from the sizes.
int make_plan(int prefix_len, int batch_size, int max_tokens, int max_qo_len, int num_qo_heads,
              int num_kv_heads, int head_dim, int blocks, sgl_prefix_plan_t& p) {
  const int st = check_sizes(prefix_len, batch_size, max_tokens, max_qo_len, num_qo_heads, num_kv_heads, head_dim);
  if (st != SGL_OK) return st;
  if (blocks < 2 || blocks > 1022) return SGL_ERR_INVALID_ARG;
  const int64_t rows = static_cast<int64_t>(max_tokens) * (num_qo_heads / num_kv_heads);
  const int64_t row_tiles = (rows + 32 * kWaves - 1) / (32 * kWaves);
  p = sgl_prefix_plan_t{};
  p.prefix_len = prefix_len, p.batch_size = batch_size, p.max_tokens = max_tokens, p.max_qo_len = max_qo_len;
  p.num_qo_heads = num_qo_heads, p.num_kv_heads = num_kv_heads, p.head_dim = head_dim;
  p.num_blocks = blocks;
  const int heads = heads_per_group(num_kv_heads);
  const int64_t units = static_cast<int64_t>(blocks) * (kWaves / heads) / (num_kv_heads / heads);
  p.max_units = static_cast<int32_t>(units < 1 ? 1 : units);
  // Two runs of a row tile and head, or as many as there are workgroups, of up to 128 rows.
  if (prefix_len > 0) p.prefix_rows = (blocks + 2 * row_tiles * num_kv_heads) * std::min<int64_t>(rows, 32 * kWaves);
  p.workspace_bytes = workspace_layout(p).total;
  return SGL_OK;
}

template <int RB>
void launch_attention(const PrefixArgs& a, hipStream_t s) {
  hipLaunchKernelGGL(prefix_attention_kernel<RB>, dim3(a.blocks), dim3(64 * kWaves), 0, s, a);
}

}  // namespace
}  // namespace sgl

using namespace sgl;

extern "C" int sgl_prefix_plan(int prefix_len, int batch_size, int max_tokens, int max_qo_len,
                               int num_qo_heads, int num_kv_heads, int head_dim,
                               sgl_prefix_plan_t* plan) {
  if (!plan) return SGL_ERR_INVALID_ARG;
  const int st = check_sizes(prefix_len, batch_size, max_tokens, max_qo_len, num_qo_heads, num_kv_heads, head_dim);
  if (st != SGL_OK) return st;
  return make_plan(prefix_len, batch_size, max_tokens, max_qo_len, num_qo_heads, num_kv_heads, head_dim,
                   std::min(2 * device_cus(), 1022), *plan);
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
  // The maximum of the scores is taken before the scale.
  if (!(sm_scale > 0.f) || !isfinite(sm_scale)) return SGL_ERR_INVALID_ARG;
  if (num_qo_heads != plan->num_qo_heads || num_kv_heads != plan->num_kv_heads ||
      head_dim != plan->head_dim)
    return SGL_ERR_INVALID_ARG;
  // A plan as sgl_prefix_plan makes it.
  sgl_prefix_plan_t p;
  int st = make_plan(plan->prefix_len, plan->batch_size, plan->max_tokens, plan->max_qo_len,
                     num_qo_heads, num_kv_heads, head_dim, plan->num_blocks, p);
  if (st != SGL_OK) return st;
  if (plan->max_units != p.max_units || plan->prefix_rows != p.prefix_rows) return SGL_ERR_INVALID_ARG;
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
  a.inv_group = (65536u + a.group - 1) / a.group;
  a.prefix = p.prefix_len, a.max_qo = p.max_qo_len, a.blocks = p.num_blocks;
  a.heads = heads_per_group(num_kv_heads), a.side = kWaves / a.heads, a.rest = num_kv_heads / a.heads;
  a.scale_log2 = sm_scale * 1.4426950408889634f;
  a.o = static_cast<uint16_t*>(o), a.o_st = o_stride_token, a.o_sh = o_stride_head;
  a.p_o = reinterpret_cast<float*>(ws + l.p_o), a.p_lse = reinterpret_cast<float*>(ws + l.p_lse);
  a.s_o = reinterpret_cast<float*>(ws + l.s_o), a.s_lse = reinterpret_cast<float*>(ws + l.s_lse);
  a.split = reinterpret_cast<FoldSplit*>(ws + l.split);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  // Row blocks of a request's own tokens. One and two, 64 requests of 300 own tokens,
  // 32q/8kv: 1 query token (4 rows) 21.0 and 21.5 us, 4 (16) 25.9 and 26.9, 5 38.6 and 29.6.
  if (p.max_qo_len * a.group <= 16) launch_attention<1>(a, s);
  else launch_attention<2>(a, s);
  st = launch_status();
  if (st != SGL_OK) return st;
  // Lanes of a row. A row has about 32,768 / rows pieces of the prefix (two workgroups of
  // tiles per 128 rows and CU), at most one a tile, and a group of 32 lanes takes 4 or 8 in
  // turn. us with 1, 2 and 8 groups: 128 rows behind 4,096 tokens 19.1, 14.4 and 12.3,
  // 1,024 behind 1,024 17.8, 13.9, 16.8, 2,048 behind 4,096 22.7, 21.1, 23.6, 4,096 behind
  // 1,024 20.1, 24.5, 32.3.
  const int64_t rows = static_cast<int64_t>(max_tokens) * num_qo_heads;
  const int sets = p.prefix_len == 0 || rows > 2048 ? 1 : rows <= 256 && p.prefix_len > 16 * pf::kBN ? 8 : 2;
  const int rows_per = 8 / sets;
  const int all_iters = (num_qo_heads + rows_per - 1) / rows_per;
  int iters = static_cast<int>(std::min<int64_t>((static_cast<int64_t>(max_tokens) * all_iters + kFoldGroups - 1) / kFoldGroups, all_iters));
  iters = std::max(iters, 1);
  const int head_groups = (all_iters + iters - 1) / iters;
  const dim3 fold(static_cast<uint32_t>(max_tokens) * head_groups);
  if (sets == 8) hipLaunchKernelGGL(prefix_fold_kernel<8>, fold, dim3(256), 0, s, a, head_groups, iters);
  else if (sets == 2) hipLaunchKernelGGL(prefix_fold_kernel<2>, fold, dim3(256), 0, s, a, head_groups, iters);
  else hipLaunchKernelGGL(prefix_fold_kernel<1>, fold, dim3(256), 0, s, a, head_groups, iters);
  return launch_status();
}
