// Mixture of experts: sgl_moe_route (the experts of each token from the router's logits)
// and sgl_moe_experts (their gate, up and down projections and the weighted sum).
#include "tile.h"

#include <algorithm>

namespace sgl {
namespace {

// ------------------------------------------------------------------ route

constexpr int kMostExperts = 512;
constexpr int kMostChosen = 32;

struct RouteArgs {
  const void* logits;
  int64_t stride;
  float* weights;
  int32_t* experts;
  int64_t tokens;
  int32_t num_experts, top_k, renormalize;
};

template <int DT>
__device__ __forceinline__ float load_logit(const void* p, int64_t i) {
  if constexpr (DT == SGL_DTYPE_F32) return static_cast<const float*>(p)[i];
  else return to_f32<DT>(static_cast<const uint16_t*>(p)[i]);
}

// Order of a logit as a whole number: larger logits are larger, NaN is below -inf, and
// -0 is 0. Never 0, which marks an expert already taken.
__device__ __forceinline__ uint32_t rank_of(float x) {
  if (x != x) return 1;
  const uint32_t b = __float_as_uint(x + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// The logit of a rank.
__device__ __forceinline__ float logit_of(uint32_t rank) {
  if (rank == 1) return __builtin_nanf("");
  return __uint_as_float(rank & 0x80000000u ? rank & 0x7fffffffu : ~rank);
}

// Largest and smallest of a row of 16 lanes, in all of them.
__device__ __forceinline__ uint32_t max16(uint32_t x) {
  x = max(x, dpp_u32<0xB1>(x));
  x = max(x, dpp_u32<0x4E>(x));
  x = max(x, dpp_u32<0x141>(x));
  return max(x, dpp_u32<0x140>(x));
}
__device__ __forceinline__ uint32_t min16(uint32_t x) {
  x = min(x, dpp_u32<0xB1>(x));
  x = min(x, dpp_u32<0x4E>(x));
  x = min(x, dpp_u32<0x141>(x));
  return min(x, dpp_u32<0x140>(x));
}

// 16 lanes a token (lane exchanges inside 16 lanes are register moves): expert l + 16 i in
// register i. Each round takes the largest rank and of its experts the lowest; lane j % 16
// keeps the j-th choice. 16,384 tokens of 128 experts, 8 chosen: 7.6 us, the rounds' eight
// dependent lane exchanges each (5 MB read and written: 0.7).
template <int DT, int V>
__global__ __launch_bounds__(256) void route_kernel(const RouteArgs a) {
  const int l = threadIdx.x & 15;
  const int64_t t = static_cast<int64_t>(gemm::group_index()) * 16 + (threadIdx.x >> 4);
  const bool real = t < a.tokens;
  const int64_t row = (real ? t : a.tokens - 1) * a.stride;
  float x[V];
  uint32_t rank[V];
  uint32_t top_rank = 0;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int e = l + 16 * i;
    x[i] = e < a.num_experts ? load_logit<DT>(a.logits, row + e) : 0.f;
  }
#pragma unroll
  for (int i = 0; i < V; ++i) {
    rank[i] = l + 16 * i < a.num_experts ? rank_of(x[i]) : 0;
    top_rank = max(top_rank, rank[i]);
  }
  const float top = logit_of(max16(top_rank));
  float total = 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i) total += l + 16 * i < a.num_experts ? expf(x[i] - top) : 0.f;
  total = group_sum<16>(total);
  uint32_t kept[kMostChosen / 16] = {};
  int32_t expert[kMostChosen / 16] = {};
  auto round = [&](int j, uint32_t& kept_rank, int32_t& kept_expert) {
    uint32_t best = 0, at = 0;
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (rank[i] > best) best = rank[i], at = i;  // of equal ones the first
    const uint32_t most = max16(best);
    const uint32_t e = min16(best == most ? l + 16 * at : 0xffffffffu);
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (e == static_cast<uint32_t>(l + 16 * i)) rank[i] = 0;
    if (l == (j & 15)) kept_rank = most, kept_expert = static_cast<int32_t>(e);
  };
  for (int j = 0; j < min(a.top_k, 16); ++j) round(j, kept[0], expert[0]);
  for (int j = 16; j < a.top_k; ++j) round(j, kept[1], expert[1]);
  float w[kMostChosen / 16], sum = 0.f;
#pragma unroll
  for (int i = 0; i < kMostChosen / 16; ++i) {
    w[i] = l + 16 * i < a.top_k ? expf(logit_of(kept[i]) - top) : 0.f;
    sum += w[i];
  }
  sum = group_sum<16>(sum);
  // A row with a NaN, or no finite logit, has a NaN total and NaN weights.
  const float under = a.renormalize ? sum + (total - total) : total;
#pragma unroll
  for (int i = 0; i < kMostChosen / 16; ++i) {
    const int j = l + 16 * i;
    if (real && j < a.top_k) {
      a.weights[t * a.top_k + j] = w[i] / under;
      a.experts[t * a.top_k + j] = expert[i];
    }
  }
}

template <int DT>
void launch_route(const RouteArgs& a, hipStream_t s) {
  const dim3 grid = gemm::rows_of((a.tokens + 15) / 16), block(256);
  if (a.num_experts <= 64) hipLaunchKernelGGL((route_kernel<DT, 4>), grid, block, 0, s, a);
  else if (a.num_experts <= 128) hipLaunchKernelGGL((route_kernel<DT, 8>), grid, block, 0, s, a);
  else if (a.num_experts <= 256) hipLaunchKernelGGL((route_kernel<DT, 16>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((route_kernel<DT, 32>), grid, block, 0, s, a);
}

// ------------------------------------------------------------------ experts

struct SortArgs {
  const int32_t* experts;  // [slots]
  int32_t* order;          // slots by expert
  int4* tiles;
  int32_t slots, num_experts, tile_rows, num_tiles;
};

constexpr int kSortThreads = 1024;
constexpr int kSortAhead = 16;  // loads of four choices a lane has in flight

// One workgroup an expert counts the slots of lower experts (its first place) and writes
// its own slots and tiles. Every one reads all choices, so that none waits for another's counts
// (65,536 choices of 128 experts 11.9 us, 6,216 5.5; with ballots over single choices, read
// twice, 18.7 and 7.8). Expert e's tiles start at entry first / tile_rows + e: a later expert's
// cannot start inside them, so no expert needs another's tiles.
__global__ __launch_bounds__(kSortThreads) void sort_kernel(const SortArgs a) {
  __shared__ int32_t lower_of[kSortThreads / kWave], own_of[kSortThreads / kWave];
  const int e = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  constexpr int kWaves = kSortThreads / kWave;
  // Wave w has the slots [w per, (w + 1) per).
  constexpr int kRun = 4 * kWave, kStep = kRun * kSortAhead;
  const int per = (a.slots + kSortThreads - 1) / kSortThreads * kWave;
  const int begin = min(a.slots, wave * per), end = min(a.slots, begin + per);
  int32_t x[kSortAhead][4];
  auto load = [&](int i) {
#pragma unroll
    for (int u = 0; u < kSortAhead; ++u) {
      const int at = i + kRun * u + 4 * lane;
      if (i + kRun * u >= end) break;
      if (i + kRun * (u + 1) <= end) {
        __builtin_memcpy(x[u], a.experts + at, 16);
      } else {
#pragma unroll
        for (int c = 0; c < 4; ++c) x[u][c] = at + c < end ? a.experts[at + c] : -1;
      }
    }
  };
  int lower = 0, own = 0;  // of this lane's choices; no expert's number is below none
  for (int i = begin; i < end; i += kStep) {
    load(i);
#pragma unroll
    for (int u = 0; u < kSortAhead; ++u) {
      if (i + kRun * u >= end) break;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        lower += static_cast<uint32_t>(x[u][c]) < static_cast<uint32_t>(e);
        own += x[u][c] == e;
      }
    }
  }
  int before = own;  // in this lane and those below
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) {
    const int low = __shfl_up(before, d, kWave);
    if (lane >= d) before += low;
    lower += __shfl_xor(lower, d, kWave);
  }
  if (lane == kWave - 1) lower_of[wave] = lower, own_of[wave] = before;
  __syncthreads();
  int first = 0, at = 0, count = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    first += lower_of[w];
    at += w < wave ? own_of[w] : 0;
    count += own_of[w];
  }
  at += first + before - own;
  for (int i = begin; i < end; i += kStep) {
    if (begin + kStep < end) load(i);  // else they are still there
#pragma unroll
    for (int u = 0; u < kSortAhead; ++u) {
      if (i + kRun * u >= end) break;
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (x[u][c] == e) a.order[at++] = i + kRun * u + 4 * lane + c;
    }
  }
  const int t0 = first / a.tile_rows + e;
  const int t1 = e + 1 == a.num_experts ? a.num_tiles : (first + count) / a.tile_rows + e + 1;
  for (int t = t0 + tid; t < t1; t += kSortThreads) {
    const int done = (t - t0) * a.tile_rows;
    a.tiles[t] = int4{e, first + done, min(a.tile_rows, count - done), 0};
  }
}

struct CombineArgs {
  const float* y;  // [slots, stride] weighted outputs of the slots
  const int32_t* experts;
  const uint16_t* res;
  uint16_t* out;
  int64_t y_st, r_st, o_st;
  int32_t tokens, hidden, top_k, num_experts, wide;
};

// out[t] = the sum of its slots in their order (+ residual); slots of no expert are skipped.
// Eight outputs a thread, eight slots' loads in flight. y is fp32: a token's terms differ in size and
// may cancel, so none is rounded before their sum.
// Bound by memory: 8 slots of 8,192 tokens x 2,048 109 us (5.2 TB/s).
template <int DT>
__global__ __launch_bounds__(256) void combine_kernel(const CombineArgs a) {
  constexpr int kAhead = 8;
  const int64_t t = gemm::group_index();
  const int h = 8 * (blockIdx.z * 256 + threadIdx.x);
  if (h >= a.hidden || t >= a.tokens) return;
  const int32_t* ids = a.experts + t * a.top_k;
  float sum[8] = {};
  for (int j0 = 0; j0 < a.top_k; j0 += kAhead) {
    u32x4_t v[kAhead][2];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int j = j0 + u;
      const u32x4_t zero = {0, 0, 0, 0};
      const bool in = j < a.top_k && ids[j] >= 0 && ids[j] < a.num_experts;
      const int64_t at = (t * a.top_k + j) * a.y_st + h;
      v[u][0] = in ? ldg128_nt<true>(a.y + at) : zero;
      v[u][1] = in ? ldg128_nt<true>(a.y + at + 4) : zero;
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
#pragma unroll
      for (int i = 0; i < 8; ++i) sum[i] += __uint_as_float(v[u][i / 4][i % 4]);
  }
  uint16_t* o = a.out + t * a.o_st + h;
  const uint16_t* r = a.res ? a.res + t * a.r_st + h : nullptr;
  if (a.wide && h + 8 <= a.hidden) {
    if (r) {
      float f[8];
      unpack8_t<DT>(ldg128(r), f);
#pragma unroll
      for (int i = 0; i < 8; ++i) sum[i] += f[i];
    }
    stg128(o, pack8_t<DT>(sum));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (h + i < a.hidden)
        o[i] = static_cast<uint16_t>(from_f32<DT>(sum[i] + (r ? to_f32<DT>(r[i]) : 0.f)));
  }
}

using gemm::aligned;

constexpr int64_t kMost = 1 << 30;  // choices: a workgroup's share of them stays an int
constexpr int kTileRows = gemm::kAnyTile;
// Slots an expert has on average at most where the weights are streamed: 16 at a time, more
// take another pass (128 experts of 2,048 x 768, 8 a token: 96 tokens 215 us, tiles 234; 128
// tokens 229 and 229). How the choices fall is not known on the host; where all are at one expert
// its passes come one behind the other (147 experts, one a token, spread and all at one: 128 tokens
// 137 and 56 us, 512 222 and 259, 1,024 248 and 503; by tiles 1,025 260 and 83).
constexpr int64_t kFewPlaces = 7;

// The workspace: slots in order, tiles, the rows h between the projections and the weighted
// outputs. Rows are padded to whole 16 bytes. h is rounded to the type: the matrix instructions of the
// down projection take 16-bit operands, and fp32 ones in two 16-bit parts would double its products.
// That is as large an error as rounding the result (against 64 bits 0.0023 to 0.0024 in bf16, 0.0017
// without it; fp16 0.00029 and 0.00021).
struct Layout {
  int64_t num_tiles, h_st, y_st, order, tiles, h, y, bytes;
};

Layout layout_of(int64_t slots, int64_t experts, int64_t hidden, int64_t inter) {
  const auto up = [](int64_t x, int64_t to) { return (x + to - 1) / to * to; };
  Layout l;
  l.num_tiles = slots / kTileRows + experts;
  l.h_st = up(inter, 8);
  l.y_st = up(hidden, 8);
  l.order = 0;
  l.tiles = up(slots * 4, 256);
  l.h = l.tiles + up(l.num_tiles * 16, 256);
  l.y = l.h + up(slots * l.h_st * 2, 256);
  l.bytes = l.y + up(slots * l.y_st * 4, 256);
  return l;
}

bool sizes_ok(int64_t tokens, int64_t top_k, int64_t experts, int64_t hidden, int64_t inter) {
  return tokens >= 0 && top_k > 0 && experts > 0 && hidden > 0 && inter > 0;
}
bool sizes_built(int64_t tokens, int64_t top_k, int64_t experts, int64_t hidden, int64_t inter) {
  return top_k <= kMost && tokens <= kMost / top_k && experts <= 65536 && hidden <= 1 << 20 &&
         inter <= 1 << 20;
}

template <int DT>
int combine(const sgl_moe_t& x, const gemm::Args& down, hipStream_t s) {
  CombineArgs c{};
  c.y = static_cast<const float*>(down.out), c.y_st = down.o_st, c.experts = x.experts;
  c.res = static_cast<const uint16_t*>(x.residual), c.r_st = x.residual_stride_row;
  c.out = static_cast<uint16_t*>(x.out), c.o_st = x.out_stride_row;
  c.tokens = static_cast<int32_t>(x.tokens), c.hidden = x.hidden, c.top_k = x.top_k, c.num_experts = x.num_experts;
  c.wide = aligned(x.out, x.out_stride_row, 16, 2) && aligned(x.residual, x.residual_stride_row, 16, 2);
  dim3 grid = gemm::rows_of(x.tokens);
  grid.z = (x.hidden + 2047) / 2048;
  hipLaunchKernelGGL(combine_kernel<DT>, grid, dim3(256), 0, s, c);
  return launch_status();
}

// Few slots: the workgroups find their expert's slots themselves, rows of h and y are slots.
template <int DT>
int run_few(const sgl_moe_t& x, gemm::Args up, gemm::Args down, hipStream_t s) {
  const int slots = static_cast<int>(x.tokens * x.top_k), tokens = static_cast<int>(x.tokens);
  gemm::StreamArgs st{};
  st.experts = x.experts, st.slots = slots, st.num_experts = x.num_experts;
  st.by_slot = slots < x.num_experts;
  const int rows = st.by_slot ? slots : x.num_experts;
  st.g = up;
  int status = gemm::launch_experts<DT, gemm::kGateUp, true>(st, rows, s);
  if (status != SGL_OK) return status;
  st.g = down;
  if (tokens <= gemm::kFewTokens && slots <= gemm::kFewSlots) {
    st.g.out = x.out, st.g.o_st = x.out_stride_row, st.g.out_f32 = 0;
    st.g.tokens = tokens;
    st.g.wide = aligned(x.out, x.out_stride_row, 8, 2) && aligned(x.residual, x.residual_stride_row, 8, 2);
    constexpr int kTiles = 2, kOut = 4 * kTiles;
    hipLaunchKernelGGL((gemm::down_few_kernel<DT, kTiles, 8>), dim3((x.hidden + kOut - 1) / kOut), dim3(512),
                       0, s, st, static_cast<const uint16_t*>(x.residual), x.residual_stride_row);
    return launch_status();
  }
  status = gemm::launch_experts<DT, gemm::kDown, false>(st, rows, s);
  if (status != SGL_OK) return status;
  return combine<DT>(x, down, s);
}

// Elements of x that the tiles' 32-bit offsets reach (every expert's rows may be anywhere in
// them). More are calls of their parts.
constexpr int64_t kReach = (1ll << 30) - 1;

// The call of `tokens` tokens from `first` on.
sgl_moe_t tokens_of(sgl_moe_t x, int64_t first, int64_t tokens) {
  x.x = static_cast<const uint16_t*>(x.x) + first * x.x_stride_row;
  x.weights += first * x.top_k, x.experts += first * x.top_k;
  if (x.residual) x.residual = static_cast<const uint16_t*>(x.residual) + first * x.residual_stride_row;
  x.out = static_cast<uint16_t*>(x.out) + first * x.out_stride_row;
  x.tokens = tokens;
  return x;
}

template <int DT>
int run(const sgl_moe_t& x, const Layout& l, char* ws, hipStream_t s) {
  const int slots = static_cast<int>(x.tokens * x.top_k);
  int32_t* order = reinterpret_cast<int32_t*>(ws + l.order);
  int4* tiles = reinterpret_cast<int4*>(ws + l.tiles);
  uint16_t* h = reinterpret_cast<uint16_t*>(ws + l.h);
  float* y = reinterpret_cast<float*>(ws + l.y);
  gemm::Args up{};
  up.places = tiles, up.order = order, up.top_k = x.top_k, up.scale = x.weights;
  gemm::Args down = up;
  up.x = static_cast<const uint16_t*>(x.x), up.x_st = x.tokens == 1 ? 0 : x.x_stride_row;
  up.w = static_cast<const uint16_t*>(x.gate_up);
  up.w_st = x.gate_up_stride_row, up.w_se = x.gate_up_stride_expert;
  up.out = h, up.o_st = l.h_st, up.wide = 2;
  up.tokens = slots, up.n = x.intermediate, up.k = x.hidden, up.act = x.activation;
  const bool up_vec = x.hidden % 8 == 0 && aligned(x.x, up.x_st, 16, 2) &&
                      aligned(x.gate_up, x.gate_up_stride_row, 16, 2) &&
                      (x.num_experts == 1 || x.gate_up_stride_expert % 8 == 0);
  down.x = h, down.x_st = l.h_st;
  down.w = static_cast<const uint16_t*>(x.down);
  down.w_st = x.down_stride_row, down.w_se = x.down_stride_expert;
  down.out = y, down.o_st = l.y_st, down.out_f32 = 1, down.wide = 2;
  down.tokens = slots, down.n = x.hidden, down.k = x.intermediate;
  const bool down_vec = x.intermediate % 8 == 0 && aligned(x.down, x.down_stride_row, 16, 2) &&
                        (x.num_experts == 1 || x.down_stride_expert % 8 == 0);
  if (up_vec && down_vec && slots <= gemm::kMostSlots && slots <= kFewPlaces * x.num_experts &&
      std::max({up.x_st, up.w_st, down.x_st, down.w_st}) <= gemm::kMostStride)
    return run_few<DT>(x, up, down, s);

  const bool fast = up_vec && down_vec &&
                    std::max({up.x_st, up.w_st, down.x_st, down.w_st}) <= gemm::kMostStride;
  if (fast && x.tokens * up.x_st > kReach) {
    const int64_t each = kReach / up.x_st;
    for (int64_t t = 0; t < x.tokens; t += each) {
      const int status = run<DT>(tokens_of(x, t, std::min(each, x.tokens - t)), l, ws, s);
      if (status != SGL_OK) return status;
    }
    return SGL_OK;
  }
  const int share = slots / x.num_experts;  // places of an expert, on average
  const int rows = !fast ? gemm::kAnyTile : share <= 64 ? 64 : share < 256 ? 128 : 256;
  const int num_tiles = slots / rows + x.num_experts;
  const SortArgs sort{x.experts, order, tiles, slots, x.num_experts, rows, num_tiles};
  hipLaunchKernelGGL(sort_kernel, dim3(x.num_experts), dim3(kSortThreads), 0, s, sort);
  int st = launch_status();
  if (st != SGL_OK) return st;
  const auto product = [&](auto mode, auto gate, const gemm::Args& a) {
    constexpr int kMode = decltype(mode)::value;
    constexpr bool kGated = decltype(gate)::value;
    if (!fast) return gemm::launch_any<DT, kMode, kGated>(a, num_tiles, s);
    if (rows == 64) return gemm::launch_tile<DT, kMode, kGated, 2, 2, 2, 1, 3>(a, num_tiles, s);
    if (rows == 128) return gemm::launch_tile<DT, kMode, kGated, 2, 2, 2, 2, 2>(a, num_tiles, s);
    return gemm::launch_tile<DT, kMode, kGated, 2, 4, 4, 2, 2>(a, num_tiles, s);
  };
  st = product(std::integral_constant<int, gemm::kGateUp>{}, std::true_type{}, up);
  if (st != SGL_OK) return st;
  st = product(std::integral_constant<int, gemm::kDown>{}, std::false_type{}, down);
  if (st != SGL_OK) return st;
  return combine<DT>(x, down, s);
}

}  // namespace
}  // namespace sgl

using namespace sgl;

extern "C" int sgl_moe_route(const void* logits, int64_t logits_stride_row, int logits_dtype,
                             int64_t tokens, int num_experts, int top_k, int renormalize,
                             float* weights, int32_t* experts, void* stream) {
  if (tokens < 0 || num_experts <= 0 || top_k <= 0 || top_k > num_experts) return SGL_ERR_INVALID_ARG;
  if (num_experts > kMostExperts || top_k > kMostChosen || tokens > kMost) return SGL_ERR_UNSUPPORTED;
  if (logits_dtype < SGL_DTYPE_BF16 || logits_dtype > SGL_DTYPE_F32) return SGL_ERR_UNSUPPORTED;
  if (tokens == 0) return SGL_OK;
  if (!logits || !weights || !experts || logits_stride_row < num_experts) return SGL_ERR_INVALID_ARG;
  const RouteArgs a{logits, logits_stride_row, weights, experts, tokens, num_experts, top_k,
                    renormalize != 0};
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (logits_dtype == SGL_DTYPE_F32) launch_route<SGL_DTYPE_F32>(a, s);
  else if (logits_dtype == SGL_DTYPE_BF16) launch_route<SGL_DTYPE_BF16>(a, s);
  else launch_route<SGL_DTYPE_F16>(a, s);
  return launch_status();
}

extern "C" int64_t sgl_moe_workspace_bytes(int64_t tokens, int top_k, int num_experts, int hidden,
                                           int intermediate) {
  if (!sizes_ok(tokens, top_k, num_experts, hidden, intermediate) ||
      !sizes_built(tokens, top_k, num_experts, hidden, intermediate))
    return 0;
  return layout_of(tokens * top_k, num_experts, hidden, intermediate).bytes;
}

extern "C" int sgl_moe_experts(const sgl_moe_t* args, void* workspace, int64_t workspace_bytes,
                               void* stream) {
  if (!args) return SGL_ERR_INVALID_ARG;
  const sgl_moe_t& x = *args;
  if (!sizes_ok(x.tokens, x.top_k, x.num_experts, x.hidden, x.intermediate)) return SGL_ERR_INVALID_ARG;
  if (x.dtype != SGL_DTYPE_BF16 && x.dtype != SGL_DTYPE_F16) return SGL_ERR_UNSUPPORTED;
  if (x.activation != SGL_ACT_SILU_AND_MUL && x.activation != SGL_ACT_GELU_AND_MUL)
    return SGL_ERR_UNSUPPORTED;
  if (!sizes_built(x.tokens, x.top_k, x.num_experts, x.hidden, x.intermediate))
    return SGL_ERR_UNSUPPORTED;
  if (x.tokens == 0) return SGL_OK;
  if (!x.x || !x.gate_up || !x.down || !x.weights || !x.experts || !x.out) return SGL_ERR_INVALID_ARG;
  if (x.x_stride_row < x.hidden || x.out_stride_row < x.hidden ||
      x.gate_up_stride_row < x.hidden || x.down_stride_row < x.intermediate ||
      (x.residual && x.residual_stride_row < x.hidden) ||
      (x.num_experts > 1 &&
       (x.gate_up_stride_expert < x.gate_up_stride_row * 2 * x.intermediate ||
        x.down_stride_expert < x.down_stride_row * x.hidden)))
    return SGL_ERR_INVALID_ARG;
  if (x.out == x.x || (x.residual == x.out && x.residual_stride_row != x.out_stride_row))
    return SGL_ERR_INVALID_ARG;
  const Layout l = layout_of(x.tokens * x.top_k, x.num_experts, x.hidden, x.intermediate);
  if (!workspace || workspace_bytes < l.bytes) return SGL_ERR_CAPACITY;
  if (!aligned16(workspace)) return SGL_ERR_ALIGNMENT;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  return x.dtype == SGL_DTYPE_BF16 ? run<SGL_DTYPE_BF16>(x, l, ws, s) : run<SGL_DTYPE_F16>(x, l, ws, s);
}
