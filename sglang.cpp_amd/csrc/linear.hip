// sgl_linear: a projection with its epilogue.
#include "tile.h"

#include <algorithm>

namespace sgl {
namespace {

bool gated(int act) { return act == SGL_ACT_SILU_AND_MUL || act == SGL_ACT_GELU_AND_MUL; }

// The tile kernels' shapes and what a stage of 64 inputs takes them (us, measured): with a
// workgroup for each CU at most, and with all a CU holds.
struct Shape {
  int rows, tokens, per_cu;
  double alone, full;
};
constexpr Shape kShapes[] = {
    {256, 256, 1, 1.55, 1.55},  // 1,340 to 1,380 TFLOP/s where they fill the CUs (8,192 x 24,576 x 4,096)
    {128, 128, 2, 0.70, 1.05},  // 1,090 there; 2,048 x 4,096 x 4,096 takes 72 us, the larger ones 100
    {64, 128, 2, 0.40, 0.55},   // 512 x 4,096 x 4,096: 28 us, the others 48 and 92
};
using gemm::kCus;
using gemm::kMostSplits;

struct Plan {
  int shape, splits;
  int64_t bytes;  // of the parts' sums
  double us;
};

// The shape and the number of parts of k with the least estimated time: rounds of
// workgroups x stages, and for parts their sums written and read at 5 TB/s and another
// launch (333 x 4,096 x 12,288: 128 x 128 tiles in five parts 59 us, in one 163; 100 x 4,096
// x 4,096: 64 x 128 in four 15.6, in one 26).
Plan plan_of(int64_t tokens, int64_t n, int64_t k, int act, bool may_split) {
  const int64_t rows = n * (gated(act) ? 2 : 1), stages = (k + 63) / 64;
  Plan best{0, 1, 0, 1e300};
  for (int i = 0; i < 3; ++i) {
    const Shape& x = kShapes[i];
    const int64_t tiles = ((rows + x.rows - 1) / x.rows) * ((tokens + x.tokens - 1) / x.tokens);
    for (int s = 1; s <= kMostSplits && (s == 1 || (may_split && tiles * s <= 2 * kCus && stages >= 4 * s)); ++s) {
      const int64_t groups = tiles * s, each = (stages + s - 1) / s;
      const int64_t bytes = s > 1 ? groups * x.rows * x.tokens * 4 : 0;
      const int64_t rounds = (groups + kCus * x.per_cu - 1) / (kCus * x.per_cu);
      const double us = 4.0 + (groups <= kCus ? x.alone : x.full) * static_cast<double>(rounds * each) +
                        (s > 1 ? 2.5 + 2.0 * static_cast<double>(bytes) / 5e6 : 0.0);
      if (us < best.us) best = Plan{i, s, bytes, us};
    }
  }
  return best;
}

// Whether the stream kernels take a call: always up to 16 tokens (their rows of x cost what
// the weights' do), above where their estimate, the weights at 5.8 TB/s or what a CU
// stages at 50 GB/s, is the lower one (48 tokens x 4,096 x 4,096: 13 us, tiles 16; 60 x
// 4,096 x 12,288: 37, tiles 29).
bool streams(int64_t tokens, int64_t n, int64_t k, int act, bool may_split) {
  if (tokens > gemm::stream_tokens(gated(act), n)) return false;
  if (tokens <= 16) return true;
  const int tiles = gemm::stream_tiles(gated(act), n, 1);
  const int64_t rows = n * (gated(act) ? 2 : 1), groups = (rows + 16 * tiles - 1) / (16 * tiles);
  const double staged = static_cast<double>((groups + kCus - 1) / kCus * (tiles + (tokens + 15) / 16)) * 32.0 *
                        static_cast<double>(k);
  const double read = 2.0 * static_cast<double>(rows) * static_cast<double>(k);
  return 2.5 + std::max(staged / 5e4, read / 5.8e6) <= plan_of(tokens, n, k, act, may_split).us;
}

template <int DT, bool GATED>
int run_tiles(gemm::Args a, void* workspace, hipStream_t s) {
  const Plan p = plan_of(a.tokens, a.n, a.k, a.act, workspace != nullptr);
  a.splits = p.splits, a.part = static_cast<float*>(workspace);
  const int64_t tiles_t = (static_cast<int64_t>(a.tokens) + kShapes[p.shape].tokens - 1) / kShapes[p.shape].tokens;
  if (p.shape == 0) return gemm::launch_tile<DT, gemm::kLinear, GATED, 2, 4, 4, 2, 2>(a, tiles_t, s);
  if (p.shape == 1) return gemm::launch_tile<DT, gemm::kLinear, GATED, 2, 2, 2, 2, 2>(a, tiles_t, s);
  return gemm::launch_tile<DT, gemm::kLinear, GATED, 1, 4, 2, 1, 3>(a, tiles_t, s);
}

template <int DT>
int run(const gemm::Args& a, bool vec, void* workspace, hipStream_t s) {
  const bool fast = vec && a.x_st <= gemm::kMostStride && a.w_st <= gemm::kMostStride;
  if (fast && streams(a.tokens, a.n, a.k, a.act, workspace != nullptr)) {
    gemm::StreamArgs st{};
    st.g = a;
    return gated(a.act) ? gemm::launch_stream<DT, true>(st, s)
                        : gemm::launch_stream<DT, false>(st, s);
  }
  if (fast) return gated(a.act) ? run_tiles<DT, true>(a, workspace, s) : run_tiles<DT, false>(a, workspace, s);
  if (gemm::takes_any_few(a))
    return gated(a.act) ? gemm::launch_any_few<DT, true>(a, s) : gemm::launch_any_few<DT, false>(a, s);
  const int64_t tiles_t = (static_cast<int64_t>(a.tokens) + gemm::kAnyTile - 1) / gemm::kAnyTile;
  return gated(a.act) ? gemm::launch_any<DT, gemm::kLinear, true>(a, tiles_t, s)
                      : gemm::launch_any<DT, gemm::kLinear, false>(a, tiles_t, s);
}

using gemm::aligned;
constexpr int64_t kMost = 0x7fffff00;  // tokens, outputs and inputs: room for a tile below 2^31

}  // namespace
}  // namespace sgl

using namespace sgl;

extern "C" int64_t sgl_linear_workspace_bytes(int64_t tokens, int64_t n, int64_t k, int activation) {
  if (tokens <= 0 || n <= 0 || k <= 0 || tokens > kMost || n > kMost || k > kMost ||
      activation < SGL_ACT_NONE || activation > SGL_ACT_GELU_AND_MUL || streams(tokens, n, k, activation, true))
    return 0;
  return plan_of(tokens, n, k, activation, true).bytes;
}

extern "C" int sgl_linear(const sgl_linear_t* args, void* workspace, int64_t workspace_bytes,
                          void* stream) {
  if (!args) return SGL_ERR_INVALID_ARG;
  const sgl_linear_t& x = *args;
  if (x.tokens < 0 || x.n <= 0 || x.k <= 0 || x.reserved != 0) return SGL_ERR_INVALID_ARG;
  if (x.dtype != SGL_DTYPE_BF16 && x.dtype != SGL_DTYPE_F16) return SGL_ERR_UNSUPPORTED;
  if (x.out_dtype != x.dtype && x.out_dtype != SGL_DTYPE_F32) return SGL_ERR_UNSUPPORTED;
  if (x.activation < SGL_ACT_NONE || x.activation > SGL_ACT_GELU_AND_MUL) return SGL_ERR_UNSUPPORTED;
  if (x.tokens > kMost || x.n > kMost || x.k > kMost) return SGL_ERR_UNSUPPORTED;
  if (x.tokens == 0) return SGL_OK;
  if (!x.x || !x.weight || !x.out) return SGL_ERR_INVALID_ARG;
  if (x.x_stride_row < x.k || x.weight_stride_row < x.k || x.out_stride_row < x.n ||
      (x.residual && x.residual_stride_row < x.n))
    return SGL_ERR_INVALID_ARG;
  if (x.out == x.x || (x.residual == x.out && (x.out_dtype != x.dtype ||
                                               x.residual_stride_row != x.out_stride_row)))
    return SGL_ERR_INVALID_ARG;
  const int64_t need = sgl_linear_workspace_bytes(x.tokens, x.n, x.k, x.activation);
  if (workspace && workspace_bytes < need) return SGL_ERR_CAPACITY;
  if (workspace && !aligned16(workspace)) return SGL_ERR_ALIGNMENT;
  gemm::Args a{};
  // A single row's stride is nothing that alignment depends on.
  const bool one = x.tokens == 1;
  a.x = static_cast<const uint16_t*>(x.x), a.x_st = one ? 0 : x.x_stride_row;
  a.w = static_cast<const uint16_t*>(x.weight), a.w_st = x.weight_stride_row;
  a.bias = static_cast<const uint16_t*>(x.bias);
  a.res = static_cast<const uint16_t*>(x.residual), a.r_st = one ? 0 : x.residual_stride_row;
  a.out = x.out, a.o_st = one ? 0 : x.out_stride_row;
  a.tokens = static_cast<int32_t>(x.tokens), a.n = static_cast<int32_t>(x.n);
  a.k = static_cast<int32_t>(x.k), a.act = x.activation;
  a.out_f32 = x.out_dtype == SGL_DTYPE_F32;
  const int64_t size = a.out_f32 ? 4 : 2;
  const int64_t rows = gated(x.activation) ? x.n : 0;
  const auto wide = [&](int64_t columns) {
    return aligned(x.out, a.o_st, std::min<int64_t>(16, columns * size), size) &&
           aligned(x.residual, a.r_st, 2 * columns, 2) && aligned(x.bias, rows, 8, 2);
  };
  a.wide = wide(8) ? 2 : wide(4) ? 1 : 0;
  const bool vec = x.k % 8 == 0 && aligned(x.x, a.x_st, 16, 2) &&
                   aligned(x.weight, x.weight_stride_row, 16, 2);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  return x.dtype == SGL_DTYPE_BF16 ? run<SGL_DTYPE_BF16>(a, vec, workspace, s)
                                   : run<SGL_DTYPE_F16>(a, vec, workspace, s);
}
