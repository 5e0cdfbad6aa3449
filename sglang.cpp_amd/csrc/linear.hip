// sgl_linear: a projection with its epilogue.
#include "tile.h"

namespace sgl {
namespace {

bool gated(int act) { return act == SGL_ACT_SILU_AND_MUL || act == SGL_ACT_GELU_AND_MUL; }

// Tiles of 256 x 256 where they fill the CUs, of 128 x 128 otherwise.
template <int DT, bool GATED>
int run_tiles(const gemm::Args& a, hipStream_t s) {
  const int64_t t = a.tokens, rows = static_cast<int64_t>(a.n) * (GATED ? 2 : 1);
  if ((t + 255) / 256 * ((rows + 255) / 256) >= 256)
    return gemm::launch_tile<DT, gemm::kLinear, GATED, 2, 4, 4, 2>(a, (t + 255) / 256, s);
  return gemm::launch_tile<DT, gemm::kLinear, GATED, 2, 2, 2, 2>(a, (t + 127) / 128, s);
}

template <int DT>
int run(const gemm::Args& a, bool vec, hipStream_t s) {
  if (vec && a.tokens <= (gated(a.act) ? gemm::stream_tokens<true>() : gemm::stream_tokens<false>()) && a.x_st <= gemm::kMostStride && a.w_st <= gemm::kMostStride) {
    gemm::StreamArgs st{};
    st.g = a;
    return gated(a.act) ? gemm::launch_stream<DT, gemm::kLinear, true>(st, a.tokens, 1, s)
                        : gemm::launch_stream<DT, gemm::kLinear, false>(st, a.tokens, 1, s);
  }
  if (vec && a.x_st <= gemm::kMostStride && a.w_st <= gemm::kMostStride)
    return gated(a.act) ? run_tiles<DT, true>(a, s) : run_tiles<DT, false>(a, s);
  const int64_t tiles_t = (static_cast<int64_t>(a.tokens) + gemm::kAnyTile - 1) / gemm::kAnyTile;
  return gated(a.act) ? gemm::launch_any<DT, gemm::kLinear, true>(a, vec, tiles_t, s)
                      : gemm::launch_any<DT, gemm::kLinear, false>(a, vec, tiles_t, s);
}

bool aligned(const void* p, int64_t stride, int64_t bytes, int64_t size) {
  return !p || (reinterpret_cast<uintptr_t>(p) % bytes == 0 && stride * size % bytes == 0);
}

constexpr int64_t kMost = 0x7fffff00;  // tokens, outputs and inputs: room for a tile below 2^31

}  // namespace
}  // namespace sgl

using namespace sgl;

extern "C" int64_t sgl_linear_workspace_bytes(int64_t tokens, int64_t n, int64_t k, int activation) {
  (void)tokens, (void)n, (void)k, (void)activation;
  return 0;
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
  a.x = static_cast<const uint16_t*>(x.x), a.x_st = x.x_stride_row;
  a.w = static_cast<const uint16_t*>(x.weight), a.w_st = x.weight_stride_row;
  a.bias = static_cast<const uint16_t*>(x.bias);
  a.res = static_cast<const uint16_t*>(x.residual), a.r_st = x.residual_stride_row;
  a.out = x.out, a.o_st = x.out_stride_row;
  a.tokens = static_cast<int32_t>(x.tokens), a.n = static_cast<int32_t>(x.n);
  a.k = static_cast<int32_t>(x.k), a.act = x.activation;
  a.out_f32 = x.out_dtype == SGL_DTYPE_F32;
  const int64_t size = a.out_f32 ? 4 : 2;
  a.wide = aligned(x.out, x.out_stride_row, 4 * size, size) &&
           aligned(x.residual, x.residual_stride_row, 8, 2) &&
           aligned(x.bias, gated(x.activation) ? x.n : 0, 8, 2);
  const bool vec = x.k % 8 == 0 && aligned(x.x, x.x_stride_row, 16, 2) &&
                   aligned(x.weight, x.weight_stride_row, 16, 2);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  return x.dtype == SGL_DTYPE_BF16 ? run<SGL_DTYPE_BF16>(a, vec, s) : run<SGL_DTYPE_F16>(a, vec, s);
}
