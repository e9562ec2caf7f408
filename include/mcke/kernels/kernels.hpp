// mcke/kernels/kernels.hpp -- the kernel launcher API.
//
// Same names, argument order and error behaviour as the reference's
// include/mcke/kernels/kernels.hpp:59-302; each launcher is an inline wrapper
// over the C-ABI in mcke_amd.h (libmcke_amd.so), which owns the gfx950 kernels.
// Launchers never allocate and never synchronise; work goes onto `stream`.
#pragma once

#include <cstddef>
#include <cstdint>
#include <string>

#include "mcke/core/dtype.hpp"
#include "mcke/core/status.hpp"
#include "mcke/kernels/gemm_tile.hpp"
#include "mcke/runtime/stream.hpp"
#include "mcke_amd.h"

namespace mcke::kernels {

namespace detail {
inline Status status_of(int rc) {
  if (rc == MCKE_STATUS_OK) return OkStatus();
  return Status(static_cast<StatusCode>(rc), mcke_last_error());
}
inline mcke_gemm_tile to_c(const GemmTile& t) { return mcke_gemm_tile{t.bm, t.bn, t.bk, t.tm, t.tn}; }
}  // namespace detail

[[nodiscard]] inline Status launch_vector_add_f32(const float* a, const float* b, float* out,
                                                 std::size_t n, rt::StreamHandle stream) {
  return detail::status_of(mcke_launch_vector_add_f32(a, b, out, n, stream));
}

enum class Activation : std::uint8_t { kNone, kRelu, kGeluErf, kGeluTanh };

[[nodiscard]] inline Status launch_bias_act_f32(const float* x, const float* bias, float* y,
                                               std::int64_t rows, std::int64_t cols,
                                               Activation act, int vector_width,
                                               rt::StreamHandle stream, int max_row_blocks = 0) {
  return detail::status_of(mcke_launch_bias_act_f32(x, bias, y, rows, cols, static_cast<int>(act),
                                                    vector_width, stream, max_row_blocks));
}

[[nodiscard]] inline Status launch_bias_add_f32(const float* x, const float* bias, float* y,
                                               std::int64_t rows, std::int64_t cols,
                                               int vector_width, rt::StreamHandle stream) {
  return detail::status_of(mcke_launch_bias_add_f32(x, bias, y, rows, cols, vector_width, stream));
}

[[nodiscard]] inline Status launch_activation_f32(const float* x, float* y, std::int64_t n,
                                                 Activation act, int vector_width,
                                                 rt::StreamHandle stream) {
  return detail::status_of(
      mcke_launch_activation_f32(x, y, n, static_cast<int>(act), vector_width, stream));
}

// Largest width in {4, 2, 1} legal for this pointer and column count.
[[nodiscard]] inline int max_vector_width_f32(const void* p, std::int64_t cols) noexcept {
  const auto addr = reinterpret_cast<std::uintptr_t>(p);
  for (int w = 4; w > 1; w >>= 1)
    if (cols % w == 0 && addr % (sizeof(float) * static_cast<std::size_t>(w)) == 0) return w;
  return 1;
}

enum class ReduceKind : std::uint8_t { kSum, kMax, kMean };
enum class ReduceVariant : std::uint8_t { kSmemTree, kWarpShuffle, kTwoPass };

[[nodiscard]] inline std::size_t row_reduce_workspace_bytes(std::int64_t rows, std::int64_t cols,
                                                           ReduceVariant variant) noexcept {
  return mcke_row_reduce_workspace_bytes(rows, cols, static_cast<int>(variant));
}

[[nodiscard]] inline Status launch_row_reduce_f32(const float* x, float* out, std::int64_t rows,
                                                 std::int64_t cols, ReduceKind kind,
                                                 ReduceVariant variant, rt::StreamHandle stream) {
  return detail::status_of(mcke_launch_row_reduce_f32(x, out, rows, cols, static_cast<int>(kind),
                                                      static_cast<int>(variant), stream));
}

[[nodiscard]] inline Status launch_row_reduce_f32(const float* x, float* out, std::int64_t rows,
                                                 std::int64_t cols, ReduceKind kind,
                                                 ReduceVariant variant, float* workspace,
                                                 std::size_t workspace_bytes,
                                                 rt::StreamHandle stream) {
  return detail::status_of(mcke_launch_row_reduce_ws_f32(
      x, out, rows, cols, static_cast<int>(kind), static_cast<int>(variant), workspace,
      workspace_bytes, stream));
}

enum class SoftmaxVariant : std::uint8_t { kThreePass, kOnlineOnePass };

[[nodiscard]] inline Status launch_row_softmax_f32(const float* x, float* y, std::int64_t rows,
                                                  std::int64_t cols, SoftmaxVariant variant,
                                                  rt::StreamHandle stream) {
  return detail::status_of(
      mcke_launch_row_softmax_f32(x, y, rows, cols, static_cast<int>(variant), stream));
}

[[nodiscard]] inline Status launch_gemm_f32(const float* a, const float* b, float* c,
                                           std::int64_t m, std::int64_t n, std::int64_t k,
                                           float alpha, float beta, GemmVariant variant,
                                           GemmTile tile, rt::StreamHandle stream) {
  const mcke_gemm_tile t = detail::to_c(tile);
  return detail::status_of(mcke_launch_gemm_f32(a, b, c, m, n, k, alpha, beta,
                                                static_cast<int>(variant), &t, stream));
}

// No reference counterpart: launch_gemm_f32 (kMfmaF32, beta = 0) and
// launch_bias_act_f32 in one launch, y = act(alpha * A B + bias[col]), with the
// bits of the two launches in sequence (mcke_launch_gemm_bias_act_f32).
[[nodiscard]] inline Status launch_gemm_bias_act_f32(const float* a, const float* b,
                                                    const float* bias, float* y, std::int64_t m,
                                                    std::int64_t n, std::int64_t k, float alpha,
                                                    Activation act, GemmTile tile,
                                                    rt::StreamHandle stream) {
  const mcke_gemm_tile t = detail::to_c(tile);
  return detail::status_of(mcke_launch_gemm_bias_act_f32(a, b, bias, y, m, n, k, alpha,
                                                         static_cast<int>(act), &t, stream));
}

struct GemmKernelAttrs {
  int regs_per_thread = 0;
  std::size_t static_smem_bytes = 0;
  std::size_t local_bytes = 0;
  int threads_per_block = 0;
  int max_blocks_per_sm_api = 0;
};

[[nodiscard]] inline StatusOr<GemmKernelAttrs> gemm_kernel_attrs(GemmVariant variant, GemmTile tile) {
  const mcke_gemm_tile t = detail::to_c(tile);
  mcke_kernel_attrs a{};
  MCKE_RETURN_IF_ERROR(detail::status_of(mcke_gemm_kernel_attrs(static_cast<int>(variant), &t, &a)));
  GemmKernelAttrs out;
  out.regs_per_thread = a.regs_per_thread;
  out.static_smem_bytes = a.static_smem_bytes;
  out.local_bytes = a.local_bytes;
  out.threads_per_block = a.threads_per_block;
  out.max_blocks_per_sm_api = a.max_blocks_per_sm_api;
  return out;
}

// No reference counterpart: the MFMA tile this build picks for a shape.
[[nodiscard]] inline GemmTile mfma_default_tile(std::int64_t m, std::int64_t n, std::int64_t k) {
  mcke_gemm_tile t{};
  (void)mcke_gemm_mfma_default_tile(m, n, k, &t);
  return GemmTile{t.bm, t.bn, t.bk, t.tm, t.tn};
}

// ---------------------------------------------------------------------------
// 16-bit-input GEMM.  No reference counterpart: the reference reserves
// DType::kF16 / kBF16 (dtype.hpp:33-41) but launches fp32 only.  A and B hold
// `ab` values (kBF16 or kF16), products accumulate in fp32, C holds `c` values
// (kF32 or `ab`).  Argument order, validation and status codes follow
// launch_gemm_f32.
// ---------------------------------------------------------------------------
[[nodiscard]] inline Status launch_gemm_lp(const void* a, const void* b, void* c, DType ab, DType cd,
                                          std::int64_t m, std::int64_t n, std::int64_t k,
                                          float alpha, float beta, GemmTile tile,
                                          rt::StreamHandle stream) {
  const mcke_gemm_tile t = detail::to_c(tile);
  return detail::status_of(mcke_launch_gemm_lp(a, b, c, static_cast<int>(ab), static_cast<int>(cd),
                                               m, n, k, alpha, beta, &t, stream));
}

// y = act(alpha * A B + bias[col]) + residual on 16-bit operands in one launch; bias and
// residual may be null, residual may be y (mcke_launch_gemm_lp_bias_act).
[[nodiscard]] inline Status launch_gemm_lp_bias_act(const void* a, const void* b, const void* bias,
                                                   const void* residual, void* y, DType ab,
                                                   DType yd, DType bias_dtype, std::int64_t m,
                                                   std::int64_t n, std::int64_t k, float alpha,
                                                   Activation act, GemmTile tile,
                                                   rt::StreamHandle stream) {
  const mcke_gemm_tile t = detail::to_c(tile);
  return detail::status_of(mcke_launch_gemm_lp_bias_act(
      a, b, bias, residual, y, static_cast<int>(ab), static_cast<int>(yd),
      static_cast<int>(bias_dtype), m, n, k, alpha, static_cast<int>(act), &t, stream));
}

// The 16-bit GEMM tile this build picks for a shape.
[[nodiscard]] inline GemmTile lp_default_tile(std::int64_t m, std::int64_t n, std::int64_t k) {
  mcke_gemm_tile t{};
  (void)mcke_gemm_lp_default_tile(m, n, k, &t);
  return GemmTile{t.bm, t.bn, t.bk, t.tm, t.tn};
}

// Whether the 16-bit GEMM is instantiated for a tile: (256,256,64,16,16),
// (128,128,64,8,8) or (64,64,64,4,4).
[[nodiscard]] constexpr bool gemm_lp_tile_is_supported(const GemmTile& t) {
  return t.bk == 64 && t.bm == t.bn && (t.bm == 256 || t.bm == 128 || t.bm == 64) &&
         t.tm == t.bm / 16 && t.tn == t.bn / 16;
}

// ---------------------------------------------------------------------------
// Layer norm and token log probabilities.  No reference counterparts; formulas,
// optional (null) operands and special rows are those of mcke_amd.h.
// ---------------------------------------------------------------------------
[[nodiscard]] inline Status launch_layer_norm(const void* x, const void* weight, const void* bias,
                                             void* y, float* mean, float* rstd, DType dtype,
                                             DType param_dtype, std::int64_t rows,
                                             std::int64_t cols, float eps,
                                             rt::StreamHandle stream) {
  return detail::status_of(mcke_launch_layer_norm(x, weight, bias, y, mean, rstd,
                                                  static_cast<int>(dtype),
                                                  static_cast<int>(param_dtype), rows, cols, eps,
                                                  stream));
}

[[nodiscard]] inline std::size_t layer_norm_backward_workspace_bytes(std::int64_t rows,
                                                                    std::int64_t cols) noexcept {
  return mcke_layer_norm_backward_workspace_bytes(rows, cols);
}

[[nodiscard]] inline Status launch_layer_norm_backward(
    const void* dy, const void* x, const void* weight, const float* mean, const float* rstd,
    void* dx, void* dweight, void* dbias, DType dtype, DType param_dtype, std::int64_t rows,
    std::int64_t cols, void* workspace, std::size_t workspace_bytes, rt::StreamHandle stream) {
  return detail::status_of(mcke_launch_layer_norm_backward(
      dy, x, weight, mean, rstd, dx, dweight, dbias, static_cast<int>(dtype),
      static_cast<int>(param_dtype), rows, cols, workspace, workspace_bytes, stream));
}

[[nodiscard]] inline std::size_t token_logprobs_workspace_bytes(std::int64_t rows,
                                                               std::int64_t vocab,
                                                               int top_k) noexcept {
  return mcke_token_logprobs_workspace_bytes(rows, vocab, top_k);
}

[[nodiscard]] inline Status launch_token_logprobs(
    const void* logits, const std::int64_t* tokens, float* logprobs, float* entropy, float* lse,
    float* top_logprobs, std::int64_t* top_ids, DType dtype, std::int64_t rows,
    std::int64_t vocab, std::int64_t row_stride, float scale, int top_k, void* workspace,
    std::size_t workspace_bytes, rt::StreamHandle stream) {
  return detail::status_of(mcke_launch_token_logprobs(
      logits, tokens, logprobs, entropy, lse, top_logprobs, top_ids, static_cast<int>(dtype), rows,
      vocab, row_stride, scale, top_k, workspace, workspace_bytes, stream));
}

[[nodiscard]] inline Status launch_token_logprobs_backward(
    const void* logits, const std::int64_t* tokens, const float* lse, const float* entropy,
    const float* dlogprobs, const float* dentropy, void* dlogits, DType dtype, std::int64_t rows,
    std::int64_t vocab, std::int64_t row_stride, float scale, rt::StreamHandle stream) {
  return detail::status_of(mcke_launch_token_logprobs_backward(
      logits, tokens, lse, entropy, dlogprobs, dentropy, dlogits, static_cast<int>(dtype), rows,
      vocab, row_stride, scale, stream));
}

// ---------------------------------------------------------------------------
// Embedding, bias + activation kept in 8 bits, cross entropy of hidden states.  No
// reference counterparts; formulas, optional (null) operands and special rows are
// those of mcke_amd.h.
// ---------------------------------------------------------------------------
[[nodiscard]] inline Status launch_embedding(const std::int64_t* tokens, const void* table,
                                            void* out, DType table_dtype, DType out_dtype,
                                            std::int64_t rows, std::int64_t vocab,
                                            std::int64_t cols, float scale,
                                            rt::StreamHandle stream) {
  return detail::status_of(mcke_launch_embedding(tokens, table, out, static_cast<int>(table_dtype),
                                                 static_cast<int>(out_dtype), rows, vocab, cols,
                                                 scale, stream));
}

[[nodiscard]] inline std::size_t embedding_backward_workspace_bytes(std::int64_t rows,
                                                                   std::int64_t vocab,
                                                                   std::int64_t cols) noexcept {
  return mcke_embedding_backward_workspace_bytes(rows, vocab, cols);
}

[[nodiscard]] inline Status launch_embedding_backward(
    const std::int64_t* tokens, const void* dout, void* dtable, DType dout_dtype,
    DType table_dtype, std::int64_t rows, std::int64_t vocab, std::int64_t cols, float scale,
    bool accumulate, void* workspace, std::size_t workspace_bytes, rt::StreamHandle stream) {
  return detail::status_of(mcke_launch_embedding_backward(
      tokens, dout, dtable, static_cast<int>(dout_dtype), static_cast<int>(table_dtype), rows,
      vocab, cols, scale, accumulate ? 1 : 0, workspace, workspace_bytes, stream));
}

[[nodiscard]] inline Status launch_bias_act_checkpoint8(
    const void* x, const void* bias, void* y, std::uint8_t* codes, std::uint8_t* exponents,
    DType dtype, DType bias_dtype, std::int64_t rows, std::int64_t cols, Activation act,
    rt::StreamHandle stream) {
  return detail::status_of(mcke_launch_bias_act_checkpoint8(
      x, bias, y, codes, exponents, static_cast<int>(dtype), static_cast<int>(bias_dtype), rows,
      cols, static_cast<int>(act), stream));
}

[[nodiscard]] inline std::size_t bias_act_checkpoint8_backward_workspace_bytes(
    std::int64_t rows, std::int64_t cols) noexcept {
  return mcke_bias_act_checkpoint8_backward_workspace_bytes(rows, cols);
}

[[nodiscard]] inline Status launch_bias_act_checkpoint8_backward(
    const void* dy, const std::uint8_t* codes, const std::uint8_t* exponents, void* dx, void* y,
    void* dbias, DType dtype, DType bias_dtype, std::int64_t rows, std::int64_t cols,
    Activation act, void* workspace, std::size_t workspace_bytes, rt::StreamHandle stream) {
  return detail::status_of(mcke_launch_bias_act_checkpoint8_backward(
      dy, codes, exponents, dx, y, dbias, static_cast<int>(dtype), static_cast<int>(bias_dtype),
      rows, cols, static_cast<int>(act), workspace, workspace_bytes, stream));
}

[[nodiscard]] inline std::size_t linear_cross_entropy_workspace_bytes(std::int64_t rows,
                                                                     std::int64_t vocab,
                                                                     std::int64_t dim) noexcept {
  return mcke_linear_cross_entropy_workspace_bytes(rows, vocab, dim);
}

[[nodiscard]] inline Status launch_linear_cross_entropy(
    const void* hidden, const void* weight, const std::int64_t* targets, float* loss, float* lse,
    DType dtype, std::int64_t rows, std::int64_t vocab, std::int64_t dim, float scale,
    void* workspace, std::size_t workspace_bytes, rt::StreamHandle stream) {
  return detail::status_of(mcke_launch_linear_cross_entropy(
      hidden, weight, targets, loss, lse, static_cast<int>(dtype), rows, vocab, dim, scale,
      workspace, workspace_bytes, stream));
}

[[nodiscard]] inline std::size_t linear_cross_entropy_backward_workspace_bytes(
    std::int64_t rows, std::int64_t vocab, std::int64_t dim) noexcept {
  return mcke_linear_cross_entropy_backward_workspace_bytes(rows, vocab, dim);
}

[[nodiscard]] inline Status launch_linear_cross_entropy_backward(
    const void* hidden, const void* weight, const std::int64_t* targets, const float* lse,
    const float* dloss, const float* dlse, void* dhidden, void* dweight, DType dtype,
    std::int64_t rows, std::int64_t vocab, std::int64_t dim, float scale, void* workspace,
    std::size_t workspace_bytes, rt::StreamHandle stream) {
  return detail::status_of(mcke_launch_linear_cross_entropy_backward(
      hidden, weight, targets, lse, dloss, dlse, dhidden, dweight, static_cast<int>(dtype), rows,
      vocab, dim, scale, workspace, workspace_bytes, stream));
}

}  // namespace mcke::kernels
