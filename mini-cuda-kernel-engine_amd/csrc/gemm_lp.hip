// gemm_lp.hip -- the 16-bit-input GEMM entry points (bf16 / fp16 in, fp32
// accumulation, fp32 or 16-bit out) over gemm_lp_launch.hpp.
//
// The reference reserves DType::kF16 and kBF16 (include/mcke/core/dtype.hpp:33-41)
// for tensor-core inputs but ships only the fp32 launcher (kernels.hpp:265-269,
// gemm.cu:829-882).  mcke_launch_gemm_lp keeps that launcher's argument order,
// validation and status codes, with the two dtypes added after the pointers.
#include <hip/hip_runtime.h>

#include <string>

#include "common.hpp"
#include "gemm_lp_launch.hpp"

namespace mcke_amd {
namespace {

// (ab_dtype, c_dtype) -> 0..3, or -1 when the pair is not supported.
int lp_combo(int ab, int cd) {
  if (ab == MCKE_DTYPE_BF16) return cd == MCKE_DTYPE_F32 ? 0 : cd == MCKE_DTYPE_BF16 ? 1 : -1;
  if (ab == MCKE_DTYPE_F16) return cd == MCKE_DTYPE_F32 ? 2 : cd == MCKE_DTYPE_F16 ? 3 : -1;
  return -1;
}

int check_combo(const char* who, int ab, int cd, int* combo, const char* out = "c_dtype") {
  if (ab != MCKE_DTYPE_BF16 && ab != MCKE_DTYPE_F16)
    return invalid(std::string(who) + ": ab_dtype must be MCKE_DTYPE_BF16 or MCKE_DTYPE_F16, got " +
                   std::to_string(ab));
  *combo = lp_combo(ab, cd);
  if (*combo < 0)
    return invalid(std::string(who) + ": " + out + " must be MCKE_DTYPE_F32 or ab_dtype, got " +
                   std::to_string(cd));
  return ok();
}

int check_tile(const char* who, const mcke_gemm_tile* tile, int* ti) {
  *ti = lp_tile_index(tile);
  if (*ti < 0)
    return invalid(std::string(who) +
                   ": instantiated for tiles (bm,bn,bk,tm,tn) = (256,256,64,16,16), "
                   "(128,128,64,8,8) and (64,64,64,4,4); no fallback is applied");
  return ok();
}

}  // namespace
}  // namespace mcke_amd

using namespace mcke_amd;

extern "C" {

int mcke_launch_gemm_lp(const void* a, const void* b, void* c, int ab_dtype, int c_dtype,
                        int64_t m, int64_t n, int64_t k, float alpha, float beta,
                        const mcke_gemm_tile* tile, void* stream) {
  int combo = -1, ti = -1;
  if (int rc = check_combo("launch_gemm_lp", ab_dtype, c_dtype, &combo)) return rc;
  if (int rc = check_tile("launch_gemm_lp", tile, &ti)) return rc;
  if (m == 0 || n == 0) return ok();
  if (m < 0 || n < 0 || k < 0) return invalid("launch_gemm_lp: negative extent");
  if (!a || !b || !c) return invalid("launch_gemm_lp: null pointer");
  if (a == c || b == c)
    return invalid("launch_gemm_lp: output aliases an input, which violates the "
                   "__restrict__ contract");
  if (m > 2147483647LL || n > 2147483647LL || k > 2147483647LL)
    return invalid("launch_gemm_lp: extent exceeds INT32_MAX");
  // 16-byte loads of eight elements need k % 8, n % 8 and 16-byte aligned bases;
  // the C vector stores need C 16-byte aligned as well.
  const bool vec = (k % 8 == 0) && (n % 8 == 0) && aligned(a, 16) && aligned(b, 16) &&
                   aligned(c, 16);
  const LpArgs<NoEpilogue> x{static_cast<const uint16_t*>(a), static_cast<const uint16_t*>(b), c,
                             static_cast<int>(m), static_cast<int>(n), static_cast<int>(k), alpha,
                             beta, {}, static_cast<hipStream_t>(stream)};
  switch (combo) {
    case 0: return LpTable<__bf16, float>::launch(ti, x, vec);
    case 1: return LpTable<__bf16, __bf16>::launch(ti, x, vec);
    case 2: return LpTable<_Float16, float>::launch(ti, x, vec);
    default: return LpTable<_Float16, _Float16>::launch(ti, x, vec);
  }
}

int mcke_launch_gemm_lp_bias_act(const void* a, const void* b, const void* bias,
                                 const void* residual, void* y, int ab_dtype, int y_dtype,
                                 int bias_dtype, int64_t m, int64_t n, int64_t k, float alpha,
                                 int activation, const mcke_gemm_tile* tile, void* stream) {
  int combo = -1, ti = -1;
  if (int rc = check_combo("launch_gemm_lp_bias_act", ab_dtype, y_dtype, &combo, "y_dtype"))
    return rc;
  if (bias_dtype != MCKE_DTYPE_F32 && bias_dtype != ab_dtype)
    return invalid("launch_gemm_lp_bias_act: bias_dtype must be MCKE_DTYPE_F32 or ab_dtype, got " +
                   std::to_string(bias_dtype));
  if (int rc = check_tile("launch_gemm_lp_bias_act", tile, &ti)) return rc;
  if (activation < MCKE_ACT_NONE || activation > MCKE_ACT_GELU_TANH)
    return invalid("launch_gemm_lp_bias_act: unknown Activation");
  if (m == 0 || n == 0) return ok();
  if (m < 0 || n < 0 || k < 0) return invalid("launch_gemm_lp_bias_act: negative extent");
  if ((k > 0 && (!a || !b)) || !y) return invalid("launch_gemm_lp_bias_act: null pointer");
  if (m > 2147483647LL || n > 2147483647LL || k > 2147483647LL)
    return invalid("launch_gemm_lp_bias_act: extent exceeds INT32_MAX");
  const uint64_t um = m, un = n, uk = k, ye = dtype_bytes(y_dtype), be = dtype_bytes(bias_dtype);
  if (!aligned(a, 2) || !aligned(b, 2) || !aligned(y, ye) || !aligned(residual, ye) ||
      !aligned(bias, be))
    return invalid("launch_gemm_lp_bias_act: a pointer is not aligned to its type");
  if (overlap(y, um * un * ye, a, 2 * um * uk) || overlap(y, um * un * ye, b, 2 * uk * un) ||
      overlap(y, um * un * ye, bias, be * un))
    return invalid("launch_gemm_lp_bias_act: output overlaps an input, which violates the "
                   "__restrict__ contract");
  if (residual != y && overlap(y, um * un * ye, residual, um * un * ye))
    return invalid("launch_gemm_lp_bias_act: the residual overlaps the output without being it");
  const bool vec = (k % 8 == 0) && (n % 8 == 0) && aligned(a, 16) && aligned(b, 16) &&
                   aligned(y, 16);
  const LpArgs<Epilogue> x{static_cast<const uint16_t*>(a), static_cast<const uint16_t*>(b), y,
                           static_cast<int>(m), static_cast<int>(n), static_cast<int>(k), alpha,
                           0.0f, Epilogue{bias, residual, bias_dtype, activation},
                           static_cast<hipStream_t>(stream)};
  switch (combo) {
    case 0: return launch_fused_bf16_f32(ti, x, vec);
    case 1: return launch_fused_bf16_bf16(ti, x, vec);
    case 2: return launch_fused_f16_f32(ti, x, vec);
    default: return launch_fused_f16_f16(ti, x, vec);
  }
}

int mcke_gemm_lp_kernel_attrs(int ab_dtype, int c_dtype, const mcke_gemm_tile* tile,
                              mcke_kernel_attrs* out) {
  if (!out) return invalid("gemm_lp_kernel_attrs: null out");
  int combo = -1, ti = -1;
  if (int rc = check_combo("gemm_lp_kernel_attrs", ab_dtype, c_dtype, &combo)) return rc;
  if (int rc = check_tile("gemm_lp_kernel_attrs", tile, &ti)) return rc;
  LpKernel kern = nullptr;
  switch (combo) {
    case 0: kern = LpTable<__bf16, float>::kernel(ti); break;
    case 1: kern = LpTable<__bf16, __bf16>::kernel(ti); break;
    case 2: kern = LpTable<_Float16, float>::kernel(ti); break;
    default: kern = LpTable<_Float16, _Float16>::kernel(ti); break;
  }
  hipFuncAttributes fa{};
  MCKE_HIP_TRY(hipFuncGetAttributes(&fa, kern));
  out->regs_per_thread = fa.numRegs;
  out->agprs_per_thread = 0;
  out->static_smem_bytes = fa.sharedSizeBytes;
  out->local_bytes = fa.localSizeBytes;
  out->threads_per_block = kMfmaThreads;
  int blocks = 0;
  MCKE_HIP_TRY(hipOccupancyMaxActiveBlocksPerMultiprocessor(&blocks, kern, kMfmaThreads, 0));
  out->max_blocks_per_sm_api = blocks;
  return ok();
}

int mcke_gemm_lp_default_tile(int64_t m, int64_t n, int64_t k, mcke_gemm_tile* out) {
  if (!out) return invalid("gemm_lp_default_tile: null out");
  (void)k;
  // The largest tile that still fills most of a 256-CU part.  Measured on MI355X: 256 x 256
  // wins at 4096^3 (256 tiles) and at 3072 x 4096 x 1024 (192 tiles, bf16: 32.1 us against
  // 33.6), 128 x 128 at 2048^3 (256 tiles: 23.2 us against 37.2 for 64 x 64) and down to
  // 80 tiles (a launch of fewer than 208 that are not whole still splits K where K is short or
  // odd), 64 x 64 at 1024^3 (64 tiles of 128: 12.4 us against 8.8).
  auto tiles = [&](int64_t t) { return ((m + t - 1) / t) * ((n + t - 1) / t); };
  if (tiles(256) >= 192) *out = mcke_gemm_tile{256, 256, kLpBK, 16, 16};
  else if (tiles(128) >= 80) *out = mcke_gemm_tile{128, 128, kLpBK, 8, 8};
  else *out = mcke_gemm_tile{64, 64, kLpBK, 4, 4};
  return ok();
}

}  // extern "C"
