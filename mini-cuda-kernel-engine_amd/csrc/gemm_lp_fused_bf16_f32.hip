// The 16-bit product with its epilogue, bf16 operands and f32 output.
#include "gemm_lp_launch.hpp"

namespace mcke_amd {

int launch_fused_bf16_f32(int ti, const LpArgs<Epilogue>& x, bool vec) {
  return LpTable<__bf16, float>::launch(ti, x, vec);
}

}  // namespace mcke_amd
