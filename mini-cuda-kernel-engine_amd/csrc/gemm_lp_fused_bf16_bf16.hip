// The 16-bit product with its epilogue, bf16 operands and bf16 output.
#include "gemm_lp_launch.hpp"

namespace mcke_amd {

int launch_fused_bf16_bf16(int ti, const LpArgs<Epilogue>& x, bool vec) {
  return LpTable<__bf16, __bf16>::launch(ti, x, vec);
}

}  // namespace mcke_amd
