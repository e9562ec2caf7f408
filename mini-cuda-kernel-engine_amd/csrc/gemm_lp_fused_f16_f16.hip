// The 16-bit product with its epilogue, f16 operands and f16 output.
#include "gemm_lp_launch.hpp"

namespace mcke_amd {

int launch_fused_f16_f16(int ti, const LpArgs<Epilogue>& x, bool vec) {
  return LpTable<_Float16, _Float16>::launch(ti, x, vec);
}

}  // namespace mcke_amd
