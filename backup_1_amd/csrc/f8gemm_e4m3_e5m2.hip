// Scaled 8-bit products of e4m3 rows with e5m2 columns.
#include "f8gemm_launch.hpp"

namespace decx_hip {

int f8gemm_launch_e4m3_e5m2(const F8GemmArgs& g, bool e8m0) { return launch_f8gemm_kind<0, 1>(g, e8m0); }

}  // namespace decx_hip
