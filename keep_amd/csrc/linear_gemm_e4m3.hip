// The dense projection's products through LDS (linear_gemm_dev.h) on e4m3 values.
#include "linear_gemm_dev.h"

namespace keep {

void linear_gemm_e4m3(const LinearGemmArgs& a, int mode, int tile, hipStream_t s) { linear_gemm_mode<e4m3s>(a, mode, tile, s); }

}  // namespace keep
