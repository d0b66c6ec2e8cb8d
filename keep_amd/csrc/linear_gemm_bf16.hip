// The dense projection's products through LDS (linear_gemm_dev.h) on bf16 values.
#include "linear_gemm_dev.h"

namespace keep {

void linear_gemm_bf16(const LinearGemmArgs& a, int mode, int tile, hipStream_t s) { linear_gemm_mode<bf16s>(a, mode, tile, s); }

}  // namespace keep
