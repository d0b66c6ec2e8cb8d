// The dense projection's products through LDS (linear_gemm_dev.h) on f32 values.
#include "linear_gemm_dev.h"

namespace keep {

void linear_gemm_f32(const LinearGemmArgs& a, int mode, int tile, hipStream_t s) { linear_gemm_mode<float>(a, mode, tile, s); }

}  // namespace keep
