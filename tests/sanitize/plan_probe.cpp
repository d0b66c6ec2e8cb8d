// The plan of a dense projection's products (linear.hip's own rule) for calls given on the standard input, a line each:
// dtype M N K grad -> "mode tile slices" of the forward product, and with grad of dx's and dW's. Host code alone, without the
// HIP runtime: nothing is launched, and the kernels' registration at the start has nowhere to go.
#include <cstdio>

#include "../../keep_amd/csrc/linear.hip"

namespace keep {
void linear_gemm_bf16(const LinearGemmArgs&, int, int, hipStream_t) {}
void linear_gemm_f16(const LinearGemmArgs&, int, int, hipStream_t) {}
void linear_gemm_f32(const LinearGemmArgs&, int, int, hipStream_t) {}
void linear_gemm_e4m3(const LinearGemmArgs&, int, int, hipStream_t) {}
}  // namespace keep

extern "C" {
void** __hipRegisterFatBinary(const void*) { return nullptr; }
void __hipRegisterFunction(void**, const void*, char*, const char*, unsigned, void*, void*, void*, void*, int*) {}
void __hipUnregisterFatBinary(void**) {}
}

int main() {
  int dtype, grad;
  long long M, N, K;
  while (std::scanf("%d %lld %lld %lld %d", &dtype, &M, &N, &K, &grad) == 5) {
    const LinearPlan f = linear_plan(dtype, LINEAR_FORWARD, N, M, K);
    std::printf("%d %d %d", LINEAR_FORWARD, f.tile, f.slices);
    if (grad) {
      const LinearGradPlan g = linear_grad_plan(dtype, M, N, K);
      std::printf(" %d %d %d %d %d %d", LINEAR_ROWS, g.rows.tile, g.rows.slices, LINEAR_WEIGHT, g.weight.tile, g.weight.slices);
    }
    std::printf("\n");
  }
}
