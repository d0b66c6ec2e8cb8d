// Argument probes of the entry points of the norms, the choice of experts and the dense projections, built like
// dense_probe.cpp: all-zero / all-null, -1 and huge arguments, then sizes whose products would overflow behind pointers that
// are not null. Every call must return KEEP_OK or KEEP_EINVAL without reading memory and without undefined behaviour. The
// products through LDS, whose launches no probe reaches, are left out of the build.
#include <cstdio>
#include <cstring>
#include <limits>
#include <type_traits>

#include "../../keep_amd/csrc/linear_dev.h"

namespace keep {
static int reached = 0;
void linear_gemm_bf16(const LinearGemmArgs&, int, int, hipStream_t) { ++reached; }
void linear_gemm_f16(const LinearGemmArgs&, int, int, hipStream_t) { ++reached; }
void linear_gemm_f32(const LinearGemmArgs&, int, int, hipStream_t) { ++reached; }
void linear_gemm_e4m3(const LinearGemmArgs&, int, int, hipStream_t) { ++reached; }
}  // namespace keep

template <class T>
T fill(int mode) {
  if constexpr (std::is_pointer_v<T>) return mode < 3 ? nullptr : (T)(uintptr_t)256;
  else if (mode == 0) return T(0);
  else if (mode == 1) return T(-1);
  else if (mode == 2) return std::numeric_limits<T>::max() / 3;
  else return sizeof(T) == 8 ? T(0x7fffffff) : T(1);  // every size at its limit
}

static int failures = 0;

template <class R, class... A>
void probe(const char* name, R (*f)(A...)) {
  for (int mode = 0; mode < 4; ++mode) {
    R r = f(fill<A>(mode)...);
    if constexpr (std::is_same_v<R, int>) {
      if (r != KEEP_OK && r != KEEP_EINVAL) {
        std::printf("FAIL %s mode %d returned %d: %s\n", name, mode, (int)r, keep_last_error());
        ++failures;
      }
    } else if (r < 0) {
      std::printf("FAIL %s mode %d returned %lld\n", name, mode, (long long)r);
      ++failures;
    }
  }
}

#define PROBE(f) probe(#f, &f)

int main() {
  PROBE(keep_rmsnorm);
  PROBE(keep_rmsnorm_quant);
  PROBE(keep_rmsnorm_grad);
  PROBE(keep_rmsnorm_grad_workspace_bytes);
  PROBE(keep_route_experts);
  PROBE(keep_route_experts_grad);
  PROBE(keep_linear);
  PROBE(keep_linear_workspace_bytes);
  PROBE(keep_linear_q8);
  PROBE(keep_linear_grad);
  PROBE(keep_linear_grad_workspace_bytes);
  // one size in range, the others at their limits
  const int64_t m = 0x7fffffff, top = 1 << 20;
  void* p = (void*)(uintptr_t)256;
  if (keep_linear(p, m, 1, m, p, m, m, m, p, 1, 2, p, 1, p, p, 1, p, m, nullptr) != KEEP_EINVAL) ++failures;
  if (keep_linear(p, 4 * top, 1, m, p, 4 * top, top, top, p, 1, 2, p, 1, p, p, 1, p, m, nullptr) != KEEP_EINVAL) ++failures;
  if (keep_linear_grad(p, p, 2, p, top, p, top, 1, m, top, top, p, p, p, 1, p, m, nullptr) != KEEP_EINVAL) ++failures;
  if (keep_linear_workspace_bytes(KEEP_E4M3, 1 << 17, top, top) < 0) ++failures;
  if (keep_linear_grad_workspace_bytes(0, 1 << 17, top, top) <= 0) ++failures;
  if (keep_rmsnorm_grad_workspace_bytes(m, 16384) <= 0) ++failures;
  if (keep_rmsnorm_grad(p, 2, p, 2, p, (float*)p, m, 16384, p, 2, p, p, p, p, 64, nullptr) != KEEP_EINVAL) ++failures;
  if (keep_route_experts(p, 0, m, 1024, 8, nullptr, 1, 1, 0, 1, 1.f, (int32_t*)p, (float*)p, nullptr, nullptr) != KEEP_EINVAL)
    ++failures;
  if (std::strlen(keep_last_error()) == 0) ++failures;  // the probes above left a message
  if (keep::reached) ++failures;
  std::printf("%s: %d failures\n", failures ? "FAIL" : "ok", failures);
  return failures ? 1 : 0;
}
