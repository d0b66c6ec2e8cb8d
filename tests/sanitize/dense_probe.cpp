// Argument probes of the entry points of the dense routed products, the
// adapters, the typed combine and the plan over several workgroups, built like
// abi_probe.cpp: all-zero / all-null, -1 and huge arguments, then sizes whose
// products would overflow behind pointers that are not null. Every call must
// return KEEP_OK or KEEP_EINVAL without reading memory and without undefined
// behaviour.
#include <cstdio>
#include <cstring>
#include <limits>
#include <type_traits>

#include "keep_amd.h"

template <class T>
T fill(int mode) {
  if constexpr (std::is_pointer_v<T>) return mode < 3 ? nullptr : (T)(uintptr_t)256;
  else if (mode == 0) return T(0);
  else if (mode == 1) return T(-1);
  else if (mode == 2) return std::numeric_limits<T>::max() / 3;
  else if (mode == 3) return sizeof(T) == 8 ? T(0x7fffffff) : T(1);  // every size at its limit
  else return sizeof(T) == 8 ? T(128) : T(mode == 4 ? 1 : 9);        // and a small one, with a flag that is no type
}

static int failures = 0;

template <class R, class... A>
void probe(const char* name, R (*f)(A...)) {
  for (int mode = 0; mode < 6; ++mode) {
    if (mode == 4 && sizeof(R) == 4) continue;  // (valid sizes: a launch)
    R r = f(fill<A>(mode)...);
    if constexpr (std::is_same_v<R, int>) {
      if (r != KEEP_OK && r != KEEP_EINVAL && !(r == 1 && std::strstr(name, "supported"))) {
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
  PROBE(keep_route_combine_rows);
  PROBE(keep_route_combine_grad);
  PROBE(keep_route_plan_blocks);
  PROBE(keep_route_plan_blocks_workspace_bytes);
  PROBE(keep_gather_mm);
  PROBE(keep_gather_mm_tile_supported);
  PROBE(keep_gather_mm_grad_weight);
  PROBE(keep_lora);
  PROBE(keep_lora_workspace_bytes);
  PROBE(keep_lora_rank_stride);
  PROBE(keep_lora_backward);
  PROBE(keep_lora_backward_workspace_bytes);
  // the rank in range, every other size at its limit
  const int64_t m = 0x7fffffff;
  void* p = (void*)(uintptr_t)256;
  if (keep_lora(p, 1, m, p, p, nullptr, (int32_t*)p, m, 1, m, 128, m, m, nullptr, 1, nullptr, 0, p, m, p, 1, nullptr) !=
      KEEP_EINVAL)
    ++failures;
  if (keep_lora_backward(p, 1, m, p, p, nullptr, (int32_t*)p, m, 1, 1024, 128, m, m, (float*)p, p, p, p, p, 1, p, m,
                         nullptr) != KEEP_EINVAL)
    ++failures;
  if (keep_lora_backward_workspace_bytes(0, m, m, m, 128, m, m, 1, 1) != 0) ++failures;
  if (keep_lora_backward_workspace_bytes(0, 64, 2, 4, 16, 64, 32, 1, 1) <= 0) ++failures;
  if (std::strlen(keep_last_error()) == 0) ++failures;  // the probes above left a message
  std::printf("%s: %d failures\n", failures ? "FAIL" : "ok", failures);
  return failures ? 1 : 0;
}
