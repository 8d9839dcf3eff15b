// Host run of the division by 15 that scales go through (kv4_quant.cuh): every mantissa, at the ends
// of the range that spans of a group have and between, against the correctly rounded quotient.
#include <cmath>
#include <cstdint>
#include <cstdio>

#include "../../llm_fa_b200/csrc/kv4_quant.cuh"

int main() {
  // halves of spans: 2^-118 is below that of the least whose scale counts, 15 * 2^-120; 2^127 is the
  // largest exponent
  for (int e : {-118, -117, -116, -60, -1, 0, 3, 126, 127}) {
    for (uint32_t m = 0; m < (1u << 23); ++m) {
      const float x = std::ldexp(1.f + std::ldexp(static_cast<float>(m), -23), e);
      const volatile float by = 15.f;
      if (llmfa::kv4_fifteenth(x) != x / by) {
        std::printf("failed: %a\n", x);
        return 1;
      }
    }
  }
  std::printf("ok\n");
  return 0;
}
