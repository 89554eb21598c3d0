// The sampling operator's workspace over its whole range of shapes (CPU only: no GPU call). Prints the largest, in bytes.
#include <algorithm>
#include <cstdint>
#include <cstdio>

#include "qmm_requests.h"
#include "qmm_requests_kernels.h"

int main() {
  int64_t most = 0;
  for (int cus : {256, 304, 80, 1})
    for (int64_t v = 1; v <= QMM4_SAMPLE_MAX_VOCAB; v += std::max<int64_t>(1, v / 37))
      for (int64_t m = 1; m <= 1 << 20; m += std::max<int64_t>(1, m / 5)) most = std::max(most, qmm4::sample_workspace(m, v, cus));
  for (int cus : {256, 304, 80, 1})
    for (int64_t m : {1, 3, 255, 256, 257, 1 << 20}) most = std::max(most, qmm4::sample_workspace(m, QMM4_SAMPLE_MAX_VOCAB, cus));
  std::printf("%lld\n", (long long)most);
  // A batch of a model's vocabulary stays one batch: 4 bytes per logit and 8 per slice.
  const int64_t model = qmm4::sample_workspace(256, 151936, 256);
  return model >= 256LL * 151936 * 4 ? 0 : 1;
}
