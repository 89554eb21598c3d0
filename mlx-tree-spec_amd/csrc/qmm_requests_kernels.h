// Launch interface of the per-request operators (include/qmm_requests.h) between their C ABI and kernels.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace qmm4 {

// An index array of 32- or 64-bit integers.
struct Index {
  const void* p;
  bool wide;
  __device__ __forceinline__ int64_t operator[](int64_t i) const {
    return wide ? static_cast<const int64_t*>(p)[i] : static_cast<const int32_t*>(p)[i];
  }
};

// The first factor of the adapters: A [L, R, K], scale [L]; row m uses adapters[m] if that lies in 0 .. L - 1.
struct LoraTables {
  const uint16_t* a;
  const float* scale;
  Index adapters;
  int64_t L;
  int R;
};
// The shrink's grid, and what it needs of the split-K workspace (counters at zero, fp32 tiles).
struct LoraShrinkPlan {
  int rows, across, depth, slices;
  size_t counter_bytes, part_bytes;
};
LoraShrinkPlan lora_shrink_plan(const LoraTables& lora, int M, int K, int cus);
// t [M, R]: t[m, j] = scale * sum_k x[m, k] A[a, j, k] as two bf16 numbers in a word (rows without an adapter are not
// written).
hipError_t launch_lora_shrink(const LoraShrinkPlan& plan, const LoraTables& lora, const uint16_t* x, uint32_t* t,
                              float* part, uint32_t* cnt, int M, int K, hipStream_t stream);

// What a projection's kernel adds to its sums: sum_j t[m, j] B[a, n, j] for the rows with an adapter.
struct LoraAdd {
  const uint32_t* t;
  const uint16_t* b;
  Index adapters;
  int64_t L;
  int R;
};
// The same to a finished y: y[m, n] = bf16(y[m, n] + ..).
hipError_t launch_lora_expand(const LoraAdd& lora, uint16_t* y, int M, int N, hipStream_t stream);

struct RopeHeads {
  const uint16_t* x;
  int64_t row, head;  // strides in elements
  const uint16_t* weight;
  uint16_t* out;      // [M, heads, D]
  int heads;
};
struct RopeParams {
  RopeHeads q, k;
  Index positions;
  const void* inv_freq;
  bool freq64;
  float eps;
  int D, P;
};
hipError_t launch_qk_norm_rope(const RopeParams& p, int64_t M, bool interleaved, hipStream_t stream);

// A setting of each row: an array, or one value where it is null.
template <class T>
struct PerRow {
  const T* p;
  T value;
};
struct SampleParams {
  const uint16_t* logits;
  int64_t row_stride;
  const float* uniform;
  PerRow<float> temperature, top_p, min_p;
  PerRow<int32_t> top_k;
  int64_t* tokens;
  float* logprobs;
  int V;
};
// The workspace for M rows on a GPU of `cus` CUs, in bytes.
int64_t sample_workspace(int64_t M, int64_t V, int cus);
hipError_t launch_sample(const SampleParams& p, int64_t M, void* workspace, int cus, hipStream_t stream);

}  // namespace qmm4
