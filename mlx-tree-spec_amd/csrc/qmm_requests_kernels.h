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

// Adapters a: A [L, R, K], B [L, N, R], scale [L]; row m uses adapters[m] if that lies in 0 .. L - 1.
struct LoraTables {
  const uint16_t* a;
  const uint16_t* b;
  const float* scale;
  Index adapters;
  int64_t L;
  int R;
};
// t[m, j] = scale * sum_k x[m, k] A[a, j, k] (0 for rows without an adapter), fp32 [M, R].
hipError_t launch_lora_shrink(const LoraTables& lora, const uint16_t* x, float* t, int64_t M, int64_t K,
                              hipStream_t stream);
// y[m, n] = bf16(y[m, n] + sum_j t[m, j] B[a, n, j]) for rows with an adapter.
hipError_t launch_lora_expand(const LoraTables& lora, const float* t, uint16_t* y, int64_t M, int64_t N,
                              hipStream_t stream);

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
  __device__ __forceinline__ T operator[](int64_t m) const { return p ? p[m] : value; }
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
