// Low-rank adapters of many requests beside a shared projection (include/qmm_requests.h):
//   t[m, j] = scale[a] * sum_k x[m, k] A[a, j, k]      shrink, a = adapters[m]
//   y[m, n] += sum_j t[m, j] B[a, n, j]                expand
// Sums and t are fp32; y is rounded to bf16 once.
#include "qmm4_common.h"
#include "qmm_requests_kernels.h"

namespace qmm4 {

namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float dot8(u32x4 a, u32x4 b, float acc) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    acc = __builtin_fmaf(bf16_to_f32(a[e] & 0xFFFFu), bf16_to_f32(b[e] & 0xFFFFu), acc);
    acc = __builtin_fmaf(bf16_to_f32(a[e] >> 16), bf16_to_f32(b[e] >> 16), acc);
  }
  return acc;
}

// One wave per two values of t; a workgroup's four waves take 8 neighbouring j of one row.
__global__ __launch_bounds__(kThreads) void lora_shrink_kernel(LoraTables T, const uint16_t* __restrict__ x,
                                                               float* __restrict__ t, int64_t K) {
  const int64_t m = blockIdx.x;
  const int lane = threadIdx.x & 63, j = blockIdx.y * 8 + (threadIdx.x >> 6) * 2;
  const int64_t a = T.adapters[m];
  if (a < 0 || a >= T.L) {
    if (lane < 2) t[m * T.R + j + lane] = 0.0f;
    return;
  }
  const uint16_t* xr = x + m * K;
  const uint16_t* ar = T.a + (a * T.R + j) * K;
  float s0 = 0.0f, s1 = 0.0f;
  for (int64_t k = lane * 8; k < K; k += 512) {
    const u32x4 xv = *reinterpret_cast<const u32x4*>(xr + k);
    s0 = dot8(xv, *reinterpret_cast<const u32x4*>(ar + k), s0);
    s1 = dot8(xv, *reinterpret_cast<const u32x4*>(ar + K + k), s1);
  }
  s0 = norm_wave_sum(s0);
  s1 = norm_wave_sum(s1);
  const float scale = T.scale[a];
  if (lane < 2) t[m * T.R + j + lane] = scale * (lane ? s1 : s0);
}

constexpr int kExpandRows = 4;

// One thread per column, for kExpandRows rows.
__global__ __launch_bounds__(kThreads) void lora_expand_kernel(LoraTables T, const float* __restrict__ t,
                                                               uint16_t* __restrict__ y, int64_t M, int64_t N) {
  const int64_t n = (int64_t)blockIdx.y * kThreads + threadIdx.x;
  if (n >= N) return;
  for (int r = 0; r < kExpandRows; ++r) {
    const int64_t m = (int64_t)blockIdx.x * kExpandRows + r;
    if (m >= M) break;
    const int64_t a = T.adapters[m];
    if (a < 0 || a >= T.L) continue;
    const uint16_t* b = T.b + (a * N + n) * T.R;
    float sum = 0.0f;
    for (int j = 0; j < T.R; j += 8) {
      const u32x4 bv = *reinterpret_cast<const u32x4*>(b + j);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        sum = __builtin_fmaf(t[m * T.R + j + 2 * e], bf16_to_f32(bv[e] & 0xFFFFu), sum);
        sum = __builtin_fmaf(t[m * T.R + j + 2 * e + 1], bf16_to_f32(bv[e] >> 16), sum);
      }
    }
    y[m * N + n] = (uint16_t)bf16_rne(bf16_to_f32(y[m * N + n]) + sum);
  }
}

}  // namespace

hipError_t launch_lora_shrink(const LoraTables& lora, const uint16_t* x, float* t, int64_t M, int64_t K,
                              hipStream_t stream) {
  if (M <= 0) return hipSuccess;
  hipLaunchKernelGGL(lora_shrink_kernel, dim3((unsigned)M, (unsigned)(lora.R / 8)), dim3(kThreads), 0, stream, lora, x, t, K);
  return hipGetLastError();
}

hipError_t launch_lora_expand(const LoraTables& lora, const float* t, uint16_t* y, int64_t M, int64_t N,
                              hipStream_t stream) {
  if (M <= 0 || N <= 0) return hipSuccess;
  const dim3 grid((unsigned)((M + kExpandRows - 1) / kExpandRows), (unsigned)((N + kThreads - 1) / kThreads));
  hipLaunchKernelGGL(lora_expand_kernel, grid, dim3(kThreads), 0, stream, lora, t, y, M, N);
  return hipGetLastError();
}

}  // namespace qmm4
