// Low-rank adapters of many requests beside a shared projection (include/qmm_requests.h):
//   t[m, j] = scale[a] * sum_k x[m, k] A[a, j, k]      shrink, a = adapters[m]
//   y[m, n] += sum_j t[m, j] B[a, n, j]                expand
// Sums are fp32; t is kept to 2^-18 of its value (qmm_lora.h). The expand is the last step of the projection's own
// kernels; the one here serves projections that run elsewhere.
//
// Shrink: a workgroup takes 16 rows and 16 values of j for one of the adapters that its rows have (the z-th of them:
// a tree's nodes or a prompt's rows share one, so most z end at once) and a slice of K, its 8 waves a part of it each,
// as 16 x 16 x 32 matrix products. Rows are loaded with 16 neighbouring lanes each and put in matrix order through LDS
// of the wave's own (loads in matrix order, a row to each neighbouring lane, reach less than half the rate). The 8
// sums meet in LDS; slices, where there are several, are added by the last workgroup to arrive, in their order.
#include "qmm4_common.h"
#include "qmm4_lds.h"
#include "qmm_lora.h"
#include "qmm_requests_kernels.h"

namespace qmm4 {

namespace {

constexpr int kWaves = 8;
constexpr int kMaxSlices = 8;
constexpr int kThreads = 64 * kWaves;

// t as two bf16 numbers: the value rounded, and what that left out (nothing, where the value is not finite).
__device__ __forceinline__ uint32_t split_bf16(float v) {
  const uint32_t hi = bf16_rne(v);
  const float rest = v - bf16_to_f32(hi);
  return hi << 16 | ((hi & 0x7F80u) == 0x7F80u ? 0u : bf16_rne(rest));
}

constexpr int kUnit = 128;               // k per step of a wave
constexpr int kWaveLds = 2 * 16 * kUnit * 2;  // bytes: 16 rows of x and of A
constexpr int kCoherent = 16;            // buffer access flag: coherent across the XCDs' L2s

struct Shrink {
  LoraTables T;
  const uint16_t* x;
  uint32_t* t;
  float* part;    // slices > 1: fp32 tiles [tile][slice][lane][4]
  uint32_t* cnt;  // arrivals per tile (0 between launches)
  int M, K, slices, across, units;  // units of kUnit k, the last one possibly short
  int first;  // not in slices: the first row
};

template <bool SLICED>
__global__ __launch_bounds__(kThreads) void lora_shrink_kernel(Shrink P) {
  extern __shared__ __attribute__((aligned(16))) u32x4 lds[];
  const LoraTables& T = P.T;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int slices = SLICED ? P.slices : 1, slice = SLICED ? blockIdx.x % slices : 0;
  const int m0 = SLICED ? blockIdx.x / slices * 16 : P.first + ((blockIdx.x >> 3) / P.across * 8 + (blockIdx.x & 7)) * 16;
  const int j0 = (SLICED ? blockIdx.y : (blockIdx.x >> 3) % P.across) * 16;
  if (!SLICED && m0 >= P.M) return;
  const int64_t id = T.adapters[min(m0 + (lane & 15), P.M - 1)];
  const int a = m0 + (lane & 15) < P.M && id >= 0 && id < T.L ? (int)id : -1;
  // The z-th adapter of the rows.
  uint32_t todo = (uint32_t)__ballot(a >= 0) & 0xFFFFu, rows = 0;
  int d = 0;
  for (int z = 0; z <= (int)blockIdx.z; ++z) {
    if (todo == 0) return;
    d = __builtin_amdgcn_readlane(a, __ffs((int)todo) - 1);
    rows = (uint32_t)__ballot(a == d) & 0xFFFFu;
    todo &= ~rows;
  }
  const float scale = T.scale[d];
  const int part = slice * kWaves + wave, parts = slices * kWaves;
  const int ub = (int)((int64_t)part * P.units / parts), ue = (int)((int64_t)(part + 1) * P.units / parts);
  // Load i: row 4 i + lane / 16 of the tile, 16-byte piece lane % 16 of the unit.
  const int r4 = lane >> 4, piece = lane & 15;
  const uint16_t* xr = P.x + (int64_t)(m0 + r4) * P.K + piece * 8;
  const uint16_t* ar = T.a + ((int64_t)d * T.R + j0 + r4) * P.K + piece * 8;
  u32x4* const lx = lds + wave * (kWaveLds / 16);
  u32x4* const la = lx + 16 * 16;
  f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
  // Units in flight: a sliced wave has 1 or 2 (4 x 5120 4.8 us with 1 and with 2, 64 x 17408 rank 32 7.0 and 7.2), one with
  // all of K several (2000 x 5120 rank 64 15.5, 15.0 and 14.7 us with 1, 2 and 3, 20.7 with 4).
  constexpr int kBatch = SLICED ? 1 : 3;
  for (int u0 = ub; u0 < ue; u0 += kBatch) {
    u32x4 xv[kBatch][4], av[kBatch][4];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int u = u0 + b;
      const bool in = u < ue && u * kUnit + piece * 8 < P.K;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        xv[b][i] = av[b][i] = u32x4{0u, 0u, 0u, 0u};
        if (in && (rows >> (4 * i + r4) & 1)) xv[b][i] = *reinterpret_cast<const u32x4*>(xr + (int64_t)(4 * i) * P.K + u * kUnit);
        if (in && j0 + 4 * i + r4 < T.R) av[b][i] = *reinterpret_cast<const u32x4*>(ar + (int64_t)(4 * i) * P.K + u * kUnit);
      }
    }
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      if (u0 + b >= ue) break;
      // (A wave's LDS accesses are done in order; the fences keep the compiler's.)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = 4 * i + r4;
        lx[row * 16 + (piece ^ row)] = xv[b][i];
        la[row * 16 + (piece ^ row)] = av[b][i];
      }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        const int at = (lane & 15) * 16 + ((4 * p + r4) ^ (lane & 15));
        acc = Mfma<16>::mma(as_bf16x8(lx[at]), as_bf16x8(la[at]), acc);
      }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
  }
  __syncthreads();
  f32x4* const sums = reinterpret_cast<f32x4*>(lds);
  sums[wave * 64 + lane] = acc;
  __syncthreads();
  if (wave != 0) return;
#pragma unroll
  for (int w = 1; w < kWaves; ++w) {
    const f32x4 v = sums[w * 64 + lane];
    acc[0] += v[0]; acc[1] += v[1]; acc[2] += v[2]; acc[3] += v[3];
  }
  if constexpr (SLICED) {
    const uint32_t tile = (blockIdx.z * gridDim.y + blockIdx.y) * (gridDim.x / slices) + blockIdx.x / slices;
    const __amdgpu_buffer_rsrc_t rp = __builtin_amdgcn_make_buffer_rsrc(
        P.part, 0, rsrc_bytes((unsigned long long)gridDim.x * gridDim.y * gridDim.z * 1024), kBufferRsrcWord3);
    const uint32_t o = tile * (uint32_t)slices * 1024u + (uint32_t)lane * 16u;
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, acc), rp, o + (uint32_t)slice * 1024u, 0, kCoherent);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    uint32_t before = 0;
    if (lane == 0) before = __hip_atomic_fetch_add(&P.cnt[tile], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (__builtin_amdgcn_readfirstlane(before) != (uint32_t)slices - 1) return;
    f32x4 v[kMaxSlices];
#pragma unroll
    for (int q = 0; q < kMaxSlices; ++q) {
      v[q] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      if (q < slices)
        v[q] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rp, o + (uint32_t)q * 1024u, 0, kCoherent));
    }
    acc = v[0];
#pragma unroll
    for (int q = 1; q < kMaxSlices; ++q) {
      acc[0] += v[q][0]; acc[1] += v[q][1]; acc[2] += v[q][2]; acc[3] += v[q][3];
    }
    if (lane == 0) __hip_atomic_store(&P.cnt[tile], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  const int jj = j0 + (lane & 15);
  if (jj >= T.R) return;
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if (rows >> (4 * r4 + r) & 1) P.t[(int64_t)(m0 + 4 * r4 + r) * T.R + jj] = split_bf16(scale * acc[r]);
}

// One wave per 16 x 64 values of y (of every so many rows, where there are more than a grid's).
__global__ __launch_bounds__(256) void lora_expand_kernel(LoraAdd E, uint16_t* __restrict__ y, int M, int N) {
  const int lane = threadIdx.x & 63, across = (N + 255) / 256, rows = gridDim.x / across * 16;
  const int n0 = (blockIdx.x % across * 4 + (threadIdx.x >> 6)) * 64;
  for (int m0 = blockIdx.x / across * 16; m0 < M; m0 += rows) {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int col = n0 + c * 16 + (lane & 15);
      const f32x4 d = lora_tile16(E, f32x4{0.0f, 0.0f, 0.0f, 0.0f}, m0, col, M, N);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int m = m0 + 4 * (lane >> 4) + r;
        if (col < N && lora_adapter(E, m, M) >= 0) {
          uint16_t* p = y + (int64_t)m * N + col;
          *p = (uint16_t)bf16_rne(bf16_to_f32(*p) + d[r]);
        }
      }
    }
  }
}

LdsAllowance g_sliced, g_whole;

}  // namespace

// Few tiles: K in up to 8 slices of at least 512, while that gives a CU no second workgroup (counted for one adapter per
// 16 rows). One / 4 / 8 slices: 4 x 5120 rank 16 of 4 adapters 6.1 / 5.3 / 4.8 us, 16 rows of one 6.3 / 5.3 / 4.7, 64 x
// 17408 rank 32 of 4 adapters 14.9 / 7.8 / 6.9; many tiles, 2000 x 5120 rank 64, 15.0 / 30 / 47. (4 or 16 waves instead of
// 8: 4 x 5120 0.2 or 0.5 more, many tiles no better; tiles of 4 values of j: no better in slices.)
LoraShrinkPlan lora_shrink_plan(const LoraTables& lora, int M, int K, int cus) {
  LoraShrinkPlan p;
  const int most = M < 16 ? M : 16;  // adapters of 16 rows
  p.rows = (M + 15) / 16;
  p.across = (lora.R + 15) / 16;
  p.depth = (int)(lora.L < most ? lora.L : most);
  const int64_t tiles = (int64_t)p.rows * p.across;
  int64_t s = cus / tiles;
  if (s > K / 512) s = K / 512;
  p.slices = s < 1 ? 1 : s > kMaxSlices ? kMaxSlices : (int)s;
  p.counter_bytes = p.slices > 1 ? (size_t)(tiles * p.depth) * sizeof(uint32_t) : 0;
  p.part_bytes = p.slices > 1 ? (size_t)(tiles * p.depth * p.slices) * 1024 : 0;
  return p;
}

hipError_t launch_lora_shrink(const LoraShrinkPlan& plan, const LoraTables& lora, const uint16_t* x, uint32_t* t,
                              float* part, uint32_t* cnt, int M, int K, hipStream_t stream) {
  constexpr size_t kLds = (size_t)kWaves * kWaveLds;
  Shrink P{lora, x, t, part, cnt, M, K, plan.slices, plan.across, (K + kUnit - 1) / kUnit, 0};
  if (plan.slices > 1) {
    const hipError_t e = g_sliced.allow(reinterpret_cast<const void*>(&lora_shrink_kernel<true>), kLds);
    if (e != hipSuccess) return e;
    const dim3 grid((unsigned)(plan.rows * plan.slices), (unsigned)plan.across, (unsigned)plan.depth);
    hipLaunchKernelGGL(lora_shrink_kernel<true>, grid, dim3(kThreads), kLds, stream, P);
  } else {
    // Workgroups 8 apart (of one XCD) in turn take the tiles of j of the same rows: x comes into one L2 instead of up to 8
    // (2000 x 5120 rank 64: 20.9 -> 15.5 us).
    const hipError_t e = g_whole.allow(reinterpret_cast<const void*>(&lora_shrink_kernel<false>), kLds);
    if (e != hipSuccess) return e;
    constexpr int kMost = 1 << 18;  // tiles of rows per launch (a grid may have 2^32 threads along x)
    for (int tile = 0; tile < plan.rows; tile += kMost) {
      const int rows = plan.rows - tile < kMost ? plan.rows - tile : kMost;
      P.first = tile * 16;
      const dim3 grid((unsigned)((rows + 7) / 8 * 8 * plan.across), 1, (unsigned)plan.depth);
      hipLaunchKernelGGL(lora_shrink_kernel<false>, grid, dim3(kThreads), kLds, stream, P);
    }
  }
  return hipGetLastError();
}

hipError_t launch_lora_expand(const LoraAdd& lora, uint16_t* y, int M, int N, hipStream_t stream) {
  if (M <= 0 || N <= 0) return hipSuccess;
  const int64_t across = (N + 255) / 256, most = (1 << 23) / across;  // (a grid may have 2^32 threads along x)
  const int64_t rows = (M + 15) / 16 < most ? (M + 15) / 16 : most;
  hipLaunchKernelGGL(lora_expand_kernel, dim3((unsigned)(rows * across)), dim3(256), 0, stream, lora, y, M, N);
  return hipGetLastError();
}

}  // namespace qmm4
