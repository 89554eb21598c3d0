// The second factor of the adapters, added to a projection's fp32 sums before they are rounded
// (include/qmm_requests.h): sum[m, n] += sum_j t[m, j] B[a, n, j] for the rows m with an adapter a.
//
// t comes from the shrink kernel as two bf16 numbers whose sum is the value to 2^-18 of it (the high one in the
// upper half of a word): matrix instructions then take it at nearly fp32's precision for two instead of one, on
// work that is R / K of the projection's.
//
// What is not finite in t or B gives what the formula gives: t's low part, which is zero or of either sign, takes B
// with such values as zeros (times an infinity it would add NaN, or the other infinity), and the high part takes B as
// it is, wherever a product is added to rows of its own adapter only. (The GEMM's tiles of several adapters are not
// such a place: lora_nonfinite there. Alternating runs of 64 x 17408 -> 5120 rank 32: 35.9 us without the zeros, 35.8
// with them.)
#pragma once

#include "qmm4_common.h"
#include "qmm_requests_kernels.h"

namespace qmm4 {

// The rows' adapter, or -1.
__device__ __forceinline__ int lora_adapter(const LoraAdd& E, int m, int M) {
  if (m >= M) return -1;
  const int64_t a = E.adapters[m];
  return a >= 0 && a < E.L ? (int)a : -1;
}

// The adapters of rows m0 .. m0 + 3, loaded where a kernel starts and looked at where it ends (each lane for itself).
struct LoraIds {
  uint32_t lo[4], hi[4];
  __device__ __forceinline__ void load(const LoraAdd& E, int m0, int M) {
    const uint32_t* p = static_cast<const uint32_t*>(E.adapters.p);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int64_t m = min(m0 + r, M - 1);
      lo[r] = p[E.adapters.wide ? 2 * m : m];
      hi[r] = p[E.adapters.wide ? 2 * m + 1 : m];
    }
  }
  __device__ __forceinline__ void adapters(const LoraAdd& E, int m0, int M, int (&a)[4]) const {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int64_t id = E.adapters.wide ? (int64_t)((uint64_t)hi[r] << 32 | lo[r]) : (int64_t)(int32_t)lo[r];
      a[r] = m0 + r < M && id >= 0 && id < E.L ? (int)id : -1;
    }
  }
};

// 8 values of t (row m from j) as high and low parts.
__device__ __forceinline__ void lora_split(u32x4 v0, u32x4 v1, bf16x8* hi, bf16x8* lo) {
  u32x4 h, l;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    h[e] = __builtin_amdgcn_perm(v0[2 * e + 1], v0[2 * e], 0x07060302u);
    l[e] = __builtin_amdgcn_perm(v0[2 * e + 1], v0[2 * e], 0x05040100u);
    h[2 + e] = __builtin_amdgcn_perm(v1[2 * e + 1], v1[2 * e], 0x07060302u);
    l[2 + e] = __builtin_amdgcn_perm(v1[2 * e + 1], v1[2 * e], 0x05040100u);
  }
  *hi = as_bf16x8(h);
  *lo = as_bf16x8(l);
}

// Whether one of 8 bf16 values is not finite.
__device__ __forceinline__ bool lora_any_nonfinite(u32x4 v) {
  uint32_t over = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) over |= (v[e] & 0x7FFF7FFFu) + 0x00800080u;
  return (over & 0x80008000u) != 0;
}
// 8 bf16 values with those that are not finite as zeros.
__device__ __forceinline__ u32x4 lora_finite(u32x4 v) {
  typedef int16_t i16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int e = 0; e < 4; ++e)
    v[e] &= ~__builtin_bit_cast(uint32_t, __builtin_bit_cast(i16x2, (v[e] & 0x7FFF7FFFu) + 0x00800080u) >> 15);
  return v;
}

// acc + the products of 8 values of t and b.
__device__ __forceinline__ float lora_dot8(const uint32_t* t, const uint16_t* b, float acc) {
  const u32x4 t0 = *reinterpret_cast<const u32x4*>(t), t1 = *reinterpret_cast<const u32x4*>(t + 4);
  const u32x4 bv = *reinterpret_cast<const u32x4*>(b);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t v = e < 4 ? t0[e] : t1[e - 4];
    const float tv = __uint_as_float(v & 0xFFFF0000u) + __uint_as_float(v << 16);
    acc = __builtin_fmaf(tv, bf16_to_f32(e & 1 ? bv[e / 2] >> 16 : bv[e / 2] & 0xFFFFu), acc);
  }
  return acc;
}

// One value, each lane for itself.
__device__ __forceinline__ float lora_value(const LoraAdd& E, float acc, int m, int col, int M, int N) {
  const int a = lora_adapter(E, m, M);
  if (a < 0) return acc;
  const uint32_t* t = E.t + (int64_t)m * E.R;
  const uint16_t* b = E.b + ((int64_t)a * N + col) * E.R;
  float sum = 0.0f;
  for (int j = 0; j < E.R; j += 8) sum = lora_dot8(t + j, b + j, sum);
  return acc + sum;
}

// Four rows m0 .. m0 + 3 of one column (below N), each lane for itself: the loads of the four go out together, those of
// a row without an adapter from where another's would be, and its sum is dropped. AHEAD: times 8 values of j at once (2:
// 24 x 2560 -> 4100 of 8 bits with 32 adapters 15.7 -> 14.9 us; 1 where the kernel has no registers for it).
template <int AHEAD>
__device__ __forceinline__ f32x4 lora_rows4(const LoraAdd& E, f32x4 acc, const int (&a)[4], int m0, int col, int M, int N) {
  float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  const uint32_t* t[4];
  const uint16_t* b[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    t[r] = E.t + (int64_t)min(m0 + r, M - 1) * E.R;
    b[r] = E.b + ((int64_t)max(a[r], 0) * N + col) * E.R;
  }
#pragma unroll AHEAD
  for (int j = 0; j < E.R; j += 8) {
#pragma unroll
    for (int r = 0; r < 4; ++r) sum[r] = lora_dot8(t[r] + j, b[r] + j, sum[r]);
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) acc[r] += a[r] >= 0 ? sum[r] : 0.0f;
  return acc;
}
template <int AHEAD>
__device__ __forceinline__ f32x4 lora_rows4(const LoraAdd& E, f32x4 acc, int m0, int col, int M, int N) {
  int a[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) a[r] = lora_adapter(E, m0 + r, M);
  return lora_rows4<AHEAD>(E, acc, a, m0, col, M, N);
}

// A wave's 16 x 16 tile in accumulator layout (element r of a lane: row m0 + 4 (lane / 16) + r, column col, 16
// columns by lane % 16). All lanes take part. Each adapter of the tile's rows gives a tile of its own, added to its
// rows only: a row's sum takes nothing of another's adapter, whatever that holds. Rows past the second adapter (a
// batch of single rows) go lane by lane, all loads at once, instead of one adapter's round trip after another's.
__device__ __forceinline__ f32x4 lora_tile16(const LoraAdd& E, f32x4 acc, int m0, int col, int M, int N) {
  const int lane = threadIdx.x & 63, row = m0 + (lane & 15), chunk = (lane >> 4) * 8;
  const int a = lora_adapter(E, row, M);
  uint32_t todo = (uint32_t)__ballot(a >= 0) & 0xFFFFu;
  for (int i = 0; i < 2 && todo != 0; ++i) {
    const int d = __builtin_amdgcn_readlane(a, __ffs((int)todo) - 1);
    const bool mine = a == d;
    const uint32_t rows = (uint32_t)__ballot(mine) & 0xFFFFu;
    todo &= ~rows;
    f32x4 part = {0.0f, 0.0f, 0.0f, 0.0f};
    const uint32_t* t = E.t + (int64_t)row * E.R;
    const uint16_t* b = E.b + ((int64_t)d * N + col) * E.R;
#pragma unroll 2
    for (int k0 = 0; k0 < E.R; k0 += 32) {
      const int k = k0 + chunk;
      u32x4 t0 = {0u, 0u, 0u, 0u}, t1 = t0, bv = t0;
      if (mine && k < E.R) {
        t0 = *reinterpret_cast<const u32x4*>(t + k);
        t1 = *reinterpret_cast<const u32x4*>(t + k + 4);
      }
      if (col < N && k < E.R) bv = *reinterpret_cast<const u32x4*>(b + k);
      bf16x8 hi, lo;
      lora_split(t0, t1, &hi, &lo);
      part = Mfma<16>::mma(hi, as_bf16x8(bv), part);
      part = Mfma<16>::mma(lo, as_bf16x8(lora_finite(bv)), part);
    }
    const uint32_t own = rows >> (4 * (lane >> 4));
#pragma unroll
    for (int r = 0; r < 4; ++r) acc[r] += own >> r & 1 ? part[r] : 0.0f;
  }
  if (todo != 0) {
    int rest[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = 4 * (lane >> 4) + r;
      const int of = __shfl(a, i);
      rest[r] = todo >> i & 1 ? of : -1;
    }
    acc = lora_rows4<2>(E, acc, rest, m0 + 4 * (lane >> 4), min(col, N - 1), M, N);
  }
  return acc;
}

// Rows 8 rq + 4 (lane / 32) .. + 3 of a wave's 32 x 32 tile from row m0, column col (32 columns by lane % 32): four
// values of its accumulator layout. All lanes take part, rq is the same in all.
__device__ __forceinline__ f32x4 lora_part32(const LoraAdd& E, int m0, int rq, int col, int M, int N) {
  const int lane = threadIdx.x & 63, row = m0 + (lane & 31), chunk = (lane >> 5) * 8;
  const int a = lora_adapter(E, row, M);
  const bool ours = (lane & 31) >> 3 == rq;  // (t of other rows need not be read)
  uint32_t todo = (uint32_t)__ballot(a >= 0) & 0xFFu << 8 * rq;
  f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
  while (todo != 0) {
    const int d = __builtin_amdgcn_readlane(a, __ffs((int)todo) - 1);
    const bool mine = a == d && ours;
    const uint32_t rows = (uint32_t)__ballot(mine);
    todo &= ~rows;
    f32x16 part;
#pragma unroll
    for (int r = 0; r < 16; ++r) part[r] = 0.0f;
    const uint32_t* t = E.t + (int64_t)row * E.R;
    const uint16_t* b = E.b + ((int64_t)d * N + col) * E.R;
#pragma unroll 4
    for (int k0 = 0; k0 < E.R; k0 += 16) {
      const int k = k0 + chunk;
      u32x4 t0 = {0u, 0u, 0u, 0u}, t1 = t0, bv = t0;
      if (mine && k < E.R) {
        t0 = *reinterpret_cast<const u32x4*>(t + k);
        t1 = *reinterpret_cast<const u32x4*>(t + k + 4);
      }
      if (col < N && k < E.R) bv = *reinterpret_cast<const u32x4*>(b + k);
      bf16x8 hi, lo;
      lora_split(t0, t1, &hi, &lo);
      part = Mfma<32>::mma(lo, as_bf16x8(lora_finite(bv)), Mfma<32>::mma(hi, as_bf16x8(bv), part));
    }
    const uint32_t own = rows >> (8 * rq + 4 * (lane >> 5));
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float v = rq == 0 ? part[r] : rq == 1 ? part[4 + r] : rq == 2 ? part[8 + r] : part[12 + r];
      acc[r] += own >> r & 1 ? v : 0.0f;
    }
  }
  return acc;
}

}  // namespace qmm4
