// New keys and values into the paged cache (include/qmm_cache.h).
//
// A key's 16-byte pieces lie in the cache as in the row: they are stored whole. A value's do not: 16 bytes of the cache hold
// one dimension of E neighbouring tokens. Rows whose tokens share such a piece are stored together by the first of them,
// whole pieces where all E are there (prompts), single elements where not (decode). Bound by latency up to some hundred rows,
// by HBM past that.
#include "qmm4_common.h"
#include "qmm_cache_kernels.h"

namespace qmm4 {

namespace {

constexpr int kThreads = 256;
// Values of a row whose codes the 8-bit form holds in LDS at once.
constexpr int kTile = 1024;

// How many of the rows from m on the workgroup of row m stores: those whose tokens follow its own within the aligned E, if no
// earlier row has the token before it there. 0: an earlier row's workgroup stores it.
template <int E>
__device__ __forceinline__ int run_of(const int32_t* slots, int64_t m, int64_t M, int slot) {
  if ((slot & (E - 1)) != 0 && m > 0 && slots[m - 1] == slot - 1) return 0;
  const int lane = threadIdx.x & 63;
  const bool follows = lane < E - (slot & (E - 1)) && m + lane < M && slots[m + lane] == slot + lane;
  return __builtin_ctzll(~__ballot(follows));
}

__global__ __launch_bounds__(kThreads) void store_kv_kernel(CacheRows K, CacheRows V, const int32_t* slots, CacheArrays C, int64_t M,
                                                            int D) {
  const int64_t m = blockIdx.x;
  const int tid = threadIdx.x, slot = slots[m], page_size = 1 << C.page_shift;
  if ((uint32_t)slot >= (uint64_t)C.pages << C.page_shift) return;
  const int64_t head0 = (int64_t)(slot >> C.page_shift) * C.heads;
  const int off = slot & (page_size - 1), chunks = D / 8;
  for (int i = tid; i < C.heads * chunks; i += kThreads) {
    const int h = i / chunks, c = i - h * chunks;
    const u32x4 x = *reinterpret_cast<const u32x4*>(K.x + m * K.row + h * K.head + c * 8);
    static_cast<u32x4*>(C.keys)[((head0 + h) * chunks + c) * page_size + off] = x;
  }
  const int run = run_of<8>(slots, m, M, slot);
  if (run == 0) return;
  // A pair of dimensions each thread.
  for (int i = tid; i < C.heads * D / 2; i += kThreads) {
    const int h = i / (D / 2), d = (i - h * (D / 2)) * 2;
    const uint16_t* x = V.x + m * V.row + h * V.head + d;
    uint32_t v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < run ? *reinterpret_cast<const uint32_t*>(x + j * V.row) : 0u;
    uint16_t* y = static_cast<uint16_t*>(C.values) + (((head0 + h) * (page_size / 8) + off / 8) * D + d) * 8;
    if (run == 8) {
      u32x4 lo, hi;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        lo[j] = (v[2 * j] & 0xFFFFu) | v[2 * j + 1] << 16;
        hi[j] = v[2 * j] >> 16 | (v[2 * j + 1] & 0xFFFF0000u);
      }
      reinterpret_cast<u32x4*>(y)[0] = lo;
      reinterpret_cast<u32x4*>(y)[1] = hi;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (j < run) {
          y[(off & 7) + j] = (uint16_t)v[j];
          y[(off & 7) + j + 8] = (uint16_t)(v[j] >> 16);
        }
      }
    }
  }
}

// 16 values of a head, at most 16 lanes a head: their codes, four to a word, and the head's scale (in all its lanes).
// |x| is compared as bits, where NaN is above infinity above what is finite. The division by the scale is a correctly rounded
// one, so that a code is off from x / scale by half and 2^-17 at most.
__device__ __forceinline__ u32x4 codes16(u32x4 a, u32x4 b, float* scale) {
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    top = max(top, max(a[e] & 0x7FFFu, (a[e] >> 16) & 0x7FFFu));
    top = max(top, max(b[e] & 0x7FFFu, (b[e] >> 16) & 0x7FFFu));
  }
#pragma unroll
  for (int off = 1; off < 16; off <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, off));
  const bool finite = top < 0x7F80u;
  const float s = finite ? __fdiv_rn(bf16_to_f32(top), 127.0f) : __uint_as_float(0x7FC00000u);
  *scale = s;
  u32x4 out;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    uint32_t packed = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = w * 4 + e;
      const uint32_t word = i < 8 ? a[i / 2] : b[i / 2 - 4];
      const float x = bf16_to_f32(i & 1 ? word >> 16 : word & 0xFFFFu);
      const float c = finite && s > 0.0f ? rintf(__fdiv_rn(x, s)) : 0.0f;
      packed |= ((uint32_t)(int)fminf(fmaxf(c, -127.0f), 127.0f) & 0xFFu) << (8 * e);
    }
    out[w] = packed;
  }
  return out;
}

// The same into codes of 8 bits.
__global__ __launch_bounds__(kThreads) void store_kv8_kernel(CacheRows K, CacheRows V, const int32_t* slots, CacheArrays C, int64_t M,
                                                             int D) {
  __shared__ __attribute__((aligned(16))) uint8_t s_codes[16][kTile + 16];
  const int64_t m = blockIdx.x;
  const int tid = threadIdx.x, slot = slots[m], page_size = 1 << C.page_shift;
  if ((uint32_t)slot >= (uint64_t)C.pages << C.page_shift) return;
  const int64_t head0 = (int64_t)(slot >> C.page_shift) * C.heads;
  const int off = slot & (page_size - 1), chunks = D / 16;
  const int c = tid & 15, group = tid >> 4;
  const u32x4 none = {0u, 0u, 0u, 0u};
  for (int h0 = 0; h0 < C.heads; h0 += 16) {
    const int h = h0 + group;
    const bool here = h < C.heads && c < chunks;
    const u32x4* x = reinterpret_cast<const u32x4*>(K.x + m * K.row + h * K.head + c * 16);
    u32x4 a = none, b = none;
    if (here) {
      a = x[0];
      b = x[1];
    }
    float scale;
    const u32x4 codes = codes16(a, b, &scale);
    if (here) {
      static_cast<u32x4*>(C.keys)[((head0 + h) * chunks + c) * page_size + off] = codes;
      if (c == 0) C.key_scales[((head0 + h) << C.page_shift) + off] = scale;
    }
  }
  const int run = run_of<16>(slots, m, M, slot);
  if (run == 0) return;
  const int per = kTile / D;  // heads of a tile
  for (int h0 = 0; h0 < C.heads; h0 += per) {
    const int heads = min(per, C.heads - h0);
    __syncthreads();
    for (int i0 = 0; i0 < run * heads; i0 += 16) {
      const int i = i0 + group, j = i / heads, h = h0 + i - j * heads;
      const bool here = i < run * heads && c < chunks;
      const u32x4* x = reinterpret_cast<const u32x4*>(V.x + (m + j) * V.row + h * V.head + c * 16);
      u32x4 a = none, b = none;
      if (here) {
        a = x[0];
        b = x[1];
      }
      float scale;
      const u32x4 codes = codes16(a, b, &scale);
      if (here) {
        *reinterpret_cast<u32x4*>(&s_codes[j][(h - h0) * D + c * 16]) = codes;
        if (c == 0) C.value_scales[((head0 + h) << C.page_shift) + off + j] = scale;
      }
    }
    __syncthreads();
    for (int i = tid; i < heads * D; i += kThreads) {
      const int h = i / D, d = i - h * D;
      uint8_t* y = static_cast<uint8_t*>(C.values) + (((head0 + h0 + h) * (page_size / 16) + off / 16) * D + d) * 16;
      if (run == 16) {
        u32x4 v;
#pragma unroll
        for (int w = 0; w < 4; ++w)
          v[w] = s_codes[4 * w][i] | s_codes[4 * w + 1][i] << 8 | s_codes[4 * w + 2][i] << 16 | (uint32_t)s_codes[4 * w + 3][i] << 24;
        *reinterpret_cast<u32x4*>(y) = v;
      } else {
        for (int j = 0; j < run; ++j) y[(off & 15) + j] = s_codes[j][i];
      }
    }
  }
}

}  // namespace

hipError_t launch_store_kv(const CacheRows& k, const CacheRows& v, const int32_t* slots, const CacheArrays& cache, int64_t M,
                           int D, bool q8, hipStream_t stream) {
  if (q8) hipLaunchKernelGGL(store_kv8_kernel, dim3((unsigned)M), dim3(kThreads), 0, stream, k, v, slots, cache, M, D);
  else hipLaunchKernelGGL(store_kv_kernel, dim3((unsigned)M), dim3(kThreads), 0, stream, k, v, slots, cache, M, D);
  return hipGetLastError();
}

}  // namespace qmm4
