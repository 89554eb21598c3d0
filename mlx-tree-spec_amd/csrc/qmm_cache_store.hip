// New keys and values into the paged cache (include/qmm_cache.h).
//
// A key's 16-byte pieces lie in the cache as in the row, those of neighbouring tokens side by side. A value's do not: 16 bytes of
// the cache hold one dimension of E neighbouring tokens. Rows whose tokens share such a piece are a run, and a run is stored by
// one workgroup: in whole pieces where all E tokens are there (prompts), in single elements where not (decode); lines of the
// cache are not written in parts by several XCDs. A workgroup takes the runs that begin in its block of rows, up to 16 rows at a
// time, for some 256 values of each, of keys or of values. Bound by latency up to some hundred rows (16 rows of 4 heads of 256:
// 3.2 us), by HBM past that (4096 rows of 8 heads of 128, 34 MB in and out: 9.7 us, 3.5 TB/s; 1500 of 4 heads of 256 into 8 bits: 8.2).
#include "qmm4_common.h"
#include "qmm_cache_kernels.h"

namespace qmm4 {

namespace {

constexpr int kThreads = 256;
constexpr int kWindow = 16;  // rows at a time
constexpr int kWidth = 256;  // values of a row's part

// 16 values of a head, at most 16 lanes a head: their codes, four to a word, and the head's scale (in all its lanes).
// |x| is compared as bits, where NaN is above infinity above what is finite. x / scale is a product with the scale's inverse,
// corrected by its remainder (a division's own steps for every value take four times as many instructions): off by little more
// than its rounding, so that a code is off from x / scale by half and 2^-17 at most. Both are raised where the inverse would not be
// finite.
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
  const float up = s < 0x1p-100f ? 0x1p100f : 1.0f, divisor = s * up, inverse = __fdiv_rn(1.0f, divisor);
  u32x4 out;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    uint32_t packed = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = w * 4 + e;
      const uint32_t word = i < 8 ? a[i / 2] : b[i / 2 - 4];
      const float x = bf16_to_f32(i & 1 ? word >> 16 : word & 0xFFFFu) * up, y = x * inverse;
      const float c = finite && s > 0.0f ? rintf(__builtin_fmaf(__builtin_fmaf(-y, divisor, x), inverse, y)) : 0.0f;
      packed |= ((uint32_t)(int)fminf(fmaxf(c, -127.0f), 127.0f) & 0xFFu) << (8 * e);
    }
    out[w] = packed;
  }
  return out;
}

struct StoreParams {
  CacheRows k, v;
  const int32_t* slots;
  CacheArrays cache;
  int64_t M;
  int D, block, heads;  // rows of a block; heads of a part
};

template <bool Q8>
__global__ __launch_bounds__(kThreads) void store_kv_kernel(StoreParams S) {
  constexpr int E = Q8 ? 16 : 8;
  __shared__ __attribute__((aligned(16))) uint8_t s_codes[Q8 ? kWindow : 1][kWidth + 16];
  __shared__ int s_slot[kWindow], s_run[kWindow + 1];
  const CacheArrays& C = S.cache;
  const int tid = threadIdx.x, lane = tid & 63, D = S.D, page_size = 1 << C.page_shift;
  const int64_t m0 = (int64_t)blockIdx.x * S.block;
  const bool keys = (blockIdx.y & 1) == 0;
  const int h0 = (blockIdx.y >> 1) * S.heads, heads = min(S.heads, C.heads - h0);
  const CacheRows& X = keys ? S.k : S.v;
  // Where runs begin among the block's rows and those behind it (a run has at most 16; past the last row: one more).
  const int64_t m = m0 + lane;
  const int slot = m < S.M ? S.slots[m] : -1, before = m > 0 && m < S.M ? S.slots[m - 1] : -1;
  const uint64_t begins = __ballot(m == 0 || m >= S.M || (slot & (E - 1)) == 0 || (uint32_t)before + 1 != (uint32_t)slot || lane >= 48);
  const int last = S.block + __builtin_ctzll(begins >> S.block);
  for (int a = __builtin_ctzll(begins); a < last;) {
    // Whole runs of up to 16 rows.
    const int most = min(a + kWindow, last);
    const int e = most == last ? last : 63 - __builtin_clzll(begins & ((2ull << most) - 1)), rows = e - a;
    const uint64_t mine = (begins >> a) & ((1ull << rows) - 1);
    const int runs = __builtin_popcountll(mine);
    if (tid < 64 && lane >= a && lane < e) {
      s_slot[lane - a] = (uint32_t)slot < (uint64_t)C.pages << C.page_shift ? slot : -1;
      if (begins >> lane & 1) s_run[__builtin_popcountll(mine & ((1ull << (lane - a)) - 1))] = lane - a;
    }
    if (tid == 0) s_run[runs] = rows;
    __syncthreads();

    if (Q8) {
      // 16 lanes to a head of a row; neighbouring ones: the rows, whose keys' pieces lie side by side.
      const int c = lane & 15, chunks = D / 16, pairs = rows * heads;
      constexpr int kAhead = 2, kGroups = kThreads / 16;
      for (int i0 = 0; i0 < pairs; i0 += kGroups * kAhead) {
        u32x4 x[kAhead][2];
#pragma unroll
        for (int n = 0; n < kAhead; ++n) {
          const int i = i0 + kGroups * n + tid / 16, h = i / rows, j = i - h * rows;
          x[n][0] = x[n][1] = u32x4{0u, 0u, 0u, 0u};
          if (i < pairs && c < chunks && s_slot[j] >= 0) {
            const u32x4* p = reinterpret_cast<const u32x4*>(X.x + (m0 + a + j) * X.row + (h0 + h) * X.head + c * 16);
            x[n][0] = p[0];
            x[n][1] = p[1];
          }
        }
#pragma unroll
        for (int n = 0; n < kAhead; ++n) {
          const int i = i0 + kGroups * n + tid / 16, h = i / rows, j = i - h * rows;
          if (i0 + kGroups * n >= pairs) break;  // (the same for all: their lanes exchange)
          float scale;
          const u32x4 codes = codes16(x[n][0], x[n][1], &scale);
          if (i >= pairs || c >= chunks || s_slot[j] < 0) continue;
          const int off = s_slot[j] & (page_size - 1);
          const int64_t head = (int64_t)(s_slot[j] >> C.page_shift) * C.heads + h0 + h;
          if (c == 0) (keys ? C.key_scales : C.value_scales)[(head << C.page_shift) + off] = scale;
          if (keys) static_cast<u32x4*>(C.keys)[(head * chunks + c) * page_size + off] = codes;
          else *reinterpret_cast<u32x4*>(&s_codes[j][h * D + c * 16]) = codes;
        }
      }
      if (!keys) {
        __syncthreads();
        for (int i = tid; i < runs * heads * D; i += kThreads) {
          const int k = i / (heads * D), d = i - k * (heads * D), j0 = s_run[k], run = s_run[k + 1] - j0, at = s_slot[j0];
          if (at < 0) continue;
          const int off = at & (page_size - 1), h = d / D;
          const int64_t head = (int64_t)(at >> C.page_shift) * C.heads + h0 + h;
          uint8_t* y = static_cast<uint8_t*>(C.values) + ((head * (page_size / 16) + off / 16) * D + (d - h * D)) * 16;
          if (run == 16) {
            u32x4 v;
#pragma unroll
            for (int w = 0; w < 4; ++w)
              v[w] = s_codes[4 * w][d] | s_codes[4 * w + 1][d] << 8 | s_codes[4 * w + 2][d] << 16 | (uint32_t)s_codes[4 * w + 3][d] << 24;
            *reinterpret_cast<u32x4*>(y) = v;
          } else {
            for (int j = 0; j < run; ++j) y[(off & 15) + j] = s_codes[j0 + j][d];
          }
        }
      }
    } else if (keys) {
      // Neighbouring lanes: the rows, then the next piece.
      constexpr int kAhead = 2;
      const int width = rows > 8 ? 16 : rows > 4 ? 8 : rows > 2 ? 4 : rows;  // (a power of two)
      const int j = tid & (width - 1), step = kThreads / width, chunks = D / 8, pieces = heads * chunks;
      const int at = j < rows ? s_slot[j] : -1, off = at & (page_size - 1);
      const int64_t head0 = (int64_t)(at >> C.page_shift) * C.heads + h0;
      const uint16_t* row = X.x + (m0 + a + j) * X.row + h0 * X.head;
      for (int i0 = tid / width; i0 < pieces; i0 += step * kAhead) {
        u32x4 x[kAhead];
#pragma unroll
        for (int n = 0; n < kAhead; ++n) {
          const int i = i0 + n * step, h = i / chunks;
          if (at >= 0 && i < pieces) x[n] = *reinterpret_cast<const u32x4*>(row + h * X.head + (i - h * chunks) * 8);
        }
#pragma unroll
        for (int n = 0; n < kAhead; ++n) {
          const int i = i0 + n * step;
          if (at >= 0 && i < pieces) static_cast<u32x4*>(C.keys)[(head0 * chunks + i) * page_size + off] = x[n];
        }
      }
    } else {
      // A pair of dimensions of a run each thread.
      const int pairs = heads * (D / 2);
      for (int i = tid; i < runs * pairs; i += kThreads) {
        const int k = i / pairs, d2 = (i - k * pairs) * 2, h = d2 / D, d = d2 - h * D, j0 = s_run[k], run = s_run[k + 1] - j0;
        const int at = s_slot[j0];
        if (at < 0) continue;
        const int off = at & (page_size - 1);
        const uint16_t* x = X.x + (m0 + a + j0) * X.row + (h0 + h) * X.head + d;
        uint32_t v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = j < run ? *reinterpret_cast<const uint32_t*>(x + j * X.row) : 0u;
        const int64_t head = (int64_t)(at >> C.page_shift) * C.heads + h0 + h;
        uint16_t* y = static_cast<uint16_t*>(C.values) + ((head * (page_size / 8) + off / 8) * D + d) * 8;
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
    a = e;
    __syncthreads();
  }
}

}  // namespace

hipError_t launch_store_kv(const CacheRows& k, const CacheRows& v, const int32_t* slots, const CacheArrays& cache, int64_t M,
                           int D, bool q8, hipStream_t stream) {
  // A row to a block where there are few: 16 of as many requests 4.1 us (7.4 with blocks of 16), 200 5.8 (8.3); 512 of a prompt 4.7
  // with blocks of 16 (8.2 with blocks of one), 4096 10 (42).
  const int block = M <= 256 ? 1 : 16, heads = kWidth / D;
  const StoreParams p{k, v, slots, cache, M, D, block, heads};
  const dim3 grid((unsigned)((M + block - 1) / block), (unsigned)((cache.heads + heads - 1) / heads * 2));
  if (q8) hipLaunchKernelGGL(store_kv_kernel<true>, grid, dim3(kThreads), 0, stream, p);
  else hipLaunchKernelGGL(store_kv_kernel<false>, grid, dim3(kThreads), 0, stream, p);
  return hipGetLastError();
}

}  // namespace qmm4
