// Attention of a step's new rows over a paged key-value cache, split over the cache's length and joined
// (include/qmm_cache.h). With G query heads to a key head, a request of n rows has n G query rows for each key head:
//   s = scale q . k_t,   m = max s,   l = sum exp(s - m),   o = sum exp(s - m) v_t,   out = o / l  (* sigmoid(gate))
//
// Both products run on 16x16x32 matrix instructions with the tokens' side as the first operand:
//   S^T = K Q^T  (16 tokens x 16 query rows),   O^T = V^T P^T  (16 dimensions x 16 query rows)
// The cache's layout makes 16 bytes of keys (8 dimensions of a token) and of values (8 tokens of a dimension) operands as they
// lie: a wave loads them from memory to registers, 1 KB an instruction in whole runs of 256 bytes, without LDS. S^T leaves
// each lane with the probabilities of one query row; the order of tokens within a step is chosen (row 4 g + i of
// tile tt is token E g + 4 tt + i) so that they are the second operand of O^T without a move between lanes.
//
// A wave takes 16 QT query rows and every KW-th step of 4 E tokens of its workgroup's split; waves of the same rows join their
// results through LDS, splits through memory (fp32) and a second kernel. While one step's probabilities are made, the next step's
// keys are on their way, and its values while the products with the present ones run.
//
// The running maximum moves only where a logit passes it by more than 2^8: probabilities up to 256 lose nothing in fp32, and
// most steps need no exchange between lanes.
#include "qmm4_common.h"
#include "qmm4_lds.h"
#include "qmm_cache_kernels.h"

namespace qmm4 {

namespace {

constexpr float kLog2e = 1.44269504f;
// How far (in powers of two) a logit may pass the running maximum.
constexpr float kSlack = 8.0f;

template <int D, int QT, bool Q8>
struct PagedTraits {
  static constexpr int E = Q8 ? 16 : 8;      // elements of 16 bytes
  static constexpr int kStep = 4 * E;        // tokens of a wave's step
  static constexpr int kKT = E / 4;          // tiles of 16 tokens
  static constexpr int kKC = D / (4 * E);    // 16-byte pieces of a key for each lane
  static constexpr int kQK = D / 32;         // matrix instructions along D
  static constexpr int kVT = D / 16;         // tiles of 16 dimensions
  // Registers of o, q, s, keys, values and scales; with what else there is more than 256: one wave to a SIMD.
  static constexpr int kRegisters = 4 * (QT * (kVT + kQK + kKT) + kKT * kKC + kVT + (Q8 ? 3 * kKT : 0));
  static constexpr int kWaves = kRegisters > 176 ? 4 : 8;
  static constexpr size_t kJoin = (size_t)(kWaves / 2) * QT * (kVT * 1024 + 128);  // LDS of a join
};

// 8 codes -> bf16 (exact).
__device__ __forceinline__ bf16x8 codes8(uint32_t lo, uint32_t hi) {
  u32x4 r;
  r.x = pack_bf16x2((float)(int8_t)(lo & 0xFFu), (float)(int8_t)((lo >> 8) & 0xFFu));
  r.y = pack_bf16x2((float)(int8_t)((lo >> 16) & 0xFFu), (float)(int8_t)(lo >> 24));
  r.z = pack_bf16x2((float)(int8_t)(hi & 0xFFu), (float)(int8_t)((hi >> 8) & 0xFFu));
  r.w = pack_bf16x2((float)(int8_t)((hi >> 16) & 0xFFu), (float)(int8_t)(hi >> 24));
  return as_bf16x8(r);
}

__device__ __forceinline__ f32x4 mma(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

__device__ __forceinline__ float sigmoid(float x) { return 1.0f / (1.0f + __expf(-x)); }

// A query row, null where there is none.
struct QueryAddress {
  const uint16_t* x;
};

// What a wave knows of one of its query rows (the one of lane % 16 in tile qt).
struct QueryRow {
  uint64_t bits;  // the step's rows that it sees (all ones without ancestors)
  bool valid;
};

template <int D, int QT, bool Q8>
struct PagedWave {
  using T = PagedTraits<D, QT, Q8>;
  static constexpr int E = T::E;

  const PagedParams& S;
  const int32_t* table;
  int lane, r16, g, h, length, context;
  bf16x8 q[QT][T::kQK];
  QueryRow row[QT];
  int seen[QT];  // no token from this on is seen
  float m[QT], l[QT];
  f32x4 o[QT][T::kVT];
  u32x4 kf[T::kKT][T::kKC], vf[T::kVT];
  f32x4 ks[Q8 ? T::kKT : 1], vs[Q8 ? T::kKT : 1];
  bool odd = false;  // a value that is not finite was left out

  __device__ __forceinline__ PagedWave(const PagedParams& s) : S(s) {}

  // The first token of a group of E, within the request's.
  __device__ __forceinline__ int group(int token) const { return min(token, (length - 1) & ~(E - 1)); }
  // Its page (any within the cache where the table names none).
  __device__ __forceinline__ int page(int token) const {
    const int p = table[group(token) >> S.cache.page_shift];
    return max(0, min(p, (int)S.cache.pages - 1));
  }

  __device__ __forceinline__ void load_keys(int t, int page) {
    const int shift = S.cache.page_shift, tok = group(t + E * (r16 >> 2)) & ((1 << shift) - 1);
    const char* p = static_cast<const char*>(S.cache.keys) +
                    (((((int64_t)page * S.cache.heads + h) * (D / E) + g) << shift) + tok + (r16 & 3)) * 16;
#pragma unroll
    for (int c = 0; c < T::kKC; ++c)
#pragma unroll
      for (int tt = 0; tt < T::kKT; ++tt) kf[tt][c] = *reinterpret_cast<const u32x4*>(p + ((int64_t)c << (shift + 6)) + tt * 64);
  }

  __device__ __forceinline__ void load_values(int t, int page) {
    const int shift = S.cache.page_shift, tok = group(t + E * g) & ((1 << shift) - 1);
    const char* p = static_cast<const char*>(S.cache.values) +
                    ((((((int64_t)page * S.cache.heads + h) << shift) + tok) / E) * D + r16) * 16;
#pragma unroll
    for (int dt = 0; dt < T::kVT; ++dt) vf[dt] = *reinterpret_cast<const u32x4*>(p + dt * 256);
  }

  __device__ __forceinline__ void load_scales(int t, int page) {
    if constexpr (Q8) {
      const int shift = S.cache.page_shift, tok = group(t + E * g) & ((1 << shift) - 1);
      const int64_t at = (((int64_t)page * S.cache.heads + h) << shift) + tok;
#pragma unroll
      for (int tt = 0; tt < T::kKT; ++tt) {
        ks[tt] = *reinterpret_cast<const f32x4*>(S.cache.key_scales + at + 4 * tt);
        vs[tt] = *reinterpret_cast<const f32x4*>(S.cache.value_scales + at + 4 * tt);
      }
    }
  }

  // Token of value i of tile tt, relative to the step's first.
  __device__ __forceinline__ int token(int tt, int i) const { return E * g + 4 * tt + i; }
  // Whether the row sees a token: all of the context, and of what follows up to `seen` what its bits say. (Without branches:
  // hipcc 7.2 has lost the selected value of nested divergent ones here.)
  __device__ __forceinline__ bool sees(int qt, int tok) const {
    const int j = tok - context;
    return (j < 0) | ((tok < seen[qt]) & ((uint32_t)(row[qt].bits >> (j & 63)) & 1u));
  }

  // Zeros in a step's values in place of tokens past the last, which the cache need not hold, and of what is not finite:
  // a probability of zero would not keep it from the rows that do not see it. `odd`: there was some of it.
  __device__ __forceinline__ void clean_values(int t) {
    if constexpr (!Q8) {
      const int past = t + E * g - length;
      bool any = false;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint32_t keep = past + 2 * w >= 0 ? 0u : past + 2 * w + 1 >= 0 ? 0xFFFFu : 0xFFFFFFFFu;
#pragma unroll
        for (int dt = 0; dt < T::kVT; ++dt) {
          uint32_t x = vf[dt][w] & keep;
          const bool lo = (x & 0x7F80u) == 0x7F80u, hi = (x & 0x7F800000u) == 0x7F800000u;
          any |= lo | hi;
          x = lo ? x & 0xFFFF0000u : x;
          vf[dt][w] = hi ? x & 0xFFFFu : x;
        }
      }
      odd |= __any(any) != 0;
    }
  }

  // What those values add to o for the rows that see them: the wave's steps from t on again, token by token.
  __device__ __forceinline__ void add_odd_values(int t, int end, int stride, const QueryAddress (&at)[QT]) {
    const int shift = S.cache.page_shift;
    for (; t < end; t += stride) {
      if (t + T::kStep <= context) continue;
      for (int tok = t; tok < min(t + T::kStep, length); ++tok) {
        const int64_t head = (int64_t)max(0, min(table[tok >> shift], (int)S.cache.pages - 1)) * S.cache.heads + h;
        const int off = tok & ((1 << shift) - 1);
        const uint16_t* v = static_cast<const uint16_t*>(S.cache.values) + ((((head << shift) + off) / 8) * D) * 8 + off % 8;
        const uint16_t* k = static_cast<const uint16_t*>(S.cache.keys) + (((head * (D / 8)) << shift) + off) * 8;
        bool any = false;
        for (int d = lane; d < D; d += 64) any |= (v[d * 8] & 0x7F80u) == 0x7F80u;
        if (!__any(any)) continue;
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) {
          float x = 0.0f;
          for (int d = g; d < D; d += 4)
            x += at[qt].x ? bf16_to_f32(at[qt].x[d]) * bf16_to_f32(k[((int64_t)(d / 8) << shift) * 8 + d % 8]) : 0.0f;
          x += __shfl_xor(x, 16);
          x += __shfl_xor(x, 32);
          const float p = __builtin_amdgcn_exp2f(x * (S.scale * kLog2e) - m[qt]);
          const bool see = sees(qt, tok);
#pragma unroll
          for (int dt = 0; dt < T::kVT; ++dt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t y = v[(dt * 16 + 4 * g + i) * 8];
              const float add = p * bf16_to_f32(y);
              o[qt][dt][i] += (see & ((y & 0x7F80u) == 0x7F80u)) ? add : 0.0f;
            }
        }
      }
    }
  }

  // One step of kStep tokens from t, whose keys and values are loaded; MORE: those of t + stride are, meanwhile (kp, vp: their
  // pages on entry; on return those of t + 2 stride).
  template <bool MORE>
  __device__ __forceinline__ void step(int t, int stride, int* kp, int* vp) {
    f32x4 s[QT][T::kKT];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt)
#pragma unroll
      for (int tt = 0; tt < T::kKT; ++tt) s[qt][tt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int c = 0; c < T::kKC; ++c)
#pragma unroll
      for (int tt = 0; tt < T::kKT; ++tt) {
        if constexpr (Q8) {
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const bf16x8 k = codes8(kf[tt][c][2 * half], kf[tt][c][2 * half + 1]);
#pragma unroll
            for (int qt = 0; qt < QT; ++qt) s[qt][tt] = mma(k, q[qt][2 * c + half], s[qt][tt]);
          }
        } else {
#pragma unroll
          for (int qt = 0; qt < QT; ++qt) s[qt][tt] = mma(as_bf16x8(kf[tt][c]), q[qt][c], s[qt][tt]);
        }
      }
    const float unit = S.scale * kLog2e;
    f32x4 vscale[Q8 ? T::kKT : 1];
    if constexpr (Q8) {
#pragma unroll
      for (int tt = 0; tt < T::kKT; ++tt) {
        vscale[tt] = vs[tt];
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) s[qt][tt] *= ks[tt] * unit;
      }
    } else {
#pragma unroll
      for (int qt = 0; qt < QT; ++qt)
#pragma unroll
        for (int tt = 0; tt < T::kKT; ++tt) s[qt][tt] *= unit;
    }
    __builtin_amdgcn_sched_barrier(0);
    int next_page = 0;
    if constexpr (MORE) {
      next_page = *vp;
      load_keys(t + stride, *kp);
      load_scales(t + stride, next_page);
      *kp = page(t + 2 * stride + E * (r16 >> 2));
      *vp = page(t + 2 * stride + E * g);
    }
    __builtin_amdgcn_sched_barrier(0);
    const bool masked = t + T::kStep > context;
    bf16x8 p[QT][E / 8];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      if (masked) {
#pragma unroll
        for (int tt = 0; tt < T::kKT; ++tt)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[qt][tt][i] = sees(qt, t + token(tt, i)) ? s[qt][tt][i] : -__builtin_inff();
      }
      float top = s[qt][0][0];
#pragma unroll
      for (int tt = 0; tt < T::kKT; ++tt)
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, s[qt][tt][i]);
      if (__any(top > m[qt] + kSlack)) {
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(fmaxf(top, __shfl_xor(top, 32)), m[qt]);
        // (Nothing seen yet: l and o are zero.)
        const float f = m[qt] == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m[qt] - top);
        if (m[qt] != -__builtin_inff()) {
          l[qt] *= f;
#pragma unroll
          for (int dt = 0; dt < T::kVT; ++dt) o[qt][dt] *= f;
        }
        m[qt] = top;
      }
      const float ref = m[qt] == -__builtin_inff() ? 0.0f : m[qt];
      float e[E];
#pragma unroll
      for (int tt = 0; tt < T::kKT; ++tt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          e[tt * 4 + i] = __builtin_amdgcn_exp2f(s[qt][tt][i] - ref);
          l[qt] += e[tt * 4 + i];
        }
      if constexpr (Q8) {
#pragma unroll
        for (int tt = 0; tt < T::kKT; ++tt)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float x = e[tt * 4 + i] * vscale[tt][i];
            e[tt * 4 + i] = masked && !sees(qt, t + token(tt, i)) ? 0.0f : x;
          }
      }
#pragma unroll
      for (int half = 0; half < E / 8; ++half) {
        u32x4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = pack_bf16x2(e[half * 8 + 2 * i], e[half * 8 + 2 * i + 1]);
        p[qt][half] = as_bf16x8(w);
      }
    }
    if constexpr (!Q8) {
      if (masked) clean_values(t);
    }
#pragma unroll
    for (int dt = 0; dt < T::kVT; ++dt) {
#pragma unroll
      for (int half = 0; half < E / 8; ++half) {
        const bf16x8 v = Q8 ? codes8(vf[dt][(2 * half) & 3], vf[dt][(2 * half + 1) & 3]) : as_bf16x8(vf[dt]);
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) o[qt][dt] = mma(v, p[qt][half], o[qt][dt]);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (MORE) load_values(t + stride, next_page);
    __builtin_amdgcn_sched_barrier(0);
  }

  // Steps t, t + stride, .. below end.
  __device__ __forceinline__ void run(int t, int end, int stride) {
    if (t >= end) return;
    const int vpage = page(t + E * g);
    load_keys(t, page(t + E * (r16 >> 2)));
    load_scales(t, vpage);
    load_values(t, vpage);
    int kp = page(t + stride + E * (r16 >> 2)), vp = page(t + stride + E * g);
    for (; t + stride < end; t += stride) step<true>(t, stride, &kp, &vp);
    step<false>(t, stride, &kp, &vp);
  }
};

template <int D, int QT, bool Q8>
__global__ __launch_bounds__((PagedTraits<D, QT, Q8>::kWaves * 64)) void paged_kernel(PagedParams S) {
  using T = PagedTraits<D, QT, Q8>;
  extern __shared__ __attribute__((aligned(16))) char s_join[];
  const int heads = S.cache.heads, item = blockIdx.x / heads;
  if (item >= S.plan.words[0]) return;
  const int r = S.plan.items()[2 * item], split = S.plan.items()[2 * item + 1];
  const int n = S.plan.count()[r], length = S.plan.length()[r], per = S.plan.per()[r], first = S.plan.first()[r];
  const int64_t rows = (int64_t)n * S.G, heads_q = (int64_t)heads * S.G;
  const bool whole = per >= length;
  const int wave = threadIdx.x >> 6;

  PagedWave<D, QT, Q8> W(S);
  W.lane = threadIdx.x & 63;
  W.r16 = W.lane & 15;
  W.g = W.lane >> 4;
  W.h = blockIdx.x - item * heads;
  W.length = length;
  W.context = length - n;
  W.table = S.table + (int64_t)r * S.capacity;

  for (int64_t row0 = (int64_t)blockIdx.y * kPagedRows; row0 < rows; row0 += (int64_t)gridDim.y * kPagedRows) {
    // RW tiles of rows side by side (a power of two), KW waves to each, which take turns along the split.
    const int tiles = (int)min((rows - row0 + 16 * QT - 1) / (16 * QT), (int64_t)kPagedRows / (16 * QT));
    int RW = 1;
    while (RW < tiles) RW *= 2;
    const int rw = wave % RW, kw = wave / RW, KW = T::kWaves / RW;
    int last = 0;  // the last row of the wave's tiles
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      const int64_t at = row0 + (rw * QT + qt) * 16 + W.r16;
      const int i = (int)(at / S.G), hq = W.h * S.G + (int)(at - (int64_t)i * S.G);
      W.row[qt].valid = at < rows;
      W.row[qt].bits = ~0ull;
      W.seen[qt] = min(length, W.context + min(i, n) + 1);
      if (S.ancestors) {
        W.row[qt].bits = W.row[qt].valid ? (uint64_t)S.ancestors[first + i] : 0;
        W.seen[qt] = min(length, W.context + 64);
      }
      const uint16_t* x = S.q.x + (int64_t)(first + i) * S.q.row + (int64_t)hq * S.q.head;
#pragma unroll
      for (int c = 0; c < T::kQK; ++c) {
        const int d = Q8 ? (c / 2) * 64 + W.g * 16 + (c & 1) * 8 : c * 32 + W.g * 8;
        u32x4 v = {0u, 0u, 0u, 0u};
        if (W.row[qt].valid) v = *reinterpret_cast<const u32x4*>(x + d);
        W.q[qt][c] = as_bf16x8(v);
      }
      W.m[qt] = -__builtin_inff();
      W.l[qt] = 0.0f;
#pragma unroll
      for (int dt = 0; dt < T::kVT; ++dt) W.o[qt][dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      last = max(last, (int)min((row0 + (rw * QT + qt) * 16 + 15) / S.G, (int64_t)n - 1));
    }
    const int begin = split * per;
    int end = min(begin + per, length);
    if (!S.ancestors) end = min(end, W.context + last + 1);  // (nothing later is seen)
    if (rw < tiles) {
      const int t = begin + kw * T::kStep, stride = KW * T::kStep;
      W.run(t, end, stride);
      if (!Q8 && W.odd) {
        QueryAddress at[QT];
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) {
          const int64_t row = row0 + (rw * QT + qt) * 16 + W.r16;
          const int i = (int)(row / S.G), hq = W.h * S.G + (int)(row - (int64_t)i * S.G);
          at[qt].x = W.row[qt].valid ? S.q.x + (int64_t)(first + i) * S.q.row + (int64_t)hq * S.q.head : nullptr;
        }
        W.add_odd_values(t, end, stride, at);
        W.odd = false;
      }
    }

#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      W.l[qt] += __shfl_xor(W.l[qt], 16);
      W.l[qt] += __shfl_xor(W.l[qt], 32);
    }
    // The waves of the same rows: the upper half hands over to the lower.
    for (int half = KW / 2; half > 0; half /= 2) {
      f32x4* s_o = reinterpret_cast<f32x4*>(s_join);
      float* s_ml = reinterpret_cast<float*>(s_join + (size_t)(T::kWaves / 2) * QT * T::kVT * 1024);
      __syncthreads();
      if (kw >= half && kw < 2 * half) {
        const int slot = (kw - half) * RW + rw;
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) {
#pragma unroll
          for (int dt = 0; dt < T::kVT; ++dt) s_o[((slot * QT + qt) * T::kVT + dt) * 64 + W.lane] = W.o[qt][dt];
          if (W.g == 0) {
            s_ml[(slot * QT + qt) * 32 + W.r16] = W.m[qt];
            s_ml[(slot * QT + qt) * 32 + 16 + W.r16] = W.l[qt];
          }
        }
      }
      __syncthreads();
      if (kw < half) {
        const int slot = kw * RW + rw;
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) {
          const float m2 = s_ml[(slot * QT + qt) * 32 + W.r16], l2 = s_ml[(slot * QT + qt) * 32 + 16 + W.r16];
          const float top = fmaxf(W.m[qt], m2);
          const float f1 = W.m[qt] == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(W.m[qt] - top);
          const float f2 = m2 == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m2 - top);
          W.m[qt] = top;
          W.l[qt] = W.l[qt] * f1 + l2 * f2;
#pragma unroll
          for (int dt = 0; dt < T::kVT; ++dt)
            W.o[qt][dt] = W.o[qt][dt] * f1 + s_o[((slot * QT + qt) * T::kVT + dt) * 64 + W.lane] * f2;
        }
      }
    }
    if (kw == 0 && rw < tiles) {
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) {
        const int64_t at = row0 + (rw * QT + qt) * 16 + W.r16;
        const int i = (int)(at / S.G), hq = W.h * S.G + (int)(at - (int64_t)i * S.G);
        if (!W.row[qt].valid) continue;
        if (whole) {
          const bool empty = S.ancestors && W.context == 0 && (W.row[qt].bits & (n < 64 ? (1ull << n) - 1 : ~0ull)) == 0;
          const float inv = empty ? 0.0f : 1.0f / W.l[qt];
          const int64_t out = ((int64_t)(first + i) * heads_q + hq) * D;
          const uint16_t* gate = S.gate.x ? S.gate.x + (int64_t)(first + i) * S.gate.row + (int64_t)hq * S.gate.head : nullptr;
#pragma unroll
          for (int dt = 0; dt < T::kVT; ++dt) {
            const int d = dt * 16 + W.g * 4;
            f32x4 x = W.o[qt][dt] * inv;
            if (gate) {
              const u32x2 y = *reinterpret_cast<const u32x2*>(gate + d);
              x[0] *= sigmoid(bf16_to_f32(y[0] & 0xFFFFu));
              x[1] *= sigmoid(bf16_to_f32(y[0] >> 16));
              x[2] *= sigmoid(bf16_to_f32(y[1] & 0xFFFFu));
              x[3] *= sigmoid(bf16_to_f32(y[1] >> 16));
            }
            *reinterpret_cast<u32x2*>(S.out + out + d) = u32x2{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3])};
          }
        } else {
          const int64_t part = ((int64_t)S.plan.part()[r] + (int64_t)split * n + i) * heads_q + hq;
#pragma unroll
          for (int dt = 0; dt < T::kVT; ++dt) *reinterpret_cast<f32x4*>(S.part + part * D + dt * 16 + W.g * 4) = W.o[qt][dt];
          if (W.g == 0) {
            S.part_ml[part * 2] = W.m[qt];
            S.part_ml[part * 2 + 1] = W.l[qt];
          }
        }
      }
    }
  }
}

constexpr int kJoinThreads = 256;

// The splits of each row and head joined; zeros for rows without a request. kLanes lanes of 4 dimensions to a split.
template <int D>
__global__ __launch_bounds__(kJoinThreads) void paged_join_kernel(PagedParams S, int64_t m0) {
  constexpr int kLanes = D <= 64 ? 16 : D <= 128 ? 32 : 64, kSlices = kJoinThreads / kLanes;
  __shared__ f32x4 s_o[kSlices][kLanes];
  __shared__ float s_m[kSlices], s_l[kSlices];
  const int64_t row = m0 + blockIdx.y, heads_q = gridDim.x;
  const int hq = blockIdx.x, c = threadIdx.x % kLanes, slice = threadIdx.x / kLanes;
  const int r = S.request[row];
  const int64_t out = (row * heads_q + hq) * D;
  if (r < 0) {
    if (threadIdx.x < D / 4) *reinterpret_cast<u32x2*>(S.out + out + threadIdx.x * 4) = u32x2{0u, 0u};
    return;
  }
  const int n = S.plan.count()[r], length = S.plan.length()[r], per = S.plan.per()[r];
  if (per >= length) return;
  const int i = (int)row - S.plan.first()[r], splits = (length + per - 1) / per;
  const int64_t part = ((int64_t)S.plan.part()[r] + i) * heads_q + hq, stride = (int64_t)n * heads_q;
  float m = -__builtin_inff(), l = 0.0f;
  f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int s = slice; s < splits; s += kSlices) {
    const int64_t at = part + s * stride;
    const float m2 = S.part_ml[at * 2], l2 = S.part_ml[at * 2 + 1];
    const f32x4 o2 = c * 4 < D ? *reinterpret_cast<const f32x4*>(S.part + at * D + c * 4) : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const float top = fmaxf(m, m2);
    const float f1 = m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m - top);
    const float f2 = m2 == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m2 - top);
    m = top;
    l = l * f1 + l2 * f2;
    o = o * f1 + o2 * f2;
  }
  s_o[slice][c] = o;
  if (c == 0) {
    s_m[slice] = m;
    s_l[slice] = l;
  }
  __syncthreads();
  if (slice != 0 || c * 4 >= D) return;
  float top = -__builtin_inff();
#pragma unroll
  for (int s = 0; s < kSlices; ++s) top = fmaxf(top, s_m[s]);
  l = 0.0f;
  o = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int s = 0; s < kSlices; ++s) {
    const float f = s_m[s] == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(s_m[s] - top);
    l += s_l[s] * f;
    o += s_o[s][c] * f;
  }
  const uint64_t bits = S.ancestors ? (uint64_t)S.ancestors[row] : 0;
  const bool empty = S.ancestors && length == n && (bits & (n < 64 ? (1ull << n) - 1 : ~0ull)) == 0;
  o *= empty ? 0.0f : 1.0f / l;
  if (S.gate.x) {
    const u32x2 y = *reinterpret_cast<const u32x2*>(S.gate.x + row * S.gate.row + (int64_t)hq * S.gate.head + c * 4);
    o[0] *= sigmoid(bf16_to_f32(y[0] & 0xFFFFu));
    o[1] *= sigmoid(bf16_to_f32(y[0] >> 16));
    o[2] *= sigmoid(bf16_to_f32(y[1] & 0xFFFFu));
    o[3] *= sigmoid(bf16_to_f32(y[1] >> 16));
  }
  *reinterpret_cast<u32x2*>(S.out + out + c * 4) = u32x2{pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3])};
}

template <int D, int QT, bool Q8>
hipError_t launch_tiles(const PagedParams& p, int64_t M, const PagedShape& shape, hipStream_t stream) {
  using T = PagedTraits<D, QT, Q8>;
  static LdsAllowance allowance;
  const void* f = reinterpret_cast<const void*>(&paged_kernel<D, QT, Q8>);
  if (T::kJoin > 64 * 1024)
    if (hipError_t e = allowance.allow(f, T::kJoin)) return e;
  const int64_t blocks = ((int64_t)p.max_rows * p.G + kPagedRows - 1) / kPagedRows;
  const dim3 grid((unsigned)((shape.splits + p.plan.R) * p.cache.heads), (unsigned)(blocks < 4096 ? blocks : 4096));
  if (blocks > 0 && p.plan.R > 0) hipLaunchKernelGGL((paged_kernel<D, QT, Q8>), grid, dim3(T::kWaves * 64), T::kJoin, stream, p);
  return hipGetLastError();
}

template <int D>
hipError_t launch_dim(const PagedParams& p, int64_t M, const PagedShape& shape, bool q8, hipStream_t stream) {
  const bool one = (int64_t)p.max_rows * p.G <= 16;
  hipError_t e = hipErrorInvalidValue;
  if constexpr (D % 64 == 0) {
    if (q8) e = one ? launch_tiles<D, 1, true>(p, M, shape, stream) : launch_tiles<D, 2, true>(p, M, shape, stream);
  }
  if (!q8) e = one ? launch_tiles<D, 1, false>(p, M, shape, stream) : launch_tiles<D, 2, false>(p, M, shape, stream);
  if (e != hipSuccess) return e;
  constexpr int64_t kRows = 65535;
  const int64_t heads = (int64_t)p.cache.heads * p.G;
  for (int64_t m0 = 0; m0 < M; m0 += kRows)
    hipLaunchKernelGGL((paged_join_kernel<D>), dim3((unsigned)heads, (unsigned)(M - m0 < kRows ? M - m0 : kRows)),
                       dim3(kJoinThreads), 0, stream, p, m0);
  return hipGetLastError();
}

}  // namespace

PagedShape paged_shape(int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t max_rows, int cus) {
  const int G = (int)(heads / kv_heads);
  return {G, (2 * cus + kv_heads - 1) / kv_heads};
}

int64_t paged_partial_rows(const PagedShape& s, int64_t M, int64_t R, int64_t max_rows) {
  const int64_t items = s.splits + R, by_block = kPagedRows * items + M * s.G, by_rows = items * max_rows * s.G;
  return by_block < by_rows ? by_block : by_rows;
}

hipError_t launch_paged_attention(const PagedParams& p, int64_t M, const PagedShape& shape, int D, bool q8, hipStream_t stream) {
  switch (D) {
    case 64: return launch_dim<64>(p, M, shape, q8, stream);
    case 96: return launch_dim<96>(p, M, shape, q8, stream);
    case 128: return launch_dim<128>(p, M, shape, q8, stream);
    case 192: return launch_dim<192>(p, M, shape, q8, stream);
    default: return launch_dim<256>(p, M, shape, q8, stream);
  }
}

}  // namespace qmm4
