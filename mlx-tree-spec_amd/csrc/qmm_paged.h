// What the paged attention's two kernels share (qmm_paged.hip, qmm_paged_tile.hip): a wave's query rows, their softmax, what
// they see, and how waves and splits are joined.
//
// Both products run on 16x16x32 matrix instructions with the tokens' side as the first operand:
//   S^T = K Q^T  (16 tokens x 16 query rows),   O^T = V^T P^T  (16 dimensions x 16 query rows)
// The cache's layout makes pieces of keys (8 dimensions of a token) and of values (8 tokens of a dimension) operands as they
// lie, or behind a conversion from 8 bits. S^T leaves each lane with probabilities of one query row (lane % 16); the order of
// tokens within a step of 32 is chosen (row 4 g + i of tile tt is token 8 g + 4 tt + i, g = lane / 16) so that they are the
// second operand of O^T without a move between lanes.
//
// The running maximum moves only where a logit passes it by more than 2^8, so that most steps need no exchange between lanes. It
// is held above the largest logit by those 2^8 and by the tokens that a request may have: all its probabilities together stay
// below 1, and no sum of finite values overflows, whatever their size, nor does a probability times a scale of 8 bits. What this takes
// is as many powers of two of how small a probability may be (2^-126). (The bound on the tokens comes with the call: the widest kernels
// have no vector register for a request's own.)
#pragma once

#include "qmm4_common.h"
#include "qmm_cache_kernels.h"

namespace qmm4 {

constexpr float kLog2e = 1.44269504f;
// The running maximum before any token is seen: below every finite logit (in powers of two), finite itself, so that no difference
// of two is NaN.
constexpr float kNone = -0x1p127f;

// The largest of three. (v_max3_f32 by itself: fmaxf has every operand made quiet first.)
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

__device__ __forceinline__ f32x4 paged_mma(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// Byte BYTE of w, signed, as a float: one instruction. (Written out: from C++ hipcc 7.2 takes two, and keeps a loaded word's bytes
// in registers of their own from the load on.)
template <int BYTE>
__device__ __forceinline__ float code(uint32_t w) {
  float f;
  if constexpr (BYTE == 0) asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_0" : "=v"(f) : "v"(w));
  if constexpr (BYTE == 1) asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_1" : "=v"(f) : "v"(w));
  if constexpr (BYTE == 2) asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_2" : "=v"(f) : "v"(w));
  if constexpr (BYTE == 3) asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_3" : "=v"(f) : "v"(w));
  return f;
}
// 8 codes -> bf16 (exact).
__device__ __forceinline__ bf16x8 codes8(uint32_t lo, uint32_t hi) {
  return as_bf16x8(u32x4{pack_bf16x2(code<0>(lo), code<1>(lo)), pack_bf16x2(code<2>(lo), code<3>(lo)),
                         pack_bf16x2(code<0>(hi), code<1>(hi)), pack_bf16x2(code<2>(hi), code<3>(hi))});
}

__device__ __forceinline__ float sigmoid(float x) { return 1.0f / (1.0f + __expf(-x)); }

// x * sigmoid(gate) of 4 neighbouring dimensions, rounded.
__device__ __forceinline__ u32x2 gated_bf16(f32x4 x, bool gated, u32x2 y) {
  if (gated) {
    x[0] *= sigmoid(bf16_to_f32(y[0] & 0xFFFFu));
    x[1] *= sigmoid(bf16_to_f32(y[0] >> 16));
    x[2] *= sigmoid(bf16_to_f32(y[1] & 0xFFFFu));
    x[3] *= sigmoid(bf16_to_f32(y[1] >> 16));
  }
  return u32x2{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3])};
}

// 8 tokens' values of one dimension, the first of them `past` behind the request's tokens (below 0: before their end), with zeros in
// place of the tokens past the last, which the cache need not hold, and of what is not finite (*odd: there was some): a
// probability of zero would not keep it from the rows that do not see it.
__device__ __forceinline__ u32x4 clean_values(u32x4 v, int past, bool* odd) {
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const uint32_t keep = past + 2 * w >= 0 ? 0u : past + 2 * w + 1 >= 0 ? 0xFFFFu : 0xFFFFFFFFu;
    uint32_t x = v[w] & keep;
    const bool lo = (x & 0x7F80u) == 0x7F80u, hi = (x & 0x7F800000u) == 0x7F800000u;
    *odd |= lo | hi;
    x = lo ? x & 0xFFFF0000u : x;
    v[w] = hi ? x & 0xFFFFu : x;
  }
  return v;
}

// Whether a row without a context sees none of its request's n rows: its result is zero.
__device__ __forceinline__ bool paged_empty(const int64_t* ancestors, int64_t row, int length, int n) {
  if (!ancestors || length != n) return false;
  return ((uint64_t)ancestors[row] & (n < 64 ? (1ull << n) - 1 : ~0ull)) == 0;
}

// Q8: a cache of codes with scales. CODES: the products' operands are read as codes (else as bf16 numbers, which codes may have been
// made before).
template <int D, int QT, bool Q8, bool CODES = Q8>
struct PagedRows {
  static constexpr int E = Q8 ? 16 : 8;  // elements of 16 bytes of the cache
  static constexpr int kStep = 32;       // tokens of a wave's step
  static constexpr int kKT = 2;          // tiles of 16 tokens
  static constexpr int kKC = D / (CODES ? 64 : 32);  // 16-byte pieces of a key's operands for each lane
  static constexpr int kQK = D / 32;     // matrix instructions along D
  static constexpr int kVT = D / 16;     // tiles of 16 dimensions
  // LDS of a wave that hands over its results.
  static constexpr int kHandBytes = QT * (kVT * 1024 + 128);

  const PagedParams& S;
  const PagedItem& I;
  const int32_t* table;  // the request's row
  int lane, r16, g, h, length, context;
  float unit;  // of a logit, in powers of two
  bf16x8 q[QT][kQK];
  uint64_t bits[QT];  // the step's rows that the row sees (all ones without ancestors)
  int seen[QT];       // no token from this on is seen
  float m[QT], l[QT];
  f32x4 o[QT][kVT];
  bool odd = false;  // a value that is not finite was left out

  __device__ __forceinline__ PagedRows(const PagedParams& s, const PagedItem& item, int head) : S(s), I(item), h(head) {
    lane = threadIdx.x & 63;
    r16 = lane & 15;
    g = lane >> 4;
    length = I.length;
    context = length - I.rows;
    table = S.table + (int64_t)I.request * S.capacity;
    // (Never 0: what is masked has to stay at -infinity.)
    unit = S.scale == 0.0f ? 0x1p-149f : fabsf(S.scale) * kLog2e;
  }

  // Query row `at` of the request's n G: its row of the step and its head.
  __device__ __forceinline__ void place(int at, int* i, int* hq) const {
    *i = (int)((uint32_t)at / (uint32_t)S.G);
    *hq = h * S.G + at - *i * S.G;
  }
  __device__ __forceinline__ const uint16_t* query(int at) const {
    int i, hq;
    place(at, &i, &hq);
    return at < I.rows * S.G ? S.q.x + (int64_t)(I.first + i) * S.q.row + (int64_t)hq * S.q.head : nullptr;
  }

  // The wave's query rows from `row0` on, with their sign turned where scale is negative (what the maximum is taken of rises
  // with the logit then). Returns one past the last token that any of them sees.
  __device__ __forceinline__ int load_rows(int row0) {
    int end = 0;
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      const int at = row0 + qt * 16 + r16;
      int i, hq;
      place(at, &i, &hq);
      const uint16_t* x = query(at);
      bits[qt] = ~0ull;
      seen[qt] = min(length, context + min(i, I.rows) + 1);
      if (S.ancestors) {
        bits[qt] = x ? (uint64_t)S.ancestors[I.first + i] : 0;
        seen[qt] = min(length, context + 64);
      }
#pragma unroll
      for (int c = 0; c < kQK; ++c) {
        const int d = CODES ? (c / 2) * 64 + g * 16 + (c & 1) * 8 : c * 32 + g * 8;
        u32x4 v = {0u, 0u, 0u, 0u};
        if (x) v = *reinterpret_cast<const u32x4*>(x + d);
        q[qt][c] = as_bf16x8(v);
      }
      m[qt] = kNone;
      l[qt] = 0.0f;
#pragma unroll
      for (int dt = 0; dt < kVT; ++dt) o[qt][dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      end = max(end, min((row0 + qt * 16 + 15) / S.G, I.rows - 1));
    }
    if (S.scale < 0.0f) {  // (behind a branch: nothing else waits for the rows here)
#pragma unroll
      for (int qt = 0; qt < QT; ++qt)
#pragma unroll
        for (int c = 0; c < kQK; ++c) q[qt][c] = as_bf16x8(__builtin_bit_cast(u32x4, q[qt][c]) ^ 0x80008000u);
    }
    return S.ancestors ? length : context + end + 1;
  }

  // The first token of a group of 8, within the request's.
  __device__ __forceinline__ int group(int token) const { return min(token, (length - 1) & ~7); }
  // A page of the cache, whatever the table holds.
  __device__ __forceinline__ int valid_page(int page) const { return (int)min((uint32_t)page, (uint32_t)S.cache.pages - 1); }

  // Whether the row sees a token: all of the context, and of what follows up to `seen` what its bits say. (Without branches:
  // hipcc 7.2 has lost the selected value of nested divergent ones here.)
  __device__ __forceinline__ bool sees(int qt, int tok) const {
    const int j = tok - context;
    return (j < 0) | ((tok < seen[qt]) & ((uint32_t)(bits[qt] >> (j & 63)) & 1u));
  }

  // The probabilities of a step's tokens from t, whose products are s, as the second operand of the values' product; m, l and
  // o move with them. 8 bits: kscale multiplies the products, vscale the probabilities.
  __device__ __forceinline__ void softmax(int t, f32x4 (&s)[QT][kKT], const f32x4* kscale, const f32x4* vscale,
                                          bf16x8 (&p)[QT]) {
    const bool masked = t + kStep > context;
    if constexpr (Q8) {
#pragma unroll
      for (int qt = 0; qt < QT; ++qt)
#pragma unroll
        for (int tt = 0; tt < kKT; ++tt) s[qt][tt] *= kscale[tt];
    }
    if (masked) {
#pragma unroll
      for (int qt = 0; qt < QT; ++qt)
#pragma unroll
        for (int tt = 0; tt < kKT; ++tt)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[qt][tt][i] = sees(qt, t + 8 * g + 4 * tt + i) ? s[qt][tt][i] : -__builtin_inff();
    }
    // Arguments of the exponentials beside the present maximum, which stays where none passes the largest logit by more than kPagedSlack.
    float e[QT][8];
    const auto arguments = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int qt = 0; qt < QT; ++qt)
#pragma unroll
        for (int j = 0; j < 8; ++j) e[qt][j] = __builtin_fmaf(s[qt][j / 4][j % 4], unit, -m[qt]);
    };
    arguments();
    float top = kNone;
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      top = max3(top, max3(e[qt][0], e[qt][1], e[qt][2]), max3(e[qt][3], e[qt][4], e[qt][5]));
      top = max3(top, e[qt][6], e[qt][7]);
    }
    if (__any(top > -S.tokens)) {
#pragma unroll
      for (int qt = 0; qt < QT; ++qt) {
        float now = s[qt][0][0];
#pragma unroll
        for (int j = 1; j < 8; ++j) now = fmaxf(now, s[qt][j / 4][j % 4]);
        now = __builtin_fmaf(now, unit, S.tokens);
        now = fmaxf(now, __shfl_xor(now, 16));
        now = fmaxf(fmaxf(now, __shfl_xor(now, 32)) + kPagedSlack, m[qt]);
        const float f = __builtin_amdgcn_exp2f(m[qt] - now);
        l[qt] *= f;
#pragma unroll
        for (int dt = 0; dt < kVT; ++dt) o[qt][dt] *= f;
        m[qt] = now;
      }
      arguments();
    }
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      float sum[4];
#pragma unroll
      for (int j = 0; j < 8; ++j) e[qt][j] = __builtin_amdgcn_exp2f(e[qt][j]);
#pragma unroll
      for (int j = 0; j < 4; ++j) sum[j] = e[qt][j] + e[qt][j + 4];
      l[qt] += (sum[0] + sum[1]) + (sum[2] + sum[3]);
    }
    if constexpr (Q8) {
#pragma unroll
      for (int qt = 0; qt < QT; ++qt)
#pragma unroll
        for (int j = 0; j < 8; ++j) e[qt][j] *= vscale[j / 4][j % 4];
      if (masked) {  // (what is not there may have a scale that is not a number)
#pragma unroll
        for (int qt = 0; qt < QT; ++qt)
#pragma unroll
          for (int j = 0; j < 8; ++j) e[qt][j] = sees(qt, t + 8 * g + j) ? e[qt][j] : 0.0f;
      }
    }
    // (bf16, as the values are: the matrix instructions of 32 bits are a sixteenth as fast. Half a step each, 2^-8, beside a sum of them
    // that stays in 32 bits: against 64 bits 1.3 to 1.4 times the error of products in fp32, whose result is rounded to bf16 as well.)
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      u32x4 w;
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = pack_bf16x2(e[qt][2 * i], e[qt][2 * i + 1]);
      p[qt] = as_bf16x8(w);
    }
  }

  // What those values add to o for the rows that see them: the wave's steps t, t + stride, .. again, token by token, where what
  // was made clean, `reach` tokens from the step's first on, ends past the context.
  __device__ __forceinline__ void add_odd_values(int t, int end, int stride, int reach, int row0) {
    if (Q8 || !__any(odd)) return;
    odd = false;
    const int shift = S.cache.page_shift;
    for (; t < end; t += stride) {
      if (t + reach <= context) continue;
      for (int tok = t; tok < min(t + kStep, length); ++tok) {
        const int64_t head = (int64_t)valid_page(table[tok >> shift]) * S.cache.heads + h;
        const int off = tok & ((1 << shift) - 1);
        const uint16_t* v = static_cast<const uint16_t*>(S.cache.values) + ((((head << shift) + off) / 8) * D) * 8 + off % 8;
        const uint16_t* k = static_cast<const uint16_t*>(S.cache.keys) + (((head * (D / 8)) << shift) + off) * 8;
        bool any = false;
        for (int d = lane; d < D; d += 64) any |= (v[d * 8] & 0x7F80u) == 0x7F80u;
        if (!__any(any)) continue;
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) {
          const uint16_t* y = query(row0 + qt * 16 + r16);
          float x = 0.0f;
          for (int d = g; d < D; d += 4)
            x += y ? bf16_to_f32(y[d]) * bf16_to_f32(k[((int64_t)(d / 8) << shift) * 8 + d % 8]) : 0.0f;
          x += __shfl_xor(x, 16);
          x += __shfl_xor(x, 32);
          const float p = __builtin_amdgcn_exp2f(x * (S.scale * kLog2e) - m[qt]);
          const bool see = sees(qt, tok);
#pragma unroll
          for (int dt = 0; dt < kVT; ++dt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t z = v[(dt * 16 + 4 * g + i) * 8];
              const float add = p * bf16_to_f32(z);
              o[qt][dt][i] += (see & ((z & 0x7F80u) == 0x7F80u)) ? add : 0.0f;
            }
        }
      }
    }
  }

  // l of a row in all of its lanes.
  __device__ __forceinline__ void sum_lanes() {
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      l[qt] += __shfl_xor(l[qt], 16);
      l[qt] += __shfl_xor(l[qt], 32);
    }
  }

  // The wave's results to LDS (kHandBytes), and another wave's, of the same rows, joined to its own.
  __device__ __forceinline__ void hand_over(char* lds) const {
    f32x4* s_o = reinterpret_cast<f32x4*>(lds);
    float* s_ml = reinterpret_cast<float*>(lds + QT * kVT * 1024);
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
#pragma unroll
      for (int dt = 0; dt < kVT; ++dt) s_o[(qt * kVT + dt) * 64 + lane] = o[qt][dt];
      if (g == 0) {
        s_ml[qt * 32 + r16] = m[qt];
        s_ml[qt * 32 + 16 + r16] = l[qt];
      }
    }
  }
  __device__ __forceinline__ void take_over(const char* lds) {
    const f32x4* s_o = reinterpret_cast<const f32x4*>(lds);
    const float* s_ml = reinterpret_cast<const float*>(lds + QT * kVT * 1024);
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      const float m2 = s_ml[qt * 32 + r16], l2 = s_ml[qt * 32 + 16 + r16], top = fmaxf(m[qt], m2);
      const float f1 = __builtin_amdgcn_exp2f(m[qt] - top), f2 = __builtin_amdgcn_exp2f(m2 - top);
      m[qt] = top;
      l[qt] = l[qt] * f1 + l2 * f2;
#pragma unroll
      for (int dt = 0; dt < kVT; ++dt) o[qt][dt] = o[qt][dt] * f1 + s_o[(qt * kVT + dt) * 64 + lane] * f2;
    }
  }

  // The rows' results, or where the request has several splits the part of this one.
  __device__ __forceinline__ void write(int row0) const {
    const int64_t heads = (int64_t)S.cache.heads * S.G;
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      const int at = row0 + qt * 16 + r16;
      if (at >= I.rows * S.G) continue;
      int i, hq;
      place(at, &i, &hq);
      if (I.part < 0) {
        const float inv = paged_empty(S.ancestors, I.first + i, length, I.rows) ? 0.0f : 1.0f / l[qt];
        uint16_t* out = S.out + ((int64_t)(I.first + i) * heads + hq) * D + 4 * g;
        const uint16_t* gate = S.gate.x ? S.gate.x + (int64_t)(I.first + i) * S.gate.row + (int64_t)hq * S.gate.head + 4 * g : nullptr;
#pragma unroll
        for (int dt = 0; dt < kVT; ++dt)
          *reinterpret_cast<u32x2*>(out + dt * 16) =
              gated_bf16(o[qt][dt] * inv, gate != nullptr, gate ? *reinterpret_cast<const u32x2*>(gate + dt * 16) : u32x2{0u, 0u});
      } else {
        const int64_t part = ((int64_t)I.part + i) * heads + hq;
#pragma unroll
        for (int dt = 0; dt < kVT; ++dt) *reinterpret_cast<f32x4*>(S.part + part * D + dt * 16 + g * 4) = o[qt][dt];
        if (g == 0) {
          S.part_ml[part * 2] = m[qt];
          S.part_ml[part * 2 + 1] = l[qt];
        }
      }
    }
  }
};

// The kernel of more than 16 query rows to a key head.
hipError_t launch_paged_tile(const PagedParams& p, int D, bool q8, hipStream_t stream);

}  // namespace qmm4
