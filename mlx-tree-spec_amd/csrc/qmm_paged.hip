// Attention of a step's new rows over a paged key-value cache, split over the cache's length and joined
// (include/qmm_cache.h). With G query heads to a key head, a request of n rows has n G query rows for each key head:
//   s = scale q . k_t,   m = max s,   l = sum exp(s - m),   o = sum exp(s - m) v_t,   out = o / l  (* sigmoid(gate))
//
// This file: up to 16 query rows to a key head (decode), the join of splits, and the choice. Every byte of the cache is used
// once, for 16 rows at most: bound by HBM. A wave loads its operands from memory to registers, 1 KB an instruction in whole
// runs of 64 bytes and more, without LDS, and takes every KW-th step of its workgroup's split; while a step's probabilities
// are made the next step's keys are on their way, and its values while the products with the present ones run. Waves join
// through LDS, splits through memory (fp32) and a second kernel.
#include "qmm_paged.h"

namespace qmm4 {

namespace {

template <int D, bool Q8>
struct RowsTraits {
  using R = PagedRows<D, 1, Q8>;
  // Registers of o, q, s, keys, values and scales; with what else there is more than 256: one wave to a SIMD.
  static constexpr int kRegisters = 4 * (R::kVT + R::kQK + R::kKT + R::kKT * R::kKC + R::kVT + (Q8 ? 3 * R::kKT : 0));
  static constexpr int kWaves = kRegisters > 176 ? 4 : 8;
  static constexpr size_t kJoin = (size_t)(kWaves / 2) * R::kHandBytes;
};

template <int D, bool Q8>
struct PagedWave : PagedRows<D, 1, Q8> {
  using R = PagedRows<D, 1, Q8>;
  static constexpr int E = R::E;
  u32x4 kf[R::kKT][R::kKC], vf[R::kVT];
  f32x4 ks[Q8 ? R::kKT : 1], vs[Q8 ? R::kKT : 1];

  using R::R;

  __device__ __forceinline__ int page(int token) const {
    return this->valid_page(this->table[this->group(token) >> this->S.cache.page_shift]);
  }

  __device__ __forceinline__ void load_keys(int t, int page) {
    const CacheArrays& C = this->S.cache;
    const int shift = C.page_shift, tok = this->group(t + E * (this->r16 >> 2)) & ((1 << shift) - 1);
    const char* p = static_cast<const char*>(C.keys) +
                    (((((int64_t)page * C.heads + this->h) * (D / E) + this->g) << shift) + tok + (this->r16 & 3)) * 16;
#pragma unroll
    for (int c = 0; c < R::kKC; ++c)
#pragma unroll
      for (int tt = 0; tt < R::kKT; ++tt) kf[tt][c] = *reinterpret_cast<const u32x4*>(p + ((int64_t)c << (shift + 6)) + tt * 64);
  }

  __device__ __forceinline__ void load_values(int t, int page) {
    const CacheArrays& C = this->S.cache;
    const int shift = C.page_shift, tok = this->group(t + E * this->g) & ((1 << shift) - 1);
    const char* p = static_cast<const char*>(C.values) +
                    ((((((int64_t)page * C.heads + this->h) << shift) + tok) / E) * D + this->r16) * 16;
#pragma unroll
    for (int dt = 0; dt < R::kVT; ++dt) vf[dt] = *reinterpret_cast<const u32x4*>(p + dt * 256);
  }

  __device__ __forceinline__ void load_scales(int t, int page) {
    if constexpr (Q8) {
      const CacheArrays& C = this->S.cache;
      const int shift = C.page_shift, tok = this->group(t + E * this->g) & ((1 << shift) - 1);
      const int64_t at = (((int64_t)page * C.heads + this->h) << shift) + tok;
#pragma unroll
      for (int tt = 0; tt < R::kKT; ++tt) {
        ks[tt] = *reinterpret_cast<const f32x4*>(C.key_scales + at + 4 * tt);
        vs[tt] = *reinterpret_cast<const f32x4*>(C.value_scales + at + 4 * tt);
      }
    }
  }

  // One step from t, whose keys and values are loaded; MORE: those of t + stride are, meanwhile (kp, vp: their pages on entry;
  // on return those of t + 2 stride).
  template <bool MORE>
  __device__ __forceinline__ void step(int t, int stride, int* kp, int* vp) {
    f32x4 s[R::kKT], kscale[Q8 ? R::kKT : 1], vscale[Q8 ? R::kKT : 1];
#pragma unroll
    for (int tt = 0; tt < R::kKT; ++tt) s[tt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int c = 0; c < R::kKC; ++c)
#pragma unroll
      for (int tt = 0; tt < R::kKT; ++tt) {
        if constexpr (Q8) {
          s[tt] = paged_mma(codes8(kf[tt][c][0], kf[tt][c][1]), this->q[0][2 * c], s[tt]);
          s[tt] = paged_mma(codes8(kf[tt][c][2], kf[tt][c][3]), this->q[0][2 * c + 1], s[tt]);
        } else {
          s[tt] = paged_mma(as_bf16x8(kf[tt][c]), this->q[0][c], s[tt]);
        }
      }
    if constexpr (Q8) {
#pragma unroll
      for (int tt = 0; tt < R::kKT; ++tt) {
        kscale[tt] = ks[tt];
        vscale[tt] = vs[tt];
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    int next_page = 0;
    if constexpr (MORE) {
      next_page = *vp;
      load_keys(t + stride, *kp);
      load_scales(t + stride, next_page);
      *kp = page(t + 2 * stride + E * (this->r16 >> 2));
      *vp = page(t + 2 * stride + E * this->g);
    }
    __builtin_amdgcn_sched_barrier(0);
    bf16x8 p[E / 8];
    this->softmax(t, 0, s, kscale, vscale, p);
    if (!Q8 && t + R::kStep > this->context) {
#pragma unroll
      for (int dt = 0; dt < R::kVT; ++dt) vf[dt] = this->clean(vf[dt], t);
    }
#pragma unroll
    for (int dt = 0; dt < R::kVT; ++dt) {
      if constexpr (Q8) {
        this->o[0][dt] = paged_mma(codes8(vf[dt][0], vf[dt][1]), p[0], this->o[0][dt]);
        this->o[0][dt] = paged_mma(codes8(vf[dt][2], vf[dt][3]), p[E / 8 - 1], this->o[0][dt]);
      } else {
        this->o[0][dt] = paged_mma(as_bf16x8(vf[dt]), p[0], this->o[0][dt]);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (MORE) load_values(t + stride, next_page);
    __builtin_amdgcn_sched_barrier(0);
  }

  // Steps t, t + stride, .. below end.
  __device__ __forceinline__ void run(int t, int end, int stride) {
    if (t >= end) return;
    const int vpage = page(t + E * this->g);
    load_keys(t, page(t + E * (this->r16 >> 2)));
    load_scales(t, vpage);
    load_values(t, vpage);
    int kp = page(t + stride + E * (this->r16 >> 2)), vp = page(t + stride + E * this->g);
    for (; t + stride < end; t += stride) step<true>(t, stride, &kp, &vp);
    step<false>(t, stride, &kp, &vp);
  }
};

template <int D, bool Q8>
__global__ __launch_bounds__((RowsTraits<D, Q8>::kWaves * 64)) void paged_rows_kernel(PagedParams S) {
  using T = RowsTraits<D, Q8>;
  using R = PagedRows<D, 1, Q8>;
  __shared__ __attribute__((aligned(16))) char s_join[T::kJoin];
  const int item = blockIdx.x / S.cache.heads;
  if (item >= S.plan.words[0]) return;
  const int split = S.plan.items()[2 * item + 1];
  PagedWave<D, Q8> W(S, S.plan.items()[2 * item], blockIdx.x - item * S.cache.heads);
  const int wave = threadIdx.x >> 6, per = S.plan.per()[W.r];
  const int sees = W.load_rows(0), begin = split * per, end = min(min(begin + per, W.length), sees);
  const int t = begin + wave * R::kStep, stride = T::kWaves * R::kStep;
  W.run(t, end, stride);
  W.add_odd_values(t, end, stride, 0);
  W.sum_lanes();
  // The upper half of the waves hands over to the lower.
#pragma unroll
  for (int half = T::kWaves / 2; half > 0; half /= 2) {
    __syncthreads();
    if (wave >= half && wave < 2 * half) W.hand_over(s_join + (wave - half) * R::kHandBytes);
    __syncthreads();
    if (wave < half) W.take_over(s_join + wave * R::kHandBytes);
  }
  if (wave == 0) W.write(0, split);
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
  uint16_t* out = S.out + (row * heads_q + hq) * D + c * 4;
  if (r < 0) {
    if (slice == 0 && c * 4 < D) *reinterpret_cast<u32x2*>(out) = u32x2{0u, 0u};
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
  o *= paged_empty(S.ancestors, row, length, n) ? 0.0f : 1.0f / l;
  *reinterpret_cast<u32x2*>(out) =
      gated_bf16(o, S.gate.x ? S.gate.x + row * S.gate.row + (int64_t)hq * S.gate.head + c * 4 : nullptr);
}

template <int D>
void launch_rows(const PagedParams& p, int64_t items, bool q8, hipStream_t stream) {
  const dim3 grid((unsigned)(items * p.cache.heads));
  if constexpr (D % 64 == 0) {
    if (q8) hipLaunchKernelGGL((paged_rows_kernel<D, true>), grid, dim3(RowsTraits<D, true>::kWaves * 64), 0, stream, p);
  }
  if (!q8) hipLaunchKernelGGL((paged_rows_kernel<D, false>), grid, dim3(RowsTraits<D, false>::kWaves * 64), 0, stream, p);
}

template <int D>
void launch_join(const PagedParams& p, int64_t M, hipStream_t stream) {
  constexpr int64_t kRows = 65535;
  const unsigned heads = (unsigned)(p.cache.heads * p.G);
  for (int64_t m0 = 0; m0 < M; m0 += kRows)
    hipLaunchKernelGGL((paged_join_kernel<D>), dim3(heads, (unsigned)(M - m0 < kRows ? M - m0 : kRows)), dim3(kJoinThreads), 0,
                       stream, p, m0);
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

hipError_t launch_paged_rows(const PagedParams& p, int64_t items, int D, bool q8, hipStream_t stream) {
  switch (D) {
    case 64: launch_rows<64>(p, items, q8, stream); break;
    case 96: launch_rows<96>(p, items, q8, stream); break;
    case 128: launch_rows<128>(p, items, q8, stream); break;
    case 192: launch_rows<192>(p, items, q8, stream); break;
    default: launch_rows<256>(p, items, q8, stream);
  }
  return hipGetLastError();
}

hipError_t launch_paged_attention(const PagedParams& p, int64_t M, const PagedShape& shape, int D, bool q8, hipStream_t stream) {
  const int64_t items = shape.splits + p.plan.R, rows = (int64_t)p.max_rows * p.G;
  if (p.plan.R > 0 && rows > 0) {
    const hipError_t e = rows <= 16 ? launch_paged_rows(p, items, D, q8, stream)
                                    : launch_paged_tile(p, items, D, q8, stream);
    if (e != hipSuccess) return e;
  }
  switch (D) {
    case 64: launch_join<64>(p, M, stream); break;
    case 96: launch_join<96>(p, M, stream); break;
    case 128: launch_join<128>(p, M, stream); break;
    case 192: launch_join<192>(p, M, stream); break;
    default: launch_join<256>(p, M, stream);
  }
  return hipGetLastError();
}

}  // namespace qmm4
