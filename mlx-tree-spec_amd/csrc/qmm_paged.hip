// Attention of a step's new rows over a paged key-value cache, split over the cache's length and joined
// (include/qmm_cache.h). With G query heads to a key head, a request of n rows has n G query rows for each key head:
//   s = scale q . k_t,   m = max s,   l = sum exp(s - m),   o = sum exp(s - m) v_t,   out = o / l  (* sigmoid(gate))
//
// This file: up to 16 query rows to a key head (decode) of heads up to 128 or 8 bits, the join of splits, and the choice. Every
// byte of the cache is used once, for 16 rows at most: bound by HBM (64 requests of up to 16000 tokens, 8 key heads of 128, 2.4 GB:
// 415 us, 5.8 TB/s; 16 of up to 40000 in 8 bits, 4 of 256: 140-144 us, 5.4 TB/s). A wave loads its operands from memory to registers,
// 1 KB an instruction in whole runs of 64 bytes and more, without LDS, and takes every 8th step of its workgroup's split; while
// a step's probabilities are made the next step's keys are on their way, and its values while the products with the present ones
// run. Waves join through LDS, splits through memory (fp32) and a second kernel (5.3 us for 64 splits of 24 heads of 256).
// That one looks at every row and head, whether they were cut or not (a prompt of 4096 rows of 32 heads, which is not: 47 us of 420).
#include <algorithm>
#include <type_traits>

#include "qmm4_lds.h"
#include "qmm_paged.h"

namespace qmm4 {

namespace {

constexpr int kRowsWaves = 8;

template <int D, bool Q8>
struct PagedWave : PagedRows<D, 1, Q8> {
  using R = PagedRows<D, 1, Q8>;
  using Piece = std::conditional_t<Q8, u32x2, u32x4>;  // 8 tokens of a dimension
  u32x4 kf[R::kKT][R::kKC];
  Piece vf[R::kVT];
  f32x4 ks[Q8 ? R::kKT : 1], vs[Q8 ? R::kKT : 1];

  using R::R;

  __device__ __forceinline__ int page(int token) const {
    return this->valid_page(this->table[this->group(token) >> this->S.cache.page_shift]);
  }

  __device__ __forceinline__ void load_keys(int t, int page) {
    const CacheArrays& C = this->S.cache;
    const int shift = C.page_shift, tok = this->group(t + 8 * (this->r16 >> 2)) & ((1 << shift) - 1);
    const char* p = static_cast<const char*>(C.keys) +
                    (((((int64_t)page * C.heads + this->h) * (D / R::E) + this->g) << shift) + tok + (this->r16 & 3)) * 16;
#pragma unroll
    for (int c = 0; c < R::kKC; ++c)
#pragma unroll
      for (int tt = 0; tt < R::kKT; ++tt) kf[tt][c] = *reinterpret_cast<const u32x4*>(p + ((int64_t)c << (shift + 6)) + tt * 64);
  }

  __device__ __forceinline__ void load_values(int t, int page) {
    const CacheArrays& C = this->S.cache;
    const int shift = C.page_shift, tok = this->group(t + 8 * this->g) & ((1 << shift) - 1);
    const char* p = static_cast<const char*>(C.values) +
                    ((((((int64_t)page * C.heads + this->h) << shift) + tok) / R::E) * D + this->r16) * 16 + (Q8 ? tok & 8 : 0);
#pragma unroll
    for (int dt = 0; dt < R::kVT; ++dt) vf[dt] = *reinterpret_cast<const Piece*>(p + dt * 256);
  }

  __device__ __forceinline__ void load_scales(int t, int page) {
    if constexpr (Q8) {
      const CacheArrays& C = this->S.cache;
      const int shift = C.page_shift, tok = this->group(t + 8 * this->g) & ((1 << shift) - 1);
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
    f32x4 s[1][R::kKT], kscale[Q8 ? R::kKT : 1], vscale[Q8 ? R::kKT : 1];
#pragma unroll
    for (int tt = 0; tt < R::kKT; ++tt) s[0][tt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int c = 0; c < R::kKC; ++c) {
#pragma unroll
      for (int tt = 0; tt < R::kKT; ++tt) {
        if constexpr (Q8) {
          s[0][tt] = paged_mma(codes8(kf[tt][c][0], kf[tt][c][1]), this->q[0][2 * c], s[0][tt]);
          s[0][tt] = paged_mma(codes8(kf[tt][c][2], kf[tt][c][3]), this->q[0][2 * c + 1], s[0][tt]);
        } else {
          s[0][tt] = paged_mma(as_bf16x8(kf[tt][c]), this->q[0][c], s[0][tt]);
        }
      }
      if constexpr (Q8) __builtin_amdgcn_sched_barrier(0);  // (few codes at a time in registers)
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
      *kp = page(t + 2 * stride + 8 * (this->r16 >> 2));
      *vp = page(t + 2 * stride + 8 * this->g);
    }
    __builtin_amdgcn_sched_barrier(0);
    bf16x8 p[1];
    this->softmax(t, s, kscale, vscale, p);
    if constexpr (!Q8) {
      if (t + R::kStep > this->context) {
#pragma unroll
        for (int dt = 0; dt < R::kVT; ++dt) vf[dt] = clean_values(vf[dt], t + 8 * this->g - this->length, &this->odd);
      }
    }
#pragma unroll
    for (int dt = 0; dt < R::kVT; ++dt) {
      if constexpr (Q8) this->o[0][dt] = paged_mma(codes8(vf[dt][0], vf[dt][1]), p[0], this->o[0][dt]);
      else this->o[0][dt] = paged_mma(as_bf16x8(vf[dt]), p[0], this->o[0][dt]);
      if (Q8 && dt % 4 == 3) __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (MORE) load_values(t + stride, next_page);
    __builtin_amdgcn_sched_barrier(0);
  }

  // Steps t, t + stride, .. below end; the query rows are loaded behind the first keys and values.
  __device__ __forceinline__ void run(int t, int end, int stride) {
    const bool any = t < end;
    if (any) {
      // (The first tokens' page came with the item: one load less to wait for.)
      const bool known = this->S.cache.page_shift >= 6 && t < this->I.begin + kPagedUnit;
      const int vpage = known ? this->valid_page(this->I.page) : page(t + 8 * this->g);
      load_keys(t, known ? vpage : page(t + 8 * (this->r16 >> 2)));
      load_scales(t, vpage);
      load_values(t, vpage);
    }
    this->load_rows(0);
    if (!any) return;
    int kp = page(t + stride + 8 * (this->r16 >> 2)), vp = page(t + stride + 8 * this->g);
    for (; t + stride < end; t += stride) step<true>(t, stride, &kp, &vp);
    step<false>(t, stride, &kp, &vp);
  }
};

template <int D, bool Q8>
__global__ __launch_bounds__(kRowsWaves * 64) void paged_rows_kernel(PagedParams S) {
  using R = PagedRows<D, 1, Q8>;
  extern __shared__ __attribute__((aligned(16))) char s_join[];
  const int item = blockIdx.x / S.cache.heads;
  const PagedItem I = S.plan.items()[item];
  if (item >= S.plan.words[0]) return;
  PagedWave<D, Q8> W(S, I, blockIdx.x - item * S.cache.heads);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), t = I.begin + wave * R::kStep, stride = kRowsWaves * R::kStep;
  W.run(t, I.end, stride);
  W.add_odd_values(t, I.end, stride, R::kStep, 0);
  W.sum_lanes();
  // The upper half of the waves hands over to the lower (where it has anything).
  const int steps = (I.end - I.begin + R::kStep - 1) / R::kStep;
#pragma unroll
  for (int half = kRowsWaves / 2; half > 0; half /= 2) {
    if (half >= steps) continue;
    __syncthreads();
    if (wave >= half && wave < 2 * half) W.hand_over(s_join + (wave - half) * R::kHandBytes);
    __syncthreads();
    if (wave < half) W.take_over(s_join + wave * R::kHandBytes);
  }
  if (wave == 0) W.write(0);
}

constexpr int kJoinThreads = 256;

// The splits of each row and head joined; zeros for rows without a request. kLanes lanes of 4 dimensions to a split, up to 8 splits
// of each loaded together.
template <int D>
__global__ __launch_bounds__(kJoinThreads) void paged_join_kernel(PagedParams S, int64_t m0) {
  constexpr int kLanes = D <= 64 ? 16 : D <= 128 ? 32 : 64, kSlices = kJoinThreads / kLanes;
  __shared__ f32x4 s_o[kSlices][kLanes];
  __shared__ float s_m[kSlices], s_l[kSlices];
  const int64_t row = m0 + blockIdx.y, heads_q = gridDim.x;
  const int hq = blockIdx.x, c = threadIdx.x % kLanes, slice = threadIdx.x / kLanes;
  const int r = S.request[row];
  uint16_t* out = S.out + (row * heads_q + hq) * D + c * 4;
  u32x2 gate = {0u, 0u};  // (loaded here: nothing has to wait for it at the end)
  if (S.gate.x && c * 4 < D) gate = *reinterpret_cast<const u32x2*>(S.gate.x + row * S.gate.row + (int64_t)hq * S.gate.head + c * 4);
  if (r < 0) {
    if (slice == 0 && c * 4 < D) *reinterpret_cast<u32x2*>(out) = u32x2{0u, 0u};
    return;
  }
  const PagedRequest Q = S.plan.requests()[r];
  if (Q.splits <= 1) return;
  const int64_t part = ((int64_t)Q.part + (row - Q.first)) * heads_q + hq, stride = (int64_t)Q.rows * heads_q;
  float m = -__builtin_inff(), l = 0.0f;
  f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
  const auto gather = [&](auto ahead) __attribute__((always_inline)) {
    constexpr int kAhead = decltype(ahead)::value;
    for (int s0 = slice; s0 < Q.splits; s0 += kSlices * kAhead) {
      float m2[kAhead], l2[kAhead];
      f32x4 o2[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        // (Past the last: the first again, with nothing in it.)
        const bool here = s0 + j * kSlices < Q.splits;
        const int64_t at = part + (here ? s0 + j * kSlices : s0) * stride;
        m2[j] = here ? S.part_ml[at * 2] : -__builtin_inff();
        l2[j] = S.part_ml[at * 2 + 1];
        o2[j] = *reinterpret_cast<const f32x4*>(S.part + at * D + (c * 4 < D ? c * 4 : 0));
      }
      float top = m;
#pragma unroll
      for (int j = 0; j < kAhead; ++j) top = fmaxf(top, m2[j]);
      const float f = m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m - top);
      m = top;
      l *= f;
      o *= f;
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        if (m2[j] == -__builtin_inff()) continue;
        const float f2 = __builtin_amdgcn_exp2f(m2[j] - top);
        l += l2[j] * f2;
        o += o2[j] * f2;
      }
    }
  };
  if (Q.splits <= 2 * kSlices) gather(std::integral_constant<int, 2>{});
  else if (Q.splits <= 4 * kSlices) gather(std::integral_constant<int, 4>{});
  else gather(std::integral_constant<int, 8>{});
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
  o *= paged_empty(S.ancestors, row, Q.length, Q.rows) ? 0.0f : 1.0f / l;
  *reinterpret_cast<u32x2*>(out) = gated_bf16(o, S.gate.x != nullptr, gate);
}

template <int D, bool Q8>
hipError_t launch_rows(const PagedParams& p, hipStream_t stream) {
  constexpr size_t kLds = (size_t)(kRowsWaves / 2) * PagedRows<D, 1, Q8>::kHandBytes;
  static LdsAllowance allowance;
  if (kLds > 64 * 1024)
    if (hipError_t e = allowance.allow(reinterpret_cast<const void*>(&paged_rows_kernel<D, Q8>), kLds)) return e;
  hipLaunchKernelGGL((paged_rows_kernel<D, Q8>), dim3((unsigned)p.items * p.cache.heads), dim3(kRowsWaves * 64), kLds, stream, p);
  return hipGetLastError();
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
  // A workgroup fills a CU (nearly: its registers or LDS). Many requests of different lengths are spread better in two rounds than
  // in one by the rows kernel (64 of 2000 to 16000 tokens: 416 us for one of 443), which joins no more for it; few are cut for
  // one round (one of 200000 tokens: 141 us in all, 147 cut for two), and those of the tile kernel always (64 nodes over 32000 tokens:
  // 58 us, 66).
  const int64_t round = (cus + kv_heads - 1) / kv_heads;
  return {G, round, max_rows * G > 16 ? round : (2 * cus + kv_heads - 1) / kv_heads};
}

int64_t paged_partial_rows(const PagedShape& s, int64_t R, int64_t max_rows) {
  // A request of n row blocks and L tokens that is cut has more than `chunk` tokens, so fewer than 2 L / chunk splits; chunk is at
  // least the sum of all n L over s.splits. So the blocks of all splits of such requests are below 2 s.splits.
  return std::min<int64_t>(2 * kPagedRows * s.splits, (s.splits + R) * max_rows * s.G);
}

static hipError_t launch_paged_rows(const PagedParams& p, int D, bool q8, hipStream_t stream) {
  switch (D) {
    case 64: return q8 ? launch_rows<64, true>(p, stream) : launch_rows<64, false>(p, stream);
    case 96: return launch_rows<96, false>(p, stream);
    case 128: return q8 ? launch_rows<128, true>(p, stream) : launch_rows<128, false>(p, stream);
    case 192: return launch_rows<192, true>(p, stream);
    default: return launch_rows<256, true>(p, stream);
  }
}

hipError_t launch_paged_attention(const PagedParams& p, int64_t M, int D, bool q8, hipStream_t stream) {
  const int64_t rows = (int64_t)p.max_rows * p.G;
  if (p.plan.R > 0 && rows > 0) {
    // bf16 heads of 192 and more take the tile kernel from the first row on: their step is more than 8 waves' registers hold, while one
    // wave that multiplies keeps up with the loads of 8 into LDS (one request of 2000 tokens, 6 heads of 256 to a key head: 6.3 us, 7.6
    // with waves of their own; 16 of up to 8000: 63, 65). Smaller heads and codes are fewer bytes beside as much work for that wave
    // (64 of up to 16000, 4 of 128: 434 us, 428; 16 of up to 8000, one of 64: 60, 56; 8 bits, 16 of up to 40000, 6 of 256: 210, 140).
    const bool tile = rows > 16 || (D > 128 && !q8);
    const hipError_t e = tile ? launch_paged_tile(p, D, q8, stream) : launch_paged_rows(p, D, q8, stream);
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
