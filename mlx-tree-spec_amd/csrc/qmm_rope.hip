// The RMS norms of query and key heads and their rotation at each row's position, in one pass
// (include/qmm_requests.h). Per head x of D values, P frequencies:
//   n = x * inv * w,  inv = 1 / sqrt(sum(x^2) / D + eps);  angle_i = position * inv_freq[i]
//   halves:       (n[i], n[i + P])      -> (n[i] cos - n[i + P] sin, n[i + P] cos + n[i] sin)
//   interleaved:  (n[2i], n[2i + 1])    -> the same
// fp32, one rounding to bf16 at the end. An angle at position 10^6 is off by 0.06 in fp32: it is taken in
// turns in fp64, reduced there to half a turn either side of zero, and only then made fp32.
//
// A head takes G lanes, 16 bytes (8 values) each, G the power of two from D / 8 up, so that its sum stays within the
// lanes of one wave. A workgroup takes up to 4 x 256 / G heads of one row: its P sines and cosines are computed once,
// into LDS, while all its heads are on their way; a lane keeps its place within the head, so that its weights, sines
// and cosines serve every head. The partner half of a rotated pair is loaded too (from L1: a lane exchange of 8 values
// through LDS costs more).
#include "qmm4_common.h"
#include "qmm_requests_kernels.h"

namespace qmm4 {

namespace {

constexpr int kThreads = 256;
constexpr int kMaxP = 256;
constexpr int kMaxTurns = 4;

enum { kHalves, kHalvesUnaligned, kInterleaved };

// v of another lane of the 16 (DPP control), added.
template <int CTRL>
__device__ __forceinline__ float add_dpp(float v) {
  return v + __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), CTRL, 0xF, 0xF, true));
}
// Sum over groups of G neighbouring lanes, in all of them: pairs, quads, 8 (mirrored within 8) and 16 (mirrored).
__device__ __forceinline__ float group_sum(float v, int G) {
  if (G > 1) v = add_dpp<0xB1>(v);
  if (G > 2) v = add_dpp<0x4E>(v);
  if (G > 4) v = add_dpp<0x141>(v);
  if (G > 8) v = add_dpp<0x140>(v);
  if (G > 16) v += __shfl_xor(v, 16);
  if (G > 32) v += __shfl_xor(v, 32);
  return v;
}

__device__ __forceinline__ float value8(u32x4 v, int e) { return bf16_to_f32(e & 1 ? v[e / 2] >> 16 : v[e / 2] & 0xFFFFu); }

// TURNS: heads of each group of lanes.
template <int MODE, int TURNS>
__global__ __launch_bounds__(kThreads) void qk_norm_rope_kernel(RopeParams S, int64_t m0, int G, bool past_l2) {
  __shared__ __attribute__((aligned(16))) float s_cos[kMaxP], s_sin[kMaxP];
  const int tid = threadIdx.x, per = kThreads / G;
  const int64_t m = m0 + blockIdx.x;
  const int c = tid & (G - 1), h0 = blockIdx.y * (TURNS * per) + tid / G;
  const int heads = S.q.heads + S.k.heads;
  const bool in_head = c < S.D / 8;
  // kHalves (P % 8 == 0): a chunk of 8 is in the first half of the pairs, the second, or past them.
  const int pc = S.P / 8;
  const bool lo = c < pc, hi = !lo && c < 2 * pc, turned = MODE == kHalves && (lo || hi) && in_head;
  const int partner = lo ? c + pc : c - pc;
  u32x4 xv[TURNS], xp[MODE == kHalves ? TURNS : 1];
  const uint16_t* head[TURNS];
#pragma unroll
  for (int t = 0; t < TURNS; ++t) {
    const int h = h0 + t * per;
    const bool is_q = h < S.q.heads;
    const RopeHeads& H = is_q ? S.q : S.k;
    head[t] = H.x + m * H.row + (int64_t)(is_q ? h : h - S.q.heads) * H.head;
    xv[t] = u32x4{0u, 0u, 0u, 0u};
    if (h < heads && in_head) xv[t] = *reinterpret_cast<const u32x4*>(head[t] + c * 8);
    if constexpr (MODE == kHalves) {
      xp[t] = u32x4{0u, 0u, 0u, 0u};
      if (h < heads && turned) xp[t] = *reinterpret_cast<const u32x4*>(head[t] + partner * 8);
    }
  }
  // Weights of this lane's chunk, and of its partner's, for q and k.
  u32x4 wv[2], wp[2];
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const uint16_t* w = s ? S.k.weight : S.q.weight;
    wv[s] = wp[s] = u32x4{0u, 0u, 0u, 0u};
    if (in_head && (s ? S.k.heads : S.q.heads) > 0) {
      wv[s] = *reinterpret_cast<const u32x4*>(w + c * 8);
      if (turned) wp[s] = *reinterpret_cast<const u32x4*>(w + partner * 8);
    }
  }
  const double pos = (double)S.positions[m];
  for (int i = tid; i < S.P; i += kThreads) {
    const double f = S.freq64 ? static_cast<const double*>(S.inv_freq)[i] : (double)static_cast<const float*>(S.inv_freq)[i];
    const double turns = pos * (f * 0.15915494309189535);  // 1 / 2 pi
    float sn, cs;
    sincospif((float)(2.0 * (turns - rint(turns))), &sn, &cs);
    s_cos[i] = cs;
    s_sin[i] = sn;
  }
  __syncthreads();
  // Value e of the chunk turns by cs[e] and, with its partner, by sn[e] (of the sign that its place has).
  float cs[8], sn[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    cs[e] = 1.0f;
    sn[e] = 0.0f;
  }
  if constexpr (MODE == kHalves) {
    if (turned) {
      const int i = (lo ? c : c - pc) * 8;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        cs[e] = s_cos[i + e];
        sn[e] = lo ? -s_sin[i + e] : s_sin[i + e];
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int d = c * 8 + e, i = MODE == kInterleaved ? d / 2 : d < S.P ? d : d - S.P;
      if (d < 2 * S.P) {
        cs[e] = s_cos[i];
        sn[e] = (MODE == kInterleaved ? (e & 1) == 0 : d < S.P) ? -s_sin[i] : s_sin[i];
      }
    }
  }
#pragma unroll
  for (int t = 0; t < TURNS; ++t) {
    const int h = h0 + t * per;
    const bool is_q = h < S.q.heads;
    float n[8], ss = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      n[e] = value8(xv[t], e);
      ss = __builtin_fmaf(n[e], n[e], ss);
    }
    ss = group_sum(ss, G);
    // (An inverse root of one half step more than a rounded one: a fiftieth of the result's own rounding.)
    const float inv = __builtin_amdgcn_rsqf(ss / (float)S.D + S.eps);
    const u32x4 w = is_q ? wv[0] : wv[1];
#pragma unroll
    for (int e = 0; e < 8; ++e) n[e] *= inv * value8(w, e);
    u32x4 o;
    float r[8];
    if constexpr (MODE == kHalves) {
      const u32x4 w2 = is_q ? wp[0] : wp[1];
#pragma unroll
      for (int e = 0; e < 8; ++e) r[e] = n[e] * cs[e] + (value8(xp[t], e) * (inv * value8(w2, e))) * sn[e];
    } else if constexpr (MODE == kInterleaved) {
#pragma unroll
      for (int e = 0; e < 8; ++e) r[e] = n[e] * cs[e] + n[e ^ 1] * sn[e];
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int d = c * 8 + e;
        float other = 0.0f;
        if (h < heads && in_head && d < 2 * S.P) {
          const int p = d < S.P ? d + S.P : d - S.P;
          other = bf16_to_f32(head[t][p]) * (inv * bf16_to_f32((is_q ? S.q.weight : S.k.weight)[p]));
        }
        r[e] = n[e] * cs[e] + other * sn[e];
      }
    }
    if (h < heads && in_head) {
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = pack_bf16x2(r[2 * e], r[2 * e + 1]);
      const RopeHeads& H = is_q ? S.q : S.k;
      u32x4* out = reinterpret_cast<u32x4*>(H.out + (m * H.heads + (is_q ? h : h - S.q.heads)) * S.D + c * 8);
      if (past_l2) __builtin_nontemporal_store(o, out);
      else *out = o;
    }
  }
}

template <int MODE>
void launch_mode(const RopeParams& p, int64_t M, int G, hipStream_t stream) {
  const int heads = p.q.heads + p.k.heads, per = kThreads / G;
  const int groups = (heads + per - 1) / per;  // turns that a row needs in all
  // Several turns to a workgroup (fewer sines) where there are rows enough to fill the GPU: 64 x 40 heads x 128 3.2 us in
  // 3 workgroups a row, 4.0 in one; 4096 rows 18.6 and 16.5.
  const int most = M >= 512 ? kMaxTurns : 1;
  const int blocks = (groups + most - 1) / most, turns = (groups + blocks - 1) / blocks;
  // Results that no L2 (4 MiB each) will hold for their reader do not push the inputs out of it: 4096 x 40 heads x 128
  // 19.5 -> 16.5 us, 1024 x 28 x 256 9.0 -> 7.2, 1500 x 32 x 64 5.2 -> 4.8.
  const bool past_l2 = M * heads * p.D * 2 > 4 << 20;
  constexpr int64_t kRows = 1 << 23;  // (a grid may have 2^32 threads along x)
  for (int64_t m0 = 0; m0 < M; m0 += kRows) {
    const dim3 grid((unsigned)(M - m0 < kRows ? M - m0 : kRows), (unsigned)blocks);
    switch (turns) {
      case 1: hipLaunchKernelGGL((qk_norm_rope_kernel<MODE, 1>), grid, dim3(kThreads), 0, stream, p, m0, G, past_l2); break;
      case 2: hipLaunchKernelGGL((qk_norm_rope_kernel<MODE, 2>), grid, dim3(kThreads), 0, stream, p, m0, G, past_l2); break;
      case 3: hipLaunchKernelGGL((qk_norm_rope_kernel<MODE, 3>), grid, dim3(kThreads), 0, stream, p, m0, G, past_l2); break;
      default: hipLaunchKernelGGL((qk_norm_rope_kernel<MODE, 4>), grid, dim3(kThreads), 0, stream, p, m0, G, past_l2); break;
    }
  }
}

}  // namespace

hipError_t launch_qk_norm_rope(const RopeParams& p, int64_t M, bool interleaved, hipStream_t stream) {
  if (M <= 0 || p.q.heads + p.k.heads <= 0) return hipSuccess;
  int G = 1;
  while (G * 8 < p.D) G *= 2;
  if (interleaved) launch_mode<kInterleaved>(p, M, G, stream);
  else if (p.P % 8 == 0) launch_mode<kHalves>(p, M, G, stream);
  else launch_mode<kHalvesUnaligned>(p, M, G, stream);
  return hipGetLastError();
}

}  // namespace qmm4
