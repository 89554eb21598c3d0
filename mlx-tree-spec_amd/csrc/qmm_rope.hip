// The RMS norms of query and key heads and their rotation at each row's position, in one pass
// (include/qmm_requests.h). Per head x of D values, P frequencies:
//   n = x * inv * w,  inv = 1 / sqrt(sum(x^2) / D + eps);  angle_i = position * inv_freq[i]
//   halves:       (n[i], n[i + P])      -> (n[i] cos - n[i + P] sin, n[i + P] cos + n[i] sin)
//   interleaved:  (n[2i], n[2i + 1])    -> the same
// fp32, one rounding to bf16 at the end. An angle at position 10^6 is off by 0.06 in fp32: it is taken in
// turns in fp64, reduced there to half a turn either side of zero, and only then made fp32.
//
// A head takes G lanes, 16 bytes (8 values) each, G the power of two from D / 8 up, so that its sum stays within
// the lanes of one wave. Each workgroup's heads are of one row: its P sines and cosines are computed once, into
// LDS.
#include "qmm4_common.h"
#include "qmm_requests_kernels.h"

namespace qmm4 {

namespace {

constexpr int kThreads = 256;
constexpr int kMaxP = 256;

enum { kHalves, kHalvesUnaligned, kInterleaved };

template <int MODE>
__global__ __launch_bounds__(kThreads) void qk_norm_rope_kernel(RopeParams S, int G) {
  __shared__ float s_cos[kMaxP], s_sin[kMaxP];
  const int tid = threadIdx.x;
  const int64_t m = blockIdx.x;
  const int c = tid & (G - 1);
  int h = blockIdx.y * (kThreads / G) + tid / G;
  const bool live = h < S.q.heads + S.k.heads && c < S.D / 8;
  const bool is_q = h < S.q.heads;
  h = is_q ? h : h - S.q.heads;
  const RopeHeads& H = is_q ? S.q : S.k;
  const uint16_t* x = H.x + m * H.row + (int64_t)h * H.head;
  u32x4 xv = {0u, 0u, 0u, 0u}, wv = xv;
  if (live) {
    xv = *reinterpret_cast<const u32x4*>(x + c * 8);
    wv = *reinterpret_cast<const u32x4*>(H.weight + c * 8);
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
  float n[8], ss = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    n[e] = bf16_to_f32(e & 1 ? xv[e / 2] >> 16 : xv[e / 2] & 0xFFFFu);
    ss = __builtin_fmaf(n[e], n[e], ss);
  }
  for (int off = G / 2; off > 0; off >>= 1) ss += __shfl_xor(ss, off);
  const float inv = norm_inv(ss, S.D, S.eps);
#pragma unroll
  for (int e = 0; e < 8; ++e) n[e] *= inv * bf16_to_f32(e & 1 ? wv[e / 2] >> 16 : wv[e / 2] & 0xFFFFu);
  __syncthreads();

  float o[8];
  if constexpr (MODE == kInterleaved) {
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const int i = c * 4 + e / 2;
      const float cs = i < S.P ? s_cos[i] : 1.0f, sn = i < S.P ? s_sin[i] : 0.0f;
      o[e] = n[e] * cs - n[e + 1] * sn;
      o[e + 1] = n[e + 1] * cs + n[e] * sn;
    }
  } else if constexpr (MODE == kHalves) {  // P % 8 == 0: a chunk's partners are one other chunk
    const int pc = S.P / 8;
    const bool lo = c < pc, hi = !lo && c < 2 * pc;
    const int partner = lo ? c + pc : hi ? c - pc : c;
    const int lane = (tid & 63) - c + partner;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float other = __shfl(n[e], lane);
      const int i = (lo ? c : c - pc) * 8 + e;
      o[e] = lo ? n[e] * s_cos[i] - other * s_sin[i] : hi ? n[e] * s_cos[i] + other * s_sin[i] : n[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int d = c * 8 + e;
      o[e] = n[e];
      if (live && d < 2 * S.P) {
        const int i = d < S.P ? d : d - S.P, p = d < S.P ? d + S.P : d - S.P;
        const float other = bf16_to_f32(x[p]) * (inv * bf16_to_f32(H.weight[p]));
        o[e] = d < S.P ? n[e] * s_cos[i] - other * s_sin[i] : n[e] * s_cos[i] + other * s_sin[i];
      }
    }
  }
  if (live) {
    u32x4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = pack_bf16x2(o[2 * e], o[2 * e + 1]);
    *reinterpret_cast<u32x4*>(H.out + (m * H.heads + h) * S.D + c * 8) = v;
  }
}

}  // namespace

hipError_t launch_qk_norm_rope(const RopeParams& p, int64_t M, bool interleaved, hipStream_t stream) {
  const int heads = p.q.heads + p.k.heads;
  if (M <= 0 || heads <= 0) return hipSuccess;
  int G = 1;
  while (G * 8 < p.D) G *= 2;
  const int per = kThreads / G;
  const dim3 grid((unsigned)M, (unsigned)((heads + per - 1) / per));
  if (interleaved) hipLaunchKernelGGL(qk_norm_rope_kernel<kInterleaved>, grid, dim3(kThreads), 0, stream, p, G);
  else if (p.P % 8 == 0) hipLaunchKernelGGL(qk_norm_rope_kernel<kHalves>, grid, dim3(kThreads), 0, stream, p, G);
  else hipLaunchKernelGGL(qk_norm_rope_kernel<kHalvesUnaligned>, grid, dim3(kThreads), 0, stream, p, G);
  return hipGetLastError();
}

}  // namespace qmm4
