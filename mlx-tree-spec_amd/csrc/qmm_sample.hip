// The next token of each row from bf16 logits and a random number: temperature, top-k, top-p and min-p
// (include/qmm_requests.h).
//
// A bf16 logit has fewer than 2^16 values, and equal logits have equal weights: the order of falling logits is a
// histogram over the values, and top-k, top-p and the cumulative mass are sums over it. So nothing is sorted, and
// exp is taken once per value that occurs, in fp64 (a mass next to a border decides a token). The token is the
// j-th occurrence of one value, found by a second pass over the row.
//
// One workgroup per row: the histogram lies in LDS, one half of the values (positive, then negative) at a time,
// and the values that occur go to a list in the workspace, in falling order.
#include "qmm4_common.h"
#include "qmm4_lds.h"
#include "qmm_requests_kernels.h"

namespace qmm4 {

namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kBins = 32768;             // values of one half
constexpr int kNegative = 0x7f81;        // rank of the largest negative value
constexpr int kValues = 0xff00;          // ranks 0 (+infinity) .. 0xfeff (the lowest finite value)

// Rank of a bf16 value in falling order (0: +infinity, -0 equal to +0), or -1 for -infinity and NaN.
__device__ __forceinline__ int rank_of(uint32_t b) {
  const int mag = (int)(b & 0x7FFFu);
  if (mag > 0x7F80) return -1;
  if (!(b & 0x8000u) || mag == 0) return 0x7F80 - mag;
  return mag == 0x7F80 ? -1 : 0x7F80 + mag;
}
__device__ __forceinline__ double value_of(int rank) {
  const uint32_t b = rank <= 0x7F80 ? 0x7F80 - rank : 0x8000 | (rank - 0x7F80);
  return (double)bf16_to_f32(b);
}

struct Entry {
  uint32_t rank, count;
};

// Exclusive prefix and total of v over the workgroup. s: kWaves + 1 values of LDS, free for use again after the
// next barrier.
template <class T>
__device__ __forceinline__ T block_prefix(T v, T* s, T* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  T inc = v;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const T o = __shfl_up(inc, off);
    if (lane >= off) inc += o;
  }
  __syncthreads();
  if (lane == 63) s[wave] = inc;
  __syncthreads();
  T before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    if (i == wave) before = all;
    all += s[i];
  }
  *total = all;
  return before + (inc - v);
}

__global__ __launch_bounds__(kThreads) void sample_kernel(SampleParams S, Entry* __restrict__ lists) {
  extern __shared__ uint32_t hist[];  // kBins
  __shared__ double s_d[kWaves];
  __shared__ uint32_t s_u[kWaves];
  __shared__ uint32_t s_rank, s_index;
  __shared__ int s_entry;
  __shared__ double s_logprob;
  const int tid = threadIdx.x, lane = tid & 63;
  const int64_t m = blockIdx.x;
  const uint16_t* row = S.logits + m * S.row_stride;
  Entry* list = lists + m * kValues;

  // The values that occur, in falling order, with their counts.
  uint32_t entries = 0;
  for (int half = 0; half < 2; ++half) {
    const int base = half ? kNegative : 0, size = half ? kValues - kNegative : kNegative;
    for (int i = tid; i < kBins; i += kThreads) hist[i] = 0;
    __syncthreads();
    for (int i = tid; i < S.V; i += kThreads) {
      const int r = rank_of(row[i]);
      if (r >= base && r < base + size) atomicAdd(&hist[r - base], 1u);
    }
    __syncthreads();
    // Each thread lists 32 neighbouring bins.
    uint32_t here = 0, total;
    for (int i = 0; i < kBins / kThreads; ++i) here += hist[tid * (kBins / kThreads) + i] != 0;
    uint32_t at = entries + block_prefix(here, s_u, &total);
    for (int i = 0; i < kBins / kThreads; ++i) {
      const int bin = tid * (kBins / kThreads) + i;
      if (hist[bin] != 0) list[at++] = Entry{(uint32_t)(base + bin), hist[bin]};
    }
    entries += total;
    __syncthreads();
  }
  if (entries == 0) {
    if (tid == 0) {
      S.tokens[m] = -1;
      S.logprobs[m] = -__builtin_inff();
    }
    return;
  }

  const float temp = S.temperature[m], top_p = S.top_p[m], min_p = S.min_p[m];
  const int32_t top_k = S.top_k[m];
  const double largest = value_of((int)list[0].rank);
  auto weight = [&](const Entry& e) {  // (the largest value itself has 1, also where it is infinite)
    return e.rank == list[0].rank ? 1.0 : exp((value_of((int)e.rank) - largest) / (double)temp);
  };
  if (tid == 0) {
    s_entry = 0;
    s_rank = list[0].rank;
    s_index = 0;
    s_logprob = 0.0;
  }
  if (temp > 0.0f) {
    // Entries of this thread: a run of neighbours. Each pass recomputes their weights.
    const uint32_t per = (entries + kThreads - 1) / kThreads;
    const uint32_t i0 = min(entries, tid * per), i1 = min(entries, i0 + per);
    uint32_t count = 0, all_count;
    for (uint32_t i = i0; i < i1; ++i) count += list[i].count;
    const uint32_t before_count = block_prefix(count, s_u, &all_count);
    const uint32_t limit = top_k > 0 ? (uint32_t)top_k : 0xFFFFFFFFu;
    auto in_top_k = [&](uint32_t i, uint32_t before) { return before >= limit ? 0u : min(list[i].count, limit - before); };
    double mass = 0.0, total;
    uint32_t b = before_count;
    for (uint32_t i = i0; i < i1; ++i) {
      mass += in_top_k(i, b) * weight(list[i]);
      b += list[i].count;
    }
    const double before_mass = block_prefix(mass, s_d, &total);
    // Kept of an entry: those with the mass before them below top_p * total, and a weight of at least min_p.
    const double bound = (double)top_p * total;
    auto kept = [&](uint32_t i, uint32_t before, double mass_before, double w) {
      uint32_t n = in_top_k(i, before);
      if (top_p < 1.0f) {
        const double fit = ceil((bound - mass_before) / w);
        n = fit <= 0.0 ? 0u : fit < (double)n ? (uint32_t)fit : n;
      }
      if (w < (double)min_p) n = 0;
      return i == 0 ? max(n, 1u) : n;
    };
    double kept_mass = 0.0, all_kept, mb = before_mass;
    b = before_count;
    for (uint32_t i = i0; i < i1; ++i) {
      const double w = weight(list[i]);
      kept_mass += kept(i, b, mb, w) * w;
      mb += in_top_k(i, b) * w;
      b += list[i].count;
    }
    double before_kept = block_prefix(kept_mass, s_d, &all_kept);
    const float u = S.uniform[m];
    const double target = (double)(u > 0.0f ? u : 0.0f) * all_kept;
    // The entry in which the cumulative mass passes the target; where rounding leaves none, the last kept one.
    int hit = -1;
    uint32_t hit_index = 0;
    double hit_weight = 1.0;
    b = before_count;
    mb = before_mass;
    for (uint32_t i = i0; i < i1; ++i) {
      const double w = weight(list[i]);
      const uint32_t n = kept(i, b, mb, w);
      if (n > 0 && w > 0.0 && before_kept <= target) {
        const double j = floor((target - before_kept) / w);
        hit = (int)i;
        hit_index = j < (double)(n - 1) ? (uint32_t)j : n - 1;
        hit_weight = w;
      }
      before_kept += n * w;
      mb += in_top_k(i, b) * w;
      b += list[i].count;
    }
    __syncthreads();
    if (hit >= 0) atomicMax(&s_entry, hit);
    __syncthreads();
    if (hit >= 0 && hit == s_entry) {
      s_rank = list[hit].rank;
      s_index = hit_index;
      s_logprob = log(hit_weight / all_kept);
    }
  }
  __syncthreads();

  // The s_index-th occurrence (from 0) of the value, by index: kThreads logits at a time.
  const int rank = (int)s_rank;
  uint32_t left = s_index;
  for (int i0 = 0; i0 < S.V; i0 += kThreads) {
    const int i = i0 + tid;
    const bool is = i < S.V && rank_of(row[i]) == rank;
    const unsigned long long votes = __ballot(is);
    __syncthreads();
    if (lane == 0) s_u[tid >> 6] = __popcll(votes);
    __syncthreads();
    uint32_t before = 0, all = 0;
    for (int w = 0; w < kWaves; ++w) {
      if (w == (tid >> 6)) before = all;
      all += s_u[w];
    }
    before += __popcll(votes & ((1ull << lane) - 1));
    if (is && before == left) {
      S.tokens[m] = i;
      S.logprobs[m] = (float)s_logprob;
    }
    if (left < all) break;
    left -= all;
  }
}

LdsAllowance g_allowance;

}  // namespace

int64_t sample_workspace(int64_t M, int64_t V) {
  (void)V;
  return M > 0 ? M * kValues * (int64_t)sizeof(Entry) : 0;
}

hipError_t launch_sample(const SampleParams& p, int64_t M, void* workspace, hipStream_t stream) {
  if (M <= 0) return hipSuccess;
  constexpr size_t kLds = kBins * sizeof(uint32_t);
  hipError_t e = g_allowance.allow(reinterpret_cast<const void*>(&sample_kernel), kLds);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(sample_kernel, dim3((unsigned)M), dim3(kThreads), kLds, stream, p, static_cast<Entry*>(workspace));
  return hipGetLastError();
}

}  // namespace qmm4
