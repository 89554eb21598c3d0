// The next token of each row from bf16 logits and a random number: temperature, top-k, top-p and min-p
// (include/qmm_requests.h).
//
// A bf16 logit has fewer than 2^16 values, and equal logits have equal weights: the order of falling logits is a
// histogram over the values, and top-k, top-p and the cumulative mass are prefix sums over it. So nothing is
// sorted, and exp is taken once per value that occurs, in fp64: a mass next to a border decides a token. The token
// is the j-th occurrence of one value, found by looking at the logits again.
//
// Two kernels where V is too large for one workgroup per row (its counts would not fit 16 bits, and 152k logits
// take one CU about 10 us of LDS atomics):
//   count   one workgroup per slice of a row: the slice's histogram in LDS (16-bit counts, 128 KB), written out as
//           a list of (value, count) in falling order;
//   pick    one workgroup per row: the slices' lists added into one histogram (32-bit counts) over the range of
//           values that occur, then the sums over it; the slice that holds the occurrence is found in the lists
//           again, and only that slice is read.
// Up to 65535 logits one pick kernel counts its row itself. The sums go over blocks of the histogram, one per wave
// and turn (neighbouring blocks on different waves: the values that occur lie close together): a block's count
// and masses, a prefix over the blocks, then only the two blocks with the borders value by value.
#include "qmm4_common.h"
#include "qmm4_lds.h"
#include "qmm_requests_kernels.h"

namespace qmm4 {

namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kValues = 0xff00;    // ranks 0 (+infinity) .. 0xfeff (the lowest finite value)
constexpr int kMaxSlice = 32768;   // logits per slice: its counts fit 16 bits
constexpr int kMinSlice = 4096;
constexpr int kMaxSlices = 512;
constexpr int kMaxBatch = 256;     // rows per launch: bounds the workspace

// Rank of a bf16 value in falling order (0: +infinity, -0 equal to +0), or -1 for -infinity and NaN.
__device__ __forceinline__ int rank_of(uint32_t b) {
  const int mag = (int)(b & 0x7FFFu);
  const int r = (b & 0x8000u) && mag != 0 ? 0x7F80 + mag : 0x7F80 - mag;
  return mag > 0x7F80 || b == 0xFF80u ? -1 : r;
}
__device__ __forceinline__ double value_of(int rank) {
  return (double)bf16_to_f32(rank <= 0x7F80 ? 0x7F80 - rank : 0x8000 | (rank - 0x7F80));
}

// Logits [begin, end) of a row in groups of 8 within 16-byte lines: group 0 up to the first line's start, the last
// one up to the end (single loads), whole lines between. Places outside hold -infinity.
struct Groups {
  const uint16_t* row;
  int begin, end, line0, count;
  __device__ Groups(const uint16_t* r, int b, int e) : row(r), begin(b), end(e) {
    const int past = (int)((reinterpret_cast<uintptr_t>(r + b) >> 1) & 7);
    line0 = b + (past ? 8 - past : 0);
    count = e > line0 ? 1 + (e - line0 + 7) / 8 : 1;
  }
  __device__ int first(int g) const { return line0 + (g - 1) * 8; }  // index of the group's place 0
  __device__ u32x4 load(int g) const {
    const int i0 = first(g);
    if (g > 0 && i0 + 8 <= end) return *reinterpret_cast<const u32x4*>(row + i0);
    u32x4 v;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int i = i0 + e;
      const uint32_t b = i >= begin && i < end ? row[i] : 0xFF80u;
      if (e & 1) v[e / 2] |= b << 16;
      else v[e / 2] = b;
    }
    return v;
  }
};
__device__ __forceinline__ uint32_t place(u32x4 v, int e) { return e & 1 ? v[e / 2] >> 16 : v[e / 2] & 0xFFFFu; }

// Inclusive prefix over the 64 lanes.
template <class T>
__device__ __forceinline__ T wave_prefix(T v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const T o = __shfl_up(v, off);
    if (lane >= off) v += o;
  }
  return v;
}
template <class T>
__device__ __forceinline__ T wave_sum(T v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
  return v;
}
__device__ __forceinline__ int wave_min(int v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = min(v, __shfl_xor(v, off));
  return v;
}
__device__ __forceinline__ int wave_max(int v) { return -wave_min(-v); }

// 16-bit counts of the logits in groups, two to a word; returns the smallest rank this thread saw.
__device__ __forceinline__ int count_groups(const Groups& G, uint32_t* hist) {
  int lowest = kValues;
  constexpr int kBatch = 4;
  for (int g0 = threadIdx.x; g0 < G.count; g0 += kBatch * kThreads) {
    u32x4 v[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int g = g0 + i * kThreads;
      v[i] = g < G.count ? G.load(g) : u32x4{0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u};
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int r = rank_of(place(v[i], e));
        if (r >= 0) {
          atomicAdd(&hist[r >> 1], r & 1 ? 0x10000u : 1u);
          lowest = min(lowest, r);
        }
      }
    }
  }
  return lowest;
}

template <int BYTES>
__device__ __forceinline__ void zero_lds(uint32_t* p) {
  for (int i = threadIdx.x; i < BYTES / 16; i += kThreads) reinterpret_cast<u32x4*>(p)[i] = u32x4{0u, 0u, 0u, 0u};
}

// Where a batch's lists lie: n [rows][slices], entries [rows][slices][slice], an entry rank << 16 | count (a slice's
// list padded to a multiple of 4 with count 0).
struct Lists {
  uint32_t* n;
  uint32_t* entries;
  int slice, slices;
  __device__ uint32_t* list(int64_t m, int s) const { return entries + (m * slices + s) * (int64_t)slice; }
};

constexpr int kBytes16 = 65536 * 2;

__global__ __launch_bounds__(kThreads) void sample_count_kernel(SampleParams S, Lists L) {
  extern __shared__ uint32_t hist[];
  __shared__ uint32_t s_n[kWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t m = blockIdx.y;
  const int begin = blockIdx.x * L.slice, end = min(S.V, begin + L.slice);
  zero_lds<kBytes16>(hist);
  __syncthreads();
  count_groups(Groups(S.logits + m * S.row_stride, begin, end), hist);
  __syncthreads();
  // Each wave lists 4096 neighbouring values, 8 to a lane and turn.
  constexpr int kTurns = 8;
  const u32x4* h = reinterpret_cast<const u32x4*>(hist) + wave * (kTurns * 64);
  uint32_t mine = 0;
  for (int t = 0; t < kTurns; ++t) {
    const u32x4 v = h[t * 64 + lane];
#pragma unroll
    for (int e = 0; e < 8; ++e) mine += place(v, e) != 0;
  }
  mine = wave_sum(mine);
  if (lane == 0) s_n[wave] = mine;
  __syncthreads();
  uint32_t at = 0, total = 0;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    if (i == wave) at = total;
    total += s_n[i];
  }
  uint32_t* list = L.list(m, blockIdx.x);
  for (int t = 0; t < kTurns; ++t) {
    const u32x4 v = h[t * 64 + lane];
    uint32_t c = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) c += place(v, e) != 0;
    if (__ballot(c != 0) == 0) continue;
    const uint32_t inc = wave_prefix(c);
    uint32_t o = at + inc - c;
    const uint32_t rank = (uint32_t)((wave * kTurns + t) * 512 + lane * 8);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t n = place(v, e);
      if (n != 0) list[o++] = (rank + e) << 16 | n;
    }
    at += __shfl(inc, 63);
  }
  if (tid == 0) L.n[m * L.slices + blockIdx.x] = total;
  if (tid < 4 && (total & 3) != 0 && tid >= (int)(total & 3)) list[(total & ~3u) + tid] = 0;
}

// One row. MERGE: from the slices' lists, else from the row itself.
template <bool MERGE>
__global__ __launch_bounds__(kThreads) void sample_pick_kernel(SampleParams S, Lists L) {
  constexpr int kPerLane = MERGE ? 4 : 8;        // values of a block to a lane (16 bytes of the histogram)
  constexpr int kBlock = 64 * kPerLane;
  constexpr int kTurns = MERGE ? 9 : 8;          // blocks of each wave
  constexpr int kBlocks = kTurns * kWaves;
  constexpr int kSpan = kBlocks * kBlock;        // values of one histogram: 36864, or all 65536
  constexpr int kParts = MERGE ? 2 : 1;          // histograms that cover the values
  constexpr int kPerScan = (kParts * kBlocks + 63) / 64;
  extern __shared__ uint32_t hist[];
  __shared__ uint32_t s_count[kPerScan * 64], s_before[kPerScan * 64];
  __shared__ double s_mass[kPerScan * 64], s_kept[kPerScan * 64];
  __shared__ int s_lo[kWaves], s_hi[kWaves];
  __shared__ uint32_t s_u[kWaves], s_occ[MERGE ? kMaxSlices : 1];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t m = blockIdx.x;
  const uint16_t* row = S.logits + m * S.row_stride;

  float temp = S.temperature[m];
  float top_p = S.top_p[m], min_p = S.min_p[m];
  const float u = S.uniform[m];
  const int32_t top_k = S.top_k[m];
  // Settings that leave the first of the order only: as top-k 1.
  const bool first_only = !(temp > 0.0f) || top_p <= 0.0f || min_p > 1.0f;
  const uint32_t limit = first_only ? 1u : top_k > 0 ? (uint32_t)top_k : 0xFFFFFFFFu;
  if (first_only) {
    temp = top_p = 1.0f;
    min_p = 0.0f;
  }

  for (int i = tid; i < kPerScan * 64; i += kThreads) {
    s_count[i] = 0;
    s_mass[i] = s_kept[i] = 0.0;
  }
  // The histogram of values base + part * kSpan ..; `lowest`: the first value that occurs, parts: histograms
  // that the values which occur span.
  int base = 0, lowest, parts = 1;
  auto build = [&](int part) {
    if constexpr (MERGE) {
      __syncthreads();
      zero_lds<kSpan * 4>(hist);
      __syncthreads();
      const int from = base + part * kSpan;
      for (int s = wave; s < L.slices; s += kWaves) {
        const int n4 = ((int)L.n[m * L.slices + s] + 3) / 4;
        const u32x4* list = reinterpret_cast<const u32x4*>(L.list(m, s));
        constexpr int kBatch = 8;
        for (int i0 = lane; i0 < n4; i0 += kBatch * 64) {
          u32x4 v[kBatch];
#pragma unroll
          for (int i = 0; i < kBatch; ++i) v[i] = i0 + i * 64 < n4 ? list[i0 + i * 64] : u32x4{0u, 0u, 0u, 0u};
#pragma unroll
          for (int i = 0; i < kBatch; ++i) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int r = (int)(v[i][e] >> 16) - from;
              if (r >= 0 && r < kSpan && (v[i][e] & 0xFFFFu) != 0) atomicAdd(&hist[r], v[i][e] & 0xFFFFu);
            }
          }
        }
      }
      __syncthreads();
    }
  };
  int last = -1;
  if constexpr (MERGE) {
    int lo = kValues, hi = -1;
    for (int s = tid; s < L.slices; s += kThreads) {
      const uint32_t n = L.n[m * L.slices + s];
      if (n == 0) continue;
      const uint32_t* list = L.list(m, s);
      lo = min(lo, (int)(list[0] >> 16));
      hi = max(hi, (int)(list[n - 1] >> 16));
    }
    lo = wave_min(lo);
    hi = wave_max(hi);
    if (lane == 0) {
      s_lo[wave] = lo;
      s_hi[wave] = hi;
    }
    __syncthreads();
    lowest = kValues;
    for (int i = 0; i < kWaves; ++i) {
      lowest = min(lowest, s_lo[i]);
      last = max(last, s_hi[i]);
    }
    base = lowest & ~3;
    parts = last - base >= kSpan ? 2 : 1;
  } else {
    zero_lds<kBytes16>(hist);
    __syncthreads();
    const int lo = wave_min(count_groups(Groups(row, 0, S.V), hist));
    if (lane == 0) s_lo[wave] = lo;
    __syncthreads();
    lowest = kValues;
    for (int i = 0; i < kWaves; ++i) lowest = min(lowest, s_lo[i]);
  }
  if (lowest == kValues) {
    if (tid == 0) {
      S.tokens[m] = -1;
      S.logprobs[m] = -__builtin_inff();
    }
    return;
  }

  const double largest = value_of(lowest);
  auto weight = [&](int rank) {  // (the largest value itself has 1, also where it is infinite)
    const double d = value_of(rank) - largest;
    return rank == lowest ? 1.0 : largest == __builtin_inf() ? 0.0 : exp(d / (double)temp);
  };
  auto counts = [&](int b, uint32_t (&c)[kPerLane]) {
    const u32x4 v = reinterpret_cast<const u32x4*>(hist)[(b % kBlocks) * 64 + lane];
#pragma unroll
    for (int e = 0; e < kPerLane; ++e) c[e] = MERGE ? v[e % 4] : place(v, e);
  };
  auto rank_at = [&](int b, int e) { return base + b * kBlock + lane * kPerLane + e; };
  // Counts within top-k, from the count before the lane's values.
  auto within = [&](uint32_t (&c)[kPerLane], uint32_t before) {
#pragma unroll
    for (int e = 0; e < kPerLane; ++e) {
      const uint32_t all = c[e];
      c[e] = before >= limit ? 0u : min(all, limit - before);
      before += all;
    }
  };
  auto lane_before = [&](const uint32_t (&c)[kPerLane]) {
    uint32_t n = 0;
#pragma unroll
    for (int e = 0; e < kPerLane; ++e) n += c[e];
    return wave_prefix(n) - n;
  };

  // Each block's count, then its mass within top-k and the part of it with a weight of at least min_p.
  for (int part = 0; part < parts; ++part) {
    build(part);
    for (int t = 0; t < kTurns; ++t) {
      const int b = part * kBlocks + t * kWaves + wave;
      uint32_t c[kPerLane], n = 0;
      counts(b, c);
#pragma unroll
      for (int e = 0; e < kPerLane; ++e) n += c[e];
      if (__ballot(n != 0) == 0) continue;
      n = wave_sum(n);
      if (lane == 0) s_count[b] = n;
    }
    __syncthreads();
    if (wave == 0) {
      uint32_t v[kPerScan], sum = 0;
#pragma unroll
      for (int i = 0; i < kPerScan; ++i) sum += v[i] = s_count[lane * kPerScan + i];
      uint32_t before = wave_prefix(sum) - sum;
#pragma unroll
      for (int i = 0; i < kPerScan; ++i) {
        s_before[lane * kPerScan + i] = before;
        before += v[i];
      }
    }
    __syncthreads();
    for (int t = 0; t < kTurns; ++t) {
      const int b = part * kBlocks + t * kWaves + wave;
      if (s_count[b] == 0 || s_before[b] >= limit) continue;
      uint32_t c[kPerLane];
      counts(b, c);
      if (s_before[b] + s_count[b] > limit) within(c, s_before[b] + lane_before(c));
      double mass = 0.0, kept = 0.0;
#pragma unroll
      for (int e = 0; e < kPerLane; ++e) {
        if (c[e] == 0) continue;
        const double w = weight(rank_at(b, e)), mw = c[e] * w;
        mass += mw;
        kept += w < (double)min_p ? 0.0 : mw;
      }
      mass = wave_sum(mass);
      kept = wave_sum(kept);
      if (lane == 0) {
        s_mass[b] = mass;
        s_kept[b] = kept;
      }
    }
  }
  __syncthreads();

  // Every wave finds the same: the block in which the mass before reaches top_p of the whole, what is kept, and the
  // block in which the kept mass passes the target.
  double mass_before[kPerScan], kept_before[kPerScan], total, kept_total;
  {
    double a = 0.0, k = 0.0;
#pragma unroll
    for (int i = 0; i < kPerScan; ++i) {
      mass_before[i] = a;
      kept_before[i] = k;
      a += s_mass[lane * kPerScan + i];
      k += s_kept[lane * kPerScan + i];
    }
    const double ia = wave_prefix(a), ik = wave_prefix(k);
    total = __shfl(ia, 63);
    kept_total = __shfl(ik, 63);
#pragma unroll
    for (int i = 0; i < kPerScan; ++i) {
      mass_before[i] += ia - a;
      kept_before[i] += ik - k;
    }
  }
  // One block value by value: counts kept (c), weights, and the kept mass before each of the lane's values.
  const double bound = (double)top_p * total;
  const bool has_bound = top_p < 1.0f;
  int built = parts - 1;
  auto open_block = [&](int b, double mass0, double kept0, uint32_t (&c)[kPerLane], double (&w)[kPerLane],
                        double (&before)[kPerLane]) {
    if (b / kBlocks != built) {
      built = b / kBlocks;
      build(built);
    }
    counts(b, c);
    within(c, s_before[b] + lane_before(c));
    double mass = 0.0;
#pragma unroll
    for (int e = 0; e < kPerLane; ++e) {
      w[e] = c[e] != 0 ? weight(rank_at(b, e)) : 0.0;
      mass += c[e] * w[e];
    }
    double mb = mass0 + (wave_prefix(mass) - mass), kept = 0.0;
#pragma unroll
    for (int e = 0; e < kPerLane; ++e) {
      const double all = c[e] * w[e];
      if (has_bound && c[e] != 0) {  // of a value, those with less than the bound before them
        const double fit = ceil((bound - mb) / w[e]);
        c[e] = fit <= 0.0 ? 0u : fit < (double)c[e] ? (uint32_t)fit : c[e];
      }
      if (w[e] < (double)min_p) c[e] = 0;
      mb += all;
      before[e] = kept;
      kept += c[e] * w[e];
    }
    const double inc = wave_prefix(kept);
#pragma unroll
    for (int e = 0; e < kPerLane; ++e) before[e] += kept0 + (inc - kept);
    return kept0 + __shfl(inc, 63);  // kept up to the block's end
  };
  // The last block with some kept mass for which `before` lies below a limit (or at it).
  auto find = [&](auto&& ok, double* mass0, double* kept0) {
    int b = -1;
#pragma unroll
    for (int i = 0; i < kPerScan; ++i)
      if (s_kept[lane * kPerScan + i] > 0.0 && ok(i)) b = lane * kPerScan + i;
    b = wave_max(b);
    double mm = 0.0, kk = 0.0;
#pragma unroll
    for (int i = 0; i < kPerScan; ++i)
      if (i == b % kPerScan) {
        mm = mass_before[i];
        kk = kept_before[i];
      }
    *mass0 = __shfl(mm, b / kPerScan);
    *kept0 = __shfl(kk, b / kPerScan);
    return b;
  };
  uint32_t c[kPerLane];
  double w[kPerLane], before[kPerLane], mass0, kept0;
  int border = kParts * kBlocks;
  if (has_bound) {
    border = find([&](int i) { return mass_before[i] < bound; }, &mass0, &kept0);
    kept_total = open_block(border, mass0, kept0, c, w, before);
  }
  const double target = (double)(u > 0.0f ? u : 0.0f) * kept_total;
  const int block = find([&](int i) { return lane * kPerScan + i <= border && kept_before[i] <= target; }, &mass0, &kept0);
  if (block != border) open_block(block, mass0, kept0, c, w, before);
  // The last value with some mass that starts at or before the target, and the occurrence of it that passes it.
  int slot = -1;
#pragma unroll
  for (int e = 0; e < kPerLane; ++e)
    if (c[e] != 0 && w[e] > 0.0 && before[e] <= target) slot = e;
  const unsigned long long lanes = __ballot(slot >= 0);
  const int owner = 63 - __builtin_clzll(lanes | 1);
  slot = __shfl(slot, owner);
  uint32_t index = 0;
  double hit_weight = 1.0;
#pragma unroll
  for (int e = 0; e < kPerLane; ++e)
    if (e == slot) {
      const double j = floor((target - before[e]) / w[e]);
      index = j < (double)(c[e] - 1) ? (uint32_t)j : c[e] - 1;
      hit_weight = w[e];
    }
  uint32_t left = __shfl(index, owner);
  hit_weight = __shfl(hit_weight, owner);
  const int rank = base + block * kBlock + owner * kPerLane + max(slot, 0);

  // The slice with the occurrence: the value's count in each list, found by two looks of a wave.
  int begin = 0, end = S.V;
  if constexpr (MERGE) {
    for (int s = wave; s < L.slices; s += kWaves) {
      const int n = (int)L.n[m * L.slices + s];
      const uint32_t* list = L.list(m, s);
      const int step = (n + 63) / 64;
      const unsigned long long le = __ballot(lane * step < n && (int)(list[min(lane * step, max(n - 1, 0))] >> 16) <= rank);
      uint32_t occ = 0;
      if (le != 0) {
        const int from = (63 - __builtin_clzll(le)) * step;
        for (int i = lane; i < step; i += 64) {
          const uint32_t v = from + i < n ? list[from + i] : 0xFFFFFFFFu;
          if ((int)(v >> 16) == rank) occ = v & 0xFFFFu;
        }
      }
      occ = wave_sum(occ);
      if (lane == 0) s_occ[s] = occ;
    }
    __syncthreads();
    int slice = L.slices - 1;
    for (int s = 0; s < L.slices; ++s) {
      if (left < s_occ[s]) {
        slice = s;
        break;
      }
      left -= s_occ[s];
    }
    begin = slice * L.slice;
    end = min(S.V, begin + L.slice);
  }
  const Groups G(row, begin, end);
  for (int g0 = 0; g0 < G.count; g0 += kThreads) {
    const int g = g0 + tid;
    uint32_t hits = 0;
    if (g < G.count) {
      const u32x4 v = G.load(g);
#pragma unroll
      for (int e = 0; e < 8; ++e) hits |= (rank_of(place(v, e)) == rank ? 1u : 0u) << e;
    }
    const uint32_t n = __popc(hits), inc = wave_prefix(n);
    __syncthreads();
    if (lane == 63) s_u[wave] = inc;
    __syncthreads();
    uint32_t ahead = inc - n, all = 0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
      if (i < wave) ahead += s_u[i];
      all += s_u[i];
    }
    if (left >= ahead && left < ahead + n) {
      for (uint32_t skip = left - ahead; skip > 0; --skip) hits &= hits - 1;
      S.tokens[m] = G.first(g) + (__ffs((int)hits) - 1);
      S.logprobs[m] = (float)log(hit_weight / kept_total);
    }
    if (left < all) break;
    left -= all;
  }
}

LdsAllowance g_count, g_pick, g_merge;

constexpr size_t kMergeBytes = 36864 * sizeof(uint32_t);

struct Plan {
  int slice, slices;
  int64_t batch;
};
// Slices of a row: enough workgroups (one per CU: the histogram takes most of its LDS) for the GPU, at least 4096
// logits each.
Plan plan_of(int64_t M, int V, int cus) {
  const int64_t batch = M < kMaxBatch ? M : kMaxBatch;
  int64_t s = cus / batch;
  if (s > V / kMinSlice) s = V / kMinSlice;
  if (s < (V + kMaxSlice - 1) / kMaxSlice) s = (V + kMaxSlice - 1) / kMaxSlice;
  if (s > kMaxSlices) s = kMaxSlices;
  const int slice = (int)(((V + s - 1) / s + 7) / 8 * 8);
  return {slice, (V + slice - 1) / slice, batch};
}
constexpr int kOneKernelV = 65535;  // counts fit 16 bits

}  // namespace

int64_t sample_workspace(int64_t M, int64_t V, int cus) {
  if (M <= 0 || V <= kOneKernelV) return 16;
  const Plan p = plan_of(M, (int)V, cus);
  return ((p.batch * p.slices + 3) / 4 * 4 + p.batch * p.slices * (int64_t)p.slice) * (int64_t)sizeof(uint32_t);
}

hipError_t launch_sample(const SampleParams& p, int64_t M, void* workspace, int cus, hipStream_t stream) {
  hipError_t e;
  auto rows_from = [&](int64_t m0) {
    SampleParams q = p;
    q.logits += m0 * p.row_stride;
    q.uniform += m0;
    auto step = [&](auto& s) {
      if (s.p) s.p += m0;
    };
    step(q.temperature);
    step(q.top_k);
    step(q.top_p);
    step(q.min_p);
    q.tokens += m0;
    q.logprobs += m0;
    return q;
  };
  if (p.V <= kOneKernelV) {
    e = g_pick.allow(reinterpret_cast<const void*>(&sample_pick_kernel<false>), kBytes16);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(sample_pick_kernel<false>, dim3((unsigned)M), dim3(kThreads), kBytes16, stream, p, Lists{});
    return hipGetLastError();
  }
  e = g_count.allow(reinterpret_cast<const void*>(&sample_count_kernel), kBytes16);
  if (e == hipSuccess) e = g_merge.allow(reinterpret_cast<const void*>(&sample_pick_kernel<true>), kMergeBytes);
  if (e != hipSuccess) return e;
  const Plan plan = plan_of(M, p.V, cus);
  uint32_t* ws = static_cast<uint32_t*>(workspace);
  const Lists lists{ws, ws + (plan.batch * plan.slices + 3) / 4 * 4, plan.slice, plan.slices};
  for (int64_t m0 = 0; m0 < M; m0 += plan.batch) {
    const int64_t rows = M - m0 < plan.batch ? M - m0 : plan.batch;
    const SampleParams q = rows_from(m0);
    hipLaunchKernelGGL(sample_count_kernel, dim3(plan.slices, (unsigned)rows), dim3(kThreads), kBytes16, stream, q, lists);
    hipLaunchKernelGGL(sample_pick_kernel<true>, dim3((unsigned)rows), dim3(kThreads), kMergeBytes, stream, q, lists);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace qmm4
