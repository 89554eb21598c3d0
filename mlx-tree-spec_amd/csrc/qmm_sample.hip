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
// Up to 65535 logits one pick kernel counts its row itself.
//
// The sums run over the values that occur, up to 4096 of them (a page) listed in LDS, 4 neighbours to a thread: a
// prefix over the workgroup gives the count before each thread, its counts within top-k, their masses; another the
// mass before it, what top-p and min-p keep of it; a third the kept mass before it, and with it the value that
// passes the target. More values (152k logits of a model have about 3500; past 4096 they lie many octaves apart)
// take their pages in turn, once per sum.
//
// What bounds it: a row's steps follow each other in one workgroup, and its 16 waves get through about 150
// instructions each a microsecond; the steps are kept to few instructions per value and wave.
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

// Rank of a bf16 value in falling order (0: +infinity, -0 equal to +0); outside 0 .. kValues - 1 for -infinity and
// NaN.
__device__ __forceinline__ int rank_of(uint32_t b) {
  const int mag = (int)(b & 0x7FFFu);
  return 0x7F80 + (b & 0x8000u ? mag : -mag);
}
__device__ __forceinline__ double value_of(int rank) {
  return (double)bf16_to_f32(rank <= 0x7F80 ? 0x7F80 - rank : 0x8000 | (rank - 0x7F80));
}

// Logits [begin, end) of a row: whole 16-byte lines of 8 (line g from index first(g)), and up to 7 logits either side
// of them, which `edge` holds for threads 0 .. 15 in index order around the lines. Places outside hold -infinity.
constexpr uint32_t kNone = 0xFF80u;
struct Lines {
  const uint16_t* row;
  int begin, end, line0, count;
  __device__ Lines(const uint16_t* r, int b, int e) : row(r), begin(b), end(e) {
    const int past = (int)((reinterpret_cast<uintptr_t>(r + b) >> 1) & 7);
    line0 = min(e, b + (past ? 8 - past : 0));
    count = (e - line0) / 8;
  }
  __device__ int first(int g) const { return line0 + g * 8; }
  // Lines past the last are loads of the last one, made -infinity: no branch keeps loads apart.
  __device__ u32x4 load(int g) const {
    const u32x4 none = {kNone << 16 | kNone, kNone << 16 | kNone, kNone << 16 | kNone, kNone << 16 | kNone};
    if (count == 0) return none;
    const u32x4 v = *reinterpret_cast<const u32x4*>(row + first(min(g, count - 1)));
    return g < count ? v : none;
  }
  __device__ int edge_index(int t) const { return t < 8 ? begin + t : first(count) + t - 8; }
  __device__ bool has_edge(int t) const { return t < 8 ? begin + t < line0 : t < 16 && first(count) + t - 8 < end; }
  __device__ uint32_t edge(int t) const { return has_edge(t) ? row[edge_index(t)] : kNone; }
};
__device__ __forceinline__ uint32_t place(u32x4 v, int e) { return e & 1 ? v[e / 2] >> 16 : v[e / 2] & 0xFFFFu; }

// v of the lane that the DPP control names, 0 where there is none or its row is masked out.
template <int CTRL, int ROWS, class T>
__device__ __forceinline__ T dpp(T v) {
  if constexpr (sizeof(T) == 8) {
    const u32x2 p = __builtin_bit_cast(u32x2, v);
    return __builtin_bit_cast(T, u32x2{dpp<CTRL, ROWS>(p.x), dpp<CTRL, ROWS>(p.y)});
  } else {
    return (T)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false);
  }
}
template <class T>
__device__ __forceinline__ T lane_value(T v, int lane) {  // lane: the same in all lanes
  if constexpr (sizeof(T) == 8) {
    const u32x2 p = __builtin_bit_cast(u32x2, v);
    return __builtin_bit_cast(T, u32x2{lane_value(p.x, lane), lane_value(p.y, lane)});
  } else {
    return (T)__builtin_amdgcn_readlane((int)v, lane);
  }
}
// Inclusive prefix over the 64 lanes: within rows of 16 by shifts of 1, 2, 4 and 8 lanes, then the last lane of rows
// 0 and 2 to the row behind, and of the first half to the second. (Register moves: the same through LDS permutes
// cost 6 round trips of about 50 ns each, a tenth of the pick kernel.)
template <class T>
__device__ __forceinline__ T wave_prefix(T v) {
  v += dpp<0x111, 0xF>(v);
  v += dpp<0x112, 0xF>(v);
  v += dpp<0x114, 0xF>(v);
  v += dpp<0x118, 0xF>(v);
  v += dpp<0x142, 0xA>(v);
  v += dpp<0x143, 0xC>(v);
  return v;
}
// Over the first 16 lanes (of other lanes: anything).
template <class T>
__device__ __forceinline__ T row_prefix(T v) {
  v += dpp<0x111, 0xF>(v);
  v += dpp<0x112, 0xF>(v);
  v += dpp<0x114, 0xF>(v);
  v += dpp<0x118, 0xF>(v);
  return v;
}
template <class T>
__device__ __forceinline__ T wave_sum(T v) { return lane_value(wave_prefix(v), 63); }
// The largest of values >= -1 over the first 16 lanes, or all.
__device__ __forceinline__ int row_max(int v) {
  v += 1;  // (a DPP without a source lane gives 0)
  v = max(v, dpp<0x111, 0xF>(v));
  v = max(v, dpp<0x112, 0xF>(v));
  v = max(v, dpp<0x114, 0xF>(v));
  v = max(v, dpp<0x118, 0xF>(v));
  return lane_value(v, 15) - 1;
}
__device__ __forceinline__ int wave_max(int v) {
  v += 1;
  v = max(v, dpp<0x111, 0xF>(v));
  v = max(v, dpp<0x112, 0xF>(v));
  v = max(v, dpp<0x114, 0xF>(v));
  v = max(v, dpp<0x118, 0xF>(v));
  v = max(v, dpp<0x142, 0xA>(v));
  v = max(v, dpp<0x143, 0xC>(v));
  return lane_value(v, 63) - 1;
}
// The smallest of values up to kValues.
__device__ __forceinline__ int row_min(int v) { return kValues - row_max(kValues - v); }
__device__ __forceinline__ int wave_min(int v) { return kValues - wave_max(kValues - v); }

// 16-bit counts of the logits, two to a word; returns the smallest rank this thread saw. `held`: the lines loaded
// last (lines threadIdx.x + i kThreads where there are at most kBatch * kThreads of them). `between` runs while the
// first loads are under way.
constexpr int kBatch = 4;
template <class F>
__device__ __forceinline__ int count_lines(const Lines& G, uint32_t* hist, u32x4 (&held)[kBatch], F&& between) {
  int lowest = kValues;
  auto count = [&](uint32_t b) {  // -infinity and NaN go to bins past the values, one for each lane
    int r = rank_of(b);
    r = (uint32_t)r < (uint32_t)kValues ? r : kValues + (int)(threadIdx.x & 63);
    atomicAdd(&hist[r >> 1], r & 1 ? 0x10000u : 1u);
    lowest = min(lowest, r);
  };
  const uint32_t edge = G.edge(threadIdx.x);
  for (int g0 = threadIdx.x, at = 0; at < max(G.count, 1); g0 += kBatch * kThreads, at += kBatch * kThreads) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i) held[i] = G.load(g0 + i * kThreads);
    if (at == 0) {
      __builtin_amdgcn_sched_barrier(0);
      between();
      count(edge);
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (at + i * kThreads >= G.count) break;
#pragma unroll
      for (int e = 0; e < 8; ++e) count(place(held[i], e));
    }
  }
  __syncthreads();
  if (threadIdx.x < 32) hist[kValues / 2 + threadIdx.x] = 0;
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
  extern __shared__ __attribute__((aligned(16))) uint32_t hist[];
  __shared__ uint32_t s_n[kWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t m = blockIdx.y;
  const int begin = blockIdx.x * L.slice, end = min(S.V, begin + L.slice);
  u32x4 held[kBatch];
  count_lines(Lines(S.logits + m * S.row_stride, begin, end), hist, held, [&] {
    zero_lds<kBytes16>(hist);
    __syncthreads();
  });
  __syncthreads();
  // Each wave lists 4096 neighbouring values, 64 words of two at a time: a comparison is a mask of the lanes, and a
  // lane's place in the list the number of values below it.
  constexpr int kLooks = 32;
  const uint32_t* h = hist + wave * (kLooks * 64) + lane;
  uint32_t mine = 0, looks = 0;
#pragma unroll
  for (int t = 0; t < kLooks; ++t) {
    const uint32_t v = h[t * 64];
    const int seen = __popcll(__ballot((v & 0xFFFFu) != 0)) + __popcll(__ballot(v > 0xFFFFu));
    mine += seen;
    looks |= seen != 0 ? 1u << t : 0;
  }
  if (lane == 0) s_n[wave] = mine;
  __syncthreads();
  const uint32_t waves = row_prefix(s_n[lane & 15]), total = lane_value(waves, 15);
  uint32_t at = wave ? lane_value(waves, wave - 1) : 0u;
  uint32_t* list = L.list(m, blockIdx.x);
  for (; looks != 0; looks &= looks - 1) {
    const int t = __ffs((int)looks) - 1;
    const uint32_t v = h[t * 64];
    const unsigned long long lo = __ballot((v & 0xFFFFu) != 0), hi = __ballot(v > 0xFFFFu);
    uint32_t o = __builtin_amdgcn_mbcnt_hi((uint32_t)(lo >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)lo, at));
    o = __builtin_amdgcn_mbcnt_hi((uint32_t)(hi >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)hi, o));
    const uint32_t r = (uint32_t)((wave * kLooks + t) * 64 + lane) * 2;
    if ((v & 0xFFFFu) != 0) list[o++] = r << 16 | (v & 0xFFFFu);
    if (v > 0xFFFFu) list[o] = (r + 1) << 16 | v >> 16;
    at += __popcll(lo) + __popcll(hi);
  }
  if (tid == 0) L.n[m * L.slices + blockIdx.x] = total;
  if (tid < 4 && (total & 3) != 0 && tid >= (int)(total & 3)) list[(total & ~3u) + tid] = 0;
}

// One row. MERGE: from the slices' lists, else from the row itself.
template <bool MERGE>
__global__ __launch_bounds__(kThreads) void sample_pick_kernel(SampleParams S, Lists L) {
  constexpr int kSpan = MERGE ? 36 * kThreads : 65536;  // values of one histogram: +-512 with all between, or all
  constexpr int kPer = 4;                         // listed values of a page to a thread
  constexpr int kPage = kPer * kThreads;
  extern __shared__ __attribute__((aligned(16))) uint32_t hist[];
  __shared__ uint16_t s_page[kPage];
  __shared__ int s_lo[kWaves], s_hi[kWaves];
  __shared__ double s_d[2][kWaves];
  __shared__ uint32_t s_u[kBatch][kWaves], s_n[MERGE ? kMaxSlices : 1], s_occ[MERGE ? kMaxSlices : 1];
  __shared__ uint32_t s_hit[2];
  __shared__ double s_weight;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t m = blockIdx.x;
  const uint16_t* row = S.logits + m * S.row_stride;

  float temp = S.temperature[m], top_p = S.top_p[m], min_p = S.min_p[m];
  const float u = S.uniform[m];
  const int32_t top_k = S.top_k[m];
  // Settings that leave the first of the order only: as top-k 1.
  const bool first_only = !(temp > 0.0f) || top_p <= 0.0f || min_p > 1.0f;
  const uint32_t limit = first_only ? 1u : top_k > 0 ? (uint32_t)top_k : 0xFFFFFFFFu;
  if (first_only) {
    temp = top_p = 1.0f;
    min_p = 0.0f;
  }

  // `lowest`: the first value that occurs. The histogram holds values from `base`; a second one (part 1) those past
  // its end, where there are any.
  int lowest = kValues, base = 0, parts = 1;
  u32x4 held[kBatch];
  if constexpr (MERGE) {
    int lo = kValues, hi = -1;
    for (int s = tid; s < L.slices; s += kThreads) {
      const uint32_t n = L.n[m * L.slices + s];
      s_n[s] = n;
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
    lowest = row_min(s_lo[lane & 15]);
    base = lowest & ~3;
    parts = row_max(s_hi[lane & 15]) - base >= kSpan ? 2 : 1;
  } else {
    const int lo = wave_min(count_lines(Lines(row, 0, S.V), hist, held, [&] {
      zero_lds<kBytes16>(hist);
      __syncthreads();
    }));
    if (lane == 0) s_lo[wave] = lo;
    __syncthreads();
    lowest = row_min(s_lo[lane & 15]);
  }
  if (lowest == kValues) {
    if (tid == 0) {
      S.tokens[m] = -1;
      S.logprobs[m] = -__builtin_inff();
    }
    return;
  }
  const double largest = value_of(lowest), per_temp = 1.0 / (double)temp;

  // Prefix of v over the workgroup's threads, and its total. `slot` alternates between calls.
  auto block_prefix = [&](auto v, auto* slot, auto* total) __attribute__((always_inline)) {
    const auto inc = wave_prefix(v);
    if (lane == 63) slot[wave] = inc;
    __syncthreads();
    const auto waves = row_prefix(slot[lane & 15]);
    *total = lane_value(waves, 15);
    return (wave ? lane_value(waves, wave - 1) : decltype(v)(0)) + (inc - v);
  };

  // Three sums over the pages: the mass within top-k, the part of it that is kept, and up to the target. With one page
  // the threads keep their values from sum to sum.
  double total = 0.0, kept_total = 0.0, target = 0.0;
  int built = MERGE ? -1 : 0;
  bool one_page = true;
  uint32_t c[kPer], n[kPer];
  double w[kPer], mass = 0.0, mass_before = 0.0, kept = 0.0, kept_before = 0.0;
  int rank[kPer], per = 0;
  for (int sum = 0; sum < 3; ++sum) {
    uint32_t count_sum = 0;
    double mass_sum = 0.0, kept_sum = 0.0;
    for (int part = 0; part < parts; ++part) {
      const int from = base + part * kSpan;
      if (MERGE && built != part) {
        __syncthreads();
        zero_lds<kSpan * 4>(hist);
        __syncthreads();
        built = part;
        for (int s = wave; s < L.slices; s += kWaves) {
          const int n4 = ((int)s_n[s] + 3) / 4;
          const u32x4* list = reinterpret_cast<const u32x4*>(L.list(m, s));
          constexpr int kAhead = 8;
          for (int i0 = lane; i0 < n4; i0 += kAhead * 64) {
            u32x4 v[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; ++i) v[i] = list[min(i0 + i * 64, n4 - 1)];
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
#pragma unroll
              for (int e = 0; e < 4; ++e) {  // (what is not for this histogram goes behind it, one word for each lane)
                const int r = (int)(v[i][e] >> 16) - from;
                const bool in = i0 + i * 64 < n4 && (uint32_t)r < (uint32_t)kSpan;
                atomicAdd(&hist[in ? r : kSpan + lane], v[i][e] & 0xFFFFu);
              }
            }
          }
        }
        __syncthreads();
      }
      uint32_t entries = 0;
      for (uint32_t first = 0; first == 0 || first < entries; first += kPage) {
        if (sum == 0 || !one_page) {
          // The page's values: those that occur, the first-th and on. A wave lists kLooks * 64 neighbouring words of the
          // histogram, 64 at a time: a comparison is a mask of the lanes, and a lane's place in the list the number of
          // them below it. (Neighbouring groups of 64 to different waves took two more barriers and 0.4 us.)
          constexpr int kLooks = kSpan / (MERGE ? 1 : 2) / kThreads;
          const uint32_t* h = hist + wave * (kLooks * 64) + lane;
          uint32_t here = 0;
#pragma unroll 9
          for (int t = 0; t < kLooks; ++t) {
            const uint32_t v = h[t * 64];
            if constexpr (MERGE) here += __popcll(__ballot(v != 0));
            else here += __popcll(__ballot((v & 0xFFFFu) != 0)) + __popcll(__ballot(v > 0xFFFFu));
          }
          __syncthreads();  // (the page before is read)
          uint32_t at = block_prefix(lane == 0 ? here : 0u, s_u[0], &entries);
          at = lane_value(at, 0) - first;
          if (sum == 0 && part == 0 && first == 0) one_page = parts == 1 && entries <= kPage;
#pragma unroll 9
          for (int t = 0; t < kLooks; ++t) {
            const uint32_t v = h[t * 64];
            const unsigned long long lo = __ballot(MERGE ? v != 0 : (v & 0xFFFFu) != 0), hi = MERGE ? 0 : __ballot(v > 0xFFFFu);
            if ((lo | hi) == 0) continue;
            uint32_t o = __builtin_amdgcn_mbcnt_hi((uint32_t)(lo >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)lo, at));
            const uint32_t r = (uint32_t)((wave * kLooks + t) * 64 + lane) * (MERGE ? 1 : 2);
            if constexpr (!MERGE)
              o = __builtin_amdgcn_mbcnt_hi((uint32_t)(hi >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)hi, o));
            if ((MERGE ? v != 0 : (v & 0xFFFFu) != 0) && o < (uint32_t)kPage) s_page[o] = (uint16_t)r;
            if constexpr (!MERGE) {
              o += (v & 0xFFFFu) != 0;
              if (v > 0xFFFFu && o < (uint32_t)kPage) s_page[o] = (uint16_t)(r + 1);
            }
            at += __popcll(lo) + __popcll(hi);
          }
          __syncthreads();
          // Counts within top-k and their masses. (Equal weights of neighbours: none of the values is taken twice.)
          const uint32_t in_page = min(entries - first, (uint32_t)kPage);
          per = (int)((in_page + kThreads - 1) / kThreads);
          uint32_t own = 0, page_count, all[kPer];
#pragma unroll
          for (int e = 0; e < kPer; ++e) {
            all[e] = c[e] = n[e] = 0;
            w[e] = 0.0;
            if (e >= per) continue;
            const uint32_t i = tid * per + e;
            const bool is = i < in_page;
            const uint32_t r = is ? s_page[i] : 0u;
            rank[e] = from + (int)r;
            all[e] = !is ? 0u : MERGE ? hist[r] : r & 1 ? hist[r >> 1] >> 16 : hist[r >> 1] & 0xFFFFu;
            own += all[e];
          }
          uint32_t before = count_sum + block_prefix(own, s_u[1], &page_count);
          count_sum += page_count;
          double page_mass;
          mass = 0.0;
#pragma unroll
          for (int e = 0; e < kPer; ++e) {
            if (e >= per) break;
            c[e] = before >= limit ? 0u : min(all[e], limit - before);
            before += all[e];
            // (The largest value itself has 1, also where it is infinite.)
            const double d = value_of(rank[e]) - largest;
            w[e] = rank[e] == lowest ? 1.0 : largest == __builtin_inf() ? 0.0 : exp(d * per_temp);
            if (c[e] == 0) w[e] = 0.0;
            mass += c[e] * w[e];
          }
          mass_before = mass_sum + block_prefix(mass, s_d[0], &page_mass);
          mass_sum += page_mass;
        }
        if (sum == 1 || (sum == 2 && !one_page)) {
          // Kept of a value: those with less mass before them than the bound, and a weight of at least min_p.
          if (top_p < 1.0f || min_p > 0.0f) {
            const double bound = (double)top_p * total;
            double mb = mass_before, page_kept;
            kept = 0.0;
#pragma unroll
            for (int e = 0; e < kPer; ++e) {
              if (e >= per) break;
              const double end = mb + c[e] * w[e];
              n[e] = c[e];
              if (top_p < 1.0f && end > bound) {  // (the division is for one value of all: 4 in each thread took 0.7 us)
                n[e] = 0;
                if (mb < bound) n[e] = min(c[e], (uint32_t)ceil((bound - mb) / w[e]));
              }
              if (w[e] < (double)min_p) n[e] = 0;
              mb = end;
              kept += n[e] * w[e];
            }
            kept_before = kept_sum + block_prefix(kept, s_d[1], &page_kept);
            kept_sum += page_kept;
          } else {
#pragma unroll
            for (int e = 0; e < kPer; ++e) n[e] = c[e];
            kept = mass;
            kept_before = mass_before;
            kept_sum = one_page ? total : mass_sum;
          }
        }
        if (sum == 2) {
          // The last thread with some kept mass that starts at or before the target holds the value that passes it (up
          // to rounding: then its last one).
          const int thread = wave_max(kept > 0.0 && kept_before <= target ? tid : -1);
          if (lane == 0) s_hi[wave] = thread;
          __syncthreads();
          if (tid == row_max(s_hi[lane & 15])) {
            uint32_t hit_n = 1, hit_rank = 0;
            double kb = kept_before, hit_before = 0.0, hit_weight = 1.0;
#pragma unroll
            for (int e = 0; e < kPer; ++e) {
              if (n[e] != 0 && w[e] > 0.0 && kb <= target) {
                hit_n = n[e];
                hit_rank = (uint32_t)rank[e];
                hit_before = kb;
                hit_weight = w[e];
              }
              kb += n[e] * w[e];
            }
            const double j = floor((target - hit_before) / hit_weight);
            s_hit[0] = hit_rank;
            s_hit[1] = j < (double)(hit_n - 1) ? (uint32_t)j : hit_n - 1;
            s_weight = hit_weight;
          }
          __syncthreads();
        }
        if (one_page) break;
      }
    }
    if (sum == 0) total = mass_sum;
    if (sum == 1) {
      kept_total = kept_sum;
      target = (double)(u > 0.0f ? u : 0.0f) * kept_total;
    }
  }
  const int hit = (int)s_hit[0];
  uint32_t left = s_hit[1];
  const double hit_weight = s_weight;

  // The slice with the occurrence: the value's count in each list, found by two looks of a wave.
  int begin = 0, end = S.V;
  if constexpr (MERGE) {
    for (int s = wave; s < L.slices; s += kWaves) {
      const int n = (int)s_n[s];
      const uint32_t* list = L.list(m, s);
      const int step = (n + 63) / 64;
      const unsigned long long le = __ballot(lane * step < n && (int)(list[min(lane * step, max(n - 1, 0))] >> 16) <= hit);
      uint32_t occ = 0;
      if (le != 0) {
        const int from = (63 - __builtin_clzll(le)) * step;
        for (int i = lane; i < step; i += 64) {
          const uint32_t v = from + i < n ? list[from + i] : 0xFFFFFFFFu;
          if ((int)(v >> 16) == hit) occ = v & 0xFFFFu;
        }
      }
      occ = wave_sum(occ);
      if (lane == 0) s_occ[s] = occ;
    }
    __syncthreads();
    int slice = L.slices - 1;
    for (int s0 = 0; s0 < L.slices; s0 += 64) {
      const uint32_t occ = s0 + lane < L.slices ? s_occ[s0 + lane] : 0, inc = wave_prefix(occ);
      const unsigned long long past = __ballot(left < inc);
      if (past != 0) {
        const int at = __ffsll(past) - 1;
        slice = s0 + at;
        left -= lane_value(inc - occ, at);
        break;
      }
      left -= lane_value(inc, 63);
    }
    begin = slice * L.slice;
    end = min(S.V, begin + L.slice);
  }
  auto found = [&](int index) {
    S.tokens[m] = index;
    S.logprobs[m] = (float)log(hit_weight / kept_total);
  };
  // The value's bits; zero has two forms.
  const uint32_t bits = hit <= 0x7F80 ? 0x7F80 - hit : 0x8000 | (hit - 0x7F80), other = bits == 0 ? 0x8000u : bits;
  auto matches = [&](uint32_t b) { return b == bits || b == other; };
  // Occurrences in index order: the logits before the lines, the lines, the logits behind them.
  const Lines G(row, begin, end);
  const unsigned long long edges = __ballot(matches(G.edge(lane)));  // (of lanes 0 .. 15, in every wave)
  const uint32_t head = __popcll(edges & 0xFF);
  if (left < head) {
    unsigned long long e = edges & 0xFF;
    for (; left > 0; --left) e &= e - 1;
    if (tid == 0) found(G.edge_index(__ffsll(e) - 1));
    return;
  }
  left -= head;
  const bool in_registers = !MERGE && G.count <= kBatch * kThreads;
  for (int g0 = 0; g0 < G.count; g0 += kBatch * kThreads) {
    uint32_t hits[kBatch], inc[kBatch];
    if (!in_registers) {
#pragma unroll
      for (int i = 0; i < kBatch; ++i) held[i] = G.load(g0 + i * kThreads + tid);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      hits[i] = 0;
      if (g0 + i * kThreads >= G.count) break;
#pragma unroll
      for (int e = 0; e < 8; ++e) hits[i] |= (matches(place(held[i], e)) ? 1u : 0u) << e;
      inc[i] = wave_prefix((uint32_t)__popc(hits[i]));
      if (lane == 63) s_u[i][wave] = inc[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (g0 + i * kThreads >= G.count) break;
      const uint32_t waves = row_prefix(s_u[i][lane & 15]);
      const uint32_t n = __popc(hits[i]);
      const uint32_t ahead = (wave ? lane_value(waves, wave - 1) : 0u) + inc[i] - n, all = lane_value(waves, 15);
      if (left >= ahead && left < ahead + n) {
        for (uint32_t skip = left - ahead; skip > 0; --skip) hits[i] &= hits[i] - 1;
        found(G.first(g0 + i * kThreads + tid) + __ffs((int)hits[i]) - 1);
      }
      if (left < all) return;
      left -= all;
    }
  }
  unsigned long long e = edges >> 8 & 0xFF;
  for (; left > 0 && (e & (e - 1)) != 0; --left) e &= e - 1;
  if (tid == 0) found(G.edge_index(8 + max(__ffsll(e) - 1, 0)));
}

LdsAllowance g_count, g_pick, g_merge;

constexpr size_t kMergeBytes = (36864 + 64) * sizeof(uint32_t);

struct Plan {
  int slice, slices;
  int64_t batch;
};
// Slices of a row: enough workgroups (one per CU: the histogram takes most of its LDS) for the GPU, at least 4096
// logits each.
Plan plan_of(int64_t M, int V, int cus) {
  const int64_t batch = M < kMaxBatch ? M : kMaxBatch;
  int64_t s = cus / batch;
  if (s > kWaves) s = kWaves;  // (a list to each wave of the merge: 37 slices of one row took it 7 us, 16 take 3)
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
