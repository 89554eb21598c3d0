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
// The sums run over the values that occur, up to 4096 of them (a page) listed in LDS, 4 neighbours to a thread: one
// prefix over the workgroup, of counts and masses. What top-k, top-p and min-p keep is a beginning of the order, so
// each of them is a place in that prefix, and so is the target: the thread that holds it works it out and writes it
// down for the others. More values (152k logits of a model have about 3500; past 4096 they lie many octaves apart) take
// their pages in turn, once per place to be found.
//
// What bounds it: a row's steps follow each other in one workgroup, each a few hundred ns of LDS round trips and
// barriers, and a CU gets through 2400 vector instructions of its waves each a microsecond; both kernels are kept to
// few instructions per value. On the GPU: 1 x 151936 20.1 us, 32 x 151936 (all settings) 22.8 us, 200 x 32001 14.4 us
// (13.4 in a row of eager calls). Of these the count kernel takes 6.8 and 7.7, and the counting of the last, inside the
// pick kernel, 4.5. The prefix after prefix of counts, masses and what is kept that was here
// first, with 64 words to a look, took 27, 30 and 18 us.
#include <type_traits>

#include "qmm4_common.h"
#include "qmm4_lds.h"
#include "qmm_requests_kernels.h"

namespace qmm4 {

namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kFirstRank = 0x7F, kLastRank = 0xFF7E;  // +infinity, the lowest finite value
constexpr int kNoRank = 0x10000;
constexpr int kMaxSlice = 32768;   // logits per slice: its counts fit 16 bits
constexpr int kMinSlice = 4096;
constexpr int kMaxSlices = 512;
constexpr int kMaxBatch = 256;     // rows per launch, and
constexpr int kMaxLogits = 1 << 28;  // their logits: bound the lists at 1 GiB (any row fits; past 2^20 logits a row:
                                     // 64 x 2^24 1.27 -> 1.82 ms, with 1 instead of 4 GiB)

// A rank is a bf16 value's number in falling order: 0x7FFF - b for bits b of a positive value, b - 1 of a negative one
// (0x7FFF for both zeros). -infinity (kLastRank + 1) and NaN lie either side of kFirstRank .. kLastRank.
__device__ __forceinline__ uint32_t bits_of(int rank) { return rank <= 0x7FFF ? 0x7FFF - rank : rank + 1; }
__device__ __forceinline__ double value_of(int rank) { return (double)bf16_to_f32(bits_of(rank)); }
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef int16_t i16x2 __attribute__((ext_vector_type(2)));
// The ranks of two values.
__device__ __forceinline__ u16x2 ranks_of(uint32_t b) {
  const uint32_t negative = __builtin_bit_cast(uint32_t, __builtin_bit_cast(i16x2, b) >> 15);
  return __builtin_bit_cast(u16x2, b ^ (0x7FFF7FFFu & ~negative)) + __builtin_bit_cast(u16x2, negative);
}
__device__ __forceinline__ u16x2 min2(u16x2 a, u16x2 b) {  // (a minimum with 1 would be compiled into comparisons)
  u16x2 r;
  asm("v_pk_min_u16 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
  return r;
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
// The smallest of ranks up to kNoRank.
__device__ __forceinline__ int row_min(int v) { return kNoRank - row_max(kNoRank - v); }
__device__ __forceinline__ int wave_min(int v) { return kNoRank - wave_max(kNoRank - v); }

// 16-bit counts of the logits, two to a word; returns the smallest rank this thread saw, NaN's included. `held`: the
// lines loaded last (lines threadIdx.x + i kThreads where there are at most kBatch * kThreads of them). `between` runs
// while the first loads are under way. Two logits at a time up to their addresses, 9 instructions each (one at a time
// 14: 200 x 32001 14.1 us instead of 13.5).
constexpr int kBatch = 4;
template <class F>
__device__ __forceinline__ int count_lines(const Lines& G, uint32_t* hist, u32x4 (&held)[kBatch], F&& between) {
  const uint16_t lane = threadIdx.x & 63;
  const u16x2 last = {kLastRank, kLastRank}, one = {1, 1}, lanes = {lane, lane};
  u16x2 lowest = {0xFFFF, 0xFFFF};
  auto count = [&](uint32_t b) {
    u16x2 r = ranks_of(b);
    lowest = min2(lowest, r);
    // -infinity goes to a bin of each lane's own past the values (a masked row would add to one word). NaN goes to some
    // bin past them or, around the 16 bits, in front of them.
    r += min2(__builtin_elementwise_sub_sat(r, last), one) * lanes;
    atomicAdd(&hist[r.x >> 1], __umul24(r.x & 1u, 0xFFFFu) + 1u);
    atomicAdd(&hist[r.y >> 1], __umul24(r.y & 1u, 0xFFFFu) + 1u);
  };
  const uint32_t edge = G.edge(threadIdx.x);
  for (int g0 = threadIdx.x, at = 0; at < max(G.count, 1); g0 += kBatch * kThreads, at += kBatch * kThreads) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i) held[i] = G.load(g0 + i * kThreads);
    if (at == 0) {
      __builtin_amdgcn_sched_barrier(0);
      between();
      count(kNone << 16 | edge);
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (at + i * kThreads >= G.count) break;
#pragma unroll
      for (int e = 0; e < 4; ++e) count(held[i][e]);
    }
  }
  __syncthreads();
  // What lies either side of the values is cleared.
  constexpr int kFront = kFirstRank / 2, kBack = kLastRank / 2;  // words that the first and the last value share with it
  const int t = threadIdx.x;
  if (t < kFront) hist[t] = 0;
  if (t == kFront) hist[t] &= 0xFFFF0000u;
  if (t > kFront && t <= kFront + 0x7FFF - kBack) hist[kBack + t - kFront] = 0;
  if (t == kThreads - 1) hist[kBack] &= 0xFFFFu;
  return min((int)lowest.x, (int)lowest.y);
}

// The smallest rank of the workgroup's logits (kNoRank: none), `mine` from count_lines. With a NaN among them
// it is looked for in the histogram.
__device__ __forceinline__ int lowest_rank(const uint32_t* hist, int mine, int* s_lo) {
  for (;;) {
    mine = wave_min(mine);
    if ((threadIdx.x & 63) == 0) s_lo[threadIdx.x >> 6] = mine;
    __syncthreads();
    const int lowest = row_min(s_lo[threadIdx.x & (kWaves - 1)]);
    if (lowest >= kFirstRank) return lowest <= kLastRank ? lowest : kNoRank;
    __syncthreads();
    mine = kNoRank;
    for (int w = threadIdx.x; w < 32768; w += kThreads) {
      const uint32_t n = hist[w];
      if (n != 0) mine = min(mine, 2 * w + ((n & 0xFFFFu) == 0));
    }
  }
}

template <int BYTES>
__device__ __forceinline__ void zero_lds(uint32_t* p) {
  for (int i = threadIdx.x; i < BYTES / 16; i += kThreads) reinterpret_cast<u32x4*>(p)[i] = u32x4{0u, 0u, 0u, 0u};
}

// Where a batch's lists lie: heads [rows][slices], entries [rows][slices][slice], an entry rank << 16 | count (a
// slice's list padded to a multiple of 4 with count 0).
struct Head {
  uint32_t n, lowest;  // entries, and the smallest rank (kNoRank where there is none)
};
struct Lists {
  Head* heads;
  uint32_t* entries;
  int slice, slices;
  __device__ uint32_t* list(int64_t m, int s) const { return entries + (m * slices + s) * (int64_t)slice; }
};

// How many of four counts, or of eight of 16 bits, are not zero.
template <bool PAIRS>
__device__ __forceinline__ uint32_t occurring(u32x4 v) {
  uint32_t n = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if constexpr (PAIRS) n += __popc((((v[e] & 0x7FFF7FFFu) + 0x7FFF7FFFu) | v[e]) & 0x80008000u);
    else n += min(v[e], 1u);
  }
  return n;
}

// before(total) with the number of values that occur in a histogram, then emit(o, r, n) for each, r its number, n its
// count and o its place among them in rising r. PAIRS: 16-bit counts, two to a word.
// A wave looks at 256 neighbouring words at a time (16 bytes a lane), the next wave at the next: occurring values crowd
// in a few octaves. A lane's place is a prefix over the wave, and over the looks before (look [WORDS / 256] in LDS,
// summed by each wave itself). HELD: the words stay in registers between the two, else they are read again.
template <bool PAIRS, int WORDS, bool HELD, class T, class F>
__device__ __forceinline__ void list_values(const uint32_t* hist, uint32_t* look, T&& before, F&& emit) {
  constexpr int kLooks = WORDS / 256 / kWaves, kHalf = PAIRS ? 2 : 1;
  constexpr int kSums = (kLooks * kWaves + 63) / 64;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  auto words = [&](int t) { return reinterpret_cast<const u32x4*>(hist)[(t * kWaves + wave) * 64 + lane]; };
  auto none = [](u32x4 v) { return __ballot((v.x | v.y | v.z | v.w) != 0) == 0; };
  u32x4 v[HELD ? kLooks : 1];
  uint32_t own[HELD ? kLooks : 1], mine = 0;  // (own: the lane's prefix within the look, without itself)
  auto sum = [&](int t, u32x4 v, uint32_t& own) {
    own = 0;
    if (none(v)) return;
    const uint32_t n = occurring<PAIRS>(v), inc = wave_prefix(n), all = lane_value(inc, 63);  // (in every lane)
    own = inc - n;
    mine = lane == t ? all : mine;
  };
  if constexpr (HELD) {
#pragma unroll
    for (int t = 0; t < kLooks; ++t) v[t] = words(t);
#pragma unroll
    for (int t = 0; t < kLooks; ++t) sum(t, v[t], own[t]);
  } else {
#pragma clang loop unroll(disable)
    for (int t = 0; t < kLooks; ++t) sum(t, words(t), own[0]);
  }
  if (lane < kLooks) look[lane * kWaves + wave] = mine;
  __syncthreads();
  uint32_t ahead[kSums], total = 0;
#pragma unroll
  for (int i = 0; i < kSums; ++i) {
    const uint32_t n = i * 64 + lane < kLooks * kWaves ? look[i * 64 + lane] : 0, inc = wave_prefix(n);
    ahead[i] = total + inc - n;
    total += lane_value(inc, 63);
  }
  before(total);
  auto list = [&](int t, u32x4 v, uint32_t o) {
    if (none(v)) return;
#pragma unroll
    for (int e = 0; e < 4 * kHalf; ++e) {
      const uint32_t n = !PAIRS ? v[e] : e & 1 ? v[e / 2] >> 16 : v[e / 2] & 0xFFFFu;
      if (n != 0) emit(o++, (uint32_t)((t * kWaves + wave) * 256 + lane * 4) * kHalf + e, n);
    }
  };
  if constexpr (HELD) {
#pragma unroll
    for (int t = 0; t < kLooks; ++t) list(t, v[t], own[t] + lane_value(ahead[t * kWaves / 64], t * kWaves % 64 + wave));
  } else {
#pragma clang loop unroll(disable)
    for (int t = 0; t < kLooks; ++t) {
      uint32_t at = ahead[0];
#pragma unroll
      for (int i = 1; i < kSums; ++i) at = t * kWaves / 64 == i ? ahead[i] : at;
      sum(t, words(t), own[0]);
      list(t, words(t), own[0] + lane_value(at, t * kWaves % 64 + wave));
    }
  }
}

constexpr int kBytes16 = 65536 * 2;

__global__ __launch_bounds__(kThreads) void sample_count_kernel(SampleParams S, Lists L) {
  extern __shared__ __attribute__((aligned(16))) uint32_t hist[];
  __shared__ uint32_t s_look[128];
  __shared__ int s_lo[kWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t m = blockIdx.y;
  const int begin = blockIdx.x * L.slice, end = min(S.V, begin + L.slice);
  u32x4 held[kBatch];
  const int mine = count_lines(Lines(S.logits + m * S.row_stride, begin, end), hist, held, [&] {
    zero_lds<kBytes16>(hist);
    __syncthreads();
  });
  const int lowest = lowest_rank(hist, mine, s_lo);
  uint32_t* list = L.list(m, blockIdx.x);
  list_values<true, 32768, true>(
      hist, s_look,
      [&](uint32_t n) {
        if (tid == 0) L.heads[m * L.slices + blockIdx.x] = {n, (uint32_t)lowest};
        if (tid < 4 && (n & 3) != 0 && tid >= (int)(n & 3)) list[(n & ~3u) + tid] = 0;
      },
      [&](uint32_t o, uint32_t r, uint32_t n) { list[o] = r << 16 | n; });
}

// (The loop over pages would keep the constants of an inlined exp in 50 registers and the rest in memory: 0.8 us, in
// rows that never come to it.)
__device__ __attribute__((noinline)) double exp_called(double x) { return exp(x); }

// One row. MERGE: from the slices' lists, else from the row itself.
template <bool MERGE>
__global__ __launch_bounds__(kThreads) void sample_pick_kernel(SampleParams S, Lists L) {
  constexpr int kSpan = MERGE ? 36864 : 65536;  // values of one histogram: +-512 with all between, or all
  constexpr int kPage = 4096, kPer = kPage / kThreads;  // listed values at a time, of them to a thread
  extern __shared__ __attribute__((aligned(16))) uint32_t hist[];
  __shared__ uint16_t s_page[kPage];
  __shared__ int s_lo[kWaves];
  __shared__ double s_mass[kWaves];
  __shared__ uint32_t s_u[kBatch][kWaves], s_look[kSpan / 256], s_n[MERGE ? kMaxSlices : 1], s_occ[MERGE ? kMaxSlices : 1];
  __shared__ uint32_t s_count[kWaves], s_above[kWaves], s_far;
  struct Cut {  // an end of what is kept: the mass before it, the last value kept (its number in the order), how often
    double mass;
    uint32_t index, n;
  };
  __shared__ Cut s_cut[3];
  __shared__ uint32_t s_hit[2];
  __shared__ double s_weight;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t m = blockIdx.x;
  const uint16_t* row = S.logits + m * S.row_stride;

  // (Each with a load, one value for all or not: loads behind a branch wait for each other.)
  const uint32_t* const any = reinterpret_cast<const uint32_t*>(S.uniform);
  auto setting = [&](auto s) {
    const uint32_t v = (s.p ? reinterpret_cast<const uint32_t*>(s.p) : any)[m];
    return s.p ? __builtin_bit_cast(decltype(s.value), v) : s.value;
  };
  float temp = setting(S.temperature), top_p = setting(S.top_p), min_p = setting(S.min_p);
  const float u = S.uniform[m];
  const int32_t top_k = setting(S.top_k);
  // Settings that leave the first of the order only.
  const bool first_only = !(temp > 0.0f) || top_p <= 0.0f || min_p > 1.0f || top_k == 1;
  const uint32_t limit = top_k > 0 ? (uint32_t)top_k : 0xFFFFFFFFu;

  // `lowest`: the first value that occurs. The histogram holds values from `base`; a second one (part 1) those past
  // its end, where there are any.
  int lowest, base = 0;
  u32x4 held[kBatch];
  if constexpr (MERGE) {
    int lo = kNoRank;
    for (int s = tid; s < L.slices; s += kThreads) {
      const Head head = L.heads[m * L.slices + s];
      s_n[s] = head.n;
      lo = min(lo, (int)head.lowest);
    }
    if (tid == 0) s_far = 0;
    zero_lds<kSpan * 4>(hist);
    lowest = lowest_rank(hist, lo, s_lo);
    base = lowest & ~3;
  } else {
    const int mine = count_lines(Lines(row, 0, S.V), hist, held, [&] {
      zero_lds<kBytes16>(hist);
      __syncthreads();
    });
    lowest = lowest_rank(hist, mine, s_lo);
  }
  if (lowest == kNoRank) {
    if (tid == 0) {
      S.tokens[m] = -1;
      S.logprobs[m] = -__builtin_inff();
    }
    return;
  }

  uint32_t hit = lowest, left = 0;
  double hit_weight = 1.0, kept_total = 1.0;
  if (!first_only) {
    const double largest = value_of(lowest), per_temp = 1.0 / (double)temp;
    const bool some = limit < (uint32_t)S.V;  // (top-k may end the order)
    // Four walks through the pages: the masses and counts; the end that top-k sets; those of top-p and min-p; the value
    // that passes the target. The order's masses before each thread's values are the same in each: an end is a place in
    // them, and the thread that holds it writes it down. One page is walked where it stands, in registers; more are
    // listed again for each walk.
    double target = 0.0;
    Cut cut = {0.0, 0xFFFFFFFFu, 0};
    uint32_t c[kPer], count = 0, count_before = 0, entries = 0;
    double w[kPer], mass = 0.0, mass_before = 0.0;
    double lane_waves = 0.0;  // of lane i: the mass before wave i's values; lane_has: whether those have any
    bool lane_has = false;
    int rank[kPer], per = 0;
    // Sums over the values so far.
    uint32_t count_sum = 0, above_sum = 0, above_total = 0, index0 = 0;
    double mass_sum = 0.0;
    // The lists' values from `from` on into the histogram (cleared before).
    auto merge = [&](int from) __attribute__((always_inline)) {
      bool far = false;
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
            if (i0 + i * 64 >= n4) break;
#pragma unroll
            for (int e = 0; e < 4; ++e) {  // (what is not for this histogram goes behind it, one word for each lane)
              const int r = (int)(v[i][e] >> 16) - from;
              atomicAdd(&hist[min((uint32_t)r, (uint32_t)(kSpan + lane))], v[i][e] & 0xFFFFu);
              far |= r >= kSpan;
            }
          }
        }
      }
      if (far) s_far = 1;
      __syncthreads();
    };
    // A page of a histogram: the values that occur, the first-th and on, with their weights and masses.
    auto list_page = [&](auto held, int from, uint32_t first) __attribute__((always_inline)) {
      list_values<!MERGE, kSpan / (MERGE ? 1 : 2), decltype(held)::value>(
          hist, s_look, [&](uint32_t n) { entries = n; },
          [&](uint32_t o, uint32_t r, uint32_t) {
            o -= first;
            if (o < (uint32_t)kPage) s_page[o] = (uint16_t)r;
          });
      __syncthreads();
      const uint32_t in_page = min(entries - first, (uint32_t)kPage);
      per = (int)((in_page + kThreads - 1) / kThreads);
      uint32_t above = 0;
      count = 0;
      mass = 0.0;
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        c[e] = 0;
        w[e] = 0.0;
        if (e >= per) continue;
        const uint32_t i = tid * per + e;
        const bool is = i < in_page;
        const uint32_t r = is ? s_page[i] : 0u;
        rank[e] = from + (int)r;
        c[e] = !is ? 0u : MERGE ? hist[r] : r & 1 ? hist[r >> 1] >> 16 : hist[r >> 1] & 0xFFFFu;
      }
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        if (e >= per) break;
        // (The largest value itself has 1, also where it is infinite.)
        const double d = value_of(rank[e]) - largest;
        w[e] = rank[e] == lowest ? 1.0 : largest == __builtin_inf() ? 0.0 : (decltype(held)::value ? exp(d * per_temp) : exp_called(d * per_temp));
        if (c[e] == 0) w[e] = 0.0;
        if (min_p > 0.0f) above += __popcll(__ballot(w[e] >= (double)min_p));
        count += c[e];
        mass += c[e] * w[e];
      }
      const double mass_inc = wave_prefix(mass);
      uint32_t count_inc = 0;
      if (some) count_inc = wave_prefix(count);
      if (lane == 63) {
        s_mass[wave] = mass_inc;
        s_count[wave] = count_inc;
        s_above[wave] = above;
      }
      __syncthreads();
      const double of_wave = s_mass[lane & (kWaves - 1)], waves = mass_sum + row_prefix(of_wave);
      lane_waves = dpp<0x111, 0xF>(waves);
      if (lane == 0) lane_waves = mass_sum;
      lane_has = lane < kWaves && of_wave > 0.0;
      mass_before = lane_value(lane_waves, wave) + (mass_inc - mass);
      mass_sum = lane_value(waves, kWaves - 1);
      if (some) {
        const uint32_t counts = count_sum + row_prefix(s_count[lane & (kWaves - 1)]);
        count_before = (wave ? lane_value(counts, wave - 1) : count_sum) + (count_inc - count);
        count_sum = lane_value(counts, kWaves - 1);
      }
      if (min_p > 0.0f) above_sum += lane_value(row_prefix(s_above[lane & (kWaves - 1)]), kWaves - 1);
    };
    auto decide = [&](int walk) __attribute__((always_inline)) {
      const uint32_t page0 = index0, own0 = page0 + tid * per;  // numbers in the order: the page's first, the thread's
      // Whether this thread is the page's last with some mass that starts before x (or at x), up to value number `last`.
      auto holds = [&](double x, bool at, uint32_t last) __attribute__((always_inline)) {
        const unsigned long long in = __ballot(lane_has && (lane_waves < x || (at && lane_waves == x)) && page0 + lane * 64 * per <= last);
        if (in == 0 || wave != 63 - __builtin_clzll(in)) return false;
        const unsigned long long threads = __ballot(mass > 0.0 && (mass_before < x || (at && mass_before == x)) && own0 <= last);
        return threads != 0 && lane == 63 - __builtin_clzll(threads);
      };
      if (walk == 1 && count_before < limit && limit - count_before <= count) {
        uint32_t cb = count_before;
        double mb = mass_before;
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
          if (cb < limit && limit - cb <= c[e]) s_cut[0] = {mb + (limit - cb) * w[e], own0 + e, limit - cb};
          cb += c[e];
          mb += c[e] * w[e];
        }
      }
      if (walk == 2) {
        const double bound = (double)top_p * cut.mass;
        if (top_p < 1.0f && holds(bound, false, 0xFFFFFFFFu)) {  // kept: with less mass than the bound before them
          Cut end = cut;
          double mb = mass_before;
#pragma unroll
          for (int e = 0; e < kPer; ++e) {
            const double after = mb + c[e] * w[e];
            if (w[e] > 0.0 && mb < bound) {
              const uint32_t n = after > bound ? min(c[e], (uint32_t)ceil((bound - mb) / w[e])) : c[e];
              end = {mb + n * w[e], own0 + e, n};
            }
            mb = after;
          }
          s_cut[1] = end;
        }
        if (min_p > 0.0f && above_total - 1 - own0 < (uint32_t)per) {
          double mb = mass_before;
#pragma unroll
          for (int e = 0; e < kPer; ++e) {
            mb += c[e] * w[e];
            if (own0 + e == above_total - 1) s_cut[2] = {mb, own0 + e, c[e]};
          }
        }
      }
      if (walk == 3 && holds(target, true, cut.index)) {  // (up to rounding: then the last value kept)
        uint32_t hit_n = 1, hit_rank = 0;
        double mb = mass_before, hit_before = 0.0, weight = 1.0;
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
          if (own0 + e <= cut.index && w[e] > 0.0 && mb <= target) {
            hit_n = own0 + e == cut.index ? cut.n : c[e];
            hit_rank = (uint32_t)rank[e];
            hit_before = mb;
            weight = w[e];
          }
          mb += c[e] * w[e];
        }
        const double j = floor((target - hit_before) / weight);
        s_hit[0] = hit_rank;
        s_hit[1] = j < (double)(hit_n - 1) ? (uint32_t)j : hit_n - 1;
        s_weight = weight;
      }
    };
    // Behind a walk: what it found.
    auto walked = [&](int walk) __attribute__((always_inline)) {
      __syncthreads();
      if (walk == 1) cut = s_cut[0];
      if (walk == 2 && top_p < 1.0f && s_cut[1].mass < cut.mass) cut = s_cut[1];
      if (walk == 2 && min_p > 0.0f && s_cut[2].mass < cut.mass) cut = s_cut[2];
    };
    const bool by_mass = top_p < 1.0f || min_p > 0.0f;
    if constexpr (MERGE) merge(base);
    const int parts = MERGE && s_far != 0 ? 2 : 1;
    list_page(std::true_type(), base, 0);
    if (parts == 1 && entries <= kPage) {
      const uint32_t count_total = count_sum;
      above_total = above_sum;
      cut.mass = mass_sum;
      if (some && limit < count_total) {
        decide(1);
        walked(1);
      }
      if (by_mass) {
        decide(2);
        walked(2);
      }
      target = (double)(u > 0.0f ? u : 0.0f) * cut.mass;
      decide(3);
      walked(3);
    } else {
      uint32_t count_total = 0;
      int built = 0;
#pragma clang loop unroll(disable)
      for (int walk = 0; walk < 4; ++walk) {
        if (walk == 1 && !(some && limit < count_total)) continue;
        if (walk == 2 && !by_mass) continue;
        count_sum = above_sum = index0 = 0;
        mass_sum = 0.0;
        for (int part = 0; part < parts; ++part) {
          if (MERGE && built != part) {
            __syncthreads();
            zero_lds<kSpan * 4>(hist);
            __syncthreads();
            built = part;
            merge(base + part * kSpan);
          }
          for (uint32_t first = 0; first == 0 || first < entries; first += kPage) {
            list_page(std::false_type(), base + part * kSpan, first);
            decide(walk);
            index0 += min(entries - first, (uint32_t)kPage);
          }
        }
        walked(walk);
        if (walk == 0) {
          count_total = count_sum;
          above_total = above_sum;
          cut.mass = mass_sum;
        }
        target = (double)(u > 0.0f ? u : 0.0f) * cut.mass;
      }
    }
    hit = s_hit[0];
    left = s_hit[1];
    hit_weight = s_weight;
    kept_total = cut.mass;
  }


  // The slice with the occurrence: the value's count in each list, found by two looks of a wave.
  int begin = 0, end = S.V;
  if constexpr (MERGE) {
    for (int s = wave; s < L.slices; s += kWaves) {
      const int n = (int)s_n[s];
      const uint32_t* list = L.list(m, s);
      const int step = (n + 63) / 64;
      const unsigned long long le = __ballot(lane * step < n && list[min(lane * step, max(n - 1, 0))] >> 16 <= hit);
      uint32_t occ = 0;
      if (le != 0) {
        const int from = (63 - __builtin_clzll(le)) * step;
        for (int i = lane; i < step; i += 64) {
          const uint32_t v = from + i < n ? list[from + i] : 0xFFFFFFFFu;  // (no rank)
          if (v >> 16 == hit) occ = v & 0xFFFFu;
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
  // The value's bits; of zero without the sign.
  const uint32_t bits = bits_of((int)hit), mask = bits == 0 ? 0x7FFFu : 0xFFFFu;
  auto matches = [&](uint32_t b) { return (b & mask) == bits; };
  auto line_misses = [&](u32x4 v) {  // how many of a line's 8 do not match
    u32x4 d;
#pragma unroll
    for (int e = 0; e < 4; ++e) d[e] = (v[e] ^ bits * 0x10001u) & mask * 0x10001u;
    return occurring<true>(d);
  };
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
    uint32_t n[kBatch], inc[kBatch];
    if (!in_registers) {
#pragma unroll
      for (int i = 0; i < kBatch; ++i) held[i] = G.load(g0 + i * kThreads + tid);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (g0 + i * kThreads >= G.count) break;
      n[i] = 8 - line_misses(held[i]);
      inc[i] = wave_prefix(n[i]);
      if (lane == 63) s_u[i][wave] = inc[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (g0 + i * kThreads >= G.count) break;
      const uint32_t waves = row_prefix(s_u[i][lane & (kWaves - 1)]), all = lane_value(waves, kWaves - 1);
      const uint32_t ahead = (wave ? lane_value(waves, wave - 1) : 0u) + inc[i] - n[i];
      if (left >= ahead && left < ahead + n[i]) {
        uint32_t hits = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) hits |= (matches(place(held[i], e)) ? 1u : 0u) << e;
        for (uint32_t skip = left - ahead; skip > 0; --skip) hits &= hits - 1;
        found(G.first(g0 + i * kThreads + tid) + __ffs((int)hits) - 1);
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
  const int64_t most = kMaxLogits / V < kMaxBatch ? kMaxLogits / V : kMaxBatch;
  const int64_t batch = M < most ? M : most;
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
  return (p.batch * p.slices + 1) / 2 * 16 + p.batch * p.slices * (int64_t)p.slice * (int64_t)sizeof(uint32_t);
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
  char* ws = static_cast<char*>(workspace);
  const Lists lists{reinterpret_cast<Head*>(ws), reinterpret_cast<uint32_t*>(ws + (plan.batch * plan.slices + 1) / 2 * 16),
                    plan.slice, plan.slices};
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
