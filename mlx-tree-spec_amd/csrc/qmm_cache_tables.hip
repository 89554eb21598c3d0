// One step of the paged cache's tables (include/qmm_cache.h): pages given back and taken, the new rows' places, and the plan of
// the step's attention, on the GPU, so that no length has to reach the host.
//
// All of it is prefix sums over the requests (rows, pages back, pages taken, splits) and work over their flat results: item i of
// a sum belongs to the last request whose prefix is at most i, found by a binary search in LDS. One workgroup does it, since
// every part waits for a sum over all requests; only rows past kInOne go to a second launch of many workgroups, which finds its
// requests in the plan (without one, as with kept rows, the first places all). Bound by
// latency: a chain of four prefix sums, and of two loads (the requests' numbers, then page numbers), which is why a row's page is
// read from where this step finds it (the table, or the free list) and not out of the table behind its update, and why the
// first page numbers are on their way while the plan is made.
// 16 requests of one row: 5.4 us, of which an empty launch takes 1.8; 100 of 16 rows 7.9; 24 of 50000 rows 9.4-10.3, and 3.3-4.0 for the rows.
#include <hip/hip_runtime.h>

#include "qmm_cache.h"
#include "qmm_cache_kernels.h"

namespace qmm4 {

namespace {

constexpr int kPer = 2;  // requests of a thread, neighbours
constexpr int kMost = 1024;
// Rows that the one workgroup places itself. (24 requests, two steps: 2000 rows 15.1 us in one launch, 16.5 in two; 4000 rows 16.2
// and 16.6; 10000 rows 20.2 and 16.8.)
constexpr int kInOne = 4096;
static_assert(kMost * kPer >= QMM4_CACHE_MAX_REQUESTS && kMost * 64 >= QMM4_CACHE_MAX_KEEP, "requests, words of kept rows");

// Sums over a wave's lanes up to and with each: shifts by 1, 2, 4 and 8 within rows of 16, then the rows' totals.
__device__ __forceinline__ int wave_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);
  return x;
}

// Exclusive prefix sums over the workgroup's threads of N numbers (below 2^31 in a wave), and their totals. One barrier; s: the
// waves' totals, of two sets in turn (a set is written again behind the next sum's barrier).
template <int N, int WAVES>
__device__ __forceinline__ void block_scan(const int (&v)[N], int64_t (&before)[N], int64_t (&total)[N], int (*s)[WAVES]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int x[N];
#pragma unroll
  for (int n = 0; n < N; ++n) x[n] = wave_scan(v[n]);
  if (lane == 63) {
#pragma unroll
    for (int n = 0; n < N; ++n) s[n][wave] = x[n];
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < N; ++n) {
    before[n] = x[n] - v[n];
    total[n] = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const int t = s[n][w];
      before[n] += w < wave ? t : 0;
      total[n] += t;
    }
  }
}

// The last of R (> 0) rising numbers that is at most i (s[0] <= i).
__device__ __forceinline__ int last_at_most(const int* s, int R, int i) {
  int lo = 0, hi = R;  // s[lo] <= i < s[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (s[mid] <= i) lo = mid;
    else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ int slot_of(int shift, int page, int position) {
  return (int)(((uint32_t)page << shift) + (uint32_t)(position & ((1 << shift) - 1)));
}

__device__ __forceinline__ void place(const CacheStepParams& S, int m, int slot, int position, int request) {
  S.slots[m] = slot;
  S.positions[m] = position;
  S.request[m] = request;
}

template <int THREADS>
__global__ __launch_bounds__(THREADS) void cache_step_kernel(CacheStepParams S) {
  constexpr int kWaves = THREADS / 64, kRequests = THREADS * kPer;
  __shared__ int s_scan[2][4][kWaves];
  __shared__ int s_first[kRequests], s_rows[kRequests], s_base[kRequests], s_left[kRequests], s_back[kRequests], s_took[kRequests];
  static_assert(sizeof(uint64_t) * THREADS == sizeof(int) * kRequests, "s_part below");
  __shared__ uint64_t s_bits[THREADS];  // kept rows, and how many there are before each 64
  __shared__ int s_kept[THREADS];
  const int tid = threadIdx.x, lane = tid & 63, R = S.R, shift = S.page_shift, page = 1 << shift;
  const auto pages_of = [&](int tokens) { return (tokens + page - 1) >> shift; };
  int n[kPer], had[kPer], base[kPer];
  int64_t total3[3], before3[3], total1[1], before1[1], total2[2], before2[2];

  const int in_list = *S.free_count;
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    const int r = tid * kPer + e;
    n[e] = had[e] = base[e] = 0;
    if (r < R) {
      const int most = (int)(S.capacity << shift), length = max(0, min(S.lengths[r], most));
      base[e] = S.base ? max(0, min(S.base[r], length)) : length;
      n[e] = max(0, min(S.rows[r], min(S.max_rows, S.total)));
      had[e] = pages_of(length);
    }
  }
  const int words = S.keep ? (S.total + 63) / 64 : 0;
  for (int w = tid >> 6; w < words; w += kWaves) {
    const int m = w * 64 + lane;
    const uint64_t kept = __ballot(m < S.total && S.keep[m] != 0);
    if (lane == 0) s_bits[w] = kept;
  }
  if (S.keep) __syncthreads();

  // Rows, the pages that go back, kept rows.
  int sums[3] = {0, 0, tid < words ? __builtin_popcountll(s_bits[tid]) : 0};
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    sums[0] += n[e];
    sums[1] += had[e] - pages_of(base[e]);
  }
  block_scan<3, kWaves>(sums, before3, total3, s_scan[0]);
  if (tid < words) s_kept[tid] = (int)before3[2];
  const int64_t back = total3[1];
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    const int r = tid * kPer + e;
    if (r < R) {
      const int first = (int)min(before3[0], (int64_t)S.total);
      before3[0] += n[e];
      n[e] = (int)min(before3[0], (int64_t)S.total) - first;
      s_first[r] = first;
      s_rows[r] = n[e];
      s_base[r] = base[e];
      s_left[r] = pages_of(base[e]);
      s_back[r] = (int)min(before3[1], (int64_t)1 << 30);
      before3[1] += had[e] - s_left[r];
    }
  }
  // (Pages of broken tables past the list's room are dropped.)
  const int count = max(0, min(in_list, S.pages)), room = (int)min(back, (int64_t)(S.pages - count)), available = count + room;
  __syncthreads();
  if (back > 0) {
    for (int i = tid; i < (int)min(back, (int64_t)1 << 30); i += THREADS) {
      const int r = last_at_most(s_back, R, i);
      int32_t* entry = S.table + (int64_t)r * S.capacity + s_left[r] + (i - s_back[r]);
      if (i < room) S.free_pages[count + room - 1 - i] = *entry;
      *entry = -1;
    }
    __syncthreads();
  }

  // Kept rows before row m.
  const auto kept_before = [&](int m) {
    if (m >= S.total) return (int)total3[2];
    return s_kept[m >> 6] + __builtin_popcountll(s_bits[m >> 6] & ((1ull << (m & 63)) - 1));
  };
  // Pages to take. a: rows that get a place, refused requests have none.
  int a[kPer], need[kPer], sum_need[1] = {0};
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    const int r = tid * kPer + e;
    a[e] = need[e] = 0;
    if (r < R) {
      a[e] = S.keep ? kept_before(s_first[r] + n[e]) - kept_before(s_first[r]) : n[e];
      const int want = pages_of(base[e] + a[e]);
      if (want > S.capacity) a[e] = -1;
      else need[e] = want - s_left[r];
      sum_need[0] += need[e];
    }
  }
  block_scan<1, kWaves>(sum_need, before1, total1, s_scan[1]);
  int64_t cost = 0;
  int taken[1] = {0}, blocks = 0;
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    const int r = tid * kPer + e;
    if (r < R) {
      // (Behind a refused request no other takes pages: the flat index below ends at what is taken.)
      s_took[r] = (int)min(before1[0], (int64_t)available);
      before1[0] += need[e];
      if (need[e] > 0 && before1[0] > available) a[e] = -1;
      else taken[0] += need[e];
      if (a[e] < 0) {
        a[e] = 0;
        s_rows[r] = -1 - n[e];
      }
      S.lengths[r] = base[e] + a[e];
      if (S.plan.words && s_rows[r] > 0) {
        const int64_t rows = (int64_t)s_rows[r] * S.G;
        blocks += (int)((rows + kPagedRows - 1) / kPagedRows);
        cost += (int64_t)(base[e] + a[e]) * ((rows + kPagedRows - 1) / kPagedRows);
      }
    }
  }
  int took = (int)total1[0];
  if (total1[0] > available) {
    block_scan<1, kWaves>(taken, before1, total1, s_scan[0]);
    took = (int)total1[0];
    __syncthreads();
  }
  // The sum of the costs, in parts of 22 bits, whose sums in a wave stay below 2^31 (a cost is below 2^54).
  const int parts[4] = {blocks, (int)(cost & 0x3FFFFF), (int)(cost >> 22 & 0x3FFFFF), (int)(cost >> 44)};
  int64_t total4[4], before4[4];
  block_scan<4, kWaves>(parts, before4, total4, s_scan[0]);

  // A request's page, new ones from the list.
  const auto page_of = [&](int r, int column) {
    const int fresh = column - s_left[r];
    return fresh < 0 ? S.table[(int64_t)r * S.capacity + column] : S.free_pages[available - 1 - (s_took[r] + fresh)];
  };
  const auto take = [&](int i, int* r, int* column) {
    *r = last_at_most(s_took, R, i);
    *column = s_left[*r] + (i - s_took[*r]);
    return S.free_pages[available - 1 - i];
  };
  const auto locate = [&](int m, int* slot, int* position, int* request) {
    *slot = *position = *request = -1;
    const int r = R > 0 ? last_at_most(s_first, R, m) : 0;
    if (R > 0 && m - s_first[r] < s_rows[r] && (!S.keep || (s_bits[m >> 6] >> (m & 63) & 1))) {
      *request = r;
      *position = s_base[r] + (S.keep ? kept_before(m) - kept_before(s_first[r]) : m - s_first[r]);
      *slot = slot_of(shift, page_of(r, *position >> shift), *position);
    }
  };
  // The first page and the first row of each thread: loaded here, stored behind the plan.
  const bool place_here = S.total <= kInOne || !S.plan.words;
  int take_r = 0, take_column = 0, take_page = 0, slot, position, request;
  if (tid < took) take_page = take(tid, &take_r, &take_column);
  if (place_here && tid < S.total) locate(tid, &slot, &position, &request);

  if (S.plan.words) {
    // The attention's splits: as many tokens each as leave S.splits in all (a request of several row blocks counts as often). Every
    // request ends in a split that is not full; up to half a round of row blocks, less than their number beside what fills one round
    // is aimed at (one workgroup more than the GPU holds at once takes as long again). More blocks, where one round is aimed at: as
    // many splits as blocks, since twice as many would be two rounds (a prompt of one request is not cut, and has no partial sums).
    const int64_t all = total4[1] + (total4[2] << 22) + (total4[3] << 44);
    const int64_t aim = S.round >= 2 * total4[0]   ? S.round - total4[0] + 1
                        : S.splits > S.round ? S.splits
                                             : min(S.splits, total4[0]);
    const int64_t chunk = max((int64_t)kPagedUnit, ((all + aim - 1) / aim + kPagedUnit - 1) / kPagedUnit * kPagedUnit);
    // A request's record up to its partial rows. (Without keep every row of a request that is not refused has a place.)
    const auto record = [&](int r) {
      PagedRequest q = {s_first[r], max(0, s_rows[r]), 0, kPagedUnit, 0, 0, {0, 0}};
      q.length = s_base[r] + q.rows;
      if (q.rows > 0) {
        const uint32_t length = q.length, pieces = chunk >= length ? 1 : (length + (uint32_t)chunk - 1) / (uint32_t)chunk;
        q.per = ((length + pieces - 1) / pieces + kPagedUnit - 1) / kPagedUnit * kPagedUnit;
        q.splits = (length + (uint32_t)q.per - 1) / (uint32_t)q.per;
      }
      return q;
    };
    PagedRequest q[kPer];
    int sum_splits[2] = {0, 0};
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      q[e] = {0, 0, 0, 0, 0, 0, {0, 0}};
      if (tid * kPer + e < R) q[e] = record(tid * kPer + e);
      sum_splits[0] += q[e].splits;
      sum_splits[1] += q[e].splits > 1 ? q[e].splits * q[e].rows : 0;
    }
    block_scan<2, kWaves>(sum_splits, before2, total2, s_scan[1]);
    // (s_back has served, and without keep s_bits does not: the requests' first items and partial rows.)
    int* s_part = reinterpret_cast<int*>(s_bits);
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const int r = tid * kPer + e;
      if (r < R) {
        s_part[r] = q[e].part = (int)before2[1];
        S.plan.requests()[r] = q[e];
        before2[1] += q[e].splits > 1 ? q[e].splits * q[e].rows : 0;
        s_back[r] = (int)before2[0];
        before2[0] += q[e].splits;
      }
    }
    if (tid == 0) S.plan.words[0] = (int)total2[0];
    __syncthreads();
    for (int i = tid; i < (int)total2[0]; i += THREADS) {
      const int r = last_at_most(s_back, R, i), split = i - s_back[r];
      const PagedRequest t = record(r);
      const int begin = split * t.per;
      S.plan.items()[i] = {r, t.first, t.rows, t.length, begin, min(t.length, begin + t.per),
                           t.splits > 1 ? s_part[r] + split * t.rows : -1, page_of(r, begin >> shift)};
    }
  }

  if (tid == 0) *S.free_count = available - took;
  for (int i = tid; i < took; i += THREADS) {
    if (i != tid) take_page = take(i, &take_r, &take_column);
    S.table[(int64_t)take_r * S.capacity + take_column] = take_page;
  }
  if (place_here) {
    for (int m = tid; m < S.total; m += THREADS) {
      if (m != tid) locate(m, &slot, &position, &request);
      place(S, m, slot, position, request);
    }
  }
}

// The places of many rows, from the plan.
__global__ __launch_bounds__(kMost) void cache_rows_kernel(CacheStepParams S) {
  __shared__ int s_first[QMM4_CACHE_MAX_REQUESTS];
  for (int r = threadIdx.x; r < S.R; r += kMost) s_first[r] = S.plan.requests()[r].first;
  __syncthreads();
  const int m = blockIdx.x * kMost + threadIdx.x;
  if (m >= S.total) return;
  int slot = -1, position = -1, request = -1;
  if (S.R > 0) {
    const int r = last_at_most(s_first, S.R, m), n = S.plan.requests()[r].rows;
    if (m - s_first[r] < n) {
      request = r;
      position = S.plan.requests()[r].length - n + (m - s_first[r]);
      slot = slot_of(S.page_shift, S.table[(int64_t)r * S.capacity + (position >> S.page_shift)], position);
    }
  }
  place(S, m, slot, position, request);
}

}  // namespace

hipError_t launch_cache_step(const CacheStepParams& p, hipStream_t stream) {
  // Fewer threads, whose barriers and sums are shorter, where two rows each are enough (a step of 16 requests 6.2 us, 9.6 with 1024
  // threads; of 600 11.5, 12.4).
  const int n = p.R > p.total ? p.R : p.total;
  if (n <= 512) hipLaunchKernelGGL(cache_step_kernel<256>, dim3(1), dim3(256), 0, stream, p);
  else if (n <= 1024) hipLaunchKernelGGL(cache_step_kernel<512>, dim3(1), dim3(512), 0, stream, p);
  else hipLaunchKernelGGL(cache_step_kernel<kMost>, dim3(1), dim3(kMost), 0, stream, p);
  if (p.total > kInOne && p.plan.words)
    hipLaunchKernelGGL(cache_rows_kernel, dim3((p.total + kMost - 1) / kMost), dim3(kMost), 0, stream, p);
  return hipGetLastError();
}

}  // namespace qmm4
