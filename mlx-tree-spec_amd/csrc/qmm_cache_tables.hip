// One step of the paged cache's tables (include/qmm_cache.h): pages given back and taken, the new rows' places, and the plan of
// the step's attention, on the GPU, so that no length has to reach the host.
//
// All of it is prefix sums over the requests (rows, pages back, pages taken, splits) and work over their flat results: item i of
// a sum belongs to the last request whose prefix is at most i, found by a binary search in LDS. One workgroup does it, since
// every part waits for a sum over all requests; only rows past kInOne go to a second launch of many workgroups.
#include <hip/hip_runtime.h>

#include "qmm_cache.h"
#include "qmm_cache_kernels.h"

namespace qmm4 {

namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kMaxRequests = QMM4_CACHE_MAX_REQUESTS;
constexpr int kPer = (kMaxRequests + kThreads - 1) / kThreads;  // requests of a thread, neighbours
// Rows that the one workgroup places itself.
constexpr int kInOne = 4096;

// Exclusive prefix sum over the workgroup's threads, and the total. s: kWaves + 1 words, free again after the next barrier.
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* s, int64_t* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int64_t x = v;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int64_t y = __shfl_up(x, off);
    if (lane >= off) x += y;
  }
  __syncthreads();
  if (lane == 63) s[wave] = x;
  __syncthreads();
  int64_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const int64_t t = s[w];
    before += w < wave ? t : 0;
    all += t;
  }
  *total = all;
  return before + x - v;
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

__device__ __forceinline__ void place(const CacheStepParams& S, int m, int slot, int position, int request) {
  S.slots[m] = slot;
  S.positions[m] = position;
  S.request[m] = request;
}

__device__ __forceinline__ int slot_of(const CacheStepParams& S, int r, int position) {
  const uint32_t page = S.table[(int64_t)r * S.capacity + (position >> S.page_shift)];
  return (int)((page << S.page_shift) + (uint32_t)(position & ((1 << S.page_shift) - 1)));
}

__global__ __launch_bounds__(kThreads) void cache_step_kernel(CacheStepParams S) {
  __shared__ int64_t s_scan[kWaves];
  __shared__ int s_first[kMaxRequests], s_rows[kMaxRequests], s_base[kMaxRequests], s_off[kMaxRequests], s_left[kMaxRequests],
      s_kept[kMaxRequests];
  const int tid = threadIdx.x, R = S.R, page = 1 << S.page_shift;
  const auto pages_of = [&](int64_t tokens) { return (int)((tokens + page - 1) >> S.page_shift); };
  int n[kPer], had[kPer], base[kPer];
  int64_t total;

  // Kept rows before each row (into positions for now).
  if (S.keep) {
    int64_t before = 0;
    for (int m0 = 0; m0 < S.total; m0 += kThreads) {
      const int m = m0 + tid;
      const int v = m < S.total && S.keep[m] != 0;
      const int64_t at = before + block_scan(v, s_scan, &total);
      if (m < S.total) S.positions[m] = (int)at;
      before += total;
      __syncthreads();
    }
    if (tid == 0) s_scan[0] = before;
    __syncthreads();
  }
  const int all_kept = S.keep ? (int)s_scan[0] : 0;

  // Rows, bases and the pages that go back.
  int64_t sum_n = 0, sum_back = 0;
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    const int r = tid * kPer + e;
    n[e] = had[e] = base[e] = 0;
    if (r < R) {
      const int64_t most = S.capacity << S.page_shift;
      const int length = (int)max((int64_t)0, min((int64_t)S.lengths[r], most));
      base[e] = S.base ? max(0, min(S.base[r], length)) : length;
      n[e] = max(0, min(S.rows[r], min(S.max_rows, S.total)));
      had[e] = pages_of(length);
      s_left[r] = pages_of(base[e]);
      s_base[r] = base[e];
      sum_back += had[e] - s_left[r];
      sum_n += n[e];
    }
  }
  int64_t at_n = block_scan(sum_n, s_scan, &total);
  int64_t at_back = block_scan(sum_back, s_scan, &total);
  const int64_t back = total;
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    const int r = tid * kPer + e;
    if (r < R) {
      const int64_t first = min(at_n, (int64_t)S.total);
      at_n += n[e];
      n[e] = (int)(min(at_n, (int64_t)S.total) - first);
      s_first[r] = (int)first;
      s_rows[r] = n[e];
      s_off[r] = (int)min(at_back, (int64_t)1 << 30);
      at_back += had[e] - s_left[r];
    }
  }
  const int count = max(0, min(*S.free_count, S.pages));
  __syncthreads();

  // (Pages of broken tables past the list's room are dropped.)
  const int room = (int)min(back, (int64_t)(S.pages - count));
  for (int i = tid; i < (int)min(back, (int64_t)1 << 30); i += kThreads) {
    const int r = last_at_most(s_off, R, i);
    int32_t* entry = S.table + (int64_t)r * S.capacity + s_left[r] + (i - s_off[r]);
    if (i < room) S.free_pages[count + room - 1 - i] = *entry;
    *entry = -1;
  }
  const int available = count + room;
  __syncthreads();

  // Pages to take. a: rows that get a place, refused requests have none.
  int a[kPer], need[kPer];
  int64_t sum_need = 0;
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    const int r = tid * kPer + e;
    a[e] = need[e] = 0;
    if (r < R) {
      a[e] = n[e];
      if (S.keep) {
        const int first = s_first[r], end = first + n[e];
        const int kept = first < S.total ? S.positions[first] : all_kept;
        a[e] = (end < S.total ? S.positions[end] : all_kept) - kept;
        s_kept[r] = kept;
      }
      const int64_t want = ((int64_t)base[e] + a[e] + page - 1) >> S.page_shift;
      if (want > S.capacity) a[e] = -1;
      else need[e] = (int)want - s_left[r];
      sum_need += need[e];
    }
  }
  int64_t at_need = block_scan(sum_need, s_scan, &total);
  int64_t cost = 0, blocks = 0, taken = 0;
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    const int r = tid * kPer + e;
    if (r < R) {
      s_off[r] = (int)min(at_need, (int64_t)available);
      at_need += need[e];
      if (need[e] > 0 && at_need > available) a[e] = -1;
      else taken += need[e];
      // (Behind a refused request no other takes pages: the flat index below ends at what is taken.)
      if (a[e] < 0) {
        a[e] = 0;
        s_rows[r] = -1 - n[e];
      }
      S.lengths[r] = base[e] + a[e];
      if (S.plan.words) {
        const int64_t rows = s_rows[r] > 0 ? (int64_t)s_rows[r] * S.G : 0;
        blocks += (rows + kPagedRows - 1) / kPagedRows;
        cost += (int64_t)(base[e] + a[e]) * ((rows + kPagedRows - 1) / kPagedRows);
      }
    }
  }
  block_scan(taken, s_scan, &total);
  const int took = (int)total;
  __syncthreads();
  if (tid == 0) *S.free_count = available - took;
  for (int i = tid; i < took; i += kThreads) {
    const int r = last_at_most(s_off, R, i);
    S.table[(int64_t)r * S.capacity + s_left[r] + (i - s_off[r])] = S.free_pages[available - 1 - i];
  }
  __syncthreads();

  // The rows' places.
  if (S.total <= kInOne || S.keep) {
    for (int m = tid; m < S.total; m += kThreads) {
      int slot = -1, position = -1, request = -1;
      const int r = R > 0 ? last_at_most(s_first, R, m) : 0;
      if (R > 0 && m - s_first[r] < s_rows[r] && (!S.keep || S.keep[m])) {
        request = r;
        position = s_base[r] + (S.keep ? S.positions[m] - s_kept[r] : m - s_first[r]);
        slot = slot_of(S, r, position);
      }
      place(S, m, slot, position, request);
    }
  }
  if (!S.plan.words) return;

  // The attention's splits: as many tokens each as leave S.splits in all (a request of several row blocks counts as often). Every
  // request ends in a split that is not full; where those are few, their number is taken off, so that the splits do not pass
  // S.splits by them (one workgroup more than the GPU holds at once takes as long again).
  block_scan(cost, s_scan, &total);
  int64_t all_blocks;
  block_scan(blocks, s_scan, &all_blocks);
  const int64_t aim = S.splits > 2 * all_blocks ? S.splits - all_blocks : S.splits;
  const int64_t chunk = max((int64_t)kPagedUnit, ((total + aim - 1) / aim + kPagedUnit - 1) / kPagedUnit * kPagedUnit);
  PagedRequest q[kPer];
  int64_t sum_splits = 0, sum_part = 0;
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    const int r = tid * kPer + e;
    q[e] = {0, 0, 0, kPagedUnit, 0, 0, {0, 0}};
    if (r < R) {
      q[e].first = s_first[r];
      q[e].rows = max(0, s_rows[r]);
      q[e].length = base[e] + a[e];
      if (q[e].rows > 0) {
        const int64_t pieces = (q[e].length + chunk - 1) / chunk;
        q[e].per = (int)(((q[e].length + pieces - 1) / pieces + kPagedUnit - 1) / kPagedUnit * kPagedUnit);
        q[e].splits = (q[e].length + q[e].per - 1) / q[e].per;
      }
      sum_splits += q[e].splits;
      sum_part += q[e].splits > 1 ? (int64_t)q[e].splits * q[e].rows : 0;
    }
  }
  int64_t at_part = block_scan(sum_part, s_scan, &total);
  int64_t at_splits = block_scan(sum_splits, s_scan, &total);
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    const int r = tid * kPer + e;
    if (r < R) {
      q[e].part = (int)at_part;
      S.plan.requests()[r] = q[e];
      at_part += q[e].splits > 1 ? (int64_t)q[e].splits * q[e].rows : 0;
      s_off[r] = (int)at_splits;
      at_splits += q[e].splits;
    }
  }
  if (tid == 0) S.plan.words[0] = (int)total;
  __syncthreads();
  for (int i = tid; i < (int)total; i += kThreads) {
    const int r = last_at_most(s_off, R, i), split = i - s_off[r];
    const PagedRequest& t = S.plan.requests()[r];
    S.plan.items()[i] = {r, t.first, t.rows, t.length, split * t.per, min(t.length, (split + 1) * t.per),
                         t.splits > 1 ? t.part + split * t.rows : -1, 0};
  }
}

// The places of many rows, from the plan.
__global__ __launch_bounds__(kThreads) void cache_rows_kernel(CacheStepParams S) {
  __shared__ int s_first[kMaxRequests];
  for (int r = threadIdx.x; r < S.R; r += kThreads) s_first[r] = S.plan.requests()[r].first;
  __syncthreads();
  const int m = blockIdx.x * kThreads + threadIdx.x;
  if (m >= S.total) return;
  int slot = -1, position = -1, request = -1;
  if (S.R > 0) {
    const int r = last_at_most(s_first, S.R, m), n = S.plan.requests()[r].rows;
    if (m - s_first[r] < n) {
      request = r;
      position = S.plan.requests()[r].length - n + (m - s_first[r]);
      slot = slot_of(S, r, position);
    }
  }
  place(S, m, slot, position, request);
}

}  // namespace

hipError_t launch_cache_step(const CacheStepParams& p, hipStream_t stream) {
  hipLaunchKernelGGL(cache_step_kernel, dim3(1), dim3(kThreads), 0, stream, p);
  if (p.total > kInOne && !p.keep)
    hipLaunchKernelGGL(cache_rows_kernel, dim3((p.total + kThreads - 1) / kThreads), dim3(kThreads), 0, stream, p);
  return hipGetLastError();
}

}  // namespace qmm4
