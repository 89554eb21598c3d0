// Launch interface of the paged key-value cache (include/qmm_cache.h) between its C ABI and kernels.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace qmm4 {

// Query rows (rows of the step x query heads of a key head) of one workgroup of the attention.
constexpr int kPagedRows = 128;
// How far (in powers of two) a logit may pass the largest one before it without moving the running maximum.
constexpr int kPagedSlack = 8;
// Tokens at which a request's cache may be cut into splits.
constexpr int kPagedUnit = 64;

// The plan of a step's attention, in words: how many items there are (a block of 8), a record of each request, one of each
// item. An item is one split of one request's tokens, for every key head.
struct PagedRequest {
  int32_t first, rows;   // its rows of the step
  int32_t length;        // its tokens, the rows among them
  int32_t per, splits;   // tokens of a split; splits
  int32_t part;          // first partial row (of more than one split)
  int32_t unused[2];
};
struct PagedItem {
  int32_t request, first, rows, length;
  int32_t begin, end;  // its tokens
  int32_t part;        // its first partial row, or -1: it is the request's only one
  int32_t page;        // the page of its first token
};
struct CachePlan {
  int32_t* words;
  int R;
  static constexpr int kHead = 8, kRecord = 8;
  __host__ __device__ PagedRequest* requests() const { return reinterpret_cast<PagedRequest*>(words + kHead); }
  __host__ __device__ PagedItem* items() const { return reinterpret_cast<PagedItem*>(words + kHead + (int64_t)kRecord * R); }
};
static_assert(sizeof(PagedRequest) == CachePlan::kRecord * 4 && sizeof(PagedItem) == CachePlan::kRecord * 4, "records");

// How a step's attention is cut: at most `splits` + R items.
struct PagedShape {
  int G;           // query heads of a key head
  int64_t round;   // pieces for each key head whose workgroups the GPU holds at once
  int64_t splits;  // pieces of the whole that are aimed at, at most
};
PagedShape paged_shape(int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t max_rows, int cus);
// Query rows of all partial results (of requests that are cut), for each key head, at most.
int64_t paged_partial_rows(const PagedShape& s, int64_t R, int64_t max_rows);

struct CacheStepParams {
  int32_t *lengths, *table, *free_pages, *free_count;
  const int32_t *rows, *base;
  const uint8_t* keep;
  int32_t *slots, *positions, *request;
  CachePlan plan;  // (words null: none)
  int64_t capacity;
  int R, pages, total, max_rows, page_shift, G;
  int64_t round, splits;
};
hipError_t launch_cache_step(const CacheStepParams& p, hipStream_t stream);

// k or v, element (m, h, d) at x[m * row + h * head + d].
struct CacheRows {
  const uint16_t* x;
  int64_t row, head;
};
struct CacheArrays {
  void *keys, *values;
  float *key_scales, *value_scales;  // (8 bits)
  int64_t pages;
  int page_shift, heads;
};
hipError_t launch_store_kv(const CacheRows& k, const CacheRows& v, const int32_t* slots, const CacheArrays& cache, int64_t M,
                           int D, bool q8, hipStream_t stream);

struct PagedParams {
  CacheRows q, gate;  // (gate.x null: none)
  CacheArrays cache;
  const int32_t *table, *request;
  CachePlan plan;
  const int64_t* ancestors;
  uint16_t* out;
  float *part, *part_ml;  // partial sums [rows, Hq, D]; their running maximum and sum of exponentials [rows, Hq, 2]
  int32_t capacity;
  float scale;
  float tokens;  // that a request may have, as a power of two, rounded up
  int G, max_rows;
  int items;  // records of items in the plan
};
// (With the tile kernel's own two arguments three 64-byte lines: with a fourth, cold at its start, 4 x 16 nodes of 6 heads of 256 took
// 25.1 us in place of 24.7.)
static_assert(sizeof(PagedParams) <= 184, "arguments");
hipError_t launch_paged_attention(const PagedParams& p, int64_t M, int D, bool q8, hipStream_t stream);

}  // namespace qmm4
