// Launch interface of the paged key-value cache (include/qmm_cache.h) between its C ABI and kernels.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace qmm4 {

// Query rows (rows of the step x query heads of a key head) of one workgroup of the attention.
constexpr int kPagedRows = 128;
// Tokens at which a request's cache may be cut into splits.
constexpr int kPagedUnit = 64;

// The plan of a step's attention: 8 words (the first: how many items there are), then arrays of R, then the items. Item: one
// split of one request's tokens, for every key head.
struct CachePlan {
  int32_t* words;
  int R;
  __host__ __device__ int32_t* first() const { return words + 8; }                 // first row
  __host__ __device__ int32_t* count() const { return words + 8 + (int64_t)R; }    // rows
  __host__ __device__ int32_t* length() const { return words + 8 + 2 * (int64_t)R; }  // tokens, the rows among them
  __host__ __device__ int32_t* per() const { return words + 8 + 3 * (int64_t)R; }     // tokens of a split
  __host__ __device__ int32_t* part() const { return words + 8 + 4 * (int64_t)R; }    // first partial row
  __host__ __device__ int32_t* items() const { return words + 8 + 5 * (int64_t)R; }   // (request, split)
};

// How a step's attention is cut: at most `splits` + R items.
struct PagedShape {
  int G;           // query heads of a key head
  int64_t splits;  // pieces of the whole that are aimed at, for each key head
};
PagedShape paged_shape(int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t max_rows, int cus);
// Query rows of all partial results, for each key head, at most.
int64_t paged_partial_rows(const PagedShape& s, int64_t M, int64_t R, int64_t max_rows);

struct CacheStepParams {
  int32_t *lengths, *table, *free_pages, *free_count;
  const int32_t *rows, *base;
  const uint8_t* keep;
  int32_t *slots, *positions, *request;
  CachePlan plan;  // (words null: none)
  int64_t capacity;
  int R, pages, total, max_rows, page_shift, G;
  int64_t splits;
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
  float *part, *part_ml;  // partial sums [rows, Hq, D]; their largest logit and sum of exponentials [rows, Hq, 2]
  int64_t capacity;
  float scale;
  int G, max_rows;
};
hipError_t launch_paged_attention(const PagedParams& p, int64_t M, const PagedShape& shape, int D, bool q8, hipStream_t stream);

}  // namespace qmm4
