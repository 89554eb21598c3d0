// C ABI of the paged key-value cache (declared in include/qmm_cache.h): argument checks and launches.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <exception>
#include <mutex>

#include "qmm4.h"
#include "qmm4_dispatch.h"
#include "qmm_cache.h"
#include "qmm_cache_kernels.h"

namespace {

using qmm4::hip_error;
using qmm4::set_error;

bool aligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

// No exception leaves a C entry point.
template <class F>
int guarded(F&& f) {
  try {
    qmm4::clear_error();
    return f();
  } catch (const std::exception&) {
    return QMM4_ERR_NOMEM;
  }
}

int current_cus(int* cus) {
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return hip_error(e, "hipGetDevice");
  std::lock_guard<std::mutex> lock(qmm4::api_mutex());
  qmm4::DeviceInfo* di = nullptr;
  if (int rc = qmm4::device_info(dev, &di)) return rc;
  *cus = qmm4::device_cus(di);
  return QMM4_OK;
}

int64_t clamp_rows(int64_t max_rows) { return max_rows < QMM4_CACHE_MAX_ROWS ? max_rows : QMM4_CACHE_MAX_ROWS; }

int check_pages(int64_t pages, int64_t page_size, int64_t capacity) {
  if (page_size < 16 || page_size > 1024 || (page_size & (page_size - 1)) != 0)
    return set_error(QMM4_ERR_INVALID, "page_size=%lld must be a power of two from 16 to 1024", (long long)page_size);
  const int64_t most = (1LL << 30) / page_size;
  if (pages < 0 || capacity < 0 || pages > most || capacity > most)
    return set_error(QMM4_ERR_INVALID, "%lld pages, %lld per request, of %lld tokens: up to 2^30 tokens are supported",
                     (long long)pages, (long long)capacity, (long long)page_size);
  return QMM4_OK;
}

int check_heads(int64_t heads, int64_t kv_heads) {
  if (heads < 1 || heads > 1024 || kv_heads < 1 || heads % kv_heads != 0)
    return set_error(QMM4_ERR_INVALID, "%lld query heads and %lld key heads: the first must be a multiple of the second, at most 1024",
                     (long long)heads, (long long)kv_heads);
  return QMM4_OK;
}

int check_requests(int64_t R, int64_t rows, int64_t max_rows) {
  if (R < 0 || R > QMM4_CACHE_MAX_REQUESTS || rows < 0 || rows > QMM4_CACHE_MAX_ROWS || max_rows < 0)
    return set_error(QMM4_ERR_INVALID, "%lld requests, %lld rows, at most %lld each: up to %d requests and %d rows are supported",
                     (long long)R, (long long)rows, (long long)max_rows, QMM4_CACHE_MAX_REQUESTS, QMM4_CACHE_MAX_ROWS);
  return QMM4_OK;
}

// The most rows of a request, where their query rows to a key head can be counted.
int check_query_rows(int64_t heads, int64_t kv_heads, int64_t max_rows) {
  if (clamp_rows(max_rows) * (heads / kv_heads) > (1LL << 30))
    return set_error(QMM4_ERR_INVALID, "up to %lld rows of a request of %lld query heads to a key head: up to 2^30 of both are supported",
                     (long long)max_rows, (long long)(heads / kv_heads));
  return QMM4_OK;
}

int check_format(int64_t D, int bits, const float* key_scales, const float* value_scales) {
  if (bits != 16 && bits != 8) return set_error(QMM4_ERR_UNSUPPORTED, "bits=%d: caches of 16 (bf16) or 8 bits are supported", bits);
  if (D != 64 && D != 96 && D != 128 && D != 192 && D != 256)
    return set_error(QMM4_ERR_UNSUPPORTED, "heads of %lld values: 64, 96, 128, 192 and 256 are supported", (long long)D);
  if (bits == 8 && D == 96) return set_error(QMM4_ERR_UNSUPPORTED, "heads of 96 values: not in a cache of 8 bits");
  if ((bits == 8) != (key_scales != nullptr) || (bits == 8) != (value_scales != nullptr))
    return set_error(QMM4_ERR_INVALID, "a cache of 8 bits has scales for keys and values, one of bf16 has none");
  if (!aligned(key_scales, 16) || !aligned(value_scales, 16)) return set_error(QMM4_ERR_INVALID, "scales must be 16-byte aligned");
  return QMM4_OK;
}

int rows_ok(const void* x, int64_t row, int64_t head, const char* what) {
  if (!aligned(x, 16) || row % 8 != 0 || head % 8 != 0)
    return set_error(QMM4_ERR_INVALID, "%s must be 16-byte aligned with strides that are multiples of 8", what);
  return QMM4_OK;
}

int log2_of(int64_t v) {
  int s = 0;
  while ((1LL << s) < v) ++s;
  return s;
}

int shape_of(int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t max_rows, qmm4::PagedShape* out) {
  int cus = 0;
  if (int rc = current_cus(&cus)) return rc;
  *out = qmm4::paged_shape(heads, kv_heads, head_dim, max_rows, cus);
  return QMM4_OK;
}

qmm4::CacheRows rows_of(const void* x, int64_t row, int64_t head) { return {static_cast<const uint16_t*>(x), row, head}; }

}  // namespace

extern "C" {

int64_t qmm4_cache_plan_words(int64_t R, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t max_rows) {
  int64_t words = 0;
  const int rc = guarded([&] {
    if (int bad = check_heads(heads, kv_heads)) return bad;
    if (int bad = check_requests(R, 0, max_rows)) return bad;
    if (int bad = check_query_rows(heads, kv_heads, max_rows)) return bad;
    qmm4::PagedShape s;
    if (int bad = shape_of(heads, kv_heads, head_dim, clamp_rows(max_rows), &s)) return bad;
    words = qmm4::CachePlan::kHead + qmm4::CachePlan::kRecord * (2 * R + s.splits);
    return (int)QMM4_OK;
  });
  return rc ? rc : words;
}

int qmm4_cache_step(int32_t* lengths, int32_t* block_table, int32_t* free_pages, int32_t* free_count, const int32_t* rows,
                    const int32_t* base, const uint8_t* keep, int32_t* slots, int32_t* positions, int32_t* request,
                    int32_t* plan, int64_t R, int64_t capacity, int64_t pages, int64_t total, int64_t max_rows,
                    int64_t page_size, int64_t heads, int64_t kv_heads, int64_t head_dim, void* hip_stream) {
  return guarded([&] {
    if (int rc = check_pages(pages, page_size, capacity)) return rc;
    if (int rc = check_heads(heads, kv_heads)) return rc;
    if (int rc = check_requests(R, total, max_rows)) return rc;
    if (int rc = check_query_rows(heads, kv_heads, max_rows)) return rc;
    if (capacity > (1LL << 22))
      return set_error(QMM4_ERR_INVALID, "%lld pages per request: up to 2^22 are supported", (long long)capacity);
    if (keep && total > QMM4_CACHE_MAX_KEEP)
      return set_error(QMM4_ERR_INVALID, "%lld rows with keep: up to %d are supported", (long long)total, QMM4_CACHE_MAX_KEEP);
    if (R == 0 && total == 0 && !plan) return (int)QMM4_OK;
    if ((R > 0 && (!lengths || !rows || (capacity > 0 && !block_table))) || !free_count || (pages > 0 && !free_pages) ||
        (total > 0 && (!slots || !positions || !request)))
      return set_error(QMM4_ERR_INVALID, "null pointer argument");
    if (!aligned(plan, 16)) return set_error(QMM4_ERR_INVALID, "plan must be 16-byte aligned");
    for (const void* p : {(const void*)lengths, (const void*)block_table, (const void*)free_pages, (const void*)free_count,
                          (const void*)rows, (const void*)base, (const void*)slots, (const void*)positions,
                          (const void*)request})
      if (!aligned(p, 4)) return set_error(QMM4_ERR_INVALID, "tables must be aligned to their elements");
    qmm4::PagedShape s;
    const int64_t most = clamp_rows(max_rows);
    if (int rc = shape_of(heads, kv_heads, head_dim, most, &s)) return rc;
    const qmm4::CacheStepParams p{lengths, block_table, free_pages, free_count, rows, base, keep, slots, positions, request,
                                  {keep ? nullptr : plan, (int)R}, capacity, (int)R, (int)pages, (int)total, (int)most,
                                  log2_of(page_size), s.G, s.round, s.splits};
    const hipError_t e = qmm4::launch_cache_step(p, static_cast<hipStream_t>(hip_stream));
    if (e != hipSuccess) return hip_error(e, "cache table kernel launch");
    return (int)QMM4_OK;
  });
}

int qmm4_store_kv_bf16(const void* k, int64_t k_row, int64_t k_head, const void* v, int64_t v_row, int64_t v_head,
                       const int32_t* slots, void* keys, void* values, float* key_scales, float* value_scales, int64_t M,
                       int64_t Hk, int64_t D, int64_t pages, int64_t page_size, int bits, void* hip_stream) {
  return guarded([&] {
    if (int rc = check_format(D, bits, key_scales, value_scales)) return rc;
    if (int rc = check_pages(pages, page_size, 0)) return rc;
    if (int rc = check_heads(Hk, Hk)) return rc;
    if (int rc = check_requests(0, M, 0)) return rc;
    if (M == 0 || pages == 0) return (int)QMM4_OK;
    if (!k || !v || !slots || !keys || !values) return set_error(QMM4_ERR_INVALID, "null pointer argument");
    if (int rc = rows_ok(k, k_row, k_head, "k")) return rc;
    if (int rc = rows_ok(v, v_row, v_head, "v")) return rc;
    if (!aligned(keys, 16) || !aligned(values, 16) || !aligned(slots, 4))
      return set_error(QMM4_ERR_INVALID, "keys and values must be 16-byte aligned, slots to their elements");
    const qmm4::CacheArrays cache{keys, values, key_scales, value_scales, pages, log2_of(page_size), (int)Hk};
    const hipError_t e = qmm4::launch_store_kv(rows_of(k, k_row, k_head), rows_of(v, v_row, v_head), slots, cache, M, (int)D,
                                               bits == 8, static_cast<hipStream_t>(hip_stream));
    if (e != hipSuccess) return hip_error(e, "cache store kernel launch");
    return (int)QMM4_OK;
  });
}

int64_t qmm4_paged_workspace(int64_t M, int64_t R, int64_t Hq, int64_t Hk, int64_t D, int64_t max_rows) {
  int64_t bytes = 0;
  const int rc = guarded([&] {
    if (int bad = check_heads(Hq, Hk)) return bad;
    if (int bad = check_requests(R, M, max_rows)) return bad;
    if (int bad = check_query_rows(Hq, Hk, max_rows)) return bad;
    if (int bad = check_format(D, 16, nullptr, nullptr)) return bad;
    qmm4::PagedShape s;
    if (int bad = shape_of(Hq, Hk, D, clamp_rows(max_rows), &s)) return bad;
    bytes = std::max<int64_t>(16, qmm4::paged_partial_rows(s, R, clamp_rows(max_rows)) * Hk * (D + 2) * (int64_t)sizeof(float));
    return (int)QMM4_OK;
  });
  return rc ? rc : bytes;
}

int qmm4_paged_attention_bf16(const void* q, int64_t q_row, int64_t q_head, const void* keys, const void* values,
                              const float* key_scales, const float* value_scales, const int32_t* block_table,
                              const int32_t* request, const int32_t* plan, const int64_t* ancestors, const void* gate,
                              int64_t gate_row, int64_t gate_head, void* out, void* workspace, float scale, int64_t M,
                              int64_t R, int64_t Hq, int64_t Hk, int64_t D, int64_t pages, int64_t page_size,
                              int64_t capacity, int64_t max_rows, int bits, void* hip_stream) {
  return guarded([&] {
    if (int rc = check_format(D, bits, key_scales, value_scales)) return rc;
    if (int rc = check_pages(pages, page_size, capacity)) return rc;
    if (int rc = check_heads(Hq, Hk)) return rc;
    if (int rc = check_requests(R, M, max_rows)) return rc;
    if (int rc = check_query_rows(Hq, Hk, max_rows)) return rc;
    if (!std::isfinite(scale)) return set_error(QMM4_ERR_INVALID, "scale must be finite");
    if (M == 0) return (int)QMM4_OK;
    if (!q || !keys || !values || !request || !plan || !out || !workspace || (R > 0 && !block_table))
      return set_error(QMM4_ERR_INVALID, "null pointer argument");
    if (int rc = rows_ok(q, q_row, q_head, "q")) return rc;
    if (int rc = rows_ok(gate, gate_row, gate_head, "gate")) return rc;
    if (!aligned(keys, 16) || !aligned(values, 16) || !aligned(out, 16) || !aligned(workspace, 16) || !aligned(block_table, 4) ||
        !aligned(request, 4) || !aligned(plan, 16) || !aligned(ancestors, 8))
      return set_error(QMM4_ERR_INVALID, "keys, values, out and workspace must be 16-byte aligned, tables to their elements");
    if (pages == 0 || capacity == 0)
      return set_error(QMM4_ERR_INVALID, "a cache without pages has nothing to attend to");
    const int64_t most = clamp_rows(max_rows);
    qmm4::PagedShape s;
    if (int rc = shape_of(Hq, Hk, D, most, &s)) return rc;
    float* part = static_cast<float*>(workspace);
    const int64_t rows = qmm4::paged_partial_rows(s, R, most) * Hk;
    const qmm4::PagedParams p{rows_of(q, q_row, q_head), rows_of(gate, gate_row, gate_head),
                              {const_cast<void*>(keys), const_cast<void*>(values), const_cast<float*>(key_scales),
                               const_cast<float*>(value_scales), pages, log2_of(page_size), (int)Hk},
                              block_table, request, {const_cast<int32_t*>(plan), (int)R}, ancestors,
                              static_cast<uint16_t*>(out), part, part + rows * D, (int32_t)capacity, scale,
                              (float)log2_of(capacity * page_size), s.G, (int)most, (int)(s.splits + R)};
    const hipError_t e = qmm4::launch_paged_attention(p, M, (int)D, bits == 8, static_cast<hipStream_t>(hip_stream));
    if (e != hipSuccess) return hip_error(e, "paged attention kernel launch");
    return (int)QMM4_OK;
  });
}

}  // extern "C"
