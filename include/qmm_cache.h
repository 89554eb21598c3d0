/*
 * C ABI of the paged key-value cache (libqmm4.so): what lies between a layer's attention inputs and its tail in a batched
 * decode or tree-verify step (src/mlx_tree_spec/tree_verify.py:311-402).
 *
 * A cache is a pool of pages of `page_size` tokens (a power of two from 16 to 1024). A request's tokens lie in the pages
 * that its row of block_table names, in order; slot s is token s % page_size of page s / page_size. The pages' free list,
 * block tables and lengths live on the GPU and belong to all layers; each layer has its own keys and values:
 *   keys    [pages, Hk, D / E, page_size, E]      values [pages, Hk, page_size / E, D, E]
 * with E = 8 for bf16 and E = 16 for 8-bit codes (int8), whose scales are fp32 [pages, Hk, page_size] for keys and for
 * values: a value is code * scale. (16 bytes of either are an operand of the matrix instruction as they lie.)
 *
 * Conventions as in qmm4.h: device pointers on the current device, bf16 arrays as raw 16-bit words, work enqueued on
 * `hip_stream`, 0 or a negative QMM4_ERR_* code with its message in qmm4_last_error(). A workspace is the caller's (16-byte
 * aligned, of at least the bytes that the function for it names, not in use by another call at the same time); its content
 * need not be kept or cleared between calls.
 */
#ifndef MI355X_QMM_CACHE_H
#define MI355X_QMM_CACHE_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define QMM4_CACHE_MAX_REQUESTS 2048
#define QMM4_CACHE_MAX_ROWS (1 << 22)
#define QMM4_CACHE_MAX_KEEP (1 << 16)

/*
 * One step of the tables. For request r of R, with page = page_size:
 *   b = base[r] (null: lengths[r]) within 0 .. lengths[r];   n = rows[r] within 0 .. max_rows, cut where the n so far reach
 *   `total`: the request's rows lie behind the n of each request before it (so max_rows has to be at least every one's rows);
 *   a = n, or those of the n with keep != 0.
 * Every request gives back its pages past ceil(b / page) (their entries of block_table become -1); then pages for
 * ceil((b + a) / page) are taken from the end of the free list in the order of requests, so that pages given back and taken
 * again by the same requests are the same ones. A request whose tokens would not fit its row of block_table is refused, and so
 * is every one that needs pages from the first on for which too few are left: a refused one has a = 0.
 *   lengths[r] becomes b + a; the k-th of its a rows gets position b + k, its slot, and request r; rows without a place
 *   (not kept, refused, behind the last request) get -1 in all three.
 *   lengths, rows, base: int32 [R]; block_table: int32 [R, capacity]; free_pages: int32 [pages] (room for every page of the
 *   cache), whose first free_count[0] are free; keep: one byte per row [total], or null; slots, positions, request: int32 [total].
 *   plan: int32 [qmm4_cache_plan_words(..)] for qmm4_paged_attention_bf16 on this step, 16-byte aligned, or null where no
 *   attention follows (with keep none is made).
 *   Requires R <= QMM4_CACHE_MAX_REQUESTS, total <= QMM4_CACHE_MAX_ROWS (with keep QMM4_CACHE_MAX_KEEP), max_rows >= 0, capacity
 *   <= 2^22, pages * page_size and capacity * page_size <= 2^30, heads % kv_heads == 0, heads <= 1024. Numbers in the tables
 *   that cannot be (lengths past the table, a count past the list) are taken as the nearest that can.
 */
int64_t qmm4_cache_plan_words(int64_t R, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t max_rows);
int qmm4_cache_step(int32_t* lengths, int32_t* block_table, int32_t* free_pages, int32_t* free_count, const int32_t* rows,
                    const int32_t* base, const uint8_t* keep, int32_t* slots, int32_t* positions, int32_t* request,
                    int32_t* plan, int64_t R, int64_t capacity, int64_t pages, int64_t total, int64_t max_rows,
                    int64_t page_size, int64_t heads, int64_t kv_heads, int64_t head_dim, void* hip_stream);

/*
 * New keys and values into the cache: row m at slots[m]; rows whose slot lies outside 0 .. pages * page_size - 1 are
 * skipped. Slots of different rows have to differ. 8 bits: scale = max |x| / 127 over a row's head, code = x / scale
 * rounded to the nearest (even); a head of zeros has scale 0, one with an infinity or NaN stands for NaN throughout.
 *   k, v: bf16, element (m, h, d) at k[m * k_row + h * k_head + d] (strides in elements, multiples of 8, k and v 16-byte
 *   aligned); slots: int32 [M]. bits: 16 (keys and values bf16, scales null) or 8.
 *   Requires D in 64, 96, 128, 192, 256 (8 bits: not 96), Hk <= 1024, M <= QMM4_CACHE_MAX_ROWS, pages * page_size <= 2^30,
 *   keys and values 16-byte aligned.
 */
int qmm4_store_kv_bf16(const void* k, int64_t k_row, int64_t k_head, const void* v, int64_t v_row, int64_t v_head,
                       const int32_t* slots, void* keys, void* values, float* key_scales, float* value_scales, int64_t M,
                       int64_t Hk, int64_t D, int64_t pages, int64_t page_size, int bits, void* hip_stream);

/*
 * Attention of a step's rows over their requests' cached tokens, the step's own (stored before) among them:
 *   out[m, h] = sum_t p_t values[t, h / G],   p = softmax over the visible t of scale * q[m, h] . keys[t, h / G],  G = Hq / Hk
 * times sigmoid(gate[m, h]) where gate is not null. Row i of a request of n rows and length L sees its tokens t < L - n, and
 * token L - n + j of the step where j <= i, or, with ancestors, where j < 64 and bit j of ancestors[row] is set (its own bit too).
 * Rows that see nothing, and rows without a request, give zeros. What is not finite in a token that a row does not see does not
 * reach it. Products and sums are fp32, probabilities are rounded to bf16 for their product with the values (8 bits: with
 * the scale in them), the result is rounded once. No sum of finite values overflows, whatever their size; probabilities below
 * 2^-117 capacity page_size of a row's largest may count as zero.
 *   q, gate: bf16 with strides as for k above; out: bf16 [M, Hq, D] contiguous, overlapping no input; block_table, request,
 *   plan: those of qmm4_cache_step, made with the same R, total = M, heads, kv_heads, D and max_rows on this device;
 *   ancestors: int64 [M] or null. Requires D as above, Hq % Hk == 0, scale finite.
 */
int64_t qmm4_paged_workspace(int64_t M, int64_t R, int64_t Hq, int64_t Hk, int64_t D, int64_t max_rows);
int qmm4_paged_attention_bf16(const void* q, int64_t q_row, int64_t q_head, const void* keys, const void* values,
                              const float* key_scales, const float* value_scales, const int32_t* block_table,
                              const int32_t* request, const int32_t* plan, const int64_t* ancestors, const void* gate,
                              int64_t gate_row, int64_t gate_head, void* out, void* workspace, float scale, int64_t M,
                              int64_t R, int64_t Hq, int64_t Hk, int64_t D, int64_t pages, int64_t page_size,
                              int64_t capacity, int64_t max_rows, int bits, void* hip_stream);

#ifdef __cplusplus
}
#endif

#endif /* MI355X_QMM_CACHE_H */
