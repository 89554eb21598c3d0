/*
 * C ABI of the per-request operators of a batched step (libqmm4.so): what differs from request to request
 * beside the shared quantized projections of qmm4.h.
 *
 * A step concatenates the rows of several requests (src/mlx_tree_spec/tree_verify.py:414-447) and runs each
 * projection once over all of them. These take each row's own adapter, position or sampling settings.
 *
 * Conventions as in qmm4.h: device pointers on the current device, bf16 arrays as raw 16-bit words, work
 * enqueued on `hip_stream`, 0 or a negative QMM4_ERR_* code with its message in qmm4_last_error(). A workspace
 * is the caller's (16-byte aligned, of at least the bytes the _workspace function names, not in use by another
 * call at the same time); its content need not be kept or cleared between calls.
 */
#ifndef MI355X_QMM_REQUESTS_H
#define MI355X_QMM_REQUESTS_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Largest rank of an adapter, head width and vocabulary below. */
#define QMM4_LORA_MAX_RANK 256
#define QMM4_HEAD_MAX_DIM 512
#define QMM4_SAMPLE_MAX_VOCAB (1 << 24)

/*
 * y[m] = x[m] dequant(w)^T + scale[a] * (x[m] A[a]^T) B[a]^T for a = adapters[m]: a shared quantized projection with
 * each row's low-rank adapter. Rows whose adapter lies outside 0 .. L - 1 (-1 by convention) have the projection alone,
 * with its bits.
 *   x, w, scales, biases, y and their requirements: those of qmm4_affine_bf16 (bits 4, group_size 64, K % 128 == 0,
 *   N % 16 == 0), else of qmm_affine_general_bf16; lora_a: bf16 [L, R, K]; lora_b: bf16 [L, N, R]; lora_scale: fp32
 *   [L]; adapters: int32 or int64 [M] (adapter_bits 32 or 64).
 *   The sums of both products are fp32 and rounded once; between its factors the second one is kept (in `workspace`) to
 *   2^-18 of its value. What is not finite in x, lora_a or lora_b gives what the formula gives, in the rows that use
 *   it and in no other (an infinite lora_scale: infinities or NaN in its rows). Requires R % 8 == 0, 8 <= R <= QMM4_LORA_MAX_RANK, L <= 2^30, M <= 2^26, lora_a,
 *   lora_b and workspace 16-byte aligned, lora_scale 4-byte, adapters by their own size. M == 0 or N == 0 is a no-op.
 *   Deterministic.
 */
int64_t qmm4_lora_workspace(int64_t M, int64_t R);
int qmm4_affine_lora_bf16(const void* x, const uint32_t* w, const void* scales, const void* biases,
                          const void* lora_a, const void* lora_b, const float* lora_scale, const void* adapters,
                          int adapter_bits, void* y, void* workspace, int64_t M, int64_t N, int64_t K, int64_t L,
                          int64_t R, int group_size, int bits, int transpose, void* hip_stream);

/*
 * y[m] += scale[a] * (x[m] A[a]^T) B[a]^T in place, for a projection that ran elsewhere: the same arguments (K % 8 == 0,
 * any N, M <= 2^26, each other at most 2^30), y added to in fp32 and rounded again. L == 0 is a no-op.
 */
int qmm4_lora_add_bf16(const void* x, const void* lora_a, const void* lora_b, const float* lora_scale,
                       const void* adapters, int adapter_bits, void* y, void* workspace, int64_t M, int64_t N,
                       int64_t K, int64_t L, int64_t R, void* hip_stream);

/*
 * The RMS norms of the query and key heads and their rotation at each row's position, in one pass: the step
 * between the q/k projections and attention (src/mlx_tree_spec/tree_verify.py:311-328). Per head of D values
 *   n = x / sqrt(mean(x^2) + eps) * weight,   angle_i = positions[m] * inv_freq[i], i < P,
 *   (n[i], n[i + P]) -> (n[i] cos - n[i + P] sin, n[i + P] cos + n[i] sin)       (interleaved: n[2i], n[2i + 1])
 * and n past 2 P unrotated; fp32 throughout (squares too: a sum of squares past 2^128 gives zeros, a mean square
 * under 2^-126 beside eps 0 is lost; angles reduced in 64 bits), one rounding to bf16.
 *   q: bf16, element (m, h, d) at q[m * q_row + h * q_head + d], k alike (strides in elements, multiples of 8);
 *   q_weight, k_weight: bf16 [D]; positions: int32 or int64 [M]; inv_freq: fp32 or fp64 [P]; q_out: bf16
 *   [M, Hq, D], k_out: bf16 [M, Hk, D], contiguous, overlapping no input.
 *   Requires D % 8 == 0, D <= QMM4_HEAD_MAX_DIM, 0 <= 2 P <= D, eps finite and >= 0, M <= 2^30, Hq + Hk <= 65536,
 *   q, k, weights and outputs 16-byte aligned. M == 0 or no heads: a no-op; either head count may be 0.
 */
int qmm4_qk_norm_rope_bf16(const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row, int64_t k_head,
                           const void* q_weight, const void* k_weight, float eps, const void* positions,
                           int position_bits, const void* inv_freq, int freq_bits, void* q_out, void* k_out,
                           int64_t M, int64_t Hq, int64_t Hk, int64_t D, int64_t P, int interleaved,
                           void* hip_stream);

/*
 * The next token of each row from its logits and a random number in [0, 1). With w = exp((l - max l) / T), in
 * the order of falling logits (equal ones by index):
 *   kept = the first top_k; of them the shortest prefix whose mass reaches top_p of theirs; of them those with
 *   w >= min_p; at least the first.   token = the first kept one whose cumulative mass exceeds u * the kept mass.
 * logprobs: log(w / kept mass) of the token. Masses are held in 64 bits.
 *   logits: bf16, row m at logits + m * row_stride (elements); uniform: fp32 [M]; tokens: int64 [M]; logprobs:
 *   fp32 [M]. temperature, top_p, min_p fp32 [M] and top_k int32 [M], each a device array or null: then the
 *   value behind it holds for every row. temperature <= 0 or NaN: the first of the order; top_k <= 0, top_p >= 1
 *   or NaN, min_p <= 0 or NaN: off. NaN logits count as -infinity; a row with nothing above it: token -1,
 *   log probability -infinity. u outside [0, 1) (or NaN) is taken as its nearest end (NaN: 0).
 *   Requires 1 <= V <= QMM4_SAMPLE_MAX_VOCAB, M <= 2^20, row_stride >= V (M > 1), logits 2-byte, fp32 and int32
 *   arrays 4-byte, tokens 8-byte aligned. Deterministic.
 */
/* On the current device, at most 1025 MiB (4 bytes a logit up to there); negative: an error code. */
int64_t qmm4_sample_workspace(int64_t M, int64_t V);
int qmm4_sample_bf16(const void* logits, int64_t M, int64_t V, int64_t row_stride, const float* uniform,
                     const float* temperature, float temperature_value, const int32_t* top_k, int32_t top_k_value,
                     const float* top_p, float top_p_value, const float* min_p, float min_p_value, int64_t* tokens,
                     float* logprobs, void* workspace, void* hip_stream);

#ifdef __cplusplus
}
#endif

#endif /* MI355X_QMM_REQUESTS_H */
