/*
 * cruise_decoder.h -- C ABI of the decoder operators on device tensors: the
 * pieces of one decode step around the paged cache, for any number of rows and
 * any context length (cruise_decoder_step in cruise_epoch.h is the whole step
 * for the engine's four rows).
 *
 * Plain C types only.  Every pointer is caller-owned device memory on `device`,
 * every call queues its kernels on `stream` (a cudaStream_t; NULL is the legacy
 * default stream) and returns without waiting; calls may be captured into a
 * CUDA graph.  A call keeps no state: calls on different streams or threads
 * may overlap as long as what they write does not.  Nothing is allocated.
 * dtype: 0 bf16, 1 fp16, 2 fp32.  The current device of the calling thread is
 * left as it was.
 * Return 0, -1 for invalid arguments, or a CUDA error code;
 * cruise_decoder_last_error() explains both.
 */
#ifndef CRUISE_DECODER_H
#define CRUISE_DECODER_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Head norms, rotation and the paged store of `tokens` tokens in one pass.
 * qkv [tokens][(num_heads + 2 num_kv_heads) head_dim]: query heads, key heads,
 * value heads, rows qkv_stride elements apart; dtype 0 or 1; head_dim 64 or 128.
 * Per head of q and k: with q_norm and k_norm (both or neither, [head_dim] of
 * dtype) x / sqrt(mean(x^2) + eps) * norm; then the rotation of the first
 * `rotary` elements, x cos + rotate_half(x) sin, rotate_half swapping the
 * halves of the rotated part with the sign of the first reversed (rotary a
 * multiple of 16, at most head_dim).  rope_cos and rope_sin: [rope_rows][rotary]
 * of rope_dtype 0 or 2, the row of position[t].  fp32 arithmetic, one rounding.
 * Rotated q goes to q_out [tokens][num_heads head_dim] (rows q_stride elements
 * apart); rotated k and v to slot[t] of key_cache and value_cache,
 * [num_blocks][block_size][num_kv_heads][head_dim] with block_stride elements
 * between blocks.  A slot outside [0, num_blocks block_size) stores nothing; a
 * position outside [0, rope_rows) stores nothing and gives zeros in q_out.
 * Two tokens must not have the same slot (either's values may stay).
 * Pointers 16-byte aligned, strides multiples of 8 elements; q_out and the
 * caches must not overlap the inputs, nor q_out the caches (from first to last
 * byte), nor a block of one cache a block of the other (the blocks may
 * alternate). */
int32_t cruise_decoder_rotate_store(
    const void *qkv, int64_t qkv_stride, int32_t tokens, int32_t num_heads,
    int32_t num_kv_heads, int32_t head_dim, int32_t dtype,
    const int64_t *position, const int32_t *slot, const void *q_norm,
    const void *k_norm, float eps, const void *rope_cos, const void *rope_sin,
    int32_t rope_dtype, int32_t rope_rows, int32_t rotary, void *q_out,
    int64_t q_stride, void *key_cache, void *value_cache, int64_t num_blocks,
    int32_t block_size, int64_t block_stride, int32_t device, void *stream);

/* Attention of one new token per row over the paged cache.
 * q [rows][num_heads head_dim] (rows q_stride elements apart), dtype 0 or 1,
 * head_dim 64 or 128, num_heads a multiple of num_kv_heads.  Row r attends to
 * its positions t < min(seq_len[r], table_width block_size), position t in slot
 * t % block_size of block block_table[r][t / block_size] (rows table_stride
 * entries apart).  out [rows][num_heads head_dim] (rows out_stride elements
 * apart) = softmax(scale q K^T) V, lse (may be NULL) [rows][num_heads] fp32 the
 * natural logarithm of the softmax's sum.  Positions whose block lies outside
 * [0, num_blocks) are left out; a row with no position left gets zeros and
 * lse -inf.  The values of table entries past a row's length do not matter; the
 * launch is planned by table_width, so one close to the lengths is faster.
 * workspace: cruise_decoder_attention_workspace() bytes, 16-byte aligned, not
 * shared by calls that may overlap (its contents do not matter between calls);
 * NULL where that returns 0.  Other pointers 16-byte aligned (block_table,
 * seq_len, lse 4-byte), strides of q, out and blocks multiples of 8 elements;
 * out must not overlap the inputs; num_blocks block_stride at most 2^35,
 * table_width block_size below 2^31 - 256. */
int32_t cruise_decoder_attention(
    const void *q, int64_t q_stride, int32_t rows, int32_t num_heads,
    int32_t num_kv_heads, int32_t head_dim, int32_t dtype,
    const void *key_cache, const void *value_cache, int64_t num_blocks,
    int32_t block_size, int64_t block_stride, const int32_t *block_table,
    int64_t table_stride, int32_t table_width, const int32_t *seq_len,
    float scale, void *out, int64_t out_stride, float *lse, void *workspace,
    int64_t workspace_bytes, int32_t device, void *stream);

/* Workspace bytes of cruise_decoder_attention for these sizes on `device`
 * (capacity = table_width block_size); 0 when it needs none, -1 for sizes it
 * refuses. */
int64_t cruise_decoder_attention_workspace(int32_t rows, int32_t num_heads,
                                           int32_t num_kv_heads,
                                           int32_t head_dim, int64_t capacity,
                                           int32_t device);

/* Rules on the logits and the greedy choice, in one pass.
 * logits [rows][vocab] of dtype 0, 1 or 2, rows logits_stride elements apart.
 * For every token, in fp32 and in this order:
 *   x = logit, plus bias_value where the token is in the row's bias list;
 *   token in the history: x = x > 0 ? x / repetition : x * repetition;
 *   count > 0: x = x - frequency * count; x = x - presence;
 *   allowed bit 0: x = -inf.
 * (So an infinite or NaN penalty acts on the tokens it is for, and no others.)
 * history [rows][history_width] (rows history_stride entries apart) holds
 * history_len[r] tokens, the first prompt_len[r] of them the prompt; count is
 * the token's occurrences after the prompt.  Entries outside the vocabulary do
 * not count.  repetition, frequency, presence: [rows] fp32, NULL for 1, 0, 0.
 * bias_token, bias_value [rows][bias_width] (rows bias_stride apart) with
 * bias_len[r] entries, increasing tokens within a row (entries of one token add
 * up).  allowed: bit
 * n % 32 of word n / 32 of a row (rows allowed_stride words apart).  active
 * [rows]: rows with 0 get token -1, nothing else of theirs is written.  Each
 * group may be NULL.
 * token[r] = the first maximum above -inf; -1 where there is none; -2 where a
 * processed value is NaN or +inf.  processed (may be NULL) [rows][vocab] fp32,
 * rows processed_stride apart: the x; it may be the logits themselves (fp32,
 * same stride), else must not overlap them.  token, processed and, with append,
 * history must not overlap one another or the other inputs.  append: token[r] >= 0
 * is written to history[r][history_len[r]] where that is inside history_width
 * (history_len itself is the caller's to advance).  4-byte alignment suffices (logits: their
 * own size).  The launch is planned by history_width and bias_width, so a width
 * close to the lengths is faster.  vocab at most 2^20; fewer than 2^30 history and bias entries
 * together, beyond 390000 logits at most 20000. */
int32_t cruise_decoder_choose(
    const void *logits, int64_t logits_stride, int32_t rows, int32_t vocab,
    int32_t dtype, const int32_t *active, int32_t *history,
    int64_t history_stride, int32_t history_width, const int32_t *prompt_len,
    const int32_t *history_len, const float *repetition,
    const float *frequency, const float *presence, const int32_t *bias_token,
    const float *bias_value, int64_t bias_stride, int32_t bias_width,
    const int32_t *bias_len, const uint32_t *allowed, int64_t allowed_stride,
    float *processed, int64_t processed_stride, int64_t *token, int32_t append,
    int32_t device, void *stream);

/* Why this thread's last decoder operator failed ("" after a success). */
const char *cruise_decoder_last_error(void);

#ifdef __cplusplus
}
#endif

#endif /* CRUISE_DECODER_H */
