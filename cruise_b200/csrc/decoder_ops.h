// decoder_ops.h -- the decoder operators on device tensors, as the host code
// of this library launches them (the C ABI in include/cruise_decoder.h and the
// engine).  Every launch goes to the stream it is given and returns without
// waiting; the arguments are checked by the caller-facing entries.
#pragma once

#include <cstdint>
#include <cuda_runtime.h>

namespace cruise {
namespace ops {

enum ElementType : int32_t { kBf16 = 0, kFp16 = 1, kFp32 = 2 };

// Head norms, rotation and the paged store of `tokens` tokens.
struct RotateArgs {
  const void *qkv;            // [tokens][>= (nq + 2 nkv) d]: q heads | k heads | v heads
  int64_t qkv_stride;         // elements between tokens
  int32_t tokens, nq, nkv, d;
  int32_t dtype;              // kBf16 or kFp16: qkv, norms, q_out and caches
  const int64_t *position;    // [tokens]
  const int32_t *slot;        // [tokens]; < 0: not stored
  const void *q_norm, *k_norm;   // [d] or nullptr
  float eps;
  const void *rope_cos, *rope_sin;   // [rope_rows][rotary]
  int32_t rope_dtype;         // kBf16 or kFp32
  int32_t rope_rows, rotary;
  void *q_out;                // [tokens][nq d], rows q_stride elements apart
  int64_t q_stride;
  void *key_cache, *value_cache;     // [num_blocks][block_size][nkv][d], blocks block_stride elements apart
  int64_t num_blocks, block_stride;
  int32_t block_size;
};

// Attention of one new token per row over the paged cache.
struct AttentionArgs {
  const void *q;              // [rows][nq d], rows q_stride elements apart
  int64_t q_stride;
  int32_t rows, nq, nkv, d;
  int32_t dtype;
  const void *key_cache, *value_cache;
  int64_t num_blocks, block_stride;
  int32_t block_size;
  const int32_t *block_table;   // [rows][table_width], rows table_stride entries apart
  int64_t table_stride;
  int32_t table_width;
  const int32_t *seq_len;       // [rows]
  float scale;
  void *out;                  // [rows][nq d], rows out_stride elements apart
  int64_t out_stride;
  float *lse;                 // [rows][nq] or nullptr
  void *workspace;            // attention_workspace() bytes, 16-byte aligned
};

// Rules on the logits and the greedy choice.
struct ChooseArgs {
  const void *logits;         // [rows][vocab], rows logits_stride elements apart
  int64_t logits_stride;
  int32_t rows, vocab;
  int32_t dtype;              // kFp32, kBf16 or kFp16
  const int32_t *active;      // [rows] or nullptr: 0 leaves the row alone (token -1)
  int32_t *history;           // [rows][history_width], rows history_stride entries apart, or nullptr
  int64_t history_stride;
  int32_t history_width;
  const int32_t *prompt_len, *history_len;   // [rows]
  const float *repetition, *frequency, *presence;   // [rows] or nullptr
  const int32_t *bias_token;  // [rows][bias_width], increasing within a row, or nullptr
  const float *bias_value;    // [rows][bias_width]
  int64_t bias_stride;
  int32_t bias_width;
  const int32_t *bias_len;    // [rows]
  const uint32_t *allowed;    // [rows][ceil(vocab / 32)] bit masks, rows allowed_stride words apart, or nullptr
  int64_t allowed_stride;
  float *processed;           // [rows][vocab], rows processed_stride elements apart, or nullptr
  int64_t processed_stride;
  int64_t *token;             // [rows]
  int32_t append;             // 1: history[r][history_len[r]] = token where it fits
};

// Whether [a, a + na) and [b, b + nb) bytes overlap.
inline bool overlap(const void *a, int64_t na, const void *b, int64_t nb) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return na > 0 && nb > 0 && x < y + static_cast<uintptr_t>(nb) && y < x + static_cast<uintptr_t>(na);
}

// Bytes from the first to the last element of rows `stride` elements apart.
inline int64_t extent(int64_t rows, int64_t stride, int64_t width, int64_t size) {
  return rows > 0 ? ((rows - 1) * stride + width) * size : 0;
}

cudaError_t launch_rotate_store(const RotateArgs &a, int device, cudaStream_t stream);
int64_t attention_workspace(int32_t rows, int32_t nq, int32_t nkv, int32_t d, int64_t capacity, int device);
cudaError_t launch_paged_attention(const AttentionArgs &a, int device, cudaStream_t stream);
cudaError_t launch_choose(const ChooseArgs &a, int device, cudaStream_t stream);

}  // namespace ops
}  // namespace cruise
