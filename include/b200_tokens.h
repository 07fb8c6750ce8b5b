/*
 * C ABI of the token operators: attention over the tokens of a batch or of packed sequences with a learned bias of the relative
 * position, the relative position added to the pair tensor, and dropout with a residual add whose mask is never stored. Part of
 * libb200_trimul.so; error codes, b200_trimul_strerror and b200_trimul_last_cuda_error are those of b200_trimul.h, data types
 * (B200_BLOCKS_*) those of b200_blocks.h.
 *
 *  - Pointers are device pointers; calls are asynchronous on `cuda_stream`, may be issued from any host thread and captured into a
 *    graph. The caller owns every buffer; the library allocates nothing.
 *  - Results are deterministic (fixed orders of summation). Arithmetic, softmax statistics and sums are fp32, each output is rounded
 *    once; the attention's probabilities and the gradients of its scores are rounded to the activations' type as operands of products.
 *  - Numbers on the device that the host cannot check (offsets, bucket numbers) are brought into their ranges by the kernels: what
 *    lies outside gives unspecified results, not accesses out of bounds.
 */
#ifndef B200_TOKENS_H_
#define B200_TOKENS_H_

#include "b200_blocks.h"

#ifdef __cplusplus
extern "C" {
#endif

#define B200_ATTENTION_MAX_WIDTH 128
#define B200_ATTENTION_MAX_BIAS 65504.f
#define B200_POSITION_MAX_REACH 256
#define B200_POSITION_MAX_BUCKETS 512

/* A tensor [rows, heads, d]: element strides of its first two dimensions (multiples of 8); the last is contiguous. */
typedef struct {
  const void* data;
  long long row_stride, head_stride;
} b200_attention_tensor;

/* What a call works on. Sequence s has the rows offsets[s] .. offsets[s + 1] (int32 [sequences + 1], non-decreasing, the first 0, the
 * last at most `rows`), or, with offsets null, `length` rows each (rows = sequences * length). */
typedef struct {
  long long rows;
  int sequences, length;
  int heads, kv_heads; /* heads a multiple of kv_heads: query head h reads head h / (heads / kv_heads) */
  int d;               /* 8 .. 128, a multiple of 8 */
  int dtype;           /* B200_BLOCKS_BF16 or _F16 */
  int causal;
  float scale;         /* of the scores */
  const int* offsets;
  const uint8_t* mask; /* [rows], 0: the row neither attends nor is attended to; null: all do */
  /* bias table[bucket_of[clip(j - i, -reach, reach) + reach], head] of key j and query i of a sequence; table null: none. -inf: the pair
   * does not count; finite ones beyond +-B200_ATTENTION_MAX_BIAS count as that. */
  const void* table;    /* [buckets, heads] */
  int table_dtype;      /* dtype or B200_BLOCKS_F32 */
  const int* bucket_of; /* int32 [2 reach + 1] */
  int buckets, reach;
} b200_attention_call;

/*
 * o_i = sum_j softmax_j(scale q_i . k_j + bias) v_j, o [rows, heads, d] contiguous. Rows without a key (masked ones, rows of no
 * sequence) are zero, and what masked rows hold is never used. For a backward (both null: not kept): rest, of o's type and shape, what
 * rounding o took away (2^11 times as much in fp16), and lse, fp32 [heads, rows], log2 of the softmax's denominators.
 */
int b200_token_attention_forward(const b200_attention_call* call, const b200_attention_tensor* q, const b200_attention_tensor* k,
                                 const b200_attention_tensor* v, void* o, void* rest, float* lse, void* cuda_stream);

/*
 * Gradients from dO (strides as for q), the forward's inputs, o, rest and lse: dq [rows, heads, d], dk and dv [rows, kv_heads, d], contiguous,
 * and, where it is not null, dtable (table_dtype). Workspace: 1024-byte aligned, b200_token_attention_workspace_bytes of the same call; where
 * dtable is null, that of the call without a table is enough (the gradient of a table takes 4 (2 reach + 1) bytes a head and tile of
 * 128 rows of a sequence, and one tile a sequence more).
 */
int b200_token_attention_workspace_bytes(const b200_attention_call* call, size_t* out_bytes);
int b200_token_attention_backward(const b200_attention_call* call, const b200_attention_tensor* q, const b200_attention_tensor* k,
                                  const b200_attention_tensor* v, const void* o, const void* rest, const float* lse,
                                  const b200_attention_tensor* d_o, void* dq,
                                  void* dk, void* dv, void* dtable, void* workspace, size_t workspace_bytes, void* cuda_stream);

/*
 * y[b, i, j] = z[b, i, j] + table[bucket_of[clip(index[b, j] - index[b, i], -reach, reach) + reach]], or + table[buckets - 1] where
 * chain[b, i] != chain[b, j]; z, y [b, n, n, c] in bf16, fp16 or fp32 (y may be z), table fp32 [buckets, c], index and chain [b, n]
 * int64 (wide) or int32, chain null: one chain.
 */
int b200_relative_position_forward(const void* z, const float* table, const void* index, const void* chain, const int* bucket_of, void* y,
                                   int b, int n, int c, int buckets, int reach, int wide, int dtype, void* cuda_stream);
/* dtable (fp32) from dy; the gradient of z is dy. Workspace as above. */
int b200_relative_position_workspace_bytes(int b, int n, int c, int buckets, size_t* out_bytes);
int b200_relative_position_backward(const void* dy, const void* index, const void* chain, const int* bucket_of, float* dtable,
                                    void* workspace, size_t workspace_bytes, int b, int n, int c, int buckets, int reach, int wide,
                                    int dtype, void* cuda_stream);

/*
 * y = x + keep * u * 65536 / (65536 - threshold) (x null: without it) for u [outer, shared, inner], whose rows `shared` use one mask
 * [outer, inner]: element m of it stays where half m % 8 (low half of each word first) of Philox-4x32-10 with the counter (m / 8, key[1]
 * + call) and the key key[0] is at least `threshold` (0 .. 65536; at 65536 nothing stays and u adds nothing). key: int64 [2]. y may be x
 * or u. The gradient of u is the same call on dy without x.
 */
int b200_block_dropout(const void* x, const void* u, const long long* key, unsigned long long call, void* y, long long outer, long long shared,
                       long long inner, int threshold, int dtype, void* cuda_stream);

/* As b200_blocks_read_status, for the kernels of this header. */
int b200_tokens_read_status(void* cuda_stream, int* code);

#ifdef __cplusplus
}
#endif
#endif /* B200_TOKENS_H_ */
