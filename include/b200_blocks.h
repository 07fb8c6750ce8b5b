/*
 * C ABI of the block operators: what surrounds the triangle update and the pair Transition in a block, for token, pair and
 * alignment tensors of any width. Part of libb200_trimul.so; error codes, b200_trimul_strerror and b200_trimul_last_cuda_error
 * are those of b200_trimul.h.
 *
 *  - Pointers are device pointers; calls are asynchronous on `cuda_stream`, may be issued from any host thread and captured into a
 *    graph. The caller owns every buffer; the library allocates nothing.
 *  - dtype of the activations: B200_BLOCKS_BF16, _F32 or _F16. Norm parameters and the residual scale are fp32.
 *  - Results are deterministic (fixed orders of summation). All arithmetic is fp32, each output is rounded once; the feed-forward also
 *    rounds h, da and db to the activations' type (operands of 16-bit products; h of up to four rows stays fp32). In fp16 a finite h,
 *    and a finite y of up to four rows, beyond 65504 become that; da, db and every other result become infinite there, and what is
 *    infinite or NaN on the way is never made finite.
 *  - Device-side waits are bounded: one that gives up lets the kernel finish and leaves a positive code that
 *    b200_blocks_read_status returns (and clears).
 */
#ifndef B200_BLOCKS_H_
#define B200_BLOCKS_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define B200_BLOCKS_BF16 0
#define B200_BLOCKS_F32 1
#define B200_BLOCKS_F16 2

#define B200_NORM_NONE 0
#define B200_NORM_LAYER 1
#define B200_NORM_RMS 2

#define B200_ACT_SILU 0
#define B200_ACT_GELU 1 /* with the error function */

#define B200_NORM_MAX_WIDTH 4096

/*
 * The join of two blocks on rows of width d (1 .. 4096), and without u (and y, gate, mask, scale) the plain norm h = norm_pre(x):
 *   t = norm_post(u);  y = x + valid * scale * sigmoid(gate) * t;  h = norm_pre(y)
 * x, u, y, h: [rows, d]. gate: logits [rows / gate_rows, d], row r of x uses gate row r / gate_rows (1: a row each; rows: one for
 * all), null: no gate. mask: uint8 [rows], 0: y = x there, whatever u and gate hold. scale, post_w, post_b, pre_w, pre_b: fp32 [d],
 * null: 1 or 0. post_kind B200_NORM_NONE: t = u; pre_kind B200_NORM_NONE: no h (the parameters of a norm that is not there are not
 * read). h is the norm of the unrounded y. y may be x and h may be u (a thread reads its row's elements before it writes them).
 * post_stats, pre_stats: fp32 [rows, 2], mean and 1 / sigma, for the backward (null: not kept).
 */
int b200_block_join_forward(const void* x, const void* u, const void* gate, const uint8_t* mask, const float* scale,
                            const float* post_w, const float* post_b, const float* pre_w, const float* pre_b, void* y, void* h,
                            float* post_stats, float* pre_stats, long long rows, int d, long long gate_rows, int dtype,
                            int post_kind, int pre_kind, float post_eps, float pre_eps, void* cuda_stream);

/*
 * Gradients of the above from dy and dh (either may be null: zero), the forward's inputs and statistics. Outputs that are null are
 * left out: dx, du [rows, d], dgate [rows / gate_rows, d] in the activations' type, d_scale, d_post_w, d_post_b, d_pre_w, d_pre_b
 * fp32 [d] (d_scale, d_post_w and d_post_b need u, the last two a norm after the block). Every output is overwritten. In rows that the
 * mask leaves out du and dgate are zero and nothing is added to the sums.
 * Workspace: b200_block_join_workspace_bytes, 1024-byte aligned.
 */
int b200_block_join_workspace_bytes(long long rows, int d, long long gate_rows, size_t* out_bytes);
int b200_block_join_backward(const void* dy, const void* dh, const void* x, const void* u, const void* gate, const uint8_t* mask,
                             const float* scale, const float* post_w, const float* post_b, const float* pre_w, const float* pre_b,
                             const float* post_stats, const float* pre_stats, void* dx, void* du, void* dgate, float* d_scale,
                             float* d_post_w, float* d_post_b, float* d_pre_w, float* d_pre_b, void* workspace,
                             size_t workspace_bytes, long long rows, int d, long long gate_rows, int dtype, int post_kind,
                             int pre_kind, void* cuda_stream);

/*
 * Gated feed-forward: y = (act(x w_a^T) * (x w_b^T)) w_s^T, x and y [rows, d], w_a and w_b [hidden, d], w_s [d, hidden], d and hidden
 * multiples of 8, rows up to 2^31 - 257. dtype B200_BLOCKS_BF16 or _F16; weight_dtype the same or B200_BLOCKS_F32 (rounded to dtype
 * in each call). Workspaces: 1024-byte aligned, b200_ff_workspace_bytes of the same sizes (backward 0 or 1).
 */
int b200_ff_workspace_bytes(long long rows, int d, int hidden, int weight_dtype, int backward, size_t* out_bytes);
/* For a backward: bytes that the forward of these sizes keeps (h, and a = x w_a^T and b = x w_b^T to 10 bits and more with a power of
 * two for 16 neighbouring units of a row: what is below 2^-25 of the largest of them loses bits), 0 where the backward forms them again
 * faster. A forward and its backward get the same buffer as `kept` (1024-byte aligned), or both null. */
int b200_ff_kept_bytes(long long rows, int d, int hidden, size_t* out_bytes);
int b200_ff_forward(const void* x, const void* w_a, const void* w_b, const void* w_s, void* y, void* kept, void* workspace,
                    size_t workspace_bytes, long long rows, int d, int hidden, int dtype, int weight_dtype, int activation,
                    void* cuda_stream);

/* Gradients from dy [rows, d] and the forward's inputs: dx (dtype), dw_a, dw_b, dw_s (weight_dtype, the weights' shapes). Null
 * outputs are left out, the others overwritten. */
int b200_ff_backward(const void* dy, const void* x, const void* w_a, const void* w_b, const void* w_s, const void* kept, void* dx,
                     void* dw_a, void* dw_b, void* dw_s, void* workspace, size_t workspace_bytes, long long rows, int d, int hidden, int dtype,
                     int weight_dtype, int activation, void* cuda_stream);

/* Synchronises `cuda_stream`; *code: 0, or the code of the first wait of one of these kernels on the current device that gave up
 * since the last call (then cleared). */
int b200_blocks_read_status(void* cuda_stream, int* code);

#ifdef __cplusplus
}
#endif
#endif /* B200_BLOCKS_H_ */
