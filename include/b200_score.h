/* libb200score.so -- scoring text with the FP8 weights of the decode path, for B200 (sm_100a):
 * the FP8 128x128 block-scaled matrix product for any number of tokens, the log probabilities of
 * given tokens (with entropy, rank and the top alternatives), and the FP8 head straight to log
 * probabilities, without its logits. Same conventions as b200_lmhead.h: plain pointers and sizes,
 * an int status (0 = ok, negative = argument error, positive = cudaError_t), caller-owned outputs
 * and scratch, no allocation, work enqueued on `stream` only.
 */
#ifndef B200_SCORE_H
#define B200_SCORE_H

#include <cuda_runtime_api.h>

#ifdef __cplusplus
extern "C" {
#endif

/* y[m, n] = sum over the 128-K blocks b of xs[m, b] * ws[n / 128, b] * sum_{k in b} qx[m, k] wq[n, k],
 * the blocks' sums scaled and added in fp32, one rounding to y's type (0 = bf16, 1 = f16, 2 = f32).
 * qx e4m3 [M, K] with row stride ldx bytes; xs fp32 [M, ceil(K/128)] with element strides xs_row and
 * xs_col (row-major or group-major); ws fp32 [ceil(N/128), ceil(K/128)] with row stride ws_row.
 * packed 0: wq e4m3 [N, K] row-major with row stride ldw bytes; packed 1: the FP8 head's strip
 * layout of b200_lmhead.h (N % 16 == 0, K % 128 == 0, ldw unused). y [M, N] with row stride ldy
 * elements. K % 16 == 0, ldx and ldw multiples of 16, 16-byte aligned qx and wq (a TMA copy's rules);
 * a last group of fewer than 128 K and a last block of fewer than 128 rows have scales of their own.
 * Returns 0, -1 M outside [0, 2^30], -2 bad N (at most 2^30), -3 bad K (at most 2^30), -4 a stride below its
 * row length or not a multiple of 16, -5 bad dtype, -8 more than 2^30 tiles, -10 misaligned pointer, -12 no
 * tensor map, -13 a build whose register count is not the one the kernels were written for. */
int b200_fp8_block_gemm(const void* qx, long long ldx, const float* xs, long long xs_row, long long xs_col,
                        const void* wq, long long ldw, int packed, const float* ws, long long ws_row, void* y,
                        long long ldy, int y_dtype, int M, int N, int K, cudaStream_t stream);

/* Row statistics of logits [M, V] (dtype 0 = bf16, 1 = f16, 2 = f32; row stride ld elements, unit column
 * stride) and of one token per row: with d_v = x_v - max x, S = sum e^{d_v}, W = sum e^{d_v} d_v,
 *   logprob = d_t - ln S, entropy = ln S - W / S, lse = max x + ln S, rank = 1 + #{v : x_v > x_t},
 * and the top_k (0..64, <= V) largest logits, equal ones by the lower id: top_ids [M, top_k] int64,
 * top_logprob fp32 [M, top_k]. ids int64 [M]; rank int64 [M]; logprob / entropy / lse fp32 [M].
 * -inf logits have probability 0. A row of nothing but -inf: lse and every logprob -inf, entropy 0.
 * A row with a NaN or +inf: logprob, entropy and lse NaN (NaN comes first among the top ids). An id
 * outside [0, V): logprob NaN, rank 0. Returns 0, -1 M outside [0, 2^27], -2 V outside [1, 2^30], -4 ld < V, -5 bad dtype,
 * -6 bad top_k, -10 a pointer that is not a multiple of its element. */
int b200_token_logprobs(const void* logits, int dtype, long long ld, int M, int V, const long long* ids, int top_k,
                        float* logprob, long long* rank, float* entropy, float* lse, long long* top_ids,
                        float* top_logprob, cudaStream_t stream);

/* The product of b200_fp8_block_gemm (same operands and codes) reduced to logprob, entropy and lse as
 * in b200_token_logprobs, on the fp32 logits, which are never written. workspace:
 * b200_fp8_head_logprobs_workspace_bytes(M, N) bytes, 16-byte aligned, no initialisation needed; calls
 * that share it must not overlap. Extra code: -9 workspace missing or too small. */
long long b200_fp8_head_logprobs_workspace_bytes(int M, int N);
int b200_fp8_head_logprobs(const void* qx, long long ldx, const float* xs, long long xs_row, long long xs_col,
                           const void* wq, long long ldw, int packed, const float* ws, long long ws_row,
                           const long long* ids, int M, int N, int K, float* logprob, float* entropy, float* lse,
                           void* workspace, long long workspace_bytes, cudaStream_t stream);

/* Device error word of these kernels (1 = a bounded pipeline wait ran out: what that call could not compute
 * is NaN, an element of the product or a row's logprob, entropy and lse); reset != 0 clears it. Synchronous
 * with the default stream: synchronize any other stream first. A wait gives up after 2^18 tries, about a
 * second, or as many as B200_SCORE_WAIT_TRIES in the environment says at the first call (0: at once). */
int b200_score_error(int reset);

#ifdef __cplusplus
}
#endif

#endif /* B200_SCORE_H */
