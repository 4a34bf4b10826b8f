/* C ABI of the int8 and token-routing operators in libgpu_kernels_nvfp4_bench.so (B200 / sm_100a only).
 *
 * The conventions are those of nvfp4_capi.h: every function returns 0, or 1 after storing a message that
 * gpu_kernels_nvfp4_last_error() returns; no exception crosses this boundary; streams are void* (cudaStream_t); pointers
 * are device pointers and, unless said otherwise, 16-byte aligned; the device they belong to is the current one. All
 * calls are asynchronous on their stream and may be captured into a CUDA graph; none allocates, and none keeps anything
 * for the next. Data types are 0 = bf16, 1 = fp16, 2 = fp32. A matrix with no rows is valid and launches nothing.
 * A product that gave up waiting inside the kernel is reported by gpu_kernels_nvfp4_validate(NULL).
 */
#ifndef GPU_KERNELS_OPERATORS_CAPI_H
#define GPU_KERNELS_OPERATORS_CAPI_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- int8 with a scale for each token (row of x) and each channel (row of the weights) ---- */

/* x [rows, K], any K >= 1 -> codes [rows, K] int8, scales [rows] fp32 (4-byte aligned). amax = max |x| of a row,
 * scale = amax / 127, code = the integer nearest to 127 x / amax (the exact quotient), ties to the even one. A zero row
 * has scale 0 and codes 0; a row that holds a NaN or an infinity has scale NaN and codes 0. */
int gpu_kernels_int8_quantize(const void* x, int dtype, void* codes, void* scales, long long rows, int K, void* stream);
/* codes * scale -> fp32 [rows, K]. */
int gpu_kernels_int8_dequantize(const void* codes, const void* scales, void* out_f32, long long rows, int K, void* stream);
/* C [M, N] = (a [M, K] b [N, K]^T) * a_scales[m] * b_scales[n]: exact integer sums, FP32 scaling, rounded to C's type.
 * K a multiple of 16, at most 131056; N a multiple of 8; M and N up to 2^30. a_scales 4-byte aligned. Any int8 code, -128 included. */
int gpu_kernels_int8_gemm(const void* a, const void* b, const void* a_scales, const void* b_scales, void* C, int out_dtype,
                          int M, int N, int K, void* stream);
/* The same for activations x [M, K] that are quantised on the way; codes [M, K] and scales [M] are workspace and hold what
 * gpu_kernels_int8_quantize would give. The product requests its first weights while the quantiser runs. */
int gpu_kernels_int8_linear(const void* x, int dtype, const void* b, const void* b_scales, void* codes, void* scales, void* C,
                            int out_dtype, int M, int N, int K, void* stream);
/* rows [R, K] sorted by expert, offsets [experts + 1] int32 (device): expert e's rows are [offsets[e], offsets[e + 1]) and
 * are multiplied by weights[e] of [experts, N, K] (scales [experts, N]); C [R, N]. Rows of no expert (in front of
 * offsets[0], at or behind offsets[experts]) are left as they were, or with zero_rest cleared. At most 1024 experts,
 * experts * N up to 2^30. Offsets are clipped to 0..R; where they decrease, the largest so far counts. */
int gpu_kernels_int8_grouped_gemm(const void* rows, const void* weights, const void* row_scales, const void* weight_scales,
                                  const void* offsets, int experts, void* C, int out_dtype, int R, int N, int K, int zero_rest,
                                  void* stream);
/* What a product of these sizes runs (experts = 0: a dense one): info[0..4] = {CTA pairs, tokens on the MMA's N side,
 * width of that side, CTAs that share a tile's K loop, ring stages}. */
int gpu_kernels_int8_tiles(int rows, int N, int K, int experts, int* info);

/* ---- tokens to their experts' rows and back. Route i (of tokens * topk) is a choice of token i / topk. ---- */

/* ids [routes] int32 or int64 (id_bytes 4 or 8): offsets [experts + 1], position [routes] = row of each route,
 * source [routes] = route of each row, int32 each. Rows are ordered by expert, then by route; routes of no expert (ids
 * outside [0, experts)) come last, from row offsets[experts] on. At most 1024 experts. 4-byte aligned pointers (ids: 8
 * where 64-bit). workspace: gpu_kernels_tokens_sort_workspace bytes of the caller's (NULL where that is 0), not shared
 * with a call that may run at the same time. */
int gpu_kernels_tokens_sort(const void* ids, int id_bytes, int routes, int experts, void* offsets, void* position, void* source,
                            void* workspace, void* stream);
size_t gpu_kernels_tokens_sort_workspace(int routes, int experts);
/* rows [tokens * topk, hidden]: x [tokens, hidden] in that order; `live` points to the number of live rows
 * (offsets + experts); the rows behind are cleared. Every row is the place of one route: a position outside the rows is
 * skipped, a row that no position names is not written. Pointers need the alignment of their type only; 16-byte aligned rows
 * are copied 16 bytes at a time. */
int gpu_kernels_tokens_gather(const void* x, int dtype, int tokens, int topk, int hidden, const void* position, const void* live,
                              void* rows, void* stream);
/* The same, quantised: codes [tokens * topk, K] and scales [tokens * topk]; K a multiple of 16. */
int gpu_kernels_tokens_gather_int8(const void* x, int dtype, int tokens, int topk, int K, const void* position, const void* live,
                                   void* codes, void* scales, void* stream);
/* y [tokens, hidden] = per token the sum over its live routes, in their order and in FP32, of weights[route] (fp32; NULL:
 * 1) times the route's row; rows that are not live are not read. With NULL weights this is the gradient of the gather. */
int gpu_kernels_tokens_combine(const void* rows, int dtype, const void* weights, const void* position, const void* live, int tokens,
                               int topk, int hidden, void* y, void* stream);
/* The gradients of gpu_kernels_tokens_combine: d_rows[position[i]] = weights[i] * d_y[token] (zero where not live) and
 * d_weights[i] = <d_y[token], rows[position[i]]> (zero where not live). Either may be NULL; rows may be NULL without
 * d_weights. */
int gpu_kernels_tokens_combine_backward(const void* d_y, int dtype, const void* rows, const void* weights, const void* position,
                                        const void* live, int tokens, int topk, int hidden, void* d_rows, void* d_weights,
                                        void* stream);

#ifdef __cplusplus
}
#endif

#endif
