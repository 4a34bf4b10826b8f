// Declarations shared by the translation units of the int8 and token-routing operators (not installed).
#pragma once

#include "nvfp4_internal.h"

#include <atomic>

namespace nvfp4_b200 {

extern std::atomic<unsigned long long> g_launches;

// nvfp4_gemm.cu: tensor map of a matrix of bytes [rows, row_bytes], tiles of box_rows x 128 bytes under the 128-byte
// swizzle; a tile that reaches beyond the matrix reads zeros there.
CUtensorMap byte_rows_map(const void* p, size_t rows, size_t row_bytes, int box_rows);

inline size_t dtype_bytes(int dtype) { return dtype == DTYPE_F32 ? 4 : 2; }

// int8_quant.cu
// x [rows, K] -> codes [rows, K] and scales [rows].
void int8_quantise(const void* x, int dtype, int8_t* codes, float* scales, long long rows, int K, cudaStream_t stream);
// The same, row t of x to the rows position[t * topk + j] of codes and scales; zeros from row *live on.
void int8_gather(const void* x, int dtype, long long tokens, int topk, int K, const int* position, const int* live, int8_t* codes,
                 float* scales, cudaStream_t stream);
void int8_dequantise(const int8_t* codes, const float* scales, float* out, long long rows, int K, cudaStream_t stream);

// int8_gemm.cu
struct Int8Tiles {
    int pair;       // 1: CTA pairs
    int swap;       // 1: channels on the MMA's M side, tokens on its N side
    int width;      // values of the MMA's N side per tile
    int split;      // CTAs that share a tile's K loop (one cluster)
    int stages;
    int subs;       // boxes of 128 K values per operand and ring stage
};
// rows x n x k; experts > 0: rows dealt to that many experts.
Int8Tiles int8_tiles(int rows, int n, int k, int experts, int device);
// Throws where the sizes, types or pointers of a product do not do.
void int8_gemm_check(const void* a, const void* b, const float* a_scales, const float* b_scales, const void* C, int out_dtype,
                     int M, int N, int K);
// early: the kernel in front of this one in the stream writes a and a_scales but not b, and lets this one start only
// after everything older than itself has finished.
void int8_gemm(const int8_t* a, const int8_t* b, const float* a_scales, const float* b_scales, void* C, int out_dtype, int M,
               int N, int K, bool early, cudaStream_t stream);
void int8_grouped_gemm(const int8_t* rows, const int8_t* weights, const float* row_scales, const float* weight_scales,
                       const int* offsets, int experts, void* C, int out_dtype, int R, int N, int K, bool zero_rest,
                       cudaStream_t stream);

// tokens.cu
void tokens_sort(const void* ids, int id_bytes, int routes, int experts, int* offsets, int* position, int* source, int* workspace,
                 cudaStream_t stream);
size_t tokens_sort_workspace(int routes, int experts);
void tokens_gather(const void* x, int dtype, int tokens, int topk, int hidden, const int* position, const int* live, void* rows,
                   cudaStream_t stream);
void tokens_combine(const void* rows, int dtype, const float* weights, const int* position, const int* live, int tokens, int topk,
                    int hidden, void* y, cudaStream_t stream);
void tokens_combine_backward(const void* d_y, int dtype, const void* rows, const float* weights, const int* position,
                             const int* live, int tokens, int topk, int hidden, void* d_rows, float* d_weights, cudaStream_t stream);

}  // namespace nvfp4_b200
