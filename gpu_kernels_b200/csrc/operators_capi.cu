// extern "C" surface of the int8 and token-routing operators (declared in include/operators_capi.h). As in nvfp4_capi.cu,
// exceptions end here: the message is stored and the entry point returns 1.
#include "operators_capi.h"
#include "operators_internal.h"

#include <cstring>

namespace nvfp4_b200 {
void set_last_error(const char* message);
}

namespace {

using namespace nvfp4_b200;

template <typename F>
int guarded(F&& body) {
    try {
        require_sm100();
        body();
        return 0;
    } catch (const std::exception& e) {
        set_last_error(e.what());
    } catch (...) {
        set_last_error("unknown error");
    }
    return 1;
}

const int8_t* i8(const void* p) { return static_cast<const int8_t*>(p); }
const float* f32(const void* p) { return static_cast<const float*>(p); }
const int* i32(const void* p) { return static_cast<const int*>(p); }
cudaStream_t on(void* stream) { return static_cast<cudaStream_t>(stream); }

}  // namespace

extern "C" {

int gpu_kernels_int8_quantize(const void* x, int dtype, void* codes, void* scales, long long rows, int K, void* stream) {
    return guarded([&] { int8_quantise(x, dtype, static_cast<int8_t*>(codes), static_cast<float*>(scales), rows, K, on(stream)); });
}

int gpu_kernels_int8_dequantize(const void* codes, const void* scales, void* out, long long rows, int K, void* stream) {
    return guarded([&] { int8_dequantise(i8(codes), f32(scales), static_cast<float*>(out), rows, K, on(stream)); });
}

int gpu_kernels_int8_gemm(const void* a, const void* b, const void* a_scales, const void* b_scales, void* C, int out_dtype,
                          int M, int N, int K, void* stream) {
    return guarded([&] { int8_gemm(i8(a), i8(b), f32(a_scales), f32(b_scales), C, out_dtype, M, N, K, false, on(stream)); });
}

int gpu_kernels_int8_linear(const void* x, int dtype, const void* b, const void* b_scales, void* codes, void* scales, void* C,
                            int out_dtype, int M, int N, int K, void* stream) {
    return guarded([&] {
        // both are checked before the first is launched
        int8_gemm_check(codes, b, f32(scales), f32(b_scales), C, out_dtype, M, N, K);
        int8_quantise(x, dtype, static_cast<int8_t*>(codes), static_cast<float*>(scales), M, K, on(stream));
        // The quantiser waits for everything in front of it before it lets the product start, and does not write the
        // weights: the product may read them at once.
        int8_gemm(i8(codes), i8(b), f32(scales), f32(b_scales), C, out_dtype, M, N, K, true, on(stream));
    });
}

int gpu_kernels_int8_grouped_gemm(const void* rows, const void* weights, const void* row_scales, const void* weight_scales,
                                  const void* offsets, int experts, void* C, int out_dtype, int R, int N, int K, int zero_rest,
                                  void* stream) {
    return guarded([&] {
        int8_grouped_gemm(i8(rows), i8(weights), f32(row_scales), f32(weight_scales), i32(offsets), experts, C, out_dtype, R, N, K,
                          zero_rest != 0, on(stream));
    });
}

int gpu_kernels_int8_tiles(int rows, int N, int K, int experts, int* info) {
    return guarded([&] {
        if (!info || rows < 1 || N < 1 || K < 1 || experts < 0 || rows > 1 << 30 || N > 1 << 30 || experts > 1024)
            throw std::invalid_argument("int8 tiles: positive sizes (rows and N up to 2^30, 1024 experts) and an output");
        int device = 0;
        cuda_check(cudaGetDevice(&device));
        const Int8Tiles t = int8_tiles(rows, N, K, experts, device);
        const int values[5] = {t.pair, t.swap, t.width, t.split, t.stages};
        std::memcpy(info, values, sizeof(values));
    });
}

size_t gpu_kernels_tokens_sort_workspace(int routes, int experts) {
    return routes < 0 || experts < 1 ? 0 : tokens_sort_workspace(routes, experts);
}

int gpu_kernels_tokens_sort(const void* ids, int id_bytes, int routes, int experts, void* offsets, void* position, void* source,
                            void* workspace, void* stream) {
    return guarded([&] {
        tokens_sort(ids, id_bytes, routes, experts, static_cast<int*>(offsets), static_cast<int*>(position), static_cast<int*>(source),
                    static_cast<int*>(workspace), on(stream));
    });
}

int gpu_kernels_tokens_gather(const void* x, int dtype, int tokens, int topk, int hidden, const void* position, const void* live,
                              void* rows, void* stream) {
    return guarded([&] { tokens_gather(x, dtype, tokens, topk, hidden, i32(position), i32(live), rows, on(stream)); });
}

int gpu_kernels_tokens_gather_int8(const void* x, int dtype, int tokens, int topk, int K, const void* position, const void* live,
                                   void* codes, void* scales, void* stream) {
    return guarded([&] {
        int8_gather(x, dtype, tokens, topk, K, i32(position), i32(live), static_cast<int8_t*>(codes), static_cast<float*>(scales), on(stream));
    });
}

int gpu_kernels_tokens_combine(const void* rows, int dtype, const void* weights, const void* position, const void* live, int tokens,
                               int topk, int hidden, void* y, void* stream) {
    return guarded([&] { tokens_combine(rows, dtype, f32(weights), i32(position), i32(live), tokens, topk, hidden, y, on(stream)); });
}

int gpu_kernels_tokens_combine_backward(const void* d_y, int dtype, const void* rows, const void* weights, const void* position,
                                        const void* live, int tokens, int topk, int hidden, void* d_rows, void* d_weights,
                                        void* stream) {
    return guarded([&] {
        tokens_combine_backward(d_y, dtype, rows, f32(weights), i32(position), i32(live), tokens, topk, hidden, d_rows,
                                static_cast<float*>(d_weights), on(stream));
    });
}

}  // extern "C"
