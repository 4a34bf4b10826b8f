// Per-token int8 quantiser, the same into expert order, and the dequantiser, for sm_100a.
//
// Row r of x [rows, K]: amax = max |x|, scale = amax / 127 (FP32), code = the integer nearest to 127 x / amax, ties to
// the even one. The quotient is the exact one, so that a value on a border gets the code the definition gives it (with
// amax = 2x, for example, 127 x / amax is 63.5): see code_of. A zero row has scale 0 and codes 0. A row that holds a NaN
// or an infinity has scale NaN and codes 0: what is computed from it is NaN, not a number that looks sound.
//
// HBM-bound: the row is read once, held in registers while its maximum is taken, and written as codes (8192 x 8192 bf16
// 31.6 us, 6.4 TB/s; FP32 52 us; 8192 x 8191 bf16 34.7). A row is that of 4 to 32 threads, or of a block of as many warps as
// hold it (with a warp for each short row 128 values took 4.0 times what their bytes take, now 1.2; with blocks of 256 or
// 512 threads for each long one 4836 x 8784 FP32 took 64 us, now 38). Threads take 16 values each, one 16-byte store of
// codes. The elements of all rows are one flat array cut into groups of 16, so loads and stores are aligned whatever K is;
// what a row has in front of its first whole group and behind its last one (up to 15 values each) is taken one by one.
#include "operators_internal.h"
#include "ptx.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

namespace nvfp4_b200 {
namespace {

template <typename T> struct Bits;                              // magnitude of a value as an ordered unsigned integer
template <> struct Bits<__nv_bfloat16> {
    static constexpr uint32_t NOT_FINITE = 0x7F80u;
    static __device__ float widen(uint32_t b) { return __uint_as_float(b << 16); }
};
template <> struct Bits<__half> {
    static constexpr uint32_t NOT_FINITE = 0x7C00u;
    static __device__ float widen(uint32_t b) { return __half2float(__ushort_as_half(static_cast<unsigned short>(b))); }
};
template <> struct Bits<float> {
    static constexpr uint32_t NOT_FINITE = 0x7F800000u;
    static __device__ float widen(uint32_t b) { return __uint_as_float(b); }
};

// What a row's codes are made with. f = a power of two that keeps products and quotients of rows of very large or very
// small values inside FP32's normal range; 1 for all others.
struct RowScale {
    float amax, times, divisor, reciprocal;                     // times = 127 f, divisor = amax f, reciprocal = 1 / divisor
    __device__ RowScale(float a) : amax(a) {
        const float f = a > 0x1p100f ? 0x1p-64f : a < 0x1p-60f ? 0x1p64f : 1.0f;
        times = 127.0f * f;
        divisor = a * f;
        reciprocal = a > 0.0f ? 1.0f / divisor : 0.0f;
    }
};

constexpr float ROUND = 12582912.0f;                            // 1.5 * 2^23: adding it rounds to an integer, ties to even, in the low bits

// 127 x / amax rounded to an integer, in the low byte of the result. 16-bit inputs: p = 127 x is exact (at most 18
// significant bits). q0 = p * reciprocal is within 2 ulp of the quotient; its residual p - q0 * amax is exact in an FMA,
// and one correction gives the quotient rounded once: exactly k + 1/2 where that is the quotient, and never k + 1/2
// elsewhere, since a quotient of such operands that is no tie lies at least 2^-19 (relative) away from one. FP32 inputs:
// p is rounded, so a quotient within 2^-14 of a tie is decided by comparing 127 |x| with (k + 1/2) amax, both exact in
// 64 bits.
template <typename T>
__device__ __forceinline__ uint32_t code_of(float x, const RowScale& s) {
    const float p = x * s.times;
    const float q0 = p * s.reciprocal;
    float q = __fmaf_rn(__fmaf_rn(-q0, s.divisor, p), s.reciprocal, q0);
    if constexpr (sizeof(T) == 4) {
        const float n = rintf(q);
        if (fabsf(q - n) > 0.5f - 0x1p-14f) {
            const float k = floorf(fabsf(q));
            const double value = 127.0 * fabs(double(x)), tie = (double(k) + 0.5) * double(s.amax);
            const float low_even = k - 2.0f * floorf(0.5f * k);
            q = copysignf(value > tie || (value == tie && low_even != 0.0f) ? k + 1.0f : k, q);
        }
    }
    return __float_as_uint(q + ROUND);
}

template <typename T>
struct Group {                                                  // 16 values as loaded
    uint4 raw[sizeof(T)];

    __device__ __forceinline__ uint32_t word(int i) const {
        const uint4& v = raw[i / 4];
        return i % 4 == 0 ? v.x : i % 4 == 1 ? v.y : i % 4 == 2 ? v.z : v.w;
    }
    __device__ __forceinline__ void load(const T* x, size_t group) {
        const uint4* p = reinterpret_cast<const uint4*>(x + group * 16);
        #pragma unroll
        for (int i = 0; i < int(sizeof(T)); ++i) raw[i] = __ldg(p + i);
    }
    __device__ __forceinline__ uint32_t magnitude(uint32_t sofar) const {   // 16-bit types: two maxima side by side
        #pragma unroll
        for (int i = 0; i < int(4 * sizeof(T)); ++i) {
            if constexpr (sizeof(T) == 2) sofar = __vmaxu2(sofar, word(i) & 0x7FFF7FFFu);
            else sofar = max(sofar, word(i) & 0x7FFFFFFFu);
        }
        return sofar;
    }
    __device__ __forceinline__ uint4 codes(const RowScale& s) const {
        uint32_t out[4];
        #pragma unroll
        for (int q = 0; q < 4; ++q) {
            uint32_t c[4];
            #pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int at = 4 * q + i;
                float x;
                if constexpr (sizeof(T) == 2) x = Bits<T>::widen(at % 2 ? word(at / 2) >> 16 : word(at / 2) & 0xFFFFu);
                else x = Bits<T>::widen(word(at));
                c[i] = code_of<T>(x, s);
            }
            out[q] = __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
        }
        return make_uint4(out[0], out[1], out[2], out[3]);
    }
};

// TPR: threads per row, up to 32 (a warp or part of one) or at most that many (a block of as many as it takes); NV: groups
// of 16 that each of them holds in registers; what a row has beyond those is read twice, the second time from L2. ROUTED: the row's codes go to `topk` rows of the output instead of its own.
template <typename T, int TPR, int NV, bool ROUTED, bool WHOLE>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR)
int8_quantise_kernel(const T* __restrict__ x, int8_t* __restrict__ codes, float* __restrict__ scales, long long rows, int K,
                     const int* __restrict__ position, const int* __restrict__ live, int topk) {
    ptx::chain_point();
    const int tpr = TPR <= 32 ? TPR : int(blockDim.x), t = TPR <= 32 ? threadIdx.x % TPR : threadIdx.x;
    long long row = TPR <= 32 ? (long long)(blockIdx.x) * (256 / TPR) + threadIdx.x / TPR : blockIdx.x;
    if (TPR == 32 && row >= rows) return;
    if (TPR < 32) row = min(row, rows - 1);                     // (what a warp has behind the last row writes that row's codes again)
    const size_t begin = size_t(row) * K, end = begin + K;
    const size_t whole_from = WHOLE ? begin : min(end, (begin + 15) / 16 * 16), whole_to = WHOLE ? end : max(whole_from, end / 16 * 16);
    const size_t g0 = whole_from / 16, g1 = g0 + (whole_to - whole_from) / 16;
    // This thread's values outside the whole groups, 32 places in all: sixteen in front of them and as many behind.
    constexpr int SINGLES = WHOLE ? 0 : TPR < 32 ? 32 / TPR : 1;
    size_t place[SINGLES ? SINGLES : 1];
    bool has_single[SINGLES ? SINGLES : 1];
    uint32_t single_bits[SINGLES ? SINGLES : 1], top = 0u;
    #pragma unroll
    for (int i = 0; i < SINGLES; ++i) {
        const int at = t + i * TPR;
        place[i] = at < 16 ? begin + at : whole_to + (at - 16);
        has_single[i] = at < 32 && place[i] < (at < 16 ? whole_from : end);
        single_bits[i] = 0u;
        if (has_single[i]) {
            if constexpr (sizeof(T) == 2) single_bits[i] = __ldg(reinterpret_cast<const unsigned short*>(x) + place[i]);
            else single_bits[i] = __ldg(reinterpret_cast<const uint32_t*>(x) + place[i]);
        }
    }
    // A warp holds 32 NV groups in a row: its loads and stores differ by constants.
    const size_t first = g0 + t / 32 * (32 * NV) + t % 32;
    Group<T> held[NV];
    #pragma unroll
    for (int j = 0; j < NV; ++j)
        if (first + j * 32 < g1) held[j].load(x, first + j * 32);
    #pragma unroll
    for (int i = 0; i < SINGLES; ++i) top = max(top, single_bits[i] & (sizeof(T) == 2 ? 0x7FFFu : 0x7FFFFFFFu));
    for (size_t group = g0 + t + NV * tpr; !WHOLE && group < g1; group += tpr) {
        Group<T> v;
        v.load(x, group);
        top = v.magnitude(top);
    }
    #pragma unroll
    for (int j = 0; j < NV; ++j)
        if (first + j * 32 < g1) top = held[j].magnitude(top);
    if constexpr (sizeof(T) == 2) top = max(top & 0xFFFFu, top >> 16);
    if constexpr (TPR < 32) {
        #pragma unroll
        for (int d = TPR / 2; d; d /= 2) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
    } else {
        top = __reduce_max_sync(0xFFFFFFFFu, top);
    }
    if constexpr (TPR > 32) {
        __shared__ uint32_t warp_top[TPR / 32];
        if (threadIdx.x % 32 == 0) warp_top[threadIdx.x / 32] = top;
        __syncthreads();
        const uint32_t mine = threadIdx.x % 32 < blockDim.x / 32 ? warp_top[threadIdx.x % 32] : 0u;
        top = __reduce_max_sync(0xFFFFFFFFu, mine);
    }
    const bool finite = top < Bits<T>::NOT_FINITE;
    const RowScale s(finite ? Bits<T>::widen(top) : 0.0f);
    const float scale = finite ? s.amax / 127.0f : __int_as_float(0x7FC00000);
    auto emit = [&](const Group<T>& v, size_t group) {
        const uint4 c = finite ? v.codes(s) : make_uint4(0u, 0u, 0u, 0u);
        if constexpr (ROUTED) {                                  // K is a multiple of 16: whole groups
            const long long out_rows = rows * topk;
            const int end_live = __ldg(live);
            for (int j = 0; j < topk; ++j) {
                const int to = __ldg(position + row * topk + j);
                if (to < 0 || to >= out_rows) continue;
                reinterpret_cast<uint4*>(codes)[size_t(to) * (K / 16) + (group - g0)] = to < end_live ? c : make_uint4(0u, 0u, 0u, 0u);
            }
        } else {
            reinterpret_cast<uint4*>(codes)[group] = c;
        }
    };
    #pragma unroll
    for (int i = 0; i < SINGLES; ++i)
        if (has_single[i]) codes[place[i]] = finite ? int8_t(code_of<T>(Bits<T>::widen(single_bits[i]), s)) : int8_t(0);
    #pragma unroll
    for (int j = 0; j < NV; ++j)
        if (first + j * 32 < g1) emit(held[j], first + j * 32);
    for (size_t group = g0 + t + NV * tpr; !WHOLE && group < g1; group += tpr) {
        Group<T> v;
        v.load(x, group);
        emit(v, group);
    }
    if constexpr (ROUTED) {
        const int end_live = __ldg(live);
        for (int j = t; j < topk; j += tpr) {
            const int to = __ldg(position + row * topk + j);
            if (to >= 0 && to < rows * topk) scales[to] = to < end_live ? scale : 0.0f;
        }
    } else if (t == 0) {
        scales[row] = scale;
    }
}

// The codes of all rows as one flat array, four to a thread at a time: a warp reads 128 bytes and writes 512, both in one
// run: 8192 x 8192 51.9 us, 6.5 TB/s (with sixteen codes and four 16-byte stores to a thread 76). A group of four that reaches into
// the next row takes each value's own scale.
constexpr int DEQUANT_GROUPS = 4;                               // groups per thread, a block's threads apart

// Index: 32 bits wide where the number of values allows (a 64-bit division for each group took 59 us).
template <typename Index>
__global__ void __launch_bounds__(256)
int8_dequantise_kernel(const int8_t* __restrict__ codes, const float* __restrict__ scales, float* __restrict__ out, size_t values, int K) {
    ptx::chain_point();
    const Index first = Index(blockIdx.x) * (256 * DEQUANT_GROUPS) + threadIdx.x, groups = Index(values / 4);
    char4 c[DEQUANT_GROUPS];
    #pragma unroll
    for (int j = 0; j < DEQUANT_GROUPS; ++j)
        if (first + j * 256 < groups) c[j] = __ldg(reinterpret_cast<const char4*>(codes) + first + j * 256);
    #pragma unroll
    for (int j = 0; j < DEQUANT_GROUPS; ++j) {
        const Index group = first + j * 256;
        if (group >= groups) continue;
        const Index row = group * 4 / uint32_t(K);
        const uint32_t column = uint32_t(group * 4 - row * uint32_t(K));
        float s[4];
        s[0] = s[1] = s[2] = s[3] = __ldg(scales + row);
        if (column + 3 >= uint32_t(K)) {
            #pragma unroll
            for (int i = 1; i < 4; ++i) s[i] = __ldg(scales + (group * 4 + i) / uint32_t(K));
        }
        reinterpret_cast<float4*>(out)[group] = make_float4(float(c[j].x) * s[0], float(c[j].y) * s[1], float(c[j].z) * s[2], float(c[j].w) * s[3]);
    }
    if (blockIdx.x == 0 && threadIdx.x < values % 4) {          // what is left behind the last group
        const size_t i = values / 4 * 4 + threadIdx.x;
        out[i] = float(codes[i]) * __ldg(scales + i / uint32_t(K));
    }
}

template <typename T, bool ROUTED>
void launch(const void* x, int8_t* codes, float* scales, long long rows, int K, const int* position, const int* live, int topk,
            cudaStream_t stream) {
    auto go = [&](auto kernel, int threads, int per_block = 1) {
        launch_chained(kernel, dim3(unsigned((rows + per_block - 1) / per_block)), dim3(threads), 0, stream,
                       static_cast<const T*>(x), codes, scales, rows, K, position, live, topk);
        g_launches.fetch_add(1, std::memory_order_relaxed);
    };
    const int groups = K / 16;
    // As many warps as hold the row, `most` threads at most.
    auto block = [&](int held, int most) { return std::max(64, std::min(most, (groups + 32 * held - 1) / (32 * held) * 32)); };
    // A group held is 8 registers of 16-bit values and 16 of FP32: of those no more than two, as blocks of one SM are to be
    // at different points of their rows. Longer FP32 rows are read again from L2 (K = 28672 1.65 times the time its bytes
    // take, with four groups 2.2; 14336 in one group to a thread 1.24, in two 1.4; 12288 1.27 and 1.16). 16-bit rows of 4608
    // to 16384 values take 1.00 to 1.04 times what their bytes take.
    constexpr bool SHORT = sizeof(T) == 2;
    constexpr int MOST = SHORT ? 4 : 2;
    if (K % 16 || groups > (SHORT ? 2048 : 1024)) {
        if constexpr (!ROUTED) {                                 // (routed rows are whole groups: here only the longest)
            if (groups <= 8) return go(int8_quantise_kernel<T, 8, 1, ROUTED, false>, 256, 32);
            if (groups <= 16) return go(int8_quantise_kernel<T, 16, 1, ROUTED, false>, 256, 16);
            if (groups <= 64) return go(int8_quantise_kernel<T, 32, 2, ROUTED, false>, 256, 8);
            if (groups <= 512) return go(int8_quantise_kernel<T, 256, 2, ROUTED, false>, block(2, 256));
        }
        go(int8_quantise_kernel<T, 512, MOST, ROUTED, false>, block(MOST, 512));
    } else if (groups <= 4) go(int8_quantise_kernel<T, 4, 1, ROUTED, true>, 256, 64);
    else if (groups <= 8) go(int8_quantise_kernel<T, 8, 1, ROUTED, true>, 256, 32);
    else if (groups <= 16) go(int8_quantise_kernel<T, 16, 1, ROUTED, true>, 256, 16);
    else if (groups <= 32) go(int8_quantise_kernel<T, 32, 1, ROUTED, true>, 256, 8);
    else if (groups <= 64) go(int8_quantise_kernel<T, 32, 2, ROUTED, true>, 256, 8);
    else if constexpr (SHORT) {
        if (groups <= 96) go(int8_quantise_kernel<T, 32, 3, ROUTED, true>, 256, 8);
        else if (groups <= 128) go(int8_quantise_kernel<T, 32, 4, ROUTED, true>, 256, 8);
        else if (groups <= 512) go(int8_quantise_kernel<T, 256, 2, ROUTED, true>, block(2, 256));
        else if (groups <= 1024) go(int8_quantise_kernel<T, 256, 4, ROUTED, true>, block(4, 256));
        else go(int8_quantise_kernel<T, 512, 4, ROUTED, true>, block(4, 512));
    } else {
        if (groups <= 256) go(int8_quantise_kernel<T, 256, 1, ROUTED, true>, block(1, 256));
        else if (groups <= 512) go(int8_quantise_kernel<T, 256, 2, ROUTED, true>, block(2, 256));
        else if (groups <= 768) go(int8_quantise_kernel<T, 512, 2, ROUTED, true>, block(2, 512));
        else go(int8_quantise_kernel<T, 1024, 1, ROUTED, true>, block(1, 1024));
    }
}

template <bool ROUTED>
void dispatch(const void* x, int dtype, int8_t* codes, float* scales, long long rows, int K, const int* position, const int* live,
              int topk, cudaStream_t stream) {
    switch (dtype) {
        case DTYPE_BF16: return launch<__nv_bfloat16, ROUTED>(x, codes, scales, rows, K, position, live, topk, stream);
        case DTYPE_F16: return launch<__half, ROUTED>(x, codes, scales, rows, K, position, live, topk, stream);
        case DTYPE_F32: return launch<float, ROUTED>(x, codes, scales, rows, K, position, live, topk, stream);
        default: throw std::invalid_argument("int8: dtype must be 0 (bf16), 1 (fp16) or 2 (fp32)");
    }
}

void check_rows(long long rows, int K) {
    if (rows < 0 || rows > 0x7FFFFFFFll || K < 1) throw std::invalid_argument("int8 quantise: rows must be 0..2^31-1 and K positive");
}

}  // namespace

void int8_quantise(const void* x, int dtype, int8_t* codes, float* scales, long long rows, int K, cudaStream_t stream) {
    check_rows(rows, K);
    if (rows == 0) return;
    if (!x || !codes || !scales) throw std::invalid_argument("int8 quantise: null pointer");
    if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(codes)) & 15)
        throw std::invalid_argument("int8 quantise: x and codes must be 16-byte aligned");
    dispatch<false>(x, dtype, codes, scales, rows, K, nullptr, nullptr, 1, stream);
}

void int8_gather(const void* x, int dtype, long long tokens, int topk, int K, const int* position, const int* live, int8_t* codes,
                 float* scales, cudaStream_t stream) {
    check_rows(tokens, K);
    if (topk < 1 || tokens * topk > 0x7FFFFFFFll) throw std::invalid_argument("int8 gather: topk must be positive and tokens * topk below 2^31");
    if (K % 16) throw std::invalid_argument("int8 gather: K must be a multiple of 16 (as the product of the rows wants it)");
    if (tokens == 0) return;
    if (!x || !codes || !scales || !position || !live) throw std::invalid_argument("int8 gather: null pointer");
    if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(codes)) & 15)
        throw std::invalid_argument("int8 gather: x and codes must be 16-byte aligned");
    dispatch<true>(x, dtype, codes, scales, tokens, K, position, live, topk, stream);
}

void int8_dequantise(const int8_t* codes, const float* scales, float* out, long long rows, int K, cudaStream_t stream) {
    check_rows(rows, K);
    if (rows == 0) return;
    if (!codes || !scales || !out) throw std::invalid_argument("int8 dequantise: null pointer");
    if ((reinterpret_cast<uintptr_t>(codes) | reinterpret_cast<uintptr_t>(out)) & 15)
        throw std::invalid_argument("int8 dequantise: codes and out must be 16-byte aligned");
    const size_t values = size_t(rows) * K, blocks = (values + 4 * 256 * DEQUANT_GROUPS - 1) / (4 * 256 * DEQUANT_GROUPS);
    if (blocks > 0x7FFFFFFFull) throw std::invalid_argument("int8 dequantise: too many values");
    auto kernel = values < (size_t(1) << 31) ? int8_dequantise_kernel<uint32_t> : int8_dequantise_kernel<size_t>;
    launch_chained(kernel, dim3(unsigned(blocks)), dim3(256), 0, stream, codes, scales, out, values, K);
    g_launches.fetch_add(1, std::memory_order_relaxed);
}

}  // namespace nvfp4_b200
