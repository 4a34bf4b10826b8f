// Tokens to their experts' rows and back, for sm_100a: the stable order of a router's choices, the copy of the tokens'
// rows into that order, the weighted sum of the experts' rows, and the gradients of both.
//
// A route is one of a token's topk choices; route i belongs to token i / topk. The order gives every route a row:
// expert by expert, inside an expert in the order of the routes, and behind the last expert the routes of no expert
// (ids outside [0, experts)). position[i] is route i's row, source[r] the route of row r, offsets[e] the first row of
// expert e, offsets[experts] the number of live rows. Rows at or beyond it belong to dropped routes: they are zeros
// where this file writes rows, and are not read where it reads them.
#include "operators_internal.h"
#include "ptx.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

namespace nvfp4_b200 {
namespace {

// ---- the order ------------------------------------------------------------------------------------------------------
// A counting sort in one launch of one cluster. The routes are cut into one contiguous part per warp of the cluster; a
// warp counts its part in a row of counters of its own, 32 routes at a time (lanes with the same expert find each other
// by __match_any_sync, the lowest of them adds their number), so no atomics are needed and the order is stable. Sums
// over the warps and, through distributed shared memory, over the CTAs give each (warp, expert) its first row; a second
// walk over the same routes hands the rows out. The bytes are nothing (1 MB at 131072 routes): latency is the bound.
constexpr int SORT_MAX_EXPERTS = 1024;

template <typename Id, int THREADS>
__global__ void __launch_bounds__(THREADS)
tokens_sort_kernel(const Id* __restrict__ ids, int routes, int experts, int* __restrict__ offsets, int* __restrict__ position,
                   int* __restrict__ source) {
    ptx::chain_point();
    constexpr int WARPS = THREADS / 32;
    const int keys = experts + 1;                               // the last one: dropped
    extern __shared__ int counters[];                           // [WARPS][keys], then the CTA's totals and first rows [keys] each
    int* totals = counters + WARPS * keys;
    int* first = totals + keys;
    __shared__ int warp_sum[WARPS];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    uint32_t ctas;
    asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(ctas));
    const uint32_t rank = ptx::cluster_ctarank();
    for (int i = threadIdx.x; i < WARPS * keys; i += THREADS) counters[i] = 0;
    __syncthreads();
    const long long parts = (long long)(ctas) * WARPS;
    const long long part = ((routes + parts - 1) / parts + 31) / 32 * 32;
    const long long begin = (long long)(rank * WARPS + warp) * part;
    const int steps = begin < routes ? int((min((long long)(routes), begin + part) - begin + 31) / 32) : 0;
    int* own = counters + warp * keys;
    auto key_of = [&](int step) {
        const long long i = begin + step * 32 + lane;
        if (step >= steps || i >= routes) return -1;            // no route: matches only its own kind
        const long long id = (long long)(__ldg(ids + i));
        return id >= 0 && id < experts ? int(id) : experts;
    };
    // The keys of four steps are loaded ahead of the four that are counted.
    auto walk = [&](auto&& body) {
        int ahead[4];
        #pragma unroll
        for (int j = 0; j < 4; ++j) ahead[j] = key_of(j);
        for (int step = 0; step < steps; step += 4) {
            int now[4];
            #pragma unroll
            for (int j = 0; j < 4; ++j) { now[j] = ahead[j]; ahead[j] = key_of(step + 4 + j); }
            #pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t peers = __match_any_sync(0xFFFFFFFFu, now[j]);
                body(step + j, now[j], peers);
                __syncwarp();
            }
        }
    };
    walk([&](int, int key, uint32_t peers) {
        if (key >= 0 && lane == __ffs(peers) - 1) own[key] += __popc(peers);
    });
    __syncthreads();
    for (int e = threadIdx.x; e < keys; e += THREADS) {         // counts -> routes of the same expert in the warps before
        int sum = 0;
        #pragma unroll 8
        for (int w = 0; w < WARPS; ++w) {
            const int c = counters[w * keys + e];
            counters[w * keys + e] = sum;
            sum += c;
        }
        totals[e] = sum;
    }
    __syncwarp();
    ptx::cluster_arrive();
    ptx::cluster_wait();
    // Every CTA: the routes of each expert in the whole cluster and in the CTAs before it, and the sum of the former over
    // the experts before, a run of consecutive experts per thread.
    const int run = (experts + THREADS - 1) / THREADS, e0 = min(experts, int(threadIdx.x) * run), e1 = min(experts, e0 + run);
    int sum = 0;
    for (int e = e0; e < e1; ++e) {
        int all = 0, before = 0;
        for (uint32_t c = 0; c < ctas; ++c) {
            int n;
            asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(n) : "r"(ptx::map_to_cta(ptx::smem_u32(totals + e), c)) : "memory");
            before += c < rank ? n : 0;
            all += n;
        }
        first[e] = sum + before;                                // still without the experts of the threads before
        sum += all;
    }
    int dropped_before = 0;
    if (threadIdx.x == 0) {
        for (uint32_t c = 0; c < rank; ++c) {
            int n;
            asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(n) : "r"(ptx::map_to_cta(ptx::smem_u32(totals + experts), c)) : "memory");
            dropped_before += n;
        }
    }
    __syncwarp();
    ptx::cluster_arrive();                                      // (waited for at the end: the others may still be reading)
    int upto = sum;                                             // inclusive over the warp
    #pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const int n = __shfl_up_sync(0xFFFFFFFFu, upto, d);
        if (lane >= d) upto += n;
    }
    if (lane == 31) warp_sum[warp] = upto;
    __syncthreads();
    int start = upto - sum, total = 0;
    #pragma unroll
    for (int w = 0; w < WARPS; ++w) {
        const int n = warp_sum[w];
        start += w < warp ? n : 0;
        total += n;
    }
    // offsets[e] is the first row of e over all CTAs; this CTA's first row lies behind those of the CTAs before it
    if (rank == 0) {
        for (int e = e0; e < e1; ++e) offsets[e] = start + first[e];
        if (threadIdx.x == 0) offsets[experts] = total;
    }
    for (int e = e0; e < e1; ++e) first[e] += start;
    if (threadIdx.x == 0) first[experts] = total + dropped_before;
    __syncthreads();
    walk([&](int step, int key, uint32_t peers) {
        const int leader = __ffs(peers) - 1;
        int row = 0;
        if (key >= 0 && lane == leader) {
            row = first[key] + own[key];
            own[key] += __popc(peers);
        }
        row = __shfl_sync(0xFFFFFFFFu, row, leader);
        if (key >= 0) {
            const long long i = begin + step * 32 + lane;
            row += __popc(peers & ((1u << lane) - 1u));
            position[i] = row;
            source[row] = int(i);
        }
    });
    __syncwarp();
    ptx::cluster_wait();
}

// ---- rows -------------------------------------------------------------------------------------------------------------

template <typename T> __device__ __forceinline__ float widen(T v);
template <> __device__ __forceinline__ float widen(float v) { return v; }
template <> __device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float widen(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T narrow(float v);
template <> __device__ __forceinline__ float narrow(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 narrow(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half narrow(float v) { return __float2half_rn(v); }

// N values of T, loaded and stored at once: 16 bytes, or one value where rows do not start on 16-byte boundaries.
template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
    T v[N];
};
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> load(const T* p) {
    if constexpr (sizeof(T) * N == 16) {
        const uint4 raw = __ldg(reinterpret_cast<const uint4*>(p));
        return *reinterpret_cast<const Pack<T, N>*>(&raw);
    } else {
        return *reinterpret_cast<const Pack<T, N>*>(p);
    }
}
template <typename T, int N>
__device__ __forceinline__ void store(T* p, const Pack<T, N>& v) {
    if constexpr (sizeof(T) * N == 16) *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(&v);
    else *reinterpret_cast<Pack<T, N>*>(p) = v;
}
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> zeros() {
    Pack<T, N> z;
    #pragma unroll
    for (int i = 0; i < N; ++i) z.v[i] = narrow<T>(0.0f);
    return z;
}

constexpr int ROW_THREADS = 128;
constexpr int GATHER_PACKS = 2;                                 // packs of a row per thread

// rows[position[t, j]] = x[t] for every route j of token t: the token's row is read once. One block per token and
// segment of the row.
template <typename T, int N>
__global__ void __launch_bounds__(ROW_THREADS)
tokens_gather_kernel(const T* __restrict__ x, T* __restrict__ rows, const int* __restrict__ position, const int* __restrict__ live,
                     int tokens, int topk, int hidden, int segments) {
    ptx::chain_point();
    const int token = blockIdx.x / segments, packs = hidden / N;
    const int p0 = (blockIdx.x - token * segments) * (ROW_THREADS * GATHER_PACKS) + threadIdx.x;
    Pack<T, N> v[GATHER_PACKS];
    #pragma unroll
    for (int u = 0; u < GATHER_PACKS; ++u)
        if (p0 + u * ROW_THREADS < packs) v[u] = load<T, N>(x + size_t(token) * hidden + size_t(p0 + u * ROW_THREADS) * N);
    const int end_live = __ldg(live);
    for (int j = 0; j < topk; ++j) {
        const int to = __ldg(position + size_t(token) * topk + j);
        if (to < 0 || to >= tokens * topk) continue;
        #pragma unroll
        for (int u = 0; u < GATHER_PACKS; ++u)
            if (p0 + u * ROW_THREADS < packs)
                store<T, N>(rows + size_t(to) * hidden + size_t(p0 + u * ROW_THREADS) * N, to < end_live ? v[u] : zeros<T, N>());
    }
}

// y[t] = sum over the live routes j of token t, in their order, of weights[t, j] * rows[position[t, j]] (weights null: of
// the rows as they are, which is the gradient of the gather): FP32 sums, rounded once. Up to eight rows are in flight.
template <typename T, int N, bool WEIGHTED>
__global__ void __launch_bounds__(ROW_THREADS)
tokens_combine_kernel(const T* __restrict__ rows, const float* __restrict__ weights, const int* __restrict__ position,
                      const int* __restrict__ live, int tokens, int topk, int hidden, int segments, T* __restrict__ y) {
    ptx::chain_point();
    constexpr int AHEAD = 8;
    const int token = blockIdx.x / segments, packs = hidden / N;
    const int p = (blockIdx.x - token * segments) * ROW_THREADS + threadIdx.x;
    if (p >= packs) return;
    const int end_live = min(__ldg(live), tokens * topk);
    float sum[N];
    #pragma unroll
    for (int i = 0; i < N; ++i) sum[i] = 0.0f;
    for (int j0 = 0; j0 < topk; j0 += AHEAD) {
        Pack<T, N> v[AHEAD];
        int from[AHEAD];
        #pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            from[j] = j0 + j < topk ? __ldg(position + size_t(token) * topk + j0 + j) : -1;
            if (from[j] >= end_live) from[j] = -1;
            if (from[j] >= 0) v[j] = load<T, N>(rows + size_t(from[j]) * hidden + size_t(p) * N);
        }
        #pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            if (from[j] < 0) continue;
            const float w = WEIGHTED ? __ldg(weights + size_t(token) * topk + j0 + j) : 1.0f;
            #pragma unroll
            for (int i = 0; i < N; ++i) sum[i] = WEIGHTED ? __fmaf_rn(w, widen(v[j].v[i]), sum[i]) : sum[i] + widen(v[j].v[i]);
        }
    }
    Pack<T, N> out;
    #pragma unroll
    for (int i = 0; i < N; ++i) out.v[i] = narrow<T>(sum[i]);
    store<T, N>(y + size_t(token) * hidden + size_t(p) * N, out);
}

// d_rows[position[t, j]] = weights[t, j] * d_y[t] (null: not asked for), d_weights[t, j] = <d_y[t], rows[position[t, j]]>
// (null: not asked for, the rows are then not read). A block per token: the token's gradient is read once for eight
// routes, whose sums stay in registers; lanes, then warps, are added in a fixed order.
template <typename T, int N>
__global__ void __launch_bounds__(256)
tokens_combine_backward_kernel(const T* __restrict__ d_y, const T* __restrict__ rows, const float* __restrict__ weights,
                               const int* __restrict__ position, const int* __restrict__ live, int tokens, int topk, int hidden,
                               T* __restrict__ d_rows, float* __restrict__ d_weights) {
    ptx::chain_point();
    constexpr int GROUP = 8, WARPS = 8;
    __shared__ float partial[GROUP][WARPS];
    const int token = blockIdx.x, packs = hidden / N, end_live = __ldg(live);
    for (int j0 = 0; j0 < topk; j0 += GROUP) {
        int at[GROUP];
        float w[GROUP], dot[GROUP];
        #pragma unroll
        for (int j = 0; j < GROUP; ++j) {
            at[j] = j0 + j < topk ? __ldg(position + size_t(token) * topk + j0 + j) : -1;
            if (at[j] >= tokens * topk) at[j] = -1;
            w[j] = at[j] >= 0 && at[j] < end_live ? __ldg(weights + size_t(token) * topk + j0 + j) : 0.0f;
            dot[j] = 0.0f;
        }
        for (int p = threadIdx.x; p < packs; p += 256) {
            const Pack<T, N> g = load<T, N>(d_y + size_t(token) * hidden + size_t(p) * N);
            #pragma unroll
            for (int j = 0; j < GROUP; ++j) {
                if (at[j] < 0) continue;
                const size_t place = size_t(at[j]) * hidden + size_t(p) * N;
                if (d_weights && at[j] < end_live) {
                    const Pack<T, N> r = load<T, N>(rows + place);
                    #pragma unroll
                    for (int i = 0; i < N; ++i) dot[j] = __fmaf_rn(widen(g.v[i]), widen(r.v[i]), dot[j]);
                }
                if (d_rows) {
                    Pack<T, N> out;
                    #pragma unroll
                    for (int i = 0; i < N; ++i) out.v[i] = narrow<T>(at[j] < end_live ? w[j] * widen(g.v[i]) : 0.0f);
                    store<T, N>(d_rows + place, out);
                }
            }
        }
        if (!d_weights) continue;
        #pragma unroll
        for (int j = 0; j < GROUP; ++j) {
            #pragma unroll
            for (int d = 16; d > 0; d /= 2) dot[j] += __shfl_xor_sync(0xFFFFFFFFu, dot[j], d);
            if (threadIdx.x % 32 == 0) partial[j][threadIdx.x / 32] = dot[j];
        }
        __syncthreads();
        if (threadIdx.x < GROUP && j0 + int(threadIdx.x) < topk) {
            float sum = 0.0f;
            #pragma unroll
            for (int i = 0; i < WARPS; ++i) sum += partial[threadIdx.x][i];
            d_weights[size_t(token) * topk + j0 + threadIdx.x] = sum;
        }
        __syncthreads();
    }
}

void check_routes(int tokens, int topk, int hidden) {
    if (tokens < 0 || topk < 1 || hidden < 1) throw std::invalid_argument("tokens: topk and hidden must be positive, tokens not negative");
    if ((long long)(tokens) * topk > 0x7FFFFFFFll) throw std::invalid_argument("tokens: tokens * topk must be below 2^31");
}

bool whole_packs(int hidden, size_t size, std::initializer_list<const void*> pointers) {
    uintptr_t bits = 0;
    for (const void* p : pointers) bits |= reinterpret_cast<uintptr_t>(p);
    return size_t(hidden) * size % 16 == 0 && (bits & 15) == 0;
}

// The grid of (token, segment of `per` packs) blocks.
unsigned blocks(int tokens, int packs, int per, int& segments) {
    segments = (packs + per - 1) / per;
    const long long n = (long long)(tokens) * segments;
    if (n > 0x7FFFFFFFll) throw std::invalid_argument("tokens: too many rows for one launch");
    return unsigned(n);
}

// body(value of the type, number of values per pack)
template <typename F>
void by_type(int dtype, bool whole, F&& body) {
    auto with = [&](auto value) {
        using T = decltype(value);
        if (whole) body(value, std::integral_constant<int, int(16 / sizeof(T))>{});
        else body(value, std::integral_constant<int, 1>{});
    };
    switch (dtype) {
        case DTYPE_BF16: return with(__nv_bfloat16{});
        case DTYPE_F16: return with(__half{});
        case DTYPE_F32: return with(float{});
        default: throw std::invalid_argument("tokens: dtype must be 0 (bf16), 1 (fp16) or 2 (fp32)");
    }
}

template <typename Id, int THREADS>
void launch_sort(const void* ids, int routes, int experts, int* offsets, int* position, int* source, unsigned ctas, cudaStream_t stream) {
    auto kernel = tokens_sort_kernel<Id, THREADS>;
    const size_t smem = size_t(THREADS / 32 + 2) * (experts + 1) * sizeof(int);
    if (smem > 48 * 1024) cuda_check(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)));
    cudaLaunchAttribute attrs[2]{};
    attrs[0].id = cudaLaunchAttributeClusterDimension;
    attrs[0].val.clusterDim = {ctas, 1, 1};
    attrs[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[1].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = attrs;
    cfg.numAttrs = 2;
    cuda_check(cudaLaunchKernelEx(&cfg, kernel, static_cast<const Id*>(ids), routes, experts, offsets, position, source));
    g_launches.fetch_add(1, std::memory_order_relaxed);
}

}  // namespace

void tokens_sort(const void* ids, int id_bytes, int routes, int experts, int* offsets, int* position, int* source, cudaStream_t stream) {
    if (experts < 1 || experts > SORT_MAX_EXPERTS) throw std::invalid_argument("tokens sort: 1..1024 experts");
    if (routes < 0) throw std::invalid_argument("tokens sort: the number of routes must not be negative");
    if (id_bytes != 4 && id_bytes != 8) throw std::invalid_argument("tokens sort: ids are 32- or 64-bit integers");
    if (!offsets || (routes > 0 && (!ids || !position || !source))) throw std::invalid_argument("tokens sort: null pointer");
    // A small batch is sorted by one CTA of eight warps; from 2048 routes on eight CTAs of 32 share them.
    const bool small = routes < 2048;
    if (id_bytes == 8) {
        if (small) launch_sort<long long, 256>(ids, routes, experts, offsets, position, source, 1, stream);
        else launch_sort<long long, 1024>(ids, routes, experts, offsets, position, source, 8, stream);
    } else {
        if (small) launch_sort<int, 256>(ids, routes, experts, offsets, position, source, 1, stream);
        else launch_sort<int, 1024>(ids, routes, experts, offsets, position, source, 8, stream);
    }
}

void tokens_gather(const void* x, int dtype, int tokens, int topk, int hidden, const int* position, const int* live, void* rows,
                   cudaStream_t stream) {
    check_routes(tokens, topk, hidden);
    if (tokens == 0) return;
    if (!x || !position || !live || !rows) throw std::invalid_argument("tokens gather: null pointer");
    by_type(dtype, whole_packs(hidden, dtype_bytes(dtype), {x, rows}), [&](auto value, auto n) {
        using T = decltype(value);
        constexpr int N = decltype(n)::value;
        int segments;
        const unsigned grid = blocks(tokens, hidden / N, ROW_THREADS * GATHER_PACKS, segments);
        launch_chained(tokens_gather_kernel<T, N>, dim3(grid), dim3(ROW_THREADS), 0, stream, static_cast<const T*>(x),
                       static_cast<T*>(rows), position, live, tokens, topk, hidden, segments);
    });
    g_launches.fetch_add(1, std::memory_order_relaxed);
}

void tokens_combine(const void* rows, int dtype, const float* weights, const int* position, const int* live, int tokens, int topk,
                    int hidden, void* y, cudaStream_t stream) {
    check_routes(tokens, topk, hidden);
    if (tokens == 0) return;
    if (!rows || !position || !live || !y) throw std::invalid_argument("tokens combine: null pointer");
    by_type(dtype, whole_packs(hidden, dtype_bytes(dtype), {rows, y}), [&](auto value, auto n) {
        using T = decltype(value);
        constexpr int N = decltype(n)::value;
        int segments;
        const unsigned grid = blocks(tokens, hidden / N, ROW_THREADS, segments);
        auto kernel = weights ? tokens_combine_kernel<T, N, true> : tokens_combine_kernel<T, N, false>;
        launch_chained(kernel, dim3(grid), dim3(ROW_THREADS), 0, stream, static_cast<const T*>(rows), weights, position, live, tokens,
                       topk, hidden, segments, static_cast<T*>(y));
    });
    g_launches.fetch_add(1, std::memory_order_relaxed);
}

void tokens_combine_backward(const void* d_y, int dtype, const void* rows, const float* weights, const int* position,
                             const int* live, int tokens, int topk, int hidden, void* d_rows, float* d_weights, cudaStream_t stream) {
    check_routes(tokens, topk, hidden);
    if (tokens == 0 || (!d_rows && !d_weights)) return;
    if (!d_y || !weights || !position || !live || (d_weights && !rows)) throw std::invalid_argument("tokens combine backward: null pointer");
    by_type(dtype, whole_packs(hidden, dtype_bytes(dtype), {d_y, rows, d_rows}), [&](auto value, auto n) {
        using T = decltype(value);
        constexpr int N = decltype(n)::value;
        launch_chained(tokens_combine_backward_kernel<T, N>, dim3(unsigned(tokens)), dim3(256), 0, stream, static_cast<const T*>(d_y),
                       static_cast<const T*>(rows), weights, position, live, tokens, topk, hidden, static_cast<T*>(d_rows), d_weights);
    });
    g_launches.fetch_add(1, std::memory_order_relaxed);
}

}  // namespace nvfp4_b200
