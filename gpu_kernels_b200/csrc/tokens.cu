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
#include <climits>

namespace nvfp4_b200 {
namespace {

// ---- the order ------------------------------------------------------------------------------------------------------
// A stable counting sort. The bytes are nothing (2 MB at 131072 routes); latency is the bound, and on few SMs the 4-byte
// stores of `source`, each in a sector of its own: as one cluster of eight CTAs 131072 routes of 256 experts took 32 us, on
// 64 CTAs they take 14 (six routes, one token's: 1.8 us).
// Three forms: up to SMALL routes every route is compared with every other; up to one block's worth (BLOCK) one CTA
// counts and hands out rows; beyond, a first launch counts each block's routes and a second one, with a CTA for each of
// the same blocks, adds up the counts of the blocks before its own.
constexpr int SORT_MAX_EXPERTS = 1024;
constexpr int SMALL = 256, BLOCK = 1024, SORT_WARPS = BLOCK / 32;
constexpr size_t SORT_STATIC = SORT_WARPS * sizeof(int);        // tokens_sort_kernel's static shared memory, which counts as well

template <typename Id>
__device__ __forceinline__ int key_of(const Id* ids, long long i, int experts) {
    const long long id = (long long)(__ldg(ids + i));
    return id >= 0 && id < experts ? int(id) : experts;         // `experts`: dropped
}

// A route's row is the number of routes with a smaller key, or with the same key in front of it; an expert's first row is
// the number of routes with a smaller key.
template <typename Id>
__global__ void __launch_bounds__(SMALL)
tokens_sort_small_kernel(const Id* __restrict__ ids, int routes, int experts, int* __restrict__ offsets, int* __restrict__ position,
                         int* __restrict__ source) {
    ptx::chain_point();
    __shared__ __align__(16) int keys[SMALL];
    const int i = threadIdx.x, own = i < routes ? key_of(ids, i, experts) : INT_MAX;
    keys[i] = own;
    __syncthreads();
    const int4* four = reinterpret_cast<const int4*>(keys);
    const int fours = (routes + 3) / 4;
    int row = 0;
    #pragma unroll 4
    for (int j = 0; j < fours; ++j) {
        const int4 k = four[j];
        row += (k.x < own || (k.x == own && 4 * j < i)) + (k.y < own || (k.y == own && 4 * j + 1 < i)) +
               (k.z < own || (k.z == own && 4 * j + 2 < i)) + (k.w < own || (k.w == own && 4 * j + 3 < i));
    }
    if (i < routes) {
        position[i] = row;
        source[row] = i;
    }
    for (int e = i; e <= experts; e += SMALL) {
        int first = 0;
        #pragma unroll 4
        for (int j = 0; j < fours; ++j) {
            const int4 k = four[j];
            first += (k.x < e) + (k.y < e) + (k.z < e) + (k.w < e);
        }
        offsets[e] = first;
    }
}

// counts[block][key]: the routes of each key (dropped ones last) in a block of `part` routes.
template <typename Id>
__global__ void __launch_bounds__(BLOCK)
tokens_count_kernel(const Id* __restrict__ ids, int routes, int experts, int part, int* __restrict__ counts) {
    ptx::chain_point();
    extern __shared__ int count[];
    for (int e = threadIdx.x; e <= experts; e += BLOCK) count[e] = 0;
    __syncthreads();
    const long long begin = (long long)(blockIdx.x) * part, end = min((long long)(routes), begin + part);
    for (long long i = begin + threadIdx.x; i < end; i += BLOCK) atomicAdd(&count[key_of(ids, i, experts)], 1);
    __syncthreads();
    for (int e = threadIdx.x; e <= experts; e += BLOCK) counts[size_t(blockIdx.x) * (experts + 1) + e] = count[e];
}

// A warp counts a contiguous part of its block's routes in a row of counters of its own, 32 routes at a time: lanes with
// the same expert find each other by one ballot per bit of the key, the lowest of them adds their number, so no atomics
// are needed and the order is stable. Sums over the warps and the blocks before give each (warp, expert) its first row; a
// second walk over the same routes hands the rows out.
template <typename Id>
__global__ void __launch_bounds__(BLOCK)
tokens_sort_kernel(const Id* __restrict__ ids, int routes, int experts, int part, const int* __restrict__ counts,
                   int* __restrict__ offsets, int* __restrict__ position, int* __restrict__ source) {
    ptx::chain_point();
    const int keys = experts + 1, bits = 32 - __clz(experts);
    extern __shared__ int counters[];                           // [SORT_WARPS][keys], then for each key, [keys] each:
    int* first = counters + SORT_WARPS * keys;                  // its routes in the blocks before, later its first row in this block
    int* others = first + keys;                                 // its routes in the other blocks
    __shared__ int warp_sum[SORT_STATIC / sizeof(int)];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    for (int i = threadIdx.x; i < (SORT_WARPS + 2) * keys; i += BLOCK) counters[i] = 0;
    __syncthreads();
    if (counts) {
        const int all = int(gridDim.x) * keys, mine = int(blockIdx.x) * keys;
        #pragma unroll 8
        for (int i = threadIdx.x; i < all; i += BLOCK) {
            const int n = __ldcg(counts + i), e = i % keys;
            if (n == 0) continue;
            if (i < mine) atomicAdd(first + e, n);
            if (i < mine || i >= mine + keys) atomicAdd(others + e, n);
        }
    }
    const int per_warp = part / SORT_WARPS;                     // a multiple of 32
    const long long begin = (long long)(blockIdx.x) * part + warp * per_warp;
    const int steps = begin < routes ? int((min((long long)(routes), begin + per_warp) - begin + 31) / 32) : 0;
    int* own = counters + warp * keys;
    auto walk = [&](auto&& body) {
        auto key = [&](int step) {
            const long long i = begin + step * 32 + lane;
            return step < steps && i < routes ? key_of(ids, i, experts) : -1;
        };
        int next = key(0);
        for (int step = 0; step < steps; ++step) {
            const int now = next;
            next = key(step + 1);
            uint32_t peers = __ballot_sync(0xFFFFFFFFu, now >= 0);
            for (int b = 0; b < bits; ++b) {
                const bool set = (now >> b) & 1;
                const uint32_t same = __ballot_sync(0xFFFFFFFFu, set);
                peers &= set ? same : ~same;
            }
            body(step, now, peers);
            __syncwarp();
        }
    };
    walk([&](int, int key, uint32_t peers) {
        if (key >= 0 && lane == __ffs(peers) - 1) own[key] += __popc(peers);
    });
    __syncthreads();
    // A run of consecutive keys per thread: the routes of each in all blocks, and the first row of each in this block (in
    // front of it: the smaller keys of all blocks, the same key of the blocks before).
    const int run = (keys + BLOCK - 1) / BLOCK, e0 = min(keys, int(threadIdx.x) * run), e1 = min(keys, e0 + run);
    int sum = 0;
    for (int e = e0; e < e1; ++e) {
        int here = 0;
        #pragma unroll 8
        for (int w = 0; w < SORT_WARPS; ++w) {
            const int c = counters[w * keys + e];
            counters[w * keys + e] = here;
            here += c;
        }
        first[e] += sum;                                        // still without the keys of the threads before
        sum += here + others[e];
    }
    int upto = sum;                                             // inclusive over the warp
    #pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const int n = __shfl_up_sync(0xFFFFFFFFu, upto, d);
        if (lane >= d) upto += n;
    }
    if (lane == 31) warp_sum[warp] = upto;
    __syncthreads();
    int start = upto - sum;
    #pragma unroll
    for (int w = 0; w < SORT_WARPS; ++w) start += w < warp ? warp_sum[w] : 0;
    for (int e = e0; e < e1; ++e) {
        first[e] += start;
        if (blockIdx.x == 0) offsets[e] = first[e];             // (no block before the first)
    }
    __syncthreads();
    walk([&](int step, int key, uint32_t peers) {
        const int leader = key >= 0 ? __ffs(peers) - 1 : lane;
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
}

// Blocks of the larger form, and the routes of each (a multiple of BLOCK).
int sort_blocks(int routes, int& part) {
    constexpr int MOST = 64;
    part = int((((long long)(routes) + MOST - 1) / MOST + BLOCK - 1) / BLOCK * BLOCK);
    return int(((long long)(routes) + part - 1) / part);
}

// ---- rows -------------------------------------------------------------------------------------------------------------

template <typename T> struct Format;                            // one 32-bit word as FP32 values, and back
template <> struct Format<float> {
    static __device__ __forceinline__ float get(uint32_t w, int) { return __uint_as_float(w); }
    static __device__ __forceinline__ uint32_t put(float a, float) { return __float_as_uint(a); }
};
template <> struct Format<__nv_bfloat16> {
    static __device__ __forceinline__ float get(uint32_t w, int i) { return __uint_as_float(i ? w & 0xFFFF0000u : w << 16); }
    static __device__ __forceinline__ uint32_t put(float a, float b) {
        const __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&p);
    }
};
template <> struct Format<__half> {
    static __device__ __forceinline__ float get(uint32_t w, int i) { return __half2float(__ushort_as_half(static_cast<unsigned short>(i ? w >> 16 : w))); }
    static __device__ __forceinline__ uint32_t put(float a, float b) {
        const __half2 p = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&p);
    }
};

// N values of T that are loaded and stored at once: 16 bytes, or as many as divide a row where rows do not start on
// 16-byte boundaries.
template <typename T, int N>
struct Pack {
    static constexpr int BYTES = int(sizeof(T)) * N, WORDS = BYTES < 4 ? 1 : BYTES / 4, PER_WORD = 4 / int(sizeof(T));
    using Word = typename std::conditional<BYTES == 16, uint4, typename std::conditional<BYTES == 8, uint2,
                 typename std::conditional<BYTES == 4, uint32_t, unsigned short>::type>::type>::type;
    uint32_t w[WORDS];

    __device__ __forceinline__ void load(const T* p) {
        const Word v = __ldg(reinterpret_cast<const Word*>(p));
        if constexpr (BYTES == 16) { w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w; }
        else if constexpr (BYTES == 8) { w[0] = v.x; w[1] = v.y; }
        else w[0] = v;
    }
    __device__ __forceinline__ void store(T* p) const {
        if constexpr (BYTES == 16) *reinterpret_cast<Word*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
        else if constexpr (BYTES == 8) *reinterpret_cast<Word*>(p) = make_uint2(w[0], w[1]);
        else *reinterpret_cast<Word*>(p) = Word(w[0]);
    }
    __device__ __forceinline__ float operator[](int i) const { return Format<T>::get(w[i / PER_WORD], i % PER_WORD); }
    __device__ __forceinline__ void set(const float (&v)[N]) {
        #pragma unroll
        for (int i = 0; i < N; i += PER_WORD) w[i / PER_WORD] = Format<T>::put(v[i], i + 1 < N ? v[i + 1] : 0.0f);
    }
    __device__ __forceinline__ void clear() {
        #pragma unroll
        for (int i = 0; i < WORDS; ++i) w[i] = 0u;
    }
};

// A block of ROW_THREADS threads per token and segment of its row. A segment is one pack per thread or two, and eight of
// fewer than 16 bytes, whose blocks would be over before they have begun.
constexpr int ROW_THREADS = 128;
constexpr int NARROW = 8;
template <typename T, int N> constexpr int GATHER_PACKS = sizeof(T) * N == 16 ? 2 : NARROW;

// rows[position[t, j]] = x[t] for every route j of token t: the token's row is read once. Bound by HBM, mostly its writes
// (4096 tokens of 4096 bf16 values, topk 6: 38.6 us, 6.1 TB/s).
template <typename T, int N>
__global__ void __launch_bounds__(ROW_THREADS)
tokens_gather_kernel(const T* __restrict__ x, T* __restrict__ rows, const int* __restrict__ position, const int* __restrict__ live,
                     int tokens, int topk, int hidden, int segments) {
    ptx::chain_point();
    constexpr int PACKS = GATHER_PACKS<T, N>;
    const int token = blockIdx.x / segments, packs = hidden / N;
    const int p0 = (blockIdx.x - token * segments) * (ROW_THREADS * PACKS) + threadIdx.x;
    Pack<T, N> v[PACKS];
    #pragma unroll
    for (int u = 0; u < PACKS; ++u)
        if (p0 + u * ROW_THREADS < packs) v[u].load(x + size_t(token) * hidden + size_t(p0 + u * ROW_THREADS) * N);
    const int end_live = __ldg(live);
    for (int j = 0; j < topk; ++j) {
        const int to = __ldg(position + size_t(token) * topk + j);
        if (to < 0 || to >= tokens * topk) continue;
        T* row = rows + size_t(to) * hidden;
        #pragma unroll
        for (int u = 0; u < PACKS; ++u) {
            if (p0 + u * ROW_THREADS >= packs) continue;
            Pack<T, N> out = v[u];
            if (to >= end_live) out.clear();
            out.store(row + size_t(p0 + u * ROW_THREADS) * N);
        }
    }
}

// y[t] = sum over the live routes j of token t, in their order, of weights[t, j] * rows[position[t, j]] (weights null: of
// the rows as they are, which is the gradient of the gather): FP32 sums, rounded once. GROUP rows are in flight at a time,
// PACKS packs of each: about eight loads, since fewer leave HBM waiting (rows of 4096 bf16 values: topk 1 takes 1.26 times
// what its bytes take, with one pack in flight 1.73; topk 2 1.11 and 1.24) and registers bound the rest (topk 8 in two
// rounds of four rows and two packs 1.09, with eight rows at once 1.31; topk 6 with six 1.14).
template <typename T, int GROUP, int PACKS>
__global__ void __launch_bounds__(ROW_THREADS)
tokens_combine_kernel(const T* __restrict__ rows, const float* __restrict__ weights, const int* __restrict__ position,
                      const int* __restrict__ live, int tokens, int topk, int hidden, int segments, T* __restrict__ y) {
    ptx::chain_point();
    constexpr int N = 16 / int(sizeof(T));
    const int token = blockIdx.x / segments, packs = hidden / N;
    const int p = (blockIdx.x - token * segments) * (ROW_THREADS * PACKS) + threadIdx.x;
    if (p >= packs) return;
    const int end_live = min(__ldg(live), tokens * topk);
    float sum[PACKS][N];
    #pragma unroll
    for (int u = 0; u < PACKS; ++u)
        #pragma unroll
        for (int i = 0; i < N; ++i) sum[u][i] = 0.0f;
    for (int j0 = 0; j0 < topk; j0 += GROUP) {
        Pack<T, N> v[GROUP][PACKS];
        bool there[GROUP];
        #pragma unroll
        for (int j = 0; j < GROUP; ++j) {
            const int from = j0 + j < topk ? __ldg(position + size_t(token) * topk + j0 + j) : -1;
            there[j] = from >= 0 && from < end_live;
            #pragma unroll
            for (int u = 0; u < PACKS; ++u)
                if (there[j] && p + u * ROW_THREADS < packs) v[j][u].load(rows + size_t(from) * hidden + size_t(p + u * ROW_THREADS) * N);
        }
        #pragma unroll
        for (int j = 0; j < GROUP; ++j) {
            if (!there[j]) continue;
            const float w = weights ? __ldg(weights + size_t(token) * topk + j0 + j) : 1.0f;
            #pragma unroll
            for (int u = 0; u < PACKS; ++u)
                #pragma unroll
                for (int i = 0; i < N; ++i) sum[u][i] = __fmaf_rn(w, v[j][u][i], sum[u][i]);
        }
    }
    #pragma unroll
    for (int u = 0; u < PACKS; ++u) {
        if (p + u * ROW_THREADS >= packs) break;
        Pack<T, N> out;
        out.set(sum[u]);
        out.store(y + size_t(token) * hidden + size_t(p + u * ROW_THREADS) * N);
    }
}

// The same for rows of narrower packs (an odd number of values, say): eight packs of one row in flight per thread instead
// of one pack of several rows, so that what surrounds a load is paid once for eight (1000 tokens of 2975 bf16 values, topk
// 2: 4.9 us, pack by pack 20.7).
template <typename T, int N>
__global__ void __launch_bounds__(ROW_THREADS)
tokens_combine_narrow_kernel(const T* __restrict__ rows, const float* __restrict__ weights, const int* __restrict__ position,
                             const int* __restrict__ live, int tokens, int topk, int hidden, int segments, T* __restrict__ y) {
    ptx::chain_point();
    const int token = blockIdx.x / segments, packs = hidden / N;
    const int p0 = (blockIdx.x - token * segments) * (ROW_THREADS * NARROW) + threadIdx.x;
    const int end_live = min(__ldg(live), tokens * topk);
    float sum[NARROW][N];
    #pragma unroll
    for (int u = 0; u < NARROW; ++u)
        #pragma unroll
        for (int i = 0; i < N; ++i) sum[u][i] = 0.0f;
    for (int j = 0; j < topk; ++j) {
        const int from = __ldg(position + size_t(token) * topk + j);
        if (from < 0 || from >= end_live) continue;
        const float w = weights ? __ldg(weights + size_t(token) * topk + j) : 1.0f;
        const T* row = rows + size_t(from) * hidden;
        Pack<T, N> v[NARROW];
        #pragma unroll
        for (int u = 0; u < NARROW; ++u)
            if (p0 + u * ROW_THREADS < packs) v[u].load(row + (p0 + u * ROW_THREADS) * N);
        #pragma unroll
        for (int u = 0; u < NARROW; ++u) {
            if (p0 + u * ROW_THREADS >= packs) continue;
            #pragma unroll
            for (int i = 0; i < N; ++i) sum[u][i] = __fmaf_rn(w, v[u][i], sum[u][i]);
        }
    }
    #pragma unroll
    for (int u = 0; u < NARROW; ++u) {
        if (p0 + u * ROW_THREADS >= packs) continue;
        Pack<T, N> out;
        out.set(sum[u]);
        out.store(y + size_t(token) * hidden + (p0 + u * ROW_THREADS) * N);
    }
}

// d_rows[position[t, j]] = weights[t, j] * d_y[t] (null: not asked for), d_weights[t, j] = <d_y[t], rows[position[t, j]]>
// (null: not asked for, the rows are then not read). A block per token: the token's gradient is read once for GROUP
// routes, whose sums stay in registers; lanes, then warps, are added in a fixed order. The rows of all of them are loaded
// before the first store, and registers are capped for six blocks per SM: 4096 tokens of 4096 bf16 values, topk 6, 70.8 us
// (6.2 TB/s); with loads between the stores and 256 threads a block 100 us.
template <typename T, int GROUP>
__global__ void __launch_bounds__(ROW_THREADS, 6)
tokens_combine_backward_kernel(const T* __restrict__ d_y, const T* __restrict__ rows, const float* __restrict__ weights,
                               const int* __restrict__ position, const int* __restrict__ live, int tokens, int topk, int hidden,
                               T* __restrict__ d_rows, float* __restrict__ d_weights) {
    ptx::chain_point();
    constexpr int WARPS = ROW_THREADS / 32, N = 16 / int(sizeof(T));
    __shared__ float partial[GROUP][WARPS];
    const int token = blockIdx.x, packs = hidden / N, end_live = min(__ldg(live), tokens * topk);
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
        for (int p = threadIdx.x; p < packs; p += ROW_THREADS) {
            Pack<T, N> g, r[GROUP];
            g.load(d_y + size_t(token) * hidden + size_t(p) * N);
            if (d_weights) {
                #pragma unroll
                for (int j = 0; j < GROUP; ++j)                 // all the loads before the first store
                    if (at[j] >= 0 && at[j] < end_live) r[j].load(rows + size_t(at[j]) * hidden + size_t(p) * N);
                #pragma unroll
                for (int j = 0; j < GROUP; ++j) {
                    if (at[j] < 0 || at[j] >= end_live) continue;
                    #pragma unroll
                    for (int i = 0; i < N; ++i) dot[j] = __fmaf_rn(g[i], r[j][i], dot[j]);
                }
            }
            if (d_rows) {
                #pragma unroll
                for (int j = 0; j < GROUP; ++j) {
                    if (at[j] < 0) continue;
                    float v[N];
                    #pragma unroll
                    for (int i = 0; i < N; ++i) v[i] = w[j] * g[i];
                    Pack<T, N> out;
                    out.set(v);
                    if (at[j] >= end_live) out.clear();
                    out.store(d_rows + size_t(at[j]) * hidden + size_t(p) * N);
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

// The same for rows of narrower packs: a route at a time, eight packs of its row in flight per thread. The token's gradient
// comes from L1 after the first route.
template <typename T, int N>
__global__ void __launch_bounds__(ROW_THREADS)
tokens_combine_backward_narrow_kernel(const T* __restrict__ d_y, const T* __restrict__ rows, const float* __restrict__ weights,
                                      const int* __restrict__ position, const int* __restrict__ live, int tokens, int topk,
                                      int hidden, T* __restrict__ d_rows, float* __restrict__ d_weights) {
    ptx::chain_point();
    constexpr int WARPS = ROW_THREADS / 32;
    __shared__ float partial[2][WARPS];                         // (two, so that one barrier per route is enough)
    const int token = blockIdx.x, packs = hidden / N, end_live = min(__ldg(live), tokens * topk);
    const T* gradient = d_y + size_t(token) * hidden;
    for (int j = 0; j < topk; ++j) {
        const int at = __ldg(position + size_t(token) * topk + j);
        const bool there = at >= 0 && at < tokens * topk, counts = there && at < end_live;
        const float w = counts ? __ldg(weights + size_t(token) * topk + j) : 0.0f;
        const size_t row = there ? size_t(at) * hidden : 0;
        float dot = 0.0f;
        for (int p0 = threadIdx.x; there && p0 < packs; p0 += ROW_THREADS * NARROW) {
            Pack<T, N> g[NARROW], r[NARROW];
            #pragma unroll
            for (int u = 0; u < NARROW; ++u) {
                if (p0 + u * ROW_THREADS >= packs) continue;
                g[u].load(gradient + (p0 + u * ROW_THREADS) * N);
                if (d_weights && counts) r[u].load(rows + row + (p0 + u * ROW_THREADS) * N);
            }
            #pragma unroll
            for (int u = 0; u < NARROW; ++u) {
                if (p0 + u * ROW_THREADS >= packs) continue;
                float v[N];
                #pragma unroll
                for (int i = 0; i < N; ++i) {
                    if (d_weights && counts) dot = __fmaf_rn(g[u][i], r[u][i], dot);
                    v[i] = w * g[u][i];
                }
                if (!d_rows) continue;
                Pack<T, N> out;
                out.set(v);
                if (!counts) out.clear();
                out.store(d_rows + row + (p0 + u * ROW_THREADS) * N);
            }
        }
        if (!d_weights) continue;
        __syncwarp();
        #pragma unroll
        for (int d = 16; d > 0; d /= 2) dot += __shfl_xor_sync(0xFFFFFFFFu, dot, d);
        if (threadIdx.x % 32 == 0) partial[j % 2][threadIdx.x / 32] = dot;
        __syncthreads();
        if (threadIdx.x == 0) {
            float sum = 0.0f;
            #pragma unroll
            for (int i = 0; i < WARPS; ++i) sum += partial[j % 2][i];
            d_weights[size_t(token) * topk + j] = sum;
        }
    }
}

void check_routes(int tokens, int topk, int hidden) {
    if (tokens < 0 || topk < 1 || hidden < 1) throw std::invalid_argument("tokens: topk and hidden must be positive, tokens not negative");
    if ((long long)(tokens) * topk > 0x7FFFFFFFll) throw std::invalid_argument("tokens: tokens * topk must be below 2^31");
}

// Values that can be moved at once: the largest power of two that divides a row and whose bytes divide the addresses.
int pack_values(int hidden, size_t size, std::initializer_list<const void*> pointers) {
    uintptr_t bits = uintptr_t(hidden) * size;
    for (const void* p : pointers) bits |= reinterpret_cast<uintptr_t>(p);
    size_t bytes = 16;
    while (bytes > size && (bits & (bytes - 1))) bytes /= 2;
    return int(bytes / size);
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
void by_type(int dtype, int hidden, std::initializer_list<const void*> pointers, F&& body) {
    auto with = [&](auto value) {
        using T = decltype(value);
        const int n = pack_values(hidden, sizeof(T), pointers);
        if constexpr (sizeof(T) == 2) {
            if (n == 8) return body(value, std::integral_constant<int, 8>{});
        }
        if (n == 4) return body(value, std::integral_constant<int, 4>{});
        if (n == 2) return body(value, std::integral_constant<int, 2>{});
        return body(value, std::integral_constant<int, 1>{});
    };
    switch (dtype) {
        case DTYPE_BF16: return with(__nv_bfloat16{});
        case DTYPE_F16: return with(__half{});
        case DTYPE_F32: return with(float{});
        default: throw std::invalid_argument("tokens: dtype must be 0 (bf16), 1 (fp16) or 2 (fp32)");
    }
}
// body(number of routes whose rows are in flight at once)
template <typename F>
void by_group(int topk, F&& body) {
    if (topk <= 2) return body(std::integral_constant<int, 2>{});
    if (topk <= 4) return body(std::integral_constant<int, 4>{});
    if (topk <= 6) return body(std::integral_constant<int, 6>{});
    return body(std::integral_constant<int, 8>{});
}

size_t sort_memory(int experts) { return size_t(SORT_WARPS + 2) * (size_t(experts) + 1) * sizeof(int); }

// The limit is the function's, all threads' alike: raised once per device, to what the most experts take, and never lowered.
template <typename Id>
void allow_sort_memory() {
    static std::atomic<bool> allowed[64] = {};
    int device = 0;
    cuda_check(cudaGetDevice(&device));
    const bool known = device >= 0 && device < 64;
    if (known && allowed[device].load(std::memory_order_acquire)) return;
    cuda_check(cudaFuncSetAttribute(tokens_sort_kernel<Id>, cudaFuncAttributeMaxDynamicSharedMemorySize, int(sort_memory(SORT_MAX_EXPERTS))));
    if (known) allowed[device].store(true, std::memory_order_release);
}

template <typename Id>
void launch_sort(const Id* ids, int routes, int experts, int* offsets, int* position, int* source, int* counts, cudaStream_t stream) {
    const size_t keys = size_t(experts) + 1;
    g_launches.fetch_add(1, std::memory_order_relaxed);
    if (routes <= SMALL) {
        launch_chained(tokens_sort_small_kernel<Id>, dim3(1), dim3(SMALL), 0, stream, ids, routes, experts, offsets, position, source);
        return;
    }
    int part;
    const int blocks = sort_blocks(routes, part);
    if (blocks > 1) {
        launch_chained(tokens_count_kernel<Id>, dim3(unsigned(blocks)), dim3(BLOCK), keys * sizeof(int), stream, ids, routes, experts, part, counts);
        g_launches.fetch_add(1, std::memory_order_relaxed);
    }
    const size_t smem = sort_memory(experts);
    if (smem + SORT_STATIC > 48 * 1024) allow_sort_memory<Id>();
    launch_chained(tokens_sort_kernel<Id>, dim3(unsigned(blocks)), dim3(BLOCK), smem, stream, ids, routes, experts, part,
                   blocks > 1 ? counts : nullptr, offsets, position, source);
}

}  // namespace

size_t tokens_sort_workspace(int routes, int experts) {
    int part;
    const int blocks = routes > SMALL ? sort_blocks(routes, part) : 1;
    return blocks > 1 ? size_t(blocks) * (size_t(experts) + 1) * sizeof(int) : 0;
}

void tokens_sort(const void* ids, int id_bytes, int routes, int experts, int* offsets, int* position, int* source, int* workspace,
                 cudaStream_t stream) {
    if (experts < 1 || experts > SORT_MAX_EXPERTS) throw std::invalid_argument("tokens sort: 1..1024 experts");
    if (routes < 0) throw std::invalid_argument("tokens sort: the number of routes must not be negative");
    if (id_bytes != 4 && id_bytes != 8) throw std::invalid_argument("tokens sort: ids are 32- or 64-bit integers");
    if (!offsets || (routes > 0 && (!ids || !position || !source))) throw std::invalid_argument("tokens sort: null pointer");
    if (!workspace && tokens_sort_workspace(routes, experts)) throw std::invalid_argument("tokens sort: a batch of this size needs its workspace");
    if (id_bytes == 8) launch_sort(static_cast<const long long*>(ids), routes, experts, offsets, position, source, workspace, stream);
    else launch_sort(static_cast<const int*>(ids), routes, experts, offsets, position, source, workspace, stream);
}

void tokens_gather(const void* x, int dtype, int tokens, int topk, int hidden, const int* position, const int* live, void* rows,
                   cudaStream_t stream) {
    check_routes(tokens, topk, hidden);
    if (tokens == 0) return;
    if (!x || !position || !live || !rows) throw std::invalid_argument("tokens gather: null pointer");
    by_type(dtype, hidden, {x, rows}, [&](auto value, auto n) {
        using T = decltype(value);
        constexpr int N = decltype(n)::value;
        int segments;
        const unsigned grid = blocks(tokens, hidden / N, ROW_THREADS * GATHER_PACKS<T, N>, segments);
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
    by_type(dtype, hidden, {rows, y}, [&](auto value, auto n) {
        using T = decltype(value);
        constexpr int N = decltype(n)::value;
        auto go = [&](auto kernel, int packs) {                  // of a row, to a thread
            int segments;
            const unsigned grid = blocks(tokens, hidden / N, ROW_THREADS * packs, segments);
            launch_chained(kernel, dim3(grid), dim3(ROW_THREADS), 0, stream, static_cast<const T*>(rows), weights, position, live,
                           tokens, topk, hidden, segments, static_cast<T*>(y));
        };
        if constexpr (sizeof(T) * N == 16)
            by_group(topk, [&](auto group) {
                constexpr int GROUP = decltype(group)::value <= 6 ? decltype(group)::value : 4;
                if constexpr (GROUP <= 4) {
                    if (hidden / N > ROW_THREADS) return go(tokens_combine_kernel<T, GROUP, 2>, 2);
                }
                go(tokens_combine_kernel<T, GROUP, 1>, 1);
            });
        else go(tokens_combine_narrow_kernel<T, N>, NARROW);
    });
    g_launches.fetch_add(1, std::memory_order_relaxed);
}

void tokens_combine_backward(const void* d_y, int dtype, const void* rows, const float* weights, const int* position,
                             const int* live, int tokens, int topk, int hidden, void* d_rows, float* d_weights, cudaStream_t stream) {
    check_routes(tokens, topk, hidden);
    if (tokens == 0 || (!d_rows && !d_weights)) return;
    if (!d_y || !weights || !position || !live || (d_weights && !rows)) throw std::invalid_argument("tokens combine backward: null pointer");
    by_type(dtype, hidden, {d_y, rows, d_rows}, [&](auto value, auto n) {
        using T = decltype(value);
        constexpr int N = decltype(n)::value;
        auto go = [&](auto kernel) {
            launch_chained(kernel, dim3(unsigned(tokens)), dim3(ROW_THREADS), 0, stream, static_cast<const T*>(d_y),
                           static_cast<const T*>(rows), weights, position, live, tokens, topk, hidden, static_cast<T*>(d_rows), d_weights);
        };
        if constexpr (sizeof(T) * N == 16) by_group(topk, [&](auto group) { go(tokens_combine_backward_kernel<T, decltype(group)::value>); });
        else go(tokens_combine_backward_narrow_kernel<T, N>);
    });
    g_launches.fetch_add(1, std::memory_order_relaxed);
}

}  // namespace nvfp4_b200
