// Int8 matrix products for sm_100a: C[m, n] = (sum_k a[m, k] b[n, k]) * a_scale[m] * b_scale[n], dense or expert by expert.
//
// The sum is exact (32-bit integers; K is limited so that it cannot overflow); it is converted to FP32, multiplied by the
// token's scale, then by the channel's, and rounded to C's type: at most three roundings of 2^-24 before that one.
//
// A warp-specialised kernel of 320 threads per CTA: warp 5 streams tiles of both operands through a ring in shared memory
// by TMA (128 bytes of K per row and stage, 128-byte swizzle), warp 4 issues tcgen05.mma.kind::i8 from it, and warps 0-3
// and 6-9, two per Tensor Memory lane quarter, drain the accumulators. Two accumulators take turns, so that a tile is
// drained while the next one is computed. Two forms:
//   SWAP = false, CTA pairs: 256 tokens on the MMA's M side, up to 256 channels on its N side, persistent. For many tokens:
//     bound by the tensor cores.
//   SWAP = true, single CTAs: 128 channels on the M side, the tokens on the N side, in as narrow a tile as holds them.
//     For few tokens, where each weight byte is read once and HBM is the bound: no row of a tile is padding, and a lane
//     quarter's 32 channels are consecutive in C. Where the tiles are fewer than the SMs, a cluster of 2, 4 or 8 CTAs
//     shares a tile's K loop: their integer partial sums meet in distributed shared memory, column by column, and the order
//     in which they are added does not matter.
// Grouped: rows sorted by expert, `offsets` (device) says where each expert's rows start, and the weights are stacked
// [experts, N, K]. Every CTA counts the experts' tiles once and walks the same sequence, an expert's tokens innermost, so
// that its weights are read from HBM once. A tile that reaches into the next expert's rows (or channels) computes them
// with the wrong weights and does not store them.
#include "operators_internal.h"
#include "ptx.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <mutex>

namespace nvfp4_b200 {
namespace {

using namespace ptx;

constexpr int ROW_BYTES = 128;                                  // K values per ring stage
constexpr int MMA_K = 32;                                       // K values per tcgen05.mma of this kind
constexpr int THREADS = 320, EPI_WARPS = 8;
constexpr int MAX_STAGES = 12;
constexpr int SMEM_LIMIT = 232448;                              // 227 KiB per CTA
constexpr int MAX_EXPERTS = 1024;
constexpr int MAX_K = 131056;                                   // 16 * 8191: K * 128 * 128 < 2^31

struct Control {
    uint64_t full[MAX_STAGES], empty[MAX_STAGES];
    uint64_t acc_full[2], acc_free[2];
    uint32_t tmem_base;
    WaitCtl wait;
};
constexpr int CONTROL_BYTES = 512;
static_assert(sizeof(Control) <= CONTROL_BYTES, "control block");

struct Args {
    int M, N, ksteps;
    int width, stages, split;       // see Int8Tiles
    int y_box;                      // rows of the N side's box
    int tiles_x, tiles_y, band;     // dense: tiles along the M and the N side, M-side tiles per band
    const float* a_scale;
    const float* b_scale;
    uint8_t* c;
    int out;                        // InputDtype of C
    const int* offsets;             // grouped: [experts + 1]; null = dense
    int experts;
    int zero_rest;                  // grouped: rows of C behind the last expert's are cleared
    int early;                      // the weights may be read before the grid in front of this one has finished
    uint32_t* status;
};

struct Tile {
    int x, y;                       // first row in the M side's and in the N side's operand
    int token, token_end;           // first row of C, and the first one that is not this tile's to write
    int channel;                    // first column of C
    int scale;                      // first channel in b_scale
};

// The sequence of tiles one CTA (pair, cluster) works through; every role walks the same one.
template <int CG, bool SWAP>
struct Walk {
    const Args& g;
    const int* tile_start;          // grouped: first tile and first row of every expert, [experts + 1] each
    const int* row_start;
    int t, stride, tiles, expert;
    __device__ Walk(const Args& args, const int* ts, const int* rs, int unit, int units)
        : g(args), tile_start(ts), row_start(rs), t(unit), stride(units), expert(0) {
        tiles = g.offsets ? ts[g.experts] : g.tiles_x * g.tiles_y;
    }
    __device__ bool valid() const { return t < tiles; }
    __device__ void next() { t += stride; }
    __device__ Tile tile() {
        constexpr int X = 128 * CG;
        Tile r;
        if (g.offsets) {
            while (tile_start[expert + 1] <= t) ++expert;
            const int row0 = row_start[2 * expert], row1 = row_start[2 * expert + 1], local = t - tile_start[expert];
            const int per = SWAP ? g.width : X, count = (row1 - row0 + per - 1) / per;
            const int channel_tile = local / count, token_tile = local - channel_tile * count;
            r.token = row0 + token_tile * per;
            r.token_end = row1;
            r.channel = channel_tile * (SWAP ? X : g.width);
            r.scale = expert * g.N + r.channel;
        } else {
            // bands of `band` tiles along the M side, every other one backwards along the N side: the tiles in flight share
            // their operands in L2
            const int per_band = g.band * g.tiles_y, b = t / per_band, first = b * g.band;
            const int high = min(g.band, g.tiles_x - first), within = t - b * per_band, column = within / high;
            const int tx = first + within - column * high, ty = (b & 1) ? g.tiles_y - 1 - column : column;
            r.token = SWAP ? ty * g.width : tx * X;
            r.token_end = g.M;
            r.channel = SWAP ? tx * X : ty * g.width;
            r.scale = r.channel;
        }
        r.x = SWAP ? r.scale : r.token;
        r.y = SWAP ? r.token : r.scale;
        return r;
    }
};

__device__ __forceinline__ uint32_t pack_pair(float a, float b, int out) {
    if (out == DTYPE_BF16) {
        const __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&p);
    }
    const __half2 p = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&p);
}
__device__ __forceinline__ void store_one(uint8_t* c, size_t at, float v, int out) {
    if (out == DTYPE_F32) reinterpret_cast<float*>(c)[at] = v;
    else if (out == DTYPE_BF16) reinterpret_cast<__nv_bfloat16*>(c)[at] = __float2bfloat16_rn(v);
    else reinterpret_cast<__half*>(c)[at] = __float2half_rn(v);
}
__device__ __forceinline__ float scaled(uint32_t sum, float token, float channel) {
    return __int2float_rn(int(sum)) * token * channel;
}

template <int CG, bool SWAP>
struct Roles {
    const Args& g;
    uint32_t smem;                  // 1024-aligned address of stage 0
    uint32_t stage_bytes;
    Control* ctrl;
    const int* tile_start;
    const int* row_start;
    uint32_t rank;                  // CTA of the pair, or slice of K
    int unit, units;
    uint32_t peer_abort;
    int k0, k1;                     // this CTA's ring steps of every tile

    __device__ __forceinline__ bool wait(const uint64_t* b, uint32_t parity, uint32_t who, uint32_t tag) const {
        if (mbar_wait(smem_u32(b), parity, &ctrl->wait, g.status, who, peer_abort)) return true;
        if (who) atomicCAS(g.status + 1, 0u, tag);
        return false;
    }

    // ---- warp 5 ---------------------------------------------------------------------------------------------------
    struct Cursor {
        Walk<CG, SWAP> walk;
        Tile tile;
        int ks, k0, k1;
        __device__ Cursor(const Walk<CG, SWAP>& w, int a, int b) : walk(w), ks(a), k0(a), k1(b) {
            if (walk.valid()) tile = walk.tile();
        }
        __device__ bool valid() const { return walk.valid(); }
        __device__ void next() {
            if (++ks < k1) return;
            ks = k0;
            walk.next();
            if (walk.valid()) tile = walk.tile();
        }
    };
    // One operand's part of ring stage `stage`; x_side: the M side's.
    __device__ __forceinline__ void request(const CUtensorMap* map, bool x_side, const Cursor& c, int stage) const {
        const uint32_t dst = smem + stage * stage_bytes + (x_side ? 0u : 128u * ROW_BYTES);
        const uint32_t full = smem_u32(&ctrl->full[stage]);
        if constexpr (CG == 1) {
            tma_load_2d(dst, map, c.ks * ROW_BYTES, x_side ? c.tile.x : c.tile.y, full);
        } else {
            const int half = x_side ? 128 : g.width / 2;        // each CTA of the pair loads its half of both operands
            tma_load_2d_pair(dst, map, c.ks * ROW_BYTES, (x_side ? c.tile.x : c.tile.y) + int(rank) * half, map_to_cta(full, 0));
        }
    }
    __device__ void produce(const CUtensorMap* mapX, const CUtensorMap* mapY, int lane) const {
        const uint32_t bytes = uint32_t(CG) * (128u + uint32_t(g.y_box)) * ROW_BYTES;
        const CUtensorMap* weights = SWAP ? mapX : mapY;
        const CUtensorMap* tokens = SWAP ? mapY : mapX;
        Cursor cursor(Walk<CG, SWAP>(g, tile_start, row_start, unit, units), k0, k1);
        int stage = 0;
        uint32_t phase = 0;
        if (g.early) {
            // The first ring fill: the weights at once, the tokens once the kernel that quantises them has finished.
            Cursor ahead = cursor;
            int lead = 0;
            for (; lead < g.stages && ahead.valid(); ++lead, ahead.next())
                if (elect_one()) {
                    if (CG == 1 || rank == 0) mbar_arrive_expect_tx(smem_u32(&ctrl->full[lead]), bytes);
                    request(weights, SWAP, ahead, lead);
                }
            grid_dependency_wait();
            for (int i = 0; i < lead; ++i, cursor.next())
                if (elect_one()) request(tokens, !SWAP, cursor, i);
            if (lead == g.stages) phase = 1;
            else stage = lead;
        }
        for (; cursor.valid(); cursor.next()) {
            const bool ok = wait(&ctrl->empty[stage], phase ^ 1u, lane == 0 ? STATUS_TIMEOUT_PRODUCER : 0u, 0x50000000u | (stage << 16) | cursor.ks);
            if (!__all_sync(0xFFFFFFFFu, ok)) return;
            if (elect_one()) {
                if (CG == 1 || rank == 0) mbar_arrive_expect_tx(smem_u32(&ctrl->full[stage]), bytes);
                request(weights, SWAP, cursor, stage);
                request(tokens, !SWAP, cursor, stage);
            }
            if (++stage == g.stages) { stage = 0; phase ^= 1u; }
        }
    }

    // ---- warp 4 (of the pair's first CTA) -------------------------------------------------------------------------
    __device__ void issue(uint32_t tmem, uint32_t acc_stride, int lane) const {
        // Operand descriptors: rows of 128 bytes under the 128-byte swizzle, 8-row groups 1024 bytes apart, version 1.
        constexpr uint32_t DESC_HI = (1024u >> 4) | (1u << 14) | (2u << 29);
        // Instruction descriptor of kind::i8: 32-bit integer sums (2 at bit 4), A and B signed (1 at bits 7 and 10), both
        // K-major, N >> 3 at bit 17, M >> 4 at bit 24.
        const uint32_t idesc = (2u << 4) | (1u << 7) | (1u << 10) | (uint32_t(g.width >> 3) << 17) | (uint32_t(128 * CG >> 4) << 24);
        const uint32_t ring_lo = (smem & 0x3FFFFu) >> 4;
        int stage = 0;
        uint32_t phase = 0, iter = 0;
        bool landed = false;                                    // the probe of this stage's barrier succeeded
        for (Walk<CG, SWAP> walk(g, tile_start, row_start, unit, units); walk.valid(); walk.next(), ++iter) {
            const uint32_t b = iter & 1u, acc = tmem + b * acc_stride;
            const bool free = wait(&ctrl->acc_free[b], ((iter >> 1) & 1u) ^ 1u, lane == 0 ? STATUS_TIMEOUT_MMA : 0u, 0x60000000u | iter);
            if (!__all_sync(0xFFFFFFFFu, free)) return;
            tc_fence_after_sync();
            for (int ks = k0; ks < k1; ++ks) {
                if (!landed) {
                    const bool ok = wait(&ctrl->full[stage], phase, lane == 0 ? STATUS_TIMEOUT_MMA : 0u, 0x61000000u | (stage << 16) | ks);
                    if (!__all_sync(0xFFFFFFFFu, ok)) return;
                }
                tc_fence_after_sync();
                const int next_stage = stage + 1 == g.stages ? 0 : stage + 1;
                const uint32_t next_phase = stage + 1 == g.stages ? phase ^ 1u : phase;
                const bool probe = mbar_test_wait(smem_u32(&ctrl->full[next_stage]), next_phase);
                const uint32_t lo = ring_lo + uint32_t(stage) * (stage_bytes >> 4);
                if (elect_one()) {
                    #pragma unroll
                    for (int j = 0; j < ROW_BYTES / MMA_K; ++j)
                        mma_i8<CG>(acc, lo + (j * MMA_K >> 4), lo + ((128 * ROW_BYTES + j * MMA_K) >> 4), DESC_HI, idesc,
                                   ks == k0 && j == 0 ? 0u : 1u);
                    mma_commit<CG>(smem_u32(&ctrl->empty[stage]));
                    if (ks + 1 == k1) mma_commit<CG>(smem_u32(&ctrl->acc_full[b]));
                }
                landed = __all_sync(0xFFFFFFFFu, probe);
                stage = next_stage;
                phase = next_phase;
            }
        }
    }

    // ---- warps 0-3 and 6-9 ----------------------------------------------------------------------------------------
    // 32 accumulator columns of one lane. Tokens on the lanes: 32 channels of one row of C.
    __device__ __forceinline__ void store_row(const uint32_t (&v)[32], const Tile& t, int token, int column, int wide) const {
        if (token >= t.token_end) return;
        const float sa = __ldg(g.a_scale + token);
        uint8_t* row = g.c + size_t(token) * g.N * (g.out == DTYPE_F32 ? 4 : 2);
        #pragma unroll
        for (int q = 0; q < 4; ++q) {                           // N is a multiple of 8: eight channels are there or not
            const int n = t.channel + column + 8 * q;
            if (column + 8 * q >= wide) break;
            float f[8];
            const float4 s0 = __ldg(reinterpret_cast<const float4*>(g.b_scale + t.scale + column + 8 * q));
            const float4 s1 = __ldg(reinterpret_cast<const float4*>(g.b_scale + t.scale + column + 8 * q) + 1);
            const float s[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
            #pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = scaled(v[8 * q + i], sa, s[i]);
            if (g.out == DTYPE_F32) {
                float4* dst = reinterpret_cast<float4*>(row + size_t(n) * 4);
                dst[0] = make_float4(f[0], f[1], f[2], f[3]);
                dst[1] = make_float4(f[4], f[5], f[6], f[7]);
            } else {
                *reinterpret_cast<uint4*>(row + size_t(n) * 2) =
                    make_uint4(pack_pair(f[0], f[1], g.out), pack_pair(f[2], f[3], g.out), pack_pair(f[4], f[5], g.out), pack_pair(f[6], f[7], g.out));
            }
        }
    }
    // Channels on the lanes: one channel of 32 rows of C.
    __device__ __forceinline__ void store_columns(const uint32_t (&v)[32], const Tile& t, int channel, float sb, int column, int wide, int lane) const {
        const int token0 = t.token + column, count = min(32, wide - column);
        const float mine = lane < count ? __ldg(g.a_scale + token0 + lane) : 0.0f;
        #pragma unroll
        for (int i = 0; i < 32; ++i) {
            if (i >= count) break;
            const float sa = __shfl_sync(0xFFFFFFFFu, mine, i);
            if (channel < g.N) store_one(g.c, size_t(token0 + i) * g.N + channel, scaled(v[i], sa, sb), g.out);
        }
    }

    __device__ void drain(uint32_t tmem, uint32_t acc_stride, int quarter, int half, int lane) const {
        if (g.early) grid_dependency_wait();                    // (without it the prologue waited)
        uint32_t iter = 0;
        for (Walk<CG, SWAP> walk(g, tile_start, row_start, unit, units); walk.valid(); walk.next(), ++iter) {
            const Tile t = walk.tile();
            const uint32_t b = iter & 1u;
            const bool ready = wait(&ctrl->acc_full[b], (iter >> 1) & 1u, lane == 0 ? STATUS_TIMEOUT_EPILOGUE : 0u, 0x70000000u | iter);
            if (!__all_sync(0xFFFFFFFFu, ready)) return;
            tc_fence_after_sync();
            const uint32_t acc = tmem + b * acc_stride + (uint32_t(quarter * 32) << 16);
            const int on_lane = quarter * 32 + lane + int(CG == 2 ? rank : 0u) * 128;
            const int wide = SWAP ? min(g.width, t.token_end - t.token) : min(g.width, g.N - t.channel);     // the tile's columns
            const int channel = t.channel + on_lane;
            const float sb = SWAP && channel < g.N ? __ldg(g.b_scale + t.scale + on_lane) : 0.0f;
            for (int column = half * 32; column < wide; column += 64) {
                uint32_t v[32];
                tmem_ld_32x32(acc + column, v);
                tmem_ld_wait();
                if constexpr (SWAP) store_columns(v, t, channel, sb, column, wide, lane);
                else store_row(v, t, t.token + on_lane, column, wide);
                __syncwarp();
            }
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) {
                if constexpr (CG == 2) mbar_arrive_cluster(map_to_cta(smem_u32(&ctrl->acc_free[b]), 0));
                else mbar_arrive(smem_u32(&ctrl->acc_free[b]));
            }
        }
    }

    // One tile whose K loop the cluster shares. Column (token) c of the tile belongs to CTA c % split, which has room for
    // [split][width / split][128] partial sums at `room`; every CTA sends its own there.
    __device__ void send(uint32_t tmem, uint32_t room, int quarter, int half, int lane) const {
        Walk<CG, SWAP> walk(g, tile_start, row_start, unit, units);
        const Tile t = walk.tile();
        const bool ready = wait(&ctrl->acc_full[0], 0u, lane == 0 ? STATUS_TIMEOUT_EPILOGUE : 0u, 0x71000000u);
        if (!__all_sync(0xFFFFFFFFu, ready)) return;
        tc_fence_after_sync();
        const int wide = min(g.width, t.token_end - t.token), each = g.width / g.split, ch = quarter * 32 + lane;
        for (int column = half * 32; column < wide; column += 64) {
            uint32_t v[32];
            tmem_ld_32x32(tmem + (uint32_t(quarter * 32) << 16) + column, v);
            tmem_ld_wait();
            #pragma unroll
            for (int i = 0; i < 32; ++i) {
                const int c = column + i;
                if (c >= wide) break;
                const uint32_t at = room + uint32_t(((int(rank) * each + c / g.split) * 128 + ch) * 4);
                asm volatile("st.shared::cluster.u32 [%0], %1;" :: "r"(map_to_cta(at, uint32_t(c % g.split))), "r"(v[i]) : "memory");
            }
        }
    }
    __device__ void finish(const int* room, int thread) const {
        if (g.early) grid_dependency_wait();
        Walk<CG, SWAP> walk(g, tile_start, row_start, unit, units);
        const Tile t = walk.tile();
        const int each = g.width / g.split, wide = min(g.width, t.token_end - t.token), ch = thread % 128, channel = t.channel + ch;
        if (channel >= g.N) return;
        const float sb = __ldg(g.b_scale + t.scale + ch);
        for (int slot = thread / 128; slot * g.split + int(rank) < wide; slot += 2) {
            int sum = 0;
            for (int s = 0; s < g.split; ++s) sum += room[(s * each + slot) * 128 + ch];
            const int token = t.token + slot * g.split + int(rank);
            store_one(g.c, size_t(token) * g.N + channel, scaled(uint32_t(sum), __ldg(g.a_scale + token), sb), g.out);
        }
    }
};

template <int CG, bool SWAP>
__global__ void __launch_bounds__(THREADS, 1)
int8_gemm_kernel(const __grid_constant__ CUtensorMap mapX, const __grid_constant__ CUtensorMap mapY, const Args g) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw), smem = (raw + 1023u) & ~1023u;
    const uint32_t stage_bytes = uint32_t(128 + g.width / CG) * ROW_BYTES;
    uint8_t* behind = smem_raw + (smem - raw) + g.stages * stage_bytes;
    Control* ctrl = reinterpret_cast<Control*>(behind);
    int* tile_start = reinterpret_cast<int*>(behind + CONTROL_BYTES);        // grouped: [experts + 1]
    int* row_start = tile_start + g.experts + 1;                             // grouped: first row and first row behind, [experts][2]
    int* room = tile_start;                                                  // split: partial sums
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const bool cluster = CG == 2 || g.split > 1;
    const uint32_t rank = cluster ? cluster_ctarank() : 0u;
    const uint32_t acc_stride = uint32_t(g.width + 31) / 32u * 32u;
    uint32_t columns = 64;
    while (columns < 2 * acc_stride) columns *= 2;

    if (threadIdx.x == 0) {
        for (int s = 0; s < g.stages; ++s) {
            mbar_init(smem_u32(&ctrl->full[s]), 1);
            mbar_init(smem_u32(&ctrl->empty[s]), 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(smem_u32(&ctrl->acc_full[b]), 1);
            mbar_init(smem_u32(&ctrl->acc_free[b]), EPI_WARPS * CG);
        }
        ctrl->wait.abort = 0;
        mbar_init_fence();
    }
    if (warp == 4) {
        tmem_alloc<CG>(smem_u32(&ctrl->tmem_base), columns);
        tmem_relinquish<CG>();
    }
    if (warp == 5 && lane == 0) { prefetch_tensormap(&mapX); prefetch_tensormap(&mapY); }
    if (!g.early) chain_point();
    if (g.offsets) {
        const int per = SWAP ? g.width : 128 * CG, channel_tiles = (g.N + (SWAP ? 128 * CG : g.width) - 1) / (SWAP ? 128 * CG : g.width);
        for (int e = threadIdx.x; e < g.experts; e += THREADS) row_start[2 * e + 1] = min(max(__ldcg(g.offsets + e + 1), 0), g.M);
        __syncthreads();
        if (warp == 0) {
            // Sums over the experts before, 32 at a time. An expert's rows end where the largest offset so far says and
            // start where the expert before ended, so that no row is computed twice, whatever the offsets hold.
            int tiles_before = 0, rows_before = min(max(__ldcg(g.offsets), 0), g.M);
            if (lane == 0) tile_start[0] = 0;
            for (int e = 0; e < g.experts; e += 32) {
                const bool there = e + lane < g.experts;
                int end = there ? max(row_start[2 * (e + lane) + 1], rows_before) : rows_before;
                #pragma unroll
                for (int d = 1; d < 32; d *= 2) {
                    const int m = __shfl_up_sync(0xFFFFFFFFu, end, d);
                    if (lane >= d) end = max(end, m);
                }
                int first = __shfl_up_sync(0xFFFFFFFFu, end, 1);
                if (lane == 0) first = rows_before;
                int n = (end - first + per - 1) / per * channel_tiles;
                #pragma unroll
                for (int d = 1; d < 32; d *= 2) {
                    const int m = __shfl_up_sync(0xFFFFFFFFu, n, d);
                    if (lane >= d) n += m;
                }
                if (there) {
                    row_start[2 * (e + lane)] = first;
                    row_start[2 * (e + lane) + 1] = end;
                    tile_start[e + lane + 1] = tiles_before + n;
                }
                tiles_before += __shfl_sync(0xFFFFFFFFu, n, 31);
                rows_before = __shfl_sync(0xFFFFFFFFu, end, 31);
            }
        }
        __syncwarp();
    }
    tc_fence_before_sync();
    if (cluster) { cluster_arrive(); cluster_wait(); }
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = ctrl->tmem_base;

    const int members = CG == 2 ? 2 : g.split;
    Roles<CG, SWAP> roles{g, smem, stage_bytes, ctrl, tile_start, row_start, rank, int(blockIdx.x) / members, int(gridDim.x) / members,
                          CG == 2 ? map_to_cta(smem_u32(const_cast<uint32_t*>(&ctrl->wait.abort)), rank ^ 1u) : 0u,
                          g.split > 1 ? int(rank) * g.ksteps / g.split : 0, g.split > 1 ? int(rank + 1) * g.ksteps / g.split : g.ksteps};
    const bool drains = warp < 4 || warp >= 6;
    const int half = warp < 4 ? 0 : 1, thread = (half * 4 + (warp & 3)) * 32 + lane;
    if (warp == 5) {
        roles.produce(&mapX, &mapY, lane);
        if (g.early) grid_launch_dependents();                   // (its wait lies behind it)
    } else if (warp == 4) {
        if (CG == 1 || rank == 0) roles.issue(tmem, acc_stride, lane);
    } else if (g.split > 1) {
        roles.send(tmem, smem_u32(room), warp & 3, half, lane);
    } else {
        roles.drain(tmem, acc_stride, warp & 3, half, lane);
        if (g.offsets && g.zero_rest) {
            const size_t row_packs = size_t(g.N) * (g.out == DTYPE_F32 ? 4 : 2) / 16;
            const int first = row_start[0], end = row_start[2 * g.experts - 1];
            uint4* packs = reinterpret_cast<uint4*>(g.c);
            const size_t start = size_t(blockIdx.x) * (EPI_WARPS * 32) + thread, step = size_t(gridDim.x) * (EPI_WARPS * 32);
            for (size_t i = start; i < size_t(first) * row_packs; i += step) packs[i] = make_uint4(0u, 0u, 0u, 0u);
            for (size_t i = size_t(end) * row_packs + start; i < size_t(g.M) * row_packs; i += step) packs[i] = make_uint4(0u, 0u, 0u, 0u);
        }
    }
    __syncwarp();
    // After an abandoned wait, copies in flight get time to land before the CTA's shared memory is released.
    if (ctrl->wait.abort)
        for (int i = 0; i < 200; ++i) __nanosleep(1000);
    __syncwarp();
    tc_fence_before_sync();
    if (cluster) { cluster_arrive(); cluster_wait(); }
    __syncthreads();
    if (g.split > 1 && drains && !ctrl->wait.abort) roles.finish(room, thread);
    if (warp == 4) {
        tc_fence_after_sync();
        tmem_dealloc<CG>(tmem, columns);
    }
}

// ---- host -----------------------------------------------------------------------------------------------------------

std::mutex g_lock;

// CTAs or CTA pairs that are resident at once (one CTA per SM: its ring fills the shared memory).
template <int CG, bool SWAP>
int resident(int device) {
    static int cached[64] = {};
    std::lock_guard<std::mutex> hold(g_lock);
    if (device >= 0 && device < 64 && cached[device]) return cached[device];
    auto kernel = int8_gemm_kernel<CG, SWAP>;
    cuda_check(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_LIMIT));
    int units = 0;
    cuda_check(cudaDeviceGetAttribute(&units, cudaDevAttrMultiProcessorCount, device));
    if (CG == 2) {
        cudaLaunchAttribute attr{};
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim = {2, 1, 1};
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(unsigned(units / 2) * 2);
        cfg.blockDim = dim3(THREADS);
        cfg.dynamicSmemBytes = SMEM_LIMIT;
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
        cuda_check(cudaOccupancyMaxActiveClusters(&units, kernel, &cfg));
    }
    if (units < 1) throw std::runtime_error("int8 gemm: the kernel does not fit on this device");
    if (device >= 0 && device < 64) cached[device] = units;
    return units;
}
int resident(const Int8Tiles& t, int device) { return t.pair ? resident<2, false>(device) : resident<1, true>(device); }

int round_up(int v, int to) { return (v + to - 1) / to * to; }

size_t table_bytes(const Int8Tiles& t, int experts) {
    return experts ? size_t(3 * experts + 1) * sizeof(int) : t.split > 1 ? size_t(t.width) * 128 * sizeof(int) : 0;
}

}  // namespace

Int8Tiles int8_tiles(int rows, int n, int k, int experts, int device) {
    Int8Tiles t{};
    t.split = 1;
    const int sms = resident<1, true>(device), steps = (k + ROW_BYTES - 1) / ROW_BYTES;
    if (experts) {
        const int mean = (rows + experts - 1) / experts;
        t.pair = mean >= 256;
        t.swap = !t.pair;
        t.width = t.pair ? 256 : std::min(128, round_up(mean + mean / 2, 16));
    } else {
        t.pair = rows > 256;
        t.swap = !t.pair;
        t.width = t.pair ? 256 : round_up(rows, 16);
        const int tiles = (n + 127) / 128;
        if (t.swap)
            while (t.split < 8 && tiles * t.split * 2 <= sms && steps / (t.split * 2) >= 4) t.split *= 2;
    }
    const size_t stage = size_t(128 + t.width / (t.pair ? 2 : 1)) * ROW_BYTES;
    t.stages = int(std::min<size_t>(MAX_STAGES, (SMEM_LIMIT - 1024 - CONTROL_BYTES - table_bytes(t, experts)) / stage));
    return t;
}

namespace {

void run(const int8_t* a, const int8_t* b, const float* a_scales, const float* b_scales, const int* offsets, int experts, void* C,
         int out_dtype, int M, int N, int K, bool zero_rest, bool early, cudaStream_t stream) {
    int device = 0;
    cuda_check(cudaGetDevice(&device));
    const Int8Tiles t = int8_tiles(M, N, K, experts, device);
    const int x_tile = t.pair ? 256 : 128, y_box = std::min(t.width / (t.pair ? 2 : 1), experts || t.pair ? t.width : round_up(M, 8));
    Args g{};
    g.M = M;
    g.N = N;
    g.ksteps = (K + ROW_BYTES - 1) / ROW_BYTES;
    g.width = t.width;
    g.stages = t.stages;
    g.split = t.split;
    g.y_box = y_box;
    g.a_scale = a_scales;
    g.b_scale = b_scales;
    g.c = static_cast<uint8_t*>(C);
    g.out = out_dtype;
    g.offsets = offsets;
    g.experts = experts;
    g.zero_rest = zero_rest ? 1 : 0;
    g.early = early ? 1 : 0;
    g.status = device_status_word(device);
    const int x_rows = t.swap ? N : M, y_rows = t.swap ? M : N;
    g.tiles_x = (x_rows + x_tile - 1) / x_tile;
    g.tiles_y = (y_rows + t.width - 1) / t.width;
    long long tiles = (long long)(g.tiles_x) * g.tiles_y;
    if (experts) {                                              // at most: every expert's last tile may be partial
        const int per = t.swap ? t.width : x_tile;
        tiles = ((long long)(M) / per + std::min(M, experts)) * (t.swap ? g.tiles_x : g.tiles_y);
    }
    if (tiles > 0x3FFFFFFFll) throw std::invalid_argument("int8 gemm: too many tiles");
    const int fit = resident(t, device);
    const int units = t.split > 1 ? int(tiles) : int(std::min<long long>(tiles, fit));
    g.band = 1;
    while ((g.band + 1) * (g.band + 1) <= fit) ++g.band;        // about as many operand rows on either side in flight
    g.band = std::min(g.band, g.tiles_x);
    const CUtensorMap tokens = byte_rows_map(a, size_t(M), size_t(K), t.swap ? y_box : 128);
    const CUtensorMap weights = byte_rows_map(b, size_t(N) * std::max(1, experts), size_t(K), t.swap ? 128 : y_box);
    const int members = t.pair ? 2 : t.split;
    cudaLaunchAttribute attrs[2]{};
    attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[0].val.programmaticStreamSerializationAllowed = 1;
    attrs[1].id = cudaLaunchAttributeClusterDimension;
    attrs[1].val.clusterDim = {unsigned(members), 1, 1};
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(unsigned(units) * unsigned(members));
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = 1024 + size_t(t.stages) * (128 + t.width / (t.pair ? 2 : 1)) * ROW_BYTES + CONTROL_BYTES + table_bytes(t, experts);
    cfg.stream = stream;
    cfg.attrs = attrs;
    cfg.numAttrs = members > 1 ? 2 : 1;
    if (t.pair) cuda_check(cudaLaunchKernelEx(&cfg, int8_gemm_kernel<2, false>, tokens, weights, g));
    else cuda_check(cudaLaunchKernelEx(&cfg, int8_gemm_kernel<1, true>, weights, tokens, g));
    g_launches.fetch_add(1, std::memory_order_relaxed);
}

}  // namespace

void int8_gemm_check(const void* a, const void* b, const float* a_scales, const float* b_scales, const void* C, int out_dtype,
                     int M, int N, int K) {
    if (M < 0 || N < 1 || K < 1) throw std::invalid_argument("int8 gemm: N and K must be positive, M not negative");
    if (N % 8) throw std::invalid_argument("int8 gemm: N must be a multiple of 8 (rows of C start on 16-byte boundaries)");
    if (K % 16) throw std::invalid_argument("int8 gemm: K must be a multiple of 16 (rows of the operands start on 16-byte boundaries)");
    if (K > MAX_K) throw std::invalid_argument("int8 gemm: K must not exceed 131056 (the sum has to fit 32 bits)");
    if (out_dtype < DTYPE_BF16 || out_dtype > DTYPE_F32) throw std::invalid_argument("int8 gemm: output dtype must be 0 (bf16), 1 (fp16) or 2 (fp32)");
    if (!b || !b_scales || (M > 0 && (!a || !a_scales || !C))) throw std::invalid_argument("int8 gemm: null pointer");
    if ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) | reinterpret_cast<uintptr_t>(b_scales) | reinterpret_cast<uintptr_t>(C)) & 15)
        throw std::invalid_argument("int8 gemm: operands, channel scales and C must be 16-byte aligned");
}

void int8_gemm(const int8_t* a, const int8_t* b, const float* a_scales, const float* b_scales, void* C, int out_dtype, int M,
               int N, int K, bool early, cudaStream_t stream) {
    int8_gemm_check(a, b, a_scales, b_scales, C, out_dtype, M, N, K);
    if (M == 0) return;
    run(a, b, a_scales, b_scales, nullptr, 0, C, out_dtype, M, N, K, false, early, stream);
}

void int8_grouped_gemm(const int8_t* rows, const int8_t* weights, const float* row_scales, const float* weight_scales,
                       const int* offsets, int experts, void* C, int out_dtype, int R, int N, int K, bool zero_rest,
                       cudaStream_t stream) {
    int8_gemm_check(rows, weights, row_scales, weight_scales, C, out_dtype, R, N, K);
    if (experts < 1 || experts > MAX_EXPERTS) throw std::invalid_argument("int8 grouped gemm: 1..1024 experts");
    if ((long long)(experts) * N > 0x7FFFFFFFll) throw std::invalid_argument("int8 grouped gemm: experts * N must be below 2^31");
    if (!offsets) throw std::invalid_argument("int8 grouped gemm: null pointer");
    if (R == 0) return;
    run(rows, weights, row_scales, weight_scales, offsets, experts, C, out_dtype, R, N, K, zero_rest, false, stream);
}

}  // namespace nvfp4_b200
