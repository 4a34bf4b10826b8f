// Int8 matrix products for sm_100a: C[m, n] = (sum_k a[m, k] b[n, k]) * a_scale[m] * b_scale[n], dense or expert by expert.
//
// The sum is exact (32-bit integers; K is limited so that it cannot overflow); it is converted to FP32, multiplied by the
// token's scale, then by the channel's, and rounded to C's type: at most three roundings of 2^-24 before that one.
//
// A warp-specialised kernel of 320 threads per CTA: warp 5 streams tiles of both operands through a ring in shared memory
// by TMA (128 bytes of K per row and stage, 128-byte swizzle), warp 4 issues tcgen05.mma.kind::i8 from it, and warps 0-3
// and 6-9, two per Tensor Memory lane quarter, drain the accumulators. Two accumulators take turns, so that a tile is
// drained while the next one is computed. The forms, all persistent but the split one:
//   CTA pairs: 256 tokens on the MMA's M side, up to 256 channels on its N side. For many tokens: bound by the tensor cores.
//   Single CTAs: the same with 128 tokens and as many channels to a tile (in steps of 16) as give each SM one tile.
//   SWAP, single CTAs: 128 channels on the M side, the tokens on the N side, in as narrow a tile as holds them. For few
//     tokens, where each weight byte is read once and HBM is the bound.
//   Either kind of single CTAs, where the tiles are fewer than the SMs: a cluster of 2, 4 or 8 CTAs shares a tile's K loop.
//     Their integer partial sums meet in distributed shared memory, and the order in which they are added does not matter
//     (256 x 1024 x 8192 9.6 us, in the best form without 14.3; 512 x 520 x 16384 13.7 and 24.6).
//   Grouped, SWAP, single CTAs or pairs (256 channels): rows sorted by expert, `offsets` (device) says where each expert's
//     rows start, the weights are stacked [experts, N, K]. Every CTA counts the experts' tiles once and walks the same
//     sequence, an expert's tokens innermost, so that its weights are read from HBM once. An expert's rows are dealt evenly
//     to as few tiles as hold them; the MMA's N and the rows a tile fetches (32 to a box) follow its share. With tiles of
//     one width for all, 256 experts of unequal popularity took 1143 us instead of 891 in a loop (4096 tokens of six
//     routes). A tile that reaches into the next expert's rows (or channels) computes them with the wrong weights and does
//     not store them.
// Measured: 8192 cubed 326 us (3.37 POPS, twice the rate cuBLAS reaches in bf16; 359 under the power cap); 1 x 8192 x 8192
// 15.2 us (4.4 TB/s), 1 x 28672 x 8192 40.4 us (5.8 TB/s), 128 x 28672 x 8192 44 us; 256 experts of 4096 x 4096 with 64
// tokens of six routes each 470 us (7.1 TB/s).
#include "operators_internal.h"
#include "ptx.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <mutex>

namespace nvfp4_b200 {
namespace {

using namespace ptx;

constexpr int ROW_BYTES = 128;                                  // K values per row of a box
constexpr int MMA_K = 32;                                       // K values per tcgen05.mma of this kind
constexpr int THREADS = 320, EPI_WARPS = 8;
constexpr int MAX_STAGES = 12;
constexpr int WIDE_FROM = 96;                                   // tiles wider than this take one box per ring stage
constexpr int SMEM_LIMIT = 232448;                              // 227 KiB per CTA
constexpr int MAX_EXPERTS = 1024;
constexpr int MAX_K = 131056;                                   // 16 * 8191: K * 128 * 128 < 2^31

struct Control {
    uint64_t full[MAX_STAGES], empty[MAX_STAGES];
    uint64_t acc_full[2], acc_free[2];
    uint32_t tmem_base;
    WaitCtl wait;
};
constexpr int CONTROL_BYTES = 512 + 256 * sizeof(float);          // the control block, then a scale for each column of a tile (split)
static_assert(sizeof(Control) <= 512, "control block");

struct Args {
    int M, N;
    int kboxes, ksteps;             // K in boxes of 128 values, and in ring steps
    int width, stages, split, subs; // see Int8Tiles
    int x_box, y_box;               // rows of the M and the N side's boxes
    int tiles_x, tiles_y, band;     // dense: tiles along the M and the N side, M-side tiles per band
    const float* a_scale;
    const float* b_scale;
    uint8_t* c;
    int out;                        // InputDtype of C
    int rows_32;                    // every row of C starts on a 32-byte boundary
    const int* offsets;             // grouped: [experts + 1]; null = dense
    int experts;
    int zero_rest;                  // grouped: rows of C that are no expert's are cleared
    int early;                      // the weights may be read before the grid in front of this one has finished
    uint32_t* status;
};

struct Tile {
    int x, y;                       // first row in the M side's and in the N side's operand
    int n;                          // values on the N side: g.width, or in a grouped product as few as hold the tile's tokens
    int token, token_end;           // first row of C, and the first one that is not this tile's to write
    int channel;                    // first column of C
    int scale;                      // first channel in b_scale
};

// Grouped products are SWAP, and SWAP pairs are there for them only.
template <int CG, bool SWAP>
__device__ __forceinline__ bool grouped(const Args& g) { return SWAP && (CG == 2 || g.offsets); }

// The sequence of tiles one CTA (pair, cluster) works through; every role walks the same one.
template <int CG, bool SWAP>
struct Walk {
    const Args& g;
    const int* tile_start;          // grouped: first tile of every expert and their number, [experts + 1]
    const int* row_start;           // grouped: first row of every expert and first row behind, [experts][2]
    int t, stride, tiles, expert;
    __device__ Walk(const Args& args, const int* ts, const int* rs, int unit, int units)
        : g(args), tile_start(ts), row_start(rs), t(unit), stride(units), expert(0) {
        tiles = grouped<CG, SWAP>(g) ? ts[g.experts] : g.tiles_x * g.tiles_y;
    }
    __device__ bool valid() const { return t < tiles; }
    __device__ void next() { t += stride; }
    __device__ Tile tile() {
        constexpr int X = 128 * CG;
        Tile r;
        if (grouped<CG, SWAP>(g)) {
            while (tile_start[expert + 1] <= t) ++expert;
            const int row0 = row_start[2 * expert], row1 = row_start[2 * expert + 1], rows = row1 - row0, local = t - tile_start[expert];
            const int count = (rows + g.width - 1) / g.width, channel_tile = local / count, token_tile = local - channel_tile * count;
            const int per = ((rows + count - 1) / count + 16 * CG - 1) / (16 * CG) * (16 * CG);              // equal shares, no more than g.width
            r.token = row0 + token_tile * per;
            r.token_end = min(row1, r.token + per);
            r.n = (r.token_end - r.token + 16 * CG - 1) / (16 * CG) * (16 * CG);
            r.channel = channel_tile * X;
            r.scale = expert * g.N + r.channel;
        } else {
            // bands of `band` tiles along the M side, every other one backwards along the N side: the tiles in flight share
            // their operands in L2
            const int per_band = g.band * g.tiles_y, b = t / per_band, first = b * g.band;
            const int high = min(g.band, g.tiles_x - first), within = t - b * per_band, column = within / high;
            const int tx = first + within - column * high, ty = (b & 1) ? g.tiles_y - 1 - column : column;
            r.n = g.width;
            r.token = SWAP ? ty * g.width : tx * X;
            r.token_end = SWAP ? min(g.M, r.token + g.width) : g.M;
            r.channel = SWAP ? tx * X : ty * g.width;
            r.scale = r.channel;
        }
        r.x = SWAP ? r.scale : r.token;
        r.y = SWAP ? r.token : r.scale;
        return r;
    }
};

template <int OUT>
__device__ __forceinline__ uint32_t pack_pair(float a, float b) {
    if constexpr (OUT == DTYPE_BF16) {
        const __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&p);
    } else {
        const __half2 p = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&p);
    }
}
// body(output type): one branch per block of values instead of one per value
template <typename F>
__device__ __forceinline__ void by_out(int out, F&& body) {
    if (out == DTYPE_BF16) body(std::integral_constant<int, DTYPE_BF16>{});
    else if (out == DTYPE_F16) body(std::integral_constant<int, DTYPE_F16>{});
    else body(std::integral_constant<int, DTYPE_F32>{});
}
// COUNT (even) rows of C from `c` (the first of them) on, of which `count` are there, in the column of each lane; values[i]
// is row i's. Two 16-bit values of neighbouring lanes leave as one store: the even lane writes row i, the odd one row i + 1.
template <int OUT, int COUNT>
__device__ __forceinline__ void store_column(uint8_t* c, int ld, int column, bool there, const float (&values)[COUNT], int count, int lane) {
    if constexpr (OUT == DTYPE_F32) {
        float* dst = reinterpret_cast<float*>(c) + column;
        #pragma unroll
        for (int i = 0; i < COUNT; ++i) {
            if (i < count && there) *dst = values[i];
            dst += ld;
        }
    } else {
        uint16_t* dst = reinterpret_cast<uint16_t*>(c) + (lane & 1 ? ld + column - 1 : column);
        #pragma unroll
        for (int i = 0; i < COUNT; i += 2) {
            const uint32_t own = pack_pair<OUT>(values[i], values[i + 1]), next = __shfl_xor_sync(0xFFFFFFFFu, own, 1);
            const uint32_t pair = lane & 1 ? __byte_perm(next, own, 0x7632) : __byte_perm(own, next, 0x5410);
            if (i + (lane & 1) < count && there) *reinterpret_cast<uint32_t*>(dst) = pair;
            dst += 2 * size_t(ld);
        }
    }
}
__device__ __forceinline__ float scaled(uint32_t sum, float token, float channel) {
    return __int2float_rn(int(sum)) * token * channel;
}

// Columns of a tile that each CTA of a cluster finishes: whole groups of four, and split times as many reach all columns.
__host__ __device__ __forceinline__ int run_of(int width, int split) { return (width + 4 * split - 1) / (4 * split) * 4; }

// Boxes of 128 K values per operand and ring stage, at most (Args::subs). Two where tiles are narrow: a step's instructions
// (waits, commits, requests) then serve twice the bytes (pairs: 2048 x 1024 x 8192, width 128, 19.4 -> 17.4 us; width 192
// 20.5 either way). Wide tiles keep the finer ring, and roles of their own: in the code for two 1536 x 2048 x 8192 took 25.2
// us instead of 20.5.
constexpr int SUBS = 2;

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
    // A place in the sequence of ring steps, with what a tile's requests need, computed once per tile.
    struct Cursor {
        Walk<CG, SWAP> walk;
        int ks, k0, k1, rank;
        int x, y;                   // first rows of this CTA's part (of a pair, its half) of both operands
        int parts;                  // boxes the tile takes on the N side: one, in a grouped product as many as hold its tokens
        uint32_t bytes;             // of all boxes of 128 K values, in both CTAs of a pair
        __device__ Cursor(const Walk<CG, SWAP>& w, int a, int b, int r) : walk(w), ks(a), k0(a), k1(b), rank(r) { enter(); }
        __device__ bool valid() const { return walk.valid(); }
        __device__ void enter() {
            if (!walk.valid()) return;
            const Args& g = walk.g;
            const Tile t = walk.tile();
            x = t.x + (CG == 2 ? rank * 128 : 0);
            y = t.y + (CG == 2 ? rank * (t.n / 2) : 0);
            parts = grouped<CG, SWAP>(g) ? (t.n / CG + g.y_box - 1) / g.y_box : 1;
            bytes = uint32_t(CG) * uint32_t(g.x_box + parts * g.y_box) * ROW_BYTES;
        }
        __device__ void next() {
            if (++ks < k1) return;
            ks = k0;
            walk.next();
            enter();
        }
    };
    // Boxes of a ring step that lie in K: those beyond would be zeros.
    template <int S>
    __device__ __forceinline__ int boxes(int ks) const { return S == 1 ? 1 : min(g.subs, g.kboxes - ks * g.subs); }
    // One operand's part of ring stage `stage`; x_side: the M side's.
    template <int S>
    __device__ __forceinline__ void request(const CUtensorMap* map, bool x_side, const Cursor& c, int stage) const {
        constexpr int MOST = SWAP ? 4 : 1;                      // boxes of 32 rows in 128 (a pair: 256 / 2)
        const uint32_t dst = smem + stage * stage_bytes + (x_side ? 0u : uint32_t(g.subs) * 128u * ROW_BYTES);
        const uint32_t full = smem_u32(&ctrl->full[stage]), bar = CG == 2 ? map_to_cta(full, 0) : full;
        const uint32_t pitch = (x_side ? 128u : uint32_t(g.width / CG)) * ROW_BYTES, part = uint32_t(g.y_box) * ROW_BYTES;
        const int n = boxes<S>(c.ks);
        #pragma unroll
        for (int s = 0; s < S; ++s) {
            if (s >= n) break;
            const int k = (c.ks * g.subs + s) * ROW_BYTES;
            #pragma unroll
            for (int p = 0; p < (x_side ? 1 : MOST); ++p) {
                if (p >= (x_side ? 1 : c.parts)) break;
                if constexpr (CG == 1) tma_load_2d(dst + s * pitch + p * part, map, k, (x_side ? c.x : c.y) + p * g.y_box, bar);
                else tma_load_2d_pair(dst + s * pitch + p * part, map, k, (x_side ? c.x : c.y) + p * g.y_box, bar);
            }
        }
    }
    template <int S>
    __device__ void produce(const CUtensorMap* mapX, const CUtensorMap* mapY, int lane) const {
        const CUtensorMap* weights = SWAP ? mapX : mapY;
        const CUtensorMap* tokens = SWAP ? mapY : mapX;
        Cursor cursor(Walk<CG, SWAP>(g, tile_start, row_start, unit, units), k0, k1, int(rank));
        int stage = 0;
        uint32_t phase = 0;
        if (g.early) {
            // The first ring fill: the weights at once, the tokens once the kernel that quantises them has finished.
            Cursor ahead = cursor;
            int lead = 0;
            for (; lead < g.stages && ahead.valid(); ++lead, ahead.next())
                if (elect_one()) {
                    if (CG == 1 || rank == 0) mbar_arrive_expect_tx(smem_u32(&ctrl->full[lead]), ahead.bytes * boxes<S>(ahead.ks));
                    request<S>(weights, SWAP, ahead, lead);
                }
            grid_dependency_wait();
            for (int i = 0; i < lead; ++i, cursor.next())
                if (elect_one()) request<S>(tokens, !SWAP, cursor, i);
            if (lead == g.stages) phase = 1;
            else stage = lead;
        }
        for (; cursor.valid(); cursor.next()) {
            const bool ok = wait(&ctrl->empty[stage], phase ^ 1u, lane == 0 ? STATUS_TIMEOUT_PRODUCER : 0u, 0x50000000u | (stage << 16) | cursor.ks);
            if (!__all_sync(0xFFFFFFFFu, ok)) return;
            if (elect_one()) {
                if (CG == 1 || rank == 0) mbar_arrive_expect_tx(smem_u32(&ctrl->full[stage]), cursor.bytes * boxes<S>(cursor.ks));
                request<S>(weights, SWAP, cursor, stage);
                request<S>(tokens, !SWAP, cursor, stage);
            }
            if (++stage == g.stages) { stage = 0; phase ^= 1u; }
        }
    }

    // ---- warp 4 (of the pair's first CTA) -------------------------------------------------------------------------
    template <int S>
    __device__ void issue(uint32_t tmem, uint32_t acc_stride, int lane) const {
        // Operand descriptors: rows of 128 bytes under the 128-byte swizzle, 8-row groups 1024 bytes apart, version 1.
        constexpr uint32_t DESC_HI = (1024u >> 4) | (1u << 14) | (2u << 29);
        // Instruction descriptor of kind::i8: 32-bit integer sums (2 at bit 4), A and B signed (1 at bits 7 and 10), both
        // K-major, N >> 3 at bit 17, M >> 4 at bit 24.
        const uint32_t idesc_m = (2u << 4) | (1u << 7) | (1u << 10) | (uint32_t(128 * CG >> 4) << 24);
        const uint32_t ring_lo = (smem & 0x3FFFFu) >> 4, y_pitch = uint32_t(g.width / CG) * ROW_BYTES >> 4;
        int stage = 0;
        uint32_t phase = 0, iter = 0;
        bool landed = false;                                    // the probe of this stage's barrier succeeded
        for (Walk<CG, SWAP> walk(g, tile_start, row_start, unit, units); walk.valid(); walk.next(), ++iter) {
            const uint32_t b = iter & 1u, acc = tmem + b * acc_stride, idesc = idesc_m | (uint32_t(walk.tile().n >> 3) << 17);
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
                    const int n = boxes<S>(ks);
                    #pragma unroll
                    for (int s = 0; s < S; ++s) {
                        if (s >= n) break;
                        const uint32_t x = lo + (s * 128 * ROW_BYTES >> 4), y = lo + uint32_t(g.subs) * (128 * ROW_BYTES >> 4) + s * y_pitch;
                        #pragma unroll
                        for (int j = 0; j < ROW_BYTES / MMA_K; ++j)
                            mma_i8<CG>(acc, x + (j * MMA_K >> 4), y + (j * MMA_K >> 4), DESC_HI, idesc, ks == k0 && s == 0 && j == 0 ? 0u : 1u);
                    }
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
    // The scales of a tile, loaded before its accumulator is waited for: the lane's own (of its token, or of its channel in
    // the SWAP form) and, chunk by chunk of 32 columns, that of column `lane` of each chunk this warp drains.
    struct Scales {
        float own, across[4];
        __device__ Scales(const Args& g, const Tile& t, int on_lane, int half, int lane) {
            const float* lanes = SWAP ? g.b_scale + t.scale : g.a_scale + t.token;
            const float* columns = SWAP ? g.a_scale + t.token : g.b_scale + t.scale;
            const int tokens = t.token_end - t.token, channels = g.N - t.channel;
            own = on_lane < (SWAP ? channels : tokens) ? __ldg(lanes + on_lane) : 0.0f;
            #pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int column = half * 32 + c * 64 + lane;
                across[c] = column < (SWAP ? tokens : min(g.width, channels)) ? __ldg(columns + column) : 0.0f;
            }
        }
    };
    // 32 accumulator columns of one lane. Tokens on the lanes: 32 channels of one row of C, in 32-byte stores where every
    // row starts on a 32-byte boundary. 16-byte stores of a lane's own row write each sector of C in two halves: where rows
    // start between boundaries (N an odd multiple of 8, 16-bit values) four lanes of a pair's kernel, whose many tokens may
    // make C the bound, exchange their 16-byte pieces, so that each of four stores writes 64 bytes of eight rows
    // (4820 x 24408 x 320: 84 us, without 146; 3000 x 8200 x 1024: 24.7 and 28.2).
    template <int OUT>
    __device__ __forceinline__ void store_row(const uint32_t (&v)[32], const Tile& t, int token, float own, float across, int column, int wide, int lane) const {
        constexpr int SIZE = OUT == DTYPE_F32 ? 4 : 2, WORDS = 8 * SIZE;
        uint8_t* row = g.c + (size_t(token) * g.N + t.channel + column) * SIZE;
        const int left = wide - column, count = token < t.token_end ? left : 0;  // multiples of 8, of 16 with rows_32 and 16-bit values
        auto words = [&](uint32_t* w, int first, int n) {       // of the row's 32 values, as stored
            #pragma unroll
            for (int i = 0; i < n; ++i) {
                const int at = (first + i) * (4 / SIZE);
                const float f = scaled(v[at], own, __shfl_sync(0xFFFFFFFFu, across, at));
                if constexpr (OUT == DTYPE_F32) w[i] = __float_as_uint(f);
                else w[i] = pack_pair<OUT>(f, scaled(v[at + 1], own, __shfl_sync(0xFFFFFFFFu, across, at + 1)));
            }
        };
        if (g.rows_32) {
            #pragma unroll
            for (int q = 0; q < WORDS; q += 8) {
                uint32_t w[8];
                words(w, q, 8);
                if (q * (4 / SIZE) < count)
                    asm volatile("st.global.L1::no_allocate.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                                 :: "l"(row + q * 4), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
            }
        } else if constexpr (OUT == DTYPE_F32 || CG == 1) {
            #pragma unroll
            for (int q = 0; q < WORDS; q += 4) {
                uint32_t w[4];
                words(w, q, 4);
                if (q * (4 / SIZE) < count) *reinterpret_cast<uint4*>(row + q * 4) = make_uint4(w[0], w[1], w[2], w[3]);
            }
        } else {
            uint32_t w[WORDS];
            words(w, 0, WORDS);
            const int r = lane & 3;                              // of the four lanes: afterwards piece r of each of their rows
            #pragma unroll
            for (int bit = 1; bit < 4; bit *= 2)
                #pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (i & bit) continue;
                    #pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        uint32_t& low = w[4 * i + j];
                        uint32_t& high = w[4 * (i | bit) + j];
                        const uint32_t got = __shfl_xor_sync(0xFFFFFFFFu, r & bit ? low : high, bit);
                        if (r & bit) low = got;
                        else high = got;
                    }
                }
            uint8_t* dst = row - size_t(r) * g.N * SIZE + r * 16;
            #pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (token - r + k < t.token_end && 8 * r < left)
                    *reinterpret_cast<uint4*>(dst) = make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
                dst += size_t(g.N) * SIZE;
            }
        }
    }
    // Channels on the lanes: one channel of 32 rows of C.
    template <int OUT>
    __device__ __forceinline__ void store_columns(const uint32_t (&v)[32], const Tile& t, int channel, float own, float across, int column, int wide, int lane) const {
        const int token0 = t.token + column, count = min(32, wide - column);
        uint8_t* row = g.c + size_t(token0) * g.N * (OUT == DTYPE_F32 ? 4 : 2);
        #pragma unroll
        for (int i = 0; i < 32; i += 8) {
            if (i >= count) break;
            float f[8];
            #pragma unroll
            for (int j = 0; j < 8; ++j) f[j] = scaled(v[i + j], __shfl_sync(0xFFFFFFFFu, across, i + j), own);
            store_column<OUT>(row, g.N, channel, channel < g.N, f, count - i, lane);
            row += size_t(8) * g.N * (OUT == DTYPE_F32 ? 4 : 2);
        }
    }

    __device__ void drain(uint32_t tmem, uint32_t acc_stride, int quarter, int half, int lane) const {
        if (g.early) grid_dependency_wait();                    // (without it the prologue waited)
        uint32_t iter = 0;
        for (Walk<CG, SWAP> walk(g, tile_start, row_start, unit, units); walk.valid(); walk.next(), ++iter) {
            const Tile t = walk.tile();
            const uint32_t b = iter & 1u;
            const int on_lane = quarter * 32 + lane + int(CG == 2 ? rank : 0u) * 128;
            const Scales scales(g, t, on_lane, half, lane);
            const bool ready = wait(&ctrl->acc_full[b], (iter >> 1) & 1u, lane == 0 ? STATUS_TIMEOUT_EPILOGUE : 0u, 0x70000000u | iter);
            if (!__all_sync(0xFFFFFFFFu, ready)) return;
            tc_fence_after_sync();
            const uint32_t acc = tmem + b * acc_stride + (uint32_t(quarter * 32) << 16);
            const int wide = SWAP ? t.token_end - t.token : min(g.width, g.N - t.channel);     // the tile's columns
            #pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int column = half * 32 + c * 64;
                if (column >= wide) break;
                uint32_t v[32];
                tmem_ld_32x32(acc + column, v);
                tmem_ld_wait();
                by_out(g.out, [&](auto out) {
                    if constexpr (SWAP) store_columns<decltype(out)::value>(v, t, t.channel + on_lane, scales.own, scales.across[c], column, wide, lane);
                    else store_row<decltype(out)::value>(v, t, t.token + on_lane, scales.own, scales.across[c], column, wide, lane);
                });
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

    // One tile whose K loop the cluster shares. The tile's columns are dealt to the CTAs in runs of `each`; a CTA has room for
    // its run of every member's partial sums, [split][each / 4][128 lanes][4 columns], so that lanes send and read 16 bytes
    // in a row.
    __device__ __forceinline__ int columns_of(const Tile& t) const { return SWAP ? t.token_end - t.token : min(g.width, g.N - t.channel); }
    __device__ void send(uint32_t tmem, uint32_t room, float* column_scale, int quarter, int half, int lane) const {
        if (g.early) grid_dependency_wait();
        Walk<CG, SWAP> walk(g, tile_start, row_start, unit, units);
        const Tile t = walk.tile();
        const int thread = (half * 4 + quarter) * 32 + lane, wide = columns_of(t);          // (at least as many threads as columns)
        column_scale[thread] = thread < wide ? __ldg(SWAP ? g.a_scale + t.token + thread : g.b_scale + t.scale + thread) : 0.0f;
        const bool ready = wait(&ctrl->acc_full[0], 0u, lane == 0 ? STATUS_TIMEOUT_EPILOGUE : 0u, 0x71000000u);
        if (!__all_sync(0xFFFFFFFFu, ready)) return;
        tc_fence_after_sync();
        const int each = run_of(g.width, g.split), on_lane = quarter * 32 + lane;
        for (int column = half * 32; column < wide; column += 64) {
            uint32_t v[32];
            tmem_ld_32x32(tmem + (uint32_t(quarter * 32) << 16) + column, v);
            tmem_ld_wait();
            int owner = column / each, group = (column - owner * each) / 4;
            #pragma unroll
            for (int i = 0; i < 32; i += 4) {
                if (column + i >= wide) break;
                const uint32_t at = room + uint32_t(((int(rank) * (each / 4) + group) * 128 + on_lane) * 16);
                asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};"
                             :: "r"(map_to_cta(at, uint32_t(owner))), "r"(v[i]), "r"(v[i + 1]), "r"(v[i + 2]), "r"(v[i + 3]) : "memory");
                if (++group == each / 4) { group = 0; ++owner; }
            }
        }
    }
    __device__ void finish(const int4* room, const float* column_scale, int thread) const {
        Walk<CG, SWAP> walk(g, tile_start, row_start, unit, units);
        const Tile t = walk.tile();
        const int each = run_of(g.width, g.split), on_lane = thread % 128;
        const int first = int(rank) * each, count = min(each, columns_of(t) - first);
        const bool there = on_lane < (SWAP ? g.N - t.channel : t.token_end - t.token);
        const float own = there ? __ldg(SWAP ? g.b_scale + t.scale + on_lane : g.a_scale + t.token + on_lane) : 0.0f;
        by_out(g.out, [&](auto out) {
            constexpr int OUT = decltype(out)::value, SIZE = OUT == DTYPE_F32 ? 4 : 2;
            #pragma unroll 2
            for (int group = thread / 128; group * 4 < count; group += 2) {
                int4 sum = room[group * 128 + on_lane];
                for (int s = 1; s < g.split; ++s) {
                    const int4 v = room[(s * (each / 4) + group) * 128 + on_lane];
                    sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
                }
                const int part[4] = {sum.x, sum.y, sum.z, sum.w}, column = first + group * 4;
                float f[4];
                #pragma unroll
                for (int i = 0; i < 4; ++i)
                    f[i] = SWAP ? scaled(uint32_t(part[i]), column_scale[column + i], own) : scaled(uint32_t(part[i]), own, column_scale[column + i]);
                if constexpr (SWAP) {
                    const int channel = t.channel + on_lane;
                    store_column<OUT>(g.c + size_t(t.token + column) * g.N * SIZE, g.N, channel, there, f, count - group * 4, thread & 31);
                } else if (there) {                              // four channels of one token (their number is a multiple of four)
                    uint8_t* dst = g.c + (size_t(t.token + on_lane) * g.N + t.channel + column) * SIZE;
                    if constexpr (OUT == DTYPE_F32) *reinterpret_cast<float4*>(dst) = make_float4(f[0], f[1], f[2], f[3]);
                    else *reinterpret_cast<uint2*>(dst) = make_uint2(pack_pair<OUT>(f[0], f[1]), pack_pair<OUT>(f[2], f[3]));
                }
            }
        });
    }
};

template <int CG, bool SWAP>
__global__ void __launch_bounds__(THREADS, 1)
int8_gemm_kernel(const __grid_constant__ CUtensorMap mapX, const __grid_constant__ CUtensorMap mapY, const Args g) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw), smem = (raw + 1023u) & ~1023u;
    const uint32_t stage_bytes = uint32_t(g.subs) * uint32_t(128 + g.width / CG) * ROW_BYTES;
    uint8_t* behind = smem_raw + (smem - raw) + g.stages * stage_bytes;
    Control* ctrl = reinterpret_cast<Control*>(behind);
    int* tile_start = reinterpret_cast<int*>(behind + CONTROL_BYTES);        // grouped: [experts + 1]
    int* row_start = tile_start + g.experts + 1;                             // grouped: first row and first row behind, [experts][2]
    int4* room = reinterpret_cast<int4*>(tile_start);                        // split: partial sums
    float* column_scale = reinterpret_cast<float*>(behind + CONTROL_BYTES) - 256;     // split: at the control block's end
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
    // A pair allocates Tensor Memory together: both CTAs have to be there before either begins, and stay until both have
    // given it back. (Without this barrier a CTA that was launched later than its partner, its SM still busy with the
    // kernel in front, never got out of its allocation.)
    __syncwarp();
    if constexpr (CG == 2) { cluster_arrive(); cluster_wait(); }
    if (warp == 4) tmem_alloc<CG>(smem_u32(&ctrl->tmem_base), columns);
    if (warp == 5 && lane == 0) { prefetch_tensormap(&mapX); prefetch_tensormap(&mapY); }
    if (!g.early) chain_point();
    if (grouped<CG, SWAP>(g)) {
        const int per = g.width, channel_tiles = (g.N + 128 * CG - 1) / (128 * CG);
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
    __syncwarp();
    tc_fence_before_sync();
    if (cluster) { cluster_arrive(); cluster_wait(); }
    __syncthreads();
    tc_fence_after_sync();
    if (warp == 4) tmem_relinquish<CG>();
    const uint32_t tmem = ctrl->tmem_base;

    const int members = CG == 2 ? 2 : g.split;
    Roles<CG, SWAP> roles{g, smem, stage_bytes, ctrl, tile_start, row_start, rank, int(blockIdx.x) / members, int(gridDim.x) / members,
                          CG == 2 ? map_to_cta(smem_u32(const_cast<uint32_t*>(&ctrl->wait.abort)), rank ^ 1u) : 0u,
                          g.split > 1 ? int(rank) * g.ksteps / g.split : 0, g.split > 1 ? int(rank + 1) * g.ksteps / g.split : g.ksteps};
    const bool drains = warp < 4 || warp >= 6;
    const int half = warp < 4 ? 0 : 1, thread = (half * 4 + (warp & 3)) * 32 + lane;
    if (warp == 5) {
        if ((CG == 1 || !SWAP) && g.subs > 1) roles.template produce<SUBS>(&mapX, &mapY, lane);
        else roles.template produce<1>(&mapX, &mapY, lane);
        if (g.early) grid_launch_dependents();                   // (its wait lies behind it)
    } else if (warp == 4) {
        if (CG == 1 || rank == 0) {
            if ((CG == 1 || !SWAP) && g.subs > 1) roles.template issue<SUBS>(tmem, acc_stride, lane);
            else roles.template issue<1>(tmem, acc_stride, lane);
        }
    } else if (g.split > 1) {
        roles.send(tmem, smem_u32(room), column_scale, warp & 3, half, lane);
    } else {
        roles.drain(tmem, acc_stride, warp & 3, half, lane);
        if (grouped<CG, SWAP>(g) && g.zero_rest) {
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
    if (g.split > 1 && drains && !ctrl->wait.abort) roles.finish(room, column_scale, thread);
    if (warp == 4) {
        tc_fence_after_sync();
        tmem_dealloc<CG>(tmem, columns);
        __syncwarp();
    }
    if constexpr (CG == 2) { cluster_arrive(); cluster_wait(); }
}

// ---- host -----------------------------------------------------------------------------------------------------------

std::mutex g_lock;

// CTAs (members = 1) or clusters of that many CTAs that are resident at once (one CTA per SM: its ring fills the shared
// memory). 0 for a cluster the device has no room for.
template <int CG, bool SWAP>
int resident(int device, int members) {
    static std::atomic<int> cached[64][9] = {};
    const bool known = device >= 0 && device < 64;
    if (known) {
        const int units = cached[device][members].load(std::memory_order_acquire);         // one more than what fits
        if (units) return units - 1;
    }
    std::lock_guard<std::mutex> hold(g_lock);
    auto kernel = int8_gemm_kernel<CG, SWAP>;
    cuda_check(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_LIMIT));
    int units = 0;
    cuda_check(cudaDeviceGetAttribute(&units, cudaDevAttrMultiProcessorCount, device));
    if (members > 1) {
        cudaLaunchAttribute attr{};
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim = {unsigned(members), 1, 1};
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(unsigned(units / members) * members);
        cfg.blockDim = dim3(THREADS);
        cfg.dynamicSmemBytes = SMEM_LIMIT;
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
        cuda_check(cudaOccupancyMaxActiveClusters(&units, kernel, &cfg));
    }
    if (units < 1 && members <= 2) throw std::runtime_error("int8 gemm: the kernel does not fit on this device");
    if (known) cached[device][members].store(units + 1, std::memory_order_release);
    return units;
}
int resident(const Int8Tiles& t, int device) {
    if (t.pair) return t.swap ? resident<2, true>(device, 2) : resident<2, false>(device, 2);
    return t.swap ? resident<1, true>(device, t.split) : resident<1, false>(device, t.split);
}

int round_up(int v, int to) { return (v + to - 1) / to * to; }

size_t stage_size(const Int8Tiles& t) { return size_t(t.subs) * (128 + t.width / (t.pair ? 2 : 1)) * ROW_BYTES; }
int subs_for(const Int8Tiles& t) { return t.width > (t.pair ? 160 : WIDE_FROM) ? 1 : SUBS; }

size_t table_bytes(const Int8Tiles& t, int experts) {
    return experts ? size_t(3 * experts + 1) * sizeof(int) : t.split > 1 ? size_t(t.split) * run_of(t.width, t.split) * 128 * sizeof(int) : 0;
}

// Estimated time in ns of a dense product on tiles t: launch and first data, the K loop, the exposed end of the last tile.
// The loop takes, per 128 values of K and wave, what the tensor cores need for a column (1.04 ns), what an SM takes in of
// both operands (139 bytes a ns) or what the instructions of a step cost (164 ns in a stage of two boxes, 211 in one of
// one), whichever is longest, and at least as long as both operands need to arrive. The constants are a fit to 2896 timings
// (M = 1..4096, 13 shapes of N = 512..28672, K = 2000..16384, all forms): what they pick is 0.3 % slower than the fastest on
// the mean, 11 % at worst (192 x 1032 x 2000).
float estimate(const Int8Tiles& t, int rows, int n, int k, int fit, int sms) {
    const int x = t.pair ? 256 : 128, x_rows = t.swap ? n : rows, y_rows = t.swap ? rows : n;
    const long long tiles = (long long)((x_rows + x - 1) / x) * ((y_rows + t.width - 1) / t.width), waves = (tiles + fit - 1) / fit;
    const int few = round_up(rows, 8), boxes = (k + ROW_BYTES - 1) / ROW_BYTES;
    const int taken = t.pair ? 128 + t.width / 2 : t.swap ? 128 + std::min(t.width, few) : std::min(128, few) + t.width;
    const float step = std::max({1.04f * float(t.width), float(taken * ROW_BYTES) / 139.0f, subs_for(t) > 1 ? 164.0f : 211.0f});
    const int ctas = int(std::min((long long)(sms), tiles * (t.pair ? 2 : t.split)));
    const float hbm = (float(n) + float(rows)) * float(k) / std::min(8120.0f, 91.6f * float(ctas));
    const float loop = float(waves) * float((boxes + t.split - 1) / t.split) * step;
    return 3740.0f + (t.pair ? 700.0f : 0.0f) + std::max(hbm, loop) + 14.3f * float(t.width) + 1600.0f * float(waves - 1) +
           (t.split > 1 ? 1070.0f + 14.8f * float(t.width) : 0.0f);
}

}  // namespace

Int8Tiles int8_tiles(int rows, int n, int k, int experts, int device) {
    Int8Tiles best{};
    if (experts) {
        // By the mean number of rows. From 64 on CTA pairs, whose SMs share the tokens of a tile (32 experts of 4096 x 4096,
        // mean 128: 96 us, single CTAs 118; mean 64: 89 either way; 8 experts of 2048 x 2048, mean 32: 10.8 and 9.2). Below,
        // as wide a tile as holds half as many rows again, so that most experts are one tile.
        const int mean = (rows + experts - 1) / experts;
        best.pair = mean >= 64;
        best.swap = 1;
        best.width = best.pair ? 256 : mean <= 10 ? 16 : std::min(96, round_up(mean + mean / 2, 32));
        best.split = 1;
    } else {
        float best_ns = 0.0f;
        const int sms = resident<1, false>(device, 1);
        auto consider = [&](int pair, int swap, int width, int split) {
            const Int8Tiles t{pair, swap, width, split, 0, 0};
            const int fit = resident(t, device);
            if (fit == 0) return;
            const float ns = estimate(t, rows, n, k, fit, sms);
            if (best.width == 0 || ns < best_ns) { best = t; best_ns = ns; }
        };
        const int steps = (k + SUBS * ROW_BYTES - 1) / (SUBS * ROW_BYTES);
        if (rows <= 128)
            for (int split = 1; split <= 8 && (split == 1 || steps / split >= 2); split *= 2) consider(0, 1, round_up(rows, 16), split);
        if (rows > 128)
            for (int width = 32; width <= 256; width += 32) consider(1, 0, width, 1);
        // Single CTAs with tokens on the M side: as wide as it takes for one, two or three tiles per SM, for few tokens; and,
        // where all tiles are resident at once, a cluster to a tile.
        const int high = (rows + 127) / 128;
        if (high <= 2)
            for (int waves = 1, last = 0; waves <= 3; ++waves) {
                const int across = waves * sms / high, width = std::min(256, round_up((n + across - 1) / across, 16));
                if (width != last) consider(0, 0, width, 1);
                last = width;
            }
        for (int split = 2; split <= 8 && steps / split >= 4 && high * split <= sms; split *= 2) {
            const int across = std::max(1, resident<1, false>(device, split) / high), width = round_up((n + across - 1) / across, 16);
            if (width <= 128) consider(0, 0, width, split);
        }
    }
    best.subs = subs_for(best);
    best.stages = int(std::min<size_t>(MAX_STAGES, (SMEM_LIMIT - 1024 - CONTROL_BYTES - table_bytes(best, experts)) / stage_size(best)));
    // Weights streamed by narrow tiles from many experts: 128 KB of them requested ahead per SM, no more (256 experts of
    // 4096 x 4096, six routes of 64 tokens: 470 us, with the 192 KB there is room for 488; 1024 tokens 637 and 665). One
    // matrix is streamed faster with all of the room (1 x 28672 x 8192: 40.1 us, 41.0 with 128 KB).
    if (experts && best.subs > 1) best.stages = std::min(best.stages, 4);
    return best;
}

namespace {

void run(const int8_t* a, const int8_t* b, const float* a_scales, const float* b_scales, const int* offsets, int experts, void* C,
         int out_dtype, int M, int N, int K, bool zero_rest, bool early, cudaStream_t stream) {
    int device = 0;
    cuda_check(cudaGetDevice(&device));
    const Int8Tiles t = int8_tiles(M, N, K, experts, device);
    // Boxes of the tokens' operand: no more rows than there are (rounded up to a swizzle group), in a grouped product 32 rows
    // each. What a stage holds beyond them is whatever was there: any byte is a number, a row of the product depends on its
    // own row alone, and rows that do not exist are not stored.
    const int x_tile = t.pair ? 256 : 128, half = t.pair ? 2 : 1, few = round_up(M, 8);
    const int x_box = t.swap || t.pair ? 128 : std::min(128, few);
    const int y_box = !t.swap ? t.width / half : experts ? std::min(32, t.width) : std::min(t.width, few);
    Args g{};
    g.M = M;
    g.N = N;
    g.kboxes = (K + ROW_BYTES - 1) / ROW_BYTES;
    g.subs = t.subs;
    g.ksteps = (g.kboxes + t.subs - 1) / t.subs;
    g.width = t.width;
    g.stages = t.stages;
    g.split = t.split;
    g.x_box = x_box;
    g.y_box = y_box;
    g.a_scale = a_scales;
    g.b_scale = b_scales;
    g.c = static_cast<uint8_t*>(C);
    g.out = out_dtype;
    g.rows_32 = reinterpret_cast<uintptr_t>(C) % 32 == 0 && size_t(N) * dtype_bytes(out_dtype) % 32 == 0 ? 1 : 0;
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
        tiles = ((long long)(M) / t.width + std::min(M, experts)) * g.tiles_x;
    }
    if (tiles > 0x3FFFFFFFll) throw std::invalid_argument("int8 gemm: too many tiles");
    const int fit = resident(t, device);
    const int units = t.split > 1 ? int(tiles) : int(std::min<long long>(tiles, fit));
    g.band = 1;
    while ((g.band + 1) * (g.band + 1) <= fit) ++g.band;        // about as many operand rows on either side in flight
    g.band = std::min(g.band, g.tiles_x);
    const CUtensorMap tokens = byte_rows_map(a, size_t(M), size_t(K), t.swap ? y_box : x_box);
    const CUtensorMap weights = byte_rows_map(b, size_t(N) * std::max(1, experts), size_t(K), t.swap ? x_box : y_box);
    const int members = t.pair ? 2 : t.split;
    cudaLaunchAttribute attrs[2]{};
    attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[0].val.programmaticStreamSerializationAllowed = 1;
    attrs[1].id = cudaLaunchAttributeClusterDimension;
    attrs[1].val.clusterDim = {unsigned(members), 1, 1};
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(unsigned(units) * unsigned(members));
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = 1024 + size_t(t.stages) * stage_size(t) + CONTROL_BYTES + table_bytes(t, experts);
    cfg.stream = stream;
    cfg.attrs = attrs;
    cfg.numAttrs = members > 1 ? 2 : 1;
    if (t.pair && t.swap) cuda_check(cudaLaunchKernelEx(&cfg, int8_gemm_kernel<2, true>, weights, tokens, g));
    else if (t.pair) cuda_check(cudaLaunchKernelEx(&cfg, int8_gemm_kernel<2, false>, tokens, weights, g));
    else if (t.swap) cuda_check(cudaLaunchKernelEx(&cfg, int8_gemm_kernel<1, true>, weights, tokens, g));
    else cuda_check(cudaLaunchKernelEx(&cfg, int8_gemm_kernel<1, false>, tokens, weights, g));
    g_launches.fetch_add(1, std::memory_order_relaxed);
}

}  // namespace

void int8_gemm_check(const void* a, const void* b, const float* a_scales, const float* b_scales, const void* C, int out_dtype,
                     int M, int N, int K) {
    if (M < 0 || N < 1 || K < 1 || M > 1 << 30 || N > 1 << 30) throw std::invalid_argument("int8 gemm: N and K must be positive, M not negative, M and N at most 2^30");
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
    if ((long long)(experts) * N > 1 << 30) throw std::invalid_argument("int8 grouped gemm: experts * N must be at most 2^30");
    if (!offsets) throw std::invalid_argument("int8 grouped gemm: null pointer");
    if (R == 0) return;
    run(rows, weights, row_scales, weight_scales, offsets, experts, C, out_dtype, R, N, K, zero_rest, false, stream);
}

}  // namespace nvfp4_b200
