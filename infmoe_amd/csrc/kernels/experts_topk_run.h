// The experts' feed-forward products of a top-k routing for gfx950:
//   y_t = sum_j weights[t][j] * wo_e act(wi_e x_t [, wi_1_e x_t]),  e = ids[t][j].
//
// Launches:
//   plan     the slots (t, j) sorted by expert (stable: results do not depend on the order anything retires in) and cut
//            into row tiles, on the device (calls of more than kPlanBlock slots count per block first, long ones add the counts up);
//   product  1: rows x_t gathered by slot, activation in the epilogue, hidden rows in the weights' type;
//   product  2: hidden rows against wo, FP32 rows in slot order;
//   combine  the k rows of a token, weighted and added in order.
// Hidden rows are rounded to the weights' type, as any network of that type does between two products: it is the type the
// second product's operand has.  The rows that combine adds stay in FP32: one more rounding there would be seen in y.
//
// Included by experts_topk_{f32,f16,bf16}.hip, which compile it for one type each, side by side.
//
// Three forms of the products, by rows per expert on average (slots / E):
//   up to 8 (16 where there are no tall tiles)
//              the weights streamed once through the registers, tiles of 16 rows (up to 4 on average) or 32 (stream_kernel).
//              At 4 a tile of 64 x 128 through LDS took 1.05 ms where the stream takes 0.85 (32 experts of 4096 x 10240);
//   more       tall tiles where there are enough for the compute units (tall_kernel): 4096 tokens over the same experts take
//              4.9 ms in tiles of 64 x 128 and 2.4 in tall ones; with 96 tall tiles for 256 compute units, f32, 3009 rows
//              over 16 experts of 1000 x 1500, 0.67 ms and 0.24 in the small ones;
//   otherwise, and for rows that are not whole 16-byte pieces, tiles of 64 x 128 (product_kernel).
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>

#include "forms.h"
#include "kernels.h"
#include "row_gemm.h"
#include "row_stream.h"
#include "row_tall.h"

namespace infmoe {
namespace {

using namespace rows;
using forms::kMiniSlots;

constexpr int kPlanBlock = 1024;  // slots ranked by one workgroup
constexpr int kPlanWaves = kPlanBlock / 64;
// Blocks up to which plan_place_kernel adds the counts up itself, blocks * blocks * E of them: without the launch between, 8
// blocks of 256 experts take 26.3 us (whole call, d = h = 32; with it 27.2), 16 blocks 31.2 (30.1), 32 blocks 41.3 (38.0), 1024
// blocks 1680 (1160), 4096 blocks 19960 (4510).
constexpr int kPlanScan = 16;
constexpr int kRunTiles = 8;  // row tiles of an expert that are multiplied side by side (place_of)

// ---------------------------------------------------------------- plan
__global__ __launch_bounds__(kPlanBlock) void plan_count_kernel(int S, int E, const int* __restrict__ ids, int* __restrict__ hist) {
    extern __shared__ int s_hist[];
    for (int e = threadIdx.x; e < E; e += kPlanBlock) s_hist[e] = 0;
    __syncthreads();
    const int s = blockIdx.x * kPlanBlock + threadIdx.x;
    const int e = s < S ? ids[s] : -1;
    if (e >= 0 && e < E) atomicAdd(&s_hist[e], 1);  // integer sums: order-free
    __syncthreads();
    for (int i = threadIdx.x; i < E; i += kPlanBlock) hist[(size_t)blockIdx.x * E + i] = s_hist[i];
}

// hist[b][e] becomes the sum of the blocks before b, hist[blocks][e] that of all.  A lane per expert, the blocks cut into a
// stretch per wave: every wave adds up its own, then goes over it again from the sum of the stretches before it.
__global__ __launch_bounds__(kPlanBlock) void plan_scan_kernel(int blocks, int E, int* __restrict__ hist) {
    __shared__ int s_sum[kPlanWaves][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, e = blockIdx.x * 64 + lane;
    const int b0 = (int)((long long)blocks * wave / kPlanWaves), b1 = (int)((long long)blocks * (wave + 1) / kPlanWaves);
    int sum = 0;
    if (e < E) {
#pragma unroll 8
        for (int b = b0; b < b1; ++b) sum += hist[(size_t)b * E + e];
    }
    s_sum[wave][lane] = sum;
    __syncthreads();
    if (e >= E) return;
    int run = 0, all = 0;
    for (int w = 0; w < kPlanWaves; ++w) {
        run += w < wave ? s_sum[w][lane] : 0;
        all += s_sum[w][lane];
    }
#pragma unroll 8
    for (int b = b0; b < b1; ++b) {
        const int c = hist[(size_t)b * E + e];
        hist[(size_t)b * E + e] = run;
        run += c;
    }
    if (wave == 0) hist[(size_t)blocks * E + e] = all;
}

// Exclusive prefix of v over the workgroup's kPlanBlock threads; *total: the sum.
__device__ __forceinline__ int block_prefix(int v, int* s_wave, int* total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int run = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int up = __shfl_up(run, d);
        if (lane >= d) run += up;
    }
    if (lane == 63) s_wave[wave] = run;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kPlanWaves; ++w) {
        before += w < wave ? s_wave[w] : 0;
        all += s_wave[w];
    }
    __syncthreads();
    *total = all;
    return before + run - v;
}

// row_slot[r]: slot of the r-th row in expert order; tiles / n_tiles: its cut into tiles of at most tile_rows rows, each
// (expert, first row, rows, place in its run | length of the run << 8).  Slots
// whose id is no expert get no row.  One block (hist null) needs no counts of others; a few (scanned false) add up each other's
// counts themselves, so that no launch lies between counting and placing; many find their prefixes in hist.
__global__ __launch_bounds__(kPlanBlock) void plan_place_kernel(int S, int E, const int* __restrict__ ids, const int* __restrict__ hist,
                                                                bool scanned, int tile_rows, int* __restrict__ row_slot, int4* __restrict__ tiles,
                                                                int* __restrict__ n_tiles) {
    extern __shared__ int s_dyn[];  // [kPlanWaves][E]: rows of each expert in this block, by wave
    __shared__ int s_wave[kPlanWaves];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int i = threadIdx.x; i < kPlanWaves * E; i += kPlanBlock) s_dyn[i] = 0;
    __syncthreads();
    const int s = blockIdx.x * kPlanBlock + threadIdx.x;
    int e = s < S ? ids[s] : -1;
    if (e >= E) e = -1;
    const bool valid = e >= 0;
    // lanes of this wave with the same expert: one ballot per bit of the index
    unsigned long long same = __ballot(valid);
    for (int bit = 0; (1 << bit) < E; ++bit) {
        const unsigned long long m = __ballot(valid && ((e >> bit) & 1));
        same &= (e >> bit) & 1 ? m : ~m;
    }
    const int rank = __popcll(same & (lane == 0 ? 0ull : ~0ull >> (64 - lane)));
    if (valid && rank == 0) s_dyn[wave * E + e] = __popcll(same);
    __syncthreads();
    // thread i: expert i (E <= kPlanBlock)
    const int i = threadIdx.x;
    int count = 0, earlier = 0;
    if (i < E) {
        if (hist == nullptr) {
            for (int w = 0; w < kPlanWaves; ++w) count += s_dyn[w * E + i];
        } else if (scanned) {
            earlier = hist[(size_t)blockIdx.x * E + i];
            count = hist[(size_t)gridDim.x * E + i];
        } else {
            for (int b = 0; b < (int)gridDim.x; ++b) {
                const int c = hist[(size_t)b * E + i];
                earlier += b < (int)blockIdx.x ? c : 0;
                count += c;
            }
        }
    }
    int total = 0;
    const int offset = block_prefix(count, s_wave, &total);
    if (i < E) {
        int run = offset + earlier;
        for (int w = 0; w < kPlanWaves; ++w) {
            const int c = s_dyn[w * E + i];
            s_dyn[w * E + i] = run;
            run += c;
        }
    }
    if (blockIdx.x == 0) {
        const int mine = (count + tile_rows - 1) / tile_rows;
        int n = 0;
        const int first = block_prefix(mine, s_wave, &n);
        // as few tiles as the height allows, of one height (a multiple of 32 where tiles are that tall)
        const int even = mine > 1 ? (count + mine - 1) / mine : tile_rows;
        const int height = tile_rows > 64 ? (even + 31) / 32 * 32 : tile_rows;
        for (int j = 0; j < mine; ++j) tiles[first + j] = int4{i, offset + j * height, min(height, count - j * height), j % kRunTiles | min(kRunTiles, mine - j / kRunTiles * kRunTiles) << 8};
        if (i == 0) *n_tiles = n;
    }
    __syncthreads();
    if (valid) row_slot[s_dyn[wave * E + e] + rank] = s;
}

// ---------------------------------------------------------------- products
struct Product {
    const char* a;             // rows
    const char *b, *b1;        // weights of expert 0 (b1: the second matrix of a gated first product)
    void* c;
    const int* row_slot;
    const int4* tiles;
    const int* n_tiles;
    long long a_stride, b_expert;  // bytes
    int k_slots;               // slots per token (first product: row r is token row_slot[r] / k_slots)
    int N, K, ffn;
};

// What workgroup blockIdx.x of a grid over (row tiles x column tiles) computes.  Workgroups are dealt to the dies in turn; each
// die takes a contiguous stretch of the work, in which the row tiles of an expert (runs of up to kRunTiles) stand side by
// side column tile by column tile: those at work in a die at one time read the same weight rows, once from memory and then
// from its L2, and the same few row tiles.  (f32, 16 experts of 1000 x 1500 with 188 rows each: 240 us in plain order, in
// which every row tile fetches the weights anew.)  Returns false where the grid has room for more tiles than there are.
__device__ __forceinline__ bool place_of(const int4* __restrict__ tiles, int n_tiles, int cols, int* tile, int* col) {
    const int all = n_tiles * cols, share = (all + kXcdCount - 1) / kXcdCount;
    const int mine = blockIdx.x / kXcdCount, id = (int)(blockIdx.x % kXcdCount) * share + mine;
    if (mine >= share || id >= all) return false;
    const int t = id / cols, run = tiles[t].w, head = t - (run & 255), length = run >> 8;
    const int in_run = id - head * cols;
    *tile = head + in_run % length;
    *col = in_run / length;
    return true;
}

// FIRST: A gathered, activation, C rows in expert order in T.  Otherwise A in expert order, C rows in slot order in FP32.
template <typename T, typename S, bool FIRST, bool GATED, bool ALIGNED>
__global__ __launch_bounds__(S::kThreads) void product_kernel(Product p) {
    extern __shared__ __align__(16) char lds[];
    constexpr int NM = GATED ? 2 : 1, kOut = S::kCols / NM;  // columns of C per tile
    const int cols = (p.N + kOut - 1) / kOut;
    int t, col;
    if (!place_of(p.tiles, *p.n_tiles, cols, &t, &col)) return;
    const int n0 = col * kOut;
    const int4 tile = p.tiles[t];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = wave / S::WN, wn = wave % S::WN;
    const int row_bytes = p.K * (int)sizeof(T);
    const char* pa[S::kPiecesA];
    const char* pb[S::kPiecesB];
#pragma unroll
    for (int i = 0; i < S::kPiecesA; ++i) {
        const int r = tile.y + min((tid >> 3) + i * (S::kThreads / 8), tile.z - 1);  // (rows past the tile's repeat its last)
        pa[i] = p.a + (FIRST ? (long long)(p.row_slot[r] / p.k_slots) : (long long)r) * p.a_stride;
    }
#pragma unroll
    for (int i = 0; i < S::kPiecesB; ++i) {
        // a wave's FN column blocks are half of the first matrix, half of the second when there are two
        const int v = (tid >> 3) + i * (S::kThreads / 8), w = v / (16 * S::FN), q = v % (16 * S::FN);
        const int m = q / (16 * S::FN / NM), n = n0 + w * (16 * S::FN / NM) + q % (16 * S::FN / NM);
        pb[i] = (m ? p.b1 : p.b) + tile.x * p.b_expert + (long long)min(n, p.N - 1) * row_bytes;
    }
    v4f acc[S::FM][S::FN];
#pragma unroll
    for (int i = 0; i < S::FM; ++i)
#pragma unroll
        for (int j = 0; j < S::FN; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
    multiply<T, S, ALIGNED>(acc, lds, pa, pb, row_bytes);
#pragma unroll
    for (int i = 0; i < S::FM; ++i) {
        const int r = (wm * S::FM + i) * 16 + (lane & 15);
        if (r >= tile.z) continue;
        const int row = tile.y + r;
#pragma unroll
        for (int j = 0; j < S::FN / NM; ++j) {
            const int n = n0 + (wn * (S::FN / NM) + j) * 16 + (lane >> 4) * 4;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                if (n + q >= p.N) continue;
                if constexpr (FIRST)
                    static_cast<T*>(p.c)[(size_t)row * p.N + n + q] = (T)activate<T>(p.ffn, acc[i][j][q], GATED ? acc[i][j + S::FN / 2][q] : 0.f);
                else
                    static_cast<float*>(p.c)[(size_t)p.row_slot[row] * p.N + n + q] = acc[i][j][q];
            }
        }
    }
}

// ---- many rows per expert (row_tall.h).  The height of a tile is a run-time multiple of 32 rows.
template <typename T, int FM, bool FIRST, bool GATED>
__device__ __forceinline__ void tall_body(const Product& p, const int4& tile, int n0, char* lds) {
    constexpr int F = GATED ? 2 : 4, kWaveCols = 16 * F;
    using W = Tall<FM, F>;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave >> 2, wn = wave & 3;
    const int row_bytes = p.K * (int)sizeof(T);
    const char *pa[W::kPiecesA], *pb[4];
#pragma unroll
    for (int i = 0; i < W::kPiecesA; ++i) {
        const int r = tile.y + min(W::row_a(i), tile.z - 1);
        pa[i] = p.a + (FIRST ? (long long)(p.row_slot[r] / p.k_slots) : (long long)r) * p.a_stride + W::byte_a(i);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int v = W::row_b(i), q = v & 63, n = n0 + (v >> 6) * kWaveCols + q % kWaveCols;
        pb[i] = (q >= kWaveCols ? p.b1 : p.b) + tile.x * p.b_expert + (long long)min(n, p.N - 1) * row_bytes + W::byte_b(i);
    }
    v4f acc[FM][4];
    tall_multiply<T, FM, F>(acc, lds, pa, pb, row_bytes);
    const bool whole = p.N % (16 / (FIRST ? (int)sizeof(T) : 4)) == 0;
#pragma unroll
    for (int i = 0; i < FM; ++i) {
        const int r = (wm * FM + i) * 16 + (lane & 15);
        if (r >= tile.z) continue;
        const int row = tile.y + r, n = n0 + wn * kWaveCols + W::column();
        if constexpr (FIRST)
            write_columns<T, 4 * F>(static_cast<T*>(p.c) + (size_t)row * p.N, n, p.N, whole, [&](int c) {
                return activate<T>(p.ffn, acc[i][c >> 2][c & 3], GATED ? acc[i][(c >> 2) + 4 - F][c & 3] : 0.f);
            });
        else
            write_columns<float, 4 * F>(static_cast<float*>(p.c) + (size_t)p.row_slot[row] * p.N, n, p.N, whole,
                                        [&](int c) { return acc[i][c >> 2][c & 3]; });
    }
}

template <typename T, bool FIRST, bool GATED>
__global__ __launch_bounds__(kTallThreads) void tall_kernel(Product p) {
    extern __shared__ __align__(16) char lds[];
    constexpr int kOut = GATED ? kTallCols / 2 : kTallCols;
    const int cols = (p.N + kOut - 1) / kOut;
    int t, col;
    if (!place_of(p.tiles, *p.n_tiles, cols, &t, &col)) return;
    const int4 tile = p.tiles[t];
    const int n0 = col * kOut;
    switch ((tile.z + 31) / 32) {
        case 1:
        case 2: tall_body<T, 2, FIRST, GATED>(p, tile, n0, lds); break;
        case 3: tall_body<T, 3, FIRST, GATED>(p, tile, n0, lds); break;
        case 4: tall_body<T, 4, FIRST, GATED>(p, tile, n0, lds); break;
        case 5: tall_body<T, 5, FIRST, GATED>(p, tile, n0, lds); break;
        case 6: tall_body<T, 6, FIRST, GATED>(p, tile, n0, lds); break;
        case 7: tall_body<T, 7, FIRST, GATED>(p, tile, n0, lds); break;
        default: tall_body<T, 8, FIRST, GATED>(p, tile, n0, lds); break;
    }
}

// ---- few rows per expert: the weights streamed through the registers (row_stream.h)
// Hidden rows in slot order here, so that calls of up to kMiniSlots slots need no plan: every wave finds the slots of its
// expert among the ids by ballots.  (Up to 64 slots are one ballot; the t-th expert in use is that of the t-th slot whose
// expert does not occur before it.)
struct FewRows {
    const int* ids;
    int S, E;  // ids: null when there is a plan
};

template <typename T, int FM, int FN, bool FIRST, bool GATED, bool ALIGNED>
__global__ __launch_bounds__(kStreamThreads) void stream_kernel(Product p, FewRows few) {
    extern __shared__ __align__(16) char lds[];
    __shared__ int s_slot[kMiniSlots];
    constexpr int NM = GATED ? 2 : 1, kOut = 16 * FN / NM, kTile = 16 * FM;
    const int cols = (p.N + kOut - 1) / kOut;
    const int t = blockIdx.x / cols, n0 = blockIdx.x % cols * kOut;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int expert, count, first_row = 0;
    if (few.ids != nullptr) {
        int e = lane < few.S ? few.ids[lane] : -1;
        const bool valid = e >= 0 && e < few.E;
        unsigned long long same = __ballot(valid);
        for (int bit = 0; (1 << bit) < few.E; ++bit) {
            const unsigned long long m = __ballot(valid && ((e >> bit) & 1));
            same &= (e >> bit) & 1 ? m : ~m;
        }
        const unsigned long long below = lane == 0 ? 0ull : ~0ull >> (64 - lane);
        const bool first = valid && (same & below) == 0;
        const unsigned long long firsts = __ballot(first);
        const unsigned long long chosen = __ballot(first && __popcll(firsts & below) == t);
        if (chosen == 0) return;  // fewer experts in use
        expert = __builtin_amdgcn_readlane(e, __ffsll((long long)chosen) - 1);
        const unsigned long long mine = __ballot(valid && e == expert);
        count = __popcll(mine);
        if (wave == 0 && valid && e == expert) s_slot[__popcll(mine & below)] = lane;
        __syncthreads();
    } else {
        if (t >= *p.n_tiles) return;
        const int4 tile = p.tiles[t];
        expert = tile.x, first_row = tile.y, count = tile.z;
    }
    auto slot_of = [&](int r) { return few.ids != nullptr ? s_slot[r] : p.row_slot[first_row + r]; };
    const int row_bytes = p.K * (int)sizeof(T), steps = (row_bytes + kStepBytes - 1) / kStepBytes;
    const char* pw[FN];
#pragma unroll
    for (int j = 0; j < FN; ++j) {
        const int n = n0 + j % (FN / NM) * 16 + (lane & 15);
        pw[j] = (j >= FN / NM ? p.b1 : p.b) + expert * p.b_expert + (long long)min(n, p.N - 1) * row_bytes;
    }
    for (int r0 = 0; r0 < count; r0 += kTile) {  // (more than one round only without a plan)
        const char* px[FM];
#pragma unroll
        for (int i = 0; i < FM; ++i) {
            const int slot = slot_of(min(r0 + i * 16 + (lane & 15), count - 1));
            px[i] = p.a + (long long)(FIRST ? slot / p.k_slots : slot) * p.a_stride;
        }
        v4f acc[FM][FN];
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
        stream_steps<T, FM, FN, ALIGNED>(acc, px, pw, steps * wave / kStreamWaves, steps * (wave + 1) / kStreamWaves, row_bytes, [] {});
        if (r0 > 0) __syncthreads();  // the last round's sums have been taken
        join_waves<FM, FN, NM>(lds, acc, [&](int i, int j, const v4f(&sum)[NM]) {
            const int r = r0 + i * 16 + (lane & 15), n = n0 + j * 16 + (lane >> 4) * 4;
            if (r >= count) return;
            const size_t at = (size_t)slot_of(r) * p.N + n;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                if (n + q >= p.N) continue;
                if constexpr (FIRST)
                    static_cast<T*>(p.c)[at + q] = (T)activate<T>(p.ffn, sum[0][q], GATED ? sum[NM - 1][q] : 0.f);
                else
                    static_cast<float*>(p.c)[at + q] = sum[0][q];
            }
        });
    }
}

// ---------------------------------------------------------------- combine
// A thread per COLS columns of a token: four where there are enough of them (16-byte reads), one in small batches, where the
// time is that of one read after the other.
template <typename T, int COLS>
__global__ __launch_bounds__(256) void combine_kernel(int T_n, int d, int k, int E, const int* __restrict__ ids, const float* __restrict__ weights,
                                                      const float* __restrict__ post, T* __restrict__ y, long long y_stride) {
    typedef float Row __attribute__((ext_vector_type(COLS)));
    struct alignas(COLS * sizeof(T)) Out {
        T e[COLS];
    };
    const int n = (blockIdx.y * 256 + threadIdx.x) * COLS;
    if (n >= d) return;
    for (size_t t = blockIdx.x; t < (size_t)T_n; t += gridDim.x) {
        float sum[COLS];
#pragma unroll
        for (int q = 0; q < COLS; ++q) sum[q] = 0.f;
#pragma unroll 4
        for (int j = 0; j < k; ++j) {
            const int e = ids[t * k + j];
            const float w = weights[t * k + j];
            const Row v = *reinterpret_cast<const Row*>(post + (t * k + j) * d + n);  // (of a slot without an expert: never written)
#pragma unroll
            for (int q = 0; q < COLS; ++q) {
                sum[q] += w * (e >= 0 && e < E ? v[q] : 0.f);
            }
        }
        Out out;
#pragma unroll
        for (int q = 0; q < COLS; ++q) out.e[q] = (T)sum[q];
        *reinterpret_cast<Out*>(y + t * y_stride + n) = out;
    }
}

// ---------------------------------------------------------------- host
struct Carve {
    int *row_slot, *n_tiles, *hist;
    int4* tiles;
    char* hidden;
    float* post;
    size_t total;
};
constexpr int kMinTile = 16;

Carve carve(int T, int k, int E, int d, int h, int dtype, char* base) {
    const size_t S = (size_t)T * k, size = dtype == DTYPE_F32 ? 4 : 2;
    size_t off = 0;
    auto take = [&](size_t bytes) {
        char* at = base ? base + off : nullptr;
        off += (bytes + 255) & ~(size_t)255;
        return at;
    };
    Carve c;
    c.row_slot = reinterpret_cast<int*>(take(4 * S));
    c.n_tiles = reinterpret_cast<int*>(take(4));
    c.hist = reinterpret_cast<int*>(take(4 * ((S + kPlanBlock - 1) / kPlanBlock + 1) * E));
    c.tiles = reinterpret_cast<int4*>(take(sizeof(int4) * (S / kMinTile + std::min<size_t>(E, S))));
    c.hidden = take(S * h * size);
    c.post = reinterpret_cast<float*>(take(S * d * 4));
    c.total = off;
    return c;
}

template <typename T, typename S, bool FIRST, bool GATED>
hipError_t go(const Product& p, int max_tiles, bool aligned, hipStream_t stream) {
    const int out = S::kCols / (GATED ? 2 : 1);
    const long long grid = ((long long)max_tiles * ((p.N + out - 1) / out) + kXcdCount - 1) / kXcdCount * kXcdCount;
    if (aligned) {
        if (const hipError_t err = allow_lds_once<product_kernel<T, S, FIRST, GATED, true>>(S::kLds); err != hipSuccess) return err;
        product_kernel<T, S, FIRST, GATED, true><<<(int)grid, S::kThreads, S::kLds, stream>>>(p);
    } else {
        if (const hipError_t err = allow_lds_once<product_kernel<T, S, FIRST, GATED, false>>(S::kLds); err != hipSuccess) return err;
        product_kernel<T, S, FIRST, GATED, false><<<(int)grid, S::kThreads, S::kLds, stream>>>(p);
    }
    return hipGetLastError();
}

template <typename T, bool FIRST, bool GATED>
hipError_t go_tall(const Product& p, int max_tiles, hipStream_t stream) {
    constexpr int out = GATED ? kTallCols / 2 : kTallCols;
    const long long grid = ((long long)max_tiles * ((p.N + out - 1) / out) + kXcdCount - 1) / kXcdCount * kXcdCount;
    if (const hipError_t err = allow_lds_once<tall_kernel<T, FIRST, GATED>>(kTallLds); err != hipSuccess) return err;
    tall_kernel<T, FIRST, GATED><<<(int)grid, kTallThreads, kTallLds, stream>>>(p);
    return hipGetLastError();
}

template <typename T, int FM, int FN, bool FIRST, bool GATED>
hipError_t go_stream(const Product& p, const FewRows& few, int max_tiles, bool aligned, hipStream_t stream) {
    constexpr int out = 16 * FN / (GATED ? 2 : 1), lds = stream_lds<FM, FN>();
    const long long grid = (long long)max_tiles * ((p.N + out - 1) / out);
    if (aligned) {
        if (const hipError_t err = allow_lds_once<stream_kernel<T, FM, FN, FIRST, GATED, true>>(lds); err != hipSuccess) return err;
        stream_kernel<T, FM, FN, FIRST, GATED, true><<<(int)grid, kStreamThreads, lds, stream>>>(p, few);
    } else {
        if (const hipError_t err = allow_lds_once<stream_kernel<T, FM, FN, FIRST, GATED, false>>(lds); err != hipSuccess) return err;
        stream_kernel<T, FM, FN, FIRST, GATED, false><<<(int)grid, kStreamThreads, lds, stream>>>(p, few);
    }
    return hipGetLastError();
}

template <typename T, int FM, bool FIRST, bool GATED>
hipError_t go_few(const Product& p, const FewRows& few, int max_tiles, bool aligned, hipStream_t stream) {
    const int fn = forms::stream_blocks(max_tiles, p.N, GATED);
    if (fn == 4) return go_stream<T, FM, 4, FIRST, GATED>(p, few, max_tiles, aligned, stream);
    if (GATED || fn == 2) return go_stream<T, FM, 2, FIRST, GATED>(p, few, max_tiles, aligned, stream);
    if constexpr (!GATED) return go_stream<T, FM, 1, FIRST, GATED>(p, few, max_tiles, aligned, stream);
    return hipErrorInvalidValue;
}

template <typename T>
hipError_t run(int Tn, int k, int E, int d, int h, int ffn, const T* x, long long x_stride, const int* ids, const float* weights,
               const T* wi, const T* wi_1, const T* wo, long long wi_stride, long long wo_stride, T* y, long long y_stride,
               const Carve& c, hipStream_t stream) {
    using S = Shape<1, 4, 4, 2>;
    const int slots = Tn * k, blocks = (slots + kPlanBlock - 1) / kPlanBlock;
    auto on16 = [](const void* p, long long stride) { return ((reinterpret_cast<uintptr_t>(p) | (uintptr_t)(stride * (long long)sizeof(T))) & 15) == 0; };
    const bool in_ok = d * sizeof(T) % 16 == 0 && on16(x, x_stride) && on16(wi, wi_stride) && on16(wi_1, 0);
    const bool out_ok = h * sizeof(T) % 16 == 0 && on16(wo, wo_stride);
    const forms::Experts form = forms::experts_form(slots, E, d, h, sizeof(T), in_ok && out_ok);
    static_assert(forms::kTallTileRows == kTallRows && forms::kTallCutCols == kTallCols && forms::kSmallTileRows == S::kRows, "the tiles that forms.h counts");
    const int few_blocks = form.blocks, tile_rows = form.tile_rows, max_tiles = form.max_tiles;
    const bool mini = form.mini, tall = form.kind == forms::Experts::TALL;
    // a launch has fewer than 2^32 work items in x (where a streamed product has that many, go_few takes 64 weight rows each)
    const int out = few_blocks > 0 ? 64 : tall ? kTallCols : S::kCols, threads = few_blocks > 0 ? kStreamThreads : tall ? kTallThreads : S::kThreads;
    auto items = [&](int N, int each) { return ((long long)max_tiles * ((N + each - 1) / each) + kXcdCount) * threads; };
    if (items(h, ffn == FFN_RELU ? out : out / 2) >= 1ll << 32 || items(d, out) >= 1ll << 32) return hipErrorInvalidConfiguration;
    if (!mini) {
        if (blocks > 1) plan_count_kernel<<<blocks, kPlanBlock, 4 * E, stream>>>(slots, E, ids, c.hist);
        if (blocks > kPlanScan) plan_scan_kernel<<<(E + 63) / 64, kPlanBlock, 0, stream>>>(blocks, E, c.hist);
        const size_t lds = 4 * (size_t)kPlanWaves * E;
        if (const hipError_t err = allow_lds_once<plan_place_kernel>(4 * kPlanWaves * kRouteMaxExperts); err != hipSuccess) return err;
        plan_place_kernel<<<blocks, kPlanBlock, lds, stream>>>(slots, E, ids, blocks > 1 ? c.hist : nullptr, blocks > kPlanScan, tile_rows, c.row_slot, c.tiles, c.n_tiles);
    }
    const FewRows few{mini ? ids : nullptr, slots, E};
    Product p{};
    p.row_slot = c.row_slot, p.tiles = c.tiles, p.n_tiles = c.n_tiles, p.k_slots = k, p.ffn = ffn;
    p.a = reinterpret_cast<const char*>(x), p.a_stride = x_stride * sizeof(T);
    p.b = reinterpret_cast<const char*>(wi), p.b1 = reinterpret_cast<const char*>(wi_1), p.b_expert = wi_stride * sizeof(T);
    p.c = c.hidden, p.N = h, p.K = d;
    hipError_t err;
    if (ffn == FFN_RELU)
        err = few_blocks == 1   ? go_few<T, 1, true, false>(p, few, max_tiles, in_ok, stream)
              : few_blocks == 2 ? go_few<T, 2, true, false>(p, few, max_tiles, in_ok, stream)
              : tall            ? go_tall<T, true, false>(p, max_tiles, stream)
                                : go<T, S, true, false>(p, max_tiles, in_ok, stream);
    else
        err = few_blocks == 1   ? go_few<T, 1, true, true>(p, few, max_tiles, in_ok, stream)
              : few_blocks == 2 ? go_few<T, 2, true, true>(p, few, max_tiles, in_ok, stream)
              : tall            ? go_tall<T, true, true>(p, max_tiles, stream)
                                : go<T, S, true, true>(p, max_tiles, in_ok, stream);
    if (err != hipSuccess) return err;
    p.a = c.hidden, p.a_stride = (long long)h * sizeof(T);
    p.b = reinterpret_cast<const char*>(wo), p.b1 = nullptr, p.b_expert = wo_stride * sizeof(T);
    p.c = c.post, p.N = d, p.K = h;
    err = few_blocks == 1   ? go_few<T, 1, false, false>(p, few, max_tiles, out_ok, stream)
          : few_blocks == 2 ? go_few<T, 2, false, false>(p, few, max_tiles, out_ok, stream)
          : tall            ? go_tall<T, false, false>(p, max_tiles, stream)
                            : go<T, S, false, false>(p, max_tiles, out_ok, stream);
    if (err != hipSuccess) return err;
    const bool wide = d % 4 == 0 && (long long)Tn * d >= 1 << 20 && ((reinterpret_cast<uintptr_t>(y) | (uintptr_t)(y_stride * (long long)sizeof(T))) & (4 * sizeof(T) - 1)) == 0;
    const int tokens = std::min(Tn, 1 << 22);  // (a launch has fewer than 2^32 work items in x)
    if (wide) combine_kernel<T, 4><<<dim3(tokens, (d + 1023) / 1024), 256, 0, stream>>>(Tn, d, k, E, ids, weights, c.post, y, y_stride);
    else combine_kernel<T, 1><<<dim3(tokens, (d + 255) / 256), 256, 0, stream>>>(Tn, d, k, E, ids, weights, c.post, y, y_stride);
    return hipGetLastError();
}

}  // namespace
}  // namespace infmoe
