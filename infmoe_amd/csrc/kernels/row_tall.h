// Tiles of C = A * B^T for many rows: up to 256 rows by 256 weight rows per workgroup of eight waves, two per SIMD, each
// 16 * FM x 64.  Types and names as in row_gemm.h; rows are of whole 16-byte pieces on 16-byte boundaries.
//
// Bound by the matrix pipes as long as they are fed.  At full height a wave's step of 64 bytes of K (32 elements of 16 bits) is
// 32 instructions of 16 cycles, the operands of which are 12 reads of 1 KB from LDS.
//   * Global memory goes to LDS without passing registers, two steps (128 bytes of a row, a cache line) at a time: asked for
//     in halves, every line costs the L2 two requests, and the requests that tiles of this size make at full rate are all it
//     answers.  LDS is a ring of five units of 32 KB, in turn 256 weight rows and up to 256 rows of a pair of steps: while a
//     pair is multiplied, the next pair and the weights of the one after it are there or under way.
//   * Operands are read from LDS half a step before their products.  A step is two halves of the wave's rows: during the
//     first half's products the second half's rows are read, during the second's the next step's weights (into the other of
//     two register sets) and first rows.  A pair's one barrier stands before its last half: there the next pair has
//     arrived, and everybody has read all of this one, whose two units are requested anew.
//   * Reads and requests are issued a piece at a time between the products.
// The LDS serves a 16-byte read of 64 lanes in groups of 16: lanes 0-3, 12-15, 20-23 and 24-27, then 4-11, 16-19 and 28-31,
// and the upper half alike.  The eight pieces of a row are exchanged by (row's place among the 16 of an operand) / 2, which
// gives the 16 lanes of every group 16 different places of the 256 bytes of a bank row: no conflicts.
// Row 4 a + b of weight operand j is weight row 4 F a + 4 j + b of its block of 16 F, so that a lane (a = lane / 16) ends up
// with 4 F neighbouring columns of one row of C and writes them in whole pieces.
#pragma once

#include "row_gemm.h"

namespace infmoe {
namespace rows {

constexpr int kTallThreads = 512, kTallCols = 256, kTallRows = 256, kTallPair = 128;  // bytes of K per pair of steps
constexpr int kTallUnit = 256 * kTallPair, kTallLds = 5 * kTallUnit;

// Where the pieces behind a row's end come from.
static __device__ const v4u kTallZeros = {0, 0, 0, 0};

// 64 pieces of 16 bytes, one per lane's address, to LDS bytes [at, at + 1024) in lane order.  The transfer is in flight
// afterwards: s_waitcnt vmcnt.  (Written out because the compiler would wait for it before any read of LDS.  M0, which holds the
// LDS address, is on the clobber list so that no use of it by the compiler spans the statement; that it is a register which
// the compiler does not allocate draws a warning.)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void to_lds(const char* from, unsigned at) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(at), "v"(from) : "memory", "m0");
}
#pragma clang diagnostic pop

// What each lane of a wave requests per pair of steps (8 rows of 128 bytes a request), and where its operands lie.  F: weight
// operands that share a matrix (4, or 2 when half of the tile's weight rows are of a second matrix).
template <int FM, int F>
struct Tall {
    static constexpr int kPiecesA = (FM + 1) / 2, kPiecesB = 4;  // requests of a wave per pair

    static __device__ __forceinline__ int chunk_a(int i) { return min((int)(threadIdx.x >> 6) + 8 * i, 4 * FM - 1); }
    static __device__ __forceinline__ int chunk_b(int i) { return (threadIdx.x >> 6) * 4 + i; }
    // Tile row of this lane's i-th request of A, tile weight row (0..255, 64 per wave column) of B.
    static __device__ __forceinline__ int row_a(int i) { return chunk_a(i) * 8 + ((threadIdx.x & 63) >> 3); }
    static __device__ __forceinline__ int row_b(int i) { return chunk_b(i) * 8 + ((threadIdx.x & 63) >> 3); }
    // Byte of the 128 that the request is for.
    static __device__ __forceinline__ int byte_a(int i) { return ((threadIdx.x & 7) ^ ((row_a(i) >> 1) & 7)) << 4; }
    static __device__ __forceinline__ int byte_b(int i) {
        const int r = row_b(i);
        return ((threadIdx.x & 7) ^ (((r / (4 * F)) & 3) * 2 + ((r >> 1) & 1))) << 4;
    }
    // Column of C, relative to the wave's first, of this lane's first result; 4 F from there are its.
    static __device__ __forceinline__ int column() { return ((threadIdx.x & 63) >> 4) * 4 * F; }
};

// acc = A * B^T over `end` bytes of K (a multiple of 16).  pa / pb: this lane's addresses for its requests (byte_a / byte_b
// included).  What lies behind `end` is read as zeros.
template <typename T, int FM, int F>
__device__ __forceinline__ void tall_multiply(v4f (&acc)[FM][4], char* lds, const char* (&pa)[Tall<FM, F>::kPiecesA], const char* (&pb)[4], int end) {
    using W = Tall<FM, F>;
    static_assert(FM >= 2, "two halves of rows");
    constexpr int H0 = (FM + 1) / 2;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave >> 2, wn = wave & 3;
    const unsigned base = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
    const int m = lane & 15, g = lane >> 4;
    // place of a piece (kk * 4 + g) of the lane's row: kk only exchanges the halves of the row
    const int swap = m >> 1, at_b = (wn * 64 + (m >> 2) * 4 * F + (m & 3)) * kTallPair, at_a = (wm * 16 * FM + m) * kTallPair;
    const int place[2] = {(g ^ swap) << 4, ((4 + g) ^ swap) << 4};
    const int whole = end / kTallPair, pairs = (end + kTallPair - 1) / kTallPair;
    const char* zeros = reinterpret_cast<const char*>(&kTallZeros);
    unsigned ask = base;  // unit of the next request
    int asked_a = 0, asked_b = 0;
    auto next_unit = [&](unsigned u, int by) {
        u += by * kTallUnit;
        return u >= base + kTallLds ? u - kTallLds : u;
    };
    auto request_a = [&](unsigned unit, int i) { to_lds(pa[i], unit + min(wave + 8 * i, 4 * FM - 1) * 1024); };
    auto request_b = [&](unsigned unit, int i) { to_lds(pb[i], unit + (wave * 4 + i) * 1024); };
    // (requests go on behind the last pair, into units that nothing reads: the waits below count on their number)
    auto cut_a = [&](int k) {
#pragma unroll
        for (int i = 0; i < W::kPiecesA; ++i) pa[i] = k + W::byte_a(i) < end ? pa[i] : zeros;
    };
    auto cut_b = [&](int k) {
#pragma unroll
        for (int i = 0; i < W::kPiecesB; ++i) pb[i] = k + W::byte_b(i) < end ? pb[i] : zeros;
    };
    auto advance_a = [&] {
        ++asked_a;
#pragma unroll
        for (int i = 0; i < W::kPiecesA; ++i) pa[i] += kTallPair;
        if (asked_a >= whole) cut_a(asked_a * kTallPair);
    };
    auto advance_b = [&] {
        ++asked_b;
#pragma unroll
        for (int i = 0; i < W::kPiecesB; ++i) pb[i] += kTallPair;
        if (asked_b >= whole) cut_b(asked_b * kTallPair);
    };
    v4u xa[FM], wb[2][4];
    const char *unit_b = lds, *unit_a = lds + kTallUnit;  // of the pair at work
    auto take_b = [&](const char* unit, int kk, int j) {
        wb[kk][j] = *reinterpret_cast<const v4u*>(unit + at_b + place[kk] + ((j / F) * 16 * F + 4 * (j % F)) * kTallPair);
    };
    auto take_a = [&](const char* unit, int kk, int i) { xa[i] = *reinterpret_cast<const v4u*>(unit + at_a + place[kk] + i * 16 * kTallPair); };
    auto products = [&](int kk, int i) { mma_row<T, 4>(acc[i], wb[kk], xa[i]); };
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
    if (whole == 0) cut_a(0), cut_b(0);
#pragma unroll
    for (int q = 0; q < 5; ++q) {
        if (q % 2 == 0) {
#pragma unroll
            for (int i = 0; i < W::kPiecesB; ++i) request_b(base + q * kTallUnit, i);
            advance_b();
        } else {
#pragma unroll
            for (int i = 0; i < W::kPiecesA; ++i) request_a(base + q * kTallUnit, i);
            advance_a();
        }
    }
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" : : "n"(2 * W::kPiecesB + W::kPiecesA) : "memory");
#pragma unroll
    for (int j = 0; j < 4; ++j) take_b(unit_b, 0, j);
#pragma unroll
    for (int i = 0; i < H0; ++i) take_a(unit_a, 0, i);
#pragma unroll 1
    for (int p = 0; p < pairs; ++p) {
        // first step
#pragma unroll
        for (int i = 0; i < H0; ++i) {
            if (H0 + i < FM) take_a(unit_a, 0, H0 + i);
            products(0, i);
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            take_b(unit_b, 1, i);
            if (i < H0) take_a(unit_a, 1, i);
            if (H0 + i < FM) products(0, H0 + i);
            __builtin_amdgcn_sched_barrier(0);
        }
        // second step
#pragma unroll
        for (int i = 0; i < H0; ++i) {
            if (H0 + i < FM) take_a(unit_a, 1, H0 + i);
            products(1, i);
            __builtin_amdgcn_sched_barrier(0);
        }
        // the next pair has arrived (only the weights of the one after it are younger requests), and everybody has read all
        // of this one: its units take the rows of the pair after the next and the weights of the one behind that
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"(W::kPiecesB) : "memory");
        unit_b = unit_b + 2 * kTallUnit >= lds + kTallLds ? unit_b + 2 * kTallUnit - kTallLds : unit_b + 2 * kTallUnit;
        unit_a = unit_a + 2 * kTallUnit >= lds + kTallLds ? unit_a + 2 * kTallUnit - kTallLds : unit_a + 2 * kTallUnit;
        const unsigned then = next_unit(ask, 1);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            take_b(unit_b, 0, i);
            if (i < H0) take_a(unit_a, 0, i);
            if (i < W::kPiecesA) request_a(ask, i);
            if (H0 + i < FM) products(1, H0 + i);
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int i = 0; i < W::kPiecesB; ++i) request_b(then, i);
        ask = next_unit(ask, 2);
        advance_a();
        advance_b();
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" : : : "memory");  // nothing is under way into LDS any more
}

// COUNT neighbouring columns of one row of C, from column n on, of which those below N exist.
template <typename Out, int COUNT, typename Value>
__device__ __forceinline__ void write_columns(Out* row, int n, int N, bool whole_pieces, Value&& value) {
    constexpr int kEach = 16 / sizeof(Out);
    if (whole_pieces && n + COUNT <= N) {
#pragma unroll
        for (int c = 0; c < COUNT; c += kEach) {
            union {
                Out e[kEach];
                v4u v;
            } u;
#pragma unroll
            for (int q = 0; q < kEach; ++q) u.e[q] = (Out)value(c + q);
            *reinterpret_cast<v4u*>(row + n + c) = u.v;
        }
    } else {
#pragma unroll
        for (int c = 0; c < COUNT; ++c)
            if (n + c < N) row[n + c] = (Out)value(c);
    }
}

}  // namespace rows
}  // namespace infmoe
