// Tiles of C = A * B^T for many rows: up to 256 rows by 256 weight rows per workgroup of eight waves, two per SIMD, each
// 16 * FM x 64.  Types and names as in row_gemm.h; rows are of whole 16-byte pieces on 16-byte boundaries.
//
// Bound by the matrix pipes as long as they are fed.  At full height a wave's step of 64 bytes of K (32 elements of 16 bits) is
// 32 instructions of 16 cycles, the operands of which are 12 reads of 1 KB from LDS:
//   * global memory goes to LDS without passing registers, into a ring of four steps (128 KB); a step is waited for three
//     steps after it was requested, so up to 96 KB per compute unit are under way;
//   * operands are read from LDS half a step before their products.  A step is two halves of the wave's rows: during the
//     first half's products the second half's rows are read, during the second's the next step's weights (into the other of
//     two register sets) and first rows.  The step's one barrier stands between the halves: there the next step has
//     arrived, and everybody has read all of this one, whose place in the ring is requested anew;
//   * reads and requests are issued a piece at a time between the products.
// LDS holds rows of 64 bytes; the four pieces of a row are exchanged by (row's place among the 16 of an operand) / 4, which
// spreads the 16 rows of an operand read over all banks.
// Row 4 a + b of weight operand j is weight row 4 F a + 4 j + b of its block of 16 F, so that a lane (a = lane / 16) ends up
// with 4 F neighbouring columns of one row of C and writes them in whole pieces.
#pragma once

#include "row_gemm.h"

namespace infmoe {
namespace rows {

constexpr int kTallThreads = 512, kTallCols = 256, kTallRows = 256, kTallStep = 64;
constexpr int kTallRing = 4, kTallStage = (kTallCols + kTallRows) * kTallStep, kTallLds = kTallRing * kTallStage;

// Where the pieces behind a row's end come from.
static __device__ const v4u kTallZeros = {0, 0, 0, 0};

// 64 pieces of 16 bytes, one per lane's address, to LDS bytes [at, at + 1024) in lane order.  The transfer is in flight
// afterwards: s_waitcnt vmcnt.  (Written out because the compiler would wait for it before any read of LDS.)
__device__ __forceinline__ void to_lds(const char* from, unsigned at) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(at), "v"(from) : "memory");
}

// What each lane of a wave requests per step, and where its operands lie.  F: weight operands that share a matrix (4, or 2
// when half of the tile's weight rows are of a second matrix).
template <int FM, int F>
struct Tall {
    static constexpr int kPiecesA = (FM + 3) / 4, kPieces = kPiecesA + 2;  // requests of a wave per step

    static __device__ __forceinline__ int chunk_a(int i) { return min((int)(threadIdx.x >> 6) + 8 * i, 2 * FM - 1); }
    static __device__ __forceinline__ int chunk_b(int i) { return (threadIdx.x >> 6) * 2 + i; }
    // Tile row of this lane's i-th request of A, tile weight row (0..255, 64 per wave column) of B.
    static __device__ __forceinline__ int row_a(int i) { return chunk_a(i) * 16 + ((threadIdx.x & 63) >> 2); }
    static __device__ __forceinline__ int row_b(int i) { return chunk_b(i) * 16 + ((threadIdx.x & 63) >> 2); }
    // Byte of the 64 that the request is for.
    static __device__ __forceinline__ int byte_a() { return (((threadIdx.x & 3) ^ ((threadIdx.x >> 4) & 3)) << 4); }
    static __device__ __forceinline__ int byte_b(int i) { return ((threadIdx.x & 3) ^ ((row_b(i) / (4 * F)) & 3)) << 4; }
    // Column of C, relative to the wave's first, of this lane's first result; 4 F from there are its.
    static __device__ __forceinline__ int column() { return ((threadIdx.x & 63) >> 4) * 4 * F; }
};

// acc = A * B^T over `end` bytes of K (a multiple of 16).  pa / pb: this lane's addresses for its requests (byte_a / byte_b
// included).  Steps are taken in pairs; what lies behind `end` is read as zeros.
template <typename T, int FM, int F>
__device__ __forceinline__ void tall_multiply(v4f (&acc)[FM][4], char* lds, const char* (&pa)[Tall<FM, F>::kPiecesA], const char* (&pb)[2], int end) {
    using W = Tall<FM, F>;
    static_assert(FM >= 2, "two halves of rows");
    constexpr int H0 = (FM + 1) / 2;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave >> 2, wn = wave & 3;
    const unsigned base = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
    const int m = lane & 15, g = lane >> 4;
    const char* read_b = lds + (wn * 64 + (m >> 2) * 4 * F + (m & 3)) * kTallStep + ((g ^ (m >> 2)) << 4);
    const char* read_a = lds + (kTallCols + wm * 16 * FM + m) * kTallStep + ((g ^ (m >> 2)) << 4);
    const int whole = end / kTallStep, steps = (end + 2 * kTallStep - 1) / (2 * kTallStep) * 2;
    const char* zeros = reinterpret_cast<const char*>(&kTallZeros);
    int requested = 0;
    auto request = [&](int i) {  // i-th request of step `requested`
        const unsigned stage = base + (requested & (kTallRing - 1)) * kTallStage;
        if (i < 2) to_lds(pb[i], stage + (wave * 2 + i) * 1024);
        else if (i < W::kPieces) to_lds(pa[i - 2], stage + kTallCols * kTallStep + min(wave + 8 * (i - 2), 2 * FM - 1) * 1024);
    };
    auto cut = [&](int k) {  // the pieces of the step at byte k that lie behind the rows' end
#pragma unroll
        for (int i = 0; i < 2; ++i) pb[i] = k + W::byte_b(i) < end ? pb[i] : zeros;
#pragma unroll
        for (int i = 0; i < W::kPiecesA; ++i) pa[i] = k + W::byte_a() < end ? pa[i] : zeros;
    };
    // (requests go on behind the last step, into stages that nothing reads: the waits below count on their number)
    auto advance = [&] {
        ++requested;
#pragma unroll
        for (int i = 0; i < 2; ++i) pb[i] += kTallStep;
#pragma unroll
        for (int i = 0; i < W::kPiecesA; ++i) pa[i] += kTallStep;
        if (requested >= whole) cut(requested * kTallStep);
    };
    v4u xa[FM], wb[2][4];
    auto take_b = [&](int set, int s, int j) {
        wb[set][j] = *reinterpret_cast<const v4u*>(read_b + (s & (kTallRing - 1)) * kTallStage + ((j / F) * 16 * F + 4 * (j % F)) * kTallStep);
    };
    auto take_a = [&](int s, int i) { xa[i] = *reinterpret_cast<const v4u*>(read_a + (s & (kTallRing - 1)) * kTallStage + i * 16 * kTallStep); };
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
    if (whole == 0) cut(0);
#pragma unroll
    for (int q = 0; q < kTallRing; ++q) {
#pragma unroll
        for (int i = 0; i < W::kPieces; ++i) request(i);
        advance();
    }
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" : : "n"(3 * W::kPieces) : "memory");
#pragma unroll
    for (int j = 0; j < 4; ++j) take_b(0, 0, j);
#pragma unroll
    for (int i = 0; i < H0; ++i) take_a(0, i);
    auto step = [&](auto set_, int s) {
        constexpr int set = decltype(set_)::value;
#pragma unroll
        for (int i = 0; i < H0; ++i) {
            if (H0 + i < FM) take_a(s, H0 + i);
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] = mma(wb[set][j], xa[i], acc[i][j], T{});
            __builtin_amdgcn_sched_barrier(0);
        }
        // step s + 1 has arrived (of the requests only those of s + 2 and s + 3 are younger), and everybody has read all of
        // step s: its place takes step s + 4
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"(2 * W::kPieces) : "memory");
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            request(i);
            take_b(set ^ 1, s + 1, i);
            if (i < H0) take_a(s + 1, i);
            if (H0 + i < FM)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[H0 + i][j] = mma(wb[set][j], xa[H0 + i], acc[H0 + i][j], T{});
            __builtin_amdgcn_sched_barrier(0);
        }
        advance();
    };
#pragma unroll 1
    for (int s = 0; s < steps; s += 2) {
        step(std::integral_constant<int, 0>{}, s);
        step(std::integral_constant<int, 1>{}, s + 1);
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
