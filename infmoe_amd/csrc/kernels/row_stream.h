// Tiles of C = A * B^T for few rows of A: the weights B pass once from memory through the registers of the matrix
// instructions.  Types, operand layout and names as in row_gemm.h.
//
// With at most a few dozen rows the work is a stream of weights, so the kernel is built around bytes in flight: no LDS and
// no barrier on the way in, a lane loads its 16-byte pieces of 16 weight rows straight into the operand it multiplies.  The
// kWaves waves of a workgroup share its 16 * FN weight rows by K, each streaming its share, and add their sums through LDS
// at the end; the rows of A come through the caches (FM / FN of the weights' bytes at most, less where a tile has fewer than
// 16 rows, because lanes past the last row repeat its address).
#pragma once

#include "row_gemm.h"

namespace infmoe {
namespace rows {

constexpr int kStreamWaves = 8, kStreamThreads = 64 * kStreamWaves;

// acc += over steps [s0, s1) of 128 bytes.  px / pw: this lane's row of each block.  DEPTH steps are under way at a time, each
// in registers of its own that are asked for anew as soon as their products are issued.  between() runs behind the first
// requests: what it waits for, it waits for together with them.
template <typename T, int FM, int FN, bool ALIGNED, typename Between>
__device__ __forceinline__ void stream_steps(v4f (&acc)[FM][FN], const char* const (&px)[FM], const char* const (&pw)[FN], int s0, int s1, int end,
                                             Between&& between) {
    constexpr int DEPTH = FM + FN <= 2 ? 4 : FM + FN <= 4 ? 3 : 2;
    const int lane_at = (threadIdx.x & 63) >> 4 << 4, whole = end / kStepBytes;
    v4u w[DEPTH][2][FN], x[DEPTH][2][FM];
    const int n = s1 - s0, turn = n > 0 ? (int)(blockIdx.x / kXcdCount * 2) % n : 0;
    auto ask = [&](int d, int q) {
        const int s = s0 + (q + turn >= n ? q + turn - n : q + turn);
        const int k = s * kStepBytes + lane_at;
        if (s < whole) {
            // (the two halves of a line one after the other; kept in the caches for just that, where a hint that the
            // weights are read once lets the second half go to memory again: 5.1 TB/s, with the hint 4.0)
#pragma unroll
            for (int j = 0; j < FN; ++j)
#pragma unroll
                for (int kk = 0; kk < 2; ++kk) w[d][kk][j] = whole_piece<T, ALIGNED>(pw[j] + k + kk * 64);
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int kk = 0; kk < 2; ++kk) x[d][kk][i] = whole_piece<T, ALIGNED>(px[i] + k + kk * 64);
        } else {
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
#pragma unroll
                for (int j = 0; j < FN; ++j) w[d][kk][j] = piece<T, ALIGNED>(pw[j], k + kk * 64, end);
#pragma unroll
                for (int i = 0; i < FM; ++i) x[d][kk][i] = piece<T, ALIGNED>(px[i], k + kk * 64, end);
            }
        }
    };
#pragma unroll
    for (int d = 0; d < DEPTH; ++d)
        if (d < n) ask(d, d);
    between();
#pragma unroll 1
    for (int q = 0; q < n; q += DEPTH) {
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
            if (q + d < n) {
#pragma unroll
                for (int kk = 0; kk < 2; ++kk)
#pragma unroll
                    for (int i = 0; i < FM; ++i) mma_row<T, FN>(acc[i], w[d][kk], x[d][kk][i]);
            }
            if (q + d + DEPTH < n) ask(d, q + d + DEPTH);
        }
    }
}

// The waves' sums added: afterwards block (i, j) of thread group `lane` is the sum over waves, handed to give(i, j0, sums)
// with the NJ column blocks that belong together (j0, j0 + FN / NJ, ...).  Work is spread over all waves.
template <int FM, int FN, int NJ, typename Give>
__device__ __forceinline__ void join_waves(char* lds, const v4f (&acc)[FM][FN], Give&& give) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    v4f* part = reinterpret_cast<v4f*>(lds);  // [wave][block][lane]
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) part[(wave * FM * FN + i * FN + j) * 64 + lane] = acc[i][j];
    __syncthreads();
    for (int b = wave; b < FM * (FN / NJ); b += kStreamWaves) {
        const int i = b / (FN / NJ), j0 = b % (FN / NJ);
        v4f sum[NJ];
#pragma unroll
        for (int m = 0; m < NJ; ++m) {
            sum[m] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < kStreamWaves; ++w) sum[m] += part[(w * FM * FN + i * FN + j0 + m * (FN / NJ)) * 64 + lane];
        }
        give(i, j0, sum);
    }
}
template <int FM, int FN>
constexpr int stream_lds() { return kStreamWaves * FM * FN * 64 * (int)sizeof(v4f); }

}  // namespace rows
}  // namespace infmoe
