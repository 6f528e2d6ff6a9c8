// Tiles of C = A * B^T for rows that are gathered, grouped by expert, or carry a low-rank adapter each; shared by
// experts_topk.hip and lora.hip.  A: activation rows, B: weight rows, both K elements side by side, of f32, f16 or bf16;
// sums in FP32.
//
// Everything is laid out in bytes, so that the three types share one data path: a K step is 128 bytes of a row (64
// elements of 16 bits, 32 of 32 bits), staged through LDS in pieces of 16 bytes.  A lane of a wave's 16-row operand block
// holds 16 bytes of its row, (lane / 16) pieces into 64 bytes: for 16-bit types exactly the operand of
// v_mfma_f32_16x16x32, for f32 four operands of v_mfma_f32_16x16x4 whose k are permuted alike in A and B, which leaves the
// sum as it is.  The weights are the instruction's first operand, so that a lane's four results are four neighbouring
// columns of one row of C.
#pragma once

#include <hip/hip_runtime.h>

#include <type_traits>

#include "kernels.h"

namespace infmoe {
namespace rows {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef unsigned int v4u __attribute__((ext_vector_type(4)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

constexpr int kStepBytes = 128;

__device__ __forceinline__ v4f mma(v4u w, v4u x, v4f c, __bf16) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, w), __builtin_bit_cast(v8bf, x), c, 0, 0, 0);
}
__device__ __forceinline__ v4f mma(v4u w, v4u x, v4f c, _Float16) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, w), __builtin_bit_cast(v8h, x), c, 0, 0, 0);
}
__device__ __forceinline__ v4f mma(v4u w, v4u x, v4f c, float) {
    const v4f a = __builtin_bit_cast(v4f, w), b = __builtin_bit_cast(v4f, x);
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
    return c;
}

// acc[j] += w[j] x for N weight operands.  (For f32 the four instructions of a piece go over the sums in turn: each depends on
// the one before it with the same sum, and waits for it if nothing lies between.)
template <typename T, int N>
__device__ __forceinline__ void mma_row(v4f (&acc)[N], const v4u (&w)[N], v4u x) {
    if constexpr (sizeof(T) == 4) {
        const v4f b = __builtin_bit_cast(v4f, x);
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int j = 0; j < N; ++j) acc[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(v4f, w[j])[q], b[q], acc[j], 0, 0, 0);
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) acc[j] = mma(w[j], x, acc[j], T{});
    }
}

// 16 bytes of a row from byte k on, zeros from byte `end` on.  ALIGNED: rows start on 16-byte boundaries and `end` is a
// multiple of 16.  Otherwise whole pieces are still one load (global memory takes 16 bytes at any address); the piece across a
// row's end is the row's last 16 bytes, shifted, and only of rows shorter than that put together from elements.
template <typename T, bool ALIGNED>
__device__ __forceinline__ v4u whole_piece(const char* at) {
    if constexpr (ALIGNED) return *reinterpret_cast<const v4u*>(at);
    v4u v;
    __builtin_memcpy(&v, at, 16);
    return v;
}
template <typename T, bool ALIGNED>
__device__ __forceinline__ v4u piece(const char* row, int k, int end) {
    if constexpr (ALIGNED) {
        const v4u v = *reinterpret_cast<const v4u*>(row + min(k, end - 16));
        return k < end ? v : v4u{0, 0, 0, 0};
    } else {
        if (k + 16 <= end) return whole_piece<T, false>(row + k);
        if (k >= end) return v4u{0, 0, 0, 0};
        if (end >= 16) {
            union {
                v4u v;
                unsigned long long half[2];
            } last{whole_piece<T, false>(row + end - 16)};
            const int by = 8 * (k + 16 - end);  // bits; 8 to 120
            const unsigned long long low = last.half[0], high = last.half[1];
            last.half[0] = by >= 64 ? high >> (by - 64) : low >> by | high << (64 - by);
            last.half[1] = by >= 64 ? 0 : high >> by;
            return last.v;
        }
        union {
            T e[16 / sizeof(T)];
            v4u v;
        } u;
        u.v = v4u{0, 0, 0, 0};
        const T* p = reinterpret_cast<const T*>(row + k);
        const int left = (end - k) / (int)sizeof(T);
#pragma unroll
        for (int i = 0; i < (int)(16 / sizeof(T)) - 1; ++i)
            if (i < left) u.e[i] = p[i];
        return u.v;
    }
}

// A workgroup of WM x WN waves; a wave computes FM blocks of 16 rows by FN blocks of 16 columns.
template <int WM_, int WN_, int FM_, int FN_>
struct Shape {
    static constexpr int WM = WM_, WN = WN_, FM = FM_, FN = FN_;
    static constexpr int kThreads = 64 * WM * WN, kRows = 16 * WM * FM, kCols = 16 * WN * FN;
    static constexpr int kPiecesA = kRows * 8 / kThreads, kPiecesB = kCols * 8 / kThreads;
    static constexpr int kStage = (kRows + kCols) * kStepBytes, kLds = 2 * kStage;
    static_assert(kRows * 8 % kThreads == 0 && kCols * 8 % kThreads == 0, "whole pieces per thread");
};

// Where piece `p` (0..7) of row `row` of a stage lies: pieces are exchanged inside a row so that the 16 rows an operand
// read touches at one piece index spread over all banks.
__device__ __forceinline__ int lds_at(int row, int p) { return row * kStepBytes + ((p ^ ((row >> 1) & 7)) << 4); }

// acc += (rows of A) * (rows of B)^T over `end` bytes of K.  pa / pb: this thread's rows (piece threadIdx.x % 8 of rows
// threadIdx.x / 8 + i * kThreads / 8).  take: called with (kk, weights, rows) per 64 bytes of a step, does the products.
template <typename T, typename S, bool ALIGNED, typename Take>
__device__ __forceinline__ void walk(char* lds, const char* const (&pa)[S::kPiecesA], const char* const (&pb)[S::kPiecesB], int end, Take&& take) {
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int my_row = tid >> 3, my_piece = tid & 7;
    const int wm = wave / S::WN, wn = wave % S::WN;
    v4u ra[S::kPiecesA], rb[S::kPiecesB];
    const int steps = (end + kStepBytes - 1) / kStepBytes;
    const int whole = end / kStepBytes;  // steps without a row's end
    auto fetch = [&](int s) {
        const int k = s * kStepBytes + (my_piece << 4);
        if (s < whole) {
#pragma unroll
            for (int i = 0; i < S::kPiecesA; ++i) ra[i] = whole_piece<T, ALIGNED>(pa[i] + k);
#pragma unroll
            for (int i = 0; i < S::kPiecesB; ++i) rb[i] = whole_piece<T, ALIGNED>(pb[i] + k);
            return;
        }
#pragma unroll
        for (int i = 0; i < S::kPiecesA; ++i) ra[i] = piece<T, ALIGNED>(pa[i], k, end);
#pragma unroll
        for (int i = 0; i < S::kPiecesB; ++i) rb[i] = piece<T, ALIGNED>(pb[i], k, end);
    };
    auto store = [&](int s) {
        char* at = lds + (s & 1) * S::kStage;
#pragma unroll
        for (int i = 0; i < S::kPiecesA; ++i) *reinterpret_cast<v4u*>(at + lds_at(my_row + i * (S::kThreads / 8), my_piece)) = ra[i];
#pragma unroll
        for (int i = 0; i < S::kPiecesB; ++i)
            *reinterpret_cast<v4u*>(at + S::kRows * kStepBytes + lds_at(my_row + i * (S::kThreads / 8), my_piece)) = rb[i];
    };
    __syncthreads();  // whoever used this memory before is done with it
    fetch(0);
    store(0);
    if (steps > 1) fetch(1);
    __syncthreads();
    for (int s = 0; s < steps; ++s) {
        const char* at = lds + (s & 1) * S::kStage;
        // (the other half was last read in step s - 1, which a barrier closed)
        if (s + 1 < steps) store(s + 1);
        if (s + 2 < steps) fetch(s + 2);
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            v4u xa[S::FM], wb[S::FN];
#pragma unroll
            for (int j = 0; j < S::FN; ++j)
                wb[j] = *reinterpret_cast<const v4u*>(at + S::kRows * kStepBytes + lds_at((wn * S::FN + j) * 16 + (lane & 15), kk * 4 + (lane >> 4)));
#pragma unroll
            for (int i = 0; i < S::FM; ++i)
                xa[i] = *reinterpret_cast<const v4u*>(at + lds_at((wm * S::FM + i) * 16 + (lane & 15), kk * 4 + (lane >> 4)));
            take(wb, xa);
        }
        __syncthreads();
    }
}

template <typename T, typename S, bool ALIGNED>
__device__ __forceinline__ void multiply(v4f (&acc)[S::FM][S::FN], char* lds, const char* const (&pa)[S::kPiecesA],
                                         const char* const (&pb)[S::kPiecesB], int end) {
    walk<T, S, ALIGNED>(lds, pa, pb, end, [&](const v4u (&wb)[S::FN], const v4u (&xa)[S::FM]) {
#pragma unroll
        for (int i = 0; i < S::FM; ++i) mma_row<T, S::FN>(acc[i], wb, xa[i]);
    });
}

// The same added to the rows with keep[i] only, through a sum of its own: what a row that is not kept, or a weight it must
// not see, holds (infinities, NaN) cannot reach the others' sums.
template <typename T, typename S, bool ALIGNED>
__device__ __forceinline__ void multiply_kept(v4f (&acc)[S::FM][S::FN], char* lds, const char* const (&pa)[S::kPiecesA],
                                              const char* const (&pb)[S::kPiecesB], int end, const bool (&keep)[S::FM]) {
    walk<T, S, ALIGNED>(lds, pa, pb, end, [&](const v4u (&wb)[S::FN], const v4u (&xa)[S::FM]) {
#pragma unroll
        for (int i = 0; i < S::FM; ++i)
#pragma unroll
            for (int j = 0; j < S::FN; ++j) {
                const v4f p = mma(wb[j], xa[i], v4f{0.f, 0.f, 0.f, 0.f}, T{});
#pragma unroll
                for (int q = 0; q < 4; ++q) acc[i][j][q] += keep[i] ? p[q] : 0.f;
            }
    });
}

// Activations of the feed-forward block, on FP32 sums.  A NaN stays one.
template <typename T>
__device__ __forceinline__ float logistic(float x) {
    if constexpr (sizeof(T) == 4) return 1.f / (1.f + expf(-x));
    return __frcp_rn(1.f + __expf(-x));  // (the result is rounded to 16 bits next)
}
template <typename T>
__device__ __forceinline__ float activate(int ffn, float u, float v) {
    if (ffn == FFN_RELU) return u < 0.f ? 0.f : u;
    // gelu(u) = u Phi(u) in its tanh form: 0.5 (1 + tanh z) is the logistic function of 2 z
    if (ffn == FFN_GATED_GELU) return u * logistic<T>(u * (1.5957691216057308f + 0.07135481627260025f * u * u)) * v;
    return u * logistic<T>(u) * v;
}

}  // namespace rows
}  // namespace infmoe
