// A projection shared by all rows of a batch with a low-rank adapter per row, for gfx950:
//   y_t = W x_t + scale_a * B_a (A_a x_t),  a = adapter[t].
//
// The first launch forms u_t = scale_a * A_a x_t ([T][r], in the operands' type, as the second product takes it), the next
// computes W x_t and adds u_t B_a^T before its results leave the registers, so that y is written once and never read:
//   up to 16 rows, odd strides      W streamed through the registers (project_few_kernel)
//   many rows                       tall tiles, which go over the adapters that occur among their rows (project_tall_kernel)
//   between the two                 tall tiles with K cut over workgroups, joined by a third launch (project_split_kernel)
//   many rows of odd strides        tiles of 64 x 128 (project_kernel)
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
static_assert(forms::kTallCutCols == kTallCols && forms::kTallCutBytes == kTallPair, "the tiles that forms.h counts");

struct Args {
    const char *x, *w, *a, *b;
    char *u, *y;
    const int* adapter;
    const float* scale;
    long long x_stride, y_stride;  // bytes
    int T, d, n, r, L, u_stride;   // u_stride: bytes, a multiple of 16
};

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
    return v;
}

template <typename T>
__device__ __forceinline__ float dot_piece(v4u a, v4u b, float sum) {
    union {
        v4u v;
        T e[16 / sizeof(T)];
    } p{a}, q{b};
#pragma unroll
    for (int i = 0; i < (int)(16 / sizeof(T)); ++i) sum = fmaf((float)p.e[i], (float)q.e[i], sum);
    return sum;
}

// u of few rows: a wave per row and RJ ranks (one where rows are so few that the waves are wanted, else four, which share the
// row of x).
template <typename T, int RJ, bool ALIGNED>
__global__ __launch_bounds__(256) void shrink_few_kernel(Args p) {
    const int t = blockIdx.x, lane = threadIdx.x & 63, j0 = (blockIdx.y * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * RJ;
    const int a = p.adapter[t], padded = p.u_stride / (int)sizeof(T);
    if (a < 0 || a >= p.L || j0 >= padded) return;  // (a row without an adapter: its u is never used)
    const int end = p.d * (int)sizeof(T);
    const char *x = p.x + t * p.x_stride, *m[RJ];
#pragma unroll
    for (int q = 0; q < RJ; ++q) m[q] = p.a + ((long long)a * p.r + min(j0 + q, p.r - 1)) * end;
    float sum[RJ];
#pragma unroll
    for (int q = 0; q < RJ; ++q) sum[q] = 0.f;
    constexpr int kLoads = RJ == 1 ? 4 : 2;  // pieces of a row in flight
    int k = lane * 16;
    for (; k + (kLoads - 1) * 1024 + 16 <= end; k += kLoads * 1024) {
        v4u v[kLoads], w[RJ][kLoads];
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            v[i] = whole_piece<T, ALIGNED>(x + k + i * 1024);
#pragma unroll
            for (int q = 0; q < RJ; ++q) w[q][i] = whole_piece<T, ALIGNED>(m[q] + k + i * 1024);
        }
#pragma unroll
        for (int i = 0; i < kLoads; ++i)
#pragma unroll
            for (int q = 0; q < RJ; ++q) sum[q] = dot_piece<T>(v[i], w[q][i], sum[q]);
    }
    for (; k < end; k += 1024) {
        const v4u v = piece<T, ALIGNED>(x, k, end);
#pragma unroll
        for (int q = 0; q < RJ; ++q) sum[q] = dot_piece<T>(v, piece<T, ALIGNED>(m[q], k, end), sum[q]);
    }
    const float s = p.scale != nullptr ? p.scale[a] : 1.f;
    T* u = reinterpret_cast<T*>(p.u + (size_t)t * p.u_stride);
#pragma unroll
    for (int q = 0; q < RJ; ++q) {
        const float total = wave_sum(sum[q]) * s;
        if (lane == 0 && j0 + q < padded) u[j0 + q] = (T)(j0 + q < p.r ? total : 0.f);
    }
}

// u of many rows: 16 * FM rows of a workgroup against the adapters that occur among them, 32 ranks at a time, on the matrix
// cores (row_stream.h: A_a takes the place of the weights).
template <typename T, int FM, bool ALIGNED>
__global__ __launch_bounds__(kStreamThreads) void shrink_kernel(Args p) {
    extern __shared__ __align__(16) char lds[];
    constexpr int FN = 2;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row0 = blockIdx.x * 16 * FM, count = min(16 * FM, p.T - row0), j0 = blockIdx.y * 32;
    const int end = p.d * (int)sizeof(T), steps = (end + kStepBytes - 1) / kStepBytes;
    const int a_lane = lane < count ? p.adapter[row0 + lane] : -1;  // (16 * FM <= 64)
    const char* px[FM];
    int mine[FM];
#pragma unroll
    for (int i = 0; i < FM; ++i) {
        px[i] = p.x + (row0 + min(i * 16 + (lane & 15), count - 1)) * p.x_stride;
        mine[i] = __shfl(a_lane, i * 16 + (lane & 15));
    }
    unsigned long long left = __ballot(a_lane >= 0 && a_lane < p.L);
    bool again = false;
    while (left != 0) {  // (the same in all waves)
        const int a = __builtin_amdgcn_readlane(a_lane, __ffsll((long long)left) - 1);
        left &= ~__ballot(a_lane == a);
        const char* pw[FN];
#pragma unroll
        for (int j = 0; j < FN; ++j) pw[j] = p.a + ((long long)a * p.r + min(j0 + j * 16 + (lane & 15), p.r - 1)) * end;
        v4f acc[FM][FN];
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
        stream_steps<T, FM, FN, ALIGNED>(acc, px, pw, steps * wave / kStreamWaves, steps * (wave + 1) / kStreamWaves, end, [] {});
        if (again) __syncthreads();
        again = true;
        const float s = p.scale != nullptr ? p.scale[a] : 1.f;
        join_waves<FM, FN, 1>(lds, acc, [&](int i, int j, const v4f(&sum)[1]) {
            if (mine[i] != a) return;
            T* u = reinterpret_cast<T*>(p.u + (size_t)(row0 + i * 16 + (lane & 15)) * p.u_stride);
            const int n = j0 + j * 16 + (lane >> 4) * 4;
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (n + q < p.u_stride / (int)sizeof(T)) u[n + q] = (T)(n + q < p.r ? s * sum[0][q] : 0.f);
        });
    }
}

template <typename T, typename S>
__global__ __launch_bounds__(S::kThreads) void project_kernel(Args p) {
    extern __shared__ __align__(16) char lds[];
    __shared__ int s_adapter[S::kRows], s_list[S::kRows], s_n;
    const int cols = (p.n + S::kCols - 1) / S::kCols;
    const int row0 = blockIdx.x / cols * S::kRows, n0 = blockIdx.x % cols * S::kCols;
    const int count = min(S::kRows, p.T - row0);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = wave / S::WN, wn = wave % S::WN;
    const char* pa[S::kPiecesA];
    const char* pb[S::kPiecesB];
#pragma unroll
    for (int i = 0; i < S::kPiecesA; ++i) pa[i] = p.x + (row0 + min((tid >> 3) + i * (S::kThreads / 8), count - 1)) * p.x_stride;
    const int row_bytes = p.d * (int)sizeof(T);
#pragma unroll
    for (int i = 0; i < S::kPiecesB; ++i) pb[i] = p.w + (long long)min(n0 + (tid >> 3) + i * (S::kThreads / 8), p.n - 1) * row_bytes;

    // the adapters that occur in the tile, in the order of their first rows
    for (int i = tid; i < S::kRows; i += S::kThreads) {
        const int a = i < count ? p.adapter[row0 + i] : -1;
        s_adapter[i] = a >= 0 && a < p.L ? a : -1;
    }
    if (tid == 0) s_n = 0;
    __syncthreads();
    if (tid < 64) {
        int n = 0;
        for (int i0 = 0; i0 < S::kRows; i0 += 64) {
            const int i = i0 + lane, a = s_adapter[i];
            bool first = a >= 0 && (i == 0 || s_adapter[i - 1] != a);  // (rows of a request lie side by side: seldom more work)
            for (int j = 0; first && j < i - 1; ++j) first = s_adapter[j] != a;
            const unsigned long long m = __ballot(first);
            if (first) s_list[n + __popcll(m & (lane == 0 ? 0ull : ~0ull >> (64 - lane)))] = a;
            n += __popcll(m);
        }
        if (lane == 0) s_n = n;
    }
    v4f acc[S::FM][S::FN];
#pragma unroll
    for (int i = 0; i < S::FM; ++i)
#pragma unroll
        for (int j = 0; j < S::FN; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
    multiply<T, S, false>(acc, lds, pa, pb, row_bytes);  // (starts with a barrier)

    int mine[S::FM];
#pragma unroll
    for (int i = 0; i < S::FM; ++i) mine[i] = s_adapter[(wm * S::FM + i) * 16 + (lane & 15)];
#pragma unroll
    for (int i = 0; i < S::kPiecesA; ++i) pa[i] = p.u + (size_t)(row0 + min((tid >> 3) + i * (S::kThreads / 8), count - 1)) * p.u_stride;
    const int r_bytes = p.r * (int)sizeof(T);
    for (int q = 0; q < s_n; ++q) {
        const int a = s_list[q];
        bool keep[S::FM];
#pragma unroll
        for (int i = 0; i < S::FM; ++i) keep[i] = mine[i] == a;
#pragma unroll
        for (int i = 0; i < S::kPiecesB; ++i)
            pb[i] = p.b + ((long long)a * p.n + min(n0 + (tid >> 3) + i * (S::kThreads / 8), p.n - 1)) * r_bytes;
        multiply_kept<T, S, false>(acc, lds, pa, pb, r_bytes, keep);
    }
#pragma unroll
    for (int i = 0; i < S::FM; ++i) {
        const int r = (wm * S::FM + i) * 16 + (lane & 15);
        if (r >= count) continue;
        T* y = reinterpret_cast<T*>(p.y + (row0 + r) * p.y_stride);
#pragma unroll
        for (int j = 0; j < S::FN; ++j) {
            const int n = n0 + (wn * S::FN + j) * 16 + (lane >> 4) * 4;
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (n + q < p.n) y[n + q] = (T)acc[i][j][q];
        }
    }
}

// Many rows: tiles of 32 * FM x 256 (row_tall.h).  The adapters' part needs no LDS and no barrier: every wave goes over the
// adapters among its own 16 * FM rows and takes u and B_a from the caches straight into operands.
constexpr int kTileGroup = 4;  // row tiles that share a stretch of weight columns (below)

template <typename T, int FM>
__global__ __launch_bounds__(kTallThreads) void project_tall_kernel(Args p) {
    extern __shared__ __align__(16) char lds[];
    using W = Tall<FM, 4>;
    constexpr int kRows = 32 * FM;
    const int cols = (p.n + kTallCols - 1) / kTallCols, tiles = (p.T + kRows - 1) / kRows;
    // Workgroups are dealt to the dies in turn; each die takes a contiguous stretch of tiles, walked kTileGroup row tiles by
    // one column tile at a time: those at work in a die at one time share a few row and column tiles in its L2.
    const int share = (tiles * cols + kXcdCount - 1) / kXcdCount, id = (int)(blockIdx.x % kXcdCount) * share + (int)(blockIdx.x / kXcdCount);
    if ((int)(blockIdx.x / kXcdCount) >= share || id >= tiles * cols) return;
    const int band = id / (kTileGroup * cols), in_band = id % (kTileGroup * cols), high = min(kTileGroup, tiles - band * kTileGroup);
    const int row0 = (band * kTileGroup + in_band % high) * kRows, n0 = in_band / high * kTallCols;
    const int count = min(kRows, p.T - row0);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave >> 2, wn = wave & 3;
    const int end = p.d * (int)sizeof(T);
    const char *pa[W::kPiecesA], *pb[4];
#pragma unroll
    for (int i = 0; i < W::kPiecesA; ++i) pa[i] = p.x + (row0 + min(W::row_a(i), count - 1)) * p.x_stride + W::byte_a(i);
#pragma unroll
    for (int i = 0; i < 4; ++i) pb[i] = p.w + (long long)min(n0 + W::row_b(i), p.n - 1) * end + W::byte_b(i);
    v4f acc[FM][4];
    tall_multiply<T, FM, 4>(acc, lds, pa, pb, end);

    const int m = lane & 15, r_end = p.r * (int)sizeof(T);
    const bool whole_b = ((reinterpret_cast<uintptr_t>(p.b) | (uintptr_t)r_end) & 15) == 0;
    int mine[FM];
#pragma unroll
    for (int i = 0; i < FM; ++i) {
        const int r = (wm * FM + i) * 16 + m;
        mine[i] = r < count ? p.adapter[row0 + r] : -1;
        if (mine[i] >= p.L) mine[i] = -1;
    }
    for (;;) {
        int a = -1;  // the first adapter that is left (rows that have been served get -1)
#pragma unroll
        for (int i = FM - 1; i >= 0; --i) {
            const unsigned long long left = __ballot(mine[i] >= 0);
            if (left != 0) a = __builtin_amdgcn_readlane(mine[i], __ffsll((long long)left) - 1);
        }
        if (a < 0) break;
        const char* pw[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int n = n0 + wn * 64 + (m >> 2) * 16 + 4 * j + (m & 3);
            pw[j] = p.b + ((long long)a * p.n + min(n, p.n - 1)) * r_end;
        }
        for (int k = (lane >> 4) * 16; k - (lane >> 4) * 16 < r_end; k += 64) {
            v4u wb[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) wb[j] = k >= r_end ? v4u{0, 0, 0, 0} : whole_b ? piece<T, true>(pw[j], k, r_end) : piece<T, false>(pw[j], k, r_end);
#pragma unroll
            for (int i = 0; i < FM; ++i) {
                if (__ballot(mine[i] == a) == 0) continue;
                const size_t row = row0 + min((wm * FM + i) * 16 + m, count - 1);
                const v4u u = piece<T, true>(p.u + row * p.u_stride, k, p.u_stride);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    // a sum of its own: what another adapter's rows and weights hold (infinities, NaN) stays out of acc
                    const v4f sum = mma(wb[j], u, v4f{0.f, 0.f, 0.f, 0.f}, T{});
#pragma unroll
                    for (int q = 0; q < 4; ++q) acc[i][j][q] += mine[i] == a ? sum[q] : 0.f;
                }
                // one block's loads at a time.  (Beside the sums of tall tiles even these do not fit: 8 registers are spilled at 5
                // blocks, 45 at 6, 82 at 7 and 115 at 8, all of it here and none in the loop over K.)
                __builtin_amdgcn_sched_barrier(0);
            }
        }
#pragma unroll
        for (int i = 0; i < FM; ++i) mine[i] = mine[i] == a ? -1 : mine[i];
    }
    const bool whole = ((reinterpret_cast<uintptr_t>(p.y) | (uintptr_t)p.y_stride) & 15) == 0;
#pragma unroll
    for (int i = 0; i < FM; ++i) {
        const int r = (wm * FM + i) * 16 + m;
        if (r < count)
            write_columns<T, 16>(reinterpret_cast<T*>(p.y + (row0 + r) * p.y_stride), n0 + wn * 64 + W::column(), p.n, whole,
                                 [&](int c) { return acc[i][c >> 2][c & 3]; });
    }
}

template <typename T, int FM>
hipError_t go_tall(const Args& p, hipStream_t stream) {
    const long long all = (long long)((p.T + 32 * FM - 1) / (32 * FM)) * ((p.n + kTallCols - 1) / kTallCols);
    if (const hipError_t err = allow_lds_once<project_tall_kernel<T, FM>>(kTallLds); err != hipSuccess) return err;
    project_tall_kernel<T, FM><<<(int)((all + kXcdCount - 1) / kXcdCount * kXcdCount), kTallThreads, kTallLds, stream>>>(p);
    return hipGetLastError();
}

// Rows too few for tall tiles to fill the compute units: the tiles' K is cut over `splits` workgroups, each of which leaves FP32
// sums, and a second launch adds them and the adapters' part.  (64 rows by 10240 x 4096: 40 tiles, cut in five.  Streamed by
// project_few_kernel the rows pass every compute unit's cache once per 64 weight rows, half of all bytes: 39 us.)
template <typename T, int FM>
__global__ __launch_bounds__(kTallThreads) void project_split_kernel(Args p, float* __restrict__ sums, int splits, long long sums_stride) {
    extern __shared__ __align__(16) char lds[];
    using W = Tall<FM, 4>;
    constexpr int kRows = 32 * FM;
    const int cols = (p.n + kTallCols - 1) / kTallCols;
    const int split = blockIdx.x % splits, tile = blockIdx.x / splits;
    const int row0 = tile / cols * kRows, n0 = tile % cols * kTallCols, count = min(kRows, p.T - row0);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave >> 2, wn = wave & 3;
    const int end = p.d * (int)sizeof(T), pairs = (end + kTallPair - 1) / kTallPair;
    const int k0 = (int)((long long)pairs * split / splits) * kTallPair, k1 = min((int)((long long)pairs * (split + 1) / splits) * kTallPair, end);
    const char *pa[W::kPiecesA], *pb[4];
#pragma unroll
    for (int i = 0; i < W::kPiecesA; ++i) pa[i] = p.x + (row0 + min(W::row_a(i), count - 1)) * p.x_stride + k0 + W::byte_a(i);
#pragma unroll
    for (int i = 0; i < 4; ++i) pb[i] = p.w + (long long)min(n0 + W::row_b(i), p.n - 1) * end + k0 + W::byte_b(i);
    v4f acc[FM][4];
    tall_multiply<T, FM, 4>(acc, lds, pa, pb, k1 - k0);
#pragma unroll
    for (int i = 0; i < FM; ++i) {
        const int r = (wm * FM + i) * 16 + (lane & 15);
        if (r < count)
            write_columns<float, 16>(sums + ((long long)split * p.T + row0 + r) * sums_stride, n0 + wn * 64 + W::column(), p.n, true,
                                     [&](int c) { return acc[i][c >> 2][c & 3]; });
    }
}

// (A thread per column: the lanes of a wave read rows of B_a that lie side by side.)
template <typename T>
__global__ __launch_bounds__(256) void project_join_kernel(Args p, const float* __restrict__ sums, int splits, long long sums_stride) {
    const int t = blockIdx.y, n = blockIdx.x * 256 + threadIdx.x;
    if (n >= p.n) return;
    const int a = p.adapter[t], r_end = p.r * (int)sizeof(T);
    const float* from = sums + t * sums_stride + n;
    const long long step = p.T * sums_stride;
    float sum = 0.f, part = 0.f;
#pragma unroll 4
    for (int s = 0; s < splits; ++s) sum += from[s * step];
    if (a >= 0 && a < p.L) {
        const char *u = p.u + (size_t)t * p.u_stride, *b = p.b + ((long long)a * p.n + n) * r_end;
#pragma unroll 2
        for (int k = 0; k < r_end; k += 16)  // (u is padded to whole pieces)
            part = dot_piece<T>(*reinterpret_cast<const v4u*>(u + k), piece<T, false>(b, k, r_end), part);
    }
    reinterpret_cast<T*>(p.y + t * p.y_stride)[n] = (T)(sum + part);
}

inline size_t sums_bytes(int T, int d, int n, int size) {
    const int splits = forms::project_form(T, d, n, size, (size_t)d * size % 16 == 0).splits;
    return splits > 1 ? (size_t)splits * T * ((n + 3) / 4 * 4) * 4 : 0;
}

template <typename T, int FM>
hipError_t go_split(const Args& p, float* sums, int splits, hipStream_t stream) {
    const long long tiles = (long long)((p.T + 32 * FM - 1) / (32 * FM)) * ((p.n + kTallCols - 1) / kTallCols), stride = (p.n + 3) / 4 * 4;
    if (const hipError_t err = allow_lds_once<project_split_kernel<T, FM>>(kTallLds); err != hipSuccess) return err;
    project_split_kernel<T, FM><<<(int)(tiles * splits), kTallThreads, kTallLds, stream>>>(p, sums, splits, stride);
    const dim3 grid((p.n + 255) / 256, p.T);
    project_join_kernel<T><<<grid, 256, 0, stream>>>(p, sums, splits, stride);
    return hipGetLastError();
}

template <typename T, int FM>
hipError_t go_cut(const Args& p, float* sums, int splits, hipStream_t stream) {
    if (splits > 1) return go_split<T, FM>(p, sums, splits, stream);
    return go_tall<T, FM>(p, stream);
}

// Few rows: W streamed once through the registers, 16 * FN of its rows per workgroup; the adapters' part of an output is added
// by the lane that holds the joined sum.
template <typename T, int FM, int FN, bool ALIGNED>
__global__ __launch_bounds__(kStreamThreads) void project_few_kernel(Args p) {
    extern __shared__ __align__(16) char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n0 = blockIdx.x * 16 * FN, row0 = blockIdx.y * 16 * FM, count = min(16 * FM, p.T - row0);
    const int end = p.d * (int)sizeof(T), steps = (end + kStepBytes - 1) / kStepBytes, r_end = p.r * (int)sizeof(T);
    const char *px[FM], *pw[FN];
#pragma unroll
    for (int i = 0; i < FM; ++i) px[i] = p.x + (row0 + min(i * 16 + (lane & 15), count - 1)) * p.x_stride;
#pragma unroll
    for (int j = 0; j < FN; ++j) pw[j] = p.w + (long long)min(n0 + j * 16 + (lane & 15), p.n - 1) * end;
    v4f acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
    // the adapters' part of the outputs that this lane will hold in the end (join_waves: blocks wave, wave + kStreamWaves, ...)
    constexpr int kMine = (FM * FN + kStreamWaves - 1) / kStreamWaves;
    v4f part[kMine];
    auto adapters = [&] {
#pragma unroll
        for (int c = 0; c < kMine; ++c) {
            part[c] = v4f{0.f, 0.f, 0.f, 0.f};
            const int block = wave + c * kStreamWaves;
            const int t = row0 + block / FN * 16 + (lane & 15), n = n0 + block % FN * 16 + (lane >> 4) * 4;
            if (block >= FM * FN || t >= p.T) continue;
            const int a = p.adapter[t];
            if (a < 0 || a >= p.L) continue;
            const char *u = p.u + (size_t)t * p.u_stride, *b = p.b + ((long long)a * p.n + n) * r_end;
            for (int k = 0; k < r_end; k += 16) {
                const v4u uk = *reinterpret_cast<const v4u*>(u + k);  // (u is padded to whole pieces)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    if (n + q < p.n) part[c][q] = dot_piece<T>(uk, piece<T, false>(b + q * r_end, k, r_end), part[c][q]);
            }
        }
    };
    stream_steps<T, FM, FN, ALIGNED>(acc, px, pw, steps * wave / kStreamWaves, steps * (wave + 1) / kStreamWaves, end, adapters);
    const bool whole = ((reinterpret_cast<uintptr_t>(p.y) | (uintptr_t)p.y_stride) & (4 * sizeof(T) - 1)) == 0;
    int c = 0;
    join_waves<FM, FN, 1>(lds, acc, [&](int i, int j, v4f(&sum)[1]) {
        v4f add = part[0];
        if constexpr (kMine > 1) add = c == 0 ? part[0] : part[kMine - 1];
        ++c;
        const int t = row0 + i * 16 + (lane & 15), n = n0 + j * 16 + (lane >> 4) * 4;
        if (t >= p.T) return;
        T* y = reinterpret_cast<T*>(p.y + t * p.y_stride);
        union {
            T e[4];
            unsigned long long v[sizeof(T) / 2];
        } out;
#pragma unroll
        for (int q = 0; q < 4; ++q) out.e[q] = (T)(sum[0][q] + add[q]);
        if (whole && n + 4 <= p.n) {
            if constexpr (sizeof(T) == 2) *reinterpret_cast<unsigned long long*>(y + n) = out.v[0];
            else *reinterpret_cast<v4u*>(y + n) = __builtin_bit_cast(v4u, out);
        } else {
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (n + q < p.n) y[n + q] = out.e[q];
        }
    });
    static_assert(kMine <= 2, "two blocks a wave at most");
}

template <typename T, int FM, int FN>
hipError_t go_few(const Args& p, [[maybe_unused]] bool aligned, hipStream_t stream) {
    const dim3 grid((p.n + 16 * FN - 1) / (16 * FN), (p.T + 16 * FM - 1) / (16 * FM));
    constexpr int lds = stream_lds<FM, FN>();
    auto launch = [&](auto kernel) {
        constexpr auto k = decltype(kernel)::value;
        if (const hipError_t err = allow_lds_once<k>(lds); err != hipSuccess) return err;
        k<<<grid, kStreamThreads, lds, stream>>>(p);
        return hipGetLastError();
    };
    if constexpr (FM == 1) {  // (more rows of whole pieces go to the tall tiles)
        if (aligned) return launch(std::integral_constant<void (*)(Args), project_few_kernel<T, FM, FN, true>>{});
    }
    return launch(std::integral_constant<void (*)(Args), project_few_kernel<T, FM, FN, false>>{});
}

template <typename T, typename S>
hipError_t go(const Args& p, hipStream_t stream) {
    const long long grid = (long long)((p.T + S::kRows - 1) / S::kRows) * ((p.n + S::kCols - 1) / S::kCols);
    if (const hipError_t err = allow_lds_once<project_kernel<T, S>>(S::kLds); err != hipSuccess) return err;
    project_kernel<T, S><<<(int)grid, S::kThreads, S::kLds, stream>>>(p);
    return hipGetLastError();
}

template <typename T>
hipError_t run(const Args& p, float* sums, hipStream_t stream) {
    using S = Shape<1, 4, 4, 2>;
    const bool aligned = ((reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.w) | p.x_stride | p.d * sizeof(T)) & 15) == 0;
    const bool a_aligned = aligned && (reinterpret_cast<uintptr_t>(p.a) & 15) == 0;
    const int padded = p.u_stride / (int)sizeof(T);
    switch (forms::shrink_form(p.T, padded)) {
        case forms::Shrink::ONE_RANK: {
            const dim3 grid(p.T, (padded + 3) / 4);
            if (a_aligned) shrink_few_kernel<T, 1, true><<<grid, 256, 0, stream>>>(p);
            else shrink_few_kernel<T, 1, false><<<grid, 256, 0, stream>>>(p);
            break;
        }
        case forms::Shrink::FOUR_RANKS: {
            const dim3 grid(p.T, (padded + 15) / 16);
            if (a_aligned) shrink_few_kernel<T, 4, true><<<grid, 256, 0, stream>>>(p);
            else shrink_few_kernel<T, 4, false><<<grid, 256, 0, stream>>>(p);
            break;
        }
        case forms::Shrink::TILES: {
            constexpr int FM = 2, lds = stream_lds<FM, 2>();
            const dim3 grid((p.T + 16 * FM - 1) / (16 * FM), (p.r + 31) / 32);
            if (a_aligned) shrink_kernel<T, FM, true><<<grid, kStreamThreads, lds, stream>>>(p);
            else shrink_kernel<T, FM, false><<<grid, kStreamThreads, lds, stream>>>(p);
            break;
        }
    }
    const forms::Project form = forms::project_form(p.T, p.d, p.n, sizeof(T), aligned);
    if (form.kind == forms::Project::TILES) return go<T, S>(p, stream);
    if (form.kind == forms::Project::TALL) {
        switch (form.fm) {
            case 2: return go_cut<T, 2>(p, sums, form.splits, stream);
            case 3: return go_cut<T, 3>(p, sums, form.splits, stream);
            case 4: return go_cut<T, 4>(p, sums, form.splits, stream);
            case 5: return go_cut<T, 5>(p, sums, form.splits, stream);
            case 6: return go_cut<T, 6>(p, sums, form.splits, stream);
            case 7: return go_cut<T, 7>(p, sums, form.splits, stream);
            default: return go_cut<T, 8>(p, sums, form.splits, stream);
        }
    }
    switch (16 * form.fm + form.fn) {
        case 16 + 1: return go_few<T, 1, 1>(p, aligned, stream);
        case 16 + 2: return go_few<T, 1, 2>(p, aligned, stream);
        case 32 + 1: return go_few<T, 2, 1>(p, aligned, stream);
        case 32 + 2: return go_few<T, 2, 2>(p, aligned, stream);
        case 64 + 1: return go_few<T, 4, 1>(p, aligned, stream);
        case 64 + 2: return go_few<T, 4, 2>(p, aligned, stream);
        default: return go_few<T, 4, 4>(p, aligned, stream);
    }
}

inline int u_stride_bytes(int r, int size) { return (r * size + 15) / 16 * 16; }

}  // namespace

inline size_t u_bytes(int T, int r, int size) { return ((size_t)T * u_stride_bytes(r, size) + 255) & ~(size_t)255; }

size_t lora_project_workspace_bytes(int T, int d, int n, int r, int dtype) {
    const int size = dtype == DTYPE_F32 ? 4 : 2;
    return u_bytes(T, r, size) + sums_bytes(T, d, n, size);
}

hipError_t launch_lora_project(int T, int d, int n, int r, int L, int dtype, const void* x, long long x_stride, const void* w, const void* a,
                               const void* b, const int* adapter, const float* scale, void* y, long long y_stride, void* workspace,
                               hipStream_t stream) {
    if (T <= 0) return hipSuccess;
    const int size = dtype == DTYPE_F32 ? 4 : 2;
    auto in = [](const void* p) { return static_cast<const char*>(p); };
    const Args p{in(x), in(w), in(a), in(b), static_cast<char*>(workspace), static_cast<char*>(y), adapter, scale, x_stride * size, y_stride * size,
                 T, d, n, r, L, u_stride_bytes(r, size)};
    float* sums = reinterpret_cast<float*>(static_cast<char*>(workspace) + u_bytes(T, r, size));
    // A launch has fewer than 2^32 work items in x: at most 2^26 rows (the adapters' first product has 16 a row), and fewer than
    // 2^24 tiles of 64 x 128 with 256 work items each (tall ones have no more).  Beyond, the rows go in equal parts, none of which
    // is so short that its K would be cut.
    const long long most = std::min(1ll << 26, ((1 << 24) - 64) / ((n + 255) / 256 * 2) * 64ll);
    const int parts = (int)((T - 1) / most) + 1;
    for (int i = 0; i < parts; ++i) {
        const long long from = (long long)T * i / parts, to = (long long)T * (i + 1) / parts;
        Args part = p;
        part.T = (int)(to - from);
        part.x += from * p.x_stride, part.y += from * p.y_stride, part.u += from * p.u_stride, part.adapter += from;
        const hipError_t err = dtype == DTYPE_F32   ? run<float>(part, sums, stream)
                               : dtype == DTYPE_F16 ? run<_Float16>(part, sums, stream)
                                                    : run<__bf16>(part, sums, stream);
        if (err != hipSuccess) return err;
    }
    return hipSuccess;
}

}  // namespace infmoe
