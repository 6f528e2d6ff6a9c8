// Routing to the k best experts for gfx950: scores, groups, selection and weights in one launch.
//
//   s_e = softmax(l)_e or 1 / (1 + exp(-l_e));  c_e = s_e + bias_e;  the `top_groups` groups with the largest sums of their
//   `group_top` largest c stay;  ids = the k largest c, largest first, the lowest index among equals;
//   w = scale * s_ids (/ sum of s_ids when renormalised).
//
// Softmax and the logistic function keep the order of the logits, so where neither a bias nor a sum over a group enters,
// the logits themselves are compared, which needs no arithmetic and no tolerance.  Otherwise the choice is made on scores
// in FP32, and a row in which two neighbours of the ranking are closer than what FP32 can order (see score_error) is
// chosen once more on scores in 64 bits; a result never depends on FP32's roundings.
//
// Layout: a row of E logits takes a whole wave, or 16 neighbouring lanes of it when it has at most 64 experts, each lane with
// V <= 32 consecutive experts in registers; a group of experts takes a power of two of those lanes (slots that this leaves
// over hold minus infinity).  Consecutive experts sit in ascending lanes and slots, so "the lowest index" is "the first
// lane, then the first slot", and all exchanges are between registers of one wave: no barrier.
//
// Bound by vector instructions (131071 rows of 256 experts are 134 MB and 8 MB of results, 23 us at 6.2 TB/s, and take 68): a round of the selection is a
// maximum over the row and the removal of its place.  With a row per wave that place is scalar arithmetic on the masks of
// V comparisons; with rows of 16 lanes the same instructions serve four rows.
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include "kernels.h"

namespace infmoe {
namespace {

constexpr int kThreads = 256;
typedef unsigned long long u64;
constexpr float kInf = __builtin_inff();

struct Args {
    const void* logits;
    long long stride;  // elements between rows
    const float* bias;
    int* ids;
    float* weights;
    int T, E, k, dtype, score, groups, per, lanes_log2, top_groups, group_top, renormalize, vec;
    float scale;
};

// v of the lane that the data-parallel control names; `other` in the lanes of rows that ROWS leaves out
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ float dpp(float v, float other = 0.f) {
    return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(other), __float_as_int(v), CTRL, ROWS, 0xf, false));
}
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ double dpp(double v, double other = 0.0) {
    const int lo = __builtin_amdgcn_update_dpp(__double2loint(other), __double2loint(v), CTRL, ROWS, 0xf, false);
    return __hiloint2double(__builtin_amdgcn_update_dpp(__double2hiint(other), __double2hiint(v), CTRL, ROWS, 0xf, false), lo);
}
__device__ __forceinline__ float larger(float a, float b) { return __builtin_fmaxf(a, b); }
__device__ __forceinline__ double larger(double a, double b) { return __builtin_fmax(a, b); }
__device__ __forceinline__ float size_of(float v) { return __builtin_fabsf(v); }
__device__ __forceinline__ double size_of(double v) { return __builtin_fabs(v); }

// lane 63's value in all lanes, as a scalar
__device__ __forceinline__ float last_lane(float v) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63)); }
__device__ __forceinline__ double last_lane(double v) {
    return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(v), 63), __builtin_amdgcn_readlane(__double2loint(v), 63));
}
__device__ __forceinline__ float lane_value(float v, int lane) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane)); }
__device__ __forceinline__ double lane_value(double v, int lane) {
    return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(v), lane), __builtin_amdgcn_readlane(__double2loint(v), lane));
}

// Reductions over the G lanes of a row, the result in all of them: lane ^ 1, lane ^ 2, mirror in 8, mirror in 16; over 64
// lanes then the last lane of 16 to the next 16, and of 32 to the next 32 (the full sums and maxima arrive in lane 63).
template <int G, typename R>
__device__ __forceinline__ R row_max(R v) {
    v = larger(v, dpp<0xB1>(v));
    v = larger(v, dpp<0x4E>(v));
    v = larger(v, dpp<0x141>(v));
    v = larger(v, dpp<0x140>(v));
    if constexpr (G == 64) {
        v = larger(v, dpp<0x142, 0xa>(v, v));
        v = last_lane(larger(v, dpp<0x143, 0xc>(v, v)));
    }
    return v;
}
template <int G, typename R>
__device__ __forceinline__ R row_sum(R v) {
    v += dpp<0xB1>(v);
    v += dpp<0x4E>(v);
    v += dpp<0x141>(v);
    v += dpp<0x140>(v);
    if constexpr (G == 64) {
        v += dpp<0x142, 0xa>(v, (R)0);
        v = last_lane(v + dpp<0x143, 0xc>(v, (R)0));
    }
    return v;
}

// The sum of a lane's values from I on, V of them, in pairs
template <int I, int V, typename R, int N>
__device__ __forceinline__ R pair_sum(const R (&v)[N]) {
    if constexpr (V == 1) return v[I];
    else return pair_sum<I, V / 2>(v) + pair_sum<I + V / 2, V / 2>(v);
}

__device__ __forceinline__ float load_logit(const Args& a, long long at) {
    if (a.dtype == DTYPE_F32) return static_cast<const float*>(a.logits)[at];
    const unsigned short h = static_cast<const unsigned short*>(a.logits)[at];
    return a.dtype == DTYPE_BF16 ? __uint_as_float((unsigned)h << 16) : __half2float(__ushort_as_half(h));
}

__device__ __forceinline__ float exp_of(float x) { return __expf(x); }

// Two scores p + bias computed in FP32 are ordered as the exact ones when they lie further apart than
//   score_error(kind) * max(p_max, 2^-10) + 2^-22 * |p + bias|.
// exp_of(x) is 2^(x * log2 e) with the product rounded, so its relative error is at most (1.45 |x| + 2) u, u = 2^-24.
// Logistic, p = 1 / (1 + exp(-l)): p (1 - p) (1.45 |l| + 2) u + 3 u p <= 4 u; against p_max it is largest where all scores are
// small, (1.45 |l| + 5) u p, which from p = 2^-10 on down is at most 15 u * 2^-10.  Two such errors, either way: 30 u.
// Softmax, p = exp(l - m) / sum:
//   * of its own a score has the roundings of l - m and of the argument, (2.45 |l - m| + 2) u p with |l - m| p <= 0.37 p_max,
//     and of the product with 1 / sum: under 4 u p_max;
//   * all scores of a row share the relative error of 1 / sum: the additions, in pairs (11 at most, of up to 32 terms a lane and
//     64 lanes; empty slots add an exact zero), the terms' errors, (2.45 a + 2) u with a the mean of |l - m| under p, which is
//     below 4.5 for up to 1024 experts, and the quotient: under 26 u, times a difference of at most p_max.
//   Together 26 u + 2 * 4 u = 34 u.
// The sum with the bias is rounded once: u |p + bias|.
__device__ __forceinline__ float score_error(int kind) { return kind == SCORE_SOFTMAX ? 0x1p-18f : 0x1p-19f; }  // 64 u, 32 u

// The experts of all but the top_groups best groups masked.  R: float, or double for the rows that FP32 cannot order.  Returns
// whether the choice of groups is certain (CHECK).
template <typename R, bool CHECK, int G, int V>
__device__ __forceinline__ bool keep_groups(const Args& a, R (&c)[V], float floor_gap, int in_row) {
    const int lane = threadIdx.x & 63;
    bool sure = true;
    R one = -INFINITY, two = -INFINITY;  // the two largest of the lane's, then of its group's lanes
#pragma unroll
    for (int i = 0; i < V; ++i) {
        two = larger(two, one < c[i] ? one : c[i]);
        one = larger(one, c[i]);
    }
    for (int step = 1; step < (1 << a.lanes_log2); step <<= 1) {
        const R o1 = __shfl_xor(one, step), o2 = __shfl_xor(two, step);
        two = larger(larger(two, o2), one < o1 ? one : o1);
        one = larger(one, o1);
    }
    const R value = a.group_top == 2 ? one + two : one;
    // A group's sum is off by the errors of its scores, u |one| and u |two| of their sums with the bias, and u |value|: its terms
    // count, not the sum in which they may cancel.  Two sums that are farther apart than 2 floor_gap + 2^-21 times the terms of
    // either one (8 u, where 4 u times the larger would do) are ordered.
    const R terms = a.group_top == 2 ? size_of(one) + size_of(two) : size_of(one);
    const int group = in_row >> a.lanes_log2;
    int rank = 0;
    for (int g = 0; g < a.groups; ++g) {
        const R other = G == 64 ? lane_value(value, g << a.lanes_log2) : __shfl(value, (lane - in_row) + (g << a.lanes_log2));
        rank += other > value || (other == value && g < group);
        if (CHECK && g != group && group < a.groups && other > -INFINITY && value > -INFINITY)
            sure = sure && size_of(other - value) > 2 * (R)floor_gap + (R)0x1p-21 * terms;
    }
    if (rank >= a.top_groups)
#pragma unroll
        for (int i = 0; i < V; ++i) c[i] = -INFINITY;
    return sure;
}

// Whether two neighbours of the ranking are far enough apart for FP32.
__device__ __forceinline__ bool apart(float larger_one, float smaller, float floor_gap) {
    return !(smaller > -kInf) || larger_one - smaller > floor_gap + 0x1p-22f * size_of(larger_one);
}

// What the lanes of this wave have written to LDS is there for the others, and nothing is moved across.  (No instruction: LDS
// operations of one wave are done in order.  It is the compiler that must not take a lane's own store for its later load.)
__device__ __forceinline__ void lanes_meet() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// The k best of rows of 16 lanes from a short list, when one can be had: t, the (k + 1)-th largest among the two best of every
// lane, is reached by k + 1 experts at least and, unless many are equal or few lanes take part, by no more than 16.  Those go
// through LDS to a lane each, in order of their indices; there every lane counts who is before it, and the counts are the
// ranking.  (k + 1 rounds of choose_rounds instead: 1580 vector instructions a wave for 131071 rows of 256, 107 us.)
// Returns false, for all rows of the wave, where a list is too long.
template <bool CHECK, int V>
__device__ __forceinline__ bool choose_listed(const Args& a, const float (&c)[V], float floor_gap, int in_row, int first, float2* list, int* mine, bool* sure) {
    float one = -kInf, two = -kInf;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        two = larger(two, one < c[i] ? one : c[i]);
        one = larger(one, c[i]);
    }
    int before_one = 0, before_two = one > two;
    auto against = [&](float o1, float o2) {
        before_one += o1 > one, before_one += o2 > one;
        before_two += o1 > two, before_two += o2 > two;
    };
#define INFMOE_EACH_TURN(X) X(1) X(2) X(3) X(4) X(5) X(6) X(7) X(8) X(9) X(10) X(11) X(12) X(13) X(14) X(15)
#define INFMOE_TURN(r) against(dpp<0x120 + r>(one), dpp<0x120 + r>(two));  // of the lane r before, around the 16
    INFMOE_EACH_TURN(INFMOE_TURN)
#undef INFMOE_TURN
    float t = before_two <= a.k ? two : before_one <= a.k ? one : kInf;
    t = -row_max<16>(-t);                     // the smallest of those that at most k are before
    t = larger(t, -3.4028235e38f);            // (a masked expert is never listed)
    int here = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) here += c[i] >= t;
    int to = here;  // listed in this lane and those before it
#define INFMOE_SCAN(ctrl) to += __builtin_amdgcn_update_dpp(0, to, ctrl, 0xf, 0xf, false);
    INFMOE_SCAN(0x111) INFMOE_SCAN(0x112) INFMOE_SCAN(0x114) INFMOE_SCAN(0x118)
#undef INFMOE_SCAN
    if (__ballot(to > 16) != 0) return false;
    float2* row = list + ((threadIdx.x & 63) >> 4) * 16;
    row[in_row] = float2{-kInf, __int_as_float(-1)};
    lanes_meet();  // (listed entries replace these)
    int at = to - here;
#pragma unroll
    for (int i = 0; i < V; ++i)
        if (c[i] >= t) row[at++] = float2{c[i], __int_as_float(first + i)};
    lanes_meet();
    const float2 entry = row[in_row];
    lanes_meet();  // (ranked entries replace these)
    int rank = 0;
    // an equal one counts as before where its lane, and so its index, is lower
#define INFMOE_TURN(r)                                              \
    {                                                               \
        const float other = dpp<0x120 + r>(entry.x);                \
        rank += other > entry.x || (other == entry.x && in_row >= r); \
    }
    INFMOE_EACH_TURN(INFMOE_TURN)
#undef INFMOE_TURN
#undef INFMOE_EACH_TURN
    row[rank] = entry;
    lanes_meet();
    const float2 mine_now = row[in_row];
    *mine = in_row < a.k ? __float_as_int(mine_now.y) : -1;
    const float next = dpp<0x101>(mine_now.x, -kInf);  // of the lane behind; read by all lanes, a lane that is left out gives nothing
    if (CHECK) *sure = in_row >= a.k || apart(mine_now.x, next, floor_gap);
    return true;
}

// The k best of one row per G lanes, one after the other.  Lane j of the row gets the j-th expert in *mine (-1: nothing left
// to choose).  Returns whether the row is ordered for certain (CHECK; the same answer in all of a row's lanes).
template <typename R, bool CHECK, int G, int V>
__device__ __forceinline__ bool choose_rounds(const Args& a, R (&c)[V], float floor_gap, int in_row, u64 row_lanes, int first, int* mine) {
    const int lane = threadIdx.x & 63;
    bool sure = true;
    R before = INFINITY;
    const int rounds = CHECK ? a.k + 1 : a.k;  // the border to the first expert left out counts too
    for (int j = 0; j < rounds; ++j) {
        R best = c[0];
#pragma unroll
        for (int i = 1; i < V; ++i) best = larger(best, c[i]);
        const R top = row_max<G>(best);
        if (CHECK && j > 0) sure = sure && apart((float)before, (float)top, floor_gap);
        if (j == a.k) break;
        before = top;
        if constexpr (G == 64) {
            u64 where[V], any = 0;
#pragma unroll
            for (int i = 0; i < V; ++i) any |= where[i] = __ballot(c[i] == top);
            const int winner = any != 0 ? __builtin_ctzll(any) : 0;
            int slot = 0;
#pragma unroll
            for (int i = V - 1; i >= 0; --i) slot = (where[i] >> winner) & 1 ? i : slot;
            const int expert = __builtin_amdgcn_readlane(first, winner) + slot;
            if (in_row == j) *mine = top > -INFINITY ? expert : -1;
#pragma unroll
            for (int i = 0; i < V; ++i) c[i] = i == slot && lane == winner ? (R)-INFINITY : c[i];
        } else {
            const u64 who = __ballot(best == top) & row_lanes;
            const int winner = (who != 0 ? __builtin_ctzll(who) : 0);
            int slot = 0;
#pragma unroll
            for (int i = V - 1; i >= 0; --i) slot = c[i] == best ? i : slot;
            const int expert = __shfl(first + slot, winner);
            if (in_row == j) *mine = top > -INFINITY ? expert : -1;
#pragma unroll
            for (int i = 0; i < V; ++i) c[i] = i == slot && lane == winner ? (R)-INFINITY : c[i];
        }
    }
    return sure;
}

// Groups, then the k best.
template <typename R, bool CHECK, int G, int V>
__device__ __forceinline__ bool choose(const Args& a, R (&c)[V], float floor_gap, int in_row, u64 row_lanes, int first, float2* list, int* mine) {
    bool sure = true;
    if (a.groups > 1) sure = keep_groups<R, CHECK, G, V>(a, c, floor_gap, in_row);
    if constexpr (G == 16 && V >= 8 && sizeof(R) == 4) {
        bool ordered = true;
        if (a.k <= 15 && choose_listed<CHECK, V>(a, c, floor_gap, in_row, first, list, mine, &ordered)) return sure && ordered;
    }
    return choose_rounds<R, CHECK, G, V>(a, c, floor_gap, in_row, row_lanes, first, mine) && sure;
}

template <int G, int V>
__global__ __launch_bounds__(kThreads) void route_kernel(Args a) {
    __shared__ float2 s_list[kThreads];  // choose_listed: 64 entries a wave
    float2* list = s_list + (threadIdx.x & ~63);
    const int lane = threadIdx.x & 63, in_row = lane & (G - 1);
    const u64 row_lanes = (G == 64 ? ~0ull : ((1ull << (G & 63)) - 1)) << (lane - in_row);
    const long long row = ((long long)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6)) * (64 / G) + lane / G;
    const bool live = row < a.T;
    const long long at = (live ? row : a.T - 1) * a.stride;  // lanes past the last row repeat it and store nothing
    const int group = in_row >> a.lanes_log2;
    const int local = (in_row & ((1 << a.lanes_log2) - 1)) * V;  // of the lane's first expert in its group
    const int first = group * a.per + local;
    const int have = group < a.groups ? min(max(a.per - local, 0), V) : 0;

    float l[V];
    if (a.vec) {  // every slot taken, 16-byte pieces
        if constexpr (V % 4 == 0) {
            if (a.dtype == DTYPE_F32) {
                const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(a.logits) + at + first);
#pragma unroll
                for (int i = 0; i < V / 4; ++i) {
                    const float4 q = p[i];
                    l[4 * i] = q.x, l[4 * i + 1] = q.y, l[4 * i + 2] = q.z, l[4 * i + 3] = q.w;
                }
            }
        }
        if constexpr (V % 8 == 0) {
            if (a.dtype != DTYPE_F32) {
                const uint4* p = reinterpret_cast<const uint4*>(static_cast<const unsigned short*>(a.logits) + at + first);
#pragma unroll
                for (int i = 0; i < V / 8; ++i) {
                    const uint4 q = p[i];
                    const unsigned u[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if (a.dtype == DTYPE_BF16) {
                            l[8 * i + 2 * j] = __uint_as_float(u[j] << 16);
                            l[8 * i + 2 * j + 1] = __uint_as_float(u[j] & 0xffff0000u);
                        } else {
                            l[8 * i + 2 * j] = __half2float(__ushort_as_half((unsigned short)(u[j] & 0xffff)));
                            l[8 * i + 2 * j + 1] = __half2float(__ushort_as_half((unsigned short)(u[j] >> 16)));
                        }
                    }
                }
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) l[i] = i < have ? load_logit(a, at + first + i) : -kInf;
    }

    bool bad = false;  // no order: a NaN, or a softmax over an infinite logit
    const float finite = a.score == SCORE_SOFTMAX ? 3.4028235e38f : kInf;
#pragma unroll
    for (int i = 0; i < V; ++i) bad |= !(l[i] <= finite);

    const bool scored = a.bias != nullptr || a.group_top == 2;
    float m = 0.f, sum = 1.f;
    if (a.score == SCORE_SOFTMAX) {
        m = l[0];
#pragma unroll
        for (int i = 1; i < V; ++i) m = fmaxf(m, l[i]);
        m = row_max<G>(m);
        m = m > -kInf ? m : 0.f;  // (every expert masked)
        if (scored || !a.renormalize) {
            float e[V];
#pragma unroll
            for (int i = 0; i < V; ++i) e[i] = exp_of(l[i] - m);
            sum = row_sum<G>(pair_sum<0, V>(e));
        }
    }

    int mine = -1;
    if (!scored) {
        float c[V];
#pragma unroll
        for (int i = 0; i < V; ++i) c[i] = l[i];
        choose<float, false, G, V>(a, c, 0.f, in_row, row_lanes, first, list, &mine);
    } else {
        float c[V], b[V], peak = 0x1p-10f;
#pragma unroll
        for (int i = 0; i < V; ++i) b[i] = 0.f;
        if (a.bias != nullptr) {
            if (a.vec) {
#pragma unroll
                for (int i = 0; i < V; ++i) b[i] = a.bias[first + i];
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i) b[i] = i < have ? a.bias[first + i] : 0.f;
            }
        }
        if (a.score == SCORE_SOFTMAX) {
            const float rsum = 1.f / sum;
#pragma unroll
            for (int i = 0; i < V; ++i) c[i] = exp_of(l[i] - m) * rsum;
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) c[i] = __builtin_amdgcn_rcpf(1.f + exp_of(-l[i]));
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
            peak = fmaxf(peak, c[i]);
            c[i] = l[i] > -kInf ? c[i] + b[i] : -kInf;
            bad |= !(c[i] < kInf);
        }
        peak = row_max<G>(peak);
        bool sure = choose<float, true, G, V>(a, c, score_error(a.score) * peak, in_row, row_lanes, first, list, &mine);
        if (__ballot(!sure && !bad) != 0) {  // some row of this wave: all of its rows again, in 64 bits
            double d[V];
            if (a.score == SCORE_SOFTMAX) {
                double total = 0.0;
#pragma unroll
                for (int i = 0; i < V; ++i) total += d[i] = exp((double)l[i] - m);
                total = row_sum<G>(total);
#pragma unroll
                for (int i = 0; i < V; ++i) d[i] /= total;
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i) d[i] = 1.0 / (1.0 + exp(-(double)l[i]));
            }
#pragma unroll
            for (int i = 0; i < V; ++i) d[i] = l[i] > -kInf ? d[i] + (double)b[i] : -INFINITY;
            mine = -1;
            choose<double, false, G, V>(a, d, 0.f, in_row, row_lanes, first, list, &mine);
        }
    }
    const bool nan_row = (__ballot(bad) & row_lanes) != 0;

    // Weights.  Renormalised ones are formed relative to the largest chosen logit, so that a row of tiny scores (their sum
    // may be below FP32's range) keeps its ratios: softmax's common factor cancels; of the logistic function exp(l) / (1 + exp(l)).
    const bool filled = in_row < a.k && mine >= 0;
    const float x = filled ? load_logit(a, at + mine) : -kInf;
    float w;
    if (a.score == SCORE_SOFTMAX) {
        const float base = a.renormalize ? row_max<G>(x) : m;
        w = filled ? expf(x - base) : 0.f;
        if (!a.renormalize && filled) w /= sum;
    } else {
        const float base = a.renormalize ? fminf(row_max<G>(x), 0.f) : 0.f;
        w = !filled ? 0.f : x >= 0.f ? 1.f / (1.f + expf(-x)) : expf(x - base) / (1.f + expf(x));
    }
    if (a.renormalize) {
        const float total = row_sum<G>(w);
        w = total > 0.f ? w / total : w;
    }
    if (live && in_row < a.k) {
        a.ids[row * a.k + in_row] = nan_row ? -1 : mine;
        a.weights[row * a.k + in_row] = nan_row ? __builtin_nanf("") : a.scale * w;
    }
}

template <int G, int V>
hipError_t go(const Args& all, hipStream_t stream) {
    constexpr int rows = kThreads / G, most = (1 << 23) * rows;  // (a launch has fewer than 2^32 work items)
    Args a = all;
    for (int done = 0;;) {
        a.T = min(all.T - done, most);
        route_kernel<G, V><<<(a.T - 1) / rows + 1, kThreads, 0, stream>>>(a);
        if (a.T == all.T - done) return hipGetLastError();
        done += a.T;
        a.logits = static_cast<const char*>(a.logits) + a.T * a.stride * (a.dtype == DTYPE_F32 ? 4 : 2);
        a.ids += (size_t)a.T * a.k;
        a.weights += (size_t)a.T * a.k;
    }
}

template <int G>
hipError_t go_v(const Args& a, int v, hipStream_t stream) {
    switch (v) {
        case 1: return go<G, 1>(a, stream);
        case 2: return go<G, 2>(a, stream);
        case 4: return go<G, 4>(a, stream);
        default: break;
    }
    if (v == 8) return go<G, 8>(a, stream);
    if (v == 16) return go<G, 16>(a, stream);
    if constexpr (G == 64) return go<64, 32>(a, stream);
    return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_route_topk(int T, int E, int k, const void* logits, int dtype, long long row_stride, int score,
                             const float* bias, int groups, int top_groups, int group_top, bool renormalize, float scale,
                             int* ids, float* weights, hipStream_t stream) {
    if (T <= 0) return hipSuccess;
    Args a{logits, row_stride, bias, ids, weights, T, E, k, dtype, score, groups, E / groups, 0, top_groups, group_top, renormalize, 0, scale};
    // Rows of up to 64 experts in 16 lanes with up to four each, four rows to a wave (with few experts, a wave per row leaves
    // most lanes without work); longer ones, and such whose groups or k do not fit 16 lanes, in 64: 128 rows of 256 experts
    // in 6 us instead of 10.  From 4096 rows on every SIMD has waves enough, and what counts is instructions a row: 16
    // lanes with up to 16 experts each (131071 rows of 256 experts: 107 us, a wave per row 160).
    const int most = T >= 4096 ? 16 : 4;
    int per_lane = 0, lanes = 16;
    for (;; lanes = 64) {
        int parts = 1;
        while (parts < groups) parts *= 2;  // groups, each of lanes / parts lanes
        const int each = parts <= lanes && k <= lanes ? (a.per + lanes / parts - 1) / (lanes / parts) : 64;
        if (each <= most || lanes == 64) {
            if (each > 32) return hipErrorInvalidValue;  // (not reached: E <= 1024 and groups <= 64)
            per_lane = 1;
            while (per_lane < each) per_lane *= 2;
            while ((parts << a.lanes_log2) < lanes) ++a.lanes_log2;
            break;
        }
    }
    const int size = dtype == DTYPE_F32 ? 4 : 2;
    a.vec = a.per == (per_lane << a.lanes_log2) && (groups << a.lanes_log2) == lanes && per_lane * size % 16 == 0 &&
            row_stride * size % 16 == 0 && (reinterpret_cast<uintptr_t>(logits) & 15) == 0;
    return lanes == 16 ? go_v<16>(a, per_lane, stream) : go_v<64>(a, per_lane, stream);
}

}  // namespace infmoe
