// Top-k of a router's logits, with the weights of the chosen experts.
//
//   score s(l): softmax over the row, 1 / (1 + e^-l), or sqrt(log(1 + e^l))
//   order:      by l, or by s(l) + bias where a selection bias is given; ties to
//               the lowest index; a logit (or a biased score) of -inf or NaN is
//               never chosen
//   weight:     s of the chosen (without the bias), over their sum if asked for,
//               times a constant
//
// A wave has a row, lane i the experts i, i + 64, ...  The k largest are found one
// by one: each lane's best, a maximum over the wave, the lowest index that has it.
//
// Order by biased scores is the order of the exact scores even where fp32 cannot
// tell two apart: the k + 1 largest are found in fp32 first, and if two
// neighbours among them are nearer than fp32's error the row is done again in 64
// bits (about one row in a hundred of normal logits).  Weights are computed in 64
// bits: one exponential a lane, and far logits keep their ratios.
#pragma once

#include "exl3_fp8.hpp"

namespace exl3 {

enum Scoring : int { SCORE_SOFTMAX = 0, SCORE_SIGMOID = 1, SCORE_SQRTSOFTPLUS = 2 };

constexpr int ROUTE_MAX_TOPK = 64;
constexpr int ROUTE_MAX_EXPERTS = 2048;

// v of the lane that a DPP pattern names, `none` where it names no lane.
template <int CTRL, int ROWS, typename T>
__device__ __forceinline__ T lane_of(T v, T none) {
    if constexpr (sizeof(T) == 8) {
        const u32x2_t a = __builtin_bit_cast(u32x2_t, v), b = __builtin_bit_cast(u32x2_t, none);
        return __builtin_bit_cast(T, u32x2_t{(uint32_t)__builtin_amdgcn_update_dpp((int)b[0], (int)a[0], CTRL, ROWS, 0xf, false),
                                             (uint32_t)__builtin_amdgcn_update_dpp((int)b[1], (int)a[1], CTRL, ROWS, 0xf, false)});
    } else {
        return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, none), __builtin_bit_cast(int, v),
                                                                 CTRL, ROWS, 0xf, false));
    }
}

template <typename T>
__device__ __forceinline__ T read_lane(T v, int lane) {
    if constexpr (sizeof(T) == 8) {
        const u32x2_t a = __builtin_bit_cast(u32x2_t, v);
        return __builtin_bit_cast(T, u32x2_t{(uint32_t)__builtin_amdgcn_readlane((int)a[0], lane),
                                             (uint32_t)__builtin_amdgcn_readlane((int)a[1], lane)});
    } else {
        return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
    }
}

// op over the wave's lanes (each lane's value once), as a wave-uniform value: a
// scan of each row of 16 lanes, then of the rows; lane 63 has it all.
template <typename T, typename Op>
__device__ __forceinline__ T wave_all(T v, T none, Op op) {
    v = op(v, lane_of<0x111, 0xf>(v, none));        // row_shr:1, 2, 4, 8
    v = op(v, lane_of<0x112, 0xf>(v, none));
    v = op(v, lane_of<0x114, 0xf>(v, none));
    v = op(v, lane_of<0x118, 0xf>(v, none));
    v = op(v, lane_of<0x142, 0xa>(v, none));        // row_bcast:15, 31
    v = op(v, lane_of<0x143, 0xc>(v, none));
    return read_lane(v, 63);
}

template <typename T>
__device__ __forceinline__ T wave_sum(T v) {
    return wave_all(v, (T)0, [](T a, T b) { return a + b; });
}

template <typename T>
__device__ __forceinline__ T neg_inf() { return (T)-__builtin_inff(); }

// NaN-free values only.
template <typename T>
__device__ __forceinline__ T wave_max(T v) {
    return wave_all(v, neg_inf<T>(), [](T a, T b) { return a > b ? a : b; });
}

__device__ __forceinline__ int wave_min(int v) {
    return wave_all(v, 0x7fffffff, [](int a, int b) { return min(a, b); });
}

// softplus is max(l, 0) + log(1 + e^-|l|), which neither overflows nor loses small l.
template <typename T>
__device__ __forceinline__ T score_of(int scoring, T l, T most, T total) {
    if (scoring == SCORE_SOFTMAX) return exp(l - most) / total;
    if (scoring == SCORE_SIGMOID) return (T)1 / ((T)1 + exp(-l));
    return sqrt((l > 0 ? l : (T)0) + log1p(exp(l > 0 ? -l : l)));
}

// The `count` largest of the wave's keys in order: lane j keeps the j-th one's index
// (-1: none left) and key.  Keys are NaN-free; -inf is never chosen.
template <typename T, int N>
__device__ __forceinline__ void select_top(T (&key)[N], int count, int lane, int& chosen, T& chosen_key) {
    chosen = -1;
    chosen_key = neg_inf<T>();
    for (int j = 0; j < count; ++j) {
        T best = key[0];
        int at = 0;
#pragma unroll
        for (int i = 1; i < N; ++i)
            if (key[i] > best) {
                best = key[i];
                at = i;
            }
        const T top = wave_max(best);
        if (!(top > neg_inf<T>())) break;
        const uint64_t have = __ballot(best == top);
        const int owner = __builtin_ctzll(have);
        const int idx = have & (have - 1) ? wave_min(best == top ? at * 64 + lane : 0x7fffffff)
                                          : __builtin_amdgcn_readlane(at, owner) * 64 + owner;
        if (lane == j) {
            chosen = idx;
            chosen_key = top;
        }
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (idx == i * 64 + lane) key[i] = neg_inf<T>();
    }
}

struct RouteArgs {
    const void* logits;         // [rows][E], OutKind
    const float* bias;          // [E] or null
    void* ids;                  // [rows][topk], int32 or int64
    float* weights;             // [rows][topk]
    int64_t rows;
    int kind, E, topk, scoring, ids64, renormalize;
    float scale;
};

template <int N>
__global__ __launch_bounds__(256) void moe_route_kernel(const RouteArgs A) {
    const int lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= A.rows) return;
    const int E = A.E;
    float l[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int e = i * 64 + lane;
        float v = neg_inf<float>();
        if (e < E) {
            const int64_t at = row * E + e;
            v = A.kind == OUT_F32    ? static_cast<const float*>(A.logits)[at]
                : A.kind == OUT_BF16 ? bf16_to_f32(static_cast<const uint16_t*>(A.logits)[at])
                                     : f16_bits_to_f32(static_cast<const uint16_t*>(A.logits)[at]);
        }
        l[i] = v == v ? v : neg_inf<float>();
    }
    // the softmax's maximum and sum, where something needs them
    float most = 0.f, total = 1.f;
    const bool over_row = A.scoring == SCORE_SOFTMAX && (A.bias || !A.renormalize);
    if (over_row) {
        most = l[0];
#pragma unroll
        for (int i = 1; i < N; ++i) most = fmaxf(most, l[i]);
        most = wave_max(most);
        total = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) total += l[i] > neg_inf<float>() ? expf(l[i] - most) : 0.f;
        total = wave_sum(total);
    }
    int chosen;
    if (!A.bias) {
        float key[N], unused;
#pragma unroll
        for (int i = 0; i < N; ++i) key[i] = l[i];
        select_top<float, N>(key, A.topk, lane, chosen, unused);
    } else {
        float key[N], got;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int e = i * 64 + lane;
            const float v = l[i] > neg_inf<float>() ? score_of<float>(A.scoring, l[i], most, total) + A.bias[e]
                                                    : neg_inf<float>();
            key[i] = v == v ? v : neg_inf<float>();
        }
        const int more = min(A.topk + 1, 64);
        select_top<float, N>(key, more, lane, chosen, got);
        const float below = __shfl_down(got, 1);
        // fp32's scores are within 4e-6 of the exact ones (relative above one)
        const bool near = lane + 1 < more && chosen >= 0 && !(got - below > 0x1p-17f * fmaxf(1.f, fabsf(got)));
        if (__any(near) || more == A.topk) {
            double dmost = most, dtotal = 1.0, dkey[N], unused;
            if (A.scoring == SCORE_SOFTMAX) {
                dtotal = 0.0;
#pragma unroll
                for (int i = 0; i < N; ++i) dtotal += l[i] > neg_inf<float>() ? exp((double)l[i] - dmost) : 0.0;
                dtotal = wave_sum(dtotal);
            }
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int e = i * 64 + lane;
                const double v = l[i] > neg_inf<float>()
                                     ? score_of<double>(A.scoring, (double)l[i], dmost, dtotal) + (double)A.bias[e]
                                     : neg_inf<double>();
                dkey[i] = v == v ? v : neg_inf<double>();
            }
            select_top<double, N>(dkey, A.topk, lane, chosen, unused);
        }
        if (lane >= A.topk) chosen = -1;
    }
    // the chosen logits, one a lane
    float mine = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float v = __shfl(l[i], chosen & 63);
        if ((chosen >> 6) == i) mine = v;
    }
    double s = 0.0;
    if (A.scoring == SCORE_SOFTMAX) {
        // over their own sum only ratios count: from the largest chosen logit they cannot all underflow
        const float top = over_row && !A.renormalize ? most : wave_max(chosen >= 0 ? mine : neg_inf<float>());
        if (chosen >= 0) s = exp((double)mine - (double)top) / (A.renormalize ? 1.0 : (double)total);
    } else if (chosen >= 0) {
        s = score_of<double>(A.scoring, (double)mine, 0.0, 1.0);
    }
    if (A.renormalize) {
        const double sum = wave_sum(s);
        s = sum != 0.0 ? s / sum : 0.0;
    }
    if (lane < A.topk) {
        const int64_t at = row * A.topk + lane;
        if (A.ids64) static_cast<int64_t*>(A.ids)[at] = chosen;
        else static_cast<int32_t*>(A.ids)[at] = chosen;
        A.weights[at] = (float)(s * (double)A.scale);
    }
}

}  // namespace exl3
