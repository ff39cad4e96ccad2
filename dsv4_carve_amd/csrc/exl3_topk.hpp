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
// Instructions bound it (8000 rows of 256 experts read 8 MB): keys are integers
// that order as their numbers do, a step of a maximum one DPP instruction (8000
// rows with a bias 14.5 us, 982 instructions a row; 16 rows 4.9 us, a launch and one
// row's chain).
//
// Order by biased scores is the order of the exact scores even where fp32 cannot
// tell two apart: the k + 1 largest are found in fp32 first, and if two
// neighbours among them are nearer than fp32's error the row is done again in 64
// bits (about one row in a hundred of normal logits).  Weights are computed in 64
// bits: one exponential a lane, and far logits keep their ratios; a softmax that
// is not renormalized takes its sum over the row in them too (8000 rows of 256
// experts 10.8 us, 9.1 with renormalization).
#pragma once

#include "exl3_fp8.hpp"

namespace exl3 {

enum Scoring : int { SCORE_SOFTMAX = 0, SCORE_SIGMOID = 1, SCORE_SQRTSOFTPLUS = 2 };

constexpr int ROUTE_MAX_TOPK = 64;
constexpr int ROUTE_MAX_EXPERTS = 2048;

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

template <typename K>
__device__ __forceinline__ K wave_max(K v, K none) {
    return wave_all(v, none, [](K a, K b) { return a > b ? a : b; });
}

// softplus is max(l, 0) + log(1 + e^-|l|), which neither overflows nor loses small l.
template <typename T>
__device__ __forceinline__ T score_of(int scoring, T l, T most, T total) {
    if (scoring == SCORE_SOFTMAX) return exp(l - most) / total;
    if (scoring == SCORE_SIGMOID) return (T)1 / ((T)1 + exp(-l));
    return sqrt((l > 0 ? l : (T)0) + log1p(exp(l > 0 ? -l : l)));
}

// A key that orders as its number does, so that maxima are one integer
// instruction; -inf (and a NaN) is NO_KEY, which is never chosen, and 0 has one key.
template <typename T>
struct KeyOf;
template <>
struct KeyOf<float> {
    typedef int type;
    static constexpr int NO_KEY = INT32_MIN;
    static __device__ __forceinline__ int of(float v) {
        const int b = __float_as_int(v + 0.f);
        return v > -__builtin_inff() ? b ^ (b >> 31 & 0x7fffffff) : NO_KEY;
    }
};
template <>
struct KeyOf<double> {
    typedef long type;
    static constexpr long NO_KEY = INT64_MIN;
    static __device__ __forceinline__ long of(double v) {
        const long b = __builtin_bit_cast(long, v + 0.0);
        return v > -(double)__builtin_inff() ? b ^ (b >> 63 & 0x7fffffffffffffffl) : NO_KEY;
    }
};

// The `count` largest of the wave's keys in order: lane j keeps the j-th one's index
// (-1: none left), key and logit.
template <typename K, int N>
__device__ __forceinline__ void select_top(K (&key)[N], const float (&l)[N], K none, int count, int& chosen, K& chosen_key,
                                           float& logit) {
    const int lane = threadIdx.x & 63;
    chosen = -1;
    chosen_key = none;
    logit = 0.f;
    for (int j = 0; j < count; ++j) {
        K best = key[0];
#pragma unroll
        for (int i = 1; i < N; ++i) best = key[i] > best ? key[i] : best;
        const K top = wave_max(best, none);
        if (top == none) break;
        // the lowest index that has it: the first register, then the first lane
        uint64_t have = 0;
        int at = 0;
#pragma unroll
        for (int i = N - 1; i >= 0; --i) {
            const uint64_t h = __ballot(key[i] == top);
            at = h ? i : at;
            have = h ? h : have;
        }
        const int owner = __builtin_ctzll(have);
        float value = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (at == i) {
                value = read_lane(l[i], owner);
                key[i] = lane == owner ? none : key[i];
            }
        if (lane == j) {
            chosen = at * 64 + owner;
            chosen_key = top;
            logit = value;
        }
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
    // the softmax's maximum, where something needs it, and its sum in fp32 for a first order
    float most = 0.f, total = 1.f;
    const bool over_row = A.scoring == SCORE_SOFTMAX && (A.bias || !A.renormalize);
    if (over_row) {
        most = l[0];
#pragma unroll
        for (int i = 1; i < N; ++i) most = l[i] > most ? l[i] : most;
        most = wave_max(most, neg_inf<float>());
        if (A.bias) {
            total = 0.f;
#pragma unroll
            for (int i = 0; i < N; ++i) total += l[i] > neg_inf<float>() ? expf(l[i] - most) : 0.f;
            total = wave_sum(total);
        }
    }
    int chosen;
    float mine;                     // the chosen logit, one a lane
    typedef KeyOf<float> Key;
    int key[N], got;
    bool again = false;             // in 64 bits
    if (!A.bias) {
#pragma unroll
        for (int i = 0; i < N; ++i) key[i] = Key::of(l[i]);
        select_top<int, N>(key, l, Key::NO_KEY, A.topk, chosen, got, mine);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            key[i] = l[i] > neg_inf<float>()
                         ? Key::of(score_of<float>(A.scoring, l[i], most, total) + A.bias[i * 64 + lane])
                         : Key::NO_KEY;
        const int more = min(A.topk + 1, 64);
        select_top<int, N>(key, l, Key::NO_KEY, more, chosen, got, mine);
        // fp32's keys are within 4e-6 of the exact ones, relative to what they are made of where that is above one: the
        // key itself, or a score that a bias takes back, of any expert (sqrt(log(1 + e^l)) < 1.4 sqrt(l) from l = 1 on).
        // A key turned back is its number.
        float size = 1.f;
        if (A.scoring == SCORE_SQRTSOFTPLUS) {
#pragma unroll
            for (int i = 0; i < N; ++i) size = fmaxf(size, l[i]);
            size = sqrtf(wave_max(size, 1.f));
        }
        const float here = __int_as_float(got ^ (got >> 31 & 0x7fffffff)), below = __shfl_down(here, 1);
        const bool last = __shfl_down(chosen, 1) < 0;
        const bool near = lane + 1 < more && chosen >= 0 && !last && !(here - below > 0x1p-17f * fmaxf(size, fabsf(here)));
        again = __any(near) || more == A.topk;
        if (lane >= A.topk) chosen = -1;
    }
    double dtotal = 0.0;
    if (A.scoring == SCORE_SOFTMAX && (again || !A.renormalize)) {
#pragma unroll
        for (int i = 0; i < N; ++i) dtotal += l[i] > neg_inf<float>() ? exp((double)l[i] - (double)most) : 0.0;
        dtotal = wave_sum(dtotal);
    }
    if (again) {
        typedef KeyOf<double> Key64;
        long dkey[N], unused;
#pragma unroll
        for (int i = 0; i < N; ++i)
            dkey[i] = l[i] > neg_inf<float>()
                          ? Key64::of(score_of<double>(A.scoring, (double)l[i], (double)most, dtotal) +
                                      (double)A.bias[i * 64 + lane])
                          : Key64::NO_KEY;
        select_top<long, N>(dkey, l, Key64::NO_KEY, A.topk, chosen, unused, mine);
    }
    double s = 0.0;
    if (A.scoring == SCORE_SOFTMAX) {
        // over their own sum only ratios count: from the largest chosen logit they cannot all underflow
        const float top = over_row && !A.renormalize ? most : wave_max(chosen >= 0 ? mine : neg_inf<float>(), neg_inf<float>());
        if (chosen >= 0) s = exp((double)mine - (double)top) / (A.renormalize ? 1.0 : dtotal);
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
