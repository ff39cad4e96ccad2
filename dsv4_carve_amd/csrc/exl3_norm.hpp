// The residual's addition and the root-mean-square norm in front of a
// block-scaled product:
//
//   h = x + residual,  r = 1 / sqrt(mean(h^2) + eps),  y = h r w,
//   groups of 128 of y: a = max(max|y|, 448 * 2^-126), scale = a / 448, q = e4m3(448 y / a)
//
// y / a is (h w) / max|h w|: r cancels, and quotients of few-bit values that lie on
// a rounding border of e4m3 stay on it.  Everything between the inputs and the
// roundings is 64-bit: a quotient in fp32 rounds about one value in 2^18 to the
// other side of a border.  Most values are nowhere near one, though: an fp32 quotient
// whose both neighbours at its error's distance have the same code has that code, and
// only a wave that holds another value divides in 64 bits (SURE).
//
// y in 16 bits goes by way of fp32: 2^-14 (fp16) and 2^-17 (bf16) of its values, next to
// a border, round to the other side of it, by half a step and 2^-24.  Rounded once, 8000
// rows of 4096 with y took 56 us instead of 53 and 333 rows of 1536 4.2 instead of 3.85.
#pragma once

#include "exl3_fp8.hpp"
#include "exl3_topk.hpp"

namespace exl3 {

struct NormArgs {
    const void* x;
    const void* residual;        // fp16, bf16 or fp32 by a kernel's R; null without one
    const void* weight;
    int weight_kind;
    int64_t rows;
    int k, groups;
    double eps, inverse_k;
    bool pow2;
    uint8_t* q;
    float* scale;
    void* sum;                   // h in the residual's type; null without one
    void* normed;                // y, or null
    int normed_kind;
};

constexpr int NO_RESIDUAL = -1;

// What a group's largest |h w| makes of its values g = h w.
struct NormGroup {
    double mul, b;
    float scale;
    bool small;

    // most: the group's largest |g| (NaN left out); r: the row's factor
    __device__ __forceinline__ NormGroup(double most, double r, bool finite, bool pow2) {
        constexpr double LEAST = 448.0 * 0x1p-126;
        const double top = most * r;
        small = !(top > LEAST) || !finite;
        const double a = small ? LEAST : top;
        b = 1.0;
        if (pow2) {
            const uint64_t bits = __builtin_bit_cast(uint64_t, a);
            const int e = (int)(bits >> 52) - 1023 - 8 + ((bits & 0xfffffffffffffull) > 0xc000000000000ull ? 1 : 0);
            scale = ldexpf(1.0f, e);                               // 448 = 1.75 * 2^8
            mul = ldexp(r, -e);
        } else {
            scale = (float)(a / 448.0);
            mul = small ? r * 0x1p126 : 448.0;
            b = small ? 1.0 : most;
        }
        if (!finite) mul = r;                                      // 0 for finite values, NaN for the others
    }
};

// A group's values over its scale, correctly rounded (one correction of the remainder).
struct NormDivide {
    double mul, b, rb;

    __device__ __forceinline__ explicit NormDivide(const NormGroup& g) : mul(g.mul), b(g.b), rb(1.0 / g.b) {}
    __device__ __forceinline__ double operator()(double g) const {
        const double n = g * mul;
        const double q = n * rb;
        return fma(fma(-q, b, n), rb, q);
    }
};

// Bound of an fp32 quotient's relative error, in halves of a last bit: 1 of g, 1 of the largest, 2 of its reciprocal, 1
// of that times 448, 1 of the product and 1 of the neighbour make 7 of these 8.
constexpr float SURE = 0x1p-21f;

// 1 / sqrt(x), to the last bit or two: two steps of Newton's from the hardware's estimate.
__device__ __forceinline__ double inverse_root(double x) {
    const double y = __builtin_amdgcn_rsq(x), half = 0.5 * x;
    double z = fma(y, fma(-half * y, y, 0.5), y);
    z = fma(z, fma(-half * z, z, 0.5), z);
    return x > 0.0 && x < __builtin_inf() ? z : y;
}

template <int N>
__device__ __forceinline__ void store_kind(void* p, int kind, int64_t at, const double (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float f = (float)v[i];
        if (kind == OUT_F32) static_cast<float*>(p)[at + i] = f;
        else static_cast<uint16_t*>(p)[at + i] = kind == OUT_BF16 ? (uint16_t)pack_bf16(f, f) : f32_to_f16_bits(f);
    }
}

// Sixteen neighbouring values, 16-byte aligned.
template <int KIND>
__device__ __forceinline__ void store16(void* p, int64_t at, const float (&v)[16]) {
    if constexpr (KIND == OUT_F32) {
        float4_t* o = reinterpret_cast<float4_t*>(static_cast<float*>(p) + at);
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = float4_t{v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]};
    } else {
        u32x4_t* o = reinterpret_cast<u32x4_t*>(static_cast<uint16_t*>(p) + at);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            u32x4_t u;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float a = v[8 * i + 2 * j], b = v[8 * i + 2 * j + 1];
                u[j] = KIND == OUT_BF16 ? pack_bf16(a, b) : f32_to_f16_bits(a) | (uint32_t)f32_to_f16_bits(b) << 16;
            }
            o[i] = u;
        }
    }
}

__device__ __forceinline__ void load16_any(const void* p, int kind, int64_t at, float (&v)[16]) {
    if (kind == OUT_F32) load16<OUT_F32>(static_cast<const float*>(p) + at, v);
    else if (kind == OUT_BF16) load16<OUT_BF16>(static_cast<const uint16_t*>(p) + at, v);
    else load16<OUT_F16>(static_cast<const uint16_t*>(p) + at, v);
}

// Rows of a multiple of 16 values up to 1024 * WAVES * CHUNKS, 16-byte aligned: WAVES
// waves have a row, a lane 16 neighbouring values in each of CHUNKS pieces, held
// in registers from the sum to the quotients.  Bound by memory where rows are many
// (8000 rows of 4096 in bf16 with a residual: 42.4 us, 5.4 TB/s; all quotients in 64
// bits 52.6, of instructions), by one chain of loads, sum and stores where they are few
// (1 row: 3.2 us).
template <int X, int R, int WAVES, int CHUNKS>
__global__ __launch_bounds__(256) void fp8_norm_kernel(NormArgs A) {
    __shared__ double part[4];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * (4 / WAVES) + wave / WAVES;
    const int k = WAVES == 4 || row < A.rows ? A.k : 0;             // nothing for the waves behind the last row
    const int t = (wave % WAVES) * 64 + lane;
    const int64_t at = row * A.k;
    float h0[CHUNKS][16], h1[CHUNKS][R == NO_RESIDUAL ? 1 : 16];
    double sum = 0.0;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
        const int i = (c * WAVES * 64 + t) * 16;
        if (i < k) {
            load16<X>(static_cast<const char*>(A.x) + (at + i) * (X == OUT_F32 ? 4 : 2), h0[c]);
            if constexpr (R != NO_RESIDUAL)
                load16<R>(static_cast<const char*>(A.residual) + (at + i) * (R == OUT_F32 ? 4 : 2), h1[c]);
        } else {
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                h0[c][j] = 0.f;
                if constexpr (R != NO_RESIDUAL) h1[c][j] = 0.f;
            }
        }
    }
    const auto value = [&](int c, int j) {
        if constexpr (R == NO_RESIDUAL) return (double)h0[c][j];
        else return (double)h0[c][j] + (double)h1[c][j];
    };
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const double h = value(c, j);
            sum = fma(h, h, sum);
        }
    sum = wave_sum(sum);
    if constexpr (WAVES > 1) {
        if (lane == 0) part[wave] = sum;
        __syncthreads();
        const int first = wave / WAVES * WAVES;
        sum = part[first];
#pragma unroll
        for (int i = 1; i < WAVES; ++i) sum += part[first + i];
    }
    const double r = inverse_root(fma(sum, A.inverse_k, A.eps));
    const bool finite = sum < __builtin_inf() && r < __builtin_inf();
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
        const int i = (c * WAVES * 64 + t) * 16;
        const bool in = i < k;
        double most = 0.0;
        float w[16] = {}, g[16] = {};                                   // g: h w in 32 bits
        if (in) {
            load16_any(A.weight, A.weight_kind, i, w);
            if constexpr (R != NO_RESIDUAL) {
                float h[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) h[j] = h0[c][j] + h1[c][j];
                store16<R>(A.sum, at + i, h);
            }
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const double v = value(c, j) * (double)w[j];
                most = fmax(most, fabs(v));
                g[j] = (float)v;
            }
        }
        most = fmax(most, __shfl_xor(most, 1));
        most = fmax(most, __shfl_xor(most, 2));
        most = fmax(most, __shfl_xor(most, 4));
        const NormGroup group(most, r, finite, A.pow2);
        u32x4_t out = {0, 0, 0, 0}, differ = {0, 0, 0, 0};
        if (in) {
            if ((lane & 7) == 0) A.scale[row * A.groups + (i >> 7)] = group.scale;
            const bool plain = finite && !group.small && most > 0x1p-100 && most < 0x1p100;
            const float by = A.pow2 ? (float)group.mul : 448.f * __builtin_amdgcn_rcpf((float)most);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float lo[4], hi[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float q = g[4 * j + e] * by;
                    lo[e] = q * (1.f - SURE);
                    hi[e] = q * (1.f + SURE);
                }
                out[j] = pack_e4m3(lo[0], lo[1], lo[2], lo[3]);
                differ[j] = plain ? out[j] ^ pack_e4m3(hi[0], hi[1], hi[2], hi[3]) : ~0u;
            }
        }
        if (__builtin_amdgcn_ballot_w64((differ[0] | differ[1] | differ[2] | differ[3]) != 0)) {
            const NormDivide divide(group);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (!__builtin_amdgcn_ballot_w64(differ[j] != 0)) continue;
                float q[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) q[e] = to_odd(divide(value(c, 4 * j + e) * (double)w[4 * j + e]));
                out[j] = pack_e4m3(q[0], q[1], q[2], q[3]);
            }
        }
        if (!in) continue;
        *reinterpret_cast<u32x4_t*>(A.q + at + i) = out;
        if (A.normed) {
#pragma unroll
            for (int j = 0; j < 16; ++j) g[j] = (float)(value(c, j) * (double)w[j] * r);
            with_kind(A.normed_kind, [&](auto kind) { store16<decltype(kind)::value>(A.normed, at + i, g); });
        }
    }
}

// Any row length and alignment: a workgroup for each row, which is read twice; a
// wave for each group, two values a lane.
template <int X, int R>
__global__ __launch_bounds__(256) void fp8_norm_any_kernel(NormArgs A) {
    __shared__ double part[4];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t row = blockIdx.x, at = row * A.k;
    const auto value = [&](int i) {
        const double h = load_kind<X>(A.x, at + i);
        if constexpr (R == NO_RESIDUAL) return h;
        else return h + (double)load_kind<R>(A.residual, at + i);
    };
    double sum = 0.0;
    for (int i = threadIdx.x; i < A.k; i += 256) {
        const double h = value(i);
        sum = fma(h, h, sum);
    }
    sum = wave_sum(sum);
    if (lane == 0) part[wave] = sum;
    __syncthreads();
    sum = part[0] + part[1] + part[2] + part[3];
    const double r = inverse_root(fma(sum, A.inverse_k, A.eps));
    const bool finite = sum < __builtin_inf() && r < __builtin_inf();
    for (int b = wave; b < A.groups; b += 4) {
        double g[2] = {0.0, 0.0};
        double most = 0.0;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int i = b * FP8_BLOCK + j * 64 + lane;
            if (i < A.k) {
                const double h[1] = {value(i)};
                if constexpr (R != NO_RESIDUAL) store_kind<1>(A.sum, R, at + i, h);
                float w;
                if (A.weight_kind == OUT_F32) w = load_kind<OUT_F32>(A.weight, i);
                else if (A.weight_kind == OUT_BF16) w = load_kind<OUT_BF16>(A.weight, i);
                else w = load_kind<OUT_F16>(A.weight, i);
                g[j] = h[0] * (double)w;
                most = fmax(most, fabs(g[j]));
            }
        }
        most = wave_max(most, 0.0);
        const NormGroup group(most, r, finite, A.pow2);
        if (lane == 0) A.scale[row * A.groups + b] = group.scale;
        const NormDivide divide(group);
        const uint32_t u = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(to_odd(divide(g[0])), to_odd(divide(g[1])), 0, false);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int i = b * FP8_BLOCK + j * 64 + lane;
            if (i < A.k) {
                A.q[at + i] = (uint8_t)(u >> (8 * j));
                if (A.normed) {
                    const double y[1] = {g[j] * r};
                    store_kind<1>(A.normed, A.normed_kind, at + i, y);
                }
            }
        }
    }
}

}  // namespace exl3
