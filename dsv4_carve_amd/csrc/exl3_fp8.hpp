// Block-scaled 8-bit floats for gfx950: rows quantized in groups of 128 values,
// and the product of such rows with a matrix that has a scale for each 128x128
// block.
//
//   quantize   a = max(max|x|, 448 * 2^-126) over a group, scale = a / 448,
//              q = e4m3(448 x / a), ties to even
//   product    c[i][j] = sum_b sa[i][b] * sw[j / 128][b] * sum_{k in block b} a[i][k] * w[j][k]
//
// A block of 128 is four 16x16x32 instructions on values widened to 16 bits
// (exactly) into a cleared accumulator, whose result is scaled into the running
// sums (fp32) by one multiply-add a value.  Both operands give a lane 32 of the
// block's bytes, and a sum does not care which: lane l takes bytes
// [16g, 16g + 16) and [64 + 16g, 64 + 16g + 16) of row l % 16, g = l / 16, so that
// four lanes read 64 bytes of a row together.  The weight is the instruction's
// row operand: a lane's four results are then four neighbouring outputs of one
// row of a, under one scale.
//
// The 8-bit instruction (16x16x128, a block in one) is twice as fast, but cuts
// each product to a multiple of 2^-13 of the largest power of two among its group
// of eight before it adds them: 1e-5 of the result in the 2-norm on normal
// values, where the 16-bit one is at 3e-8.
#pragma once

#include "exl3_decode.hpp"
#include "exl3_capi_util.hpp"

namespace exl3 {

typedef int int8x32_t __attribute__((ext_vector_type(8)));      // 32 e4m3 values
typedef int i32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));

constexpr int FP8_BLOCK = 128;
constexpr float FP8_MAX = 448.0f;

__device__ __forceinline__ int8x32_t join(i32x4_t lo, i32x4_t hi) {
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));

template <bool BF16>
struct Half16 {
    typedef half8_t vec8;
    static __device__ __forceinline__ float4_t mfma(vec8 a, vec8 b, float4_t c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ vec8 widen(uint32_t lo, uint32_t hi) {
        const f16x2_t p0 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false);
        const f16x2_t p1 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true);
        const f16x2_t p2 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false);
        const f16x2_t p3 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true);
        return vec8{p0[0], p0[1], p1[0], p1[1], p2[0], p2[1], p3[0], p3[1]};
    }
    static __device__ __forceinline__ uint16_t bits(float f) { return f32_to_f16_bits(f); }
};

template <>
struct Half16<true> {
    typedef bf16x8_t vec8;
    static __device__ __forceinline__ float4_t mfma(vec8 a, vec8 b, float4_t c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ vec8 widen(uint32_t lo, uint32_t hi) {
        const bf16x2_t p0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false);
        const bf16x2_t p1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true);
        const bf16x2_t p2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false);
        const bf16x2_t p3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true);
        return vec8{p0[0], p0[1], p1[0], p1[1], p2[0], p2[1], p3[0], p3[1]};
    }
    static __device__ __forceinline__ uint16_t bits(float f) { return f32_to_bf16_rne(f); }
};

// A lane's 32 weights of one block (two 16-byte loads, as in exl3_fp8.hpp) and the inputs at the same k.
template <typename H>
struct BlockW {
    typename H::vec8 v[4];
    __device__ __forceinline__ explicit BlockW(const int8x32_t& q) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = H::widen((uint32_t)q[2 * i], (uint32_t)q[2 * i + 1]);
    }
};

template <typename H>
struct BlockX {
    typename H::vec8 v[4];
    __device__ __forceinline__ void load(const uint16_t* p, int g) {      // p: the block's first input
        const typename H::vec8* lo = reinterpret_cast<const typename H::vec8*>(p + 16 * g);
        const typename H::vec8* hi = reinterpret_cast<const typename H::vec8*>(p + 64 + 16 * g);
        v[0] = lo[0];
        v[1] = lo[1];
        v[2] = hi[0];
        v[3] = hi[1];
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = typename H::vec8{};
    }
};

template <typename H, typename X>
__device__ __forceinline__ float4_t block_product(const BlockW<H>& w, const X& x) {
    float4_t p = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; ++i) p = H::mfma(w.v[i], x.v[i], p);
    return p;
}

// One value of kind K as fp32.
template <int K>
__device__ __forceinline__ float load_kind(const void* p, int64_t i) {
    if constexpr (K == OUT_F32) return static_cast<const float*>(p)[i];
    const uint16_t h = static_cast<const uint16_t*>(p)[i];
    return K == OUT_BF16 ? bf16_to_f32(h) : f16_bits_to_f32(h);
}

// ---------------------------------------------------------------- quantization

// What a group's largest magnitude makes of its values.  448 x / a is the
// quotient correctly rounded: with a = b * 2^e, 1 <= b < 2, n = x * (448 * 2^-e)
// is exact for a 16-bit x, and n / b follows from the reciprocal of b with one
// correction of the remainder (Markstein), three operations a value in place of
// a division's ten.  It matters because quotients on a rounding border of e4m3
// are common (the scale and the values have few bits each): a multiplication by
// 448 / a alone rounds some of them the wrong way.
struct QuantGroup {
    float mul, b, r, scale;
    bool pow2;

    __device__ __forceinline__ QuantGroup(float most, bool pow2_) : pow2(pow2_) {
        const float a = fmaxf(most, FP8_MAX * 0x1p-126f);
        const uint32_t bits = __float_as_uint(a);
        const int e = (int)(bits >> 23) - 127;
        const uint32_t frac = bits & 0x7fffffu;
        const bool inf = e == 128;
        if (pow2) {
            const int s = e - 8 + (frac > 0x600000u ? 1 : 0);      // 448 = 1.75 * 2^8
            scale = inf ? a : __uint_as_float((uint32_t)(s + 127) << 23);
            mul = inf ? 0.f : __uint_as_float((uint32_t)(127 - s) << 23);
            b = r = 0.f;
        } else {
            scale = a / FP8_MAX;
            mul = __uint_as_float(((uint32_t)(127 + 8 - e) << 23) | 0x600000u);
            b = inf ? 0.f : __uint_as_float(frac | 0x3f800000u);
            r = inf ? 0.f : 1.0f / b;
        }
    }

    __device__ __forceinline__ float operator()(float x) const {
        const float n = x * mul;
        if (pow2) return n;
        const float q = n * r;
        return fmaf(fmaf(-q, b, n), r, q);
    }
};

__device__ __forceinline__ uint32_t pack_e4m3(float a, float b, float c, float d) {
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false), true);
}

// Sixteen values of kind K (16-byte aligned) as fp32.
template <int K>
__device__ __forceinline__ void load16(const void* p, float (&v)[16]) {
    if constexpr (K == OUT_F32) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float4_t f = static_cast<const float4_t*>(p)[i];
#pragma unroll
            for (int j = 0; j < 4; ++j) v[4 * i + j] = f[j];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const u32x4_t u = static_cast<const u32x4_t*>(p)[i];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                v[8 * i + 2 * j] = K == OUT_BF16 ? __uint_as_float(u[j] << 16) : f16_bits_to_f32((uint16_t)u[j]);
                v[8 * i + 2 * j + 1] =
                    K == OUT_BF16 ? __uint_as_float(u[j] & 0xffff0000u) : f16_bits_to_f32((uint16_t)(u[j] >> 16));
            }
        }
    }
}

// Rows of a multiple of 16 values, 16-byte aligned: a lane has 16 neighbouring
// values, eight lanes a group.
template <int K, bool POW2>
__global__ __launch_bounds__(256) void fp8_quantize_kernel(const void* __restrict__ x, int64_t rows, int k, int groups,
                                                           uint8_t* __restrict__ q, float* __restrict__ scale) {
    const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const uint32_t chunks = (uint32_t)groups * 8;
    const int64_t row = t / chunks;
    const int c = (int)(t - row * chunks);
    const bool in = row < rows && c * 16 < k;
    float v[16];
    float most = 0.f;
    const int64_t at = row * k + c * 16;
    if (in) {
        load16<K>(static_cast<const char*>(x) + at * (K == OUT_F32 ? 4 : 2), v);
#pragma unroll
        for (int i = 0; i < 16; ++i) most = fmaxf(most, fabsf(v[i]));
    }
#pragma unroll
    for (int d = 1; d < 8; d <<= 1) most = fmaxf(most, __shfl_xor(most, d));
    if (!in) return;
    const QuantGroup g(most, POW2);
    if ((c & 7) == 0) scale[row * groups + (c >> 3)] = g.scale;
    u32x4_t out;
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = pack_e4m3(g(v[4 * i]), g(v[4 * i + 1]), g(v[4 * i + 2]), g(v[4 * i + 3]));
    *reinterpret_cast<u32x4_t*>(q + at) = out;
}

// Any row length and alignment: a wave for each group, two values a lane.
template <int K, bool POW2>
__global__ __launch_bounds__(256) void fp8_quantize_any_kernel(const void* __restrict__ x, int64_t rows, int k,
                                                               int groups, uint8_t* __restrict__ q,
                                                               float* __restrict__ scale) {
    const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int64_t row = w / groups;
    if (row >= rows) return;
    const int g = (int)(w - row * groups), lane = threadIdx.x & 63;
    const int i0 = g * FP8_BLOCK + lane, i1 = i0 + 64;
    const float v0 = i0 < k ? load_kind<K>(x, row * k + i0) : 0.f;
    const float v1 = i1 < k ? load_kind<K>(x, row * k + i1) : 0.f;
    float most = fmaxf(fmaxf(0.f, fabsf(v0)), fabsf(v1));
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) most = fmaxf(most, __shfl_xor(most, d));
    const QuantGroup gr(most, POW2);
    if (lane == 0) scale[row * groups + g] = gr.scale;
    const uint32_t u = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(gr(v0), gr(v1), 0, false);
    if (i0 < k) q[row * k + i0] = (uint8_t)u;
    if (i1 < k) q[row * k + i1] = (uint8_t)(u >> 8);
}

// ---------------------------------------------------------------- product, few rows

// Four neighbouring outputs of one row, n0 % 4 == 0.
__device__ __forceinline__ void store_out4(void* c, int kind, int64_t row, int64_t n, int n0, const float (&v)[4],
                                           bool whole) {
    const int64_t at = row * n + n0;
    if (kind == OUT_F32) {
        float* p = static_cast<float*>(c) + at;
        if (whole) {
            *reinterpret_cast<float4_t*>(p) = float4_t{v[0], v[1], v[2], v[3]};
        } else {
            for (int i = 0; i < 4 && n0 + i < n; ++i) p[i] = v[i];
        }
        return;
    }
    uint16_t h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = kind == OUT_BF16 ? f32_to_bf16_rne(v[i]) : f32_to_f16_bits(v[i]);
    uint16_t* p = static_cast<uint16_t*>(c) + at;
    if (whole) {
        *reinterpret_cast<u32x2_t*>(p) = u32x2_t{h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16};
    } else {
        for (int i = 0; i < 4 && n0 + i < n; ++i) p[i] = h[i];
    }
}

// A lane's 32 bytes of block kb of a row of k bytes (k % 16 == 0); bytes past k are zero.
__device__ __forceinline__ int8x32_t load_block(const uint8_t* row, int kb, int g, int k) {
    const i32x4_t zero = {0, 0, 0, 0};
    const int c0 = kb * FP8_BLOCK + g * 16, c1 = c0 + 64;
    const i32x4_t lo = c0 < k ? *reinterpret_cast<const i32x4_t*>(row + c0) : zero;
    const i32x4_t hi = c1 < k ? *reinterpret_cast<const i32x4_t*>(row + c1) : zero;
    return join(lo, hi);
}

// A workgroup has 16 outputs of 16 MT rows; its waves take every WAVES-th block
// of k, with both operands straight from memory to registers, and their sums are
// joined in LDS in the order of the waves.
template <int MT, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void fp8_gemm_rows_kernel(const uint8_t* __restrict__ a,
                                                                   const float* __restrict__ a_scale, int64_t m, int k,
                                                                   const uint8_t* __restrict__ w,
                                                                   const float* __restrict__ w_scale, int n,
                                                                   void* __restrict__ c, int c_kind) {
    __shared__ float part[WAVES][MT * 4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int r = lane & 15, g = lane >> 4;
    const int n0 = blockIdx.x * 16;
    const int64_t m0 = (int64_t)blockIdx.y * 16 * MT;
    const int blocks = (k + FP8_BLOCK - 1) / FP8_BLOCK;
    const uint8_t* wr = w + (int64_t)min(n0 + r, n - 1) * k;
    const float* ws = w_scale + (int64_t)(n0 / FP8_BLOCK) * blocks;
    const uint8_t* ar[MT];
    const float* as[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int64_t row = m0 + 16 * t + r < m ? m0 + 16 * t + r : m - 1;
        ar[t] = a + row * k;
        as[t] = a_scale + row * blocks;
    }
    float acc[MT][4] = {};
#pragma unroll 2
    for (int kb = wave; kb < blocks; kb += WAVES) {
        const BlockW<Half16<true>> wv(load_block(wr, kb, g, k));
        const float s = ws[kb];
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const float4_t p = block_product<Half16<true>>(wv, BlockW<Half16<true>>(load_block(ar[t], kb, g, k)));
            const float sc = s * as[t][kb];
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[t][i] = fmaf(p[i], sc, acc[t][i]);
        }
    }
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) part[wave][4 * t + i][lane] = acc[t][i];
    __syncthreads();
    for (int t = wave; t < MT; t += WAVES) {
        float v[4] = {};
#pragma unroll
        for (int s = 0; s < WAVES; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] += part[s][4 * t + i][lane];
        const int64_t row = m0 + 16 * t + r;
        const int nn = n0 + 4 * g;
        if (row < m && nn < n) store_out4(c, c_kind, row, n, nn, v, n % 4 == 0);
    }
}

}  // namespace exl3
