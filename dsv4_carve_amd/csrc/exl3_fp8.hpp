// Block-scaled 8-bit floats for gfx950: rows quantized in groups of 128 values,
// and the product of such rows with a matrix that has a scale for each 128x128
// block.
//
//   quantize   a = max(max|x|, 448 * 2^-126) over a group, scale = a / 448,
//              q = e4m3(448 x / a), ties to even
//   product    c[i][j] = sum_b sa[i][b] * sw[j / 128][b] * sum_{k in block b} a[i][k] * w[j][k]
//
// A block of 128 goes through the matrix unit into a cleared accumulator, whose
// result is scaled into the running sums (fp32) by one multiply-add a value.  Both
// operands give a lane 32 of the block's bytes, and a sum does not care which:
// lane l takes bytes [16g, 16g + 16) and [64 + 16g, 64 + 16g + 16) of row l % 16,
// g = l / 16, so that four lanes read 64 bytes of a row together.  The weight is
// the instruction's row operand: a lane's four results are then four
// neighbouring outputs of one row of a, under one scale.
//
// The instruction is the 16-bit one (16x16x32, four a block) on values widened
// exactly, so that sums are fp32's.  The 8-bit one (16x16x128, a block in one) is
// twice as fast and is not used: it cuts each product to a multiple of 2^-13 of
// the largest power of two among its group of eight before it adds them, which a
// result that cancels feels far more than its own rounding.
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

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// A wave-uniform lane's value of 4 or 8 bytes.
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
};

// A lane's 32 e4m3 values of one block (two 16-byte loads) and 16-bit inputs at the same k.
template <typename H>
struct BlockW {
    typename H::vec8 v[4];
    BlockW() = default;
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
};

template <typename H, typename X>
__device__ __forceinline__ float4_t block_product(const BlockW<H>& w, const X& x, float4_t p = {0.f, 0.f, 0.f, 0.f}) {
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
// values, eight lanes a group.  Memory bounds it: 8000 x 4096 fp16 15.9 us, 6.2 TB/s
// read and written; 13 rows are a launch's 2.9 us.
template <int K, bool POW2>
__global__ __launch_bounds__(256) void fp8_quantize_kernel(const void* __restrict__ x, int64_t rows, int k, int groups,
                                                           uint8_t* __restrict__ q, float* __restrict__ scale) {
    const uint32_t chunks = (uint32_t)groups * 8;
    const uint32_t t = blockIdx.x * 256 + threadIdx.x, in_rows = t / chunks;        // fewer than 2^32 threads a launch
    const int64_t row = in_rows;
    const int c = (int)(t - in_rows * chunks);
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

// Any row length and alignment: a wave for each group, two values a lane, whose
// loads of two or four bytes bound it.
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

// Two values rounded to bf16 in one instruction (ties to even, a NaN stays one).
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    return __builtin_bit_cast(uint32_t, bf16x2_t{(__bf16)a, (__bf16)b});
}

// Four neighbouring outputs of one row, n0 % 4 == 0; whole: all four are in the row, and their place is aligned.
template <int KIND>
__device__ __forceinline__ void store_out4(void* c, int64_t row, int64_t n, int n0, const float (&v)[4], bool whole) {
    const int64_t at = row * n + n0;
    if constexpr (KIND == OUT_F32) {
        float* p = static_cast<float*>(c) + at;
        if (whole) {
            *reinterpret_cast<float4_t*>(p) = float4_t{v[0], v[1], v[2], v[3]};
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (n0 + i < n) p[i] = v[i];
        }
    } else {
        uint32_t h[2];
#pragma unroll
        for (int i = 0; i < 2; ++i)
            h[i] = KIND == OUT_BF16 ? pack_bf16(v[2 * i], v[2 * i + 1])
                                    : f32_to_f16_bits(v[2 * i]) | (uint32_t)f32_to_f16_bits(v[2 * i + 1]) << 16;
        uint16_t* p = static_cast<uint16_t*>(c) + at;
        if (whole) {
            *reinterpret_cast<u32x2_t*>(p) = u32x2_t{h[0], h[1]};
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (n0 + i < n) p[i] = (uint16_t)(h[i >> 1] >> (16 * (i & 1)));
        }
    }
}

// f with the output kind as a constant.
template <typename F>
__device__ __forceinline__ void with_kind(int kind, F&& f) {
    if (kind == OUT_BF16) f(std::integral_constant<int, OUT_BF16>{});
    else if (kind == OUT_F16) f(std::integral_constant<int, OUT_F16>{});
    else f(std::integral_constant<int, OUT_F32>{});
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
// of k, with both operands straight from memory to registers and through the
// 16-bit instruction, and their sums are joined in LDS in the order of the waves.
// Latency bounds it: 2 rows x 1536 x 4096 3.9 us, 1 row x 4096 x 4096 4.9 us (3.4
// TB/s of weights).
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
        if (row < m && nn < n)
            with_kind(c_kind, [&](auto kind) { store_out4<kind()>(c, row, n, nn, v, n % 4 == 0); });
    }
}

// A few rows (16 at most) of kind K, quantized on the way: the workgroup
// quantizes them whole into LDS, as fp8_quantize does, while its first weights are
// on their way, and has 16 outputs of them.  LDS holds a row's blocks (zeros past
// k) and 64 bytes more, so that four rows' chunks lie in different banks, then the
// scales.  1 row x 4096 x 4096 5.5 to 6.3 us (2.7 to 3.1 TB/s of weights): the first
// loads' latency and the row's way through LDS.
constexpr int FP8_LINEAR_WAVES = 8;
constexpr int FP8_LINEAR_DEEP = 4;                // blocks of a wave on their way

__host__ __device__ inline int fp8_linear_rows_lds(int m, int k) {
    const int blocks = (k + FP8_BLOCK - 1) / FP8_BLOCK, rows = m * (blocks * FP8_BLOCK + 64 + blocks * 4);
    const int sums = FP8_LINEAR_WAVES * 64 * 16;
    return rows > sums ? rows : sums;
}

template <int K>
__global__ __launch_bounds__(FP8_LINEAR_WAVES * 64) void fp8_linear_rows_kernel(const void* __restrict__ x, int m, int k,
                                                                                const uint8_t* __restrict__ w,
                                                                                const float* __restrict__ w_scale,
                                                                                int n, void* __restrict__ c, int c_kind) {
    typedef Half16<true> H;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int r = lane & 15, g = lane >> 4;
    const int n0 = blockIdx.x * 16, blocks = (k + FP8_BLOCK - 1) / FP8_BLOCK, stride = blocks * FP8_BLOCK + 64;
    const uint8_t* wr = w + (int64_t)min(n0 + r, n - 1) * k;
    const float* ws = w_scale + (int64_t)(n0 / FP8_BLOCK) * blocks;
    float* const scales = reinterpret_cast<float*>(lds + m * stride);        // [m][blocks]
    int8x32_t wq[FP8_LINEAR_DEEP];
    float sw[FP8_LINEAR_DEEP];
#pragma unroll
    for (int d = 0; d < FP8_LINEAR_DEEP; ++d) {
        const int kb = wave + d * FP8_LINEAR_WAVES;
        if (kb < blocks) {
            wq[d] = load_block(wr, kb, g, k);
            sw[d] = ws[kb];
        }
    }
    for (int at = tid; at < m * blocks * 8; at += FP8_LINEAR_WAVES * 64) {    // eight lanes a group: whole groups take part
        const int row = at / (blocks * 8), ch = at - row * (blocks * 8);
        float v[16] = {};
        float most = 0.f;
        if (ch * 16 < k) {
            load16<K>(static_cast<const char*>(x) + ((int64_t)row * k + ch * 16) * (K == OUT_F32 ? 4 : 2), v);
#pragma unroll
            for (int i = 0; i < 16; ++i) most = fmaxf(most, fabsf(v[i]));
        }
#pragma unroll
        for (int d = 1; d < 8; d <<= 1) most = fmaxf(most, __shfl_xor(most, d));
        const QuantGroup q(most, false);
        if ((ch & 7) == 0) scales[row * blocks + (ch >> 3)] = q.scale;
        u32x4_t out;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            out[i] = ch * 16 < k ? pack_e4m3(q(v[4 * i]), q(v[4 * i + 1]), q(v[4 * i + 2]), q(v[4 * i + 3])) : 0u;
        *reinterpret_cast<u32x4_t*>(lds + row * stride + ch * 16) = out;
    }
    __syncthreads();
    float acc[4] = {};
    const char* ar = lds + min(r, m - 1) * stride;
    const float* as = scales + min(r, m - 1) * blocks;
    for (int base = wave; base < blocks; base += FP8_LINEAR_DEEP * FP8_LINEAR_WAVES) {
#pragma unroll
        for (int d = 0; d < FP8_LINEAR_DEEP; ++d) {
            const int kb = base + d * FP8_LINEAR_WAVES, ahead = kb + FP8_LINEAR_DEEP * FP8_LINEAR_WAVES;
            if (kb >= blocks) break;
            const char* p = ar + kb * FP8_BLOCK + g * 16;
            const BlockW<H> a(join(*reinterpret_cast<const i32x4_t*>(p), *reinterpret_cast<const i32x4_t*>(p + 64)));
            const float4_t pr = block_product<H>(BlockW<H>(wq[d]), a);
            const float s = sw[d] * as[kb];
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[i] = fmaf(pr[i], s, acc[i]);
            if (ahead < blocks) {
                wq[d] = load_block(wr, ahead, g, k);
                sw[d] = ws[ahead];
            }
        }
    }
    __syncthreads();                     // the rows are read: their place takes the waves' sums
    float4_t* const part = reinterpret_cast<float4_t*>(lds);
    part[wave * 64 + lane] = float4_t{acc[0], acc[1], acc[2], acc[3]};
    __syncthreads();
    if (wave) return;
    float v[4] = {};
#pragma unroll
    for (int s = 0; s < FP8_LINEAR_WAVES; ++s) {
        const float4_t p = part[s * 64 + lane];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] += p[i];
    }
    const int nn = n0 + 4 * g;
    if (r < m && nn < n) with_kind(c_kind, [&](auto kind) { store_out4<kind()>(c, r, n, nn, v, n % 4 == 0); });
}

// ---------------------------------------------------------------- product, many rows

// Tiles of BM rows of a and BN rows of w; WM x WN waves share one, KG such sets
// take alternate blocks of k (their sums are joined in LDS at the end).  A step
// is KG blocks, which go from memory straight to LDS, one step ahead.  A row of a
// block is eight 16-byte chunks there, chunk c of row r at place c ^ (r & 7), so
// that eight rows' chunks of one k lie in different banks.
template <int BM, int BN, int WM, int WN, int KG>
struct Fp8Tile {
    static constexpr int SET = WM * WN * 64;              // threads of one set
    static constexpr int THREADS = SET * KG;
    static constexpr int MT = BM / WM / 16, NT = BN / WN / 16;
    static constexpr int NA = BM * 8 / SET, NW = BN * 8 / SET;      // chunks a thread moves in a step
    static constexpr int BUF = (BM + BN) * FP8_BLOCK;     // bytes of a block
    static constexpr int GROUP = KG < 4 ? 8 : 4;          // steps whose scales are staged together
    static constexpr int SCALES = KG * GROUP * (BM + 1);  // values of a group
    static constexpr int NS = (SCALES + THREADS - 1) / THREADS;
    static constexpr int LDS = 2 * KG * BUF + 2 * SCALES * 4;
    static_assert(BM * 8 % SET == 0 && BN * 8 % SET == 0 && SET % 64 == 0, "whole chunks, in rows of eight");
    static_assert(128 % BN == 0, "one block of w's scales");
    static_assert(KG == 1 || BM * BN * 4 * (KG - 1) <= LDS, "the sums are joined in the buffers");
    static_assert(LDS <= 160 * 1024, "LDS of a CU");
};

constexpr int FP8_TILE_MAX_K = 1 << 22;        // 128 rows of k bytes, and a few blocks more, stay below 2^31

// 16 bytes a lane from base + at + step to dst + 16 * lane, zeros where at is OUTSIDE: the buffer has 2^31 bytes, and
// an offset past its end reads as zero.
constexpr uint32_t OUTSIDE = 0x80000000u;
__device__ __forceinline__ void load_to_lds(__amdgpu_buffer_rsrc_t base, char* dst, uint32_t at, int step) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(base, (__attribute__((address_space(3))) void*)dst, 16, (int)at, step, 0, 0);
}

// Until none of this wave's loads and LDS operations is on its way.
__device__ __forceinline__ void wait_loads() { __builtin_amdgcn_s_waitcnt(7 << 4); }

// A workgroup barrier without a wait of its own; the compiler moves no memory access over it.
__device__ __forceinline__ void bare_barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

template <int BM, int BN, int WM, int WN, int KG>
__global__ __launch_bounds__(WM* WN* KG * 64) __attribute__((amdgpu_waves_per_eu(2))) void fp8_gemm_tile_kernel(const uint8_t* __restrict__ a,
                                                                        const float* __restrict__ a_scale, int m, int k,
                                                                        const uint8_t* __restrict__ w,
                                                                        const float* __restrict__ w_scale, int n,
                                                                        void* __restrict__ c, int c_kind, int tiles_m,
                                                                        int tiles_n) {
    typedef Fp8Tile<BM, BN, WM, WN, KG> T;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int tid = threadIdx.x, lane = tid & 63;
    const int set = KG == 1 ? 0 : __builtin_amdgcn_readfirstlane(tid / T::SET), st = tid - set * T::SET;
    const int wv = __builtin_amdgcn_readfirstlane(st >> 6), wm = wv / WN, wn = wv - wm * WN;
    const int r = lane & 15, g = lane >> 4;
    const int blocks = (k + FP8_BLOCK - 1) / FP8_BLOCK, steps = (blocks + KG - 1) / KG;

    // Workgroup i runs on XCD i % 8: neighbouring tiles, in groups of four tile rows, go to one XCD and its L2.
    int tm, tn;
    {
        const int total = tiles_m * tiles_n, xcd = blockIdx.x & 7, per = total / 8, more = total % 8;
        const int at = xcd * per + min(xcd, more) + (blockIdx.x >> 3);
        const int group = at / (4 * tiles_n), in = at - group * 4 * tiles_n, rows = min(4, tiles_m - group * 4);
        tn = in / rows;
        tm = group * 4 + in - tn * rows;
    }
    const int m0 = tm * BM, n0 = tn * BN;

    // this lane's chunks: rows st / 8 + i * SET / 8 of either operand, the chunk whose place is st % 8
    const int cr = st >> 3, cc = (st ^ cr) & 7;
    const __amdgpu_buffer_rsrc_t ta =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(a + (int64_t)m0 * k), 0, 0x7fffffff, 0x27000);
    const __amdgpu_buffer_rsrc_t tw =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(w + (int64_t)n0 * k), 0, 0x7fffffff, 0x27000);
    constexpr int ROWS = T::SET / 8;        // a multiple of eight: a thread's chunks have one place in their rows
    uint32_t oa[T::NA], ow[T::NW];
#pragma unroll
    for (int i = 0; i < T::NA; ++i) oa[i] = (uint32_t)(min(cr + i * ROWS, m - 1 - m0) * k + cc * 16);
#pragma unroll
    for (int i = 0; i < T::NW; ++i) ow[i] = (uint32_t)(min(cr + i * ROWS, n - 1 - n0) * k + cc * 16);
    const auto fetch = [&](int step, int stage) {
        const int at = (step * KG + set) * FP8_BLOCK;
        char* dst = lds + (stage * KG + set) * T::BUF + wv * 1024;
        if (at + FP8_BLOCK <= k) {
#pragma unroll
            for (int i = 0; i < T::NA; ++i) load_to_lds(ta, dst + i * ROWS * FP8_BLOCK, oa[i], at);
#pragma unroll
            for (int i = 0; i < T::NW; ++i) load_to_lds(tw, dst + (BM + i * ROWS) * FP8_BLOCK, ow[i], at);
        } else {            // chunks past the end of k are zeros, and no traffic
            const bool in = at + cc * 16 < k;
#pragma unroll
            for (int i = 0; i < T::NA; ++i) load_to_lds(ta, dst + i * ROWS * FP8_BLOCK, in ? oa[i] : OUTSIDE, at);
#pragma unroll
            for (int i = 0; i < T::NW; ++i) load_to_lds(tw, dst + (BM + i * ROWS) * FP8_BLOCK, in ? ow[i] : OUTSIDE, at);
        }
    };
    // scales of a group of steps as [block][BM rows of a, w's block]; a block past the end has zeros, not a neighbour's
    // value: that may be infinite
    float* const scales = reinterpret_cast<float*>(lds + 2 * KG * T::BUF);
    const auto fetch_scales = [&](float (&v)[T::NS], int first) {
#pragma unroll
        for (int i = 0; i < T::NS; ++i) {
            const int at = tid + i * T::THREADS, row = at / (KG * T::GROUP), b = at - row * (KG * T::GROUP);
            const int kb = min(first * KG + b, blocks - 1);
            const float* p = row < BM ? a_scale + (int64_t)min(m0 + row, m - 1) * blocks
                                      : w_scale + (int64_t)(n0 / FP8_BLOCK) * blocks;
            v[i] = p[kb];
        }
    };
    const auto put_scales = [&](const float (&v)[T::NS], int first) {
        float* p = scales + (first / T::GROUP & 1) * T::SCALES;
#pragma unroll
        for (int i = 0; i < T::NS; ++i) {
            const int at = tid + i * T::THREADS, row = at / (KG * T::GROUP), b = at - row * (KG * T::GROUP);
            if (at < T::SCALES) p[b * (BM + 1) + row] = first * KG + b < blocks ? v[i] : 0.f;
        }
    };

    // this lane's chunks g and g + 4 of row r of its wave's first 16 rows of either operand; the others are at constant
    // distances (the barrier keeps the compiler from folding those into one register each)
    int aa[2], aw[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int at = r * FP8_BLOCK + (((g + 4 * h) ^ (r & 7)) * 16);
        aa[h] = wm * (BM / WM) * FP8_BLOCK + at;
        aw[h] = (BM + wn * (BN / WN)) * FP8_BLOCK + at;
        asm("" : "+v"(aa[h]), "+v"(aw[h]));
    }
    float acc[T::MT][T::NT][4] = {};
    float sv[T::NS];
    fetch_scales(sv, 0);
    fetch(0, 0);
    put_scales(sv, 0);
    // Row groups i = 0 .. LAST of a step, each NT products; a product is read (into its sum) one row group after it
    // began.  A step's last row group is computed after the next step's barrier, while that step's first operands are
    // on their way from LDS.
    constexpr int LAST = T::MT - 1;
    typedef BlockW<Half16<true>> Frag;
    Frag fa = {}, fw[T::NT] = {};
    float4_t p[T::NT] = {};
    float s = 0.f, sw = 0.f, sc = 0.f;      // scales: of fa's rows, of w's block, of the products in p
    const auto sum_up = [&](int i, int j) {
#pragma unroll
        for (int q = 0; q < 4; ++q) acc[i][j][q] = fmaf(p[j][q], sc, acc[i][j][q]);
    };
    for (int step = 0; step < steps; ++step) {
        // this step has come, and every wave is done with the buffer of the one before
        wait_loads();
        bare_barrier();
        // (no branch below these: the compiler would move the sums' updates behind it, and hold every product until there)
        if (step % T::GROUP == 0) fetch_scales(sv, step + T::GROUP);
        if (step % T::GROUP == T::GROUP / 2) put_scales(sv, step + T::GROUP / 2);
        fetch(step + 1, (step + 1) & 1);
        const char* base = lds + ((step & 1) * KG + set) * T::BUF;
        const float* sp = scales + (step / T::GROUP & 1) * T::SCALES + (step % T::GROUP * KG + set) * (BM + 1);
        const auto read = [&](Frag& f, const int (&at)[2], int i) {
            f = Frag(join(*reinterpret_cast<const i32x4_t*>(base + at[0] + i * 16 * FP8_BLOCK),
                          *reinterpret_cast<const i32x4_t*>(base + at[1] + i * 16 * FP8_BLOCK)));
        };
        Frag next;
        read(next, aa, 0);
        const float sw_next = sp[BM];
        sp += wm * (BM / WM) + r;
        float s_next = sp[0];
#pragma unroll
        for (int j = 0; j < T::NT; ++j) {
            if (LAST > 0) sum_up(LAST - 1, j);
            else sum_up(0, j);
            p[j] = block_product(fw[j], fa);
            read(fw[j], aw, j);
            __builtin_amdgcn_sched_barrier(0);
        }
        sc = s * sw;
        fa = next;
        s = s_next;
        sw = sw_next;
#pragma unroll
        for (int i = 0; i < LAST; ++i) {
            read(next, aa, i + 1);
            s_next = sp[16 * (i + 1)];
#pragma unroll
            for (int j = 0; j < T::NT; ++j) {
                sum_up(i ? i - 1 : LAST, j);
                p[j] = block_product(fw[j], fa);
                __builtin_amdgcn_sched_barrier(0);
            }
            sc = s * sw;
            fa = next;
            s = s_next;
        }
    }
#pragma unroll
    for (int j = 0; j < T::NT; ++j) {
        sum_up(LAST > 0 ? LAST - 1 : 0, j);
        p[j] = block_product(fw[j], fa);
    }
    sc = s * sw;
#pragma unroll
    for (int j = 0; j < T::NT; ++j) sum_up(LAST, j);
    wait_loads();                   // the zeros of the steps past the end, before the buffers are used again or given back
    __syncthreads();
    if constexpr (KG > 1) {
        float4_t* sums = reinterpret_cast<float4_t*>(lds);
#pragma unroll
        for (int s = 1; s < KG; ++s) {
            if (set == s)
#pragma unroll
                for (int i = 0; i < T::MT; ++i)
#pragma unroll
                    for (int j = 0; j < T::NT; ++j)
                        sums[((s - 1) * T::MT * T::NT + i * T::NT + j) * T::SET + st] =
                            float4_t{acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]};
        }
        __syncthreads();
        if (set) return;
#pragma unroll
        for (int s = 1; s < KG; ++s)
#pragma unroll
            for (int i = 0; i < T::MT; ++i)
#pragma unroll
                for (int j = 0; j < T::NT; ++j) {
                    const float4_t o = sums[((s - 1) * T::MT * T::NT + i * T::NT + j) * T::SET + st];
#pragma unroll
                    for (int q = 0; q < 4; ++q) acc[i][j][q] += o[q];
                }
    }
    const bool whole = n % 4 == 0, inside = whole && m0 + BM <= m && n0 + BN <= n;
    const int row0 = m0 + wm * (BM / WM) + r, col0 = n0 + wn * (BN / WN) + 4 * g;
    with_kind(c_kind, [&](auto kind) {
        if (inside) {
#pragma unroll
            for (int i = 0; i < T::MT; ++i)
#pragma unroll
                for (int j = 0; j < T::NT; ++j)
                    store_out4<kind()>(c, row0 + 16 * i, n, col0 + 16 * j, acc[i][j], true);
        } else {
#pragma unroll
            for (int i = 0; i < T::MT; ++i)
#pragma unroll
                for (int j = 0; j < T::NT; ++j)
                    if (row0 + 16 * i < m && col0 + 16 * j < n)
                        store_out4<kind()>(c, row0 + 16 * i, n, col0 + 16 * j, acc[i][j], whole);
        }
    });
}

}  // namespace exl3
