// A paged cache of e4m3 keys and values with one power-of-two scale for each page
// and head, the write into it, and causal attention over it.
//
//   k  [pages][kv][page][dim]   k_scale [pages][kv]
//   v  [pages][kv][dim][page]   v_scale [pages][kv]      (a value's tokens are neighbours)
//
//   s_ij = scale * q_i . k_j for the keys j that query i sees (j <= i, j > i - window)
//   out_i = sum_j e^(s_ij) v_j / (sum_j e^(s_ij) + e^sink),  lse_i = log of that sum
//
// A power of two as the scale keeps a value's bits where the scale of a begun page
// grows (but for those that fall below e4m3's normal range), and e4m3's relative
// error does not depend on where in its range a value lies.
#pragma once

#include "exl3_fp8.hpp"
#include "exl3_topk.hpp"

namespace exl3 {

struct CacheView {
    uint8_t* k;
    float* k_scale;
    uint8_t* v;
    float* v_scale;
    const int* table;            // [seqs][width] pages
    int64_t table_stride;
    const int* lengths;          // [seqs], the new tokens counted
    const int* starts;           // [seqs + 1] first token of each sequence, or null: one token each
    int seqs, tokens, kv, dim, page_shift, width, pages;
};

// A sequence's tokens in a call and its length.  What a table, a length or a start
// names past its range is cut to it: no index leaves a buffer.
struct Seq {
    int first, n, len;
};

__device__ __forceinline__ Seq get_seq(const CacheView& C, int s) {
    Seq q;
    if (C.starts) {
        const int a = C.starts[s], b = C.starts[s + 1];
        q.first = min(max(a, 0), C.tokens);
        q.n = max(min(b, C.tokens) - q.first, 0);
    } else {
        q.first = s;
        q.n = 1;
    }
    const int64_t room = (int64_t)C.width << C.page_shift;
    const int len = max(C.lengths[s], 0);
    q.len = (int64_t)len < room ? len : (int)room;
    return q;
}

// A value that all lanes have alike, known as such to the compiler: control flow and
// addresses that follow from it are scalar.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int64_t uniform(int64_t v) {
    const u32x2_t a = __builtin_bit_cast(u32x2_t, v);
    return __builtin_bit_cast(int64_t, u32x2_t{(uint32_t)uniform((int)a[0]), (uint32_t)uniform((int)a[1])});
}

// Inclusive prefix sums over the wave's lanes.
__device__ __forceinline__ int64_t wave_scan(int64_t v) {
    v += lane_of<0x111, 0xf>(v, (int64_t)0);        // row_shr:1, 2, 4, 8
    v += lane_of<0x112, 0xf>(v, (int64_t)0);
    v += lane_of<0x114, 0xf>(v, (int64_t)0);
    v += lane_of<0x118, 0xf>(v, (int64_t)0);
    v += lane_of<0x142, 0xa>(v, (int64_t)0);        // row_bcast:15, 31
    v += lane_of<0x143, 0xc>(v, (int64_t)0);
    return v;
}

// a / b, 0 <= a, 0 < b; in 32 bits where both fit.
__device__ __forceinline__ int64_t divide(int64_t a, int64_t b) {
    return ((uint64_t)(a | b) >> 32) == 0 ? (int64_t)((uint32_t)a / (uint32_t)b) : a / b;
}

// The sequence that a unit of all sequences' units lies in; count(q) units each.  The
// unit is at(total), total being all of them; s is -1 where it lies behind them.  Every
// wave looks by itself: up to 64 sequences are one load and one scan.
struct Found {
    int s;
    int64_t unit;                // within the sequence
    Seq q;
};

template <typename Count, typename At>
__device__ __forceinline__ Found find_seq(const CacheView& C, Count&& count, At&& at) {
    const int lane = threadIdx.x & 63;
    const Seq none{0, 0, 0};
    Found f{-1, 0, none};
    const auto look = [&](int s0, const Seq& q, int64_t c, int64_t before, int64_t sum, int64_t want) {
        before += sum - c;
        const uint64_t hit = __builtin_amdgcn_ballot_w64(want >= before && want < before + c);
        if (!hit) return;
        const int l = __builtin_ctzll(hit);
        f.s = s0 + l;
        f.unit = want - read_lane(before, l);
        f.q = Seq{read_lane(q.first, l), read_lane(q.n, l), read_lane(q.len, l)};
    };
    if (C.seqs <= 64) {
        const Seq q = lane < C.seqs ? get_seq(C, lane) : none;
        const int64_t c = count(q), sum = wave_scan(c);
        look(0, q, c, 0, sum, at(read_lane(sum, 63)));
    } else {
        int64_t c = 0;
        for (int s = lane; s < C.seqs; s += 64) c += count(get_seq(C, s));
        const int64_t want = at(read_lane(wave_scan(c), 63));
        int64_t before = 0;
        for (int s0 = 0; s0 < C.seqs && want >= before && f.s < 0; s0 += 64) {
            const Seq q = s0 + lane < C.seqs ? get_seq(C, s0 + lane) : none;
            const int64_t n = count(q), sum = wave_scan(n);
            look(s0, q, n, before, sum, want);
            before += read_lane(sum, 63);
        }
    }
    return f;
}

// ---------------------------------------------------------------- the write

constexpr int APPEND_WAVES = 4;

struct AppendArgs {
    CacheView c;
    const void* k;
    const void* v;
    int64_t k_token, k_head, v_token, v_head;          // strides in values
};

// The pages that a sequence's new tokens lie in.
__device__ __forceinline__ int touched_pages(const CacheView& C, const Seq& q) {
    const int from = max(q.len - q.n, 0);
    return q.len > from ? ((q.len - 1) >> C.page_shift) - (from >> C.page_shift) + 1 : 0;
}

// Eight neighbouring values (16-byte aligned) as fp32; an infinity as a NaN.
template <int K>
__device__ __forceinline__ void load8_finite(const void* p, int64_t at, float (&v)[8]) {
    if constexpr (K == OUT_F32) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float4_t f = reinterpret_cast<const float4_t*>(static_cast<const float*>(p) + at)[i];
#pragma unroll
            for (int j = 0; j < 4; ++j) v[4 * i + j] = f[j];
        }
    } else {
        const u32x4_t u = *reinterpret_cast<const u32x4_t*>(static_cast<const uint16_t*>(p) + at);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[2 * j] = K == OUT_BF16 ? __uint_as_float(u[j] << 16) : f16_bits_to_f32((uint16_t)u[j]);
            v[2 * j + 1] = K == OUT_BF16 ? __uint_as_float(u[j] & 0xffff0000u) : f16_bits_to_f32((uint16_t)(u[j] >> 16));
        }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = fabsf(v[j]) == __builtin_inff() ? __builtin_nanf("") : v[j];
}

// Four codes times a power of two, rounded to e4m3 again.
__device__ __forceinline__ uint32_t rescale4(uint32_t u, float by) {
    return pack_e4m3(__builtin_amdgcn_cvt_f32_fp8((int)u, 0) * by, __builtin_amdgcn_cvt_f32_fp8((int)u, 1) * by,
                     __builtin_amdgcn_cvt_f32_fp8((int)u, 2) * by, __builtin_amdgcn_cvt_f32_fp8((int)u, 3) * by);
}

// A workgroup has one page of one head, of the keys or of the values: the new
// tokens' largest magnitude, the scale, the old codes where it grew, the new ones.
// The inputs are read twice (the second time from cache).
template <int K>
__global__ __launch_bounds__(APPEND_WAVES * 64) void fp8_cache_append_kernel(AppendArgs A) {
    __shared__ float most_of[APPEND_WAVES];
    const CacheView& C = A.c;
    const int tid = threadIdx.x, head = blockIdx.y;
    const bool values = blockIdx.z;
    int s = blockIdx.x, nth = 0;
    Seq q;
    if (C.starts) {
        const Found f = find_seq(C, [&](const Seq& x) { return (int64_t)touched_pages(C, x); },
                                 [](int64_t) { return (int64_t)blockIdx.x; });
        if (f.s < 0) return;
        s = f.s;
        nth = (int)f.unit;
        q = f.q;
    } else {
        q = get_seq(C, s);
    }
    const int page = 1 << C.page_shift, base = q.len - q.n, from = max(base, 0);
    if (q.len <= from) return;
    const int at = (from >> C.page_shift) + nth;                                  // the page's place in the sequence
    const int id = C.table[s * C.table_stride + at];
    if ((unsigned)id >= (unsigned)C.pages) return;
    const int lo = max(from - (at << C.page_shift), 0), hi = min(q.len - (at << C.page_shift), page);
    const int64_t token = q.first + (at << C.page_shift) - base;                  // the token of the page's place 0
    const int64_t stride = values ? A.v_token : A.k_token;
    const int64_t in0 = token * stride + head * (values ? A.v_head : A.k_head);
    const void* in = values ? A.v : A.k;
    const int64_t block = (int64_t)id * C.kv + head;
    uint8_t* code = (values ? C.v : C.k) + (block << C.page_shift) * C.dim;
    float* scale = (values ? C.v_scale : C.k_scale) + block;

    const int per = C.dim >> 3;                                                   // chunks of eight a token
    float most = 0.f;
    float x[8];
    for (int i = tid; i < (hi - lo) * per; i += APPEND_WAVES * 64) {
        const int t = i / per;
        load8_finite<K>(in, in0 + (lo + t) * stride + (i - t * per) * 8, x);
#pragma unroll
        for (int j = 0; j < 8; ++j) most = fmaxf(most, fabsf(x[j]));
    }
    most = wave_max(most, 0.f);
    if ((tid & 63) == 0) most_of[tid >> 6] = most;
    const float before = lo ? *scale : 0.f;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < APPEND_WAVES; ++w) most = fmaxf(most, most_of[w]);
    const float now = fmaxf(QuantGroup(most, true).scale, before);
    const float inverse = 1.0f / now, by = before / now;
    const bool grew = lo && by != 1.0f;
    if (!values) {
        if (grew)
            for (int i = tid; i < lo * C.dim / 16; i += APPEND_WAVES * 64) {
                u32x4_t u = reinterpret_cast<u32x4_t*>(code)[i];
#pragma unroll
                for (int j = 0; j < 4; ++j) u[j] = rescale4(u[j], by);
                reinterpret_cast<u32x4_t*>(code)[i] = u;
            }
        for (int i = tid; i < (hi - lo) * per; i += APPEND_WAVES * 64) {
            const int t = i / per, d = (i - t * per) * 8;
            load8_finite<K>(in, in0 + (lo + t) * stride + d, x);
            *reinterpret_cast<u32x2_t*>(code + (lo + t) * C.dim + d) =
                u32x2_t{pack_e4m3(x[0] * inverse, x[1] * inverse, x[2] * inverse, x[3] * inverse),
                        pack_e4m3(x[4] * inverse, x[5] * inverse, x[6] * inverse, x[7] * inverse)};
        }
    } else {
        // 16 tokens of one value's channel at once; what is outside [lo, hi) goes back as it was, or rescaled below lo
        const int first = grew ? 0 : lo >> 4, groups = ((hi + 15) >> 4) - first;
        for (int i = tid; i < groups * C.dim; i += APPEND_WAVES * 64) {
            const int b = i / C.dim, d = i - b * C.dim, t0 = (first + b) * 16;
            u32x4_t* p = reinterpret_cast<u32x4_t*>(code + ((int64_t)d << C.page_shift) + t0);
            u32x4_t u = {0, 0, 0, 0};
            if (t0 < lo || t0 + 16 > hi) u = *p;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t moved = grew ? rescale4(u[j], by) : u[j];
                float y[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int t = t0 + 4 * j + e;
                    const float f = t >= lo && t < hi ? load_kind<K>(in, in0 + t * stride + d) : 0.f;
                    y[e] = (fabsf(f) == __builtin_inff() ? __builtin_nanf("") : f) * inverse;
                }
                const uint32_t made = pack_e4m3(y[0], y[1], y[2], y[3]);
                uint32_t r = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int t = t0 + 4 * j + e;
                    const uint32_t m = 0xffu << (8 * e);
                    r |= m & (t < lo ? moved : t < hi ? made : u[j]);
                }
                u[j] = r;
            }
            *p = u;
        }
    }
    if (tid == 0) *scale = now;
}

// ---------------------------------------------------------------- attention

constexpr int ATTN_WAVES = 4;
constexpr int ATTN_KEYS = 64;                 // keys of a block
constexpr float ATTN_LOW = -3.402823466e+38f; // a row's reference before its first key
constexpr float ATTN_SLACK = 6.f;             // how far a logit may pass the reference (log2) before sums are rescaled
constexpr int ATTN_HEADROOM = 8;              // 16-bit weights are below 2^(SLACK + HEADROOM) < 65504

// A tile that goes on behind the share of the workgroup that begins it.
struct SharedTile {
    int first, r0, rows, head;                // the sequence's first token; the tile's rows within it; the cache head
    int last;                                 // the workgroup of its last unit; -1: there is no such tile
    int unused[3];
};

struct AttnArgs {
    CacheView c;
    const uint16_t* q;
    int64_t q_token, q_head;                  // strides in values
    int heads, group;                         // query heads, and of each cache head
    float qk_scale;                           // |scale| * log2(e)
    bool negative;                            // scale < 0
    int window;                               // 0: none
    const float* sinks;                       // [heads] or null
    uint16_t* out;                            // [tokens][heads][dim]
    float* lse;                               // [tokens][heads] or null
    float* part;                              // partial results of shared tiles, or null: a workgroup a tile
    SharedTile* shared;                       // a workgroup's shared tile
    int tiles;                                // tiles at most
    int least;                                // units that a workgroup has at least
    bool clear;                               // rows that no sequence has are zeroed
};

// Rows of a tile: ROWS neighbouring (query, head of the group) pairs of one sequence and cache head.
struct Tile {
    int r0, rows;                             // rows within the sequence, and how many there are
    int lo, hi;                               // keys that some row sees
    int full_lo, full_hi;                     // keys that every row sees
};

__device__ __forceinline__ Tile get_tile(const AttnArgs& A, const Seq& q, int t, int ROWS) {
    Tile x;
    x.r0 = t * ROWS;
    x.rows = min(ROWS, q.n * A.group - x.r0);
    const int base = q.len - q.n;
    const int qa = x.r0 / A.group, qb = (x.r0 + x.rows - 1) / A.group;
    x.hi = min(max(base + qb + 1, 0), q.len);
    x.full_hi = max(base + qa + 1, 0);
    x.lo = x.full_lo = 0;
    if (A.window) {
        x.lo = min(max(base + qa + 1 - A.window, 0), x.hi);
        x.full_lo = max(base + qb + 1 - A.window, 0);
    }
    return x;
}

__device__ __forceinline__ int tiles_of(const AttnArgs& A, const Seq& q, int ROWS) {
    return (int)(((int64_t)q.n * A.group + ROWS - 1) / ROWS);
}

// Blocks of keys that a tile goes through, one at least: a row without keys has a result too.
__device__ __forceinline__ int blocks_of(const Tile& x) {
    return max((x.hi + ATTN_KEYS - 1) / ATTN_KEYS - x.lo / ATTN_KEYS, 1);
}

__device__ __forceinline__ int64_t units_of(const AttnArgs& A, const Seq& q, int ROWS) {
    const int tiles = tiles_of(A, q, ROWS);
    int64_t n = 0;
    for (int t = 0; t < tiles; ++t) n += blocks_of(get_tile(A, q, t, ROWS));
    return n;
}

__device__ __forceinline__ float xor_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}

__device__ __forceinline__ uint32_t nan_bytes(uint32_t u) {       // 0x80 in each byte that is an e4m3 NaN
    return ((u & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
}

// One wave's rows against blocks of 64 keys.  The products are transposed: keys are
// the rows of S^T = K Q^T, so that a lane has logits of one row only (row lane % 16 of
// each 16), and lane group g = lane / 16 has keys 16 g .. 16 g + 15 of the block: key
// 16 g + 4 t + i is row 4 g + i of the t-th product.  The weights are then, as they
// are, the column operand of O^T = V^T P^T, for which a lane reads 16 neighbouring
// tokens of one channel.  A lane's 16 keys are of one page: one pair of scales.
//
// Softmax: the 16-bit operand of the second product is w = 2^(s - m + k), with a
// reference m that follows the row's largest logit with some slack, and k = log2(value
// scale) + HEADROOM - c, where c follows the row's largest log2 of weight times scale:
// so it neither overflows nor loses a row whose values are small.  (k is -64 at least:
// less counts as nothing beside the row's largest.)  The denominator is the sum of w
// 2^-k.  Sums are fp32.  A 16-bit weight has 11 bits, three more than a bf16 result;
// for an fp16 result the rest of the weight goes through the product as well (FINE).
//
// Memory wants neighbouring lanes on neighbouring bytes, the products lanes of
// different keys and channels: a wave's loads go by whole rows (16 bytes a lane) and are
// turned in LDS, in a place of its own, so that no barrier is needed.  Chunks of 16
// bytes are XORed with their row: neither side meets a bank twice in eight lanes.
// Loads are of buffers that end with the page: what lies outside is not read and comes
// back as zeros, so a call's end and a page that is none need no branch.
template <int DIM>
struct AttnStage {
    static constexpr int SUB = DIM % 128 == 0 ? 128 : 64, CS = SUB / 16, SUBS = DIM / SUB, KEYS = 64 / CS;
    static constexpr int LOADS = DIM / 16;                    // loads of 16 bytes a lane for the keys or values of a block
    static constexpr int K_BYTES = ATTN_KEYS * DIM, BYTES = 2 * K_BYTES;

    char* lds;                   // keys [64][DIM], values [DIM][64]
    int k_write, v_write, k_read[2], v_read;
    uint32_t k_off[SUBS], v_off;
    int lg;                      // log2 of the neighbouring chunks of a value's row

    __device__ __forceinline__ AttnStage(const CacheView& C, char* lds_) : lds(lds_) {
        const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
        const int key = lane / CS, chunk = lane % CS;
        const int sw = SUB == 128 ? key & 3 : (key >> 1) & 1;
        k_write = key * DIM + ((chunk ^ sw) << 4);
        const int sr = SUB == 128 ? (r & 3) | (r >> 2 & 1) << 2 : (r >> 1 & 1) | (r >> 2 & 1) << 1;
        const int row = (16 * (r >> 2) + (r & 3)) * DIM;
        k_read[0] = row + ((g ^ sr) << 4);
        k_read[1] = SUB == 128 ? row + (((4 + g) ^ sr) << 4) : k_read[0] + 64;
#pragma unroll
        for (int s = 0; s < SUBS; ++s) {
            const int c = s * SUB + chunk * 16;
            k_off[s] = c < C.dim ? key * C.dim + c : OUTSIDE; // behind the row's end: zeros
        }
        lg = min(C.page_shift, 6) - 4;
        const int v_row = lane >> lg, v_chunk = (lane & ((1 << lg) - 1)) << 4;
        v_off = (v_row << C.page_shift) + v_chunk;            // channels behind the last are outside the page
        v_write = K_BYTES + v_row * 64 + (v_chunk ^ ((v_row >> 1 & 3) << 4));
        v_read = K_BYTES + r * 64 + ((g ^ (r >> 1 & 3)) << 4);
    }

    // Bytes of a page and head from `at` on; none where ids' lane group g names no page, or without `on`.
    static __device__ __forceinline__ __amdgpu_buffer_rsrc_t part(const CacheView& C, const uint8_t* p, int head, int ids, int g,
                                                                  int at, bool on) {
        const int id = __builtin_amdgcn_readlane(ids, 16 * g);
        const bool is = on && (unsigned)id < (unsigned)C.pages;
        const uint32_t bytes = (uint32_t)C.dim << C.page_shift;                   // below 2^16, and 1024 heads of it below 2^32
        return __builtin_amdgcn_make_buffer_rsrc(
            const_cast<uint8_t*>(p) + (uint64_t)(uint32_t)(is ? id : 0) * ((uint32_t)C.kv * bytes) + (head * bytes + at), 0,
            is ? bytes - at : 0, 0x27000);
    }

    __device__ __forceinline__ void load_k(const CacheView& C, int head, int b, int ids, bool on, u32x4_t (&z)[LOADS]) const {
        const int mask = (1 << C.page_shift) - 1;
        __amdgpu_buffer_rsrc_t p[4];
#pragma unroll
        for (int g = 0; g < 4; ++g) p[g] = part(C, C.k, head, ids, g, ((b * ATTN_KEYS + 16 * g) & mask) * C.dim, on);
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            const int key = j / SUBS * KEYS;
            z[j] = __builtin_amdgcn_raw_buffer_load_b128(p[key >> 4], k_off[j % SUBS], (key & 15) * C.dim, 0);
        }
    }

    __device__ __forceinline__ void load_v(const CacheView& C, int head, int b, int ids, bool on, u32x4_t (&z)[LOADS]) const {
        const int mask = (1 << C.page_shift) - 1;
        __amdgpu_buffer_rsrc_t p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int g = (i & ((1 << (2 - lg)) - 1)) << lg;
            p[i] = part(C, C.v, head, ids, g, (b * ATTN_KEYS + 16 * g) & mask, on);
        }
#pragma unroll
        for (int j = 0; j < LOADS; ++j)
            z[j] = __builtin_amdgcn_raw_buffer_load_b128(p[j & 3], v_off + (j >> (2 - lg) << (6 - lg + C.page_shift)), 0, 0);
    }

    // Between what some lanes of the wave write and others read: LDS keeps a wave's order, the compiler has to.
    static __device__ __forceinline__ void order() { asm volatile("" ::: "memory"); }

    __device__ __forceinline__ void put_k(const u32x4_t (&z)[LOADS]) const {
        order();
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            const int key = j / SUBS * KEYS;
            const int at = key >> 4 & 1 ? k_write ^ (SUB == 128 ? 64 : 32) : k_write;
            *reinterpret_cast<u32x4_t*>(lds + at + key * DIM + j % SUBS * SUB) = z[j];
        }
        order();
    }

    __device__ __forceinline__ void put_v(const u32x4_t (&z)[LOADS]) const {
        order();
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            const int g = (j & ((1 << (2 - lg)) - 1)) << lg, channel = j >> (2 - lg) << (6 - lg);
            *reinterpret_cast<u32x4_t*>(lds + (v_write ^ (g << 4)) + channel * 64) = z[j];
        }
        order();
    }

    // 16 values of key 16 (lane % 16 / 4) + 4 t + lane % 4, from 64 k + 16 (lane / 16) on
    __device__ __forceinline__ u32x4_t key(int t, int k) const {
        return *reinterpret_cast<const u32x4_t*>(lds + k_read[k & 1] + k / 2 * 128 + 4 * t * DIM);
    }

    // 16 tokens, from 16 (lane / 16) on, of channel 16 d + lane % 16
    __device__ __forceinline__ u32x4_t& value(int d) const { return *reinterpret_cast<u32x4_t*>(lds + v_read + d * 1024); }
};

template <int DIM, bool BF16, int RB>
struct AttnWave {
    static constexpr bool FINE = !BF16;
    static constexpr int KC = DIM / 64, DT = DIM / 16;
    typedef Half16<BF16> H;
    typedef Half16<false> W;

    float4_t o[DT][RB];
    float m[RB], top[RB], c[RB], l[RB];

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            m[rb] = top[rb] = ATTN_LOW;
            c[rb] = l[rb] = 0.f;
#pragma unroll
            for (int d = 0; d < DT; ++d) o[d][rb] = float4_t{0.f, 0.f, 0.f, 0.f};
        }
    }

    // Blocks first, first + step, ... < last of the tile's keys.  No branch divides lanes in here: the compiler may leave
    // them apart in the loop around the products, and may place copies of other lanes' registers before they are back.
    __device__ __forceinline__ void run(const AttnArgs& A, const AttnStage<DIM>& S, const Seq& q, const Tile& x, int s, int head,
                                        int first, int last, int step) {
        if (first >= last) return;
        const CacheView& C = A.c;
        const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
        const int base = q.len - q.n;
        typename H::vec8 qf[RB][KC][2];
        int see_lo[RB], see_hi[RB];
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            const int row = 16 * rb + r;
            const bool in = row < x.rows;
            const int of = x.r0 + (in ? row : 0), at = of / A.group, hg = of - at * A.group;
            const uint16_t* p = A.q + (int64_t)(q.first + at) * A.q_token + (int64_t)(head * A.group + hg) * A.q_head;
#pragma unroll
            for (int k = 0; k < KC; ++k)
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const int d = 64 * k + 16 * g + 8 * u;
                    const bool is = in && d < C.dim;
                    const u32x4_t z = *reinterpret_cast<const u32x4_t*>(p + (d < C.dim ? d : 0));
                    u32x4_t v;
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] = is ? A.negative ? z[i] ^ 0x80008000u : z[i] : 0u;
                    qf[rb][k][u] = __builtin_bit_cast(typename H::vec8, v);
                }
            see_hi[rb] = in ? min(base + at + 1, q.len) : 0;
            see_lo[rb] = in && A.window ? base + at + 1 - A.window : 0;
        }
        const int* table = C.table + s * C.table_stride;
        const int pages = (q.len + (1 << C.page_shift) - 1) >> C.page_shift;
        // The page of lane group g's 16 keys.
        const auto pages_of = [&](int b) {
            const int i = (min(b, last - 1) * ATTN_KEYS + 16 * g) >> C.page_shift, id = table[min(i, pages - 1)];
            return i < pages ? id : -1;
        };
        const auto valid = [&](int id) { return (unsigned)id < (unsigned)C.pages; };
        const auto scale_of = [&](const float* p, int id) { return p[(int64_t)(valid(id) ? id : 0) * C.kv + head]; };
        // In a block that not every row sees whole, what no row sees may hold anything: its bytes become zeros (a weight of 0
        // would leave a NaN one).  A NaN that only some rows see becomes a zero too, and `nans` has it counted later.
        bool nans = false;
        const auto hide_values = [&](int b, bool here, bool keep_nans) {
            const int key0 = b * ATTN_KEYS + 16 * g;
            uint32_t keep[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                keep[j] = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int key = key0 + 4 * j + e;
                    if (here && key >= x.lo && key < x.hi) keep[j] |= 0xffu << (8 * e);
                }
            }
            uint32_t nan = 0;
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                u32x4_t v = S.value(d);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    v[j] &= keep[j];
                    const uint32_t bad = nan_bytes(v[j]);
                    nan |= bad;
                    if (!keep_nans) v[j] &= ~((bad >> 7) * 0xffu);
                }
                S.value(d) = v;
            }
            S.order();
            nans |= __builtin_amdgcn_ballot_w64(nan != 0) != 0;
        };

        u32x4_t kreg[DT], vreg[DT];
        int ids = pages_of(first), next = pages_of(first + step);  // asked for two blocks ahead: loads come back in order
        S.load_k(C, head, first, ids, true, kreg);
        float ks = scale_of(C.k_scale, ids), vs = scale_of(C.v_scale, ids);
        S.load_v(C, head, first, ids, true, vreg);
        for (int b = first; b < last; b += step) {
            const int id_here = ids;
            float kc = fmaxf(ks * A.qk_scale, 0x1p-126f), vscale = vs;
            const int after = pages_of(b + 2 * step);
            const bool more = b + step < last;
            S.put_k(kreg);
            S.load_k(C, head, b + step, next, more, kreg);
            ks = scale_of(C.k_scale, next);
            vs = scale_of(C.v_scale, next);
            float4_t p[4][RB];
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) p[t][rb] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < KC; ++k)
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const u32x4_t z = S.key(t, k);
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const typename H::vec8 key = H::widen(z[2 * u], z[2 * u + 1]);
#pragma unroll
                        for (int rb = 0; rb < RB; ++rb) p[t][rb] = H::mfma(key, qf[rb][k][u], p[t][rb]);
                    }
                }
            S.put_v(vreg);
            S.load_v(C, head, b + step, next, more, vreg);
            ids = next;
            next = after;
            if (b * ATTN_KEYS < x.full_lo || (b + 1) * ATTN_KEYS > x.full_hi ||
                __builtin_amdgcn_ballot_w64(valid(id_here)) != ~0ull) {
                const int key0 = b * ATTN_KEYS + 16 * g;
                const bool here = valid(id_here) && key0 + 15 >= x.lo && key0 < x.hi;
                kc = here ? kc : 1.f;
                vscale = here ? vscale : 1.f;
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) {
                    const int lo = here ? see_lo[rb] - key0 : 16, n = see_hi[rb] - key0;
#pragma unroll
                    for (int t = 0; t < 4; ++t)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int key = 4 * t + i;
                            p[t][rb][i] = key >= lo && key < n ? p[t][rb][i] : -__builtin_inff();
                        }
                }
                hide_values(b, here, false);
            }
            const float lv = __builtin_amdgcn_logf(vscale);
            bool grew = false;
            float most[RB];
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
                float a = p[0][rb][0];
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (t + i) a = fmaxf(a, p[t][rb][i]);
                most[rb] = a * kc;
                grew |= most[rb] > m[rb] + ATTN_SLACK || most[rb] + lv > top[rb] + ATTN_SLACK;
            }
            if (__builtin_amdgcn_ballot_w64(grew)) {
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) {
                    const float m1 = fmaxf(m[rb], xor_max(most[rb])), top1 = fmaxf(top[rb], xor_max(most[rb] + lv));
                    const float c1 = ceilf(top1 - m1);
                    const float fl = __builtin_amdgcn_exp2f(m[rb] - m1);
                    const float fo = __builtin_amdgcn_exp2f(m[rb] - m1 + (c[rb] - c1));
                    m[rb] = m1;
                    top[rb] = top1;
                    c[rb] = c1;
                    l[rb] *= fl;
#pragma unroll
                    for (int d = 0; d < DT; ++d)
#pragma unroll
                        for (int i = 0; i < 4; ++i) o[d][rb][i] *= fo;
                }
            }
            half8_t hi[RB][2], lo[RB][2];
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
                const float k = fmaxf(lv + (ATTN_HEADROOM - c[rb]), -64.f), add = k - m[rb];
                float sum = 0.f;
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float w = __builtin_amdgcn_exp2f(fmaf(p[t][rb][i], kc, add));
                        sum += w;
                        const _Float16 h = (_Float16)w;
                        hi[rb][t >> 1][4 * (t & 1) + i] = h;
                        if constexpr (FINE) lo[rb][t >> 1][4 * (t & 1) + i] = (_Float16)(w - (float)h);
                    }
                l[rb] = fmaf(sum, __builtin_amdgcn_exp2f(-k), l[rb]);
            }
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                const u32x4_t z = S.value(d);
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const half8_t v = W::widen(z[2 * u], z[2 * u + 1]);
#pragma unroll
                    for (int rb = 0; rb < RB; ++rb) {
                        o[d][rb] = W::mfma(v, hi[rb][u], o[d][rb]);
                        if constexpr (FINE) o[d][rb] = W::mfma(v, lo[rb][u], o[d][rb]);
                    }
                }
            }
        }
        if (!nans) return;
        // NaN values that were left out above: counted for the rows that see them, in products of their own.
        for (int b = first; b < last; b += step) {
            const int id = pages_of(b);
            const int key0 = b * ATTN_KEYS + 16 * g;
            const bool here = valid(id) && key0 + 15 >= x.lo && key0 < x.hi;
            S.load_v(C, head, b, id, true, vreg);
            S.put_v(vreg);
            hide_values(b, here, true);
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
                half8_t sees[2];
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const int key = key0 + 8 * u + j;
                        sees[u][j] = here && key >= see_lo[rb] && key < see_hi[rb] ? (_Float16)1.f : (_Float16)0.f;
                    }
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    const u32x4_t z = S.value(d);
                    float4_t n = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int u = 0; u < 2; ++u)
                        n = W::mfma(W::widen((nan_bytes(z[2 * u]) >> 7) * 0x38u, (nan_bytes(z[2 * u + 1]) >> 7) * 0x38u),
                                    sees[u], n);                                             // 0x38: one
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[d][rb][i] = n[i] > 0.f ? __builtin_nanf("") : o[d][rb][i];
                }
            }
        }
    }
};

template <int DIM, int RB>
struct AttnSize {
    static constexpr int ROWS = 16 * RB, PITCH = DIM + 4;
    static constexpr int JOIN = ATTN_WAVES * ROWS * (PITCH + 2) * 4, STAGE = ATTN_WAVES * AttnStage<DIM>::BYTES;
    static constexpr int LDS = JOIN > STAGE ? JOIN : STAGE;       // the blocks of the waves, then their sums
    static constexpr int WAVES_EU = RB <= 2 && DIM <= 128 ? 2 : 1;
    static constexpr int PART = ROWS * (DIM + 2);                 // floats of a partial result: rows of sums, then m and l
};

// Four outputs of one row.
template <bool BF16>
__device__ __forceinline__ void store_row4(uint16_t* p, float4_t v) {
    const uint32_t a = BF16 ? pack_bf16(v[0], v[1]) : f32_to_f16_bits(v[0]) | (uint32_t)f32_to_f16_bits(v[1]) << 16;
    const uint32_t b = BF16 ? pack_bf16(v[2], v[3]) : f32_to_f16_bits(v[2]) | (uint32_t)f32_to_f16_bits(v[3]) << 16;
    *reinterpret_cast<u32x2_t*>(p) = u32x2_t{a, b};
}

// A row's final factor and the logarithm of its sum, from its reference and sum.
__device__ __forceinline__ float finish_row(const AttnArgs& A, int head, float m, float l, float& lse) {
    float f = 1.f;
    if (A.sinks) {
        const float s = A.sinks[head] * 1.4426950408889634f, m1 = fmaxf(m, s);
        f = __builtin_amdgcn_exp2f(m - m1);
        l = l * f + __builtin_amdgcn_exp2f(s - m1);
        m = m1;
    }
    lse = l == 0.f ? -__builtin_inff() : (m + __builtin_amdgcn_logf(l)) * 0.6931471805599453f;
    return l == 0.f ? 0.f : f / l;
}

// Rows of q whose tokens no sequence has: zeros, and -inf for the logarithm.
__device__ __forceinline__ void clear_rows(const AttnArgs& A) {
    const CacheView& C = A.c;
    if (!A.clear || !C.starts) return;
    const int a = min(max(C.starts[0], 0), C.tokens), b = min(max(C.starts[C.seqs], a), C.tokens);
    const int rows = C.tokens - (b - a);
    const int64_t each = (int64_t)A.heads * C.dim / 8;
    for (int i = blockIdx.x; i < rows; i += gridDim.x) {
        const int64_t t = i < a ? i : i + (b - a);
        for (int64_t j = threadIdx.x; j < each; j += blockDim.x)
            reinterpret_cast<u32x4_t*>(A.out + t * A.heads * C.dim)[j] = u32x4_t{0, 0, 0, 0};
        if (A.lse)
            for (int j = threadIdx.x; j < A.heads; j += blockDim.x) A.lse[t * A.heads + j] = -__builtin_inff();
    }
}

// Workgroups go to the XCDs in turn (workgroup b to XCD b % 8), and what one reads its
// neighbours on the XCD find in L2: so an XCD's workgroups take neighbouring work.
constexpr int XCDS = 8;

// Workgroup b's place where each XCD's workgroups are next to each other.
__device__ __forceinline__ int by_xcd(int b, int n) {
    const int x = b % XCDS, each = n / XCDS, more = n % XCDS;
    return x * each + min(x, more) + b / XCDS;
}

// A workgroup a tile: a head's tiles in turn on the XCDs that the head has, or an XCD's heads one after another.
__device__ __forceinline__ void tile_by_xcd(int b, int tiles, int heads, int& tile, int& head) {
    const int x = b % XCDS, i = b / XCDS;
    if (heads < XCDS && XCDS % heads == 0) {
        const int of = XCDS / heads;
        head = x / of;
        tile = i * of + x % of;
    } else if (heads % XCDS == 0) {
        head = x * (heads / XCDS) + i / tiles;
        tile = i % tiles;
    } else {
        head = b / tiles;
        tile = b % tiles;
    }
}

// Units are (cache head, tile, block of keys), in this order; a workgroup has an
// equal share of them, next to each other, whatever sequences they are of.  Its four
// waves go through a tile's blocks in turn and join their sums in LDS.  A tile whose
// blocks one workgroup has all is finished; of the others each workgroup leaves a
// partial result: in its first place where the tile began before its share, in its
// second where it goes on behind it.  Without a place for partial results a workgroup
// has a tile, the last, longest ones first.
template <int DIM, bool BF16, int RB>
__global__ __launch_bounds__(ATTN_WAVES * 64, (AttnSize<DIM, RB>::WAVES_EU)) void fp8_attention_kernel(AttnArgs A) {
    typedef AttnSize<DIM, RB> Z;
    extern __shared__ __attribute__((aligned(16))) float lds[];
    const CacheView& C = A.c;
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), r = lane & 15, g = lane >> 4;
    int64_t u = 0, u1 = 0, share = 0;
    int s = 0, t = 0, head = 0, done = 0;                       // done: the tile's blocks before the share
    Seq q;
    Tile x;
    int n = 0;
    int me = blockIdx.x;
    clear_rows(A);
    if (A.part) {
        const Found f = find_seq(C, [&](const Seq& x) { return units_of(A, x, Z::ROWS); }, [&](int64_t total) {
            const int64_t all = total * C.kv;
            share = divide(all + gridDim.x - 1, gridDim.x);
            if (share < A.least) share = A.least;
            const int busy = (int)divide(all + share - 1, share);
            if (me >= busy) return (int64_t)-1;
            me = by_xcd(me, busy);
            u = share * me;
            u1 = u + share < all ? u + share : all;
            head = (int)divide(u, total);
            return u - head * total;
        });
        if (tid == 0) A.shared[me].last = -1;            // nothing to join, unless a tile goes on behind the share
        if (f.s < 0) return;
        s = f.s;
        q = f.q;
        int64_t left = f.unit;
        for (;; ++t) {
            x = get_tile(A, q, t, Z::ROWS);
            n = blocks_of(x);
            if (left < n) break;
            left -= n;
        }
        done = (int)left;
    } else {
        int tile;
        tile_by_xcd(blockIdx.x, A.tiles, C.kv, tile, head);
        if (tile >= A.tiles || head >= C.kv) return;
        const int64_t at = A.tiles - 1 - tile;
        const Found f = find_seq(C, [&](const Seq& x) { return (int64_t)tiles_of(A, x, Z::ROWS); }, [&](int64_t) { return at; });
        if (f.s < 0) return;
        s = f.s;
        q = f.q;
        t = (int)f.unit;
        x = get_tile(A, q, t, Z::ROWS);
        n = blocks_of(x);
        u1 = n;
    }
    const AttnStage<DIM> S(C, reinterpret_cast<char*>(lds) + wave * AttnStage<DIM>::BYTES);
    float* sums = lds;                                          // [wave][row][PITCH]
    float* ml = lds + ATTN_WAVES * Z::ROWS * Z::PITCH;          // [wave][row][2]
    for (;;) {
        const int64_t want = u1 - u;
        const int here = (int)(n - done < want ? n - done : want);
        const int b0 = x.lo / ATTN_KEYS + done;
        AttnWave<DIM, BF16, RB> W;
        W.clear();
        W.run(A, S, q, x, s, head, b0 + wave, min(b0 + here, (x.hi + ATTN_KEYS - 1) / ATTN_KEYS), ATTN_WAVES);
        __syncthreads();
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            const int row = 16 * rb + r;
            float l = W.l[rb];
            l += __shfl_xor(l, 16);
            l += __shfl_xor(l, 32);
            ml[(wave * Z::ROWS + row) * 2] = W.m[rb];           // by four lanes alike: no branch while the sums are live
            ml[(wave * Z::ROWS + row) * 2 + 1] = l;
            const int back = (int)W.c[rb] - ATTN_HEADROOM;
#pragma unroll
            for (int d = 0; d < DIM / 16; ++d) {
                float4_t v;
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = ldexpf(W.o[d][rb][i], back);
                *reinterpret_cast<float4_t*>(sums + (wave * Z::ROWS + row) * Z::PITCH + 16 * d + 4 * g) = v;
            }
        }
        __syncthreads();
        const bool final = here == n;
        if (!final && done == 0 && tid == 0)
            A.shared[me] = SharedTile{q.first, x.r0, x.rows, head, (int)divide(u + n - 1, share)};
        float* part = A.part + ((int64_t)me * 2 + (done == 0 ? 1 : 0)) * Z::PART;
        const int quads = C.dim / 4;
        for (int i = tid; i < x.rows * quads; i += ATTN_WAVES * 64) {
            const int row = i / quads, d = (i - row * quads) * 4;
            float m = ATTN_LOW, l = 0.f;
#pragma unroll
            for (int w = 0; w < ATTN_WAVES; ++w) m = fmaxf(m, ml[(w * Z::ROWS + row) * 2]);
            float4_t v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < ATTN_WAVES; ++w) {
                const float f = __builtin_amdgcn_exp2f(ml[(w * Z::ROWS + row) * 2] - m);
                l += f * ml[(w * Z::ROWS + row) * 2 + 1];
                const float4_t a = *reinterpret_cast<const float4_t*>(sums + (w * Z::ROWS + row) * Z::PITCH + d);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = fmaf(f, a[j], v[j]);
            }
            if (final) {
                const int at = (x.r0 + row) / A.group, h = head * A.group + x.r0 + row - at * A.group;
                const int64_t o = (int64_t)(q.first + at) * A.heads + h;
                float lse;
                const float f = finish_row(A, h, m, l, lse);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] *= f;
                store_row4<BF16>(A.out + o * C.dim + d, v);
                if (A.lse && d == 0) A.lse[o] = lse;
            } else {
                *reinterpret_cast<float4_t*>(part + row * C.dim + d) = v;
                if (d == 0) {
                    part[Z::ROWS * DIM + 2 * row] = m;
                    part[Z::ROWS * DIM + 2 * row + 1] = l;
                }
            }
        }
        u += here;
        if (u >= u1) break;
        __syncthreads();                                        // the sums' places hold blocks again
        done = 0;
        if (++t == tiles_of(A, q, Z::ROWS)) {
            t = 0;
            do {
                if (++s == C.seqs) {
                    s = 0;
                    ++head;
                }
                q = get_seq(C, s);
            } while (q.n == 0);
        }
        x = get_tile(A, q, t, Z::ROWS);
        n = blocks_of(x);
    }
}

// A tile that several workgroups share, joined: blockIdx.x is the workgroup that
// begins it, blockIdx.y takes every gridDim.y-th row.  A row's threads are groups that
// each take some of the partial results, four channels a thread; the groups' sums
// meet in LDS.
template <int DIM, bool BF16, int RB>
__global__ __launch_bounds__(ATTN_WAVES * 64) void fp8_attention_join_kernel(AttnArgs A) {
    typedef AttnSize<DIM, RB> Z;
    constexpr int QUADS = DIM / 4, GROUPS = ATTN_WAVES * 64 / QUADS;
    __shared__ float4_t sums[GROUPS][QUADS];
    __shared__ float ml[GROUPS][2];
    const CacheView& C = A.c;
    const SharedTile x = A.shared[blockIdx.x];
    const int first = blockIdx.x, group = threadIdx.x / QUADS, d = (threadIdx.x - group * QUADS) * 4;
    if (x.last < 0) return;
    const auto take = [&](int w, int row, float& m, float& l, float4_t& v) {
        const float* p = A.part + ((int64_t)w * 2 + (w == first ? 1 : 0)) * Z::PART;
        const float pm = p[Z::ROWS * DIM + 2 * row], pl = p[Z::ROWS * DIM + 2 * row + 1];
        const float4_t a = *reinterpret_cast<const float4_t*>(p + row * C.dim + d);
        const float m1 = fmaxf(m, pm), f = __builtin_amdgcn_exp2f(m - m1), g = __builtin_amdgcn_exp2f(pm - m1);
        m = m1;
        l = fmaf(g, pl, l * f);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = fmaf(g, a[j], v[j] * f);
    };
    const auto finish = [&](int row, float m, float l, float4_t v) {
        const int at = (x.r0 + row) / A.group, h = x.head * A.group + x.r0 + row - at * A.group;
        const int64_t o = (int64_t)(x.first + at) * A.heads + h;
        float lse;
        const float f = finish_row(A, h, m, l, lse);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] *= f;
        store_row4<BF16>(A.out + o * C.dim + d, v);
        if (A.lse && d == 0) A.lse[o] = lse;
    };
    if (x.last - first < 2 * GROUPS) {
        // few partial results: a row a group
        if (group >= GROUPS || d >= C.dim) return;
        for (int row = blockIdx.y * GROUPS + group; row < x.rows; row += gridDim.y * GROUPS) {
            float m = ATTN_LOW, l = 0.f;
            float4_t v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
            for (int w = first; w <= x.last; ++w) take(w, row, m, l, v);
            finish(row, m, l, v);
        }
        return;
    }
    for (int row = blockIdx.y; row < x.rows; row += gridDim.y) {
        float m = ATTN_LOW, l = 0.f;
        float4_t v = {0.f, 0.f, 0.f, 0.f};
        if (group < GROUPS && d < C.dim) {
#pragma unroll 4
            for (int w = first + group; w <= x.last; w += GROUPS) take(w, row, m, l, v);
            sums[group][d / 4] = v;
            if (d == 0) {
                ml[group][0] = m;
                ml[group][1] = l;
            }
        }
        __syncthreads();
        if (group == 0 && d < C.dim) {
#pragma unroll
            for (int i = 1; i < GROUPS; ++i) {
                const float m1 = fmaxf(m, ml[i][0]), f = __builtin_amdgcn_exp2f(m - m1), g = __builtin_amdgcn_exp2f(ml[i][0] - m1);
                m = m1;
                l = fmaf(g, ml[i][1], l * f);
                const float4_t a = sums[i][d / 4];
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = fmaf(g, a[j], v[j] * f);
            }
            finish(row, m, l, v);
        }
        __syncthreads();
    }
}

}  // namespace exl3
