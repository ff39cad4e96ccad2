// Causal attention over the 8-bit paged cache, with grouped heads.
//
//   s_ij = scale * q_i . k_j for the keys j that query i sees (j <= i, j > i - window)
//   out_i = sum_j e^(s_ij) v_j / (sum_j e^(s_ij) + e^sink),  lse_i = log of that sum
#pragma once

#include "exl3_cache.hpp"
#include "exl3_xcd.hpp"

namespace exl3 {

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
    int most;                                 // workgroups that the units are divided over at most
    int clear;                                // rows that no sequence has: 1: zeros, and -inf for the logarithm; 2: this alone
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
    x.hi = min(max(base + qb + 1, 0), q.end);
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

// Pieces of `each` blocks that the tiles of a sequence make.
__device__ __forceinline__ int64_t units_of(const AttnArgs& A, const Seq& q, int ROWS, int64_t each) {
    const int tiles = tiles_of(A, q, ROWS);
    int64_t n = 0;
    for (int t = 0; t < tiles; ++t) {
        const int blocks = blocks_of(get_tile(A, q, t, ROWS));
        n += each == 1 ? blocks : divide(blocks + each - 1, each);
    }
    return n;
}

__device__ __forceinline__ float xor_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}

__device__ __forceinline__ uint32_t nan_bytes(uint32_t u) {       // 0x80 in each byte that is an e4m3 NaN
    return ((u & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
}

// A page's scale that is NaN, infinite or negative: what sees the page is NaN.
__device__ __forceinline__ bool bad_scale(float s) {
    return __builtin_amdgcn_classf(s, 0x3 | 0x4 | 0x8 | 0x10 | 0x200);     // NaNs, -infinity, -normal, -subnormal, infinity
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
// 2^-k.  Sums are fp32.  A 16-bit weight has 11 bits; with FINE the rest of it goes
// through the product as well (22 bits).  That is nearly free where memory bounds a call
// (few rows, 64 tokens of up to 8192: 119.6 -> 121.3 us; one of 1000: 10.8 -> 10.9), and
// costs 22% where instructions do (a chunk of 512 behind 16384 keys: 171-175 -> 210; in
// tiles of 64 rows 64 sequences of up to 8 and 16 tokens 144 -> 152 and 155 -> 166, a chunk
// of 256 channels 191 -> 226): so many rows with a bf16 result, which has three bits less
// than the weight, go without.
// Against 64 bits the chunk's error, the result's rounding in it, is 1.6596e-3 of the
// result without the rest and 1.6568e-3 with it.
template <int DIM, bool BF16, int RB, bool FINE>
struct AttnRows {
    static constexpr int ROWS = 16 * RB, KC = DIM / 64, DT = DIM / 16;
    typedef Half16<BF16> H;
    typedef Half16<false> W;

    typename H::vec8 qf[RB][KC][2];
    int see_lo[RB], see_hi[RB];
    float4_t o[DT][RB];
    float m[RB], top[RB], c[RB], l[RB];

    // The rows from r0 on of sequence q and a cache head, `rows` of them (one at least).
    __device__ __forceinline__ void begin(const AttnArgs& A, const Seq& q, int r0, int rows, int head) {
        const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4, base = q.len - q.n;
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            const int row = 16 * rb + r;
            const bool in = row < rows;
            const int of = r0 + (in ? row : 0), at = of / A.group, hg = of - at * A.group;
            const uint16_t* p = A.q + (int64_t)(q.first + at) * A.q_token + (int64_t)(head * A.group + hg) * A.q_head;
#pragma unroll
            for (int k = 0; k < KC; ++k)
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const int d = 64 * k + 16 * g + 8 * u;
                    const bool is = in && d < A.c.dim;
                    const u32x4_t z = *reinterpret_cast<const u32x4_t*>(p + (d < A.c.dim ? d : 0));
                    u32x4_t v;
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] = is ? A.negative ? z[i] ^ 0x80008000u : z[i] : 0u;
                    qf[rb][k][u] = __builtin_bit_cast(typename H::vec8, v);
                }
            see_hi[rb] = in ? min(base + at + 1, q.end) : 0;
            see_lo[rb] = in && A.window ? base + at + 1 - A.window : 0;
            m[rb] = top[rb] = ATTN_LOW;
            c[rb] = l[rb] = 0.f;
#pragma unroll
            for (int d = 0; d < DT; ++d) o[d][rb] = float4_t{0.f, 0.f, 0.f, 0.f};
        }
    }

    // What no row of [lo, hi) sees may hold anything: its bytes become zeros (a weight of 0 would leave a NaN one).
    static __device__ __forceinline__ void keep_bytes(uint32_t (&keep)[4], bool here, int key0, int lo, int hi) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            keep[j] = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int key = key0 + 4 * j + e;
                if (here && key >= lo && key < hi) keep[j] |= 0xffu << (8 * e);
            }
        }
    }

    // A block of keys, key0 = its first plus 16 (lane / 16).  key(t, k): 16 bytes of key 16 (lane % 16 / 4) + 4 t + lane % 4
    // from channel 64 k + 16 (lane / 16) on; value(d): 16 tokens, from key0 on, of channel 16 d + lane % 16.  ks, vs: the
    // scales of the lane's 16 keys.  masked: not every row sees it whole, or a scale is none; the lane's keys are in a page
    // (`here`) and the rows see [lo, hi) at most.  Returns whether a value that some rows see is a NaN, by itself or by its
    // scale: it is left out (counted by add_nans).
    template <typename K, typename V>
    __device__ __forceinline__ bool step(const AttnArgs& A, bool masked, float ks, float vs, bool here, int key0, int lo, int hi, K&& key,
                                         V&& value) {
        float4_t p[4][RB];
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) p[t][rb] = float4_t{0.f, 0.f, 0.f, 0.f};
        // Two reads from LDS are on their way while the last two are multiplied: piece n of the keys is t = 2 n % 4 and the
        // next, k = n / 2; the values' follow.
        u32x4_t z[2][2];
        const auto read_key = [&](int n, int i) { return key(2 * n % 4 + i, n / 2); };
#pragma unroll
        for (int i = 0; i < 2; ++i) z[0][i] = read_key(0, i);
        // Products first: the other waves' other work goes on beside them (four prompts of up to 3000 tokens 236 -> 230 us, the
        // other way round 240; a chunk of 512 behind 16384 keys 185, 184 and 180).
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int n = 0; n < 2 * KC; ++n) {
#pragma unroll
            for (int i = 0; i < 2; ++i) z[(n + 1) & 1][i] = n + 1 < 2 * KC ? read_key(n + 1, i) : value(i);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const typename H::vec8 w = H::widen(z[n & 1][i][2 * u], z[n & 1][i][2 * u + 1]);
#pragma unroll
                    for (int rb = 0; rb < RB; ++rb) p[2 * n % 4 + i][rb] = H::mfma(w, qf[rb][n / 2][u], p[2 * n % 4 + i][rb]);
                }
            __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_s_setprio(0);
        float kc = fmaxf(ks * A.qk_scale, 0x1p-126f);
        uint32_t keep[4] = {}, nan = 0;
        if (masked) {
            here = here && key0 + 15 >= lo && key0 < hi;
            const float poison = bad_scale(ks) ? __builtin_nanf("") : 0.f;
            kc = here && !bad_scale(ks) ? kc : 1.f;
            nan = here && bad_scale(vs) ? 1u : 0u;
            vs = here && !bad_scale(vs) ? vs : 1.f;
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
                const int from = here ? see_lo[rb] - key0 : 16, n = see_hi[rb] - key0;
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int at = 4 * t + i;
                        p[t][rb][i] = at >= from && at < n ? p[t][rb][i] + poison : -__builtin_inff();
                    }
            }
            keep_bytes(keep, here, key0, lo, hi);
        }
        const float lv = __builtin_amdgcn_logf(vs);
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
        half8_t big[RB][2], rest[RB][2];
        float minus = -1.f;
        asm("" : "+s"(minus));                                  // unknown: a mixed fma reads the 16-bit weight as it is
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            const float k = fmaxf(lv + (ATTN_HEADROOM - c[rb]), -64.f), add = k - m[rb];
            float sum[4];                                       // four chains of additions
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int i = 0; i < 4; i += 2) {
                    const float w0 = __builtin_amdgcn_exp2f(fmaf(p[t][rb][i], kc, add));
                    const float w1 = __builtin_amdgcn_exp2f(fmaf(p[t][rb][i + 1], kc, add));
                    sum[i] = t ? sum[i] + w0 : w0;
                    sum[i + 1] = t ? sum[i + 1] + w1 : w1;
                    const int at = 4 * (t & 1) + i;
                    big[rb][t >> 1][at] = (_Float16)w0;
                    big[rb][t >> 1][at + 1] = (_Float16)w1;
                    if constexpr (FINE) {
                        rest[rb][t >> 1][at] = (_Float16)fmaf((float)big[rb][t >> 1][at], minus, w0);
                        rest[rb][t >> 1][at + 1] = (_Float16)fmaf((float)big[rb][t >> 1][at + 1], minus, w1);
                    }
                }
            l[rb] = fmaf((sum[0] + sum[1]) + (sum[2] + sum[3]), __builtin_amdgcn_exp2f(-k), l[rb]);
            asm volatile("" : "+v"(l[rb]));                     // now: the weights would be kept until behind the products
            __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int n = 0; n < DT / 2; ++n) {
            u32x4_t (&v)[2] = z[n & 1];
            if (n + 1 < DT / 2) {
#pragma unroll
                for (int i = 0; i < 2; ++i) z[(n + 1) & 1][i] = value(2 * n + 2 + i);
            }
            __builtin_amdgcn_sched_barrier(0);
            if (masked) {
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        v[i][j] &= keep[j];
                        const uint32_t bad = nan_bytes(v[i][j]);
                        nan |= bad;
                        v[i][j] &= ~((bad >> 7) * 0xffu);
                    }
            }
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const half8_t w = W::widen(v[i][2 * u], v[i][2 * u + 1]);
#pragma unroll
                    for (int rb = 0; rb < RB; ++rb) o[2 * n + i][rb] = W::mfma(w, big[rb][u], o[2 * n + i][rb]);
                    if constexpr (FINE) {
#pragma unroll
                        for (int rb = 0; rb < RB; ++rb) o[2 * n + i][rb] = W::mfma(w, rest[rb][u], o[2 * n + i][rb]);
                    }
                }
            __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_s_setprio(0);
        return masked && __builtin_amdgcn_ballot_w64(nan != 0) != 0;
    }

    // The NaN values of a masked block (all of the lane's, if their scale vs is none), counted for the rows that see them in
    // products of their own.
    template <typename V>
    __device__ __forceinline__ void add_nans(bool here, float vs, int key0, int lo, int hi, V&& value) {
        uint32_t keep[4];
        here = here && key0 + 15 >= lo && key0 < hi;
        keep_bytes(keep, here, key0, lo, hi);
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            half8_t sees[2];
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int at = key0 + 8 * u + j;
                    sees[u][j] = here && at >= see_lo[rb] && at < see_hi[rb] ? (_Float16)1.f : (_Float16)0.f;
                }
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                u32x4_t z = value(d);
#pragma unroll
                for (int j = 0; j < 4; ++j) z[j] = bad_scale(vs) ? 0x7f7f7f7fu : z[j];
                float4_t n = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int u = 0; u < 2; ++u)
                    n = W::mfma(W::widen((nan_bytes(z[2 * u] & keep[2 * u]) >> 7) * 0x38u,                // 0x38: one
                                         (nan_bytes(z[2 * u + 1] & keep[2 * u + 1]) >> 7) * 0x38u), sees[u], n);
#pragma unroll
                for (int i = 0; i < 4; ++i) o[d][rb][i] = n[i] > 0.f ? __builtin_nanf("") : o[d][rb][i];
            }
        }
    }

    // A row's sum over the lanes that share it, and what brings its o to the unit of that sum.
    __device__ __forceinline__ float row_sum(int rb) const {
        float a = l[rb];
        a += __shfl_xor(a, 16);
        return a + __shfl_xor(a, 32);
    }
    __device__ __forceinline__ int back(int rb) const { return (int)c[rb] - ATTN_HEADROOM; }
};

// v in another register: the one that it came in is free for the next load.
template <typename T>
__device__ __forceinline__ T moved(T v) {
    T r;
    asm volatile("v_mov_b32 %0, %1" : "=v"(r) : "v"(v));
    return r;
}

// A sequence's pages for one cache head.
struct Pages {
    const int* table;
    int pages;

    __device__ __forceinline__ Pages(const CacheView& C, const Seq& q, int s)
        : table(C.table + s * C.table_stride), pages((q.end + (1 << C.page_shift) - 1) >> C.page_shift) {}

    // The page of the 16 keys from 64 b + 16 (lane / 16) on, -1 behind the sequence's end; raw: as the table has it.
    __device__ __forceinline__ int index(const CacheView& C, int b) const { return (b * ATTN_KEYS + (threadIdx.x & 48)) >> C.page_shift; }
    __device__ __forceinline__ int raw(const CacheView& C, int b) const { return table[min(index(C, b), pages - 1)]; }
    __device__ __forceinline__ int of(const CacheView& C, int b, int raw) const { return index(C, b) < pages ? raw : -1; }
    __device__ __forceinline__ int of(const CacheView& C, int b) const { return of(C, b, raw(C, b)); }
};

__device__ __forceinline__ bool valid_page(const CacheView& C, int id) { return (unsigned)id < (unsigned)C.pages; }
__device__ __forceinline__ float scale_of(const CacheView& C, const float* p, int id, int head) {
    return p[(int64_t)(valid_page(C, id) ? id : 0) * C.kv + head];
}

// Whether some row of a tile does not see a block whole, or a scale is none.
__device__ __forceinline__ bool masked_block(const CacheView& C, const Tile& x, int b, int id, float ks, float vs) {
    return b * ATTN_KEYS < x.full_lo || (b + 1) * ATTN_KEYS > x.full_hi ||
           __builtin_amdgcn_ballot_w64(valid_page(C, id) && !bad_scale(ks) && !bad_scale(vs)) != ~0ull;
}

// Bytes of a page and head from `at` on, as a buffer that ends with the page; none where ids' lane group g names no
// page, or without `on`: what lies outside a buffer is not read and comes back as zeros.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t page_part(const CacheView& C, const uint8_t* p, int head, int ids, int g, int at,
                                                            bool on) {
    const int id = __builtin_amdgcn_readlane(ids, 16 * g);
    const bool is = on && valid_page(C, id);
    const uint32_t bytes = (uint32_t)C.dim << C.page_shift;                   // 2^16 at most, and 1024 heads of it 2^26
    return __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint8_t*>(p) + (uint64_t)(uint32_t)(is ? id : 0) * ((uint32_t)C.kv * bytes) + (head * bytes + at), 0,
        is ? bytes - at : 0, 0x27000);
}

// Memory wants neighbouring lanes on neighbouring bytes, the products lanes of
// different keys and channels: a wave's loads go by whole rows (16 bytes a lane) and are
// turned in LDS, in a place of its own, so that no barrier is needed.  Chunks of 16
// bytes are XORed with their row: neither side meets a bank twice in eight lanes.
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

    __device__ __forceinline__ void load_k(const CacheView& C, int head, int b, int ids, bool on, u32x4_t (&z)[LOADS]) const {
        const int mask = (1 << C.page_shift) - 1;
        __amdgpu_buffer_rsrc_t p[4];
#pragma unroll
        for (int g = 0; g < 4; ++g) p[g] = page_part(C, C.k, head, ids, g, ((b * ATTN_KEYS + 16 * g) & mask) * C.dim, on);
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
            p[i] = page_part(C, C.v, head, ids, g, (b * ATTN_KEYS + 16 * g) & mask, on);
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

    __device__ __forceinline__ u32x4_t key(int t, int k) const {
        return *reinterpret_cast<const u32x4_t*>(lds + k_read[k & 1] + k / 2 * 128 + 4 * t * DIM);
    }
    __device__ __forceinline__ u32x4_t value(int d) const { return *reinterpret_cast<const u32x4_t*>(lds + v_read + d * 1024); }
};

// Blocks first, first + step, ... < last of a tile's keys for one wave.  No branch divides lanes in here: the compiler may
// leave them apart in the loop around the products, and may place copies of other lanes' registers before they are back.
template <int DIM, bool BF16, int RB>
__device__ __forceinline__ void attend(const AttnArgs& A, const AttnStage<DIM>& S, AttnRows<DIM, BF16, RB, true>& R, const Seq& q,
                                       const Tile& x, int s, int head, int first, int last, int step) {
    constexpr int DT = DIM / 16;
    if (first >= last) return;
    const CacheView& C = A.c;
    const int g16 = threadIdx.x & 48;
    const Pages P(C, q, s);
    const auto key = [&](int t, int k) { return S.key(t, k); };
    const auto value = [&](int d) { return S.value(d); };
    u32x4_t kreg[DT], vreg[DT];
    int ids = P.of(C, first), raw = P.raw(C, min(first + step, last - 1));    // two blocks ahead: loads come back in order
    S.load_k(C, head, first, ids, true, kreg);
    float ks = scale_of(C, C.k_scale, ids, head), vs = scale_of(C, C.v_scale, ids, head);
    S.load_v(C, head, first, ids, true, vreg);
    bool nans = false;
    for (int b = first; b < last; b += step) {
        const bool more = b + step < last;
        const int id = ids;
        ids = P.of(C, min(b + step, last - 1), moved(raw));
        raw = P.raw(C, min(b + 2 * step, last - 1));
        S.put_k(kreg);
        const float ks_now = moved(ks), vs_now = moved(vs);
        S.load_k(C, head, b + step, ids, more, kreg);
        ks = scale_of(C, C.k_scale, ids, head);
        vs = scale_of(C, C.v_scale, ids, head);
        S.put_v(vreg);
        S.load_v(C, head, b + step, ids, more, vreg);
        // one step for both kinds of blocks: with one each, the compiler keeps the sums twice
        const bool masked = uniform((int)masked_block(C, x, b, id, ks_now, vs_now)) != 0;
        nans |= R.step(A, masked, ks_now, vs_now, !masked || valid_page(C, id), b * ATTN_KEYS + g16, x.lo, x.hi, key, value);
    }
    if (!nans) return;
    for (int b = first; b < last; b += step) {
        const int id = P.of(C, b);
        S.load_v(C, head, b, id, true, vreg);
        S.put_v(vreg);
        R.add_nans(valid_page(C, id), scale_of(C, C.v_scale, id, head), b * ATTN_KEYS + g16, x.lo, x.hi, value);
    }
}

template <int DIM, int RB>
struct AttnSize {
    static constexpr int ROWS = 16 * RB, PITCH = DIM + 4;
    static constexpr int JOIN = ATTN_WAVES * ROWS * (PITCH + 2) * 4, STAGE = ATTN_WAVES * AttnStage<DIM>::BYTES;
    static constexpr int LDS = JOIN > STAGE ? JOIN : STAGE;       // the blocks of the waves, then their sums
    static constexpr int WAVES_EU = DIM <= 128 ? 2 : 1;
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

// Rows of q whose tokens no sequence has, by A.clear.
__device__ __forceinline__ void clear_rows(const AttnArgs& A) {
    const CacheView& C = A.c;
    if (!A.clear || !C.starts) return;
    int largest = 0;
#pragma unroll 4
    for (int s0 = 0; s0 <= C.seqs; s0 += 64) {
        const int s = s0 + (threadIdx.x & 63);
        largest = max(largest, s <= C.seqs ? get_start(C, s) : 0);
    }
    const int a = get_start(C, 0), b = read_lane(wave_max_scan(largest), 63);
    const int rows = C.tokens - (b - a);
    const int64_t each = (int64_t)A.heads * C.dim / 8;
    for (int i = blockIdx.x; i < rows; i += gridDim.x) {
        const int64_t t = i < a ? i : i + (b - a);
        if (A.clear == 1)
            for (int64_t j = threadIdx.x; j < each; j += blockDim.x)
                reinterpret_cast<u32x4_t*>(A.out + t * A.heads * C.dim)[j] = u32x4_t{0, 0, 0, 0};
        if (A.lse)
            for (int j = threadIdx.x; j < A.heads; j += blockDim.x) A.lse[t * A.heads + j] = -__builtin_inff();
    }
}

// Units are (cache head, tile, block of keys), in this order; a workgroup has an
// equal share of them, next to each other, whatever sequences they are of.  Where the
// shares are hardly larger then, a share is of one tile: a second one costs a workgroup
// what about four units a wave do (16 sequences of 5 tokens, window 1024: 24.9 -> 21.1 us;
// 24 sequences of 1 token: 25.8 -> 20.7).  A tile whose blocks one workgroup has all is
// finished; of the others each workgroup leaves a partial result: in its first place
// where the tile began before its share, in its second where it goes on behind it.
// Without a place for partial results a workgroup has a tile, the last ones first (of a
// prompt the longest).
//
// Two workgroups are on a CU, and the waves of the first go first: where instructions
// bound it, 65 blocks of 64 keys and 128 rows take the first 112 us and the second 154.
// So there the first ones (the first half of an XCD's) have ATTN_FIRST : 16 - ATTN_FIRST
// of the units, where these are 16 a workgroup at least (a chunk of 512 behind 16384
// keys: 171-176 us, 180 with equal shares; 10 : 6 is like 9 : 7).
constexpr int ATTN_FIRST = 9;

template <int ROWS>
struct Work {
    static constexpr bool UNEVEN = ROWS >= 64;
    int64_t all, u, u1, share;   // units: of the call, the next, the end of the workgroup's, how many a workgroup has
    bool uneven;
    int me, s, t, head;
    int done, n, here;           // of the tile: blocks before the next unit, all of them, those of this workgroup
    Seq q;
    Tile x;

    // False if there is nothing for this workgroup.
    __device__ __forceinline__ bool find(const AttnArgs& A) {
        const CacheView& C = A.c;
        all = u = u1 = share = 0;
        uneven = false;
        me = blockIdx.x;
        t = head = done = 0;
        if (A.part) {
            int64_t mine = 0, piece = 0;                          // tiles of this lane's sequences
            int pieces = -1;                                      // a share is of one tile; -1: not known yet
            const Found f = find_seq(C, [&](const Seq& x) {
                if (pieces < 0) mine += tiles_of(A, x, ROWS);
                return units_of(A, x, ROWS, pieces > 0 ? share : 1);
            }, [&](int64_t total) {
                int64_t busy;
                if (pieces < 0) {
                    // (starts that decrease may make more units than the launch was bounded for)
                    const int64_t wgs = min(A.most, (int)gridDim.x), tiles = (C.seqs == 1 ? mine : read_lane(wave_scan(mine), 63)) * C.kv;
                    all = total * C.kv;
                    share = piece = A.least;
                    pieces = 1;
                    if (all > (wgs - tiles) * piece) {
                        share = max((int64_t)1, divide(all + wgs - 1, wgs));
                        // no more than wgs pieces have this length, or the rest of a tile
                        if (wgs > tiles) piece = max(piece, divide(all + wgs - tiles - 1, wgs - tiles));
                        pieces = wgs > tiles && piece <= share + 4 * A.least;
                    }
                    if (pieces) return COUNT_AGAIN;
                }
                if (pieces) {
                    busy = total * C.kv;
                    if (busy > min(A.most, (int)gridDim.x) && share != piece) {
                        share = piece;                            // those of the shares' length are too many
                        return COUNT_AGAIN;
                    }
                } else {
                    busy = divide(all + share - 1, share);
                    uneven = UNEVEN && all >= 16 * (int64_t)A.most && (int)gridDim.x == A.most && A.most % (2 * XCDS) == 0;
                    if (uneven) busy = A.most;
                }
                if (me >= busy) return (int64_t)-1;
                me = by_xcd(me, (int)busy);
                u = begin_of(A, me);
                u1 = min(begin_of(A, me + 1), all);
                const int64_t at = pieces ? me : u;
                head = (int)divide(at, total);
                return at - head * total;
            });
            if (threadIdx.x == 0) A.shared[me].last = -1;        // nothing to join, unless a tile goes on behind the share
            if (f.s < 0) return false;
            s = f.s;
            q = f.q;
            int64_t left = f.unit;
            for (;; ++t) {
                x = get_tile(A, q, t, ROWS);
                n = blocks_of(x);
                const int64_t units = pieces ? divide(n + share - 1, share) : n;
                if (left < units) break;
                left -= units;
            }
            if (pieces) {
                left *= share;
                u1 = u + min(share, n - left);
            }
            done = (int)left;
        } else {
            int tile;
            if (!tile_by_xcd(blockIdx.x, A.tiles, C.kv, tile, head)) return false;
            const int64_t at = A.tiles - 1 - tile;
            if (C.starts) {
                const Found f = find_slot(C, at, [&](int64_t token, int64_t i) { return token * A.group / ROWS + i; });
                if (f.s < 0 || f.unit >= tiles_of(A, f.q, ROWS)) return false;
                s = f.s;
                q = f.q;
                t = (int)f.unit;
            } else {
                const int each = (A.group + ROWS - 1) / ROWS;
                s = (int)at / each;
                t = (int)at - s * each;
                q = get_seq(C, s, 0);
            }
            x = get_tile(A, q, t, ROWS);
            n = blocks_of(x);
            u1 = n;
        }
        measure();
        return true;
    }

    // The first unit of workgroup j.
    __device__ __forceinline__ int64_t begin_of(const AttnArgs& A, int j) const {
        if (!UNEVEN || !uneven) return share * j;
        const int half = A.most / (2 * XCDS), p = j % (2 * half);
        return divide(all * (8 * (j - p) + min(p, half) * ATTN_FIRST + max(p - half, 0) * (16 - ATTN_FIRST)), 8 * A.most);
    }

    __device__ __forceinline__ void measure() {
        const int64_t want = u1 - u;
        here = (int)(n - done < want ? n - done : want);
    }
    __device__ __forceinline__ int first() const { return x.lo / ATTN_KEYS + done; }
    __device__ __forceinline__ int last() const { return min(first() + here, (x.hi + ATTN_KEYS - 1) / ATTN_KEYS); }
    __device__ __forceinline__ bool whole() const { return here == n; }

    // Where a partial result goes, of `size` floats each; tells the join of a tile that begins here.
    __device__ __forceinline__ float* part(const AttnArgs& A, int size) const {
        if (done == 0 && threadIdx.x == 0) {
            int last = me;
            if (UNEVEN && uneven)
                while (begin_of(A, last + 1) < u + n) ++last;
            else
                last = (int)divide(u + n - 1, share);
            last = min(last, (int)gridDim.x - 1);
            A.shared[me] = SharedTile{q.first, x.r0, x.rows, head, last};
        }
        return A.part + ((int64_t)me * 2 + (done == 0 ? 1 : 0)) * size;
    }

    // The next tile of the workgroup's units; false behind the last.
    __device__ __forceinline__ bool next(const AttnArgs& A) {
        const CacheView& C = A.c;
        u += here;
        if (u >= u1) return false;
        done = 0;
        if (++t == tiles_of(A, q, ROWS)) {
            t = 0;
            int before = q.first + q.n;
            do {
                if (++s == C.seqs) {
                    s = before = 0;
                    ++head;
                }
                q = get_seq(C, s, before);
                before = q.first + q.n;
            } while (q.n == 0);
        }
        x = get_tile(A, q, t, ROWS);
        n = blocks_of(x);
        measure();
        return true;
    }
};

// Few rows a sequence: the four waves of a workgroup go through a tile's blocks in
// turn, each with a place of its own in LDS, and join their sums there.  Bound by memory
// where there is much of it: 64 ragged contexts of up to 8192, 593 MB, 121 us (4.9 TB/s);
// one of 131072, 268 MB, 48 us and 5 for the join.  A short call is a chain: lookup,
// first loads, a block's instructions, join (one token of 1000 keys: 11 us with the
// join kernel).  Two workgroups of heads of up to 128 channels are on a CU.
template <int DIM, bool BF16, int RB>
__global__ __launch_bounds__(ATTN_WAVES * 64, (AttnSize<DIM, RB>::WAVES_EU)) void fp8_attention_kernel(AttnArgs A) {
    typedef AttnSize<DIM, RB> Z;
    extern __shared__ __attribute__((aligned(16))) float lds[];
    const CacheView& C = A.c;
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), r = lane & 15, g = lane >> 4;
    clear_rows(A);
    Work<Z::ROWS> w;
    if (!w.find(A)) return;
    const AttnStage<DIM> S(C, reinterpret_cast<char*>(lds) + wave * AttnStage<DIM>::BYTES);
    float* sums = lds;                                          // [wave][row][PITCH]
    float* ml = lds + ATTN_WAVES * Z::ROWS * Z::PITCH;          // [wave][row][2]
    for (;;) {
        {
            AttnRows<DIM, BF16, RB, true> R;
            R.begin(A, w.q, w.x.r0, w.x.rows, w.head);
            attend(A, S, R, w.q, w.x, w.s, w.head, w.first() + wave, w.last(), ATTN_WAVES);
            __syncthreads();
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
                const int row = 16 * rb + r;
                const float l = R.row_sum(rb);
                ml[(wave * Z::ROWS + row) * 2] = R.m[rb];       // by four lanes alike: no branch while the sums are live
                ml[(wave * Z::ROWS + row) * 2 + 1] = l;
#pragma unroll
                for (int d = 0; d < DIM / 16; ++d) {
                    float4_t v;
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] = ldexpf(R.o[d][rb][i], R.back(rb));
                    *reinterpret_cast<float4_t*>(sums + (wave * Z::ROWS + row) * Z::PITCH + 16 * d + 4 * g) = v;
                }
            }
        }
        __syncthreads();
        float* part = w.whole() ? nullptr : w.part(A, Z::PART);
        const int quads = C.dim / 4;
        for (int i = tid; i < w.x.rows * quads; i += ATTN_WAVES * 64) {
            const int row = i / quads, d = (i - row * quads) * 4;
            float m = ATTN_LOW, l = 0.f;
#pragma unroll
            for (int j = 0; j < ATTN_WAVES; ++j) m = fmaxf(m, ml[(j * Z::ROWS + row) * 2]);
            float4_t v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < ATTN_WAVES; ++j) {
                const float f = __builtin_amdgcn_exp2f(ml[(j * Z::ROWS + row) * 2] - m);
                l += f * ml[(j * Z::ROWS + row) * 2 + 1];
                const float4_t a = *reinterpret_cast<const float4_t*>(sums + (j * Z::ROWS + row) * Z::PITCH + d);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = fmaf(f, a[e], v[e]);
            }
            if (!part) {
                const int at = (w.x.r0 + row) / A.group, h = w.head * A.group + w.x.r0 + row - at * A.group;
                const int64_t o = (int64_t)(w.q.first + at) * A.heads + h;
                float lse;
                const float f = finish_row(A, h, m, l, lse);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] *= f;
                store_row4<BF16>(A.out + o * C.dim + d, v);
                if (A.lse && d == 0) A.lse[o] = lse;
            } else {
                *reinterpret_cast<float4_t*>(part + row * DIM + d) = v;
                if (d == 0) {
                    part[Z::ROWS * DIM + 2 * row] = m;
                    part[Z::ROWS * DIM + 2 * row + 1] = l;
                }
            }
        }
        if (!w.next(A)) break;
        __syncthreads();                                        // the sums' places hold blocks again
    }
}

// ---------------------------------------------------------------- many rows

// Keys and values of a block for a whole workgroup, straight from memory to LDS, in
// two places that take turns.  A load's 64 chunks of 16 bytes lie in LDS in the order
// of the lanes, so it is the lane's chunk in memory that is XORed with its row.
//   keys    [DIM / SUB][64][SUB bytes]
//   values  [pieces][DIM][16 << lg bytes]: the tokens of a page, 64 at most
template <int DIM>
struct AttnShare {
    static constexpr int SUB = DIM % 128 == 0 ? 128 : 64, CS = SUB / 16, SUBS = DIM / SUB, KEYS = 64 / CS;
    static constexpr int LOADS = DIM / 16 / ATTN_WAVES;       // of a wave, for the keys or the values
    static constexpr int K_BYTES = ATTN_KEYS * DIM, BYTES = 2 * K_BYTES;

    char* lds;
    int k_read[2], v_read;
    uint32_t k_off[SUBS], v_off;
    int lg, wave;

    __device__ __forceinline__ AttnShare(const CacheView& C, char* lds_, int wave_) : lds(lds_), wave(wave_) {
        const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
        const int key = lane / CS, place = lane % CS;
        const int sw = SUB == 128 ? key & 3 : (key >> 1) & 1;
#pragma unroll
        for (int i = 0; i < SUBS; ++i) {
            // keys 16 .. 31 and 48 .. 63 have another bit
            const int c = i * SUB + ((((place ^ sw) << 4)) ^ ((wave & 1) ? SUB / 2 : 0));
            k_off[i] = c < C.dim ? key * C.dim + c : OUTSIDE;  // behind the row's end: zeros
        }
        const int sr = SUB == 128 ? (r & 3) | (r >> 2 & 1) << 2 : (r >> 1 & 1) | (r >> 2 & 1) << 1;
        const int row = (16 * (r >> 2) + (r & 3)) * SUB;
        k_read[0] = row + ((g ^ sr) << 4);
        k_read[1] = SUB == 128 ? row + (((4 + g) ^ sr) << 4) : k_read[0] + ATTN_KEYS * SUB;
        lg = min(C.page_shift, 6) - 4;
        // a row of `1 << lg` chunks; eight lanes meet every bank once
        const int channel = lane >> lg, mask = (1 << lg) - 1;
        const auto swap = [&](int c) { return lg == 2 ? c >> 1 & 3 : lg == 1 ? c >> 2 & 1 : 0; };
        v_off = ((channel + (wave & mask) * (DIM >> lg)) << C.page_shift) + (((lane & mask) ^ swap(channel)) << 4);
        v_read = K_BYTES + ((((g >> lg) * DIM + r) << lg) + ((g & mask) ^ swap(r))) * 16;
    }

    // This wave's loads of block b: keys 16 wave .. 16 wave + 15, and its part of the piece of values that they are in. One
    // page has them all.
    __device__ __forceinline__ void load(const CacheView& C, int head, int b, int ids, bool on, int place) const {
        const int mask = (1 << C.page_shift) - 1, at = b * ATTN_KEYS;
        const int id = __builtin_amdgcn_readlane(ids, 16 * wave);
        const bool is = on && valid_page(C, id);
        const uint32_t bytes = (uint32_t)C.dim << C.page_shift;
        const uint64_t page = (uint64_t)(uint32_t)(is ? id : 0) * ((uint32_t)C.kv * bytes) + head * bytes;
        const uint32_t k_at = ((at + 16 * wave) & mask) * C.dim, v_at = (at + (wave >> lg << lg) * 16) & mask;
        const __amdgpu_buffer_rsrc_t k = __builtin_amdgcn_make_buffer_rsrc(C.k + page + k_at, 0, is ? bytes - k_at : 0, 0x27000);
        const __amdgpu_buffer_rsrc_t v = __builtin_amdgcn_make_buffer_rsrc(C.v + page + v_at, 0, is ? bytes - v_at : 0, 0x27000);
        char* to = lds + place * BYTES + wave * (16 * SUB);
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int sub = i * KEYS / 16, key = i * KEYS % 16;
            load_to_lds(k, to + (sub * ATTN_KEYS + key) * SUB, k_off[sub], key * C.dim);
        }
        to = lds + place * BYTES + K_BYTES + wave * (LOADS * 1024);
#pragma unroll
        for (int i = 0; i < LOADS; ++i)                       // behind the last channel: zeros
            load_to_lds(v, to + i * 1024, v_off + (i << (6 - lg + C.page_shift)), 0);
    }

    __device__ __forceinline__ u32x4_t key(int place, int t, int k) const {
        return *reinterpret_cast<const u32x4_t*>(lds + place * BYTES + k_read[k & 1] +
                                                 k / 2 * (ATTN_KEYS * 128) + 4 * t * SUB);
    }
    __device__ __forceinline__ u32x4_t value(int place, int d) const {
        return *reinterpret_cast<const u32x4_t*>(lds + place * BYTES + v_read + (d << (8 + lg)));
    }
};

template <int DIM, int RB>
struct ShareSize {
    static constexpr int ROWS = ATTN_WAVES * 16 * RB;
    static constexpr int LDS = 2 * AttnShare<DIM>::BYTES;
    static constexpr int PART = ROWS * (DIM + 2);
    static_assert(LDS >= ROWS * DIM * 2, "a tile's results go through the blocks' places");
};

// Many rows a sequence: each wave has rows of its own, all go through a tile's blocks
// together, with one barrier a block; the next block is on its way meanwhile.  Bound by
// vector instructions: a wave widens the codes of a whole block for its 32 rows (16 where
// heads are wider than 128, for the registers: 329 us where 32 rows spilled in 522), and
// the exponentials come on top.  512 tokens behind 16384 keys, 32 heads over 8 of 128:
// 165-175 us, 790 TFLOP/s, the matrix unit 41% busy.  The 8-bit product on the codes as
// they are (queries in two e4m3 parts) took 167 for 180, but its sums are not fp32's:
// logits were up to 2^-16 of their terms' sum off.  256 rows a workgroup of eight waves: no faster.
template <int DIM, bool BF16, int RB>
__global__ __launch_bounds__(ATTN_WAVES * 64, 2) void fp8_attention_rows_kernel(AttnArgs A) {
    typedef ShareSize<DIM, RB> Z;
    constexpr int OWN = 16 * RB;
    extern __shared__ __attribute__((aligned(16))) char share_lds[];
    const CacheView& C = A.c;
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), r = lane & 15, g = lane >> 4;
    clear_rows(A);
    Work<Z::ROWS> w;
    if (!w.find(A)) return;
    const AttnShare<DIM> S(C, share_lds, wave);
    for (;;) {
        const int first = w.first(), last = w.last();
        // this wave's rows; a wave without any takes the first one's, and stores nothing
        const int rows = w.x.rows - wave * OWN;
        const Tile x = get_tile(A, w.q, w.t * ATTN_WAVES + (rows > 0 ? wave : 0), OWN);
        AttnRows<DIM, BF16, RB, !BF16> R;
        R.begin(A, w.q, x.r0, x.rows, w.head);
        const Pages P(C, w.q, w.s);
        bool nans = false;
        if (first < last) {
            // What a block needs is asked for a whole block before, so that the wait at its beginning is for all of it alike.
            int raw = P.raw(C, first);
            int ids = P.of(C, first, raw);
            float ks = scale_of(C, C.k_scale, ids, w.head), vs = scale_of(C, C.v_scale, ids, w.head);
            S.load(C, w.head, first, ids, true, 0);
            raw = P.raw(C, min(first + 1, last - 1));
            int id, key0, place;
            float ks_now, vs_now;
            // Block b begins; 0: these rows see nothing of it, 1: all of them see it whole, 2: some do not.
            const auto top = [&](int b) {
                place = (b - first) & 1;
                id = ids;
                key0 = b * ATTN_KEYS + (lane & 48);
                wait_loads();
                bare_barrier();                                 // block b is there, and nobody reads the other place
                ks_now = moved(ks);
                vs_now = moved(vs);
                ids = P.of(C, b + 1, moved(raw));
                raw = P.raw(C, min(b + 2, last - 1));
                ks = scale_of(C, C.k_scale, ids, w.head);
                vs = scale_of(C, C.v_scale, ids, w.head);
                S.load(C, w.head, b + 1, ids, b + 1 < last, place ^ 1);
                if (uniform((int)(rows <= 0 || b * ATTN_KEYS >= x.hi || (b + 1) * ATTN_KEYS <= x.lo))) return 0;
                return uniform(masked_block(C, x, b, id, ks_now, vs_now) ? 2 : 1);
            };
            const auto key = [&](int t, int k) { return S.key(place, t, k); };
            const auto value = [&](int d) { return S.value(place, d); };
            // blocks that are seen whole have a loop of their own
            int b = first;
            for (int mode = top(b);;) {
                while (mode == 1) {
                    R.step(A, false, ks_now, vs_now, true, key0, 0, 0, key, value);
                    mode = ++b < last ? top(b) : -1;
                }
                if (mode < 0) break;
                if (mode == 2) nans |= R.step(A, true, ks_now, vs_now, valid_page(C, id), key0, x.lo, x.hi, key, value);
                if (++b == last) break;
                mode = top(b);
            }
            wait_loads();                                       // a load of nothing writes zeros
            if (__syncthreads_or(nans)) {
                for (int b = first; b < last; ++b) {
                    const int id = P.of(C, b);
                    S.load(C, w.head, b, id, true, 0);
                    wait_loads();
                    bare_barrier();
                    R.add_nans(valid_page(C, id), scale_of(C, C.v_scale, id, w.head), b * ATTN_KEYS + (lane & 48), x.lo, x.hi,
                               [&](int d) { return S.value(0, d); });
                    wait_loads();
                    bare_barrier();
                }
            }
        }
        float lse[RB];
        if (w.whole()) {
            // through LDS: rows leave it 16 bytes a lane
            uint16_t* out = reinterpret_cast<uint16_t*>(share_lds) + wave * OWN * DIM;
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
                const int row = 16 * rb + r, of = x.r0 + min(row, x.rows - 1), at = of / A.group;
                const int swap = (row & 7) << 3;                // chunks of 16 bytes XORed with their row, for the banks
                const float f = finish_row(A, w.head * A.group + of - at * A.group, R.m[rb], R.row_sum(rb), lse[rb]);
#pragma unroll
                for (int d = 0; d < DIM / 16; ++d) {
                    float4_t v;
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] = ldexpf(R.o[d][rb][i], R.back(rb)) * f;
                    store_row4<BF16>(out + row * DIM + (16 * d + 4 * g ^ swap), v);
                }
            }
            asm volatile("" ::: "memory");
            const int chunks = C.dim / 8;
            for (int i = lane; i < (rows > 0 ? x.rows : 0) * chunks; i += 64) {
                const int row = i / chunks, d = (i - row * chunks) * 8, of = x.r0 + row, at = of / A.group;
                const int64_t o = (int64_t)(w.q.first + at) * A.heads + w.head * A.group + of - at * A.group;
                *reinterpret_cast<u32x4_t*>(A.out + o * C.dim + d) = *reinterpret_cast<const u32x4_t*>(out + row * DIM + (d ^ (row & 7) << 3));
            }
            if (A.lse && rows > 0 && g == 0) {
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) {
                    const int row = 16 * rb + r, of = x.r0 + row, at = of / A.group;
                    if (row < x.rows)
                        A.lse[(int64_t)(w.q.first + at) * A.heads + w.head * A.group + of - at * A.group] = lse[rb];
                }
            }
        } else {
            float* part = w.part(A, Z::PART);
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
                const int row = wave * OWN + 16 * rb + r;      // rows behind the last have room too
#pragma unroll
                for (int d = 0; d < DIM / 16; ++d) {
                    float4_t v;
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] = ldexpf(R.o[d][rb][i], R.back(rb));
                    *reinterpret_cast<float4_t*>(part + row * DIM + 16 * d + 4 * g) = v;
                }
                part[Z::ROWS * DIM + 2 * row] = R.m[rb];
                part[Z::ROWS * DIM + 2 * row + 1] = R.row_sum(rb);
            }
        }
        if (!w.next(A)) break;
        __syncthreads();                                        // the results' places hold blocks again
    }
}

// A tile that several workgroups share, joined: blockIdx.x is the workgroup that
// begins it, blockIdx.y takes every gridDim.y-th row.  A row's threads are groups that
// each take some of the partial results, four channels a thread; the groups' sums
// meet in LDS.  3 to 5 us, mostly a launch's; 9 where the partial results are 34 MB (512
// workgroups of 128 rows).  A launch of its own: the last workgroup to come would need
// counters that are zero, and the caller's scratch is not.
template <int DIM, bool BF16, int ROWS>
__global__ __launch_bounds__(ATTN_WAVES * 64) void fp8_attention_join_kernel(AttnArgs A) {
    constexpr int PART = ROWS * (DIM + 2), QUADS = DIM / 4, GROUPS = ATTN_WAVES * 64 / QUADS;
    __shared__ float4_t sums[GROUPS][QUADS];
    __shared__ float ml[GROUPS][2];
    const CacheView& C = A.c;
    const SharedTile x = A.shared[blockIdx.x];
    const int first = blockIdx.x, group = threadIdx.x / QUADS, d = (threadIdx.x - group * QUADS) * 4;
    if (x.last < 0) return;
    const auto take = [&](int w, int row, float& m, float& l, float4_t& v) {
        const float* p = A.part + ((int64_t)w * 2 + (w == first ? 1 : 0)) * PART;
        const float pm = p[ROWS * DIM + 2 * row], pl = p[ROWS * DIM + 2 * row + 1];
        const float4_t a = *reinterpret_cast<const float4_t*>(p + row * DIM + d);
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
