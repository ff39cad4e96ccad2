// A paged cache of e4m3 keys and values with one power-of-two scale for each page
// and head, and the write into it.
//
//   k  [pages][kv][page][dim]   k_scale [pages][kv]
//   v  [pages][kv][dim][page]   v_scale [pages][kv]      (a value's tokens are neighbours)
//
// A power of two as the scale keeps a value's bits where the scale of a begun page
// grows (but for those that fall below e4m3's normal range), and e4m3's relative
// error does not depend on where in its range a value lies.  A begun page that has
// another scale is written by that one.
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

// A sequence's tokens in a call, its length and how many of its keys have room.  A token
// keeps its position where the length is past the table's row: those behind the room have
// no place, and do not take that of others.  No index leaves a buffer: pages follow from
// `end`, and starts are cut to the call's tokens.  A start that is less than one before it
// counts as the largest before it: no token has two sequences.
struct Seq {
    int first, n, len, end;
};

__device__ __forceinline__ int get_start(const CacheView& C, int s) { return min(max(C.starts[s], 0), C.tokens); }

__device__ __forceinline__ void get_length(const CacheView& C, int s, Seq& q) {
    q.len = max(C.lengths[s], 0);
    q.end = min(q.len, C.width << C.page_shift);                // the room is below 2^31
}

// before: the largest start before sequence s
__device__ __forceinline__ Seq get_seq(const CacheView& C, int s, int before) {
    Seq q;
    if (C.starts) {
        q.first = max(get_start(C, s), before);
        q.n = max(get_start(C, s + 1) - q.first, 0);
    } else {
        q.first = s;
        q.n = 1;
    }
    get_length(C, s, q);
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

// Inclusive largest values, of values that are not negative.
__device__ __forceinline__ int wave_max_scan(int v) {
    v = max(v, lane_of<0x111, 0xf>(v, 0));
    v = max(v, lane_of<0x112, 0xf>(v, 0));
    v = max(v, lane_of<0x114, 0xf>(v, 0));
    v = max(v, lane_of<0x118, 0xf>(v, 0));
    v = max(v, lane_of<0x142, 0xa>(v, 0));
    return max(v, lane_of<0x143, 0xc>(v, 0));
}

// Each lane's of the sequences s0 .. s0 + 63; `before` goes on to the next 64.
__device__ __forceinline__ Seq lane_seq(const CacheView& C, int s0, int& before) {
    const int s = s0 + (threadIdx.x & 63);
    int first = before;
    if (C.starts) {
        first = max(before, wave_max_scan(s < C.seqs ? get_start(C, s) : 0));
        before = read_lane(first, 63);
    }
    return s < C.seqs ? get_seq(C, s, first) : Seq{0, 0, 0, 0};
}

// a / b, 0 <= a, 0 < b; in 32 bits where both fit, and else bit by bit: a short call
// spends much of its time on fetching its instructions, and these are few.
__device__ __forceinline__ int64_t divide(int64_t a, int64_t b) {
    if (((uint64_t)(a | b) >> 32) == 0) return (int64_t)((uint32_t)a / (uint32_t)b);
    uint64_t r = 0, x = (uint64_t)a;
#pragma unroll 1
    for (int i = 0; i < 64; ++i) {
        r = r << 1 | x >> 63;
        x <<= 1;
        if (r >= (uint64_t)b) {
            r -= (uint64_t)b;
            x |= 1;
        }
    }
    return (int64_t)x;
}

// The sequence that a unit of all sequences' units lies in; count(q) units each.  The
// unit is at(total), total being all of them, or COUNT_AGAIN, where at has changed what a
// unit is; s is -1 where it lies behind them.  Every wave looks by itself: up to 64
// sequences are one load and one scan, one sequence is not divided over lanes.
constexpr int64_t COUNT_AGAIN = -2;
struct Found {
    int s;
    int64_t unit;                // within the sequence
    Seq q;
};

template <typename Count, typename At>
__device__ __forceinline__ Found find_seq(const CacheView& C, Count&& count, At&& at) {
    Found f{-1, 0, Seq{0, 0, 0, 0}};
    const auto look = [&](int s0, const Seq& q, int64_t c, int64_t before, int64_t sum, int64_t want) {
        before += sum - c;
        const uint64_t hit = __builtin_amdgcn_ballot_w64(want >= before && want < before + c);
        if (!hit) return;
        const int l = __builtin_ctzll(hit);
        f.s = s0 + l;
        f.unit = want - read_lane(before, l);
        f.q = Seq{read_lane(q.first, l), read_lane(q.n, l), read_lane(q.len, l), read_lane(q.end, l)};
    };
    if (C.seqs == 1) {
        f.q = get_seq(C, 0, 0);
        for (;;) {
            const int64_t c = uniform(count(f.q)), want = at(c);
            if (want == COUNT_AGAIN) continue;
            if (want >= 0 && want < c) f.s = 0;
            f.unit = want;
            break;
        }
    } else if (C.seqs <= 64) {
        int before = 0;
        const Seq q = lane_seq(C, 0, before);
        for (;;) {
            const int64_t c = count(q), sum = wave_scan(c), want = at(read_lane(sum, 63));
            if (want == COUNT_AGAIN) continue;
            look(0, q, c, 0, sum, want);
            break;
        }
    } else {
        // A lane counts `each` neighbouring sequences; those of the lane that has the unit are then a lane each.
        const int lane = threadIdx.x & 63, each = (C.seqs + 63) / 64, from = min(lane * each, C.seqs), to = min(from + each, C.seqs);
        int start = 0;
        if (C.starts) {
            for (int s = from; s < to; ++s) start = max(start, get_start(C, s));
            start = __shfl_up(wave_max_scan(start), 1);
            start = lane ? start : 0;                                         // the largest before the lane's
        }
        int64_t c, sum, want;
        do {
            c = 0;
            int before = start;
            for (int s = from; s < to; ++s) {
                const Seq q = get_seq(C, s, before);
                before = q.first;
                c += count(q);
            }
            sum = wave_scan(c);
            want = at(read_lane(sum, 63));
        } while (want == COUNT_AGAIN);
        const uint64_t hit = __builtin_amdgcn_ballot_w64(want >= sum - c && want < sum);
        if (!hit) return f;
        const int l = __builtin_ctzll(hit);
        int64_t before = read_lane(sum - c, l);
        int first = read_lane(start, l);
        for (int s0 = l * each; f.s < 0 && s0 < (l + 1) * each && s0 < C.seqs; s0 += 64) {
            const Seq q = lane_seq(C, s0, first);
            const int64_t n = s0 + lane < (l + 1) * each ? count(q) : 0, sums = wave_scan(n);
            look(s0, q, n, before, sums, want);
            before += read_lane(sums, 63);
        }
    }
    return f;
}

// The sequence that has the workgroups before(first token, s) up to before(first token
// behind it, s + 1), x among them: some more than it needs, but starts alone tell them,
// and the look ends where it is found (append to 1024 sequences of 3 tokens, 33000
// workgroups: 195 -> 123 us).
template <typename Before>
__device__ __forceinline__ Found find_slot(const CacheView& C, int64_t x, Before&& before) {
    Found f{-1, 0, Seq{0, 0, 0, 0}};
    const int lane = threadIdx.x & 63;
    int start = 0;
    for (int s0 = 0; s0 < C.seqs; s0 += 64) {
        const int s = s0 + lane;
        int first = s, end = s + 1;
        if (C.starts) {
            first = max(start, wave_max_scan(s < C.seqs ? get_start(C, s) : 0));
            end = max(first, s < C.seqs ? get_start(C, s + 1) : 0);
            start = read_lane(first, 63);
        }
        const int64_t lo = before((int64_t)first, (int64_t)s);
        const uint64_t hit = __builtin_amdgcn_ballot_w64(s < C.seqs && x >= lo && x < before((int64_t)end, (int64_t)s + 1));
        if (!hit) continue;
        const int l = __builtin_ctzll(hit);
        f.s = s0 + l;
        f.unit = x - read_lane(lo, l);
        f.q.first = read_lane(first, l);
        f.q.n = read_lane(end, l) - f.q.first;
        get_length(C, f.s, f.q);
        break;
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
    return q.end > from ? ((q.end - 1) >> C.page_shift) - (from >> C.page_shift) + 1 : 0;
}

// Eight neighbouring values (16-byte aligned), as they are in memory.
template <int K>
struct Eight {
    u32x4_t u[K == OUT_F32 ? 2 : 1];

    __device__ __forceinline__ void load(const void* p, int64_t at) {
        const u32x4_t* from = reinterpret_cast<const u32x4_t*>(static_cast<const char*>(p) + at * (K == OUT_F32 ? 4 : 2));
        u[0] = from[0];
        if constexpr (K == OUT_F32) u[1] = from[1];
    }
    // as fp32, an infinity as a NaN
    __device__ __forceinline__ void finite(float (&v)[8]) const {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if constexpr (K == OUT_F32) v[j] = __uint_as_float(u[j / 4][j % 4]);
            else if constexpr (K == OUT_BF16) v[j] = __uint_as_float(j & 1 ? u[0][j / 2] & 0xffff0000u : u[0][j / 2] << 16);
            else v[j] = f16_bits_to_f32((uint16_t)(u[0][j / 2] >> (16 * (j & 1))));
            v[j] = fabsf(v[j]) == __builtin_inff() ? __builtin_nanf("") : v[j];
        }
    }
};

// One value, from 64 bits, as an e4m3 code.
__device__ __forceinline__ uint8_t code_of(double v) {
    const float f = to_odd(v);
    return (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(f, f, 0, false);
}
__device__ __forceinline__ uint8_t rescale1(uint8_t u, float by) {
    return code_of((double)__builtin_amdgcn_cvt_f32_fp8((int)u, 0) * (double)by);
}

// Four codes times a power of two, rounded to e4m3 again.
__device__ __forceinline__ uint32_t rescale4(uint32_t u, float by) {
    return pack_e4m3(__builtin_amdgcn_cvt_f32_fp8((int)u, 0) * by, __builtin_amdgcn_cvt_f32_fp8((int)u, 1) * by,
                     __builtin_amdgcn_cvt_f32_fp8((int)u, 2) * by, __builtin_amdgcn_cvt_f32_fp8((int)u, 3) * by);
}

// Byte c of each of four words, as one word each.
__device__ __forceinline__ void transpose4(uint32_t (&w)[4]) {
    const uint32_t a = __builtin_amdgcn_perm(w[1], w[0], 0x05010400u), b = __builtin_amdgcn_perm(w[3], w[2], 0x05010400u);
    const uint32_t c = __builtin_amdgcn_perm(w[1], w[0], 0x07030602u), d = __builtin_amdgcn_perm(w[3], w[2], 0x07030602u);
    w[0] = __builtin_amdgcn_perm(b, a, 0x05040100u);
    w[1] = __builtin_amdgcn_perm(b, a, 0x07060302u);
    w[2] = __builtin_amdgcn_perm(d, c, 0x05040100u);
    w[3] = __builtin_amdgcn_perm(d, c, 0x07060302u);
}

// A workgroup, or each wave of it where tokens are few (TEAM threads), has one page of
// one head, of the keys or of the values: the new tokens' largest magnitude, the scale,
// the old codes where it grew, the new ones.  The inputs stay in registers in between,
// the first APPEND_HOLD * TEAM chunks of eight (a workgroup's: 64 tokens of 256 values,
// 128 of 128); what a page has more is read twice.  A value's codes
// are turned in LDS: tokens of a channel are neighbours in the cache.  Four chunks of
// up to 2000 tokens, 8 heads of 128 (30 MB): 12 us; read twice and values gathered two
// bytes a load 18.4.
// 13 single tokens: 4.4 us, a chain of lookup, page, inputs, reduction and store.
constexpr int APPEND_HOLD = 8;

__host__ __device__ inline int append_lds(int page, int dim) { return page * (dim + 4); }

template <int K, int TEAM>
__global__ __launch_bounds__(APPEND_WAVES * 64) void fp8_cache_append_kernel(AppendArgs A) {
    constexpr int THREADS = TEAM, TEAMS = APPEND_WAVES * 64 / TEAM;
    extern __shared__ __attribute__((aligned(16))) char append_lds_[];
    __shared__ float most_of[APPEND_WAVES];
    const CacheView& C = A.c;
    const int tid = threadIdx.x % TEAM, team = uniform((int)threadIdx.x / TEAM), head = blockIdx.y * TEAMS + team;
    char* append_codes = append_lds_ + team * append_lds(1 << C.page_shift, C.dim);        // values: [page][dim + 4]
    const bool values = blockIdx.z;
    if (head >= C.kv) return;
    int s = blockIdx.x, nth = 0;
    Seq q;
    if (C.starts) {
        // pages that new tokens lie in: at most two more than they fill
        const Found f = find_slot(C, blockIdx.x, [&](int64_t token, int64_t i) { return (token >> C.page_shift) + 2 * i; });
        if (f.s < 0 || f.unit >= touched_pages(C, f.q)) return;
        s = f.s;
        nth = (int)f.unit;
        q = f.q;
    } else {
        q = get_seq(C, s, 0);
    }
    const int page = 1 << C.page_shift, base = q.len - q.n, from = max(base, 0);
    if (q.end <= from) return;
    const int at = (from >> C.page_shift) + nth;                                  // the page's place in the sequence
    const int id = C.table[s * C.table_stride + at];
    if ((unsigned)id >= (unsigned)C.pages) return;
    const int lo = max(from - (at << C.page_shift), 0), hi = min(q.end - (at << C.page_shift), page);
    const int64_t token = q.first + (at << C.page_shift) - base;                  // the token of the page's place 0
    const int64_t stride = values ? A.v_token : A.k_token;
    const int64_t in0 = token * stride + head * (values ? A.v_head : A.k_head);
    const void* in = values ? A.v : A.k;
    const int64_t block = (int64_t)id * C.kv + head;
    uint8_t* code = (values ? C.v : C.k) + (block << C.page_shift) * C.dim;
    float* scale = (values ? C.v_scale : C.k_scale) + block;

    const int per = C.dim >> 3, chunks = (hi - lo) * per;                         // chunks of eight, of a token and new
    const float each = __builtin_amdgcn_rcpf((float)per);                         // i / per: i is below 2^13, per 32 at most
    const auto where = [&](int i, int& t, int& d) {
        t = (int)(((float)i + 0.5f) * each);
        d = (i - t * per) * 8;
        t += lo;
        return in0 + t * stride + d;
    };
    Eight<K> held[APPEND_HOLD];
    int t, d;
#pragma unroll
    for (int c = 0; c < APPEND_HOLD; ++c) {
        if (c * THREADS >= chunks) break;
        if (tid + c * THREADS < chunks) held[c].load(in, where(tid + c * THREADS, t, d));
    }
    const float before = lo ? *scale : 0.f;
    // values: 16 tokens of four channels are a thread's; what is outside [lo, hi) goes back as it was, or rescaled below lo
    const int lg = C.page_shift - 4, last = (hi + 15) >> 4, fours = values ? C.dim / 4 << lg : 0;
    const auto row = [&](int i, int e) {
        return reinterpret_cast<u32x4_t*>(code + ((int64_t)((i >> lg << 2) + e) << C.page_shift) + (i & ((1 << lg) - 1)) * 16);
    };
    const auto outside = [&](int i) {
        const int t0 = (i & ((1 << lg) - 1)) * 16;
        return t0 < hi && (t0 < lo || t0 + 16 > hi);
    };
    u32x4_t old[4];
    if (tid < fours && outside(tid)) {
#pragma unroll
        for (int e = 0; e < 4; ++e) old[e] = *row(tid, e);
    }
    float most = 0.f;
    float x[8];
    const auto largest = [&](const Eight<K>& v) {
        v.finite(x);
#pragma unroll
        for (int j = 0; j < 8; ++j) most = fmaxf(most, fabsf(x[j]));
    };
#pragma unroll
    for (int c = 0; c < APPEND_HOLD; ++c) {
        if (c * THREADS >= chunks) break;
        if (tid + c * THREADS < chunks) largest(held[c]);
    }
    for (int i = tid + APPEND_HOLD * THREADS; i < chunks; i += THREADS) {
        Eight<K> v;
        v.load(in, where(i, t, d));
        largest(v);
    }
    most = wave_max(most, 0.f);
    if constexpr (TEAM > 64) {
        if ((tid & 63) == 0) most_of[tid >> 6] = most;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < APPEND_WAVES; ++w) most = fmaxf(most, most_of[w]);
    }
    const float now = fmaxf(QuantGroup(most, true).scale, before);
    const float inverse = 1.0f / now, by = before / now;
    const bool grew = lo && by != 1.0f;
    // A begun page's scale that is not this kernel's may be no power of two: then values are divided in 64 bits, where a
    // quotient that is not on a border of e4m3 stays on its side (a product with a rounded 1 / now does not).  One by one:
    // beside the others' code, eight a step cost every call 0.3 us (13 single tokens 4.2 -> 4.5), this costs it 0.1.
    const bool exact = ((__float_as_uint(now) | __float_as_uint(before)) & 0x7fffffu) == 0;
    const auto put = [&](int i, const Eight<K>& v) {
        where(i, t, d);
        v.finite(x);
        const uint32_t a = pack_e4m3(x[0] * inverse, x[1] * inverse, x[2] * inverse, x[3] * inverse);
        const uint32_t b = pack_e4m3(x[4] * inverse, x[5] * inverse, x[6] * inverse, x[7] * inverse);
        if (values) {
            uint32_t* to = reinterpret_cast<uint32_t*>(append_codes + t * (C.dim + 4) + d);
            to[0] = a;
            to[1] = b;
        } else {
            *reinterpret_cast<u32x2_t*>(code + t * C.dim + d) = u32x2_t{a, b};
        }
    };
#pragma unroll
    for (int c = 0; c < APPEND_HOLD; ++c) {
        if (c * THREADS >= chunks) break;
        if (tid + c * THREADS < chunks) put(tid + c * THREADS, held[c]);
    }
    for (int i = tid + APPEND_HOLD * THREADS; i < chunks; i += THREADS) {
        Eight<K> v;
        where(i, t, d);
        v.load(in, in0 + t * stride + d);
        put(i, v);
    }
    if (!exact) {
        // each thread's own codes again
#pragma unroll 1
        for (int i = 0; i < ((chunks - tid + THREADS - 1) / THREADS) * 8; ++i) {
            const int64_t from = where(tid + (i >> 3) * THREADS, t, d) + (i & 7);
            d += i & 7;
            const float v = load_kind<K>(in, from);
            const uint8_t u = code_of(fabsf(v) == __builtin_inff() ? __builtin_nan("") : (double)v / (double)now);
            if (values) append_codes[t * (C.dim + 4) + d] = (char)u;
            else code[t * C.dim + d] = u;
        }
    }
    if (!values) {
        if (grew && exact)
            for (int i = tid; i < lo * C.dim / 16; i += THREADS) {
                u32x4_t u = reinterpret_cast<u32x4_t*>(code)[i];
#pragma unroll
                for (int j = 0; j < 4; ++j) u[j] = rescale4(u[j], by);
                reinterpret_cast<u32x4_t*>(code)[i] = u;
            }
        if (grew && !exact) {
#pragma unroll 1
            for (int i = tid; i < lo * C.dim; i += THREADS) code[i] = rescale1(code[i], by);
        }
    } else {
        if constexpr (TEAM > 64) __syncthreads();
        else asm volatile("" ::: "memory");                     // LDS keeps a wave's order, the compiler has to
        const int first = grew ? 0 : lo >> 4;
        for (int i = tid; i < fours; i += THREADS) {
            const int group = i & ((1 << lg) - 1), d = i >> lg << 2, t0 = group * 16;
            if (group < first || group >= last) continue;
            u32x4_t made[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint32_t w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    w[e] = *reinterpret_cast<const uint32_t*>(append_codes + (t0 + 4 * j + e) * (C.dim + 4) + d);
                transpose4(w);
#pragma unroll
                for (int e = 0; e < 4; ++e) made[e][j] = w[e];
            }
            if (outside(i)) {
                if (i != tid) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) old[e] = *row(i, e);
                }
                const auto bytes_before = [&](int t) { return (uint32_t)((1ull << (8 * min(max(t, 0), 4))) - 1); };
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t below = bytes_before(lo - t0 - 4 * j), fresh = bytes_before(hi - t0 - 4 * j) & ~below;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t u = old[e][j], moved = grew && exact ? rescale4(u, by) : u;
                        made[e][j] = (made[e][j] & fresh) | (moved & below) | (u & ~(fresh | below));
                    }
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) *row(i, e) = made[e];
            if (grew && !exact) {
#pragma unroll 1
                for (int j = 0; j < 64; ++j) {
                    uint8_t* u = reinterpret_cast<uint8_t*>(row(i, j >> 4)) + (j & 15);
                    if (t0 + (j & 15) < lo) *u = rescale1(*u, by);
                }
            }
        }
    }
    if (tid == 0) *scale = now;
}

}  // namespace exl3
