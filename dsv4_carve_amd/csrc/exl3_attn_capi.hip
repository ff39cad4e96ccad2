// C-ABI entry points of the 8-bit cache and the attention over it (declared in
// include/exl3_amd.h).
#include <algorithm>
#include <cmath>

#include "exl3_attn_launch.hpp"

using namespace exl3;

// Keys that a table's row may name: a block of them, or the next ones that a wave asks for, still ends below 2^31.
constexpr int64_t MAX_ROOM = INT32_MAX - 1023;

static int check_cache(const void* k, const void* k_scale, const void* v, const void* v_scale, int64_t pages, int64_t kv_heads,
                       int64_t page_size, int64_t dim, const void* table, int64_t width, const void* lengths,
                       const void* starts, int64_t seqs, int64_t tokens) {
    if (!k || !k_scale || !v || !v_scale || !table || !lengths) return fail("null pointer");
    if (pages < 1 || pages > INT32_MAX) return fail("pages must be in 1..2^31-1");
    if (kv_heads < 1 || kv_heads > 1024) return fail("kv_heads must be in 1..1024");
    if (page_size < 16 || page_size > 256 || (page_size & (page_size - 1)))
        return fail("page_size must be 16, 32, 64, 128 or 256");
    if (dim < 16 || dim > 256 || dim % 16) return fail("dim must be a multiple of 16 in 16..256");
    if (width < 1 || width > MAX_ROOM / page_size) return fail("a table's row must have 1..(2^31-1024)/page_size pages");
    if (seqs < 1 || seqs > (1 << 20)) return fail("seqs must be in 1..2^20");
    if (tokens < 1 || tokens > (1 << 22)) return fail("tokens must be in 1..2^22");
    if (!starts && tokens != seqs) return fail("without starts there is one token for each sequence");
    if (!aligned16(k) || !aligned16(v)) return fail("k and v must be 16-byte aligned");
    return 0;
}

static int log2_of(int64_t v) { return 63 - __builtin_clzll((unsigned long long)v); }

// Rows of a tile, and the kernel with it, by the rows that a sequence and cache head have on average.  16 and 32: the
// waves divide a tile's keys; 64 and 128: they have rows of their own and share the keys in LDS.  In us, 32 query heads
// over 8 cache heads, 64 ragged sequences of up to 8192 keys with up to 8, 16 and 32 tokens (18, 34 and 66 rows):
//            16 rows         32 rows         64 rows         128 rows
//   dim 64   88, 144, 255    76, 106, 170    100, 105, 231   112, 139, 153
//   dim 128  169, 289, 500   199, 290, 479   144, 158, 324   159, 186, 207
// and of 4 such sequences 25, 30, 46 / 37, 41, 50 / 31, 33, 39 / 43, 46, 49 (dim 128); 16 query heads over 4 of 256
// channels, the 64 sequences: 172, 260, 451 / 265, 388, 606 / 152, 158, 234 (128 rows have no room in the registers).
static int tile_rows(int64_t rows, int64_t dim, int64_t pairs, int64_t cus) {
    if (rows <= 16) return 16;
    if (dim <= 64) return rows <= 64 ? 32 : 128;
    if (dim <= 128 && rows <= 32 && pairs < cus / 2) return 16;
    return dim > 128 || rows <= 64 ? 64 : 128;
}

// Work is shared out over the workgroups that run at once, two a CU, where the waves divide the keys, and where there are
// fewer than four tiles a CU: one tile's length more or less counts then (64 sequences of up to 8192 keys, 512 tiles of
// 128 rows: 259 -> 184 us; with up to 16 tiles a CU four prompts of up to 3000 tokens, 2000 tiles, go from 230 to 401).
// Single tokens of many sequences have a workgroup a tile too, if their tables have room for few keys: a second tile costs a
// workgroup more than a new one does (8 heads of 128: 256 sequences of up to 500, 1000 and 4000 keys 51, 76 and 218 us, shared
// out 60, 85 and 225; 128 of up to 2000 69 and 75), but then the longest sequence bounds the call.  So its run, 6.6 us for
// 1024 keys, is to be no longer than the launch's rounds of two workgroups a CU, which take 7 us and more each.  Past that
// 300 sequences of 500 keys with one of 131072 take 140 us shared out and 870-910 otherwise, 128 and 256 even ones of up to
// 8192 242 and 473 against 255 and 483; but in tables with room for 131072, 300 of 500 take 85 where 74 would do, and 1024 of
// up to 128 with two cache heads 50 instead of 34.
// Rows of a shared tile are joined by a workgroup each where a tile has more than five partial results, and by one for four
// where it has fewer (us, a row each and four rows: one token of 131072 keys with one cache head 25.3 and 33.6, 24 tokens of a
// 256-channel head 20.9 and 24.2, four of four tokens of 8192 23.2 and 27.4; 16 of five tokens 23.0 and 20.8, 512 tokens of
// 1024 keys 56 and 45, of 16384 175 and 166.  64 tokens of 8192 are on the wrong side: 44 and 39).
static AttnPlan plan_attention(int64_t tokens, int64_t heads, int64_t kv_heads, int64_t dim, int64_t seqs, int64_t keys) {
    const int64_t group = heads / kv_heads, rows = (tokens + seqs - 1) / seqs * group, cus = device_cus();
    AttnPlan P{};
    P.rows = tile_rows(rows, dim, std::min(seqs, tokens) * kv_heads, cus);
    const bool few = P.rows <= 32;
    const int64_t tiles = tokens * group / P.rows + std::min(seqs, tokens), blocks = (keys + ATTN_KEYS - 1) / ATTN_KEYS;
    const bool single = tokens == seqs && keys * 2 * cus <= 1024 * tiles * kv_heads;
    P.tiles = (unsigned)(tokens * group / P.rows + seqs);                // as the kernels' find_slot counts
    if (tiles * kv_heads <= 4 * cus || (few && !single) || P.tiles * kv_heads > MAX_GRID / 2) {   // or more than a launch takes
        const int64_t each = few ? ATTN_WAVES : 1, units = tiles * kv_heads * std::max<int64_t>(blocks, 1);
        P.shares = (unsigned)std::max<int64_t>(1, std::min(2 * cus, (units + each - 1) / each + tiles * kv_heads));
        P.least = (int)each;
        P.most = (int)(2 * cus);
        P.join_rows = (unsigned)(P.shares > 5 * tiles * kv_heads ? P.rows : P.rows / 4);
    }
    return P;
}

// Partial results, and what the workgroups say of them.
static int64_t part_bytes(const AttnPlan& P, int64_t dim) {
    const int64_t padded = (dim + 63) / 64 * 64;
    return (int64_t)P.shares * 2 * P.rows * (padded + 2) * 4;
}

static int64_t attention_scratch(const AttnPlan& P, int64_t dim) {
    return P.shares ? part_bytes(P, dim) + (int64_t)P.shares * (int64_t)sizeof(SharedTile) : 0;
}

static int64_t keys_of(int64_t width, int64_t page_size, int64_t tokens, int64_t window) {
    return window ? std::min(width * page_size, window + tokens + 2 * ATTN_KEYS) : width * page_size;
}

template <int K, int TEAM>
static int launch_append(const AppendArgs& A, int64_t slots, hipStream_t s) {
    static std::atomic<uint64_t> ready{0};           // devices that know of the LDS size
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= MAX_DEVICES) return fail("no HIP device");
    if (!(ready.load() >> dev & 1)) {
        if (hipFuncSetAttribute(reinterpret_cast<const void*>(fp8_cache_append_kernel<K, TEAM>),
                                hipFuncAttributeMaxDynamicSharedMemorySize, append_lds(256, 256)) != hipSuccess)
            return fail("the device does not give the kernel its LDS");
        ready.fetch_or(1ull << dev);
    }
    constexpr int TEAMS = APPEND_WAVES * 64 / TEAM;
    hipLaunchKernelGGL((fp8_cache_append_kernel<K, TEAM>), dim3((unsigned)slots, (unsigned)((A.c.kv + TEAMS - 1) / TEAMS), 2),
                       dim3(APPEND_WAVES * 64), TEAMS * append_lds(1 << A.c.page_shift, A.c.dim), s, A);
    return check_launch();
}

// A wave a page and head where sequences are many, have few tokens and the waves' pages have room in LDS.  In us, pages of
// 64, 8 heads of 128 channels, a workgroup each and a wave each: 1, 64, 256 and 1024 sequences of a token 5.0, 6.5, 13.5, 36.3
// and 5.7, 6.4, 10.0, 28.0; 16, 256 and 1024 of 3 tokens 5.6, 24.3, 125.5 and 6.2, 15.9, 58.4; 64 of 16 8.5 and 8.1.
template <int K>
static int launch_append(const AppendArgs& A, int64_t slots, hipStream_t s) {
    const bool waves = A.c.tokens <= 16 * (int64_t)A.c.seqs && slots * A.c.kv * 2 > 4 * device_cus() &&
                       APPEND_WAVES * append_lds(1 << A.c.page_shift, A.c.dim) <= 64 * 1024;
    return waves ? launch_append<K, 64>(A, slots, s) : launch_append<K, APPEND_WAVES * 64>(A, slots, s);
}

extern "C" {

int exl3_fp8_cache_append(const void* k, int64_t k_token, int64_t k_head, const void* v, int64_t v_token, int64_t v_head,
                          int kind, int64_t tokens, uint8_t* k_cache, float* k_scale, uint8_t* v_cache, float* v_scale,
                          int64_t pages, int64_t kv_heads, int64_t page_size, int64_t dim, const int32_t* table,
                          int64_t table_stride, int64_t width, const int32_t* lengths, const int32_t* starts, int64_t seqs,
                          void* stream) {
    clear_error();
    if (!k || !v) return fail("null pointer");
    if (kind < OUT_F16 || kind > OUT_F32) return fail("kind must be 0 (fp16), 1 (bf16) or 2 (fp32)");
    if (check_cache(k_cache, k_scale, v_cache, v_scale, pages, kv_heads, page_size, dim, table, width, lengths, starts, seqs,
                    tokens))
        return -1;
    const int64_t each = kind == OUT_F32 ? 4 : 8;
    if (!aligned16(k) || !aligned16(v) || k_token % each || k_head % each || v_token % each || v_head % each)
        return fail("rows of k and v must be 16-byte aligned");
    const AppendArgs A{{k_cache, k_scale, v_cache, v_scale, table, table_stride, lengths, starts, (int)seqs, (int)tokens,
                        (int)kv_heads, (int)dim, log2_of(page_size), (int)width, (int)pages},
                       k, v, k_token, k_head, v_token, v_head};
    const int64_t slots = starts ? tokens / page_size + 2 * seqs : tokens;     // as the kernel's find_slot counts
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    if (kind == OUT_F16) return launch_append<OUT_F16>(A, slots, s);
    if (kind == OUT_BF16) return launch_append<OUT_BF16>(A, slots, s);
    return launch_append<OUT_F32>(A, slots, s);
}

int64_t exl3_fp8_attention_scratch_bytes(int64_t tokens, int64_t heads, int64_t kv_heads, int64_t dim, int64_t seqs,
                                         int64_t width, int64_t page_size, int64_t window) {
    clear_error();
    if (tokens < 1 || tokens > (1 << 22) || seqs < 1 || seqs > (1 << 20) || kv_heads < 1 || heads < kv_heads ||
        heads % kv_heads || heads > 65536 || dim < 16 || dim > 256 || dim % 16 || page_size < 16 || page_size > 256 ||
        width < 1 || width > MAX_ROOM / page_size || window < 0)
        return fail("sizes out of range");
    return attention_scratch(plan_attention(tokens, heads, kv_heads, dim, seqs, keys_of(width, page_size, tokens, window)), dim);
}

int exl3_fp8_attention(const void* q, int kind, int64_t q_token, int64_t q_head, int64_t tokens, int64_t heads,
                       const uint8_t* k_cache, const float* k_scale, const uint8_t* v_cache, const float* v_scale,
                       int64_t pages, int64_t kv_heads, int64_t page_size, int64_t dim, const int32_t* table,
                       int64_t table_stride, int64_t width, const int32_t* lengths, const int32_t* starts, int64_t seqs,
                       float scale, int64_t window, const float* sinks, void* out, float* lse, int clear, void* scratch,
                       int64_t scratch_bytes, void* stream) {
    clear_error();
    if (!q || !out) return fail("null pointer");
    if (kind != OUT_F16 && kind != OUT_BF16) return fail("kind must be 0 (fp16) or 1 (bf16)");
    if (check_cache(k_cache, k_scale, v_cache, v_scale, pages, kv_heads, page_size, dim, table, width, lengths, starts, seqs,
                    tokens))
        return -1;
    if (heads < kv_heads || heads % kv_heads || heads > 65536) return fail("heads must be a multiple of kv_heads up to 65536");
    if (tokens * heads > INT32_MAX) return fail("too many rows");
    if (!std::isfinite(scale)) return fail("scale must be finite");
    if (window < 0 || window > INT32_MAX / 2) return fail("window must be in 0..2^30");
    if (!aligned16(q) || !aligned16(out) || q_token % 8 || q_head % 8) return fail("rows of q and out must be 16-byte aligned");
    AttnPlan P = plan_attention(tokens, heads, kv_heads, dim, seqs, keys_of(width, page_size, tokens, window));
    if (!starts) P.tiles = (unsigned)(seqs * ((heads / kv_heads + P.rows - 1) / P.rows));
    const int64_t need = attention_scratch(P, dim);
    if (need && !scratch) return fail("null pointer");
    if (!aligned16(scratch)) return fail("scratch must be 16-byte aligned");
    if (scratch_bytes < need) return fail("scratch too small");
    AttnArgs A{{const_cast<uint8_t*>(k_cache), const_cast<float*>(k_scale), const_cast<uint8_t*>(v_cache),
                const_cast<float*>(v_scale), table, table_stride, lengths, starts, (int)seqs, (int)tokens, (int)kv_heads,
                (int)dim, log2_of(page_size), (int)width, (int)pages},
               static_cast<const uint16_t*>(q), q_token, q_head, (int)heads, (int)(heads / kv_heads),
               std::fabs(scale) * 1.4426950408889634f, scale < 0.f, (int)window, sinks, static_cast<uint16_t*>(out), lse,
               P.shares ? static_cast<float*>(scratch) : nullptr,
               reinterpret_cast<SharedTile*>(static_cast<char*>(scratch) + part_bytes(P, dim)), (int)P.tiles, P.least, P.most, clear == 2 ? 2 : clear != 0};
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    const bool bf16 = kind == OUT_BF16;
    if (dim <= 64) return launch_attention_64(A, P, bf16, s);
    if (dim <= 128) return launch_attention_128(A, P, bf16, s);
    if (dim <= 192) return launch_attention_192(A, P, bf16, s);
    return launch_attention_256(A, P, bf16, s);
}

}  // extern "C"
