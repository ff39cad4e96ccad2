// C-ABI entry points of the block-scaled 8-bit quantization and products
// (declared in include/exl3_amd.h).
#include <atomic>

#include "exl3_fp8.hpp"

using namespace exl3;

static int check_blocks(int64_t m, int64_t k, int64_t n) {
    if (m < 1 || n < 1 || k < 16 || k % 16) return fail("m and n must be positive and k a positive multiple of 16");
    if (k > (1 << 24) || n > (1 << 24)) return fail("k and n must be at most 2^24");
    if (m > (int64_t)65535 * 16) return fail("m must be at most 1048560");
    return 0;
}

// As many launches as the rows need: one takes MAX_GRID workgroups of 32 groups, or of 4.
template <int K>
static int launch_quantize(const void* x, int64_t rows, int k, int groups, bool pow2, uint8_t* q, float* scale,
                           hipStream_t s) {
    const bool chunks = k % 16 == 0 && aligned16(x) && aligned16(q);
    const auto kernel = chunks ? (pow2 ? fp8_quantize_kernel<K, true> : fp8_quantize_kernel<K, false>)
                               : (pow2 ? fp8_quantize_any_kernel<K, true> : fp8_quantize_any_kernel<K, false>);
    const int64_t per = chunks ? 32 : 4, most = MAX_GRID * per / groups;
    for (int64_t at = 0; at < rows; at += most) {
        const int64_t here = rows - at < most ? rows - at : most;
        hipLaunchKernelGGL(kernel, dim3((unsigned)((here * groups + per - 1) / per)), dim3(256), 0, s,
                           static_cast<const char*>(x) + at * k * (K == OUT_F32 ? 4 : 2), here, k, groups, q + at * k,
                           scale + at * groups);
        if (check_launch()) return -1;
    }
    return 0;
}

static int quantize(const void* x, int x_kind, int64_t rows, int64_t k, bool pow2, uint8_t* q, float* scale,
                    hipStream_t s) {
    const int groups = (int)((k + FP8_BLOCK - 1) / FP8_BLOCK);
    if (x_kind == OUT_F16) return launch_quantize<OUT_F16>(x, rows, (int)k, groups, pow2, q, scale, s);
    if (x_kind == OUT_BF16) return launch_quantize<OUT_BF16>(x, rows, (int)k, groups, pow2, q, scale, s);
    return launch_quantize<OUT_F32>(x, rows, (int)k, groups, pow2, q, scale, s);
}

// ---------------------------------------------------------------- choice of a tile

struct GemmArgs {
    const uint8_t* a;
    const float* a_scale;
    int64_t m;
    int k;
    const uint8_t* w;
    const float* w_scale;
    int n;
    void* c;
    int c_kind;
    hipStream_t s;
};

template <int BM, int BN, int WM, int WN, int KG>
static int launch_tile(const GemmArgs& A) {
    typedef Fp8Tile<BM, BN, WM, WN, KG> T;
    const auto kernel = fp8_gemm_tile_kernel<BM, BN, WM, WN, KG>;
    static std::atomic<uint64_t> ready{0};           // devices that know of the LDS size
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= MAX_DEVICES) return fail("no HIP device");
    if (!(ready.load() >> dev & 1)) {
        if (hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                                T::LDS) != hipSuccess)
            return fail("the device does not give the kernel its LDS");
        ready.fetch_or(1ull << dev);
    }
    const int64_t tm = (A.m + BM - 1) / BM, tn = (A.n + BN - 1) / BN;
    if (tm * tn * T::THREADS > 0xffffffffLL) return fail("too many tiles");
    hipLaunchKernelGGL(kernel, dim3((unsigned)(tm * tn)), dim3(T::THREADS), T::LDS, A.s, A.a, A.a_scale, (int)A.m, A.k,
                       A.w, A.w_scale, A.n, A.c, A.c_kind, (int)tm, (int)tn);
    return check_launch();
}

// A tile's share of the time: us for one block of k of a round of workgroups, with
// one workgroup a CU and with as many as a CU's LDS holds.
struct TileCost {
    int bm, bn, resident;
    float one, full;
    int (*launch)(const GemmArgs&);
};

// Measured in captured launches on 4096-wide k (us, this table's shapes in turn): 48
// rows x 4096 8.6 / 10.8 / 15.6 / 22.6; 128 x 4096 14.7 / 11.5 / 16.2 / 23.0; 256 x
// 4096 27.8 / 21.0 / 17.2 / 23.5 / 38.7; 512 x 4096 51.4 / 37.8 / 29.8 / 24.2 / 39.2;
// 4096 x 4096 - / - / 208 / 169 / 120.
static const TileCost TILES[] = {
    {32, 32, 1, 0.16f, 0.16f, launch_tile<32, 32, 1, 1, 8>},
    {32, 64, 1, 0.24f, 0.24f, launch_tile<32, 64, 1, 2, 4>},
    {64, 64, 2, 0.36f, 0.80f, launch_tile<64, 64, 2, 2, 2>},
    {64, 128, 1, 0.63f, 0.63f, launch_tile<64, 128, 2, 2, 2>},
    {128, 128, 2, 1.13f, 1.95f, launch_tile<128, 128, 2, 2, 1>},
};

// Rounds of workgroups, each with about 1 us that the blocks do not account for; a
// last round of one workgroup a CU takes what one takes.  Of 135 sizes (k 1536,
// 4096 and 7168, n 1536, 4096 and 12288, 4 to 4096 rows) the choice is 1% above the
// fastest kernel in the mean and more than 10% above it in two: 32 rows x 1536 x
// 1536, 6.0 us where the kernel without tiles takes 4.5, and 4096 rows
// 7168 -> 1536, 108 where 128x128 takes 98.
static const TileCost& choose_tile(int64_t m, int64_t k, int64_t n) {
    const int64_t cus = device_cus();
    const double blocks = (double)((k + FP8_BLOCK - 1) / FP8_BLOCK);
    const TileCost* best = TILES;
    double least = 0;
    for (const TileCost& t : TILES) {
        const int64_t tiles = ((m + t.bm - 1) / t.bm) * ((n + t.bn - 1) / t.bn);
        const int64_t rounds = tiles / (cus * t.resident), rest = tiles - rounds * cus * t.resident;
        const double us = (double)rounds * (1.0 + blocks * t.full) +
                          (rest ? 1.0 + blocks * (rest <= cus ? t.one : t.full) : 0.0);
        if (&t == TILES || us < least) {
            least = us;
            best = &t;
        }
    }
    return *best;
}

// The kernel goes by the sizes, not by the result's type: a 16-bit result is the
// fp32 one rounded.  Few rows have a kernel without LDS tiles: 8, and 16 where its
// workgroups are one round (us, against the best tile: 4096 x 4096 8 rows 6.5 / 7.6,
// 16 rows 7.5 / 7.7, 1536 x 4096 16 rows 4.4 / 5.9, 7168 x 4096 11.0 / 10.7; 4096 x
// 12288 8 rows 13.7 / 13.1, 16 rows 16.6 / 13.1), and so has a k whose rows are too
// long for a tile's 32-bit offsets.
static int gemm(const GemmArgs& A) {
    if (A.m <= (A.n <= 16 * (int64_t)device_cus() ? 16 : 8) || A.k > FP8_TILE_MAX_K) {
        hipLaunchKernelGGL((fp8_gemm_rows_kernel<1, 8>), dim3((unsigned)((A.n + 15) / 16), (unsigned)((A.m + 15) / 16)),
                           dim3(512), 0, A.s, A.a, A.a_scale, A.m, A.k, A.w, A.w_scale, A.n, A.c, A.c_kind);
        return check_launch();
    }
    return choose_tile(A.m, A.k, A.n).launch(A);
}

// Whether a linear's rows are quantized by the workgroups that multiply them.
// Every one of them does all the rows, so it pays while that is little for a CU
// (us in a captured step, one launch / two: 4096 x 4096 1 row 6.3 / 8.0, 8 rows
// 9.2 / 9.1; 4096 x 12288 1 row 12.0 / 13.7, 4 rows 15.0 / 14.8; 1536 x 4096 16
// rows 6.2 / 6.8), and it saves the caller a launch and the scratch.
static bool linear_in_one(int64_t m, int64_t k, int64_t n) {
    const int64_t rounds = (n + 16 * device_cus() - 1) / (16 * device_cus());
    return m <= 16 && m * k * rounds <= 32768 && fp8_linear_rows_lds((int)m, (int)k) <= 64 * 1024;
}

static int64_t linear_scratch_bytes(int64_t m, int64_t k, int64_t n) {
    return linear_in_one(m, k, n) ? 0 : align_up(m * k, 256) + m * ((k + FP8_BLOCK - 1) / FP8_BLOCK) * 4;
}

extern "C" {

int exl3_fp8_quantize(const void* x, int x_kind, int64_t rows, int64_t k, int pow2, uint8_t* q, float* scale,
                      void* stream) {
    clear_error();
    if (!x || !q || !scale) return fail("null pointer");
    if (x_kind < OUT_F16 || x_kind > OUT_F32) return fail("x_kind must be 0 (fp16), 1 (bf16) or 2 (fp32)");
    if (rows < 1 || k < 1) return fail("rows and k must be positive");
    if (k > (1 << 24)) return fail("k must be at most 2^24");
    if (rows > (int64_t)1 << 36) return fail("too many values");
    return quantize(x, x_kind, rows, k, pow2 != 0, q, scale, reinterpret_cast<hipStream_t>(stream));
}

int exl3_fp8_gemm(const uint8_t* a, const float* a_scale, int64_t m, int64_t k, const uint8_t* w, const float* w_scale,
                  int64_t n, void* c, int c_kind, void* stream) {
    clear_error();
    if (!a || !a_scale || !w || !w_scale || !c) return fail("null pointer");
    if (c_kind < OUT_F16 || c_kind > OUT_F32) return fail("c_kind must be 0 (fp16), 1 (bf16) or 2 (fp32)");
    if (check_blocks(m, k, n)) return -1;
    if (!aligned16(a) || !aligned16(w) || !aligned16(c)) return fail("a, w and c must be 16-byte aligned");
    return gemm(GemmArgs{a, a_scale, m, (int)k, w, w_scale, (int)n, c, c_kind, reinterpret_cast<hipStream_t>(stream)});
}

int64_t exl3_fp8_linear_scratch_bytes(int64_t m, int64_t k, int64_t n) {
    clear_error();
    if (check_blocks(m, k, n)) return -1;
    return linear_scratch_bytes(m, k, n);
}

int exl3_fp8_linear(const void* x, int x_kind, int64_t m, int64_t k, const uint8_t* w, const float* w_scale, int64_t n,
                    void* c, int c_kind, void* scratch, int64_t scratch_bytes, void* stream) {
    clear_error();
    if (!x || !w || !w_scale || !c) return fail("null pointer");
    if (x_kind < OUT_F16 || x_kind > OUT_F32) return fail("x_kind must be 0 (fp16), 1 (bf16) or 2 (fp32)");
    if (c_kind < OUT_F16 || c_kind > OUT_F32) return fail("c_kind must be 0 (fp16), 1 (bf16) or 2 (fp32)");
    if (check_blocks(m, k, n)) return -1;
    if (!aligned16(x) || !aligned16(w) || !aligned16(c)) return fail("x, w and c must be 16-byte aligned");
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    if (linear_in_one(m, k, n)) {
        const auto kernel = x_kind == OUT_F16    ? fp8_linear_rows_kernel<OUT_F16>
                            : x_kind == OUT_BF16 ? fp8_linear_rows_kernel<OUT_BF16>
                                                 : fp8_linear_rows_kernel<OUT_F32>;
        hipLaunchKernelGGL(kernel, dim3((unsigned)((n + 15) / 16)), dim3(FP8_LINEAR_WAVES * 64),
                           fp8_linear_rows_lds((int)m, (int)k), s, x, (int)m, (int)k, w, w_scale, (int)n, c, c_kind);
        return check_launch();
    }
    if (!scratch) return fail("null pointer");
    if (!aligned16(scratch)) return fail("scratch must be 16-byte aligned");
    if (scratch_bytes < linear_scratch_bytes(m, k, n)) return fail("scratch too small");
    uint8_t* q = static_cast<uint8_t*>(scratch);
    float* scale = reinterpret_cast<float*>(q + align_up(m * k, 256));
    const int rc = quantize(x, x_kind, m, k, false, q, scale, s);
    return rc ? rc : gemm(GemmArgs{q, scale, m, (int)k, w, w_scale, (int)n, c, c_kind, s});
}

}  // extern "C"
