// Instances of the attention kernels for heads of up to EXL3_ATTN_DIM values.
#include "exl3_attn_launch.hpp"

namespace exl3 {

template <int DIM, bool BF16, int ROWS, int LDS>
static int launch(void (*kernel)(AttnArgs), const AttnArgs& A, const AttnPlan& P, std::atomic<uint64_t>& ready, hipStream_t s) {
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= MAX_DEVICES) return fail("no HIP device");
    if (!(ready.load() >> dev & 1)) {
        if (hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, LDS) !=
            hipSuccess)
            return fail("the device does not give the kernel its LDS");
        ready.fetch_or(1ull << dev);
    }
    const unsigned grid = P.shares ? P.shares : tile_grid((int)P.tiles, A.c.kv);
    hipLaunchKernelGGL(kernel, dim3(grid), dim3(ATTN_WAVES * 64), LDS, s, A);
    if (check_launch()) return -1;
    if (P.shares < 2) return 0;
    hipLaunchKernelGGL((fp8_attention_join_kernel<DIM, BF16, ROWS>), dim3(P.shares - 1, P.join_rows), dim3(ATTN_WAVES * 64), 0, s, A);
    return check_launch();
}

template <int DIM, bool BF16, int RB>
static int launch_few(const AttnArgs& A, const AttnPlan& P, hipStream_t s) {
    static std::atomic<uint64_t> ready{0};           // devices that know of the LDS size
    typedef AttnSize<DIM, RB> Z;
    return launch<DIM, BF16, Z::ROWS, Z::LDS>(fp8_attention_kernel<DIM, BF16, RB>, A, P, ready, s);
}

template <int DIM, bool BF16, int RB>
static int launch_many(const AttnArgs& A, const AttnPlan& P, hipStream_t s) {
    static std::atomic<uint64_t> ready{0};
    typedef ShareSize<DIM, RB> Z;
    return launch<DIM, BF16, Z::ROWS, Z::LDS>(fp8_attention_rows_kernel<DIM, BF16, RB>, A, P, ready, s);
}

// The tiles that plan_attention takes for heads of up to DIM values.
template <int DIM, bool BF16>
static int launch(const AttnArgs& A, const AttnPlan& P, hipStream_t s) {
    if (P.rows == 16) return launch_few<DIM, BF16, 1>(A, P, s);
    if constexpr (DIM <= 64) {
        if (P.rows == 32) return launch_few<DIM, BF16, 2>(A, P, s);
        return launch_many<DIM, BF16, 2>(A, P, s);
    } else {
        if constexpr (DIM <= 128)
            if (P.rows == 128) return launch_many<DIM, BF16, 2>(A, P, s);
        return launch_many<DIM, BF16, 1>(A, P, s);
    }
}

#define EXL3_ATTN_CAT_(a, b) a##b
#define EXL3_ATTN_CAT(a, b) EXL3_ATTN_CAT_(a, b)

int EXL3_ATTN_CAT(launch_attention_, EXL3_ATTN_DIM)(const AttnArgs& A, const AttnPlan& P, bool bf16, hipStream_t s) {
    return bf16 ? launch<EXL3_ATTN_DIM, true>(A, P, s) : launch<EXL3_ATTN_DIM, false>(A, P, s);
}

}  // namespace exl3
