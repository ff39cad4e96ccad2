// Instances of the attention kernels for heads of up to EXL3_ATTN_DIM values.
#include "exl3_attn_launch.hpp"

namespace exl3 {

template <int DIM, bool BF16, int RB>
static int launch(const AttnArgs& A, const AttnPlan& P, hipStream_t s) {
    const auto kernel = fp8_attention_kernel<DIM, BF16, RB>;
    constexpr int LDS = AttnSize<DIM, RB>::LDS;
    static std::atomic<uint64_t> ready{0};           // devices that know of the LDS size
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= MAX_DEVICES) return fail("no HIP device");
    if (!(ready.load() >> dev & 1)) {
        if (hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, LDS) !=
            hipSuccess)
            return fail("the device does not give the kernel its LDS");
        ready.fetch_or(1ull << dev);
    }
    if (P.shares) {
        hipLaunchKernelGGL(kernel, dim3(P.shares), dim3(ATTN_WAVES * 64), LDS, s, A);
        if (check_launch()) return -1;
        if (P.shares == 1) return 0;
        hipLaunchKernelGGL((fp8_attention_join_kernel<DIM, BF16, RB>), dim3(P.shares - 1, P.join_rows), dim3(ATTN_WAVES * 64), 0,
                           s, A);
    } else {
        hipLaunchKernelGGL(kernel, dim3((P.tiles + XCDS - 1) / XCDS * XCDS * A.c.kv), dim3(ATTN_WAVES * 64), LDS, s, A);
    }
    return check_launch();
}

template <int DIM, bool BF16>
static int launch(const AttnArgs& A, const AttnPlan& P, hipStream_t s) {
    if (P.rb == 1) return launch<DIM, BF16, 1>(A, P, s);
    if constexpr (DIM <= 128)
        if (P.rb == 4) return launch<DIM, BF16, 4>(A, P, s);
    return launch<DIM, BF16, 2>(A, P, s);
}

#define EXL3_ATTN_CAT_(a, b) a##b
#define EXL3_ATTN_CAT(a, b) EXL3_ATTN_CAT_(a, b)

int EXL3_ATTN_CAT(launch_attention_, EXL3_ATTN_DIM)(const AttnArgs& A, const AttnPlan& P, bool bf16, hipStream_t s) {
    return bf16 ? launch<EXL3_ATTN_DIM, true>(A, P, s) : launch<EXL3_ATTN_DIM, false>(A, P, s);
}

}  // namespace exl3
