// C-ABI entry point of the norm in front of a block-scaled product (declared in
// include/exl3_amd.h).
#include <cmath>

#include "exl3_norm.hpp"

using namespace exl3;

static NormArgs from_row(const NormArgs& A, int64_t row, int64_t rows, int x_kind, int r_kind) {
    const auto on = [&](const void* p, int kind) {
        return p ? static_cast<const char*>(p) + row * A.k * (kind == OUT_F32 ? 4 : 2) : nullptr;
    };
    NormArgs B = A;
    B.rows = rows;
    B.x = on(A.x, x_kind);
    B.residual = on(A.residual, r_kind);
    B.sum = const_cast<char*>(on(A.sum, r_kind));
    B.normed = const_cast<char*>(on(A.normed, A.normed_kind));
    B.q = A.q + row * A.k;
    B.scale = A.scale + row * A.groups;
    return B;
}

// As many launches as the rows need: one takes MAX_GRID workgroups.
template <int X, int R>
static int launch(const NormArgs& A, hipStream_t s) {
    const bool aligned = A.k % 16 == 0 && aligned16(A.x) && aligned16(A.residual) && aligned16(A.weight) && aligned16(A.q) &&
                         aligned16(A.sum) && aligned16(A.normed);
    void (*kernel)(NormArgs) = fp8_norm_any_kernel<X, R>;
    int per = 1;
    if (aligned && A.k <= 16384) {
        if (A.k <= 1024) kernel = fp8_norm_kernel<X, R, 1, 1>, per = 4;
        else if (A.k <= 2048) kernel = fp8_norm_kernel<X, R, 2, 1>, per = 2;
        else if (A.k <= 4096) kernel = fp8_norm_kernel<X, R, 4, 1>;
        else if (A.k <= 8192) kernel = fp8_norm_kernel<X, R, 4, 2>;
        else kernel = fp8_norm_kernel<X, R, 4, 4>;
    }
    const int64_t most = MAX_GRID * per;
    for (int64_t at = 0; at < A.rows; at += most) {
        const int64_t here = A.rows - at < most ? A.rows - at : most;
        hipLaunchKernelGGL(kernel, dim3((unsigned)((here + per - 1) / per)), dim3(256), 0, s, from_row(A, at, here, X, R));
        if (check_launch()) return -1;
    }
    return 0;
}

template <int X>
static int launch(const NormArgs& A, int r_kind, hipStream_t s) {
    if (!A.residual) return launch<X, NO_RESIDUAL>(A, s);
    if (r_kind == OUT_F32) return launch<X, OUT_F32>(A, s);
    return launch<X, X>(A, s);
}

extern "C" {

int exl3_fp8_norm(const void* x, int x_kind, const void* residual, int residual_kind, const void* weight, int weight_kind,
                  int64_t rows, int64_t k, float eps, int pow2, uint8_t* q, float* scale, void* sum, void* normed,
                  int normed_kind, void* stream) {
    clear_error();
    if (!x || !weight || !q || !scale || (residual && !sum)) return fail("null pointer");
    if (x_kind < OUT_F16 || x_kind > OUT_F32) return fail("x_kind must be 0 (fp16), 1 (bf16) or 2 (fp32)");
    if (weight_kind < OUT_F16 || weight_kind > OUT_F32) return fail("weight_kind must be 0 (fp16), 1 (bf16) or 2 (fp32)");
    if (residual && residual_kind != x_kind && residual_kind != OUT_F32)
        return fail("residual_kind must be x's or 2 (fp32)");
    if (normed && (normed_kind < OUT_F16 || normed_kind > OUT_F32))
        return fail("normed_kind must be 0 (fp16), 1 (bf16) or 2 (fp32)");
    if (rows < 1 || k < 1) return fail("rows and k must be positive");
    if (k > (1 << 24)) return fail("k must be at most 2^24");
    if (rows > (int64_t)1 << 36) return fail("too many values");
    if (!(eps >= 0.f) || !std::isfinite(eps)) return fail("eps must be finite and not negative");
    const NormArgs A{x, residual, weight, weight_kind, rows, (int)k, (int)((k + FP8_BLOCK - 1) / FP8_BLOCK), (double)eps,
                     1.0 / (double)k, pow2 != 0, q, scale, residual ? sum : nullptr, normed, normed_kind};
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    if (x_kind == OUT_F16) return launch<OUT_F16>(A, residual_kind, s);
    if (x_kind == OUT_BF16) return launch<OUT_BF16>(A, residual_kind, s);
    return launch<OUT_F32>(A, residual_kind, s);
}

}  // extern "C"
