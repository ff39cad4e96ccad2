// C-ABI entry points of the block-scaled expert layer and the expert router
// (declared in include/exl3_amd.h).
#include <cmath>

#include "exl3_fp8_moe.hpp"
#include "exl3_topk.hpp"

using namespace exl3;

extern "C" {

int exl3_fp8_moe_max_rows(void) { return FP8_MOE_MAX_ROWS; }

int64_t exl3_fp8_moe_scratch_bytes(int64_t rows, int64_t topk, int64_t intermediate) {
    clear_error();
    if (rows < 1 || rows > FP8_MOE_MAX_ROWS) return fail("row count out of range (1 <= rows <= exl3_fp8_moe_max_rows())");
    if (topk < 1 || topk > FP8_MOE_MAX_TOPK) return fail("topk must be in 1..16");
    if (intermediate < 128 || intermediate % 128) return fail("intermediate must be a positive multiple of 128");
    return rows * topk * intermediate * 4;
}

int exl3_fp8_moe(const void* x, int x_kind, void* out, int out_kind, int64_t rows, int64_t hidden, int64_t intermediate,
                 int64_t n_experts, int64_t topk, const uint8_t* w13, const float* w13_scale, const uint8_t* w2,
                 const float* w2_scale, const void* topk_ids, int ids_kind, const void* topk_weights, int weights_kind,
                 const int64_t* expert_map, int64_t n_global, float swiglu_limit, void* scratch, int64_t scratch_bytes,
                 void* stream) {
    clear_error();
    if (!x || !out || !w13 || !w13_scale || !w2 || !w2_scale || !topk_ids || !topk_weights || !scratch)
        return fail("null pointer");
    if (x_kind != OUT_F16 && x_kind != OUT_BF16) return fail("x_kind must be 0 (fp16) or 1 (bf16)");
    if (out_kind < OUT_F16 || out_kind > OUT_F32) return fail("out_kind must be 0 (fp16), 1 (bf16) or 2 (fp32)");
    const int64_t need = exl3_fp8_moe_scratch_bytes(rows, topk, intermediate);
    if (need < 0) return -1;
    if (hidden < 128 || hidden % 128) return fail("hidden must be a positive multiple of 128");
    if (hidden > (1 << 20) || intermediate > (1 << 20)) return fail("hidden and intermediate must be at most 2^20");
    if (n_experts < 1 || n_experts > (1 << 16)) return fail("n_experts must be in 1..65536");
    if (!(swiglu_limit > 0.f)) return fail("swiglu_limit must be positive (infinity for none)");
    if (scratch_bytes < need) return fail("scratch too small");
    if (!aligned16(x) || !aligned16(out) || !aligned16(w13) || !aligned16(w2) || !aligned16(scratch))
        return fail("x, out, w13, w2 and scratch must be 16-byte aligned");
    Fp8MoeArgs A{x, w13, w13_scale, w2, w2_scale, static_cast<float*>(scratch), out, Route{}, out_kind, (int)rows,
                 (int)hidden, (int)intermediate, (int)n_experts, (int)topk, swiglu_limit};
    if (make_route(topk_ids, ids_kind, topk_weights, weights_kind, expert_map, n_global, A.rt)) return -1;
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    // fewer experts than slots: a workgroup row for each expert
    const int slots = (int)(rows * topk), by_expert = n_experts < slots;
    const dim3 g1((unsigned)(intermediate / 16), (unsigned)(by_expert ? n_experts : slots)), g2((unsigned)(hidden / 16));
    // An expert has slots / n_experts rows on average: with three at most, more than four are rare, and the expert's
    // weights are read again for them (us, 41 rows x 8 on half of 256 experts: 306, with 64 columns 327).
    const bool few = slots <= 3 * n_experts;
    const auto launch = [&](auto gu, auto dn) {
        hipLaunchKernelGGL(gu, g1, dim3(FP8_GU_WAVES * 64), 0, s, A, by_expert);
        const int rc = check_launch();
        if (rc) return rc;
        hipLaunchKernelGGL(dn, g2, dim3(FP8_DOWN_WAVES * 64), 0, s, A);
        return check_launch();
    };
    const auto pick = [&](auto bf16) {
        constexpr bool B = decltype(bf16)::value;
        if (rows == 1) return launch(few ? fp8_moe_gate_up_kernel<B, 0> : fp8_moe_gate_up_kernel<B, 1>, fp8_moe_down_kernel<0>);
        if (rows <= 16)
            return launch(few ? fp8_moe_gate_up_kernel<B, 0> : fp8_moe_gate_up_kernel<B, 1>, fp8_moe_down_kernel<1>);
        if (rows <= 32)
            return launch(few ? fp8_moe_gate_up_kernel<B, 0> : fp8_moe_gate_up_kernel<B, 2>, fp8_moe_down_kernel<2>);
        return launch(few ? fp8_moe_gate_up_kernel<B, 0> : fp8_moe_gate_up_kernel<B, 4>, fp8_moe_down_kernel<4>);
    };
    return x_kind == OUT_BF16 ? pick(std::true_type{}) : pick(std::false_type{});
}

int exl3_moe_route(const void* logits, int logits_kind, int64_t rows, int64_t n_experts, int64_t topk, int scoring,
                   const float* bias, int renormalize, float scale, void* ids, int ids_kind, float* weights,
                   void* stream) {
    clear_error();
    if (!logits || !ids || !weights) return fail("null pointer");
    if (logits_kind < OUT_F16 || logits_kind > OUT_F32) return fail("logits_kind must be 0 (fp16), 1 (bf16) or 2 (fp32)");
    if (ids_kind != IDS_I32 && ids_kind != IDS_I64) return fail("ids_kind must be 0 (int32) or 1 (int64)");
    if (scoring < SCORE_SOFTMAX || scoring > SCORE_SQRTSOFTPLUS)
        return fail("scoring must be 0 (softmax), 1 (sigmoid) or 2 (sqrtsoftplus)");
    if (rows < 1 || n_experts < 1 || n_experts > ROUTE_MAX_EXPERTS)
        return fail("rows must be positive and n_experts in 1..2048");
    if (topk < 1 || topk > ROUTE_MAX_TOPK || topk > n_experts) return fail("topk must be in 1..min(64, n_experts)");
    if (!std::isfinite(scale)) return fail("scale must be finite");
    if (rows > (int64_t)1 << 36) return fail("too many rows");
    const int per_lane = (int)(n_experts + 63) / 64;
    const auto launch = [&](auto kernel) {        // as often as the rows need: a workgroup has four
        for (int64_t at = 0; at < rows; at += 4 * MAX_GRID) {
            const int64_t here = rows - at < 4 * MAX_GRID ? rows - at : 4 * MAX_GRID;
            const RouteArgs A{static_cast<const char*>(logits) + at * n_experts * (logits_kind == OUT_F32 ? 4 : 2), bias,
                              static_cast<char*>(ids) + at * topk * (ids_kind == IDS_I64 ? 8 : 4), weights + at * topk,
                              here, logits_kind, (int)n_experts, (int)topk, scoring, ids_kind == IDS_I64,
                              renormalize != 0, scale};
            hipLaunchKernelGGL(kernel, dim3((unsigned)((here + 3) / 4)), dim3(256), 0,
                               reinterpret_cast<hipStream_t>(stream), A);
            if (check_launch()) return -1;
        }
        return 0;
    };
    if (per_lane <= 1) return launch(moe_route_kernel<1>);
    if (per_lane <= 2) return launch(moe_route_kernel<2>);
    if (per_lane <= 4) return launch(moe_route_kernel<4>);
    if (per_lane <= 8) return launch(moe_route_kernel<8>);
    if (per_lane <= 16) return launch(moe_route_kernel<16>);
    return launch(moe_route_kernel<32>);
}

}  // extern "C"
