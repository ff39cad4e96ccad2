// A routed-expert layer of block-scaled e4m3 matrices for a few rows, in two launches:
//
//   gate/up   act[s] = silu(min(g, L)) * clamp(u, -L, L) for each routed slot s = (row, expert e),
//             g = W13[e][:I] x[row], u = W13[e][I:] x[row]
//   down      out[row] = sum_e wt(row, e) * (W2[e] act[s])
//
// Activations stay 16-bit and the e4m3 weights are widened to their type
// (exactly) before the 16x16x32 matrix instruction: at a few rows the layer reads
// weights, and rounding activations to 8 bits would cost accuracy for nothing.
// Sums are fp32: a block of 128 is four instructions into a cleared
// accumulator, scaled into the running sum by one multiply-add a value.  The
// activation is rounded to 16 bits between the launches, the only rounding
// besides the output's.
//
// Routing is read in each workgroup, lane r of a wave holding row r (64 rows at
// most).  A row that names an expert more than once counts as its first slot,
// under the sum of the weights.
#pragma once

#include "exl3_fp8.hpp"
#include "exl3_route.hpp"

namespace exl3 {

constexpr int FP8_MOE_MAX_ROWS = 64;
constexpr int FP8_MOE_MAX_TOPK = 16;
constexpr int FP8_MOE_MAX_SLOTS = 1024;

__device__ __forceinline__ int8x32_t load_whole_block(const uint8_t* row, int g) {      // row: the block's first byte
    return join(*reinterpret_cast<const i32x4_t*>(row + 16 * g), *reinterpret_cast<const i32x4_t*>(row + 64 + 16 * g));
}

struct Fp8MoeArgs {
    const void* x;              // [rows][hidden], 16-bit
    const uint8_t* w13;         // [E][2 I][hidden]
    const float* s13;           // [E][2 I / 128][hidden / 128]
    const uint8_t* w2;          // [E][hidden][I]
    const float* s2;            // [E][hidden / 128][I / 128]
    uint16_t* act;              // [rows * topk][I], 16-bit
    void* out;                  // [rows][hidden]
    Route rt;
    int out_kind, rows, hidden, inter, E, topk;
    float limit;                // +inf: none
};

constexpr int FP8_GU_WAVES = 8;

// gate/up: a workgroup has 16 gate and the same 16 up outputs of one active
// expert.  blockIdx.y is a slot; the expert's first slot does the work for all
// the rows that name it, the other slots' workgroups end at once.
template <bool BF16, int MT>
__global__ __launch_bounds__(FP8_GU_WAVES * 64) void fp8_moe_gate_up_kernel(const Fp8MoeArgs A) {
    typedef Half16<BF16> H;
    __shared__ float part[FP8_GU_WAVES][2 * MT * 4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int r = lane & 15, g = lane >> 4;
    const int slot = blockIdx.y, S = A.rows * A.topk;
    const int e = A.rt.local(slot, A.E);
    if (e < 0) return;
    // this lane's row: its first slot of expert e, or -1
    int mine = -1;
#pragma unroll
    for (int j0 = 0; j0 < FP8_MOE_MAX_TOPK; j0 += 8) {
        if (j0 >= A.topk) break;
        int s[8], le[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) s[j] = lane < A.rows && j0 + j < A.topk ? lane * A.topk + j0 + j : S;
        A.rt.local_n<8>(s, S, A.E, le);
#pragma unroll
        for (int j = 0; j < 8; ++j) mine = mine < 0 && le[j] == e ? s[j] : mine;
    }
    if (__ballot(mine >= 0 && mine < slot)) return;
    const uint64_t mask = __ballot(mine >= 0);
    const int cnt = __popcll(mask);
    // column c is the c-th of those rows
    const int place = __popcll(mask & ((1ull << lane) - 1));
    const int col_slot = __builtin_amdgcn_ds_permute((mine >= 0 ? place : cnt + lane - place) * 4, mine);

    const int n0 = blockIdx.x * 16, I = A.inter, hidden = A.hidden, kb_n = hidden / FP8_BLOCK;
    const uint8_t* wg = A.w13 + ((int64_t)e * 2 * I + n0 + r) * hidden;
    const uint8_t* wu = wg + (int64_t)I * hidden;
    const float* sg = A.s13 + ((int64_t)e * 2 * I + n0) / FP8_BLOCK * kb_n;
    const float* su = sg + (int64_t)(I / FP8_BLOCK) * kb_n;
    const uint16_t* xr[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int cs = __shfl(col_slot, 16 * t + r);
        xr[t] = 16 * t + r < cnt ? static_cast<const uint16_t*>(A.x) + (int64_t)(cs / A.topk) * hidden : nullptr;
    }
    float ag[MT][4] = {}, au[MT][4] = {};
#pragma unroll 2
    for (int kb = wave; kb < kb_n; kb += FP8_GU_WAVES) {
        const BlockW<H> bg(load_whole_block(wg + kb * FP8_BLOCK, g));
        const BlockW<H> bu(load_whole_block(wu + kb * FP8_BLOCK, g));
        const float scg = sg[kb], scu = su[kb];
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            if (t > 0 && 16 * t >= cnt) break;
            BlockX<H> bx;
            if (xr[t]) bx.load(xr[t] + kb * FP8_BLOCK, g);
            else bx.clear();
            const float4_t pg = block_product<H>(bg, bx), pu = block_product<H>(bu, bx);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                ag[t][i] = fmaf(pg[i], scg, ag[t][i]);
                au[t][i] = fmaf(pu[i], scu, au[t][i]);
            }
        }
    }
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            part[wave][8 * t + i][lane] = ag[t][i];
            part[wave][8 * t + 4 + i][lane] = au[t][i];
        }
    __syncthreads();
    for (int t = wave; t < MT; t += FP8_GU_WAVES) {
        float gs[4] = {}, us[4] = {};
#pragma unroll
        for (int s = 0; s < FP8_GU_WAVES; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                gs[i] += part[s][8 * t + i][lane];
                us[i] += part[s][8 * t + 4 + i][lane];
            }
        const int cs = __shfl(col_slot, 16 * t + r);
        if (16 * t + r >= cnt) continue;
        uint16_t h[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            // comparisons, not fminf: a NaN stays one
            const float gv = gs[i] > A.limit ? A.limit : gs[i];
            const float uv = us[i] > A.limit ? A.limit : us[i] < -A.limit ? -A.limit : us[i];
            h[i] = H::bits(gv / (1.0f + expf(-gv)) * uv);
        }
        *reinterpret_cast<u32x2_t*>(A.act + (int64_t)cs * I + n0 + 4 * g) =
            u32x2_t{h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16};
    }
}

constexpr int FP8_DOWN_WAVES = 16;

// down: a workgroup has 16 outputs of every row and goes through all active
// experts, in the order of their first slots; a column of the matrix
// instruction is a row of the batch, and a row's routing weight joins the block's
// scale, so that the sum over experts needs no second pass and no atomics.
template <bool BF16, int MT>
__global__ __launch_bounds__(FP8_DOWN_WAVES * 64) void fp8_moe_down_kernel(const Fp8MoeArgs A) {
    typedef Half16<BF16> H;
    constexpr int THREADS = FP8_DOWN_WAVES * 64;
    __shared__ int ids[FP8_MOE_MAX_SLOTS];                // local expert of a slot, or -1
    __shared__ uint16_t list[FP8_MOE_MAX_SLOTS];          // first slots of the active experts, in order
    __shared__ uint64_t mask[FP8_MOE_MAX_SLOTS];          // their rows
    __shared__ int first_at[FP8_MOE_MAX_SLOTS];           // place of a first slot's expert in the order
    __shared__ int wave_n[FP8_DOWN_WAVES];
    __shared__ float part[FP8_DOWN_WAVES][MT * 4][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int r = lane & 15, g = lane >> 4;
    const int S = A.rows * A.topk;
    const int e = tid < S ? A.rt.local(tid, A.E) : -1;
    ids[tid] = e;
    __syncthreads();
    int first = tid;
    if (e >= 0) {
        for (int s = 0; s < tid; ++s)
            if (ids[s] == e) {
                first = s;
                break;
            }
    }
    const bool owner = e >= 0 && first == tid;
    const uint64_t own = __ballot(owner);
    if (lane == 0) wave_n[wave] = __popcll(own);
    __syncthreads();
    int before = 0, active = 0;
#pragma unroll
    for (int i = 0; i < FP8_DOWN_WAVES; ++i) {
        before += i < wave ? wave_n[i] : 0;
        active += wave_n[i];
    }
    if (owner) {
        const int at = before + __popcll(own & ((1ull << lane) - 1));
        list[at] = (uint16_t)tid;
        first_at[tid] = at;
        mask[at] = 0;
    }
    __syncthreads();
    if (e >= 0) atomicOr(reinterpret_cast<unsigned long long*>(&mask[first_at[first]]), 1ull << (tid / A.topk));
    __syncthreads();

    const int n0 = blockIdx.x * 16, I = A.inter, hidden = A.hidden, kb_n = I / FP8_BLOCK;
    float acc[MT][4] = {};
    for (int u = wave; u < active * kb_n; u += FP8_DOWN_WAVES) {
        const int j = u / kb_n, kb = u - j * kb_n;
        const int ex = ids[list[j]];
        const uint64_t rows = mask[j];
        const BlockW<H> bw(load_whole_block(A.w2 + ((int64_t)ex * hidden + n0 + r) * I + kb * FP8_BLOCK, g));
        const float sc = A.s2[((int64_t)ex * hidden + n0) / FP8_BLOCK * kb_n + kb];
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            if (!((rows >> (16 * t)) & 0xffff)) continue;
            const int row = 16 * t + r;
            const bool has = (rows >> row) & 1;
            BlockX<H> bx;
            float wt = 0.f;
            if (has) {
                int at = -1;
                for (int q = 0; q < A.topk; ++q) {
                    const int s = row * A.topk + q;
                    if (ids[s] == ex) {
                        at = at < 0 ? s : at;
                        wt += A.rt.weight(s);
                    }
                }
                bx.load(A.act + (int64_t)at * I + kb * FP8_BLOCK, g);
            } else {
                bx.clear();
            }
            const float4_t p = block_product<H>(bw, bx);
            wt *= sc;
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[t][i] = has ? fmaf(p[i], wt, acc[t][i]) : acc[t][i];
        }
    }
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) part[wave][4 * t + i][lane] = acc[t][i];
    __syncthreads();
    for (int t = wave; t < MT; t += FP8_DOWN_WAVES) {
        float v[4] = {};
#pragma unroll
        for (int s = 0; s < FP8_DOWN_WAVES; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] += part[s][4 * t + i][lane];
        const int row = 16 * t + r;
        if (row < A.rows)
            with_kind(A.out_kind, [&](auto kind) { store_out4<kind()>(A.out, row, hidden, n0 + 4 * g, v, true); });
    }
    static_assert(THREADS == FP8_MOE_MAX_SLOTS, "a thread for each slot");
}

}  // namespace exl3
