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

constexpr int FP8_GU_WAVES = 4;

// gate/up: a workgroup has 16 gate and the same 16 up outputs of one active
// expert, for all the rows that name it.  blockIdx.y is a slot, whose expert's
// first slot does the work, or with by_expert an expert; the others' workgroups
// end at once, and there are fewer of those with fewer experts than slots.  The
// expert's rows are the columns of the matrix instruction, 16 MT at a time: with
// few rows an expert, the columns left over cost neither traffic nor time.  Four
// waves a workgroup, each with two blocks of both matrices on their way: 5.6 TB/s
// of weights (the layer above, 303 us), 4.2 with eight waves of twice the
// registers a workgroup.
template <bool BF16, int MT>
__global__ __launch_bounds__(FP8_GU_WAVES * 64) void fp8_moe_gate_up_kernel(const Fp8MoeArgs A, int by_expert) {
    typedef Half16<BF16> H;
    __shared__ float part[FP8_GU_WAVES][2 * MT * 4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int r = lane & 15, g = lane >> 4;
    const int S = A.rows * A.topk;
    const int slot = by_expert ? S : blockIdx.y, e = by_expert ? blockIdx.y : A.rt.local(slot, A.E);
    if (e < 0) return;
    const int n0 = blockIdx.x * 16, I = A.inter, hidden = A.hidden, kb_n = hidden / FP8_BLOCK;
    const uint8_t* wg = A.w13 + ((int64_t)e * 2 * I + n0 + r) * hidden;
    const uint8_t* wu = wg + (int64_t)I * hidden;
    const float* sg = A.s13 + ((int64_t)e * 2 * I + n0) / FP8_BLOCK * kb_n;
    const float* su = sg + (int64_t)(I / FP8_BLOCK) * kb_n;
    struct Unit {
        int8x32_t g, u;
        float sg, su;
    };
    const auto fetch = [&](Unit& u, int kb) {
        u.g = load_whole_block(wg + kb * FP8_BLOCK, g);
        u.u = load_whole_block(wu + kb * FP8_BLOCK, g);
        u.sg = sg[kb];
        u.su = su[kb];
    };
    Unit u0, u1;
    if (wave < kb_n) fetch(u0, wave);           // on its way while the routing is read
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
    const uint64_t mask = __ballot(mine >= 0);
    if (!by_expert ? __ballot(mine >= 0 && mine < slot) != 0 : mask == 0) return;
    const int cnt = __popcll(mask);
    // column c is the c-th of those rows
    const int place = __popcll(mask & ((1ull << lane) - 1));
    const int col_slot = __builtin_amdgcn_ds_permute((mine >= 0 ? place : cnt + lane - place) * 4, mine);

    for (int c0 = 0; c0 < cnt; c0 += 16 * MT) {
        const uint16_t* xr[MT];
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const int col = c0 + 16 * t + r, cs = __shfl(col_slot, col & 63);
            xr[t] = col < cnt ? static_cast<const uint16_t*>(A.x) + (int64_t)(cs / A.topk) * hidden : nullptr;
        }
        float ag[MT][4] = {}, au[MT][4] = {};
        const auto compute = [&](const Unit& u, int kb) {
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                if (t > 0 && c0 + 16 * t >= cnt) break;
                BlockX<H> bx;
                if (xr[t]) bx.load(xr[t] + kb * FP8_BLOCK, g);
                else bx.clear();
                const float4_t pg = block_product<H>(BlockW<H>(u.g), bx), pu = block_product<H>(BlockW<H>(u.u), bx);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    ag[t][i] = fmaf(pg[i], u.sg, ag[t][i]);
                    au[t][i] = fmaf(pu[i], u.su, au[t][i]);
                }
            }
        };
        if (c0 && wave < kb_n) fetch(u0, wave);
        for (int kb = wave; kb < kb_n; kb += 2 * FP8_GU_WAVES) {
            if (kb + FP8_GU_WAVES < kb_n) fetch(u1, kb + FP8_GU_WAVES);
            compute(u0, kb);
            if (kb + 2 * FP8_GU_WAVES < kb_n) fetch(u0, kb + 2 * FP8_GU_WAVES);
            if (kb + FP8_GU_WAVES < kb_n) compute(u1, kb + FP8_GU_WAVES);
        }
        if (c0) __syncthreads();
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
            const int col = c0 + 16 * t + r, cs = __shfl(col_slot, col & 63);
            if (col >= cnt) continue;
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
}

constexpr int FP8_DOWN_WAVES = 16;

// down: a workgroup has 16 outputs of every row and goes through all active
// experts, in the order of their first slots; a column of the matrix
// instruction is a row of the batch, and a row's routing weight joins the block's
// scale, so that the sum over experts needs no second pass and no atomics.  A
// wave takes every 16th block of (expert, k), the next one's bytes on their way
// while it computes; of its row groups of 16 only those that name the expert are
// read and multiplied.  5.1 TB/s of weights with 16 rows (101 of 256 experts of
// 4096 x 2048, 165 us); three or four blocks ahead, or the inputs ahead too,
// change nothing.
template <bool BF16, int MT>
__global__ __launch_bounds__(FP8_DOWN_WAVES * 64) void fp8_moe_down_kernel(const Fp8MoeArgs A) {
    typedef Half16<BF16> H;
    static_assert(FP8_DOWN_WAVES * 64 == FP8_MOE_MAX_SLOTS, "a thread for each slot");
    struct Entry {
        int slot;
        float weight;
    };
    struct Expert {
        uint64_t rows;             // bit r: row r names it
        int id, first;             // its first entry
    };
    __shared__ __attribute__((aligned(16))) int ids[FP8_MOE_MAX_SLOTS];      // local expert of a slot, or -1
    __shared__ float wts[FP8_MOE_MAX_SLOTS];
    __shared__ Expert experts[FP8_MOE_MAX_SLOTS];                            // the active ones
    __shared__ Entry entries[FP8_MOE_MAX_SLOTS];                             // their rows, in order
    __shared__ uint16_t place[FP8_MOE_MAX_SLOTS];                            // of a first slot's expert among them
    __shared__ int wave_n[FP8_DOWN_WAVES];
    __shared__ float part[FP8_DOWN_WAVES][MT * 4][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int r = lane & 15, g = lane >> 4;
    const int S = A.rows * A.topk, row = tid / A.topk;
    const int e = tid < S ? A.rt.local(tid, A.E) : -1;
    ids[tid] = e;
    if (e >= 0) wts[tid] = A.rt.weight(tid);
    __syncthreads();
    // the first slot of this one's expert, and whether it is its row's first of it
    int first = tid;
    bool row_first = false;
    if (wave * 64 < S) {
        for (int s = (min(S, wave * 64 + 64) - 1) & ~3; s >= 0; s -= 4) {
            const i32x4_t v = *reinterpret_cast<const i32x4_t*>(&ids[s]);
#pragma unroll
            for (int i = 3; i >= 0; --i) first = v[i] == e && s + i < first ? s + i : first;
        }
        row_first = e >= 0;
        for (int s = row * A.topk; s < tid; ++s) row_first = row_first && ids[s] != e;
    }
    const bool owner = e >= 0 && first == tid;
    const uint64_t below = (1ull << lane) - 1, own = __ballot(owner);
    if (lane == 0) wave_n[wave] = __popcll(own);
    __syncthreads();
    int before = 0, active = 0;
#pragma unroll
    for (int i = 0; i < FP8_DOWN_WAVES; ++i) {
        before += i < wave ? wave_n[i] : 0;
        active += wave_n[i];
    }
    if (owner) {
        const int at = before + __popcll(own & below);
        place[tid] = (uint16_t)at;
        experts[at].id = e;
        experts[at].rows = 0;
    }
    __syncthreads();
    if (row_first) atomicOr(reinterpret_cast<unsigned long long*>(&experts[place[first]].rows), 1ull << row);
    __syncthreads();
    // entries of the experts before each: a scan over the waves' experts
    const int mine = tid < active ? __popcll(experts[tid].rows) : 0;
    int sum = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(sum, d);
        sum += lane >= d ? o : 0;
    }
    if (lane == 63) wave_n[wave] = sum;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < FP8_DOWN_WAVES; ++i) sum += i < wave ? wave_n[i] : 0;
    if (tid < active) experts[tid].first = sum - mine;
    __syncthreads();
    if (row_first) {
        float w = 0.f;
        for (int s = tid; s < (row + 1) * A.topk; ++s) w += ids[s] == e ? wts[s] : 0.f;
        const Expert& x = experts[place[first]];
        entries[x.first + __popcll(x.rows & ((1ull << row) - 1))] = Entry{tid, w};
    }
    __syncthreads();

    const int n0 = blockIdx.x * 16, I = A.inter, hidden = A.hidden, kb_n = I / FP8_BLOCK, units = active * kb_n;
    // a row group's inputs, and this lane's routing weight
    const auto inputs = [&](BlockX<H>& x, float& wt, uint64_t rows, int first, int kb, int t) {
        const int at = 16 * t + r;
        x.clear();
        wt = 0.f;
        if ((rows >> at) & 1) {
            const Entry n = entries[first + __popcll(rows & ((1ull << at) - 1))];
            wt = n.weight;
            x.load(A.act + (int64_t)n.slot * I + kb * FP8_BLOCK, g);
        }
    };
    struct Unit {
        int8x32_t w;
        uint64_t rows;
        float sc;
        int first, kb;
    };
    const auto fetch = [&](Unit& u, int at) {
        const int j = at / kb_n;
        u.kb = at - j * kb_n;
        const Expert x = experts[j];
        u.rows = x.rows;
        u.first = x.first;
        u.w = load_whole_block(A.w2 + ((int64_t)x.id * hidden + n0 + r) * I + u.kb * FP8_BLOCK, g);
        u.sc = A.s2[((int64_t)x.id * hidden + n0) / FP8_BLOCK * kb_n + u.kb];
    };
    float acc[MT][4] = {};
    const auto compute = [&](const Unit& u) {
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            if (MT > 1 && !((u.rows >> (16 * t)) & 0xffff)) continue;
            BlockX<H> x;
            float wt;
            inputs(x, wt, u.rows, u.first, u.kb, t);
            const float4_t p = block_product<H>(BlockW<H>(u.w), x);
            const bool has = (u.rows >> (16 * t + r)) & 1;      // 0 times a weight that is NaN is not 0
            wt *= u.sc;
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[t][i] = has ? fmaf(p[i], wt, acc[t][i]) : acc[t][i];
        }
    };
    Unit u0, u1;
    int at = __builtin_amdgcn_readfirstlane(wave);
    if (at < units) fetch(u0, at);
    for (; at < units; at += 2 * FP8_DOWN_WAVES) {
        if (at + FP8_DOWN_WAVES < units) fetch(u1, at + FP8_DOWN_WAVES);
        compute(u0);
        if (at + 2 * FP8_DOWN_WAVES < units) fetch(u0, at + 2 * FP8_DOWN_WAVES);
        if (at + FP8_DOWN_WAVES < units) compute(u1);
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
        const int orow = 16 * t + r;
        if (orow < A.rows)
            with_kind(A.out_kind, [&](auto kind) { store_out4<kind()>(A.out, orow, hidden, n0 + 4 * g, v, true); });
    }
}

}  // namespace exl3
