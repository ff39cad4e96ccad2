// A routed-expert layer of block-scaled e4m3 matrices for a few rows, in two launches:
//
//   gate/up   act[s] = silu(min(g, L)) * clamp(u, -L, L) for each routed slot s = (row, expert e),
//             g = W13[e][:I] x[row], u = W13[e][I:] x[row]
//   down      out[row] = sum_e wt(row, e) * (W2[e] act[s])
//
// Activations are not quantized: at a few rows the layer reads weights, and
// rounding activations to 8 bits would cost accuracy for nothing.  The e4m3
// weights are widened (exactly) to the type of x for the first product, and to
// bf16 for the second, whose activation is fp32: 24 bits, the sum of three bf16
// values, each its highest 8 bits left (exact, and no overflow).  Sums are fp32: a
// block of 128 is four 16x16x32 instructions into a cleared accumulator, scaled into
// the running sum by one multiply-add a value; the three parts of an activation are
// three columns of the instruction, whose results are added before that.
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
    float* act;                 // [rows * topk][I]
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
// few rows an expert, the columns left over cost neither traffic nor time.  MT 0
// is for rows that are few an expert, 4 at a time: their inputs come as down's do,
// one load for four rows.  Four waves a workgroup, each with two blocks of both
// matrices on their way.  Memory bounds it: 5.4 to 5.7 TB/s of weights with 16 rows
// (101 of 256 experts of 4096 x 2048, 299 to 314 us).
template <bool BF16, int MT>
__global__ __launch_bounds__(FP8_GU_WAVES * 64) void fp8_moe_gate_up_kernel(const Fp8MoeArgs A, int by_expert) {
    typedef Half16<BF16> H;
    constexpr int TILES = MT ? MT : 1, COLS = MT ? 16 * MT : 4;
    __shared__ float part[FP8_GU_WAVES][2 * TILES * 4][64];
    __shared__ i32x4_t columns[MT ? 1 : FP8_GU_WAVES][64];      // a wave's inputs of one block, 256 bytes a row
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

    for (int c0 = 0; c0 < cnt; c0 += COLS) {
        // a column past the last row has that row's inputs, and is not stored
        const auto input_row = [&](int col) {
            return static_cast<const uint16_t*>(A.x) + (int64_t)(__shfl(col_slot, min(col, cnt - 1)) / A.topk) * hidden;
        };
        const uint16_t* xr[TILES];
#pragma unroll
        for (int t = 0; t < TILES; ++t) xr[t] = MT ? input_row(c0 + 16 * t + r) : input_row(c0 + g) + 8 * r;
        float ag[TILES][4] = {}, au[TILES][4] = {};
        const auto compute = [&](const Unit& u, int kb) {
#pragma unroll
            for (int t = 0; t < TILES; ++t) {
                if (t > 0 && c0 + 16 * t >= cnt) break;
                BlockX<H> bx;
                if constexpr (MT) {
                    bx.load(xr[t] + kb * FP8_BLOCK, g);
                } else {
                    __builtin_amdgcn_wave_barrier();
                    columns[wave][lane] = *reinterpret_cast<const i32x4_t*>(xr[t] + kb * FP8_BLOCK);
                    __builtin_amdgcn_wave_barrier();
                    bx.load(reinterpret_cast<const uint16_t*>(columns[wave] + 16 * min(r, 3)), g);
                }
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
            fetch(u1, min(kb + FP8_GU_WAVES, kb_n - 1));
            compute(u0, kb);
            fetch(u0, min(kb + 2 * FP8_GU_WAVES, kb_n - 1));
            if (kb + FP8_GU_WAVES < kb_n) compute(u1, kb + FP8_GU_WAVES);
        }
        if (c0) __syncthreads();
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                part[wave][8 * t + i][lane] = ag[t][i];
                part[wave][8 * t + 4 + i][lane] = au[t][i];
            }
        __syncthreads();
        for (int t = wave; t < TILES; t += FP8_GU_WAVES) {
            float gs[4] = {}, us[4] = {};
#pragma unroll
            for (int s = 0; s < FP8_GU_WAVES; ++s)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    gs[i] += part[s][8 * t + i][lane];
                    us[i] += part[s][8 * t + 4 + i][lane];
                }
            const int col = c0 + 16 * t + r, cs = __shfl(col_slot, col & 63);
            if (col >= cnt || (!MT && r >= COLS)) continue;
            float4_t act;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                // comparisons, not fminf: a NaN stays one
                const float gv = gs[i] > A.limit ? A.limit : gs[i];
                const float uv = us[i] > A.limit ? A.limit : us[i] < -A.limit ? -A.limit : us[i];
                act[i] = gv / (1.0f + expf(-gv)) * uv;
            }
            *reinterpret_cast<float4_t*>(A.act + (int64_t)cs * I + n0 + 4 * g) = act;
        }
    }
}

constexpr int FP8_DOWN_WAVES = 16;

// Four fp32 values as three planes of bf16: their upper halves, those of what that leaves, and the 8 bits left then.
__device__ __forceinline__ void split_bf16(const float4_t& v, u32x2_t (&plane)[3]) {
    float4_t rest = v;
#pragma unroll
    for (int p = 0; p < 3; ++p) {
        uint32_t u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            u[i] = __float_as_uint(rest[i]);
            const float top = __uint_as_float(u[i] & 0xffff0000u);
            rest[i] = p == 0 && fabsf(top) == __builtin_inff() ? 0.f : rest[i] - top;      // an infinity leaves nothing
        }
        plane[p] = u32x2_t{__builtin_amdgcn_perm(u[1], u[0], 0x07060302), __builtin_amdgcn_perm(u[3], u[2], 0x07060302)};
    }
}

// down: a workgroup has 16 outputs of every row and goes through all active
// experts, in the order of their first slots; a column of the matrix
// instruction is a row of the batch, and a row's routing weight joins the block's
// scale, so that the sum over experts needs no second pass and no atomics.  A
// wave takes every 16th block of an expert and up to four rows that name it, the
// next ones' bytes on their way while it computes.  5.3 to 5.5 TB/s of weights with
// 16 rows (101 of 256 experts of 4096 x 2048, 154 to 160 us).  MT 0 is for a
// single row, whose experts one wave tells apart: one barrier before the first
// load, not eight (a layer of one row 46.1 to 47.7 us a call, 48.5 to 50.7 with
// MT 1).
template <int MT>
__global__ __launch_bounds__(FP8_DOWN_WAVES * 64) void fp8_moe_down_kernel(const Fp8MoeArgs A) {
    typedef Half16<true> H;
    constexpr int WAVES = FP8_DOWN_WAVES;
    static_assert(WAVES * 64 == FP8_MOE_MAX_SLOTS, "a thread for each slot");
    constexpr bool ONE = MT == 0;
    constexpr int TILES = ONE ? 1 : MT;
    constexpr int COLS = ONE ? 1 : 4, LOADS = (COLS + 1) / 2;      // rows of a group, and the loads that bring their inputs
    struct Entry {
        uint16_t slot, row;
        float weight;
    };
    struct Group {                 // an expert and up to COLS rows that name it, no two of them alike mod 16
        int id;
        uint16_t first, count;     // entries
    };
    __shared__ __attribute__((aligned(16))) int ids[FP8_MOE_MAX_SLOTS];      // local expert of a slot, or -1
    __shared__ float wts[FP8_MOE_MAX_SLOTS];
    __shared__ int expert_id[FP8_MOE_MAX_SLOTS];                             // the active ones
    __shared__ uint64_t expert_rows[FP8_MOE_MAX_SLOTS];                      // bit r: row r names it
    __shared__ Entry entries[FP8_MOE_MAX_SLOTS];                             // their rows, in order
    __shared__ Group groups[FP8_MOE_MAX_SLOTS];
    __shared__ uint16_t place[FP8_MOE_MAX_SLOTS];                            // of a first slot's expert among them
    __shared__ uint16_t first_of[FP8_MOE_MAX_SLOTS];                         // an expert's first entry
    __shared__ int wave_n[2][WAVES];
    __shared__ __attribute__((aligned(16))) float part[WAVES][TILES * 4][64];
    // a wave's inputs of one block: sixteen chunks of 8 values, each of twelve columns, plane 0, 1 and 2 of the group's four
    // rows in turn, and 16 bytes more, so that chunks lie in different banks
    constexpr int CHUNK = 13 * 16;
    __shared__ __attribute__((aligned(16))) char columns[WAVES][16 * CHUNK];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int r = lane & 15, g = lane >> 4;
    const int S = A.rows * A.topk;
    const uint64_t below = (1ull << lane) - 1;
    const int row = tid / A.topk;
    const int e = tid < S ? A.rt.local(tid, A.E) : -1;
    int total;                     // entries, groups from bit 16 up
    if constexpr (ONE) {
        // an expert's first slot is an entry and a group, with the weights of all its slots
        if (wave == 0) {
            const float w = e >= 0 ? A.rt.weight(tid) : 0.f;
            float sum = 0.f;
            bool is_first = e >= 0;
#pragma unroll
            for (int s = 0; s < FP8_MOE_MAX_TOPK; ++s) {
                const bool same = read_lane(e, s) == e;
                sum += same ? read_lane(w, s) : 0.f;
                is_first = is_first && !(same && s < lane);
            }
            const uint64_t active = __ballot(is_first);
            const int at = __popcll(active & below);
            if (is_first) {
                groups[at] = Group{e, (uint16_t)at, 1};
                entries[at] = Entry{(uint16_t)tid, 0, sum};
            }
            if (lane == 0) wave_n[1][0] = __popcll(active);
        }
        __syncthreads();
        total = wave_n[1][0] << 16;
    } else {
        ids[tid] = e;
        if (e >= 0) wts[tid] = A.rt.weight(tid);
        __syncthreads();
        // the first slot of this one's expert, and whether it is its row's first of it
        int first = tid;
        bool row_first = e >= 0;
        if (wave * 64 < S) {
            for (int s = (min(S, wave * 64 + 64) - 1) & ~3; s >= 0; s -= 4) {
                const i32x4_t v = *reinterpret_cast<const i32x4_t*>(&ids[s]);
#pragma unroll
                for (int i = 3; i >= 0; --i) first = v[i] == e && s + i < first ? s + i : first;
            }
            for (int s = row * A.topk; s < tid; ++s) row_first = row_first && ids[s] != e;
        }
        const bool owner = e >= 0 && first == tid;
        const uint64_t own = __ballot(owner);
        if (lane == 0) wave_n[0][wave] = __popcll(own);
        __syncthreads();
        int before = 0, active = 0;
#pragma unroll
        for (int i = 0; i < WAVES; ++i) {
            before += i < wave ? wave_n[0][i] : 0;
            active += wave_n[0][i];
        }
        if (owner) {
            const int at = before + __popcll(own & below);
            place[tid] = (uint16_t)at;
            expert_id[at] = e;
            expert_rows[at] = 0;
        }
        __syncthreads();
        if (row_first) atomicOr(reinterpret_cast<unsigned long long*>(&expert_rows[place[first]]), 1ull << row);
        __syncthreads();
        // An expert's rows in order, cut into groups: a group's rows are columns of the matrix instruction by their number
        // mod 16.
        const auto split = [](uint64_t rows, auto&& group) {
            int first = 0, count = 0;
            for (uint32_t used = 0; rows; rows &= rows - 1) {
                const uint32_t column = 1u << (__builtin_ctzll(rows) & 15);
                if (count == COLS || (used & column)) {
                    group(first, count);
                    first += count;
                    count = 0;
                    used = 0;
                }
                used |= column;
                ++count;
            }
            if (count) group(first, count);
        };
        // entries and groups of the experts before each: a scan over the waves' experts, groups from bit 16 up
        const uint64_t named = tid < active ? expert_rows[tid] : 0;
        int mine = __popcll(named);
        split(named, [&](int, int) { mine += 1 << 16; });
        int sum = mine;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int o = __shfl_up(sum, d);
            sum += lane >= d ? o : 0;
        }
        if (lane == 63) wave_n[1][wave] = sum;
        __syncthreads();
        total = 0;
#pragma unroll
        for (int i = 0; i < WAVES; ++i) {
            sum += i < wave ? wave_n[1][i] : 0;
            total += wave_n[1][i];
        }
        if (tid < active) {
            int at = (sum - mine) >> 16;
            const int entry = (sum - mine) & 0xffff;
            first_of[tid] = (uint16_t)entry;
            split(named, [&](int first, int count) {
                groups[at++] = Group{expert_id[tid], (uint16_t)(entry + first), (uint16_t)count};
            });
        }
        __syncthreads();
        if (row_first) {
            float w = 0.f;
            for (int s = tid; s < (row + 1) * A.topk; ++s) w += ids[s] == e ? wts[s] : 0.f;
            const int j = place[first];
            entries[first_of[j] + __popcll(expert_rows[j] & ((1ull << row) - 1))] = Entry{(uint16_t)tid, (uint16_t)row, w};
        }
        __syncthreads();

    }

    const int n0 = blockIdx.x * 16, I = A.inter, hidden = A.hidden, kb_n = I / FP8_BLOCK;
    const int units = (total >> 16) * kb_n;
    // Block kb of group j's expert, and the inputs of the group's rows there: the vector memory path takes 16 lanes
    // that read neighbouring bytes together and lanes of different rows one by one, so the inputs (512 bytes a row,
    // two rows a load) come in their own order and take the matrix unit's by way of LDS.  Straight to the lanes that
    // multiply them they are eight loads of four useful lanes each, and bound the kernel (231 us where it is 165).
    struct Weights {
        int8x32_t w;
        float sc;
    };
    struct Inputs {
        float4_t v[LOADS];
        float wt;
        int col, t;                // this lane's row's: which of the group's (-1: none), which 16 of the batch
        int last;                  // of the group's rows
    };
    const auto fetch_w = [&](Weights& u, int at) {
        const int j = at / kb_n, kb = at - j * kb_n, id = __builtin_amdgcn_readfirstlane(groups[j].id);
        u.w = load_whole_block(A.w2 + ((int64_t)id * hidden + n0 + r) * I + kb * FP8_BLOCK, g);
        u.sc = A.s2[((int64_t)id * hidden + n0) / FP8_BLOCK * kb_n + kb];
    };
    const auto fetch_x = [&](Inputs& u, int at) {
        const int j = at / kb_n, kb = at - j * kb_n;
        const int first = __builtin_amdgcn_readfirstlane(groups[j].first);
        const int last = __builtin_amdgcn_readfirstlane(groups[j].count) - 1;
        u.last = last;
        u.col = -1;
        u.t = 0;
        u.wt = 0.f;
#pragma unroll
        for (int i = 0; i < COLS; ++i) {
            const Entry n = entries[first + min(i, last)];
            if (i <= last && (n.row & 15) == r) {
                u.col = i;
                u.t = n.row >> 4;
                u.wt = n.weight;
            }
        }
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int slot = entries[first + min(2 * i + (lane >> 5), last)].slot;
            u.v[i] = reinterpret_cast<const float4_t*>(A.act + (int64_t)slot * I + kb * FP8_BLOCK)[lane & 31];
        }
    };
    float acc[TILES][4] = {};
    const auto compute = [&](const Weights& u, const Inputs& x) {
        __builtin_amdgcn_wave_barrier();              // the wave's own place: its LDS operations are in order
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            if (2 * i > x.last) break;                // its last rows again
            u32x2_t plane[3];
            split_bf16(x.v[i], plane);
            char* at = columns[wave] + ((lane & 31) >> 1) * CHUNK + (2 * i + (lane >> 5)) * 16 + (lane & 1) * 8;
#pragma unroll
            for (int q = 0; q < 3; ++q) *reinterpret_cast<u32x2_t*>(at + 64 * q) = plane[q];
        }
        __builtin_amdgcn_wave_barrier();
        const char* col = columns[wave] + 2 * g * CHUNK + (r < 12 ? r : r - 4) * 16;        // columns from 12 on are no row's
        BlockX<H> in;
#pragma unroll
        for (int i = 0; i < 4; ++i)                   // chunks 2g, 2g + 1, 8 + 2g and 9 + 2g
            in.v[i] = *reinterpret_cast<const H::vec8*>(col + ((i & 1) + (i >> 1) * 8) * CHUNK);
        const float4_t p3 = block_product<H>(BlockW<H>(u.w), in);
        const bool has = x.col >= 0;
        const int from = ((lane & 48) + (has ? x.col : 0)) * 4;
        float p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {                 // the parts of column c are c, c + 4 and c + 8: row_shl:4, 8
            const float sum = p3[i] + lane_of<0x104, 0xf>(p3[i], 0.f) + lane_of<0x108, 0xf>(p3[i], 0.f);
            p[i] = __int_as_float(__builtin_amdgcn_ds_bpermute(from, __float_as_int(sum)));
        }
        const float s = x.wt * u.sc;
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
            const bool here = has && (TILES == 1 || x.t == t);
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[t][i] = here ? fmaf(p[i], s, acc[t][i]) : acc[t][i];
        }
    };
    // Loads are waited for in their order, so a unit's inputs are asked for one unit ahead and before the weights of
    // two units ahead: those are still on their way while the unit is computed.  For the same reason no load is in a
    // branch (a wait behind one counts the loads of the shorter side): a group of fewer rows reads its last one's
    // inputs again, and past the end the last unit is.
    constexpr int AHEAD = 2, RING = AHEAD + 1, TURN = 2 * RING;
    Weights uw[RING];
    Inputs ux[2];
    const int me = __builtin_amdgcn_readfirstlane(wave);
    if (me < units) {
        fetch_x(ux[0], me);
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) fetch_w(uw[i], min(me + i * WAVES, units - 1));
    }
    for (int base = me; base < units; base += TURN * WAVES) {
#pragma unroll
        for (int i = 0; i < TURN; ++i) {
            const int at = base + i * WAVES;
            if (at >= units) break;
            fetch_x(ux[(i + 1) % 2], min(at + WAVES, units - 1));
            fetch_w(uw[(i + AHEAD) % RING], min(at + AHEAD * WAVES, units - 1));
            compute(uw[i % RING], ux[i % 2]);
        }
    }
#pragma unroll
    for (int t = 0; t < TILES; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) part[wave][4 * t + i][lane] = acc[t][i];
    __syncthreads();
    for (int t = wave; t < TILES; t += WAVES) {
        float v[4] = {};
#pragma unroll
        for (int s = 0; s < WAVES; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] += part[s][4 * t + i][lane];
        const int orow = 16 * t + r;
        if (orow < A.rows)
            with_kind(A.out_kind, [&](auto kind) { store_out4<kind()>(A.out, orow, hidden, n0 + 4 * g, v, true); });
    }
}

}  // namespace exl3
