// Y = X W^T + bias, and for a token with an adapter + B_a (A_a x), all mod p.
//
// A product of two field elements is sixteen products of bytes.  With w = sum_i w_i 2^(8i) and, since 2^31 = 1, 2^(8i) x mod p a
// rotation of x's 31 bits with bytes d_c(i),
//
//   sum_j w_j x_j = sum_c 2^(8c) sum_(j,i) w_(j,i) d_(j,c)(i),
//
// so the matrix's own bytes, as they lie in memory, are the one operand of a product of unsigned bytes with 32-bit sums, 4n deep, and
// each token has four columns in the other.  Nothing of W is laid out anew: it streams through shared memory once, by tensor copies.
// A sum of 4 * 8192 byte products stays below 2^31, so after 8192 columns of W the accumulators are emptied.
#pragma once
#include "m31.cuh"
#include "serving.cuh"
#include "tc_i8.cuh"

namespace zkb {

constexpr u32 LIN_ROWS = 256;                  // rows of W per tile: two accumulators of 128 that share the tokens' operand
constexpr u32 LIN_STEP = 32;                   // columns of W per step: 128 bytes, one swizzle row
constexpr u32 LIN_SEG = 256;                   // steps after which the accumulators are emptied (8192 columns)
constexpr u32 LIN_TOKENS = 64;                 // tokens per tile at most: 256 columns of an accumulator
constexpr u32 LIN_MAX_STAGES = 8;
constexpr u32 LIN_THREADS = 192;               // warp 0 copies, warp 1 issues, warps 2 to 5 empty the accumulators

// Byte c of the four rotations of x by 8i, i = 0 .. 3, for c = 0 .. 3.  All of them are bytes of x, of x >> 7, or of x without the top bits of its bytes.
__device__ __forceinline__ void digit_words(u32 x, u32 (&w)[4]) {
    const u32 t = x >> 7, m = x & 0x007f7f7fu;
    w[0] = __byte_perm(x, t, 0x4560);
    w[1] = __byte_perm(x, t, 0x5601);
    w[2] = __byte_perm(x, t, 0x6012);
    w[3] = __byte_perm(x, m, 0x4563);
}

// How a product is cut: `tiles` of LIN_ROWS rows x `tt` tokens, each `steps` deep in `segs` segments.  Tiles' steps lie one behind the other and every CTA takes `per`
// of them, so all CTAs finish together; a CTA leaves its sum over each stretch of one tile's segment in slot (CTA + tile * segs + segment), which are all different.
struct LinPlan {
    u32 tokens, m, n, tt, ntiles, mtiles, steps, segs, per, ctas, stages, stage_bytes, tmem_cols;
    u64 total;
    size_t slot_words;
};
inline LinPlan lin_plan(int sm_count, u32 tokens, u32 m, u32 n) {
    LinPlan p{};
    p.tokens = tokens; p.m = m; p.n = n;
    p.ntiles = (tokens + LIN_TOKENS - 1) / LIN_TOKENS;
    p.tt = ((tokens + p.ntiles - 1) / p.ntiles + 3) / 4 * 4;
    p.mtiles = (m + LIN_ROWS - 1) / LIN_ROWS;
    p.steps = (n + LIN_STEP - 1) / LIN_STEP;
    p.segs = (p.steps + LIN_SEG - 1) / LIN_SEG;
    p.total = (u64)p.mtiles * p.ntiles * p.steps;
    p.per = (u32)((p.total + sm_count - 1) / sm_count);
    p.ctas = (u32)((p.total + p.per - 1) / p.per);
    p.stage_bytes = LIN_ROWS * 128 + 4 * p.tt * 128;
    p.stages = 200 * 1024 / p.stage_bytes < LIN_MAX_STAGES ? 200 * 1024 / p.stage_bytes : LIN_MAX_STAGES;
    p.tmem_cols = 32;
    while (p.tmem_cols < 8 * p.tt) p.tmem_cols *= 2;
    p.slot_words = (size_t)p.tt * LIN_ROWS;
    return p;
}
// Tokens of one pass: their operand (16 bytes a value) is read by every row of tiles and should stay in L2.
inline u32 lin_chunk(u32 tokens, u32 n) {
    const u64 fit = ((u64)64 << 20) / ((u64)(n + LIN_STEP - 1) / LIN_STEP * LIN_STEP * 16) / LIN_TOKENS * LIN_TOKENS;
    const u32 most = fit < LIN_TOKENS ? LIN_TOKENS : (fit > 2048 ? 2048u : (u32)fit);
    return tokens < most ? tokens : most;
}
inline size_t lin_digit_bytes(const LinPlan& p) { return (size_t)p.ntiles * p.steps * p.tt * 512; }
inline size_t lin_slot_bytes(const LinPlan& p) { return ((size_t)p.ctas + (size_t)p.mtiles * p.ntiles * p.segs) * p.slot_words * 4; }

// The tokens' operand, in the order in which the tiles are copied: per (tile of tokens, step) 4 tt rows of 128 bytes, swizzled.
__global__ void __launch_bounds__(512) linear_digits_kernel(const u32* __restrict__ x, u64 x_stride, LinPlan p, unsigned char* __restrict__ out) {
    const u32 step = blockIdx.x, nt = blockIdx.y, tok = threadIdx.x >> 3, q = threadIdx.x & 7;
    const u32 t = nt * p.tt + tok, j = step * LIN_STEP + 4 * q;
    unsigned char* tile = out + ((size_t)nt * p.steps + step) * p.tt * 512;
    u32 w[4][4];
#pragma unroll
    for (u32 e = 0; e < 4; e++) {
        const u32 v = t < p.tokens && j + e < p.n ? x[t * x_stride + j + e] : 0u;
        u32 d[4];
        digit_words(v, d);
#pragma unroll
        for (int c = 0; c < 4; c++) w[c][e] = d[c];
    }
#pragma unroll
    for (u32 c = 0; c < 4; c++) {
        const u32 r = 4 * tok + c;
        *reinterpret_cast<uint4*>(tile + r * 128 + ((q ^ (r & 7)) << 4)) = make_uint4(w[c][0], w[c][1], w[c][2], w[c][3]);
    }
}

struct LinWalk {                               // a CTA's stretches, the same for every role
    const LinPlan& p;
    u64 at, end;
    __device__ LinWalk(const LinPlan& plan) : p(plan), at((u64)blockIdx.x * plan.per), end(at + plan.per < plan.total ? at + plan.per : plan.total) {}
    u32 mt, nt, first, count, slot;
    __device__ bool next() {
        if (at >= end) return false;
        const u32 tile = (u32)(at / p.steps);
        first = (u32)(at - (u64)tile * p.steps);
        const u32 seg = first / LIN_SEG, seg_end = (seg + 1) * LIN_SEG < p.steps ? (seg + 1) * LIN_SEG : p.steps;
        count = end - at < seg_end - first ? (u32)(end - at) : seg_end - first;
        mt = tile / p.ntiles;
        nt = tile - mt * p.ntiles;
        slot = blockIdx.x + tile * p.segs + seg;
        at += count;
        return true;
    }
};

__global__ void __launch_bounds__(LIN_THREADS) linear_bytes_kernel(const __grid_constant__ CUtensorMap map_w, LinPlan p, const unsigned char* __restrict__ digits,
                                                                   u32* __restrict__ slots, int* gave_up_out) {
    extern __shared__ __align__(16) unsigned char lin_smem[];
    __shared__ __align__(8) u64 bars[2 * LIN_MAX_STAGES + 2];
    __shared__ u32 tmem_base;
    __shared__ volatile int gave_up;
    const u32 warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const u32 base = (smem_addr(lin_smem) + 1023) & ~1023u;
    const u32 full = smem_addr(bars), empty = full + 8 * LIN_MAX_STAGES, acc_full = empty + 8 * LIN_MAX_STAGES, acc_empty = acc_full + 8;
    if (threadIdx.x == 0) {
        for (u32 s = 0; s < p.stages; s++) { mbar_init(full + 8 * s, 1); mbar_init(empty + 8 * s, 1); }
        mbar_init(acc_full, 1);
        mbar_init(acc_empty, 4);
        gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) tmem_alloc(smem_addr(&tmem_base), p.tmem_cols);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const u32 tmem = tmem_base, b_bytes = p.tt * 512;
    LinWalk walk(p);
    if (warp == 0) {
        if (lane == 0) {
            u32 it = 0;
            bool ok = true;
            while (ok && walk.next()) {
                for (u32 k = 0; k < walk.count; k++, it++) {
                    const u32 s = it % p.stages, round = it / p.stages, st = base + s * p.stage_bytes;
                    if (round && !(ok = mbar_wait(empty + 8 * s, (round - 1) & 1, &gave_up))) break;
                    mbar_expect(full + 8 * s, p.stage_bytes);
                    tensor_load_2d(st, &map_w, (int)((walk.first + k) * LIN_STEP), (int)(walk.mt * LIN_ROWS), full + 8 * s);
                    bulk_load(st + LIN_ROWS * 128, digits + ((size_t)walk.nt * p.steps + walk.first + k) * b_bytes, b_bytes, full + 8 * s);
                }
            }
            if (!ok)                             // given up: nothing of this CTA may still be in flight when it ends
                for (u32 i = it > p.stages ? it - p.stages : 0; i < it; i++)
                    for (u32 n = 0; n < (1u << 16) && !mbar_try(full + 8 * (i % p.stages), (i / p.stages) & 1); n++) {}
        }
    } else if (warp == 1) {
        if (lane == 0) {
            const u32 idesc = i8_instr_desc(4 * p.tt);
            u32 it = 0, n = 0;
            bool ok = true;
            while (ok && walk.next()) {
                if (n && !(ok = mbar_wait(acc_empty, (n - 1) & 1, &gave_up))) { mma_commit(acc_full); n++; break; }
                tc_fence_after();
                const bool two = walk.mt * LIN_ROWS + 128 < p.m;
                for (u32 k = 0; k < walk.count; k++, it++) {
                    const u32 s = it % p.stages, st = base + s * p.stage_bytes;
                    if (!(ok = mbar_wait(full + 8 * s, (it / p.stages) & 1, &gave_up))) break;
                    tc_fence_after();
                    const u64 a = smem_desc_sw128(st), b = smem_desc_sw128(st + LIN_ROWS * 128);
#pragma unroll
                    for (u32 kk = 0; kk < 4; kk++) mma_u8(tmem, a + 2 * kk, b + 2 * kk, idesc, k || kk);
                    if (two) {
#pragma unroll
                        for (u32 kk = 0; kk < 4; kk++) mma_u8(tmem + 4 * p.tt, a + (16384 >> 4) + 2 * kk, b + 2 * kk, idesc, k || kk);
                    }
                    mma_commit(empty + 8 * s);
                }
                mma_commit(acc_full);
                n++;
            }
            if (!ok)
                for (u32 i = 0; i < (1u << 16) && !mbar_try(acc_full, (n - 1) & 1); i++) {}
        }
    } else {
        const u32 quarter = warp & 3;            // the lanes of TMEM that this warp may read
        u32 n = 0;
        while (walk.next()) {
            if (!mbar_wait(acc_full, n & 1, &gave_up)) break;
            tc_fence_after();
            u32* slot = slots + (size_t)walk.slot * p.slot_words;
            for (u32 half = 0; half < 2; half++) {
                const u32 row = half * 128 + quarter * 32 + lane;
                if (walk.mt * LIN_ROWS + half * 128 >= p.m) break;
                for (u32 t0 = 0; t0 < p.tt; t0 += 16) {
                    u32 v[4][16];
#pragma unroll
                    for (u32 g = 0; g < 4; g++)
                        if (t0 + 4 * g < p.tt) tmem_load16(tmem + (quarter << 21) + half * 4 * p.tt + 4 * t0 + 16 * g, v[g]);
                    tmem_wait_load();
#pragma unroll
                    for (u32 g = 0; g < 4; g++)
                        if (t0 + 4 * g < p.tt) {
#pragma unroll
                            for (u32 e = 0; e < 4; e++)
                                slot[(size_t)(t0 + 4 * g + e) * LIN_ROWS + row] =
                                    red64((u64)v[g][4 * e] + ((u64)v[g][4 * e + 1] << 8) + ((u64)v[g][4 * e + 2] << 16) + ((u64)v[g][4 * e + 3] << 24));
                        }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(acc_empty);
            n++;
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 1) tmem_free(tmem, p.tmem_cols);
    if (threadIdx.x == 0 && gave_up) *gave_up_out = 1;
}

// Sum of one output's slots (see LinPlan).
__device__ __forceinline__ u64 lin_sum(const LinPlan& p, const u32* __restrict__ slots, u32 t, u32 i) {
    const u32 nt = t / p.tt, mt = i / LIN_ROWS, tile = mt * p.ntiles + nt;
    const size_t in = (size_t)(t - nt * p.tt) * LIN_ROWS + (i - mt * LIN_ROWS);
    const u64 begin = (u64)tile * p.steps;
    u64 s = 0;
    for (u32 seg = 0; seg < p.segs; seg++) {
        const u64 b = begin + seg * LIN_SEG, e = begin + ((seg + 1) * LIN_SEG < p.steps ? (seg + 1) * LIN_SEG : p.steps);
        for (u32 c = (u32)(b / p.per); c <= (u32)((e - 1) / p.per); c++) s += slots[((size_t)c + (size_t)tile * p.segs + seg) * p.slot_words + in];
    }
    return s;
}
__global__ void __launch_bounds__(256) linear_join_kernel(LinearArgs A, LinPlan p, const u32* __restrict__ slots, const u32* __restrict__ u) {
    const u32 i = blockIdx.x * 256 + threadIdx.x, t = blockIdx.y;
    if (i >= A.m) return;
    u64 y = lin_sum(p, slots, t, i) + (A.bias ? A.bias[i] : 0);
    const int of = u ? A.adapter_of[t] : -1;
    if (of >= 0 && (u32)of < A.num_adapters)
        for (u32 r = 0; r < A.rank; r++) y += mul31(A.b[((size_t)of * A.m + i) * A.rank + r], u[(size_t)t * A.rank + r]);
    A.y[t * A.y_stride + i] = red64(y);
}

// u[t][r] = A[of[t]][r] . x[t]; a warp per (token, r).
__global__ void __launch_bounds__(256) adapter_shrink_kernel(LinearArgs A, u32* __restrict__ u) {
    const u32 w = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (w >= A.tokens * A.rank) return;
    const u32 t = w / A.rank, r = w - t * A.rank;
    const int of = A.adapter_of[t];
    u64 acc = 0;
    if (of >= 0 && (u32)of < A.num_adapters) {
        const u32* a = A.a + ((size_t)of * A.rank + r) * A.n;
        const u32* x = A.x + t * A.x_stride;
        for (u32 j = lane; j < A.n; j += 32) acc += mul31(a[j], x[j]);
    }
    u32 s = red64(acc);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) s = add31(s, __shfl_xor_sync(0xffffffffu, s, off));
    if (lane == 0) u[w] = s;
}

// A 32 x 32 tile of Y per CTA.
__global__ void __launch_bounds__(256) adapter_linear_kernel(LinearArgs A, const u32* __restrict__ u) {
    __shared__ u32 ws[32][33], xs[32][33];
    const u32 i0 = blockIdx.x * 32, t0 = blockIdx.y * 32, tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    u64 acc[4] = {0, 0, 0, 0};
    for (u32 j0 = 0; j0 < A.n; j0 += 32) {
        for (u32 r = ty; r < 32; r += 8) {
            ws[r][tx] = i0 + r < A.m && j0 + tx < A.n ? A.w[(size_t)(i0 + r) * A.n + j0 + tx] : 0;
            xs[r][tx] = t0 + r < A.tokens && j0 + tx < A.n ? A.x[(t0 + r) * A.x_stride + j0 + tx] : 0;
        }
        __syncthreads();
        for (u32 j = 0; j < 32; j++)
            for (int k = 0; k < 4; k++) acc[k] += mul31(ws[tx][j], xs[ty + 8 * k][j]);
        __syncthreads();
    }
    const u32 i = i0 + tx;
    if (i >= A.m) return;
    for (int k = 0; k < 4; k++) {
        const u32 t = t0 + ty + 8 * k;
        if (t >= A.tokens) continue;
        u64 y = acc[k] + (A.bias ? A.bias[i] : 0);
        const int of = u ? A.adapter_of[t] : -1;
        if (of >= 0 && (u32)of < A.num_adapters)
            for (u32 r = 0; r < A.rank; r++) y += mul31(A.b[((size_t)of * A.m + i) * A.rank + r], u[(size_t)t * A.rank + r]);
        A.y[t * A.y_stride + i] = red64(y);
    }
}

}  // namespace zkb
