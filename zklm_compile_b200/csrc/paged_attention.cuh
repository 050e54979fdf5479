// One new token per sequence over its cached positions.
//
//   s_j = q . k_j,  e_j = table[rnd(s_j / 2^shift)],  out = (sum_j e_j v_j) / (sum_j e_j)
//
// in the field, s_j read as a centred integer and rounded half away from zero.  The table stands in for exp, so no running maximum is
// needed: both sums are plain sums mod p, and parts of a row join by adding.
#pragma once
#include "m31.cuh"
#include "kv_append.cuh"
#include "serving.cuh"

namespace zkb {

constexpr int PA_THREADS = 256;
constexpr u32 PA_MAX_D = 256;

// One CTA: one (sequence, head).
__global__ void __launch_bounds__(PA_THREADS) paged_attention_kernel(PagedAttnArgs A) {
    __shared__ u32 q[PA_MAX_D], e[PA_THREADS];
    __shared__ u32 out[PA_MAX_D];
    const u32 seq = blockIdx.x, head = blockIdx.y, d = A.c.d, kvh = head / (A.num_heads / A.c.num_kv_heads);
    const u32 lane = threadIdx.x & 31, warp = threadIdx.x >> 5, mask = (1u << A.c.page_bits) - 1;
    const int len = A.lens[seq];
    u32* to = A.out + ((size_t)seq * A.num_heads + head) * d;
    for (u32 i = threadIdx.x; i < d; i += PA_THREADS) { q[i] = A.q[seq * A.q_stride + (size_t)head * d + i]; out[i] = 0; }
    __syncthreads();
    int bad = len < 0 || (u64)len > ((u64)A.max_blocks << A.c.page_bits) ? SERVE_PAGE : 0;
    u32 sum = 0;
    for (int base = 0; !bad && base < len; base += PA_THREADS) {
        const int n = len - base < PA_THREADS ? len - base : PA_THREADS;
        int mine = 0;
        for (int j = warp; j < n; j += PA_THREADS / 32) {
            const u32 pos = base + j;
            const int page = A.block_table[(size_t)seq * A.max_blocks + (pos >> A.c.page_bits)];
            u32 ev = 0;
            if (page < 0 || (u32)page >= A.c.num_pages) mine = max(mine, (int)SERVE_PAGE);
            else {
                const size_t at = (size_t)page * A.c.page_stride + (((size_t)kvh << A.c.page_bits) + (pos & mask)) * d;
                u64 acc = 0;
                for (u32 i = lane; i < d; i += 32) {
                    const int z = A.c.small ? ((const int16_t*)A.c.k)[at + i] : 0;
                    const u32 kk = A.c.small ? (z < 0 ? (u32)z + ZKB_P : (u32)z) : ((const u32*)A.c.k)[at + i];
                    acc += mul31(kk, q[i]);
                }
                u32 s = red64(acc);
#pragma unroll
                for (int off = 16; off > 0; off >>= 1) s = add31(s, __shfl_xor_sync(0xffffffffu, s, off));
                long long x = centred32(s), a = x < 0 ? -x : x;
                if (A.score_shift) a = (a + (1ll << (A.score_shift - 1))) >> A.score_shift;
                x = x < 0 ? -a : a;
                const int half = (int)(A.n_table / 2);
                if (x < -half || x >= half) mine = max(mine, (int)SERVE_SCORE);
                else ev = A.table[x < 0 ? x + A.n_table : x];
            }
            if (lane == 0) e[j] = ev;
        }
        bad = __syncthreads_or(mine == SERVE_PAGE) ? SERVE_PAGE : (__syncthreads_or(mine) ? SERVE_SCORE : 0);
        if (bad) break;
        for (u32 i = threadIdx.x; i < d; i += PA_THREADS) {
            u64 acc = out[i];
            for (int j = 0; j < n; j++) {
                const u32 pos = base + j;
                const int page = A.block_table[(size_t)seq * A.max_blocks + (pos >> A.c.page_bits)];
                const size_t at = (size_t)page * A.c.page_stride + (((size_t)kvh << A.c.page_bits) + (pos & mask)) * d + i;
                const int z = A.c.small ? ((const int16_t*)A.c.v)[at] : 0;
                const u32 vv = A.c.small ? (z < 0 ? (u32)z + ZKB_P : (u32)z) : ((const u32*)A.c.v)[at];
                acc += mul31(e[j], vv);
            }
            out[i] = red64(acc);
        }
        for (int j = 0; j < n; j++) sum = add31(sum, e[j]);
        __syncthreads();
    }
    if (!bad && len > 0 && sum == 0) bad = SERVE_ZERO_SUM;
    if (bad && threadIdx.x == 0) atomicMax(A.status + seq, bad);
    const u32 inv = bad ? 0 : inv31(sum);
    for (u32 i = threadIdx.x; i < d; i += PA_THREADS) to[i] = mul31(out[i], inv);
}

}  // namespace zkb
