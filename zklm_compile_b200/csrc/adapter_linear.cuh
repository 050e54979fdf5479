// Y = X W^T + bias, and for a token with an adapter + B_a (A_a x), all mod p.
#pragma once
#include "m31.cuh"
#include "serving.cuh"

namespace zkb {

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
