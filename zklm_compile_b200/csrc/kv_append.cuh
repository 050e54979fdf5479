// Keys and values of new tokens into their pages, K and Q rotated by position on the way.
//
//   (a, b) -> (rnd((a c - b s) / 2^shift), rnd((a s + b c) / 2^shift))
//
// on the centred integers that the field elements stand for, rnd to the nearest integer and halves away from zero (the framework's
// rounding of requantised values), then back into the field.  c, s are integers of `shift` fractional bits from the caller's table, so
// the rotation is one exact map and not a matter of a sine's last bit.
#pragma once
#include "m31.cuh"
#include "serving.cuh"

namespace zkb {

constexpr int APPEND_THREADS = 256;

__device__ __forceinline__ int centred32(u32 v) { return v > ZKB_P / 2 ? (int)(v - ZKB_P) : (int)v; }
// |x| <= 2^62 -> (rounded half away from zero) mod p
__device__ __forceinline__ u32 round_to_field(long long x, u32 shift) {
    u64 m = (u64)(x < 0 ? -x : x);
    if (shift) m = (m + (1ull << (shift - 1))) >> shift;
    const u32 r = red64(m);
    return x < 0 ? neg31(r) : r;
}

// One CTA: one token, the rows (heads of k, v, q) y, y + gridDim.y, ... by warp.
__global__ void __launch_bounds__(APPEND_THREADS) kv_append_kernel(AppendArgs A) {
    const u32 t = blockIdx.x;
    u32 seq = 0;
    for (u32 base = 0; base < A.num_seqs; base += APPEND_THREADS) {
        const u32 s = base + threadIdx.x;
        seq += __syncthreads_count(s < A.num_seqs && A.row_start[s + 1] <= (int)t);
    }
    if (seq >= A.num_seqs) return;                            // behind the last sequence
    const int first = A.row_start[seq];
    if ((int)t < first) return;
    const long long pos = (long long)A.start[seq] + ((int)t - first);
    const long long block = pos >> A.c.page_bits;
    const int page = pos >= 0 && block < A.max_blocks ? A.block_table[(size_t)seq * A.max_blocks + block] : -1;
    const bool have_page = page >= 0 && (u32)page < A.c.num_pages, have_rot = A.rot == 0 || (pos >= 0 && pos < A.positions);
    if (!have_page || !have_rot) {
        if (threadIdx.x == 0) atomicMax(A.status + seq, have_page ? SERVE_ROTATION : SERVE_PAGE);
        return;
    }
    const u32 d = A.c.d, kv = A.c.num_kv_heads, half = A.rot / 2, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const u32 rows = 2 * kv + (A.q ? A.num_heads : 0);
    const int* cs = A.cos_sin + (size_t)pos * A.rot;
    bool out_of_range = false;
    for (u32 row = blockIdx.y * (APPEND_THREADS / 32) + warp; row < rows; row += gridDim.y * (APPEND_THREADS / 32)) {
        const bool is_k = row < kv, is_v = !is_k && row < 2 * kv;
        const u32 h = is_k ? row : (is_v ? row - kv : row - 2 * kv);
        const u32* src = is_k ? A.k + t * A.k_stride : (is_v ? A.v + t * A.v_stride : A.q + t * A.q_stride);
        src += (size_t)h * d;
        const size_t at = (size_t)page * A.c.page_stride + ((size_t)h << A.c.page_bits) * d + (size_t)(pos & ((1u << A.c.page_bits) - 1)) * d;
        auto put = [&](u32 i, u32 v) {
            if (!is_k && !is_v) {
                A.q_out[t * A.q_out_stride + (size_t)h * d + i] = v;
            } else if (A.c.small) {
                const int z = centred32(v);
                out_of_range |= z < -32768 || z > 32767;
                ((int16_t*)(is_k ? A.c.k : A.c.v))[at + i] = (int16_t)z;
            } else {
                ((u32*)(is_k ? A.c.k : A.c.v))[at + i] = v;
            }
        };
        const u32 rot = is_v ? 0 : A.rot;
        for (u32 p = lane; p < rot / 2; p += 32) {             // both of a pair by one thread: q may be rotated in place
            const u32 i = A.pairs ? 2 * p : p, j = A.pairs ? 2 * p + 1 : p + half;
            const long long c = cs[2 * p], s = cs[2 * p + 1], x = centred32(src[i]), y = centred32(src[j]);
            put(i, round_to_field(x * c - y * s, A.shift));
            put(j, round_to_field(x * s + y * c, A.shift));
        }
        for (u32 i = rot + lane; i < d; i += 32) put(i, src[i]);
    }
    if (out_of_range) atomicMax(A.status + seq, SERVE_RANGE);
}

}  // namespace zkb
