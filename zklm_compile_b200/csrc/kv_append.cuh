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
// |x| <= 2^62 -> x / 2^shift rounded half away from zero, mod p.  Half less one unit, where x is negative, makes the floor of a shift round away from zero there too;
// 2^32 p = 2^63 - 2^32 makes the sum positive.
__device__ __forceinline__ u32 round_to_field(long long x, u32 shift) {
    const long long away = shift ? x >> 63 : 0;
    const long long y = (x + (long long)((1ull << shift) >> 1) + away) >> shift;
    return red64((u64)y + ((u64)ZKB_P << 32));
}

// Where a token goes.  All threads of the CTA call it; false: padding, or refused (and reported).
struct AppendPlace { u32 seq; long long pos; int page; };
__device__ __forceinline__ bool append_place(const AppendArgs& A, u32 t, AppendPlace& p) {
    p.seq = 0;                                                // sequences that end before t
    for (u32 base = 0; base < A.num_seqs; base += APPEND_THREADS) {
        const u32 s = base + threadIdx.x;
        p.seq += __syncthreads_count(s < A.num_seqs && A.row_start[s + 1] <= (int)t);
    }
    if (p.seq >= A.num_seqs) return false;                    // behind the last sequence
    const int first = A.row_start[p.seq];
    if ((int)t < first) return false;
    p.pos = (long long)A.start[p.seq] + ((int)t - first);
    const long long block = p.pos >> A.c.page_bits;
    p.page = p.pos >= 0 && block < A.max_blocks ? A.block_table[(size_t)p.seq * A.max_blocks + block] : -1;
    const bool have_page = p.page >= 0 && (u32)p.page < A.c.num_pages, have_rot = A.rot == 0 || (p.pos >= 0 && p.pos < A.positions);
    if (have_page && have_rot) return true;
    if (threadIdx.x == 0) atomicMax(A.status + p.seq, have_page ? SERVE_ROTATION : SERVE_PAGE);
    return false;
}
__device__ __forceinline__ void rotate_pair(u32& a, u32& b, int c, int s, u32 shift) {
    const long long x = centred32(a), y = centred32(b);
    a = round_to_field(x * c - y * s, shift);
    b = round_to_field(x * s + y * c, shift);
}

// 16 bytes at a time, for rows, rotations and addresses that are whole groups of 16 bytes (see kv_append_launch).  What bounds it is the copy: K, V and
// Q in, the cache and Q out.  A row has `items` items: four neighbours, or where halves turn four elements and their four partners; a thread has the same item in
// every row that it takes, so its cosines and sines stay in registers.  The first rows are read before the place is looked up.
// 8111 tokens of 32 + 2 x 8 heads of 128, a quarter of each turned, into a field cache (400 MB): 69 us, 5.8 TB/s; into a 16-bit one (367 MB) 68 us.
template <bool SMALL, bool PAIRS>
__global__ void __launch_bounds__(APPEND_THREADS, 4) kv_append_vec_kernel(AppendArgs A, u32 items, u32 rot_items) {
    constexpr u32 BATCH = PAIRS ? 6 : 3;                       // rows under way, 16 bytes or 32 of each
    const u32 t = blockIdx.x, d = A.c.d, kv = A.c.num_kv_heads, half = A.rot / 2, rows = 2 * kv + (A.q ? A.num_heads : 0);
    const u32 per_pass = APPEND_THREADS / items, step = gridDim.y * per_pass, turning = per_pass * rot_items;
    // the first threads have the items that turn, so that few warps have both kinds
    const bool turns = threadIdx.x < turning, two = !PAIRS && turns;
    const u32 still = items - rot_items, rest = threadIdx.x - turning;
    const u32 item = turns ? threadIdx.x % rot_items : still ? rot_items + rest % still : 0, in_pass = turns ? threadIdx.x / rot_items : still ? rest / still : per_pass;
    const u32 e0 = PAIRS || turns ? 4 * item : A.rot + 4 * (item - rot_items), e1 = half + 4 * item;
    u32 row = in_pass < per_pass ? blockIdx.y * per_pass + in_pass : rows;
    uint4 a[BATCH], b[BATCH];
    auto load = [&](u32 from_row) {
#pragma unroll
        for (u32 k = 0; k < BATCH; k++) {
            const u32 r = from_row + k * step;
            if (r >= rows) break;
            const u32* src = r < kv ? A.k + t * A.k_stride + (size_t)r * d : r < 2 * kv ? A.v + t * A.v_stride + (size_t)(r - kv) * d : A.q + t * A.q_stride + (size_t)(r - 2 * kv) * d;
            a[k] = __ldcs(reinterpret_cast<const uint4*>(src + e0));
            if (two) b[k] = __ldcs(reinterpret_cast<const uint4*>(src + e1));
        }
    };
    load(row);
    AppendPlace p;
    if (!append_place(A, t, p)) return;
    int4 cs0 = make_int4(0, 0, 0, 0), cs1 = cs0;              // cos, sin of two pairs each
    if (turns) {
        const int4* cs = reinterpret_cast<const int4*>(A.cos_sin + (size_t)p.pos * A.rot + (PAIRS ? 4 : 8) * item);
        cs0 = cs[0];
        if (!PAIRS) cs1 = cs[1];
    }
    const size_t at = (size_t)p.page * A.c.page_stride + (size_t)(p.pos & ((1u << A.c.page_bits) - 1)) * d;
    bool out_of_range = false;
    while (row < rows) {
#pragma unroll
        for (u32 k = 0; k < BATCH; k++) {
            const u32 r = row + k * step;
            if (r >= rows) break;
            const bool is_k = r < kv, is_v = !is_k && r < 2 * kv;
            if (turns && !is_v) {
                if (PAIRS) {
                    rotate_pair(a[k].x, a[k].y, cs0.x, cs0.y, A.shift);
                    rotate_pair(a[k].z, a[k].w, cs0.z, cs0.w, A.shift);
                } else {
                    rotate_pair(a[k].x, b[k].x, cs0.x, cs0.y, A.shift);
                    rotate_pair(a[k].y, b[k].y, cs0.z, cs0.w, A.shift);
                    rotate_pair(a[k].z, b[k].z, cs1.x, cs1.y, A.shift);
                    rotate_pair(a[k].w, b[k].w, cs1.z, cs1.w, A.shift);
                }
            }
            if (!is_k && !is_v) {
                u32* to = A.q_out + t * A.q_out_stride + (size_t)(r - 2 * kv) * d;
                __stcs(reinterpret_cast<uint4*>(to + e0), a[k]);
                if (two) __stcs(reinterpret_cast<uint4*>(to + e1), b[k]);
                continue;
            }
            const size_t to = at + ((size_t)(is_k ? r : r - kv) << A.c.page_bits) * d;
            if (SMALL) {
                auto put = [&](u32 e, const uint4& v) {
                    const int z[4] = {centred32(v.x), centred32(v.y), centred32(v.z), centred32(v.w)};
#pragma unroll
                    for (int i = 0; i < 4; i++) out_of_range |= z[i] != (int)(int16_t)z[i];
                    *reinterpret_cast<uint2*>((int16_t*)(is_k ? A.c.k : A.c.v) + to + e) = make_uint2(__byte_perm(z[0], z[1], 0x5410), __byte_perm(z[2], z[3], 0x5410));
                };
                put(e0, a[k]);
                if (two) put(e1, b[k]);
            } else {
                u32* pages = (u32*)(is_k ? A.c.k : A.c.v) + to;
                *reinterpret_cast<uint4*>(pages + e0) = a[k];
                if (two) *reinterpret_cast<uint4*>(pages + e1) = b[k];
            }
        }
        row += BATCH * step;
        load(row);
    }
    if (out_of_range) atomicMax(A.status + p.seq, SERVE_RANGE);
}

// Any sizes and alignment.  One CTA: one token, the rows (heads of k, v, q) y, y + gridDim.y, ... by warp.
__global__ void __launch_bounds__(APPEND_THREADS) kv_append_kernel(AppendArgs A) {
    const u32 t = blockIdx.x;
    AppendPlace place;
    if (!append_place(A, t, place)) return;
    const u32 seq = place.seq;
    const long long pos = place.pos;
    const int page = place.page;
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
            u32 x = src[i], y = src[j];
            rotate_pair(x, y, cs[2 * p], cs[2 * p + 1], A.shift);
            put(i, x);
            put(j, y);
        }
        for (u32 i = rot + lane; i < d; i += 32) put(i, src[i]);
    }
    if (out_of_range) atomicMax(A.status + seq, SERVE_RANGE);
}

}  // namespace zkb
