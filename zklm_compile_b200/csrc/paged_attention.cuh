// One new token per sequence over its cached positions.
//
//   s_j = q . k_j,  e_j = table[rnd(s_j / 2^shift)],  out = (sum_j e_j v_j) / (sum_j e_j)
//
// in the field, s_j read as a centred integer and rounded half away from zero.  The table stands in for exp, so no running maximum is
// needed: both sums are plain sums mod p, and parts of a row join by adding.
//
// Both sums of products run on the integer tensor cores (mma.sync, unsigned bytes), with the cache's own bytes as the left operand: a
// product of field elements is sixteen products of bytes, w x = sum_c 2^(8c) sum_i w_i d_c(i) with d(i) the bytes of 2^(8i) x mod p, a
// rotation of x's 31 bits (digit_words).  A query head is four columns of the right operand.  For scores the 16 rows of a tile are
// positions and the depth runs over the bytes of a key; for the output the rows are elements of the head and the depth runs over the bytes
// of one element at several positions - either way a register of the left operand is a 32-bit word of the cache (two half words of two
// positions in a 16-bit cache), so nothing is transposed on the way.  16-bit elements are made unsigned by flipping their top bit, and
// 2^15 (sum of the other operand) is taken off at the end.
//
// What bounds it is reading the cache.  Every warp has a ring of half tiles of its own, filled by tensor copies (16 rows a copy) that an mbarrier a slot
// counts, so warps never wait for one another within a row.  (A bulk copy a row instead held the 16-bit cache to 3.4 TB/s.)  The work of a call
// is one list of blocks (positions of one sequence and key head) that the CTAs share evenly by its length, whatever the sequences' lengths are; a
// row that CTAs share is added up by the one that brings its last part.  Integer sums have no order, so results do not depend on the split.
//
// Measured, heads of 128: 48 rows of up to 6000 positions, 8 x 4 heads, field 5.8 TB/s (190 us); one row over 131071, 8 x 4 heads, 16-bit 5.4 TB/s (99 us); 64 rows
// of up to 5000, 8 x 8 heads, 16-bit 3.9 TB/s (230 us) - there 810 instructions a tile and the registers that eight heads' sums take bound it.
#pragma once
#include <type_traits>
#include "m31.cuh"
#include "kv_append.cuh"
#include "adapter_linear.cuh"
#include "serving.cuh"

namespace zkb {

constexpr u32 PA_FLUSH = 512;                 // blocks after which 32-bit sums move to 64 bits: 512 tiles x 16 positions x 4 x 255^2 < 2^31

// x^(p - 2) by powers 2^k - 1.
__device__ __forceinline__ u32 inv31_chain(u32 x) {
    auto sq = [](u32 v, int n) { for (int i = 0; i < n; i++) v = mul31(v, v); return v; };
    const u32 t2 = mul31(sq(x, 1), x), t3 = mul31(sq(t2, 1), x), t6 = mul31(sq(t3, 3), t3), t7 = mul31(sq(t6, 1), x), t14 = mul31(sq(t7, 7), t7);
    const u32 t28 = mul31(sq(t14, 14), t14), t29 = mul31(sq(t28, 1), x);
    return mul31(sq(t29, 2), x);               // 4 (2^29 - 1) + 1 = 2^31 - 3
}

// How the kernels are built for a head of up to DP elements: warps, and half tiles (16 keys or 16 values) in a warp's ring.  A half tile lies as the
// tensor copies leave it: columns of 128 bytes, 16 rows of one behind the other, the 16-byte groups of a row swizzled by the row's low bits.
// Which position becomes which row of an operand is free, and is chosen so that no two lanes of a phase meet in a bank.  Warps: as many as the registers of
// dp / 16 x nt x 4 sums a lane leave.  Twelve against eight, 131071 positions, 8 key heads with one / four heads each: 128 in 16 bits 90 / 94 against 94 / 105 us, 64 in 16 bits
// 66 / 74 against 84 / 92, 64 in the field 89 / 91 against 91 / 103; a few rows of 77 positions lose what the set-up of four more warps takes, 7.5 to 9.5 us against 7.0 to 8.5.
// Slots: about 130 to 160 KB of them.
template <int DP, bool SMALL, int NT>
struct PaShape {
    static constexpr int RB = DP * (SMALL ? 2 : 4);
    static constexpr int WARPS = RB >= 1024 ? 5 : (RB <= 256 && NT <= 2 ? 12 : 8);
    static constexpr int NS = RB >= 512 ? 2 : (RB == 256 ? (WARPS == 12 ? 3 : 4) : 6);
    static constexpr int HALF = 16 * RB;       // bytes of a slot
    static constexpr int ED = SMALL ? 256 : 512;   // bytes of a tile's weights, as digits, per tile of columns
};
struct PaWork {                                // see paged_attention_launch
    u32 slices, slice_heads, ctas;
    u32* slots;                                // [ctas][2][slice_heads][DP + 4]: sums, then the sum of weights and what went wrong
    u32* arrived;                              // [ctas], zero before and after a call: how many parts are there of the row that begins in this CTA
    u32* begun;                                // zero before and after a call: see pa_began
    int fast;                                  // tensor copies: rows are whole 16-byte groups on 16-byte boundaries, pages have 8 rows or more
    int q_vec;                                 // q is read 16 bytes at a time
    int whole;                                 // a box has all the columns of its rows
    int* gave_up;
};
enum : u32 { PA_BAD_PAGE = 1, PA_BAD_SCORE = 2 };

// How the blocks are shared is worked out by every CTA for itself from the lengths.  They are inputs, which nobody changes before the call has run; but
// should somebody, no address and no barrier may depend on its luck.  So all threads of a CTA compute by what one of them read, and a share is found in the
// lengths that it was counted by (up to PA_FEW sequences) or cut to what the arrays have.  The copies of a warp go by what the warp itself read, in bounds
// whatever it was.  What then becomes of the rows is nothing of use: a CTA that finds blocks missing or left over sets the give-up flag, and so does the
// next call if parts of a row are left in the counters, which it would add to.
constexpr u32 PA_FEW = 256;

// The blocks of a length: 0 for a sequence without positions and one whose length the block table cannot have.
ZKB_HD u32 pa_blocks(u64 positions, int l, u32 block, u32& len) {
    len = l < 0 || (u64)l > positions ? 0u : (u32)l;
    return (len + block - 1) / block;
}
// The stream of blocks that a CTA takes: sequences, in each its (key head, slice) items, in each its blocks.
struct PaWalk {
    u32 seq, kvh, slice, blk, nb, len, left;
    // Block `rest` (in shares of `per` where `aligned`) of sequence `at`, which has nb of them an item; rest < its items x its blocks.
    ZKB_HD void start(u32 at, u64 rest, u64 count, bool aligned, u32 per, u32 slices) {
        seq = at;
        const u32 parts = aligned ? (nb + per - 1) / per : nb, grp = rest >> 32 ? (u32)(rest / parts) : (u32)rest / parts;      // of an item, in what the rest is counted in
        kvh = grp / slices;
        slice = grp - kvh * slices;
        blk = (u32)(rest - (u64)grp * parts) * (aligned ? per : 1u);
        left = !aligned ? (u32)count : nb - blk < per ? nb - blk : per;
    }
    // n blocks on, within an item or to its end; true: what comes next is another sequence (next_seq).
    ZKB_HD bool step(u32 n, u32 slices, u32 kv_heads) {
        left -= n;
        blk += n;
        if (blk < nb || !left) return false;
        blk = 0;
        if (++slice < slices) return false;
        slice = 0;
        if (++kvh < kv_heads) return false;
        kvh = 0;
        return true;
    }
    // The next sequence that has blocks.  There is one while blocks are left; if not (see above) none is.
    template <class Length>
    ZKB_HD void next_seq(u32 num_seqs, u64 positions, u32 block, const Length& length) {
        do {
            if (++seq >= num_seqs) { seq = num_seqs - 1; nb = len = left = 0; return; }
            nb = pa_blocks(positions, length(seq), block, len);
        } while (nb == 0);
    }
};
// The CTAs that have a part of a row of nb blocks, from the first on; `at`: where in the list of blocks the row's block `first` lies, which CTA `cta` has.
// (A row that was not counted with these blocks may seem to begin before the list or to end behind it.)
struct PaParts { u32 first_cta, n; };
ZKB_HD PaParts pa_parts(bool aligned, u64 per, u32 ctas, u32 cta, u64 at, u32 first, u32 nb) {
    const u64 row0 = at - (first < at ? first : at);
    PaParts p;
    p.first_cta = aligned ? cta - first / (u32)per : (u32)(row0 / per);
    p.n = aligned ? (nb + (u32)per - 1) / (u32)per : (u32)((row0 + nb - 1) / per) - p.first_cta + 1;
    p.n = umin32(p.n, ctas - p.first_cta);
    return p;
}
// What is left in the counters of a row's parts is known from one more word: its high half has the parts that were brought less those that were added up, its low
// half the CTAs that began, the first of them as 1 - ctas, so that it is zero before a call, at its end, and in between not for a CTA that has not added itself.
// That CTA sees whether the call began with counters at zero; nothing is waited for.  (A word for the last CTA to clear, which has to wait for its own atomic:
// 0.4 us more in a call of 7, 0.9 in one of 19.)
ZKB_HD u32 pa_began(u32 cta, u32 ctas) { return cta ? 1u : 1u - ctas; }
ZKB_HD u32 pa_brought(u32 parts, u32 added) { return (parts - added) << 16; }
ZKB_HD bool pa_stale(u32 word) { return word != 0 && (word & 0xffffu) == 0; }

// Half tiles that a warp has copied into a ring of ns slots, `slot` being the next one's: the last of its tiles with its values or without.
ZKB_HD u32 pa_halves(u32 tiles, u32 slot, u32 ns) { return 2 * tiles % ns == slot ? 2 * tiles : 2 * tiles - 1; }

// One output row (or its part) in shared memory to where it belongs.
__device__ __forceinline__ void pa_finish(const PagedAttnArgs& A, u32 seq, u32 head, u32 e, u32 acc, u32 inv, u32 correction) {
    A.out[((size_t)seq * A.num_heads + head) * A.c.d + e] = mul31(sub31(acc, correction), inv);
}

template <int DP, bool SMALL, int NT>
__global__ void __launch_bounds__(PaShape<DP, SMALL, NT>::WARPS * 32, 1) paged_attention_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                                                                                                   PagedAttnArgs A, PaWork P) {
    using S = PaShape<DP, SMALL, NT>;
    constexpr int WARPS = S::WARPS, NS = S::NS, RB = S::RB, J = RB / 64, VJ = RB / 128, MT = DP / 16, HEADS = 2 * NT, THREADS = WARPS * 32;
    constexpr u32 BLOCK = WARPS * 16;
    extern __shared__ __align__(16) unsigned char pa_raw[];
    unsigned char* const pa_smem = pa_raw + ((0u - smem_addr(pa_raw)) & 1023u);    // the swizzle goes by addresses
    uint4* qd = reinterpret_cast<uint4*>(pa_smem + WARPS * NS * S::HALF);          // [J][NT][32]
    u32* part = reinterpret_cast<u32*>(qd + J * NT * 32);                          // [WARPS][HEADS][DP]: sums of e v
    unsigned char* digits = reinterpret_cast<unsigned char*>(part + WARPS * HEADS * DP);   // [WARPS][NT][ED]
    __shared__ u32 es_part[WARPS][HEADS], flag_part[WARPS][HEADS];                 // sums of e, and what went wrong
    __shared__ u32 off_q[HEADS], corr[HEADS], inv[HEADS], scan[32];
    __shared__ int few_lens[PA_FEW];
    __shared__ u32 found_seq, found_len;
    __shared__ u64 found_rest;
    __shared__ struct { PaWalk walk; u64 per, to; bool aligned; } share;           // as thread 0 has it
    __shared__ __align__(8) u64 bars[WARPS * NS];
    __shared__ volatile int gave_up;
    __shared__ int last_part;
    const u32 tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, q4 = lane & 3;
    const u32 grps = A.c.num_kv_heads * P.slices, hpg = A.num_heads / A.c.num_kv_heads, d = A.c.d;
    u32 begun = 0;
    if (tid == 0) {
        gave_up = 0;
        if (P.fast) { prefetch_tensor_map(&map_k); prefetch_tensor_map(&map_v); }
        begun = __ldcg(P.begun);
        atomicAdd(P.begun, pa_began(blockIdx.x, P.ctas));
    }

    // ---- this CTA's share of the blocks ---------------------------------------------------------
    // up to 256 sequences by every warp for itself, more by the CTA
    constexpr int K = PA_FEW / 32;
    const u64 positions = (u64)A.max_blocks << A.c.page_bits;
    u64 total = 0;
    u32 own_nb[K], own_len[K];
    const bool few = A.num_seqs <= PA_FEW;
    if (few) {
#pragma unroll
        for (int k = 0; k < K; k++) {
            own_nb[k] = own_len[k] = 0;
            if (32 * k + lane < A.num_seqs) own_nb[k] = pa_blocks(positions, A.lens[32 * k + lane], BLOCK, own_len[k]);
            if (warp == 0) few_lens[32 * k + lane] = own_len[k];      // for the others from the first barrier on
            total += own_nb[k];
        }
    } else {
        for (u32 s = tid; s < A.num_seqs; s += THREADS) { u32 len; total += pa_blocks(positions, A.lens[s], BLOCK, len); }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    if (!few) {
        __shared__ u64 sums[WARPS];
        if (lane == 0) sums[warp] = total;
        __syncthreads();
        total = 0;
#pragma unroll
        for (int w = 0; w < WARPS; w++) total += sums[w];
    }
    total *= grps;
    u64 per = total >> 31 ? (total + P.ctas - 1) / P.ctas : ((u32)total + P.ctas - 1) / P.ctas;      // a 64-bit division is hundreds of cycles
    // Where the rows are fewer than the CTAs each CTA keeps to one row (`aligned`: a share is `per` blocks of one item), if that costs no one much more;
    // a second row in a CTA costs as much as several blocks.
    bool aligned = false;
    if (few) {
        u32 rows = 0;
#pragma unroll
        for (int k = 0; k < K; k++) rows += __popc(__ballot_sync(0xffffffffu, own_nb[k] != 0));
        if (rows && (u64)rows * grps <= P.ctas) {
            for (u32 more = 0; more < 3 && !aligned; more++) {
                const u32 p = (u32)per + (more ? ((u32)per + 7) / 8 * more : 0);
                u32 shares = 0;
#pragma unroll
                for (int k = 0; k < K; k++) shares += (own_nb[k] + p - 1) / p;
                shares = __reduce_add_sync(0xffffffffu, shares);
                if ((u64)shares * grps <= P.ctas) {
                    aligned = true;
                    per = p;
                    total = (u64)shares * grps;
#pragma unroll
                    for (int k = 0; k < K; k++) own_nb[k] = (own_nb[k] + p - 1) / p;       // in shares from here on
                }
            }
        }
    }
    const u64 from = aligned ? blockIdx.x : per * blockIdx.x, to = aligned ? (from < total ? from + 1 : from) : from + per < total ? from + per : total;
    // rows without positions are zero
    for (u32 s = blockIdx.x; s < A.num_seqs; s += P.ctas) {
        u32 len;
        const int l = A.lens[s];
        if (pa_blocks(positions, l, BLOCK, len)) continue;
        for (u32 i = tid; i < A.num_heads * d; i += THREADS) A.out[(size_t)s * A.num_heads * d + i] = 0;
        if (tid == 0 && l != 0) atomicMax(A.status + s, (int)SERVE_PAGE);
    }
    u32 start_seq = 0, start_len = 0;          // the sequence in which block `from` lies, and the blocks of it that lie before
    u64 start_rest = 0, before = 0;
    if (from >= to) {
        // nothing for this CTA
    } else if (few) {
#pragma unroll
        for (int k = 0; k < K; k++) {
            if (32u * k >= A.num_seqs) break;
            u32 x = own_nb[k];
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) { const u32 y = __shfl_up_sync(0xffffffffu, x, o); if ((int)lane >= o) x += y; }
            const u64 end = (before + x) * grps, begin = end - (u64)own_nb[k] * grps;
            const u32 here = __ballot_sync(0xffffffffu, begin <= from && from < end);
            if (here) {
                start_seq = 32 * k + __ffs(here) - 1;
                start_rest = from - __shfl_sync(0xffffffffu, begin, __ffs(here) - 1);
                start_len = __shfl_sync(0xffffffffu, own_len[k], __ffs(here) - 1);
            }
            before += __shfl_sync(0xffffffffu, x, 31);
        }
    } else {
        if (tid == 0) { found_seq = found_len = 0; found_rest = 0; }
        for (u32 base = 0;; base += THREADS) {
            u32 len = 0, nb = base + tid < A.num_seqs ? pa_blocks(positions, A.lens[base + tid], BLOCK, len) : 0u, x = nb;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) { const u32 y = __shfl_up_sync(0xffffffffu, x, o); if ((int)lane >= o) x += y; }
            if (lane == 31) scan[warp] = x;
            __syncthreads();
            u64 w = 0, all = 0;
#pragma unroll
            for (int i = 0; i < WARPS; i++) { if (i < (int)warp) w += scan[i]; all += scan[i]; }
            const u64 end = (before + w + x) * grps, begin = end - (u64)nb * grps;
            if (nb && begin <= from && from < end) { found_seq = base + tid; found_len = len; found_rest = from - begin; }
            before += all;
            __syncthreads();
            if (before * grps > from || base + THREADS >= A.num_seqs) break;
        }
        start_seq = found_seq;
        start_len = found_len;
        start_rest = found_rest;
    }
    PaWalk cw{};
    cw.nb = pa_blocks(positions, (int)start_len, BLOCK, cw.len);
    if (cw.nb) cw.start(start_seq, start_rest, to - from, aligned, (u32)per, P.slices);
    if (pa_stale(begun) || (from < to && !cw.nb)) *P.gave_up = 1;       // see above
    if (tid == 0) { share.walk = cw; share.per = per; share.to = to; share.aligned = aligned; }
    PaWalk lw = cw;                            // the copies run ahead of the computation

    // ---- copies -------------------------------------------------------------------------------------
    const u32 ring_at = warp * NS * S::HALF, ring = smem_addr(pa_smem) + ring_at, bar0 = smem_addr(bars + warp * NS);
    const u32 mask = (1u << A.c.page_bits) - 1;
    constexpr u32 E = SMALL ? 2 : 4;
    const u32 row_bytes = d * E;
    const u64 page_bytes = A.c.page_stride * E;
    const u32 columns = (row_bytes + 127) / 128;
    if (lane == 0) {
        for (int i = 0; i < NS; i++) mbar_init(bar0 + 8 * i, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async;" ::: "memory");
    }
    __syncwarp();
    u32 bad_pages = 0, loaded = 0;             // bit k: the tile k tiles behind the last one that was copied has a bad page
    // With tensor copies a tile lies in one page (two of 8 rows), the same for all lanes, fetched a tile ahead; without, lanes 0 .. 15 look up their rows'.
    int next0 = 0, next1 = 0, page0 = -1, page1 = -1;
    auto page_of = [&](u32 pos) { return A.block_table[(size_t)lw.seq * A.max_blocks + (pos >> A.c.page_bits)]; };
    auto fetch_page = [&] {
        const u32 pos0 = lw.blk * BLOCK + warp * 16;
        if (!P.fast || !lw.left) return;
        next0 = pos0 < lw.len ? page_of(pos0) : 0;
        if (P.fast == 8) next1 = pos0 + 8 < lw.len ? page_of(pos0 + 8) : 0;
    };
    u32 slot_in = 0;
    auto load_half = [&](bool is_v) {          // the next half tile into the next slot
        if (!lw.left) return;
        const u32 pos0 = lw.blk * BLOCK + warp * 16, bar = bar0 + 8 * slot_in, kv_row = lw.kvh << A.c.page_bits;
        if (P.fast) {
            // boxes of 16 rows (8 where a page has no more), all of a row where it is whole columns of 128 bytes, else a column each
            if (!is_v) {
                const bool fine0 = (u32)next0 < A.c.num_pages, fine1 = (u32)next1 < A.c.num_pages;
                page0 = fine0 && pos0 < lw.len ? next0 : -1;
                page1 = fine1 && P.fast == 8 && pos0 + 8 < lw.len ? next1 : -1;
                bad_pages = bad_pages << 1 | (u32)(!fine0 || !fine1);
                loaded++;
            }
            const u32 bytes = columns * 128 * P.fast, dst = ring + slot_in * S::HALF, step = P.whole ? columns : 1u;
            mbar_expect_one(bar, (page0 >= 0 ? bytes : 0u) + (page1 >= 0 ? bytes : 0u));
            const CUtensorMap* map = is_v ? &map_v : &map_k;
            for (u32 c = 0; c < columns; c += step) {
                if (page0 >= 0) tensor_load_4d_one(dst + c * 2048, map, (int)(c * (128 / E)), (int)(kv_row + (pos0 & mask)), 0, page0, bar);
                if (page1 >= 0) tensor_load_4d_one(dst + c * 2048 + 1024, map, (int)(c * (128 / E)), (int)(kv_row + ((pos0 + 8) & mask)), 0, page1, bar);
            }
        } else {                               // a word at a time, nothing under way: 3.9 ms for the 48 rows in pages of four, against 0.2 by copies
            const u32 pos = pos0 + lane;
            const bool there = lane < 16 && pos < lw.len;
            const int page = there ? page_of(pos) : 0;
            const bool fine = (u32)page < A.c.num_pages;
            if (!is_v) {
                bad_pages = bad_pages << 1 | (__any_sync(0xffffffffu, !fine) ? 1u : 0u);
                loaded++;
            }
            const char* src = (const char*)(is_v ? A.c.v : A.c.k) + (u64)(u32)page * page_bytes + (u64)(kv_row + (pos & mask)) * row_bytes;
            for (int r = 0; r < 16; r++) {
                const char* from_row = (const char*)__shfl_sync(0xffffffffu, (u64)src, r);
                if (!__shfl_sync(0xffffffffu, (int)(there && fine), r)) continue;
                unsigned char* to_row = pa_smem + ring_at + slot_in * S::HALF + r * 128;
                for (u32 i = lane; i < d; i += 32) {
                    const u32 byte = i * E;
                    unsigned char* w = to_row + (byte >> 7) * 2048 + ((byte & 127) ^ ((r & 7) << 4));
                    if (SMALL) *reinterpret_cast<uint16_t*>(w) = reinterpret_cast<const uint16_t*>(from_row)[i];
                    else *reinterpret_cast<u32*>(w) = reinterpret_cast<const u32*>(from_row)[i];
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(bar);
        }
        if (is_v) {
            if (lw.step(1, P.slices, A.c.num_kv_heads)) {
                lw.next_seq(A.num_seqs, (u64)A.max_blocks << A.c.page_bits, BLOCK, [&](u32 s) { return __shfl_sync(0xffffffffu, A.lens[s], 0); });
                if (!lw.left) gave_up = 1;     // blocks are missing: nobody waits for them
            }
            fetch_page();
        }
        slot_in = slot_in + 1 == NS ? 0 : slot_in + 1;
    };
    // A thread's elements of q for a row: four words' places of one head for each of its items, fetched ahead of their use.
    constexpr int Q_ITEMS = (HEADS * J * 4 + THREADS - 1) / THREADS;
    constexpr u32 Q_WORDS = SMALL ? 8 : 4;
    u32 qv[Q_ITEMS][Q_WORDS];
    auto fetch_q = [&](u32 seq, u32 head0, u32 heads) {
#pragma unroll
        for (int it = 0; it < Q_ITEMS; it++) {
            const u32 i = tid + it * THREADS, head = i / (J * 4), e0 = (16 * (i / 4 % J) + 4 * (i & 3)) * (SMALL ? 2 : 1);
            const u32* from_q = A.q + seq * A.q_stride + (size_t)(head0 + head) * d + e0;
#pragma unroll
            for (u32 k = 0; k < Q_WORDS; k += 4) {
                if (P.q_vec) {
                    const uint4 t = head < heads && e0 + k < d ? *reinterpret_cast<const uint4*>(from_q + k) : make_uint4(0, 0, 0, 0);
                    qv[it][k] = t.x; qv[it][k + 1] = t.y; qv[it][k + 2] = t.z; qv[it][k + 3] = t.w;
                } else {
#pragma unroll
                    for (u32 e = k; e < k + 4; e++) qv[it][e] = head < heads && e0 + e < d ? from_q[e] : 0u;
                }
            }
        }
    };
    auto heads_of = [&](const PaWalk& w) { const u32 rest = hpg - w.slice * P.slice_heads; return rest < P.slice_heads ? rest : P.slice_heads; };
    auto head0_of = [&](const PaWalk& w) { return w.kvh * hpg + w.slice * P.slice_heads; };
    fetch_page();
    if (cw.left) fetch_q(cw.seq, head0_of(cw), heads_of(cw));
#pragma unroll
    for (int h = 0; h < NS; h++) load_half(h & 1);

    // keys: lane (g, q4) reads rows k_row and k_row + 8, so that a phase has two rows four apart; values: rows 2 q4 and 2 q4 + 1 (and those + 8), two apart
    const u32 k_row = (g >> 1) + 4 * (g & 1), k_at = k_row * 128 + ((q4 ^ k_row) << 4);
    const u32 v_at0 = 2 * q4 * 128 + ((g ^ (2 * q4)) << 4), v_at1 = (2 * q4 + 1) * 128 + ((g ^ (2 * q4 + 1)) << 4);
    const bool odd = q4 & 1;
    const DigitWeights weights = odd ? DigitWeights{1u << 16, 1u << 24, 1u, 1u << 8} : DigitWeights{1u, 1u << 8, 1u << 16, 1u << 24};
    u32 slot_out = 0, phase = 0;
    auto wait_half = [&] { if (!mbar_test(bar0 + 8 * slot_out, phase) && !gave_up) mbar_wait(bar0 + 8 * slot_out, phase, &gave_up); };     // no time for more of them once one ran out
    auto next_slot = [&] { if (++slot_out == NS) { slot_out = 0; phase ^= 1; } };

    // ---- the stretches of items ---------------------------------------------------------------------
    u32 computed = 0;
    __syncthreads();
    if (cw.left != share.walk.left || (cw.left && !lw.nb)) gave_up = 1;       // copies that nobody waits for, or none where they are waited for
    cw = share.walk;
    while (cw.left) {
        const u32 seq = cw.seq, head0 = head0_of(cw), heads = heads_of(cw);
        const u32 first = cw.blk, len = cw.len, nb = cw.nb, count = cw.left < nb - first ? cw.left : nb - first;
        // The right operand of the scores: a thread takes four words' places of one head, whose digits are four lanes' 16 bytes for steps 2j and 2j + 1.
#pragma unroll
        for (int it = 0; it < Q_ITEMS; it++) {
            const u32 i = tid + it * THREADS, head = i / (J * 4), j = i / 4 % J, qq = i & 3;
            if (i >= HEADS * J * 4) break;
            u32 w[4][4];                         // [column c][word]
#pragma unroll
            for (u32 k = 0; k < 4; k++) {
                u32 da[4], db[4];
                if (SMALL) {
                    digit_words(qv[it][2 * k % Q_WORDS], da);
                    digit_words(qv[it][(2 * k + 1) % Q_WORDS], db);
#pragma unroll
                    for (u32 c = 0; c < 4; c++) w[c][k] = __byte_perm(da[c], db[c], 0x5410);
                } else {
                    digit_words(qv[it][k], da);
#pragma unroll
                    for (u32 c = 0; c < 4; c++) w[c][k] = da[c];
                }
            }
#pragma unroll
            for (u32 c = 0; c < 4; c++) qd[(j * NT + head / 2) * 32 + ((head & 1) * 4 + c) * 4 + qq] = make_uint4(w[c][0], w[c][1], w[c][2], w[c][3]);
            if (SMALL) {                         // what flipped top bits add to a score, 2^15 sum q, is taken off its digits 0 and 2 at the start; J * 4 lanes have a head
                u64 sum = 0;
#pragma unroll
                for (u32 k = 0; k < Q_WORDS; k++) sum += qv[it][k];
#pragma unroll
                for (u32 o = J * 2; o > 0; o >>= 1) sum += __shfl_xor_sync(J * 4 == 32 ? 0xffffffffu : ((1u << (J * 4 % 32)) - 1) << (lane & ~(J * 4 - 1)), sum, o);
                if ((lane & (J * 4 - 1)) == 0) off_q[head] = neg31(mul31(red64(sum), 32768u));
            }
        }
        __syncthreads();

        int acc[MT][NT][4];
        u64 esum[NT];
        u32 bad = 0;                            // bit 0: a page, bit 1 + nt: a score of this lane's head
#pragma unroll
        for (int n = 0; n < NT; n++) {
            esum[n] = 0;
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int i = 0; i < 4; i++) acc[m][n][i] = 0;
        }
        bool flushed = false;
        auto flush = [&]() {                    // sums of 32 bits to the warp's sums mod p
            u32* to_part = part + (warp * HEADS + (q4 >> 1)) * DP;
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    int(&c)[4] = acc[m][n];
                    const u32 v = digit_value(c, odd, weights);
                    // rows of the tile are elements (see the left operand below)
                    const u32 e = SMALL ? 8 * (8 * (m >> 2) + g) + 2 * (m & 3) + odd : 4 * (8 * (m >> 1) + g) + 2 * (m & 1) + odd;
                    u32* at = to_part + 2 * n * DP + e;
                    *at = flushed ? add31(*at, v) : v;
                    c[0] = c[1] = c[2] = c[3] = 0;
                }
            flushed = true;
        };
        u32* ed = reinterpret_cast<u32*>(digits + warp * NT * S::ED);
        const u32 round_up = (1u << A.score_shift) >> 1;
        for (u32 b = 0; b < count; b++) {
            const u32 pos0 = (first + b) * BLOCK + warp * 16;
            // keys.  A warp behind the last position goes along with what its slot holds: none of its positions is seen, so all its weights are zero.
            wait_half();
            int sc[NT][4];
            {
                if ((bad_pages >> (loaded - 1 - computed)) & 1) bad |= 1;
                const unsigned char* kt = pa_smem + ring_at + slot_out * S::HALF;
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    sc[n][1] = sc[n][3] = 0;
                    sc[n][0] = sc[n][2] = SMALL ? (int)((off_q[2 * n + (q4 >> 1)] >> (odd ? 16 : 0)) & 0xffffu) : 0;
                }
#pragma unroll
                for (int j = 0; j < J; j++) {
                    const unsigned char* at = kt + (j >> 1) * 2048 + (j & 1 ? k_at ^ 64 : k_at);
                    uint4 a = *reinterpret_cast<const uint4*>(at), c = *reinterpret_cast<const uint4*>(at + 1024);
                    if (SMALL) {
                        a.x ^= 0x80008000u; a.y ^= 0x80008000u; a.z ^= 0x80008000u; a.w ^= 0x80008000u;
                        c.x ^= 0x80008000u; c.y ^= 0x80008000u; c.z ^= 0x80008000u; c.w ^= 0x80008000u;
                    }
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        const uint4 bq = qd[(j * NT + n) * 32 + lane];
                        mma_u8_16x8x32(sc[n], a.x, c.x, a.y, c.y, bq.x, bq.y);
                        mma_u8_16x8x32(sc[n], a.z, c.z, a.w, c.w, bq.z, bq.w);
                    }
                }
            }
            __syncwarp();                        // every lane has read its keys
            load_half(NS & 1);
            next_slot();
            {
                // one score a lane and tile of columns: position k_row (+ 8 for odd lanes), head 2n + (q4 >> 1).  Columns of a head behind the last one are zero and
                // so are their scores; nobody reads what becomes of them.
                const u32 row = k_row + (odd ? 8 : 0);
                const bool seen = pos0 + row < len;
                u32 ev[NT];
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    const u32 s = digit_value(sc[n], odd, weights), minus = ZKB_P - s;
                    const bool neg = minus < s;
                    const u32 m = (umin32(s, minus) + round_up) >> A.score_shift;
                    const u32 index = neg ? 0u - m : m;
                    const bool in = index + A.n_table / 2 < A.n_table;
                    ev[n] = seen && in ? __ldg(A.table + (index & (A.n_table - 1))) : 0u;
                    if (seen && !in) bad |= 2u << n;
                }
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    esum[n] += ev[n];
                    const u32 col = (q4 >> 1) * 4;
                    if (SMALL) {
                        // [NT][8 slots of depth][8 columns], a word for positions p and p + 1: the lane of p writes columns 0 and 1, that of p + 1 columns 2 and 3
                        // (bytes 0 and 1 of digit_words, c = 0, 1 or 2, 3)
                        const u32 other = __shfl_xor_sync(0xffffffffu, ev[n], 8);
                        const bool high = row & 1;
                        const u32 a = high ? other : ev[n], b = high ? ev[n] : other, sel = high ? 0x4312 : 0x0140;
                        const u32 x = __byte_perm(a, (a << (high ? 9 : 0)) >> (high ? 25 : 23), sel), y = __byte_perm(b, (b << (high ? 9 : 0)) >> (high ? 25 : 23), sel);
                        *reinterpret_cast<uint2*>(ed + ((n * 8 + ((row & 7) >> 1) + 4 * (row >> 3)) * 8 + col + (high ? 2 : 0))) =
                            make_uint2(__byte_perm(x, y, 0x5410), __byte_perm(x, y, 0x7632));
                    } else {                     // [NT][16 slots of depth][8 columns]
                        u32 dw[4];
                        digit_words(ev[n], dw);
                        *reinterpret_cast<uint4*>(ed + (n * 16 + (row & 8) + (row & 1) * 4 + ((row & 7) >> 1)) * 8 + col) = make_uint4(dw[0], dw[1], dw[2], dw[3]);
                    }
                }
                __syncwarp();
            }
            // values
            wait_half();
            {
                const unsigned char* vt = pa_smem + ring_at + slot_out * S::HALF;
                constexpr int KS = SMALL ? 1 : 2;
#pragma unroll
                for (int ks = 0; ks < KS; ks++) {
                    u32 b0[NT], b1[NT];
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        const u32* e8 = ed + (SMALL ? n * 64 : (n * 16 + 8 * ks) * 8);
                        b0[n] = e8[q4 * 8 + g];
                        b1[n] = e8[(q4 + 4) * 8 + g];
                    }
#pragma unroll
                    for (int j = 0; j < VJ; j++) {
                        if (SMALL) {
                            u32 v[4][4];
#pragma unroll
                            for (int r = 0; r < 4; r++) {
                                const uint4 t = *reinterpret_cast<const uint4*>(vt + (r & 1 ? v_at1 : v_at0) + (r >> 1) * 1024 + j * 2048);
                                v[r][0] = t.x; v[r][1] = t.y; v[r][2] = t.z; v[r][3] = t.w;
                            }
#pragma unroll
                            for (int i = 0; i < 4; i++) {
                                const u32 a0 = __byte_perm(v[0][i], v[1][i], 0x5410) ^ 0x80008000u, a1 = __byte_perm(v[0][i], v[1][i], 0x7632) ^ 0x80008000u;
                                const u32 a2 = __byte_perm(v[2][i], v[3][i], 0x5410) ^ 0x80008000u, a3 = __byte_perm(v[2][i], v[3][i], 0x7632) ^ 0x80008000u;
#pragma unroll
                                for (int n = 0; n < NT; n++) mma_u8_16x8x32(acc[4 * j + i][n], a0, a1, a2, a3, b0[n], b1[n]);
                            }
                        } else {
                            const uint4 v = *reinterpret_cast<const uint4*>(vt + v_at0 + ks * 1024 + j * 2048), u = *reinterpret_cast<const uint4*>(vt + v_at1 + ks * 1024 + j * 2048);
#pragma unroll
                            for (int n = 0; n < NT; n++) {
                                mma_u8_16x8x32(acc[2 * j][n], v.x, v.y, u.x, u.y, b0[n], b1[n]);
                                mma_u8_16x8x32(acc[2 * j + 1][n], v.z, v.w, u.z, u.w, b0[n], b1[n]);
                            }
                        }
                    }
                }
            }
            __syncwarp();                        // every lane has read its values and the digits
            load_half((NS + 1) & 1);
            next_slot();
            computed++;
            if ((b + 1) % PA_FLUSH == 0) flush();
        }
#pragma unroll
        for (int n = 0; n < NT; n++) {
            u32 s = red64(esum[n]);
            u32 f = (bad & 1 ? PA_BAD_PAGE : 0u) | (bad & (2u << n) ? PA_BAD_SCORE : 0u);
#pragma unroll
            for (int o = 1; o < 32; o = o == 1 ? 4 : o * 2) {                       // all lanes but the other head's
                s = add31(s, __shfl_xor_sync(0xffffffffu, s, o));
                f |= __shfl_xor_sync(0xffffffffu, f, o);
            }
            if (g == 0 && !odd) { es_part[warp][2 * n + (q4 >> 1)] = s; flag_part[warp][2 * n + (q4 >> 1)] = f; }
        }
        __syncthreads();
        const bool begins = first == 0, ends = first + count == nb;
        u32* slot = P.slots + (size_t)(2 * blockIdx.x + (begins ? 1 : 0)) * HEADS * (DP + 4);
        if (tid < heads) {                      // while the other warps store their sums
            u32 s = 0, f = 0;
#pragma unroll
            for (int w = 0; w < WARPS; w++) { s = add31(s, es_part[w][tid]); f |= flag_part[w][tid]; }
            if (begins && ends) {
                const int code = f & PA_BAD_PAGE ? SERVE_PAGE : f & PA_BAD_SCORE ? SERVE_SCORE : s == 0 ? SERVE_ZERO_SUM : 0;
                if (code) atomicMax(A.status + seq, code);
                inv[tid] = code ? 0u : inv31_chain(s);
                corr[tid] = SMALL ? mul31(s, 32768u) : 0u;
            } else {
                slot[tid * (DP + 4) + DP] = s;
                slot[tid * (DP + 4) + DP + 1] = f;
            }
        }
        __syncwarp();
        flush();
        __syncthreads();
        for (u32 i = tid; i < heads * DP; i += THREADS) {
            u64 sum = 0;
#pragma unroll
            for (int w = 0; w < WARPS; w++) sum += part[w * HEADS * DP + i];
            const u32 h = i / DP, e = i % DP;
            if (!(begins && ends)) slot[h * (DP + 4) + e] = red64(sum);
            else if (e < d) pa_finish(A, seq, head0 + h, e, red64(sum), inv[h], corr[h]);
        }
        if (!(begins && ends)) {
            // The CTA that brings a row's last part adds the parts up.  They lie in the slot of the CTA in which the row begins and those of the next ones.
            const PaParts parts = pa_parts(share.aligned, share.per, P.ctas, blockIdx.x, share.to - cw.left, first, nb);
            const u32 c0 = parts.first_cta, n = parts.n;
            __threadfence();
            __syncthreads();
            if (tid == 0) {
                const bool all = atomicAdd(P.arrived + c0, 1u) == n - 1;
                last_part = all;
                if (all) atomicSub(P.arrived + c0, n);
                atomicAdd(P.begun, pa_brought(1, all ? n : 0));
            }
            __syncthreads();
            if (last_part) {
                __threadfence();
                auto slot_of = [&](u32 k) { return P.slots + (size_t)(2 * (c0 + k) + (k ? 0 : 1)) * HEADS * (DP + 4); };
                constexpr int PER = (HEADS * DP + THREADS - 1) / THREADS;
                u64 sum[PER];                    // the elements' loads are under way while the weights are added up and inverted
#pragma unroll
                for (int v = 0; v < PER; v++) sum[v] = 0;
#pragma unroll 2
                for (u32 k = 0; k < n; k++) {
                    const u32* from_slot = slot_of(k);
#pragma unroll
                    for (int v = 0; v < PER; v++) {
                        const u32 i = tid + v * THREADS;
                        if (i < heads * DP) sum[v] += __ldcg(from_slot + i / DP * (DP + 4) + i % DP);
                    }
                }
                for (u32 h = warp; h < heads; h += WARPS) {
                    u64 s = 0;
                    u32 f = 0;
                    for (u32 k = lane; k < n; k += 32) {
                        const u32* from_slot = slot_of(k) + h * (DP + 4) + DP;
                        s += __ldcg(from_slot);
                        f |= __ldcg(from_slot + 1);
                    }
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
                    f = __reduce_or_sync(0xffffffffu, f);
                    if (lane == 0) {
                        const u32 all = red64(s);
                        const int code = f & PA_BAD_PAGE ? SERVE_PAGE : f & PA_BAD_SCORE ? SERVE_SCORE : all == 0 ? SERVE_ZERO_SUM : 0;
                        if (code) atomicMax(A.status + seq, code);
                        inv[h] = code ? 0u : inv31_chain(all);
                        corr[h] = SMALL ? mul31(all, 32768u) : 0u;
                    }
                }
                __syncthreads();
#pragma unroll
                for (int v = 0; v < PER; v++) {
                    const u32 i = tid + v * THREADS, h = i / DP, e = i % DP;
                    if (i < heads * DP && e < d) pa_finish(A, seq, head0 + h, e, red64(sum[v]), inv[h], corr[h]);
                }
            }
        }
        if (cw.step(count, P.slices, A.c.num_kv_heads)) {
            if (few) {
                cw.next_seq(A.num_seqs, (u64)A.max_blocks << A.c.page_bits, BLOCK, [&](u32 s) { return few_lens[s]; });
            } else {                            // by one thread for all
                if (tid == 0) {
                    cw.next_seq(A.num_seqs, (u64)A.max_blocks << A.c.page_bits, BLOCK, [&](u32 s) { return A.lens[s]; });
                    share.walk = cw;
                }
                __syncthreads();
                cw = share.walk;
            }
            if (!cw.left) gave_up = 1;          // blocks are missing
        }
        if (cw.left) {
            fetch_q(cw.seq, head0_of(cw), heads_of(cw));
            __syncthreads();                    // all are done with this row's arrays
        }
    }
    if (gave_up) {                              // nothing of this warp may still be in flight when it ends
        const u32 halves = pa_halves(loaded, slot_in, NS);
        for (u32 h = 0; h < NS; h++) {
            const u32 last = halves - 1 - h, use = last / NS;
            if (h < halves)
                for (u32 n = 0; n < (1u << 16) && !mbar_try(bar0 + 8 * (last % NS), use & 1); n++) {}
        }
        if (lane == 0) *P.gave_up = 1;
    }
}

// ---- launch ---------------------------------------------------------------------------------------------
struct PaChoice { u32 dp, nt, slices, slice_heads; };
// 2 nt query heads of a key head share a pass over it: as many as the sums fit into registers with (dp / 16 x nt x 4 of them a lane).
inline PaChoice pa_choice(u32 d, u32 hpg) {
    PaChoice c{};
    c.dp = d <= 64 ? 64 : (d <= 128 ? 128 : 256);
    const u32 most = c.dp == 256 ? 4 : 8;
    c.slices = (hpg + most - 1) / most;
    c.slice_heads = (hpg + c.slices - 1) / c.slices;
    c.nt = c.dp == 256 ? (c.slice_heads <= 2 ? 1 : 2) : (c.slice_heads + 1) / 2;
    return c;
}
template <int DP, bool SMALL, int NT>
inline cudaError_t pa_launch(cudaStream_t stream, const CUtensorMap (&maps)[2], const PagedAttnArgs& a, PaWork w, int* launches) {
    using S = PaShape<DP, SMALL, NT>;
    constexpr size_t smem = (size_t)S::WARPS * S::NS * S::HALF + (size_t)S::RB / 64 * NT * 512 + (size_t)S::WARPS * 2 * NT * DP * 4 + (size_t)S::WARPS * NT * S::ED + 1024;
    static_assert(smem <= 226 * 1024, "with the kernel's own arrays below the 227 KB of a CTA");
    cudaError_t e = allow_smem(paged_attention_kernel<DP, SMALL, NT>, smem);
    if (e != cudaSuccess) return e;
    const u64 most = (u64)a.num_seqs * a.c.num_kv_heads * w.slices * ((((u64)a.max_blocks << a.c.page_bits) + S::WARPS * 16 - 1) / (S::WARPS * 16));
    if (most < w.ctas) w.ctas = (u32)most;
    paged_attention_kernel<DP, SMALL, NT><<<w.ctas, S::WARPS * 32, smem, stream>>>(maps[0], maps[1], a, w);
    ++*launches;
    return cudaGetLastError();
}

}  // namespace zkb
