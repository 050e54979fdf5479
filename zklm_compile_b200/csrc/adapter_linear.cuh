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
constexpr u32 LIN_TEAM = 4, LIN_FILL = 3 * LIN_TEAM;   // warps that fill operands by plain stores: teams that take a step each
constexpr u32 LIN_THREADS = (6 + LIN_FILL) * 32;
constexpr u32 LIN_CHUNK = 2048;                // tokens of one pass

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
    u32 tokens, m, n, a_rows, tt, ntiles, mtiles, wtiles, steps, segs, per, ctas, stages, stage_bytes, tmem_cols, total;   // tiles: wtiles of W, then those of the adapters' A
    size_t slot_words;
};
inline LinPlan lin_plan(int sm_count, u32 tokens, u32 m, u32 n, u32 a_rows) {
    LinPlan p{};
    p.tokens = tokens; p.m = m; p.n = n; p.a_rows = a_rows;
    p.ntiles = (tokens + LIN_TOKENS - 1) / LIN_TOKENS;
    p.tt = ((tokens + p.ntiles - 1) / p.ntiles + 3) / 4 * 4;
    p.wtiles = (m + LIN_ROWS - 1) / LIN_ROWS;
    p.mtiles = p.wtiles + (a_rows + LIN_ROWS - 1) / LIN_ROWS;
    p.steps = (n + LIN_STEP - 1) / LIN_STEP;
    p.segs = (p.steps + LIN_SEG - 1) / LIN_SEG;
    p.total = p.mtiles * p.ntiles * p.steps;                  // below 2^32: lin_fits
    p.per = (p.total + sm_count - 1) / sm_count;
    p.ctas = (p.total + p.per - 1) / p.per;
    p.stage_bytes = LIN_ROWS * 128 + (4 * p.tt * 128 + 1023) / 1024 * 1024;
    p.stages = 200 * 1024 / p.stage_bytes < LIN_MAX_STAGES ? 200 * 1024 / p.stage_bytes : LIN_MAX_STAGES;     // 3 at least, as many as teams of warps that fill
    p.tmem_cols = 32;
    while (p.tmem_cols < 8 * p.tt) p.tmem_cols *= 2;
    p.slot_words = (size_t)p.tt * LIN_ROWS;
    return p;
}
// Whether the steps of one pass can be counted in 31 bits (2^40 products of W's elements and tokens would not).
inline bool lin_fits(u32 tokens, u32 m, u32 n, u32 a_rows) {
    return ((u64)((m + LIN_ROWS - 1) / LIN_ROWS) + (a_rows + LIN_ROWS - 1) / LIN_ROWS) * ((tokens + LIN_TOKENS - 1) / LIN_TOKENS) * ((n + LIN_STEP - 1) / LIN_STEP) < (1ull << 31);
}
// Rows of A that the product takes along with W's (all adapters for all tokens), or 0: then each token's own rank products are made apart.
// Along, an adapter's rows are read once however many tokens use it and no launch is added; apart, no adapter that no token has is read.  2560 x 2560 and twelve adapters of
// 16 for 1 / 64 / 1024 tokens: along 10.0 / 25 / 96 us, apart 10.3 / 25 / 112; 256 adapters: 16.7 / 35 / 212 and 12.3 / 29 / 140 (where the rule's second clause, which counts
// bytes, takes the slower side at 1024).
inline u32 lin_a_rows(u32 tokens, u32 m, u32 num_adapters, u32 rank) {
    const u64 rows = (u64)num_adapters * rank, tiles = (rows + LIN_ROWS - 1) / LIN_ROWS, wtiles = (m + LIN_ROWS - 1) / LIN_ROWS;
    return rows && (tiles <= (wtiles < 8 ? 1 : wtiles / 8) || tiles * LIN_ROWS <= (u64)tokens * rank / 2) && rows < (1u << 30) ? (u32)rows : 0u;
}
inline u32 lin_chunk(u32 tokens) { return tokens < LIN_CHUNK ? tokens : LIN_CHUNK; }
// For any number of tokens up to the plan's: fewer of them may be shared by more CTAs.
inline size_t lin_slot_bytes(int sm_count, const LinPlan& p) { return ((size_t)sm_count + (size_t)p.mtiles * p.ntiles * p.segs) * p.slot_words * 4; }

struct LinWalk {                               // a CTA's stretches, the same for every role
    const LinPlan& p;
    u32 at, end;
    __device__ LinWalk(const LinPlan& plan) : p(plan), at(blockIdx.x * plan.per), end(plan.total - at > plan.per ? at + plan.per : plan.total) {}
    u32 mt, nt, first, count, slot;
    __device__ bool next() {
        if (at >= end) return false;
        const u32 tile = at / p.steps;
        first = at - tile * p.steps;
        const u32 seg = first / LIN_SEG, seg_end = (seg + 1) * LIN_SEG < p.steps ? (seg + 1) * LIN_SEG : p.steps;
        count = end - at < seg_end - first ? end - at : seg_end - first;
        mt = tile / p.ntiles;
        nt = tile - mt * p.ntiles;
        slot = blockIdx.x + tile * p.segs + seg;
        at += count;
        return true;
    }
};

// Warp 0 copies W, warp 1 issues, warps 2 to 5 empty the accumulators, the others make the tokens' operand from x: 16 bytes of it a value, which would
// be four times x to copy, and a kernel of its own to make (332 against 260 us for 1024 x 4096 x 4096).  W_COPY: W by tensor copies; otherwise (rows that start on no
// 16-byte boundary) word by word, by the warps that fill.
template <bool W_COPY>
__global__ void __launch_bounds__(LIN_THREADS) linear_bytes_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_a, LinPlan p, LinearArgs A, int x_vec,
                                                                   u32* __restrict__ slots) {
    extern __shared__ __align__(16) unsigned char lin_raw[];
    __shared__ __align__(8) u64 bars[2 * LIN_MAX_STAGES + 2];
    __shared__ u32 tmem_base;
    __shared__ volatile int gave_up;
    const u32 warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    unsigned char* const smem = lin_raw + ((0u - smem_addr(lin_raw)) & 1023u);         // the swizzle goes by addresses
    const u32 base = smem_addr(smem);
    const u32 full = smem_addr(bars), empty = full + 8 * LIN_MAX_STAGES, acc_full = empty + 8 * LIN_MAX_STAGES, acc_empty = acc_full + 8;
    if (threadIdx.x == 0) {
        for (u32 s = 0; s < p.stages; s++) { mbar_init(full + 8 * s, 1 + LIN_TEAM); mbar_init(empty + 8 * s, 1); }
        mbar_init(acc_full, 1);
        mbar_init(acc_empty, 4);
        gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) tmem_alloc(smem_addr(&tmem_base), p.tmem_cols);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_launch_dependents();
    const u32 tmem = tmem_base;
    LinWalk walk(p);
    if (warp == 0) {
        u32 it = 0;
        bool ok = true;
        while (ok && walk.next()) {
            const bool of_w = walk.mt < p.wtiles;
            const CUtensorMap* map = of_w ? &map_w : &map_a;
            const int row = (int)((of_w ? walk.mt : walk.mt - p.wtiles) * LIN_ROWS);
            for (u32 k = 0; k < walk.count; k++, it++) {
                const u32 s = it % p.stages, round = it / p.stages, st = base + s * p.stage_bytes;
                if (round && !(ok = mbar_wait(empty + 8 * s, (round - 1) & 1, &gave_up))) break;
                mbar_expect_one(full + 8 * s, W_COPY ? LIN_ROWS * 128 : 0u);
                if (W_COPY) tensor_load_2d_one(st, map, (int)((walk.first + k) * LIN_STEP), row, full + 8 * s);
            }
        }
        // The kernel before this one (where it is one of the same call) makes what the join reads: the join, which waits for this kernel, must find it done.
        pdl_wait();
        if (!ok)                                 // given up: nothing of this CTA may still be in flight when it ends
            for (u32 i = it > p.stages ? it - p.stages : 0; i < it; i++)
                for (u32 n = 0; n < (1u << 16) && !mbar_try(full + 8 * (i % p.stages), (i / p.stages) & 1); n++) {}
    } else if (warp == 1) {
        const u32 idesc = i8_instr_desc(4 * p.tt);
        u32 it = 0, n = 0;
        bool ok = true;
        while (ok && walk.next()) {
            if (n && !(ok = mbar_wait(acc_empty, (n - 1) & 1, &gave_up))) { mma_commit_one(acc_full); n++; break; }
            tc_fence_after();
            const bool two = walk.mt < p.wtiles ? walk.mt * LIN_ROWS + 128 < p.m : (walk.mt - p.wtiles) * LIN_ROWS + 128 < p.a_rows;
            for (u32 k = 0; k < walk.count; k++, it++) {
                const u32 s = it % p.stages, st = base + s * p.stage_bytes;
                if (!(ok = mbar_wait(full + 8 * s, (it / p.stages) & 1, &gave_up))) break;
                tc_fence_after();
                const u64 a = smem_desc_sw128(st), b = smem_desc_sw128(st + LIN_ROWS * 128);
#pragma unroll
                for (u32 kk = 0; kk < 4; kk++) mma_u8_one(tmem, a + 2 * kk, b + 2 * kk, idesc, k || kk);
                if (two) {
#pragma unroll
                    for (u32 kk = 0; kk < 4; kk++) mma_u8_one(tmem + 4 * p.tt, a + (16384 >> 4) + 2 * kk, b + 2 * kk, idesc, k || kk);
                }
                mma_commit_one(empty + 8 * s);
            }
            mma_commit_one(acc_full);
            n++;
        }
        if (!ok)
            for (u32 i = 0; i < (1u << 16) && !mbar_try(acc_full, (n - 1) & 1); i++) {}
    } else if (warp < 6) {
        const u32 quarter = warp & 3;            // the lanes of TMEM that this warp may read
        u32 n = 0;
        while (walk.next()) {
            if (!mbar_wait(acc_full, n & 1, &gave_up)) break;
            tc_fence_after();
            u32* slot = slots + (size_t)walk.slot * p.slot_words;
            const u32 rows = walk.mt < p.wtiles ? p.m - walk.mt * LIN_ROWS : p.a_rows - (walk.mt - p.wtiles) * LIN_ROWS;
            for (u32 half = 0; half < 2; half++) {
                const u32 row = half * 128 + quarter * 32 + lane;
                if (half * 128 >= rows) break;
                const u32 from = tmem + (quarter << 21) + half * 4 * p.tt;
                for (u32 t0 = 0; t0 < p.tt; t0 += 16) {
                    u32 v[4][16];
#pragma unroll
                    for (u32 g = 0; g < 4; g++)
                        if (t0 + 4 * g < p.tt) tmem_load16(from + 4 * t0 + 16 * g, v[g]);
                    tmem_wait_load();
                    u32* to = slot + (size_t)t0 * LIN_ROWS + row;
#pragma unroll
                    for (u32 g = 0; g < 4; g++)
                        if (t0 + 4 * g < p.tt) {
#pragma unroll
                            for (u32 e = 0; e < 4; e++) {
                                // digits below 2^31: the value is below 2^56, and its two parts add up to less than 2^32, which will do for a term of a sum
                                const u64 x = v[g][4 * e] + (u64)v[g][4 * e + 1] * (1u << 8) + (u64)v[g][4 * e + 2] * (1u << 16) + (u64)v[g][4 * e + 3] * (1u << 24);
                                to[(4 * g + e) * LIN_ROWS] = ((u32)x & ZKB_P) + (u32)(x >> 31);
                            }
                        }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(acc_empty);
            n++;
        }
    } else {
        // Each team of warps takes every third step, so that three steps' loads are under way.  There are at least as many stages as teams: a team knows that
        // the stage of its last step was empty, and from that that its next one's was emptied the time before last; with fewer stages than teams it could
        // be two phases ahead, where a wait by parity sees the wrong one.  (1024 x 4096 x 4096 with teams of two 253 us, of four 248.)
        constexpr u32 teams = LIN_FILL / LIN_TEAM;
        const u32 team = (warp - 6) / LIN_TEAM, member = (warp - 6) % LIN_TEAM;
        constexpr u32 GROUPS = LIN_TOKENS / (4 * LIN_TEAM);
        // A warp's groups of four values of x, fetched a turn ahead: token 4 (4 i + member) + lane / 8 of the tile, columns 4 (lane & 7) .. of its next step.
        u32 x[GROUPS][4];
        u32 ahead = blockIdx.x * p.per + team;
        auto fetch = [&] {
            if (ahead >= walk.end) return;
            const u32 tile = ahead / p.steps, j = (ahead - tile * p.steps) * LIN_STEP + 4 * (lane & 7), tok0 = tile % p.ntiles * p.tt;
#pragma unroll
            for (u32 i = 0; i < GROUPS; i++) {
                const u32 in = 4 * (LIN_TEAM * i + member) + (lane >> 3), t = tok0 + in;
                const bool there = in < p.tt && t < p.tokens;
                const u32* at = A.x + t * A.x_stride + j;
                if (x_vec) {                     // n is a multiple of 4 then
                    const uint4 v = there && j < p.n ? *reinterpret_cast<const uint4*>(at) : make_uint4(0, 0, 0, 0);
                    x[i][0] = v.x; x[i][1] = v.y; x[i][2] = v.z; x[i][3] = v.w;
                } else {
#pragma unroll
                    for (u32 e = 0; e < 4; e++) x[i][e] = there && j + e < p.n ? at[e] : 0u;
                }
            }
        };
        fetch();
        u32 it = 0;
        bool ok = true;
        while (ok && walk.next()) {
            const bool of_w = walk.mt < p.wtiles;
            const u32 row0 = (of_w ? walk.mt : walk.mt - p.wtiles) * LIN_ROWS, rows = (of_w ? p.m : p.a_rows) - row0, most = rows < LIN_ROWS ? rows : LIN_ROWS;
            for (u32 k = 0; k < walk.count; k++, it++) {
                if (it % teams != team) continue;
                const u32 s = it % p.stages, round = it / p.stages, step = walk.first + k;
                unsigned char* st = smem + s * p.stage_bytes;
                if (round && !(ok = mbar_wait(empty + 8 * s, (round - 1) & 1, &gave_up))) break;
                if (!W_COPY) {
                    const u32 j = step * LIN_STEP + lane, bytes = j < p.n ? 4 : 0;      // past the end of a row nothing is read and zero is stored
                    const u32* src = bytes ? (of_w ? A.w : A.a) + (size_t)(row0 + member) * p.n + j : A.w;
                    const size_t next = bytes ? LIN_TEAM * (size_t)p.n : 0;
                    const u32 to = smem_addr(st) + (lane & 3) * 4;
#pragma unroll 8
                    for (u32 r = member; r < most; r += LIN_TEAM, src += next)
                        asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to + r * 128 + (((lane >> 2) ^ (r & 7)) << 4)), "l"(src), "r"(bytes) : "memory");
                }
#pragma unroll
                for (u32 i = 0; i < GROUPS; i++) {
                    const u32 t = 4 * (LIN_TEAM * i + member) + (lane >> 3), q = lane & 7;
                    if (4 * (LIN_TEAM * i + member) >= p.tt) break;
                    u32 w[4][4];
#pragma unroll
                    for (u32 e = 0; e < 4; e++) {
                        u32 d[4];
                        digit_words(x[i][e], d);
#pragma unroll
                        for (int c = 0; c < 4; c++) w[c][e] = d[c];
                    }
#pragma unroll
                    for (u32 c = 0; c < 4; c++) {
                        const u32 r = 4 * t + c;
                        *reinterpret_cast<uint4*>(st + LIN_ROWS * 128 + r * 128 + ((q ^ (r & 7)) << 4)) = make_uint4(w[c][0], w[c][1], w[c][2], w[c][3]);
                    }
                }
                ahead += teams;
                fetch();
                if (!W_COPY) asm volatile("cp.async.wait_all;" ::: "memory");
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(full + 8 * s);
            }
        }
        if (!W_COPY) asm volatile("cp.async.wait_all;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 1) tmem_free(tmem, p.tmem_cols);
    if (threadIdx.x == 0 && gave_up) *A.gave_up = 1;
}

// The slots that hold a tile (see LinPlan): segment seg's are c + tile * segs + seg for c from lin_first to lin_last.
__device__ __forceinline__ u32 lin_first(const LinPlan& p, u32 tile, u32 seg) { return (tile * p.steps + seg * LIN_SEG) / p.per; }
__device__ __forceinline__ u32 lin_last(const LinPlan& p, u32 tile, u32 seg) {
    return (tile * p.steps + ((seg + 1) * LIN_SEG < p.steps ? (seg + 1) * LIN_SEG : p.steps) - 1) / p.per;
}
// Adds the slots' sums of rows row .. row + 3 of tile mt (one tile's; `vec`: row is a multiple of 4) for a token of tile nt.  The slots are written while the join
// is already there: they are no read-only memory to the compiler, and read from L2.
__device__ __forceinline__ void lin_sum4(const LinPlan& p, const u32* slots, u32 mt, u32 nt, u32 in_tile, u32 row, bool vec, u64 (&v)[4]) {
    const u32 tile = mt * p.ntiles + nt;
    const u32* at = slots + (size_t)in_tile * LIN_ROWS + row;
    for (u32 seg = 0; seg < p.segs; seg++) {
        const u32 from = lin_first(p, tile, seg), to = lin_last(p, tile, seg);
        const u32* s = at + ((size_t)from + (size_t)tile * p.segs + seg) * p.slot_words;
        if (vec) {
#pragma unroll 4
            for (u32 c = from; c <= to; c++, s += p.slot_words) {
                const uint4 x = __ldcg(reinterpret_cast<const uint4*>(s));
                v[0] += x.x; v[1] += x.y; v[2] += x.z; v[3] += x.w;
            }
        } else {
#pragma unroll 4
            for (u32 c = from; c <= to; c++, s += p.slot_words) { v[0] += __ldcg(s); v[1] += __ldcg(s + 1); v[2] += __ldcg(s + 2); v[3] += __ldcg(s + 3); }
        }
    }
}
// Four products of field elements fit 64 bits.
__device__ __forceinline__ u64 lin_dot4(const u32* a, const u32* b) {
    const u64 s = (u64)a[0] * b[0] + (u64)a[1] * b[1] + (u64)a[2] * b[2] + (u64)a[3] * b[3];
    return (s & ZKB_P) + (s >> 31);
}
// One CTA: `blocks` times 64 rows, up to 16 tokens of a tile of tokens.  B (A x) is a product of bytes too, on the warps' tensor cores: the rows of B are the left operand as
// they lie in memory, read once for all tokens beside each other that have the same adapter (a run); each token's A x has four columns in the
// right one, zero for the adapters of other tokens; tokens of one adapter apart from each other are two runs, which read B twice (48 tokens of 9728 rows and twelve
// adapters: 45 us in any order, 36 sorted by adapter, the whole call).  What bounds it is latency, slots first: 45 us for 1024 tokens of rank 32 and 4096 rows, 21 without adapters.
constexpr u32 LIN_JOIN_ROWS = 64, LIN_JOIN_TOKENS = 16, LIN_JOIN_RANK = 64;
__global__ void __launch_bounds__(256, 3) linear_join_kernel(LinearArgs A, LinPlan p, u32 blocks, int b_vec, int y_vec, const u32* slots, const u32* u_own) {
    __shared__ uint4 ud[LIN_JOIN_RANK / 16][LIN_JOIN_TOKENS / 2][32];              // digits of A x, 64 of the rank at a time
    __shared__ __align__(16) u32 lora[LIN_JOIN_TOKENS][LIN_JOIN_ROWS + 4];
    __shared__ int of[LIN_JOIN_TOKENS], run_of[LIN_JOIN_TOKENS], run_adapter[LIN_JOIN_TOKENS], runs;
    const u32 groups = (p.tt + LIN_JOIN_TOKENS - 1) / LIN_JOIN_TOKENS, nt = blockIdx.y / groups, in_tile = (blockIdx.y - nt * groups) * LIN_JOIN_TOKENS, t0 = nt * p.tt + in_tile;
    const u32 tile_end = (nt + 1) * p.tt < p.tokens ? (nt + 1) * p.tt : p.tokens;
    if (t0 >= tile_end) return;
    const u32 count = tile_end - t0 < LIN_JOIN_TOKENS ? tile_end - t0 : LIN_JOIN_TOKENS;
    const u32 tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, quad = 4 * (tid & 15), mine = tid >> 4, begin = blockIdx.x * blocks * LIN_JOIN_ROWS, rank = A.rank;
    const u32 stop = A.m - begin < blocks * LIN_JOIN_ROWS ? A.m : begin + blocks * LIN_JOIN_ROWS;
    // what does not come from the product: before waiting for it
    int n_runs = 0;
    if (rank) {
        if (warp == 0) {                       // runs of tokens with the same adapter; lanes 0 .. 15 are the tokens
            const int a = lane < count ? A.adapter_of[t0 + lane] : -1;
            const int mine_of = a >= 0 && (u32)a < A.num_adapters ? a : -1, before = __shfl_up_sync(0xffffffffu, mine_of, 1);
            const bool begins = mine_of >= 0 && (lane == 0 || before != mine_of);
            const u32 all = __ballot_sync(0xffffffffu, begins), run = __popc(all & (0xffffffffu >> (31 - lane))) - 1;
            if (lane < LIN_JOIN_TOKENS) { of[lane] = mine_of; run_of[lane] = mine_of >= 0 ? (int)run : -1; }
            if (begins) run_adapter[run] = mine_of;
            if (lane == 0) runs = __popc(all);
        }
        __syncthreads();
        n_runs = runs;
        const u32 lines = ((stop - begin) * rank + 31) / 32;
        for (int r = 0; r < n_runs; r++)
            for (u32 k = tid; k < lines; k += 256) prefetch_l2(A.b + ((size_t)run_adapter[r] * A.m + begin) * rank + 32 * (size_t)k);
    }
    // A x from column rb of the rank on, four of it a thread, and its digits
    auto make_digits = [&](u32 rb) {
        const u32 t = tid >> 4, at = tid & 15, r0 = rb + 4 * at;
        u64 v[4] = {0, 0, 0, 0};
        if (t < count && of[t] >= 0 && r0 < rank) {
            const u32 a_row = (u32)of[t] * rank + r0, in = a_row % LIN_ROWS;       // what lies behind the adapter's last row is not used
            if (!p.a_rows) {
#pragma unroll
                for (u32 k = 0; k < 4; k++) v[k] = r0 + k < rank ? __ldcg(u_own + (size_t)(t0 + t) * rank + r0 + k) : 0u;
            } else if (in + 4 <= LIN_ROWS) {
                lin_sum4(p, slots, p.wtiles + a_row / LIN_ROWS, nt, in_tile + t, in, rank % 4 == 0, v);
            } else {                             // the four lie in two tiles: each with the last four rows of its own
                for (u32 k = 0; k < 4 && r0 + k < rank; k++) {
                    u64 x[4] = {0, 0, 0, 0};
                    const u32 r = (a_row + k) % LIN_ROWS, back = r < 4 ? r : 3;
                    lin_sum4(p, slots, p.wtiles + (a_row + k) / LIN_ROWS, nt, in_tile + t, r - back, false, x);
                    v[k] = back == 0 ? x[0] : back == 1 ? x[1] : back == 2 ? x[2] : x[3];
                }
            }
        }
        u32 w[4][4];
#pragma unroll
        for (u32 k = 0; k < 4; k++) {
            u32 d[4];
            digit_words(r0 + k < rank ? red64(v[k]) : 0u, d);
#pragma unroll
            for (u32 c = 0; c < 4; c++) w[c][k] = d[c];
        }
#pragma unroll
        for (u32 c = 0; c < 4; c++) ud[at >> 2][t >> 1][((t & 1) * 4 + c) * 4 + (at & 3)] = make_uint4(w[c][0], w[c][1], w[c][2], w[c][3]);
    };
    const u32 g = lane >> 2, q4 = lane & 3, nt0 = (warp >> 2) * 4;
    const bool odd = q4 & 1;
    const DigitWeights weights = odd ? DigitWeights{1u << 16, 1u << 24, 1u, 1u << 8} : DigitWeights{1u, 1u << 8, 1u << 16, 1u << 24};
    int run_n[4];                              // the run of this lane's column in each of the warp's tiles of columns
#pragma unroll
    for (u32 n = 0; n < 4; n++) run_n[n] = n_runs ? run_of[2 * (nt0 + n) + (lane >> 4)] : -1;
    // Rows row_a and row_a + 8 of B, columns 4 q4 .. + 3 of 16, for step x of a pass over the rank: its adapters' 16 columns one behind the other
    auto load_b = [&](u32 rb, u32 x, u32 row_a, u32 (&fa)[4], u32 (&fc)[4]) {
        const u32 chunk = x / n_runs, r = rb + 16 * chunk + 4 * q4;
        const u32* from = A.b + ((size_t)run_adapter[x - chunk * n_runs] * A.m + row_a) * rank + r;
        const u32* from8 = from + 8 * (size_t)rank;
        if (b_vec) {
            const uint4 va = r < rank && row_a < A.m ? *reinterpret_cast<const uint4*>(from) : make_uint4(0, 0, 0, 0);
            const uint4 vc = r < rank && row_a + 8 < A.m ? *reinterpret_cast<const uint4*>(from8) : make_uint4(0, 0, 0, 0);
            fa[0] = va.x; fa[1] = va.y; fa[2] = va.z; fa[3] = va.w;
            fc[0] = vc.x; fc[1] = vc.y; fc[2] = vc.z; fc[3] = vc.w;
        } else {
#pragma unroll
            for (u32 e = 0; e < 4; e++) {
                fa[e] = r + e < rank && row_a < A.m ? from[e] : 0u;
                fc[e] = r + e < rank && row_a + 8 < A.m ? from8[e] : 0u;
            }
        }
    };
    auto multiply = [&](u32 x, const u32 (&fa)[4], const u32 (&fc)[4], int (&acc)[4][4]) {
        const u32 chunk = x / n_runs;
        const int run = (int)(x - chunk * n_runs);
#pragma unroll
        for (u32 n = 0; n < 4; n++) {
            if (!__any_sync(0xffffffffu, run_n[n] == run)) continue;
            const uint4 b = run_n[n] == run ? ud[chunk][nt0 + n][lane] : make_uint4(0, 0, 0, 0);
            mma_u8_16x8x32(acc[n], fa[0], fc[0], fa[1], fc[1], b.x, b.y);
            mma_u8_16x8x32(acc[n], fa[2], fc[2], fa[3], fc[3], b.z, b.w);
        }
    };
    pdl_wait();
    if (n_runs) make_digits(0);
    // a thread has one token and four rows of a block
    const bool has = mine < count;
    for (u32 i0 = begin; i0 < stop; i0 += LIN_JOIN_ROWS) {
        const u32 i = i0 + quad, row_a = i0 + (warp & 3) * 16 + g;
        u64 y[4];
#pragma unroll
        for (u32 e = 0; e < 4; e++) y[e] = A.bias && i + e < A.m ? A.bias[i + e] : 0u;
        // rows of the tile that are behind the last one hold nothing of use, but are there
        if (has && i < A.m) lin_sum4(p, slots, i / LIN_ROWS, nt, in_tile + mine, i % LIN_ROWS, true, y);
        if (n_runs) {
            int acc[4][4] = {};
            for (u32 rb = 0; rb < rank; rb += LIN_JOIN_RANK) {
                const u32 steps = ((rank - rb < LIN_JOIN_RANK ? rank - rb : LIN_JOIN_RANK) + 15) / 16 * (u32)n_runs;
                if (rb || (rank > LIN_JOIN_RANK && i0 > begin)) {
                    __syncthreads();
                    make_digits(rb);
                }
                __syncthreads();
                for (u32 x = 0; x < steps; x += 2) {
                    u32 f[2][2][4];
                    load_b(rb, x, row_a, f[0][0], f[0][1]);
                    if (x + 1 < steps) load_b(rb, x + 1, row_a, f[1][0], f[1][1]);
                    multiply(x, f[0][0], f[0][1], acc);
                    if (x + 1 < steps) multiply(x + 1, f[1][0], f[1][1], acc);
                }
            }
#pragma unroll
            for (u32 n = 0; n < 4; n++) lora[2 * (nt0 + n) + (q4 >> 1)][(warp & 3) * 16 + g + (odd ? 8 : 0)] = digit_value(acc[n], odd, weights);
            __syncthreads();
            const uint4 v = *reinterpret_cast<const uint4*>(&lora[mine][quad]);
            y[0] += v.x; y[1] += v.y; y[2] += v.z; y[3] += v.w;
        }
        if (has && i < A.m) {
            u32* to = A.y + (t0 + mine) * A.y_stride + i;
            const uint4 v = make_uint4(red64(y[0]), red64(y[1]), red64(y[2]), red64(y[3]));
            if (y_vec && i + 4 <= A.m) {
                *reinterpret_cast<uint4*>(to) = v;
            } else {
                to[0] = v.x;
                if (i + 1 < A.m) to[1] = v.y;
                if (i + 2 < A.m) to[2] = v.z;
                if (i + 3 < A.m) to[3] = v.w;
            }
        }
    }
}

// u[t][r] = A[of[t]][r] . x[t]; a CTA per (r, t).
__global__ void __launch_bounds__(128) adapter_shrink_kernel(LinearArgs A, int vec, u32* __restrict__ u) {
    __shared__ u32 part[4];
    pdl_launch_dependents();
    const u32 r = blockIdx.x, t = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int of = A.adapter_of[t];
    if (__syncthreads_or(of < 0 || (u32)of >= A.num_adapters)) return;      // nobody reads this token's; all of the CTA or none (a number that changes meanwhile)
    const u32* a = A.a + ((size_t)of * A.rank + r) * A.n;
    const u32* x = A.x + t * A.x_stride;
    u64 acc = 0;
    if (vec) {
#pragma unroll 4
        for (u32 j = threadIdx.x; j < A.n / 4; j += 128) {
            const uint4 v = reinterpret_cast<const uint4*>(a)[j], w = reinterpret_cast<const uint4*>(x)[j];
            const u32 p[4] = {v.x, v.y, v.z, v.w}, q[4] = {w.x, w.y, w.z, w.w};
            acc += lin_dot4(p, q);
        }
    } else {
#pragma unroll 4
        for (u32 j = threadIdx.x; j < A.n; j += 128) acc += mul31(a[j], x[j]);
    }
    u32 s = red64(acc);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) s = add31(s, __shfl_xor_sync(0xffffffffu, s, off));
    if (lane == 0) part[warp] = s;
    __syncthreads();
    if (threadIdx.x == 0) u[(size_t)t * A.rank + r] = add31(add31(part[0], part[1]), add31(part[2], part[3]));
}

}  // namespace zkb
