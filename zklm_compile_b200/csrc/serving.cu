// Operators of token-by-token forward passes (see serving.cuh).
#include <cudaTypedefs.h>
#include "kv_append.cuh"
#include "paged_attention.cuh"
#include "adapter_linear.cuh"

namespace zkb {

cudaError_t kv_append_launch(cudaStream_t stream, int sm_count, const AppendArgs& a, int* launches) {
    const u32 rows = 2 * a.c.num_kv_heads + (a.q ? a.num_heads : 0);
    const uintptr_t words = (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.q | (uintptr_t)a.q_out | (uintptr_t)a.cos_sin | (a.c.small ? 0 : (uintptr_t)a.c.k | (uintptr_t)a.c.v);
    const uint64_t strides = a.k_stride | a.v_stride | a.q_stride | a.q_out_stride | a.c.page_stride | a.c.d;
    const bool vec = !(words & 15) && !(((uintptr_t)a.c.k | (uintptr_t)a.c.v) & 7) && strides % 4 == 0 && a.rot % (a.pairs ? 4 : 8) == 0;
    if (vec) {
        const u32 rot_items = a.pairs ? a.rot / 4 : a.rot / 8, items = a.pairs ? a.c.d / 4 : rot_items + (a.c.d - a.rot) / 4;
        // as many CTAs a token as give every SM a few; one for many tokens, which then amortises the look-up
        const u32 per_pass = APPEND_THREADS / items, passes = (rows + per_pass - 1) / per_pass, want = ((u32)sm_count * 4 + a.num_tokens - 1) / a.num_tokens;
        const dim3 grid(a.num_tokens, want < passes ? want : passes);
        if (a.c.small && a.pairs) kv_append_vec_kernel<true, true><<<grid, APPEND_THREADS, 0, stream>>>(a, items, rot_items);
        else if (a.c.small) kv_append_vec_kernel<true, false><<<grid, APPEND_THREADS, 0, stream>>>(a, items, rot_items);
        else if (a.pairs) kv_append_vec_kernel<false, true><<<grid, APPEND_THREADS, 0, stream>>>(a, items, rot_items);
        else kv_append_vec_kernel<false, false><<<grid, APPEND_THREADS, 0, stream>>>(a, items, rot_items);
    } else {
        kv_append_kernel<<<dim3(a.num_tokens, (rows + 7) / 8), APPEND_THREADS, 0, stream>>>(a);
    }
    ++*launches;
    return cudaGetLastError();
}

// cuTensorMapEncodeTiled, without linking the driver library.
static PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder() {
    static PFN_cuTensorMapEncodeTiled_v12000 f = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult r;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &r) != cudaSuccess || r != cudaDriverEntryPointSuccess) p = nullptr;
        return (PFN_cuTensorMapEncodeTiled_v12000)p;
    }();
    return f;
}
// rows x n words, boxes of LIN_ROWS rows x LIN_STEP words, 128-byte swizzle; what lies outside reads as zero.
static cudaError_t rows_tensor_map(CUtensorMap* map, const u32* w, u32 rows, u32 n) {
    auto encode = tensor_map_encoder();
    if (!encode) return cudaErrorNotSupported;
    const cuuint64_t dims[2] = {n, rows}, strides[1] = {(cuuint64_t)n * 4};
    const cuuint32_t box[2] = {LIN_STEP, LIN_ROWS}, unit[2] = {1, 1};
    const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, (void*)w, dims, strides, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

size_t paged_attention_counters(int sm_count) { return ((size_t)(sm_count + 1) * 4 + 255) / 256 * 256; }
size_t paged_attention_workspace(int sm_count, uint32_t num_heads, uint32_t num_kv_heads, uint32_t d, uint32_t num_seqs) {
    if (!num_seqs) return 0;
    const PaChoice c = pa_choice(d, num_heads / num_kv_heads);
    return paged_attention_counters(sm_count) + (size_t)sm_count * 2 * 2 * c.nt * (c.dp + 4) * 4;
}
cudaError_t paged_attention_launch(cudaStream_t stream, int sm_count, const PagedAttnArgs& a, int* launches) {
    const PaChoice c = pa_choice(a.c.d, a.num_heads / a.c.num_kv_heads);
    const u32 size = a.c.small ? 2 : 4;
    PaWork w{};
    w.slices = c.slices;
    w.slice_heads = c.slice_heads;
    w.ctas = (u32)sm_count;
    w.gave_up = a.gave_up;
    w.q_vec = a.c.d % 4 == 0 && a.q_stride % 4 == 0 && !((uintptr_t)a.q & 15);
    w.arrived = a.counters ? (u32*)a.counters : (u32*)a.workspace;
    w.begun = w.arrived + sm_count;
    w.slots = (u32*)((char*)a.workspace + paged_attention_counters(sm_count));
    // Tensor copies want 16-byte boundaries; a box of less than the 8 rows of the swizzle's pattern is left to plain loads.
    CUtensorMap maps[2] = {};
    const uint64_t row_bytes = (uint64_t)a.c.d * size, page_bytes = a.c.page_stride * size;
    if (a.c.page_bits >= 3 && ((u64)a.c.num_kv_heads << a.c.page_bits) < (1ull << 31) && row_bytes % 16 == 0 && page_bytes % 16 == 0 && page_bytes < (1ull << 40) && !((uintptr_t)a.c.k & 15) && !((uintptr_t)a.c.v & 15)) {
        auto encode = tensor_map_encoder();
        if (!encode) return cudaErrorNotSupported;
        w.fast = a.c.page_bits >= 4 ? 16 : 8;
        w.whole = w.fast == 16 && row_bytes % 128 == 0;
        const u32 columns = w.whole ? (u32)(row_bytes / 128) : 1u;
        const cuuint64_t dims[4] = {w.whole ? 128 / size : a.c.d, (cuuint64_t)a.c.num_kv_heads << a.c.page_bits, columns, a.c.num_pages};
        const cuuint64_t strides[3] = {row_bytes, w.whole ? 128 : row_bytes, page_bytes};
        const cuuint32_t box[4] = {128 / size, (cuuint32_t)w.fast, columns, 1}, unit[4] = {1, 1, 1, 1};
        for (int i = 0; i < 2; i++)
            if (encode(&maps[i], a.c.small ? CU_TENSOR_MAP_DATA_TYPE_UINT16 : CU_TENSOR_MAP_DATA_TYPE_UINT32, 4, i ? a.c.v : a.c.k, dims, strides, box, unit,
                       CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
                return cudaErrorInvalidValue;
    }
    const u32 which = c.dp | c.nt << 16 | (a.c.small ? 1u << 24 : 0u);
    switch (which) {
#define ZKB_PA(DP, NT)                                                                              \
    case DP | NT << 16: return pa_launch<DP, false, NT>(stream, maps, a, w, launches);                     \
    case DP | NT << 16 | 1u << 24: return pa_launch<DP, true, NT>(stream, maps, a, w, launches);
        ZKB_PA(64, 1) ZKB_PA(64, 2) ZKB_PA(64, 3) ZKB_PA(64, 4) ZKB_PA(128, 1) ZKB_PA(128, 2) ZKB_PA(128, 3) ZKB_PA(128, 4) ZKB_PA(256, 1) ZKB_PA(256, 2)
#undef ZKB_PA
    }
    return cudaErrorInvalidValue;
}

static size_t round256(size_t b) { return (b + 255) & ~size_t(255); }
// Launch that, if `early`, may begin while the kernel before it is still running (see pdl_wait in m31.cuh): only behind a kernel of the same call, whose own
// launch waited for all that came before.
template <class... KArgs, class... Args>
static cudaError_t launch_after(bool early, void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = grid; cfg.blockDim = block; cfg.dynamicSmemBytes = smem; cfg.stream = stream; cfg.attrs = at; cfg.numAttrs = early ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, KArgs(args)...);
}

// Where the parts of a call's workspace begin.
struct LinSpace { size_t slots, end; u32 chunk, a_rows; };
static LinSpace lin_space(int sm_count, u32 tokens, u32 m, u32 n, u32 num_adapters, u32 rank) {
    LinSpace w{};
    w.chunk = lin_chunk(tokens);
    w.a_rows = lin_a_rows(w.chunk, m, num_adapters, rank);
    const LinPlan p = lin_plan(sm_count, w.chunk, m, n, w.a_rows);
    w.slots = num_adapters && !w.a_rows ? round256((size_t)w.chunk * rank * 4) : 0;
    w.end = w.slots + lin_slot_bytes(sm_count, p);
    return w;
}
bool adapter_linear_fits(uint32_t tokens, uint32_t m, uint32_t n, uint32_t num_adapters, uint32_t rank) {
    return lin_fits(lin_chunk(tokens), m, n, lin_a_rows(lin_chunk(tokens), m, num_adapters, rank));
}
size_t adapter_linear_workspace(int sm_count, uint32_t tokens, uint32_t m, uint32_t n, uint32_t num_adapters, uint32_t rank) {
    return tokens ? lin_space(sm_count, tokens, m, n, num_adapters, rank).end : 0;
}
template <bool W_COPY>
static cudaError_t lin_product(cudaStream_t stream, bool early, const CUtensorMap& map_w, const CUtensorMap& map_a, const LinPlan& p, const LinearArgs& a, u32* slots) {
    const cudaError_t e = allow_smem(linear_bytes_kernel<W_COPY>, 201 * 1024);
    if (e != cudaSuccess) return e;
    const int x_vec = a.n % 4 == 0 && a.x_stride % 4 == 0 && !((uintptr_t)a.x & 15);
    const size_t smem = (size_t)p.stages * p.stage_bytes + 1024;
    return launch_after(early, linear_bytes_kernel<W_COPY>, dim3(p.ctas), dim3(LIN_THREADS), smem, stream, map_w, map_a, p, a, x_vec, slots);
}
cudaError_t adapter_linear_launch(cudaStream_t stream, int sm_count, const LinearArgs& a, int* launches) {
    const LinSpace space = lin_space(sm_count, a.tokens, a.m, a.n, a.num_adapters, a.rank);
    u32* u = (u32*)a.workspace;
    u32* slots = (u32*)((unsigned char*)a.workspace + space.slots);
    const bool copies = a.n % 4 == 0 && !((uintptr_t)a.w & 15) && !(space.a_rows && ((uintptr_t)a.a & 15)), apart = a.rank && !space.a_rows;
    const int b_vec = a.rank % 4 == 0 && !((uintptr_t)a.b & 15), y_vec = a.y_stride % 4 == 0 && !((uintptr_t)a.y & 15);
    CUtensorMap map_w = {}, map_a = {};
    cudaError_t e = cudaSuccess;
    if (copies) {
        if ((e = rows_tensor_map(&map_w, a.w, a.m, a.n)) != cudaSuccess) return e;
        if (space.a_rows && (e = rows_tensor_map(&map_a, a.a, space.a_rows, a.n)) != cudaSuccess) return e;
    }
    for (u32 t0 = 0; t0 < a.tokens; t0 += space.chunk) {
        LinearArgs c = a;
        c.tokens = a.tokens - t0 < space.chunk ? a.tokens - t0 : space.chunk;
        c.x += t0 * a.x_stride;
        c.y += t0 * a.y_stride;
        if (a.rank) c.adapter_of += t0;
        const LinPlan p = lin_plan(sm_count, c.tokens, a.m, a.n, space.a_rows);
        if (apart) {
            const int vec = a.n % 4 == 0 && a.x_stride % 4 == 0 && !((uintptr_t)a.x & 15) && !((uintptr_t)a.a & 15);
            adapter_shrink_kernel<<<dim3(a.rank, c.tokens), 128, 0, stream>>>(c, vec, u);
            ++*launches;
        }
        e = copies ? lin_product<true>(stream, apart, map_w, map_a, p, c, slots) : lin_product<false>(stream, apart, map_w, map_a, p, c, slots);
        if (e != cudaSuccess) return e;
        // four blocks of rows a CTA where there are many of them: the tokens' A x is then summed up a quarter as often (4096 rows, rank 16, 64 / 512 / 1024 tokens: one block
        // 24 / 79 / 150 us, four 35 / 77 / 141; 9728 rows 59 / 199 / 412 and 61 / 194 / 372)
        const u32 groups = (p.tt + LIN_JOIN_TOKENS - 1) / LIN_JOIN_TOKENS, row_blocks = (a.m + LIN_JOIN_ROWS - 1) / LIN_JOIN_ROWS;
        const u32 blocks = (u64)row_blocks * p.ntiles * groups > 8ull * sm_count ? 4 : 1;
        e = launch_after(true, linear_join_kernel, dim3((row_blocks + blocks - 1) / blocks, p.ntiles * groups), dim3(256), 0, stream, c, p, blocks, b_vec, y_vec, slots, u);
        if (e != cudaSuccess) return e;
        *launches += 2;
    }
    return cudaGetLastError();
}

}  // namespace zkb
