// Operators of token-by-token forward passes (see serving.cuh).
#include <cudaTypedefs.h>
#include "kv_append.cuh"
#include "paged_attention.cuh"
#include "adapter_linear.cuh"

namespace zkb {

cudaError_t kv_append_launch(cudaStream_t stream, int sm_count, const AppendArgs& a, int* launches) {
    const u32 rows = 2 * a.c.num_kv_heads + (a.q ? a.num_heads : 0);
    kv_append_kernel<<<dim3(a.num_tokens, (rows + 7) / 8), APPEND_THREADS, 0, stream>>>(a);
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

size_t paged_attention_workspace(int sm_count, uint32_t num_heads, uint32_t num_kv_heads, uint32_t d, uint32_t num_seqs) {
    if (!num_seqs) return 0;
    const PaChoice c = pa_choice(d, num_heads / num_kv_heads);
    return ((size_t)sm_count * 2 * 2 * c.nt * (c.dp + 4) + (size_t)sm_count * 2) * 4;
}
cudaError_t paged_attention_launch(cudaStream_t stream, int sm_count, const PagedAttnArgs& a, int* launches) {
    const PaChoice c = pa_choice(a.c.d, a.num_heads / a.c.num_kv_heads);
    const u32 size = a.c.small ? 2 : 4;
    PaWork w{};
    w.slices = c.slices;
    w.slice_heads = c.slice_heads;
    w.ctas = (u32)sm_count;
    w.gave_up = a.gave_up;
    w.slots = (u32*)a.workspace;
    w.desc = w.slots + (size_t)sm_count * 2 * 2 * c.nt * (c.dp + 4);
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
        ZKB_PA(64, 1) ZKB_PA(64, 2) ZKB_PA(64, 4) ZKB_PA(128, 1) ZKB_PA(128, 2) ZKB_PA(128, 4) ZKB_PA(256, 1) ZKB_PA(256, 2)
#undef ZKB_PA
    }
    return cudaErrorInvalidValue;
}

static size_t round256(size_t b) { return (b + 255) & ~size_t(255); }
size_t adapter_linear_workspace(int sm_count, uint32_t tokens, uint32_t m, uint32_t n, uint32_t num_adapters, uint32_t rank) {
    if (!tokens) return 0;
    const LinPlan p = lin_plan(sm_count, lin_chunk(tokens, n), m, n);
    return round256((num_adapters ? (size_t)tokens * rank * 4 : 0)) + round256(lin_digit_bytes(p)) + lin_slot_bytes(p);
}
cudaError_t adapter_linear_launch(cudaStream_t stream, int sm_count, const LinearArgs& a, int* launches) {
    u32* u = a.num_adapters ? (u32*)a.workspace : nullptr;
    if (u) {
        adapter_shrink_kernel<<<(a.tokens * a.rank + 7) / 8, 256, 0, stream>>>(a, u);
        ++*launches;
    }
    if (a.n % 4 || ((uintptr_t)a.w & 15) || a.tokens < 5) {
        adapter_linear_kernel<<<dim3((a.m + 31) / 32, (a.tokens + 31) / 32), 256, 0, stream>>>(a, u);
        ++*launches;
        return cudaGetLastError();
    }
    CUtensorMap map;
    cudaError_t e = rows_tensor_map(&map, a.w, a.m, a.n);
    if (e != cudaSuccess) return e;
    e = cudaFuncSetAttribute(linear_bytes_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 201 * 1024);
    if (e != cudaSuccess) return e;
    const u32 chunk = lin_chunk(a.tokens, a.n);
    unsigned char* digits = (unsigned char*)a.workspace + round256(u ? (size_t)a.tokens * a.rank * 4 : 0);
    u32* slots = (u32*)(digits + round256(lin_digit_bytes(lin_plan(sm_count, chunk, a.m, a.n))));
    for (u32 t0 = 0; t0 < a.tokens; t0 += chunk) {
        LinearArgs c = a;
        c.tokens = a.tokens - t0 < chunk ? a.tokens - t0 : chunk;
        c.x += t0 * a.x_stride;
        c.y += t0 * a.y_stride;
        if (u) c.adapter_of += t0;
        const LinPlan p = lin_plan(sm_count, c.tokens, a.m, a.n);
        linear_digits_kernel<<<dim3(p.steps, p.ntiles), 8 * p.tt, 0, stream>>>(c.x, c.x_stride, p, digits);
        linear_bytes_kernel<<<p.ctas, LIN_THREADS, (size_t)p.stages * p.stage_bytes + 1024, stream>>>(map, p, digits, slots, a.gave_up);
        linear_join_kernel<<<dim3((a.m + 255) / 256, c.tokens), 256, 0, stream>>>(c, p, slots, u ? u + (size_t)t0 * a.rank : nullptr);
        *launches += 3;
    }
    return cudaGetLastError();
}

}  // namespace zkb
