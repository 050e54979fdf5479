// Operators of token-by-token forward passes (see serving.cuh).
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

size_t paged_attention_workspace(int, uint32_t, uint32_t, uint32_t, uint32_t) { return 256; }
cudaError_t paged_attention_launch(cudaStream_t stream, int sm_count, const PagedAttnArgs& a, int* launches) {
    paged_attention_kernel<<<dim3(a.num_seqs, a.num_heads), PA_THREADS, 0, stream>>>(a);
    ++*launches;
    return cudaGetLastError();
}

size_t adapter_linear_workspace(int, uint32_t tokens, uint32_t, uint32_t, uint32_t num_adapters, uint32_t rank) {
    return num_adapters ? (size_t)tokens * rank * 4 : 0;
}
cudaError_t adapter_linear_launch(cudaStream_t stream, int sm_count, const LinearArgs& a, int* launches) {
    u32* u = a.num_adapters ? (u32*)a.workspace : nullptr;
    if (u) {
        adapter_shrink_kernel<<<(a.tokens * a.rank + 7) / 8, 256, 0, stream>>>(a, u);
        ++*launches;
    }
    adapter_linear_kernel<<<dim3((a.m + 31) / 32, (a.tokens + 31) / 32), 256, 0, stream>>>(a, u);
    ++*launches;
    return cudaGetLastError();
}

}  // namespace zkb
