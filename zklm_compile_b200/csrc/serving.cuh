// Launchers of the operators of token-by-token forward passes: the paged key-value cache, the attention that reads it and
// projections with low-rank adapters.  Kernels are in a compilation unit of their own (serving.cu); nothing here allocates, waits
// or keeps anything between calls.
#pragma once
#include <cstddef>
#include <cstdint>
#include <cuda_runtime.h>

namespace zkb {

// What a call finds wrong with a sequence on the device is added to the caller's status word of that sequence (the largest code stays).
enum : int { SERVE_PAGE = 1, SERVE_ROTATION = 2, SERVE_RANGE = 3, SERVE_SCORE = 4, SERVE_ZERO_SUM = 5 };

// Pages of [num_kv_heads][page_size][d_head] elements, `page_stride` elements apart: canonical u32, or int16 (centred values).
struct KvPages {
    void* k;
    void* v;
    uint64_t page_stride;
    uint32_t num_pages, page_bits, num_kv_heads, d;
    int small;
};

struct AppendArgs {
    KvPages c;
    const uint32_t *k, *v, *q;
    uint64_t k_stride, v_stride, q_stride, q_out_stride;   // words between tokens
    uint32_t* q_out;
    uint32_t num_heads, num_tokens, num_seqs, max_blocks;
    const int32_t *block_table, *row_start, *start;
    const int32_t* cos_sin;                                  // [positions][rot / 2][2]
    uint32_t positions, rot, shift;
    int pairs;
    int32_t* status;
};
cudaError_t kv_append_launch(cudaStream_t stream, int sm_count, const AppendArgs& a, int* launches);

struct PagedAttnArgs {
    KvPages c;
    const uint32_t* q;
    uint64_t q_stride;
    uint32_t num_heads, num_seqs, max_blocks;
    const int32_t *block_table, *lens;
    const uint32_t* table;
    uint32_t n_table, score_shift;
    uint32_t* out;                                           // [num_seqs][num_heads][d]
    int32_t* status;
    void* workspace;
    void* counters;                                          // paged_attention_counters bytes, zero before and after every call; NULL: the first of the workspace
    int* gave_up;                                            // set when a wait inside a kernel ran out, blocks of a row are missing or parts of one are left over
};
size_t paged_attention_counters(int sm_count);
size_t paged_attention_workspace(int sm_count, uint32_t num_heads, uint32_t num_kv_heads, uint32_t d, uint32_t num_seqs);
cudaError_t paged_attention_launch(cudaStream_t stream, int sm_count, const PagedAttnArgs& a, int* launches);

struct LinearArgs {
    const uint32_t *x, *w, *bias;
    uint64_t x_stride, y_stride;
    uint32_t tokens, m, n;
    const uint32_t *a, *b;                                   // [num_adapters][rank][n], [num_adapters][m][rank]
    uint32_t num_adapters, rank;
    const int32_t* adapter_of;                               // per token; outside [0, num_adapters): none
    uint32_t* y;
    void* workspace;
    int* gave_up;                                            // as above
};
bool adapter_linear_fits(uint32_t tokens, uint32_t m, uint32_t n, uint32_t num_adapters, uint32_t rank);
size_t adapter_linear_workspace(int sm_count, uint32_t tokens, uint32_t m, uint32_t n, uint32_t num_adapters, uint32_t rank);
cudaError_t adapter_linear_launch(cudaStream_t stream, int sm_count, const LinearArgs& a, int* launches);

}  // namespace zkb
