// C ABI, part 10: operators of token-by-token forward passes.  Included by zkb200.cu.
//
// All pointers are device memory and every call is enqueued on the context's stream without waiting for it.  What only the device can
// see (a page number outside the pool, a score that the table does not know) goes into the caller's status words.

namespace {

void need_words(const void* p, const char* what) {
    if (!p) throw ArgFail{ZKB_E_ARG, std::string("serving: ") + what + " is missing"};
    if ((uintptr_t)p & 3) throw ArgFail{ZKB_E_ARG, std::string("serving: ") + what + " must be 4-byte aligned"};
}
KvPages kv_pages(const zkb_kv_cache* k) {
    if (!k) throw ArgFail{ZKB_E_ARG, "serving: no cache"};
    if (k->elem != ZKB_KV_FIELD && k->elem != ZKB_KV_I16) throw ArgFail{ZKB_E_ARG, "serving: unknown element type of the cache"};
    if (!k->num_pages || !k->num_kv_heads || !k->d_head) throw ArgFail{ZKB_E_ARG, "serving: empty dimension of the cache"};
    if (k->num_pages > 0x7fffffffu || k->num_kv_heads > 65535) throw ArgFail{ZKB_E_TOO_LARGE, "serving: more than 2^31 - 1 pages or 65535 key heads"};
    if (k->d_head > ZKB_KV_MAX_D_HEAD) throw ArgFail{ZKB_E_TOO_LARGE, "serving: d_head above 256"};
    if (!k->page_size || (k->page_size & (k->page_size - 1)) || k->page_size > 65536) throw ArgFail{ZKB_E_ARG, "serving: the page size is a power of two up to 65536"};
    const uint32_t align = k->elem == ZKB_KV_I16 ? 1 : 3;
    if (!k->k_pages_dev || !k->v_pages_dev || ((uintptr_t)k->k_pages_dev & align) || ((uintptr_t)k->v_pages_dev & align))
        throw ArgFail{ZKB_E_ARG, "serving: the cache's pages are missing or not aligned to their elements"};
    const uint64_t dense = (uint64_t)k->num_kv_heads * k->page_size * k->d_head;
    if (k->page_stride && k->page_stride < dense) throw ArgFail{ZKB_E_ARG, "serving: page_stride is less than a page"};
    uint32_t bits = 0;
    while ((1u << bits) < k->page_size) bits++;
    return KvPages{k->k_pages_dev, k->v_pages_dev, k->page_stride ? k->page_stride : dense, k->num_pages, bits, k->num_kv_heads, k->d_head, k->elem == ZKB_KV_I16};
}
uint64_t serve_stride(size_t given, uint64_t least, const char* what) {
    if (given && given < least) throw ArgFail{ZKB_E_ARG, std::string("serving: ") + what + " is less than a row"};
    return given ? given : least;
}
// The caller's workspace, or the context's scratch for the length of this call (work on one stream runs in order; a captured call would
// keep an address that later calls of the context use too).
struct ServeWorkspace {
    zkb_ctx* c;
    zkb_ctx::ScratchMark mark{};
    bool own = false;
    void* p = nullptr;
    ServeWorkspace(zkb_ctx* ctx, void* given, size_t given_bytes, size_t need) : c(ctx) {
        if (given) {
            if (given_bytes < need) throw ArgFail{ZKB_E_TOO_LARGE, "serving: the workspace is too small"};
            if ((uintptr_t)given & 255) throw ArgFail{ZKB_E_ARG, "serving: the workspace must be 256-byte aligned"};
            p = given;
        } else if (need) {
            cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
            ZKB_CUDA(cudaStreamIsCapturing(c->stream, &st));
            if (st != cudaStreamCaptureStatusNone) throw ArgFail{ZKB_E_ARG, "serving: a captured call needs a workspace of its own"};
            mark = c->scratch_mark();
            p = c->scratch(need);
            own = true;
        }
    }
    ServeWorkspace(const ServeWorkspace&) = delete;
    ~ServeWorkspace() { if (own) c->scratch_release(mark); }
};
void serve_launched(zkb_ctx* c, int n, const char* file, int line) {
    for (int i = 0; i < n; i++) c->launched(file, line);
}

}  // namespace

extern "C" {

int32_t zkb_kv_append(zkb_ctx* c, const zkb_kv_cache* cache, const uint32_t* k_dev, size_t k_stride, const uint32_t* v_dev, size_t v_stride, uint32_t num_tokens,
                      const int32_t* block_table_dev, uint32_t num_seqs, uint32_t max_blocks, const int32_t* row_start_dev, const int32_t* start_dev,
                      const zkb_kv_rotation* rotation, const uint32_t* q_dev, size_t q_stride, uint32_t num_heads, uint32_t* q_out_dev, size_t q_out_stride,
                      int32_t* status_dev) {
    if (!c) return ZKB_E_ARG;
    ZKB_TRY(c, {
        c->use();
        AppendArgs a{};
        a.c = kv_pages(cache);
        const uint64_t row = (uint64_t)a.c.num_kv_heads * a.c.d, q_row = (uint64_t)num_heads * a.c.d;
        if (num_tokens > 0x7fffffffu || num_seqs > 0x7ffffffeu || num_heads > 65535) throw ArgFail{ZKB_E_TOO_LARGE, "kv_append: too many tokens, sequences or heads"};
        a.k_stride = serve_stride(k_stride, row, "k_stride");
        a.v_stride = serve_stride(v_stride, row, "v_stride");
        if (rotation) {
            if (rotation->rot_dim > a.c.d || (rotation->rot_dim & 1)) throw ArgFail{ZKB_E_ARG, "kv_append: rot_dim is even and at most d_head"};
            if (rotation->shift > 30) throw ArgFail{ZKB_E_ARG, "kv_append: a rotation has at most 30 fractional bits"};
            if (rotation->rot_dim) need_words(rotation->cos_sin_dev, "the rotation's table");
            a.cos_sin = rotation->cos_sin_dev;
            a.positions = rotation->positions;
            a.rot = rotation->rot_dim;
            a.shift = rotation->shift;
            a.pairs = rotation->pairs != 0;
        }
        if (q_dev || q_out_dev) {
            if (!num_heads) throw ArgFail{ZKB_E_ARG, "kv_append: q without heads"};
            need_words(q_dev, "q");
            need_words(q_out_dev, "q_out");
            a.q_stride = serve_stride(q_stride, q_row, "q_stride");
            a.q_out_stride = serve_stride(q_out_stride, q_row, "q_out_stride");
            if (q_dev == q_out_dev && a.q_stride != a.q_out_stride) throw ArgFail{ZKB_E_ARG, "kv_append: q in place keeps its stride"};
            a.q = q_dev;
            a.q_out = q_out_dev;
            a.num_heads = num_heads;
        }
        if (!num_tokens || !num_seqs) return ZKB_OK;
        if (!max_blocks) throw ArgFail{ZKB_E_ARG, "kv_append: a block table without places"};
        need_words(k_dev, "k"); need_words(v_dev, "v"); need_words(block_table_dev, "block_table"); need_words(row_start_dev, "row_start");
        need_words(start_dev, "start"); need_words(status_dev, "status");
        a.k = k_dev; a.v = v_dev;
        a.num_tokens = num_tokens; a.num_seqs = num_seqs; a.max_blocks = max_blocks;
        a.block_table = block_table_dev; a.row_start = row_start_dev; a.start = start_dev; a.status = status_dev;
        int n = 0;
        ZKB_CUDA(kv_append_launch(c->stream, c->sm_count, a, &n));
        serve_launched(c, n, __FILE__, __LINE__);
    });
}

static void paged_attention_dims(const KvPages& k, uint32_t num_heads, uint32_t num_seqs) {
    if (!num_heads || num_heads % k.num_kv_heads) throw ArgFail{ZKB_E_ARG, "paged_attention: num_heads is a multiple of num_kv_heads"};
    if (num_heads > 65535 || num_seqs > 0x7fffffffu) throw ArgFail{ZKB_E_TOO_LARGE, "paged_attention: too many heads or sequences"};
}
size_t zkb_paged_attention_workspace(zkb_ctx* c, const zkb_kv_cache* cache, uint32_t num_seqs, uint32_t num_heads) {
    if (!c) return 0;
    try {
        const KvPages k = kv_pages(cache);
        paged_attention_dims(k, num_heads, num_seqs);
        return paged_attention_workspace(c->sm_count, num_heads, k.num_kv_heads, k.d, num_seqs);
    } catch (const ArgFail& e) { c->err = e.msg; return 0; }
    catch (const std::bad_alloc&) { return 0; }
}
int32_t zkb_paged_attention(zkb_ctx* c, const zkb_kv_cache* cache, const uint32_t* q_dev, size_t q_stride, uint32_t num_heads, const int32_t* block_table_dev,
                            uint32_t num_seqs, uint32_t max_blocks, const int32_t* lens_dev, const uint32_t* table_out_dev, size_t n_table, uint32_t score_shift,
                            uint32_t* out_dev, int32_t* status_dev, void* workspace_dev, size_t workspace_bytes) {
    if (!c) return ZKB_E_ARG;
    ZKB_TRY(c, {
        c->use();
        PagedAttnArgs a{};
        a.c = kv_pages(cache);
        paged_attention_dims(a.c, num_heads, num_seqs);
        if (n_table != 256 && n_table != 65536) throw ArgFail{ZKB_E_ARG, "paged_attention: the exp table has 256 or 65536 entries"};
        if (score_shift > 30) throw ArgFail{ZKB_E_ARG, "paged_attention: score_shift is at most 30"};
        a.q_stride = serve_stride(q_stride, (uint64_t)num_heads * a.c.d, "q_stride");
        if (!num_seqs) return ZKB_OK;
        if (!max_blocks) throw ArgFail{ZKB_E_ARG, "paged_attention: a block table without places"};
        // the work is counted in tiles of 16 positions and up, in 32 bits a CTA
        if ((double)num_seqs * max_blocks * cache->page_size * num_heads >= (double)(1ull << 42)) throw ArgFail{ZKB_E_TOO_LARGE, "paged_attention: more than 2^42 scores"};
        need_words(q_dev, "q"); need_words(block_table_dev, "block_table"); need_words(lens_dev, "lens"); need_words(table_out_dev, "the exp table");
        need_words(out_dev, "out"); need_words(status_dev, "status");
        if (out_dev == q_dev) throw ArgFail{ZKB_E_ARG, "paged_attention: out is not q"};
        a.q = q_dev; a.num_heads = num_heads; a.num_seqs = num_seqs; a.max_blocks = max_blocks;
        a.block_table = block_table_dev; a.lens = lens_dev; a.table = table_out_dev; a.n_table = (u32)n_table; a.score_shift = score_shift;
        a.out = out_dev; a.status = status_dev;
        ServeWorkspace ws(c, workspace_dev, workspace_bytes, paged_attention_workspace(c->sm_count, num_heads, a.c.num_kv_heads, a.c.d, num_seqs));
        a.workspace = ws.p;
        a.counters = workspace_dev ? nullptr : c->serve_counts(paged_attention_counters(c->sm_count));
        a.gave_up = c->serve_flag();
        int n = 0;
        ZKB_CUDA(paged_attention_launch(c->stream, c->sm_count, a, &n));
        serve_launched(c, n, __FILE__, __LINE__);
    });
}

static void adapter_linear_dims(uint32_t tokens, uint32_t m, uint32_t n, uint32_t num_adapters, uint32_t rank) {
    if (!m || !n) throw ArgFail{ZKB_E_ARG, "adapter_linear: empty dimension"};
    if (num_adapters && !rank) throw ArgFail{ZKB_E_ARG, "adapter_linear: adapters of rank 0"};
    if (m > (1u << 24) || n > (1u << 24) || tokens > (1u << 20) || rank > 1024) throw ArgFail{ZKB_E_TOO_LARGE, "adapter_linear: more than 2^24 rows or columns, 2^20 tokens or rank 1024"};
    if (!adapter_linear_fits(tokens, m, n, num_adapters, rank)) throw ArgFail{ZKB_E_TOO_LARGE, "adapter_linear: W has more than 2^40 elements"};
}
size_t zkb_adapter_linear_workspace(zkb_ctx* c, uint32_t tokens, uint32_t m, uint32_t n, uint32_t num_adapters, uint32_t rank) {
    if (!c) return 0;
    try {
        adapter_linear_dims(tokens, m, n, num_adapters, rank);
        return adapter_linear_workspace(c->sm_count, tokens, m, n, num_adapters, rank);
    } catch (const ArgFail& e) { c->err = e.msg; return 0; }
    catch (const std::bad_alloc&) { return 0; }
}
int32_t zkb_adapter_linear(zkb_ctx* c, const uint32_t* x_dev, size_t x_stride, const uint32_t* w_dev, const uint32_t* bias_dev, uint32_t tokens, uint32_t m, uint32_t n,
                           const uint32_t* a_dev, const uint32_t* b_dev, uint32_t num_adapters, uint32_t rank, const int32_t* adapter_of_dev, uint32_t* y_dev,
                           size_t y_stride, void* workspace_dev, size_t workspace_bytes) {
    if (!c) return ZKB_E_ARG;
    ZKB_TRY(c, {
        c->use();
        adapter_linear_dims(tokens, m, n, num_adapters, rank);
        LinearArgs a{};
        a.x_stride = serve_stride(x_stride, n, "x_stride");
        a.y_stride = serve_stride(y_stride, m, "y_stride");
        if (!tokens) return ZKB_OK;
        need_words(x_dev, "x"); need_words(w_dev, "w"); need_words(y_dev, "y");
        if (bias_dev) need_words(bias_dev, "bias");
        if (y_dev == x_dev) throw ArgFail{ZKB_E_ARG, "adapter_linear: y is not x"};
        if (num_adapters) { need_words(a_dev, "the adapters' A"); need_words(b_dev, "the adapters' B"); need_words(adapter_of_dev, "adapter_of"); }
        a.x = x_dev; a.w = w_dev; a.bias = bias_dev; a.tokens = tokens; a.m = m; a.n = n; a.a = a_dev; a.b = b_dev;
        a.num_adapters = num_adapters; a.rank = num_adapters ? rank : 0; a.adapter_of = adapter_of_dev; a.y = y_dev;
        ServeWorkspace ws(c, workspace_dev, workspace_bytes, adapter_linear_workspace(c->sm_count, tokens, m, n, num_adapters, rank));
        a.workspace = ws.p;
        a.gave_up = c->serve_flag();
        int k = 0;
        ZKB_CUDA(adapter_linear_launch(c->stream, c->sm_count, a, &k));
        serve_launched(c, k, __FILE__, __LINE__);
    });
}

}  // extern "C"
