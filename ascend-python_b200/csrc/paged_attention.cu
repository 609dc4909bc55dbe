// C entries of the attention over a paged key-value cache (npu_paged_attention, npu_paged_prompt_attention): argument checks.
#include "paged_common.cuh"

namespace qmm {
namespace paged {

static bool vectors(const void *base, int64_t a, int64_t b, int64_t c) {
    return (reinterpret_cast<uintptr_t>(base) & 15) == 0 && ((a | b | c) & 7) == 0;
}

static bool words(const void *base) { return (reinterpret_cast<uintptr_t>(base) & 3) == 0; }

// The arguments of both entries as a Problem.
static int describe(Problem *p, const char *op, const void *query, int dtype, int64_t tokens, int64_t heads, int64_t stride_token,
                    int64_t stride_head, const qmm_kv_cache *cache, const int32_t *block_table, int64_t table_stride,
                    int64_t max_pages, const int32_t *seq_lens, int64_t batch, double scale, int64_t window, int64_t sinks,
                    void *out, float *lse) {
    const std::string name(op);
    QMM_REQUIRE(dtype == QMM_DTYPE_BF16 || dtype == QMM_DTYPE_F16, name + ": the query must be bf16 or f16");
    QMM_REQUIRE(cache != nullptr, name + ": no cache given");
    QMM_REQUIRE(tokens >= 0 && heads >= 0 && batch >= 0 && max_pages >= 0 && cache->pages >= 0,
                name + ": sizes must be non-negative");
    QMM_REQUIRE(window >= 0 && sinks >= 0, name + ": window and sinks must be non-negative");
    QMM_REQUIRE(window > 0 || sinks == 0, name + ": sinks have a meaning with a window only");
    QMM_REQUIRE(cache->dim >= 8 && cache->dim <= 256 && cache->dim % 8 == 0,
                name + ": the head dimension must be a multiple of 8 up to 256");
    QMM_REQUIRE(cache->page_size >= 1 && cache->page_size <= 0x7fffffff, name + ": the page size must be positive");
    QMM_REQUIRE(cache->kv_heads >= 1 && heads % cache->kv_heads == 0,
                name + ": the query's heads must be a multiple of the cache's");
    QMM_REQUIRE(tokens < 0x7fffffff && batch < 0x7fffffff && heads <= 65535 && max_pages <= 0x7fffffff && cache->pages <= 0x7fffffff,
                name + ": sizes out of range");
    const float factor = static_cast<float>(scale) * 1.4426950408889634f;  // as the kernels take it
    QMM_REQUIRE(factor - factor == 0.0f, name + ": scale_value must be finite, and so must it times log2(e) in fp32");
    QMM_REQUIRE(vectors(query, stride_token, stride_head, 0) &&
                    vectors(cache->key, cache->key_stride_page, cache->key_stride_place, cache->key_stride_head) &&
                    vectors(cache->value, cache->value_stride_page, cache->value_stride_place, cache->value_stride_head),
                name + ": query and caches must begin at 16-byte boundaries, with strides of multiples of 8 elements");
    QMM_REQUIRE(vectors(out, 0, 0, 0) && words(lse) && words(block_table) && words(seq_lens),
                name + ": out must begin at a 16-byte boundary, lse, block_table and seq_lens at 4-byte boundaries");
    p->q = query;
    p->q_st = stride_token;
    p->q_sh = stride_head;
    p->k = cache->key;
    p->v = cache->value;
    p->k_sb = cache->key_stride_page;
    p->k_st = cache->key_stride_place;
    p->k_sh = cache->key_stride_head;
    p->v_sb = cache->value_stride_page;
    p->v_st = cache->value_stride_place;
    p->v_sh = cache->value_stride_head;
    p->table = block_table;
    p->table_st = table_stride;
    p->lens = seq_lens;
    p->start = nullptr;
    p->out = out;
    p->lse = lse;
    p->batch = static_cast<int>(batch);
    p->heads = static_cast<int>(heads);
    p->kv_heads = static_cast<int>(cache->kv_heads);
    p->group = static_cast<int>(heads / cache->kv_heads);
    p->dim = static_cast<int>(cache->dim);
    p->page = static_cast<int>(cache->page_size);
    p->page_shift = -1;
    for (int s = 0; s < 31; ++s)
        if (p->page == 1 << s) p->page_shift = s;
    p->max_pages = static_cast<int>(max_pages);
    p->window = static_cast<int>(window < 0x7fffffff ? window : 0x7fffffff);
    p->sinks = static_cast<int>(sinks < 0x7fffffff ? sinks : 0x7fffffff);
    p->tokens = tokens;
    p->pages = cache->pages;
    const int64_t capacity = cache->pages == 0 ? 0 : max_pages * cache->page_size;
    p->capacity = static_cast<int>(capacity < 0x7fffff00 ? capacity : 0x7fffff00);  // indices run up to a tile further
    p->scale = static_cast<float>(scale);
    return QMM_OK;
}

}  // namespace paged
}  // namespace qmm

using qmm::fail;

extern "C" {

int qmm_paged_attention_workspace_size(int64_t batch, int64_t heads, int64_t kv_heads, int64_t dim, int64_t max_places,
                                       size_t *bytes) {
    QMM_REQUIRE(bytes != nullptr, "qmm_paged_attention_workspace_size: no result given");
    QMM_REQUIRE(batch >= 0 && heads >= 0 && kv_heads >= 1 && dim >= 0 && max_places >= 0,
                "qmm_paged_attention_workspace_size: sizes must be non-negative");
    *bytes = qmm::paged::decode_workspace(batch, heads, kv_heads, dim);
    return QMM_OK;
}

int qmm_paged_attention(const void *query, int dtype, int64_t batch, int64_t heads, int64_t query_stride_token,
                        int64_t query_stride_head, const qmm_kv_cache *cache, const int32_t *block_table, int64_t table_stride,
                        int64_t max_pages, const int32_t *seq_lens, double scale_value, int64_t window, int64_t sinks, void *out,
                        float *lse, void *workspace, size_t workspace_bytes, void *stream) {
    qmm::paged::Problem p;
    const int rc = qmm::paged::describe(&p, "qmm_paged_attention", query, dtype, batch, heads, query_stride_token,
                                        query_stride_head, cache, block_table, table_stride, max_pages, seq_lens, batch,
                                        scale_value, window, sinks, out, lse);
    if (rc != QMM_OK) return rc;
    if (batch == 0 || heads == 0) return QMM_OK;
    return qmm::paged::launch_decode(p, dtype, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}

int qmm_paged_prompt_attention_workspace_size(int64_t tokens, int64_t batch, int64_t heads, int64_t kv_heads, int64_t dim,
                                              int64_t max_places, size_t *bytes) {
    QMM_REQUIRE(bytes != nullptr, "qmm_paged_prompt_attention_workspace_size: no result given");
    QMM_REQUIRE(tokens >= 0 && batch >= 0 && heads >= 0 && kv_heads >= 1 && dim >= 0 && max_places >= 0,
                "qmm_paged_prompt_attention_workspace_size: sizes must be non-negative");
    *bytes = qmm::paged::prompt_workspace(tokens, batch, heads, kv_heads, dim, max_places);
    return QMM_OK;
}

int qmm_paged_prompt_attention(const void *query, int dtype, int64_t tokens, int64_t heads, int64_t query_stride_token,
                               int64_t query_stride_head, const qmm_kv_cache *cache, const int32_t *block_table,
                               int64_t table_stride, int64_t max_pages, const int32_t *seq_lens, const int32_t *query_start,
                               int64_t batch, double scale_value, int64_t window, int64_t sinks, void *out, float *lse,
                               void *workspace, size_t workspace_bytes, void *stream) {
    qmm::paged::Problem p;
    const int rc = qmm::paged::describe(&p, "qmm_paged_prompt_attention", query, dtype, tokens, heads, query_stride_token,
                                        query_stride_head, cache, block_table, table_stride, max_pages, seq_lens, batch,
                                        scale_value, window, sinks, out, lse);
    if (rc != QMM_OK) return rc;
    QMM_REQUIRE(qmm::paged::words(query_start), "qmm_paged_prompt_attention: query_start must begin at 4-byte boundaries");
    p.start = query_start;
    if (tokens == 0 || heads == 0) return QMM_OK;
    return qmm::paged::launch_prompt(p, dtype, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}
}
