// npu_paged_attention, npu_paged_quant_attention and npu_paged_prompt_attention: attention over a paged key-value cache, of one new
// token a sequence (over a cache of its type or of int8) and of the last tokens of a ragged batch.  The
// reference's attention operators read dense caches; these take its conventions where they apply (scale_value, the fp32 statistic as
// a second output).
//
// The scratch is a tensor of the call, not a cached buffer: the kernels need nothing of it between calls, and graphs captured
// on one stream may then be replayed at the same time on several.
#include <cmath>

#include "op_plugin/OpApiInterface.h"
#include "op_plugin/utils/paged_cache.h"

namespace op_api {

namespace {

struct Attention {
    at::Tensor q, table, lens;
    double scale;
};

void check_query(const char *op, const at::Tensor &query, const at::Tensor &block_table, const at::Tensor &seq_lens)
{
    TORCH_CHECK(query.is_cuda(), op, " expects CUDA tensors, but query is on ", query.device());
    TORCH_CHECK(block_table.device() == query.device() && seq_lens.device() == query.device(), op, ": all tensors should be on ",
                query.device());
    TORCH_CHECK(query.scalar_type() == at::kBFloat16 || query.scalar_type() == at::kHalf, op,
                ": query should be bfloat16 or float16, but it is ", query.scalar_type());
    TORCH_CHECK(query.dim() == 3, op, ": query should be [tokens, heads, dim], but it has ", query.dim(), " dimensions");
}

Attention check_attention(const char *op, const at::Tensor &query, const qmm_kv_cache &cache, const at::Tensor &block_table,
                          const at::Tensor &seq_lens, c10::optional<double> scale_value, int64_t window, int64_t sinks)
{
    TORCH_CHECK(cache.dim == query.size(2), op, ": query and cache should have the same head dimension, but they have ",
                query.size(2), " and ", cache.dim);
    TORCH_CHECK(query.size(1) % cache.kv_heads == 0, op, ": the heads of query should be a multiple of the cache's, but they are ",
                query.size(1), " and ", cache.kv_heads);
    TORCH_CHECK(block_table.dim() == 2 && block_table.scalar_type() == at::kInt, op, ": block_table should be int32 [batch, pages], "
                "but it is ", block_table.scalar_type(), " ", block_table.sizes());
    TORCH_CHECK(seq_lens.dim() == 1 && seq_lens.scalar_type() == at::kInt && seq_lens.size(0) == block_table.size(0), op,
                ": seq_lens should be int32 [", block_table.size(0), "], but it is ", seq_lens.scalar_type(), " ", seq_lens.sizes());
    TORCH_CHECK(window >= 0 && sinks >= 0, op, ": window and sinks should not be negative, but they are ", window, " and ", sinks);
    TORCH_CHECK(window > 0 || sinks == 0, op, ": sinks have a meaning with a window only");
    Attention a;
    a.q = op_plugin_utils::dense_rows(query);
    if ((reinterpret_cast<uintptr_t>(a.q.const_data_ptr()) & 15) != 0 ||
        ((op_plugin_utils::used_stride(a.q, 0) | op_plugin_utils::used_stride(a.q, 1)) & 7) != 0) {
        a.q = a.q.is_contiguous() ? a.q.clone() : a.q.contiguous();  // the kernels read 16-byte vectors
    }
    a.table = block_table.size(1) <= 1 || block_table.stride(1) == 1 ? block_table : block_table.contiguous();
    a.lens = seq_lens.contiguous();
    a.scale = scale_value.has_value() ? *scale_value : 1.0 / std::sqrt(static_cast<double>(query.size(2)));
    return a;
}

}  // namespace

::std::tuple<at::Tensor, at::Tensor> npu_paged_attention(const at::Tensor &query, const at::Tensor &key_cache,
                                                         const at::Tensor &value_cache, const at::Tensor &block_table,
                                                         const at::Tensor &seq_lens, c10::optional<double> scale_value,
                                                         int64_t window, int64_t sinks)
{
    const char *op = "npu_paged_attention";
    c10::OptionalDeviceGuard guard;
    if (query.is_cuda()) guard.reset_device(query.device());
    check_query(op, query, block_table, seq_lens);
    const qmm_kv_cache cache = op_plugin_utils::describe_cache(op, key_cache, value_cache, query);
    const Attention a = check_attention(op, query, cache, block_table, seq_lens, scale_value, window, sinks);
    const int64_t batch = seq_lens.size(0), heads = query.size(1), dim = query.size(2), pages = block_table.size(1);
    TORCH_CHECK(query.size(0) == batch, op, ": query should have one token for each of ", batch, " sequences, but it is ",
                query.sizes());
    at::Tensor out = op_plugin_utils::empty_output(query.sizes(), query, query.scalar_type());
    at::Tensor lse = op_plugin_utils::empty_output({batch, heads}, query, at::kFloat);
    size_t bytes = 0;
    EXEC_QMM_CMD(qmm_paged_attention_workspace_size, batch, heads, cache.kv_heads, dim, pages * cache.page_size, &bytes);
    at::Tensor workspace;
    if (bytes > 0) workspace = op_plugin_utils::empty_output({static_cast<int64_t>(bytes)}, query, at::kByte);
    EXEC_QMM_CMD(qmm_paged_attention, a.q.const_data_ptr(), op_plugin_utils::qmm_dtype(query.scalar_type()), batch, heads,
                 op_plugin_utils::used_stride(a.q, 0), op_plugin_utils::used_stride(a.q, 1), &cache, static_cast<const int32_t *>(a.table.const_data_ptr()), a.table.stride(0),
                 pages, static_cast<const int32_t *>(a.lens.const_data_ptr()), a.scale, window, sinks, out.data_ptr(),
                 static_cast<float *>(lse.data_ptr()), bytes > 0 ? workspace.data_ptr() : nullptr, bytes,
                 op_plugin_utils::current_stream(query));
    return ::std::tuple<at::Tensor, at::Tensor>(out, lse);
}

::std::tuple<at::Tensor, at::Tensor> npu_paged_quant_attention(const at::Tensor &query, const at::Tensor &key_cache,
                                                               const at::Tensor &value_cache, const at::Tensor &key_scale,
                                                               const at::Tensor &value_scale, const at::Tensor &block_table,
                                                               const at::Tensor &seq_lens, c10::optional<double> scale_value,
                                                               int64_t window, int64_t sinks)
{
    const char *op = "npu_paged_quant_attention";
    c10::OptionalDeviceGuard guard;
    if (query.is_cuda()) guard.reset_device(query.device());
    check_query(op, query, block_table, seq_lens);
    const auto cache = op_plugin_utils::describe_quant_cache(op, key_cache, value_cache, key_scale, value_scale, query);
    const Attention a = check_attention(op, query, cache.codes, block_table, seq_lens, scale_value, window, sinks);
    const int64_t batch = seq_lens.size(0), heads = query.size(1), dim = query.size(2), pages = block_table.size(1);
    TORCH_CHECK(query.size(0) == batch, op, ": query should have one token for each of ", batch, " sequences, but it is ",
                query.sizes());
    at::Tensor out = op_plugin_utils::empty_output(query.sizes(), query, query.scalar_type());
    at::Tensor lse = op_plugin_utils::empty_output({batch, heads}, query, at::kFloat);
    size_t bytes = 0;
    EXEC_QMM_CMD(qmm_paged_quant_attention_workspace_size, batch, heads, cache.codes.kv_heads, dim, pages * cache.codes.page_size, &bytes);
    at::Tensor workspace;
    if (bytes > 0) workspace = op_plugin_utils::empty_output({static_cast<int64_t>(bytes)}, query, at::kByte);
    EXEC_QMM_CMD(qmm_paged_quant_attention, a.q.const_data_ptr(), op_plugin_utils::qmm_dtype(query.scalar_type()), batch, heads,
                 op_plugin_utils::used_stride(a.q, 0), op_plugin_utils::used_stride(a.q, 1), &cache.codes, &cache.scales,
                 static_cast<const int32_t *>(a.table.const_data_ptr()), a.table.stride(0), pages,
                 static_cast<const int32_t *>(a.lens.const_data_ptr()), a.scale, window, sinks, out.data_ptr(),
                 static_cast<float *>(lse.data_ptr()), bytes > 0 ? workspace.data_ptr() : nullptr, bytes,
                 op_plugin_utils::current_stream(query));
    return ::std::tuple<at::Tensor, at::Tensor>(out, lse);
}

::std::tuple<at::Tensor, at::Tensor> npu_paged_prompt_attention(const at::Tensor &query, const at::Tensor &key_cache,
                                                                const at::Tensor &value_cache, const at::Tensor &block_table,
                                                                const at::Tensor &seq_lens, const at::Tensor &query_start,
                                                                c10::optional<double> scale_value, int64_t window, int64_t sinks)
{
    const char *op = "npu_paged_prompt_attention";
    c10::OptionalDeviceGuard guard;
    if (query.is_cuda()) guard.reset_device(query.device());
    check_query(op, query, block_table, seq_lens);
    const qmm_kv_cache cache = op_plugin_utils::describe_cache(op, key_cache, value_cache, query);
    const Attention a = check_attention(op, query, cache, block_table, seq_lens, scale_value, window, sinks);
    const int64_t tokens = query.size(0), heads = query.size(1), dim = query.size(2), pages = block_table.size(1);
    const int64_t batch = seq_lens.size(0);
    TORCH_CHECK(query_start.device() == query.device(), op, ": all tensors should be on ", query.device());
    TORCH_CHECK(query_start.dim() == 1 && query_start.scalar_type() == at::kInt && query_start.size(0) == batch + 1, op,
                ": query_start should be int32 [", batch + 1, "], but it is ", query_start.scalar_type(), " ", query_start.sizes());
    const at::Tensor start = query_start.contiguous();
    at::Tensor out = op_plugin_utils::empty_output(query.sizes(), query, query.scalar_type());
    at::Tensor lse = op_plugin_utils::empty_output({tokens, heads}, query, at::kFloat);
    size_t bytes = 0;
    EXEC_QMM_CMD(qmm_paged_prompt_attention_workspace_size, tokens, batch, heads, cache.kv_heads, dim, pages * cache.page_size,
                 &bytes);
    at::Tensor workspace;
    if (bytes > 0) workspace = op_plugin_utils::empty_output({static_cast<int64_t>(bytes)}, query, at::kByte);
    EXEC_QMM_CMD(qmm_paged_prompt_attention, a.q.const_data_ptr(), op_plugin_utils::qmm_dtype(query.scalar_type()), tokens, heads,
                 op_plugin_utils::used_stride(a.q, 0), op_plugin_utils::used_stride(a.q, 1), &cache, static_cast<const int32_t *>(a.table.const_data_ptr()), a.table.stride(0),
                 pages, static_cast<const int32_t *>(a.lens.const_data_ptr()), static_cast<const int32_t *>(start.const_data_ptr()),
                 batch, a.scale, window, sinks, out.data_ptr(), static_cast<float *>(lse.data_ptr()),
                 bytes > 0 ? workspace.data_ptr() : nullptr, bytes, op_plugin_utils::current_stream(query));
    return ::std::tuple<at::Tensor, at::Tensor>(out, lse);
}

}  // namespace op_api
