// npu_paged_cache_dequant: an int8 paged key-value cache read back into pages of another type.
#include "op_plugin/OpApiInterface.h"
#include "op_plugin/utils/paged_cache.h"

namespace op_api {

void npu_paged_cache_dequant(const at::Tensor &key_cache, const at::Tensor &value_cache, const at::Tensor &key_scale,
                             const at::Tensor &value_scale, const at::Tensor &block_table, const at::Tensor &seq_lens,
                             const at::Tensor &key_out, const at::Tensor &value_out, const at::Tensor &out_table,
                             const c10::optional<at::Tensor> &first_places)
{
    const char *op = "npu_paged_cache_dequant";
    TORCH_CHECK(key_cache.is_cuda(), op, " expects CUDA tensors, but key_cache is on ", key_cache.device());
    const c10::cuda::CUDAGuard guard(key_cache.device());
    const auto cache = op_plugin_utils::describe_quant_cache(op, key_cache, value_cache, key_scale, value_scale, key_cache);
    const auto type = key_out.scalar_type();
    TORCH_CHECK(type == at::kBFloat16 || type == at::kHalf || type == at::kFloat, op, ": unsupported dtype of key_out ", type);
    qmm_kv_cache out = op_plugin_utils::describe_pages(op, "key_out", key_out, "value_out", value_out, key_cache, type, "key_out");
    TORCH_CHECK(out.kv_heads == cache.codes.kv_heads && out.dim == cache.codes.dim, op, ": key_out should hold ", cache.codes.kv_heads,
                " heads of ", cache.codes.dim, ", but it is ", key_out.sizes());
    op_plugin_utils::check_written(op, {key_out, value_out});
    TORCH_CHECK(seq_lens.device() == key_cache.device() && seq_lens.dim() == 1 && seq_lens.scalar_type() == at::kInt, op,
                ": seq_lens should be int32 [batch] on ", key_cache.device(), ", but it is ", seq_lens.scalar_type(), " ", seq_lens.sizes(),
                " on ", seq_lens.device());
    const int64_t batch = seq_lens.size(0);
    for (const auto &t : {std::make_pair("block_table", &block_table), std::make_pair("out_table", &out_table)}) {
        TORCH_CHECK(t.second->device() == key_cache.device() && t.second->dim() == 2 && t.second->scalar_type() == at::kInt &&
                        t.second->size(0) == batch,
                    op, ": ", t.first, " should be int32 [", batch, ", pages] on ", key_cache.device(), ", but it is ",
                    t.second->scalar_type(), " ", t.second->sizes(), " on ", t.second->device());
    }
    at::Tensor first;
    if (first_places.has_value()) {
        TORCH_CHECK(first_places->device() == key_cache.device() && first_places->dim() == 1 && first_places->scalar_type() == at::kInt &&
                        first_places->size(0) == batch,
                    op, ": first_places should be int32 [", batch, "] on ", key_cache.device(), ", but it is ", first_places->scalar_type(),
                    " ", first_places->sizes(), " on ", first_places->device());
        first = first_places->contiguous();
    }
    const auto rows_dense = [](const at::Tensor &t) { return t.size(1) <= 1 || t.stride(1) == 1 ? t : t.contiguous(); };
    const at::Tensor from = rows_dense(block_table), to = rows_dense(out_table), lens = seq_lens.contiguous();
    // pages that share their storage with a lazy clone get their own, now that they are written
    out.key = key_out.mutable_data_ptr();
    out.value = value_out.mutable_data_ptr();
    EXEC_QMM_CMD(qmm_paged_cache_dequant, &cache.codes, &cache.scales, static_cast<const int32_t *>(from.const_data_ptr()), from.stride(0),
                 from.size(1), static_cast<const int32_t *>(lens.const_data_ptr()),
                 first.defined() ? static_cast<const int32_t *>(first.const_data_ptr()) : nullptr, batch, &out,
                 op_plugin_utils::qmm_dtype(type), static_cast<const int32_t *>(to.const_data_ptr()), to.stride(0), to.size(1),
                 op_plugin_utils::current_stream(key_cache));
}

}  // namespace op_api
