// The paged key-value cache as the operators take it: checks and the C ABI's description.
#ifndef OP_PLUGIN_UTILS_PAGED_CACHE_H_
#define OP_PLUGIN_UTILS_PAGED_CACHE_H_

#include "op_plugin/utils/qmm_api_common.h"

namespace op_plugin_utils {

// The stride of a dimension, 0 where it has one element: what stands there then is no rule for alignment.
inline int64_t used_stride(const at::Tensor &t, int64_t dim) { return t.size(dim) == 1 ? 0 : t.stride(dim); }

// A cache's keys and values, operands `key_name` and `value_name` of `op`: [pages, page size, heads, dim] of `dtype` (`whose`: why that one) on
// the device of `like`, dense in the last dimension.  A cache is never copied, so what the kernels cannot address is refused.
inline qmm_kv_cache describe_pages(const char *op, const char *key_name, const at::Tensor &key_cache, const char *value_name,
                                   const at::Tensor &value_cache, const at::Tensor &like, at::ScalarType dtype, const char *whose)
{
    for (const auto &c : {std::make_pair(key_name, &key_cache), std::make_pair(value_name, &value_cache)}) {
        TORCH_CHECK(c.second->device() == like.device(), op, ": ", c.first, " should be on ", like.device(), ", but it is on ",
                    c.second->device());
        TORCH_CHECK(c.second->dim() == 4, op, ": ", c.first, " should be [pages, page size, heads, dim], but it has ", c.second->dim(),
                    " dimensions");
        TORCH_CHECK(c.second->scalar_type() == dtype, op, ": ", c.first, " should have the dtype of ", whose, " (", dtype, "), but it is ",
                    c.second->scalar_type());
        TORCH_CHECK(c.second->size(3) <= 1 || c.second->stride(3) == 1, op, ": the last dimension of ", c.first, " should be dense");
        TORCH_CHECK(c.second->size(1) > 0 && c.second->size(2) > 0 && c.second->size(3) > 0, op, ": ", c.first,
                    " should have places, heads and a dimension, but it is ", c.second->sizes());
    }
    TORCH_CHECK(key_cache.sizes() == value_cache.sizes(), op, ": ", key_name, " and ", value_name, " should have the same shape, but they are ",
                key_cache.sizes(), " and ", value_cache.sizes());
    qmm_kv_cache c;
    c.key = key_cache.const_data_ptr();
    c.value = value_cache.const_data_ptr();
    c.pages = key_cache.size(0);
    c.page_size = key_cache.size(1);
    c.kv_heads = key_cache.size(2);
    c.dim = key_cache.size(3);
    c.key_stride_page = used_stride(key_cache, 0);
    c.key_stride_place = used_stride(key_cache, 1);
    c.key_stride_head = used_stride(key_cache, 2);
    c.value_stride_page = used_stride(value_cache, 0);
    c.value_stride_place = used_stride(value_cache, 1);
    c.value_stride_head = used_stride(value_cache, 2);
    return c;
}

// A cache of the query's type.
inline qmm_kv_cache describe_cache(const char *op, const at::Tensor &key_cache, const at::Tensor &value_cache, const at::Tensor &like)
{
    return describe_pages(op, "key_cache", key_cache, "value_cache", value_cache, like, like.scalar_type(), "the query");
}

// An int8 cache with its scales, fp32 [pages, heads, page size].
struct QuantCache {
    qmm_kv_cache codes;
    qmm_kv_scales scales;
};
inline QuantCache describe_quant_cache(const char *op, const at::Tensor &key_cache, const at::Tensor &value_cache,
                                       const at::Tensor &key_scale, const at::Tensor &value_scale, const at::Tensor &like)
{
    QuantCache c;
    c.codes = describe_pages(op, "key_cache", key_cache, "value_cache", value_cache, like, at::kChar, "a quantized cache");
    for (const auto &s : {std::make_pair("key_scale", &key_scale), std::make_pair("value_scale", &value_scale)}) {
        TORCH_CHECK(s.second->device() == like.device(), op, ": ", s.first, " should be on ", like.device(), ", but it is on ",
                    s.second->device());
        TORCH_CHECK(s.second->scalar_type() == at::kFloat && s.second->dim() == 3 && s.second->size(0) == key_cache.size(0) &&
                        s.second->size(1) == key_cache.size(2) && s.second->size(2) == key_cache.size(1),
                    op, ": ", s.first, " should be float32 [", key_cache.size(0), ", ", key_cache.size(2), ", ", key_cache.size(1),
                    "] (pages, heads, page size), but it is ", s.second->scalar_type(), " ", s.second->sizes());
    }
    c.scales.key = static_cast<const float *>(key_scale.const_data_ptr());
    c.scales.value = static_cast<const float *>(value_scale.const_data_ptr());
    c.scales.key_stride_page = used_stride(key_scale, 0);
    c.scales.key_stride_head = used_stride(key_scale, 1);
    c.scales.key_stride_place = used_stride(key_scale, 2);
    c.scales.value_stride_page = used_stride(value_scale, 0);
    c.scales.value_stride_head = used_stride(value_scale, 1);
    c.scales.value_stride_place = used_stride(value_scale, 2);
    return c;
}

// Refuses tensors that are written and whose elements share places.
inline void check_written(const char *op, at::TensorList written)
{
    for (const auto &c : written) {
        for (int64_t d = 0; d + (c.dim() == 4 ? 1 : 0) < c.dim(); ++d) {
            TORCH_CHECK(c.size(d) == 1 || c.stride(d) != 0, op, ": the places of a cache that is written should not overlap, but its strides are ",
                        c.strides());
        }
    }
}

// A [tokens, heads, dim] operand: as it is if its heads' rows are dense, else a dense copy.
inline at::Tensor dense_rows(const at::Tensor &x)
{
    return x.size(2) <= 1 || x.stride(2) == 1 ? x : x.contiguous();
}

}  // namespace op_plugin_utils

#endif  // OP_PLUGIN_UTILS_PAGED_CACHE_H_
