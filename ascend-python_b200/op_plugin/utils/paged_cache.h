// The paged key-value cache as the operators take it: checks and the C ABI's description.
#ifndef OP_PLUGIN_UTILS_PAGED_CACHE_H_
#define OP_PLUGIN_UTILS_PAGED_CACHE_H_

#include "op_plugin/utils/qmm_api_common.h"

namespace op_plugin_utils {

// The stride of a dimension, 0 where it has one element: what stands there then is no rule for alignment.
inline int64_t used_stride(const at::Tensor &t, int64_t dim) { return t.size(dim) == 1 ? 0 : t.stride(dim); }

// key_cache and value_cache of `op`: [pages, page size, heads, dim] of `dtype` on the device of `like`, dense in the last
// dimension.  A cache is never copied, so what the kernels cannot address is refused.
inline qmm_kv_cache describe_cache(const char *op, const at::Tensor &key_cache, const at::Tensor &value_cache, const at::Tensor &like)
{
    for (const auto &c : {std::make_pair("key_cache", &key_cache), std::make_pair("value_cache", &value_cache)}) {
        TORCH_CHECK(c.second->device() == like.device(), op, ": ", c.first, " should be on ", like.device(), ", but it is on ",
                    c.second->device());
        TORCH_CHECK(c.second->dim() == 4, op, ": ", c.first, " should be [pages, page size, heads, dim], but it has ", c.second->dim(),
                    " dimensions");
        TORCH_CHECK(c.second->scalar_type() == like.scalar_type(), op, ": ", c.first, " should have the dtype of the query (",
                    like.scalar_type(), "), but it is ", c.second->scalar_type());
        TORCH_CHECK(c.second->size(3) <= 1 || c.second->stride(3) == 1, op, ": the last dimension of ", c.first, " should be dense");
        TORCH_CHECK(c.second->size(1) > 0 && c.second->size(2) > 0 && c.second->size(3) > 0, op, ": ", c.first,
                    " should have places, heads and a dimension, but it is ", c.second->sizes());
    }
    TORCH_CHECK(key_cache.sizes() == value_cache.sizes(), op, ": key_cache and value_cache should have the same shape, but they are ",
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

// A [tokens, heads, dim] operand: as it is if its heads' rows are dense, else a dense copy.
inline at::Tensor dense_rows(const at::Tensor &x)
{
    return x.size(2) <= 1 || x.stride(2) == 1 ? x : x.contiguous();
}

}  // namespace op_plugin_utils

#endif  // OP_PLUGIN_UTILS_PAGED_CACHE_H_
