// npu_rotary_axes, npu_rotary_axes_cache and npu_rotary_axes_quant_cache: rotary positions on one or several axes, and the same with
// the write of keys and values into a paged cache of their type or of int8.  They have no counterpart in the reference; host conventions are those of npu_rms_norm and its
// fusion (RmsNormKernelNpuOpApi.cpp): dense outputs with the input's options, strided inputs taken as they are.
#include "op_plugin/OpApiInterface.h"
#include "op_plugin/utils/paged_cache.h"

namespace op_api {

namespace {

struct Rotary {
    at::Tensor q, k, positions, inv_freq;
    int64_t tokens, axes, position_stride_axis, position_stride_token;
    int interleaved, cyclic, position_dtype;
    std::vector<int64_t> sections;
};

int index_dtype(const char *op, const char *name, const at::Tensor &t)
{
    TORCH_CHECK(t.scalar_type() == at::kInt || t.scalar_type() == at::kLong, op, ": ", name, " should be int32 or int64, but it is ",
                t.scalar_type());
    return t.scalar_type() == at::kInt ? QMM_DTYPE_I32 : QMM_DTYPE_I64;
}

Rotary check_rotary(const char *op, const at::Tensor &query, const at::Tensor &key, const at::Tensor &positions,
                    const at::Tensor &inv_freq, at::IntArrayRef sections, c10::string_view rotary_mode, c10::string_view axis_order)
{
    TORCH_CHECK(query.is_cuda(), op, " expects CUDA tensors, but query is on ", query.device());
    TORCH_CHECK(key.device() == query.device() && positions.device() == query.device() && inv_freq.device() == query.device(), op,
                ": all tensors should be on ", query.device());
    const auto t = query.scalar_type();
    TORCH_CHECK(t == at::kBFloat16 || t == at::kHalf || t == at::kFloat, op, ": unsupported dtype ", t);
    TORCH_CHECK(key.scalar_type() == t, op, ": key should have the dtype of query (", t, "), but it is ", key.scalar_type());
    TORCH_CHECK(query.dim() == 3 && key.dim() == 3 && query.size(0) == key.size(0) && query.size(2) == key.size(2), op,
                ": query and key should be [tokens, heads, dim] with the same tokens and dim, but they are ", query.sizes(), " and ",
                key.sizes());
    TORCH_CHECK(inv_freq.dim() == 1 && inv_freq.scalar_type() == at::kFloat, op, ": inv_freq should be a float32 vector, but it is ",
                inv_freq.scalar_type(), " ", inv_freq.sizes());
    TORCH_CHECK(rotary_mode == "half" || rotary_mode == "interleave", op, ": rotary_mode should be 'half' or 'interleave', but it is '",
                rotary_mode, "'");
    TORCH_CHECK(axis_order == "blocked" || axis_order == "cyclic", op, ": axis_order should be 'blocked' or 'cyclic', but it is '",
                axis_order, "'");
    Rotary r;
    r.position_dtype = index_dtype(op, "positions", positions);
    TORCH_CHECK(positions.dim() == 1 || positions.dim() == 2, op, ": positions should be [axes, tokens] or [tokens], but they are ",
                positions.sizes());
    r.axes = positions.dim() == 1 ? 1 : positions.size(0);
    r.tokens = query.size(0);
    TORCH_CHECK(positions.size(-1) == r.tokens, op, ": positions should hold ", r.tokens, " tokens, but they are ", positions.sizes());
    r.sections = sections.vec();
    if (r.sections.empty() && r.axes == 1) {
        r.sections.push_back(inv_freq.numel());
    }
    TORCH_CHECK(static_cast<int64_t>(r.sections.size()) == r.axes, op, ": sections should have one entry for each of ", r.axes,
                " axes, but they are ", sections);
    r.q = op_plugin_utils::dense_rows(query);
    r.k = op_plugin_utils::dense_rows(key);
    r.positions = positions;
    r.inv_freq = inv_freq.contiguous();
    r.position_stride_axis = positions.dim() == 1 ? 0 : positions.stride(0);
    r.position_stride_token = positions.stride(-1);
    r.interleaved = rotary_mode == "interleave";
    r.cyclic = axis_order == "cyclic";
    return r;
}

}  // namespace

::std::tuple<at::Tensor, at::Tensor> npu_rotary_axes(const at::Tensor &query, const at::Tensor &key, const at::Tensor &positions,
                                                     const at::Tensor &inv_freq, at::IntArrayRef sections,
                                                     c10::string_view rotary_mode, c10::string_view axis_order)
{
    c10::OptionalDeviceGuard guard;
    if (query.is_cuda()) guard.reset_device(query.device());
    const Rotary r = check_rotary("npu_rotary_axes", query, key, positions, inv_freq, sections, rotary_mode, axis_order);
    at::Tensor q = op_plugin_utils::empty_output(query.sizes(), query, query.scalar_type());
    at::Tensor k = op_plugin_utils::empty_output(key.sizes(), key, key.scalar_type());
    EXEC_QMM_CMD(qmm_rotary_axes, r.q.const_data_ptr(), r.q.stride(0), r.q.stride(1), r.k.const_data_ptr(), r.k.stride(0),
                 r.k.stride(1), op_plugin_utils::qmm_dtype(query.scalar_type()), r.tokens, query.size(1), key.size(1), query.size(2),
                 r.positions.const_data_ptr(), r.position_dtype, r.position_stride_axis, r.position_stride_token,
                 static_cast<const float *>(r.inv_freq.const_data_ptr()), r.inv_freq.numel(), r.sections.data(), r.axes,
                 r.interleaved, r.cyclic, q.data_ptr(), k.data_ptr(), op_plugin_utils::current_stream(query));
    return ::std::tuple<at::Tensor, at::Tensor>(q, k);
}

at::Tensor npu_rotary_axes_cache(const at::Tensor &query, const at::Tensor &key, const at::Tensor &value,
                                 const at::Tensor &positions, const at::Tensor &inv_freq, const at::Tensor &key_cache,
                                 const at::Tensor &value_cache, const at::Tensor &slots, at::IntArrayRef sections,
                                 c10::string_view rotary_mode, c10::string_view axis_order)
{
    const char *op = "npu_rotary_axes_cache";
    c10::OptionalDeviceGuard guard;
    if (query.is_cuda()) guard.reset_device(query.device());
    const Rotary r = check_rotary(op, query, key, positions, inv_freq, sections, rotary_mode, axis_order);
    TORCH_CHECK(value.device() == query.device() && slots.device() == query.device(), op, ": all tensors should be on ", query.device());
    TORCH_CHECK(value.scalar_type() == query.scalar_type() && value.sizes() == key.sizes(), op,
                ": value should have dtype and shape of key (", key.scalar_type(), " ", key.sizes(), "), but it is ",
                value.scalar_type(), " ", value.sizes());
    qmm_kv_cache cache = op_plugin_utils::describe_cache(op, key_cache, value_cache, query);
    TORCH_CHECK(cache.kv_heads == key.size(1) && cache.dim == key.size(2), op, ": the cache should hold ", key.size(1), " heads of ",
                key.size(2), ", but it is ", key_cache.sizes());
    op_plugin_utils::check_written(op, {key_cache, value_cache});
    const int slot_dtype = index_dtype(op, "slots", slots);
    TORCH_CHECK(slots.dim() == 1 && slots.size(0) == r.tokens, op, ": slots should hold ", r.tokens, " tokens, but they are ",
                slots.sizes());
    const at::Tensor v = op_plugin_utils::dense_rows(value);
    // a cache that shares its storage with a lazy clone gets its own, now that it is written
    cache.key = key_cache.mutable_data_ptr();
    cache.value = value_cache.mutable_data_ptr();
    at::Tensor q = op_plugin_utils::empty_output(query.sizes(), query, query.scalar_type());
    EXEC_QMM_CMD(qmm_rotary_axes_cache, r.q.const_data_ptr(), r.q.stride(0), r.q.stride(1), r.k.const_data_ptr(), r.k.stride(0),
                 r.k.stride(1), v.const_data_ptr(), v.stride(0), v.stride(1), op_plugin_utils::qmm_dtype(query.scalar_type()),
                 r.tokens, query.size(1), r.positions.const_data_ptr(), r.position_dtype, r.position_stride_axis,
                 r.position_stride_token, static_cast<const float *>(r.inv_freq.const_data_ptr()), r.inv_freq.numel(),
                 r.sections.data(), r.axes, r.interleaved, r.cyclic, &cache, slots.const_data_ptr(), slot_dtype, slots.stride(0),
                 q.data_ptr(), op_plugin_utils::current_stream(query));
    return q;
}

at::Tensor npu_rotary_axes_quant_cache(const at::Tensor &query, const at::Tensor &key, const at::Tensor &value,
                                       const at::Tensor &positions, const at::Tensor &inv_freq, const at::Tensor &key_cache,
                                       const at::Tensor &value_cache, const at::Tensor &key_scale, const at::Tensor &value_scale,
                                       const at::Tensor &slots, at::IntArrayRef sections, c10::string_view rotary_mode,
                                       c10::string_view axis_order)
{
    const char *op = "npu_rotary_axes_quant_cache";
    c10::OptionalDeviceGuard guard;
    if (query.is_cuda()) guard.reset_device(query.device());
    const Rotary r = check_rotary(op, query, key, positions, inv_freq, sections, rotary_mode, axis_order);
    TORCH_CHECK(value.device() == query.device() && slots.device() == query.device(), op, ": all tensors should be on ", query.device());
    TORCH_CHECK(value.scalar_type() == query.scalar_type() && value.sizes() == key.sizes(), op,
                ": value should have dtype and shape of key (", key.scalar_type(), " ", key.sizes(), "), but it is ",
                value.scalar_type(), " ", value.sizes());
    op_plugin_utils::QuantCache cache = op_plugin_utils::describe_quant_cache(op, key_cache, value_cache, key_scale, value_scale, query);
    TORCH_CHECK(cache.codes.kv_heads == key.size(1) && cache.codes.dim == key.size(2), op, ": the cache should hold ", key.size(1),
                " heads of ", key.size(2), ", but it is ", key_cache.sizes());
    op_plugin_utils::check_written(op, {key_cache, value_cache, key_scale, value_scale});
    const int slot_dtype = index_dtype(op, "slots", slots);
    TORCH_CHECK(slots.dim() == 1 && slots.size(0) == r.tokens, op, ": slots should hold ", r.tokens, " tokens, but they are ",
                slots.sizes());
    const at::Tensor v = op_plugin_utils::dense_rows(value);
    // a cache that shares its storage with a lazy clone gets its own, now that it is written
    cache.codes.key = key_cache.mutable_data_ptr();
    cache.codes.value = value_cache.mutable_data_ptr();
    cache.scales.key = static_cast<const float *>(key_scale.mutable_data_ptr());
    cache.scales.value = static_cast<const float *>(value_scale.mutable_data_ptr());
    at::Tensor q = op_plugin_utils::empty_output(query.sizes(), query, query.scalar_type());
    EXEC_QMM_CMD(qmm_rotary_axes_quant_cache, r.q.const_data_ptr(), r.q.stride(0), r.q.stride(1), r.k.const_data_ptr(), r.k.stride(0),
                 r.k.stride(1), v.const_data_ptr(), v.stride(0), v.stride(1), op_plugin_utils::qmm_dtype(query.scalar_type()),
                 r.tokens, query.size(1), r.positions.const_data_ptr(), r.position_dtype, r.position_stride_axis,
                 r.position_stride_token, static_cast<const float *>(r.inv_freq.const_data_ptr()), r.inv_freq.numel(),
                 r.sections.data(), r.axes, r.interleaved, r.cyclic, &cache.codes, &cache.scales, slots.const_data_ptr(), slot_dtype,
                 slots.stride(0), q.data_ptr(), op_plugin_utils::current_stream(query));
    return q;
}

}  // namespace op_api
