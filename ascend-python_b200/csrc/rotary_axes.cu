// Rotary positions on several axes (npu_rotary_axes) and the same with the write into a paged key-value cache
// (npu_rotary_axes_cache).
//
// The first 2n elements of every head of the query and the key are n pairs; pair i turns by the angle
//     position[axis(i)] * inv_freq[i]
// where text has one axis and images and video have several (time, height, width).  axis(i) goes by the sections: blocked,
// sections[0] pairs on axis 0, then sections[1] on axis 1, ...; cyclic, pair i is on axis a = i mod axes while i < axes *
// sections[a], else on axis 0.  Pairs are (i, i + n) or, interleaved, (2i, 2i + 1).  Elements behind 2n are copied.
//
// Far positions: a position of 2^17 times a frequency of 1, rounded to 32 bits, is off by up to 2^-8.  The angle is therefore
// made in 64 bits, in half turns, reduced to [-1, 1] there, and only then rounded for sincospif (off by 2^-25 half turns).
// The rotation is fp32 with one rounding to the tensors' type at the end.
//
// Every element is read and written once.  One CTA a token: n of its threads make the token's sines and cosines, which all heads
// share, in shared memory.
#include "qmm_common.cuh"

namespace qmm {

namespace {

constexpr int kThreads = 256;
constexpr int kMostPairs = 128;  // head dimension <= 256
constexpr int kMostAxes = 8;

struct RotaryParams {
    const void *q, *k, *v;
    int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh;
    const void *positions;  // [axes][tokens], axes pos_sa elements apart, tokens pos_st
    int64_t pos_sa, pos_st;
    const float *inv_freq;
    void *q_out, *k_out;            // dense [tokens][heads][dim]; k_out: without a cache
    void *k_cache, *v_cache;
    int64_t kc_sb, kc_st, kc_sh, vc_sb, vc_st, vc_sh;
    const void *slots;
    int64_t slot_st;
    int64_t places;  // pages * page size
    int page;
    int heads, kv_heads, dim, pairs, axes;
    int wide_positions, wide_slots, interleaved, cyclic, cached;
    int sections[kMostAxes];
};

__device__ __forceinline__ int axis_of(const RotaryParams &p, int i) {
    if (p.cyclic) {
        const int a = i % p.axes;
        return i < p.axes * p.sections[a] ? a : 0;
    }
    int a = 0;
    for (int end = p.sections[0]; a + 1 < p.axes && i >= end; end += p.sections[a]) ++a;
    return a;
}

__device__ __forceinline__ int64_t load_index(const void *base, int64_t at, int wide) {
    return wide ? __ldg(static_cast<const long long *>(base) + at) : __ldg(static_cast<const int *>(base) + at);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const __grid_constant__ RotaryParams p) {
    __shared__ float s_cos[kMostPairs], s_sin[kMostPairs];
    pdl_launch_dependents();
    pdl_wait();
    const int64_t token = blockIdx.x;
    for (int i = threadIdx.x; i < p.pairs; i += kThreads) {
        const int64_t place = load_index(p.positions, axis_of(p, i) * p.pos_sa + token * p.pos_st, p.wide_positions);
        const double half_turns = static_cast<double>(place) * static_cast<double>(__ldg(p.inv_freq + i)) * 0.31830988618379067154;
        float s, c;
        sincospif(static_cast<float>(half_turns - 2.0 * rint(0.5 * half_turns)), &s, &c);
        s_sin[i] = s;
        s_cos[i] = c;
    }
    __syncthreads();
    int64_t slot = 0, block = 0, at = 0;
    bool write = true;
    if (p.cached) {
        slot = load_index(p.slots, token * p.slot_st, p.wide_slots);
        write = slot >= 0 && slot < p.places;
        block = write ? slot / p.page : 0;
        at = write ? slot - block * p.page : 0;
    }
    const int total = (p.heads + p.kv_heads * (p.cached ? 2 : 1)) * p.dim;
    for (int item = threadIdx.x; item < total; item += kThreads) {
        const int row = item / p.dim, e = item - row * p.dim;
        const int kind = row < p.heads ? 0 : row < p.heads + p.kv_heads ? 1 : 2;
        const int head = kind == 0 ? row : kind == 1 ? row - p.heads : row - p.heads - p.kv_heads;
        if (kind > 0 && !write) break;
        const T *src = kind == 0   ? static_cast<const T *>(p.q) + token * p.q_st + head * p.q_sh
                       : kind == 1 ? static_cast<const T *>(p.k) + token * p.k_st + head * p.k_sh
                                   : static_cast<const T *>(p.v) + token * p.v_st + head * p.v_sh;
        T *dst;
        if (kind == 0)
            dst = static_cast<T *>(p.q_out) + (token * p.heads + head) * p.dim;
        else if (!p.cached)
            dst = static_cast<T *>(p.k_out) + (token * p.kv_heads + head) * p.dim;
        else if (kind == 1)
            dst = static_cast<T *>(p.k_cache) + block * p.kc_sb + at * p.kc_st + head * p.kc_sh;
        else
            dst = static_cast<T *>(p.v_cache) + block * p.vc_sb + at * p.vc_st + head * p.vc_sh;
        if (kind == 2 || e >= 2 * p.pairs) {
            dst[e] = src[e];
            continue;
        }
        const int i = p.interleaved ? e >> 1 : e < p.pairs ? e : e - p.pairs;
        const bool second = p.interleaved ? (e & 1) != 0 : e >= p.pairs;
        const float a = to_float(src[p.interleaved ? 2 * i : i]), b = to_float(src[p.interleaved ? 2 * i + 1 : i + p.pairs]);
        dst[e] = from_float<T>(second ? fmaf(b, s_cos[i], a * s_sin[i]) : fmaf(a, s_cos[i], -(b * s_sin[i])));
    }
}

template <typename T>
int launch_rotary(const RotaryParams &p, int64_t tokens, cudaStream_t stream) {
    QMM_CUDA_OK(launch_pdl(rotary_kernel<T>, dim3(static_cast<unsigned>(tokens)), dim3(kThreads), 0, stream, p));
    return QMM_OK;
}

int rotary(const char *op, RotaryParams &p, int dtype, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t dim,
           int64_t pairs, const int64_t *sections, int64_t axes, int position_dtype, cudaStream_t stream) {
    const std::string name(op);
    QMM_REQUIRE(tokens >= 0 && heads >= 0 && kv_heads >= 0 && dim >= 0, name + ": sizes must be non-negative");
    QMM_REQUIRE(tokens <= 0x7fffffff && heads <= 65535 && kv_heads <= 65535, name + ": sizes out of range");
    QMM_REQUIRE(dim <= 256, name + ": the head dimension must not be above 256");
    QMM_REQUIRE(pairs >= 0 && 2 * pairs <= dim, name + ": more frequencies than pairs of a head");
    QMM_REQUIRE(axes >= 1 && axes <= kMostAxes, name + ": between 1 and 8 axes");
    QMM_REQUIRE(position_dtype == QMM_DTYPE_I32 || position_dtype == QMM_DTYPE_I64, name + ": positions must be int32 or int64");
    int64_t sum = 0;
    for (int a = 0; a < axes; ++a) {
        QMM_REQUIRE(sections[a] >= 0 && sections[a] <= pairs, name + ": sections must be between 0 and the number of frequencies");
        p.sections[a] = static_cast<int>(sections[a]);
        sum += sections[a];
    }
    QMM_REQUIRE(sum == pairs, name + ": the sections must add up to the number of frequencies");
    if (p.cyclic)
        for (int a = 1; a < axes; ++a)
            QMM_REQUIRE(sections[a] == 0 || a + axes * (sections[a] - 1) < pairs,
                        name + ": cyclic sections: axis 0 has too few frequencies for the others to take turns with it");
    p.heads = static_cast<int>(heads);
    p.kv_heads = static_cast<int>(kv_heads);
    p.dim = static_cast<int>(dim);
    p.pairs = static_cast<int>(pairs);
    p.axes = static_cast<int>(axes);
    p.wide_positions = position_dtype == QMM_DTYPE_I64;
    if (tokens == 0 || dim == 0) return QMM_OK;
    if (dtype == QMM_DTYPE_BF16) return launch_rotary<__nv_bfloat16>(p, tokens, stream);
    if (dtype == QMM_DTYPE_F16) return launch_rotary<__half>(p, tokens, stream);
    if (dtype == QMM_DTYPE_F32) return launch_rotary<float>(p, tokens, stream);
    return fail(QMM_ERR_INVALID_ARGUMENT, name + ": the tensors must be bf16, f16 or f32");
}

}  // namespace

}  // namespace qmm

using qmm::fail;

extern "C" {

int qmm_rotary_axes(const void *query, int64_t query_stride_token, int64_t query_stride_head, const void *key,
                    int64_t key_stride_token, int64_t key_stride_head, int dtype, int64_t tokens, int64_t heads, int64_t kv_heads,
                    int64_t dim, const void *positions, int position_dtype, int64_t position_stride_axis,
                    int64_t position_stride_token, const float *inv_freq, int64_t pairs, const int64_t *sections, int64_t axes,
                    int interleaved, int cyclic, void *query_out, void *key_out, void *stream) {
    qmm::RotaryParams p = {};
    p.q = query;
    p.q_st = query_stride_token;
    p.q_sh = query_stride_head;
    p.k = key;
    p.k_st = key_stride_token;
    p.k_sh = key_stride_head;
    p.positions = positions;
    p.pos_sa = position_stride_axis;
    p.pos_st = position_stride_token;
    p.inv_freq = inv_freq;
    p.q_out = query_out;
    p.k_out = key_out;
    p.interleaved = interleaved != 0;
    p.cyclic = cyclic != 0;
    return qmm::rotary("qmm_rotary_axes", p, dtype, tokens, heads, kv_heads, dim, pairs, sections, axes, position_dtype,
                       static_cast<cudaStream_t>(stream));
}

int qmm_rotary_axes_cache(const void *query, int64_t query_stride_token, int64_t query_stride_head, const void *key,
                          int64_t key_stride_token, int64_t key_stride_head, const void *value, int64_t value_stride_token,
                          int64_t value_stride_head, int dtype, int64_t tokens, int64_t heads, const void *positions,
                          int position_dtype, int64_t position_stride_axis, int64_t position_stride_token, const float *inv_freq,
                          int64_t pairs, const int64_t *sections, int64_t axes, int interleaved, int cyclic,
                          const qmm_kv_cache *cache, const void *slots, int slot_dtype, int64_t slot_stride, void *query_out,
                          void *stream) {
    qmm::RotaryParams p = {};
    QMM_REQUIRE(cache != nullptr, "qmm_rotary_axes_cache: no cache given");
    QMM_REQUIRE(cache->pages >= 0 && cache->page_size >= 1 && cache->pages <= 0x7fffffff && cache->page_size <= 0x7fffffff,
                "qmm_rotary_axes_cache: pages must be non-negative, their size positive");
    QMM_REQUIRE(slot_dtype == QMM_DTYPE_I32 || slot_dtype == QMM_DTYPE_I64, "qmm_rotary_axes_cache: slots must be int32 or int64");
    p.q = query;
    p.q_st = query_stride_token;
    p.q_sh = query_stride_head;
    p.k = key;
    p.k_st = key_stride_token;
    p.k_sh = key_stride_head;
    p.v = value;
    p.v_st = value_stride_token;
    p.v_sh = value_stride_head;
    p.positions = positions;
    p.pos_sa = position_stride_axis;
    p.pos_st = position_stride_token;
    p.inv_freq = inv_freq;
    p.q_out = query_out;
    p.interleaved = interleaved != 0;
    p.cyclic = cyclic != 0;
    p.cached = 1;
    p.k_cache = const_cast<void *>(cache->key);
    p.v_cache = const_cast<void *>(cache->value);
    p.kc_sb = cache->key_stride_page;
    p.kc_st = cache->key_stride_place;
    p.kc_sh = cache->key_stride_head;
    p.vc_sb = cache->value_stride_page;
    p.vc_st = cache->value_stride_place;
    p.vc_sh = cache->value_stride_head;
    p.slots = slots;
    p.slot_st = slot_stride;
    p.places = cache->pages * cache->page_size;
    p.page = static_cast<int>(cache->page_size);
    p.wide_slots = slot_dtype == QMM_DTYPE_I64;
    return qmm::rotary("qmm_rotary_axes_cache", p, dtype, tokens, heads, cache->kv_heads, cache->dim, pairs, sections, axes,
                       position_dtype, static_cast<cudaStream_t>(stream));
}
}
