// What the rotary kernels share (rotary_axes.cu: outputs and caches of the tensors' type, rotary_quant_cache.cu: an int8 cache): the
// problem's description, the axes of pairs, where a token goes in the cache, and the checks of sizes.
#pragma once

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

// Where the token goes in the cache; false: nowhere.
__device__ __forceinline__ bool find_slot(const RotaryParams &p, int64_t token, int64_t *block, int64_t *at) {
    const int64_t slot = load_index(p.slots, token * p.slot_st, p.wide_slots);
    if (slot < 0 || slot >= p.places) return false;
    *block = slot / p.page;
    *at = slot - *block * p.page;
    return true;
}

__device__ __forceinline__ float turned_first(float a, float b, float c, float s) { return fmaf(a, c, -(b * s)); }
__device__ __forceinline__ float turned_second(float a, float b, float c, float s) { return fmaf(b, c, a * s); }

// The arguments that the entries share, checked and taken over.
inline int take_sizes(const char *op, RotaryParams &p, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t dim, int64_t pairs,
                      const int64_t *sections, int64_t axes, int position_dtype) {
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
    return QMM_OK;
}

}  // namespace

}  // namespace qmm
