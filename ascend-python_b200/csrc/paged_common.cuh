// What the kernels over the paged key-value cache share: the problem's description, which keys a token sees, where a key's
// row lies, and the attention of one row by one warp.
//
// Visible keys of the token at place p (0-based) of its sequence, in places j of the cache:
//     j <= p,  j < pages of the block table * page size,  the table's entry for j names a page of the cache, and
//     window == 0  or  p - j < window  or  j < sinks.
// With window > 0 these are two ranges, [0, sink_end) and [lo, hi).  Pages that a window has left behind are never read, so
// their entries may be anything.  A row that sees no key has output 0 and a log-sum of -inf.
#pragma once

#include "qmm_common.cuh"

namespace qmm {
namespace paged {

struct Problem {
    const void *q;
    int64_t q_st, q_sh;  // strides of the query's tokens and heads, in elements
    const void *k, *v;
    int64_t k_sb, k_st, k_sh;  // strides of a cache's pages, places and heads, in elements
    int64_t v_sb, v_st, v_sh;
    const int32_t *table;  // [batch][max_pages], rows table_st apart
    int64_t table_st;
    const int32_t *lens;
    const int32_t *start;  // null: one token a sequence
    void *out;             // [tokens][heads][dim], dense
    float *lse;            // [tokens][heads]
    int batch, heads, kv_heads, group, dim, page, page_shift;  // page_shift: log2(page), or -1
    int max_pages, window, sinks;
    int64_t tokens, pages;
    int capacity;  // places that a block table's row covers
    float scale;
};

struct Range {
    int sink_end, lo, hi;
};

__host__ __device__ __forceinline__ Range visible_range(const Problem &p, int place) {
    Range r;
    const int64_t end = static_cast<int64_t>(place) + 1;
    r.lo = p.window > 0 && end > p.window ? static_cast<int>(end - p.window) : 0;
    r.sink_end = p.sinks < r.lo ? p.sinks : r.lo;
    r.hi = end < p.capacity ? static_cast<int>(end < 0 ? 0 : end) : p.capacity;
    if (r.sink_end > r.hi) r.sink_end = r.hi;
    return r;
}

__device__ __forceinline__ int page_of(const Problem &p, int j) {
    return p.page_shift >= 0 ? j >> p.page_shift : j / p.page;
}

// The page of place j (a place below the capacity) of sequence b and j's place in it; false: no page of the cache.
__device__ __forceinline__ bool find_place(const Problem &p, int b, int j, int64_t *block, int *at) {
    const int i = page_of(p, j);
    const int32_t id = __ldg(p.table + b * p.table_st + i);
    *block = id;
    *at = j - i * p.page;
    return id >= 0 && id < p.pages;
}

// The output of one row (token, head) by one warp, in fp32: the lanes take 32 keys at a time and their whole products, then all
// lanes add the keys' values for the columns lane, lane + 32, ...  Reads visible keys alone.
template <typename T>
__device__ __noinline__ void plain_row(const Problem &p, int b, int64_t token, int head, int place) {
    constexpr int kMost = 8;  // columns a lane, dim <= 256
    const int lane = threadIdx.x & 31;
    const int kvh = head / p.group;
    const T *q = static_cast<const T *>(p.q) + token * p.q_st + head * p.q_sh;
    const T *k = static_cast<const T *>(p.k) + kvh * p.k_sh;
    const T *v = static_cast<const T *>(p.v) + kvh * p.v_sh;
    const Range r = visible_range(p, place);
    float acc[kMost];
#pragma unroll
    for (int i = 0; i < kMost; ++i) acc[i] = 0.0f;
    float top = -INFINITY, total = 0.0f;
    for (int part = 0; part < 2; ++part) {
        const int end = part == 0 ? r.sink_end : r.hi;
        for (int j0 = part == 0 ? 0 : r.lo; j0 < end; j0 += 32) {
            const int j = j0 + lane;
            int64_t block = 0;
            int at = 0;
            const bool seen = j < end && find_place(p, b, j, &block, &at);
            float s = -INFINITY;
            if (seen) {
                const T *row = k + block * p.k_sb + at * p.k_st;
                float dot = 0.0f;
                for (int d = 0; d < p.dim; ++d) dot = fmaf(to_float(q[d]), to_float(row[d]), dot);
                s = dot * p.scale;
            }
            float most = s;
            for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
            const float now = fmaxf(top, most);
            const float base = now == -INFINITY ? 0.0f : now;
            const float keep = expf(top - base);
            const float e = seen ? expf(s - base) : 0.0f;
            top = now;
            total = total * keep + e;
#pragma unroll
            for (int i = 0; i < kMost; ++i) acc[i] *= keep;
            const uint32_t which = __ballot_sync(0xffffffffu, seen);
            const int64_t offset = block * p.v_sb + at * p.v_st;
            for (uint32_t left = which; left != 0; left &= left - 1) {
                const int from = __ffs(left) - 1;
                const float w = __shfl_sync(0xffffffffu, e, from);
                const T *row = v + __shfl_sync(0xffffffffu, offset, from);
#pragma unroll
                for (int i = 0; i < kMost; ++i)
                    if (lane + 32 * i < p.dim) acc[i] = fmaf(w, to_float(row[lane + 32 * i]), acc[i]);
            }
        }
    }
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    T *out = static_cast<T *>(p.out) + (token * p.heads + head) * p.dim;
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
    for (int i = 0; i < kMost; ++i)
        if (lane + 32 * i < p.dim) out[lane + 32 * i] = from_float<T>(acc[i] * inv);
}

// A row that sees nothing, by one warp.
template <typename T>
__device__ __forceinline__ void empty_row(const Problem &p, int64_t token, int head) {
    const int lane = threadIdx.x & 31;
    T *out = static_cast<T *>(p.out) + (token * p.heads + head) * p.dim;
    for (int d = lane; d < p.dim; d += 32) out[d] = from_float<T>(0.0f);
    if (lane == 0) p.lse[token * p.heads + head] = -INFINITY;
}

size_t decode_workspace(int64_t batch, int64_t heads, int64_t kv_heads, int64_t dim);
int launch_decode(const Problem &p, int dtype, void *workspace, size_t workspace_bytes, cudaStream_t stream);
size_t prompt_workspace(int64_t tokens, int64_t batch, int64_t heads, int64_t kv_heads, int64_t dim, int64_t places);
int launch_prompt(const Problem &p, int dtype, void *workspace, size_t workspace_bytes, cudaStream_t stream);

}  // namespace paged
}  // namespace qmm
