// What the kernels over the paged key-value cache share: the problem's description, which keys a token sees, where a key's
// row lies, and the attention of rows by plain sums.
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

// Plain attention, in fp32, of rows of one sequence and one key-value head, by one warp: part `part` of `parts`, every `parts`-th 32
// keys.  The lanes take a key each for its products with the query rows (`q`: shared memory, fp32, kPlainDim apart; place < 0: no row),
// then keys' values for eight columns a lane; keys of up to 128 dimensions two at a time.  Reads keys alone that a row sees, and a
// row takes those alone that it sees itself.
constexpr int kPlainDim = 256;
struct RowPart {
    float acc[8];      // relative to exp(top), of columns 8 * lane ... (the same in both halves of the warp for two keys at a time)
    float top, total;  // the same in all lanes
};
template <typename T, int R>
__device__ __noinline__ void rows_part(const Problem &p, int b, int kvh, const int *place, const float *q, int part, int parts, RowPart *out) {
    const int lane = threadIdx.x & 31;
    const bool two = p.dim <= 128;
    const int half = two ? lane >> 4 : 0, column = (two ? lane & 15 : lane) * 8;
    const T *k = static_cast<const T *>(p.k) + kvh * p.k_sh;
    const T *v = static_cast<const T *>(p.v) + kvh * p.v_sh + (column < p.dim ? column : 0);
    Range of[R];
    int sink_end = 0, lo = 0x7fffffff, hi = 0;
    float acc[R][8] = {}, top[R], total[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        of[r] = visible_range(p, place[r]);
        top[r] = -INFINITY;
        total[r] = 0.0f;
        if (of[r].hi == 0) continue;
        sink_end = max(sink_end, of[r].sink_end);
        lo = min(lo, of[r].lo);
        hi = max(hi, of[r].hi);
    }
    for (int range = 0; range < 2; ++range) {
        const int end = range == 0 ? sink_end : hi;
        for (int64_t j0 = (range == 0 ? 0 : lo) + 32ll * part; j0 < end; j0 += 32ll * parts) {
            const int j = static_cast<int>(j0) + lane;  // (a capacity leaves room for a tile behind it)
            int64_t block = 0;
            int at = 0;
            uint32_t sees = 0;  // a bit a row
#pragma unroll
            for (int r = 0; r < R; ++r) sees |= (range == 0 ? j < of[r].sink_end : j >= of[r].lo && j < of[r].hi) ? 1u << r : 0u;
            if (sees != 0 && !find_place(p, b, j, &block, &at)) sees = 0;
            float e[R] = {};
            if (sees != 0) {
                const uint4 *row = reinterpret_cast<const uint4 *>(k + block * p.k_sb + at * p.k_st);
                const int chunks = p.dim / 8;
                for (int c = 0; c < chunks; c += 4) {  // four parts of a key under way together
                    uint4 x[4];
#pragma unroll
                    for (int n = 0; n < 4; ++n) x[n] = c + n < chunks ? __ldg(row + c + n) : make_uint4(0, 0, 0, 0);
#pragma unroll
                    for (int n = 0; n < 4; ++n) {
                        if (c + n >= chunks) break;
                        const T *y = reinterpret_cast<const T *>(&x[n]);
#pragma unroll
                        for (int i = 0; i < 8; i += 4) {
#pragma unroll
                            for (int r = 0; r < R; ++r) {
                                const float4 z = *reinterpret_cast<const float4 *>(q + r * kPlainDim + (c + n) * 8 + i);
                                e[r] = fmaf(z.w, to_float(y[i + 3]), fmaf(z.z, to_float(y[i + 2]), fmaf(z.y, to_float(y[i + 1]), fmaf(z.x, to_float(y[i]), e[r]))));
                            }
                        }
                    }
                }
            }
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const bool seen = sees >> r & 1;
                const float s = seen ? e[r] * p.scale : -INFINITY;
                float most = s;
                for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
                const float now = fmaxf(top[r], most);
                const float base = now == -INFINITY ? 0.0f : now;
                const float keep = expf(top[r] - base);
                e[r] = seen ? expf(s - base) : 0.0f;
                top[r] = now;
                total[r] = total[r] * keep + e[r];
#pragma unroll
                for (int i = 0; i < 8; ++i) acc[r][i] *= keep;
            }
            const int64_t offset = block * p.v_sb + at * p.v_st;
            // four values of a lane under way together
#pragma unroll 1
            for (int from = half; from < 32; from += two ? 8 : 4) {
                uint4 x[4];
                uint32_t which[4];
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    const int key = from + (two ? 2 * n : n);
                    which[n] = __shfl_sync(0xffffffffu, sees, key);
                    const T *row = v + __shfl_sync(0xffffffffu, offset, key);
                    x[n] = make_uint4(0, 0, 0, 0);
                    if (which[n] != 0) x[n] = __ldg(reinterpret_cast<const uint4 *>(row));
                }
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    const T *y = reinterpret_cast<const T *>(&x[n]);
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        const float w = __shfl_sync(0xffffffffu, e[r], from + (two ? 2 * n : n));
                        if (!(which[n] >> r & 1)) continue;
#pragma unroll
                        for (int i = 0; i < 8; ++i) acc[r][i] = fmaf(w, to_float(y[i]), acc[r][i]);
                    }
                }
            }
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        for (int o = 16; o > 0; o >>= 1) total[r] += __shfl_xor_sync(0xffffffffu, total[r], o);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float other = __shfl_xor_sync(0xffffffffu, acc[r][i], 16);
            out[r].acc[i] = acc[r][i] + (two ? other : 0.0f);
        }
        out[r].top = top[r];
        out[r].total = total[r];
    }
}

// A query row to shared memory for rows_part, by one warp.
template <typename T>
__device__ __forceinline__ void stage_query(const Problem &p, int64_t token, int head, float *q) {
    const T *src = static_cast<const T *>(p.q) + token * p.q_st + head * p.q_sh;
    for (int d = threadIdx.x & 31; d < p.dim; d += 32) q[d] = to_float(src[d]);
}

// The output of a row of which a warp has everything.
template <typename T>
__device__ __forceinline__ void write_row(const Problem &p, int64_t token, int head, const RowPart &r) {
    const int lane = threadIdx.x & 31;
    if (lane * 8 >= p.dim) return;
    const float inv = r.total == 0.0f ? 0.0f : 1.0f / r.total;
    *reinterpret_cast<uint4 *>(static_cast<T *>(p.out) + (token * p.heads + head) * p.dim + lane * 8) =
        make_uint4(pack2<T>(r.acc[0] * inv, r.acc[1] * inv), pack2<T>(r.acc[2] * inv, r.acc[3] * inv), pack2<T>(r.acc[4] * inv, r.acc[5] * inv),
                   pack2<T>(r.acc[6] * inv, r.acc[7] * inv));
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
