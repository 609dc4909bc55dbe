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
// Bound by HBM: every element is read and written once.  One CTA for two tokens: its threads have their first loads under way
// while n of them make a token's sines and cosines, which all heads share, in shared memory.  8192 tokens, 32/8 heads of 128 on
// three axes: 29 us, 5.8 TB/s, 0.89 of a copy (one token a CTA 38 us, four 32).
#include "rotary_axes.cuh"

namespace qmm {

namespace {

// The cosine and sine of a token's pair.
__device__ __forceinline__ void make_turn(const RotaryParams &p, int64_t token, int pair, float *c, float *s) {
    const int64_t place = load_index(p.positions, axis_of(p, pair) * p.pos_sa + token * p.pos_st, p.wide_positions);
    const double half_turns = static_cast<double>(place) * static_cast<double>(__ldg(p.inv_freq + pair)) * 0.31830988618379067154;
    sincospif(static_cast<float>(half_turns - 2.0 * rint(0.5 * half_turns)), s, c);
}

template <typename T>
struct Vec {
    static constexpr int kElems = 16 / sizeof(T);
    static __device__ __forceinline__ void unpack(const uint4 &w, float (&f)[kElems]) {
        const T *x = reinterpret_cast<const T *>(&w);
#pragma unroll
        for (int i = 0; i < kElems; ++i) f[i] = to_float(x[i]);
    }
    static __device__ __forceinline__ uint4 pack(const float (&f)[kElems]) {
        uint4 w;
        T *x = reinterpret_cast<T *>(&w);
#pragma unroll
        for (int i = 0; i < kElems; ++i) x[i] = from_float<T>(f[i]);
        return w;
    }
};

// Whether rows `stride` elements apart begin at 16-byte boundaries.
template <typename T>
bool aligned(const void *base, int64_t a, int64_t b, int64_t c = 0) {
    return (reinterpret_cast<uintptr_t>(base) & 15) == 0 && ((a | b | c) & (Vec<T>::kElems - 1)) == 0;
}

// Row `row` of a token: first the query's heads, then the key's, then the value's.
template <typename T>
__device__ __forceinline__ void find_row(const RotaryParams &p, int64_t token, int row, int64_t block, int64_t at, const T **src, T **dst) {
    if (row < p.heads) {
        *src = static_cast<const T *>(p.q) + token * p.q_st + row * p.q_sh;
        *dst = static_cast<T *>(p.q_out) + (token * p.heads + row) * p.dim;
    } else if (row < p.heads + p.kv_heads) {
        const int head = row - p.heads;
        *src = static_cast<const T *>(p.k) + token * p.k_st + head * p.k_sh;
        *dst = p.cached ? static_cast<T *>(p.k_cache) + block * p.kc_sb + at * p.kc_st + head * p.kc_sh
                        : static_cast<T *>(p.k_out) + (token * p.kv_heads + head) * p.dim;
    } else {
        const int head = row - p.heads - p.kv_heads;
        *src = static_cast<const T *>(p.v) + token * p.v_st + head * p.v_sh;
        *dst = static_cast<T *>(p.v_cache) + block * p.vc_sb + at * p.vc_st + head * p.vc_sh;
    }
}

// An element a thread: any alignment.
template <typename T>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const __grid_constant__ RotaryParams p) {
    __shared__ float s_cos[kMostPairs], s_sin[kMostPairs];
    pdl_launch_dependents();
    pdl_wait();
    const int64_t token = blockIdx.x;
    for (int i = threadIdx.x; i < p.pairs; i += kThreads) make_turn(p, token, i, s_cos + i, s_sin + i);
    __syncthreads();
    int64_t block = 0, at = 0;
    const bool write = !p.cached || find_slot(p, token, &block, &at);
    const int rows = p.heads + (write ? p.kv_heads * (p.cached ? 2 : 1) : 0);
    for (int item = threadIdx.x; item < rows * p.dim; item += kThreads) {
        const int row = item / p.dim, e = item - row * p.dim;
        const T *src;
        T *dst;
        find_row(p, token, row, block, at, &src, &dst);
        if (row >= p.heads + p.kv_heads || e >= 2 * p.pairs) {
            dst[e] = src[e];
            continue;
        }
        const int i = p.interleaved ? e >> 1 : e < p.pairs ? e : e - p.pairs;
        const bool second = p.interleaved ? (e & 1) != 0 : e >= p.pairs;
        const float a = to_float(src[p.interleaved ? 2 * i : i]), b = to_float(src[p.interleaved ? 2 * i + 1 : i + p.pairs]);
        dst[e] = from_float<T>(second ? turned_second(a, b, s_cos[i], s_sin[i]) : turned_first(a, b, s_cos[i], s_sin[i]));
    }
}

// 16-byte vectors.  A part of a row is, with halves, the vector of the first elements of its pairs and that of the second ones, or
// one vector behind the pairs; interleaved, one vector.  The first kAhead rows are under
// way while the sines and cosines are made.
//
// TOKENS a CTA: two where there are enough, so that 64 pairs' sines and cosines keep half the threads busy and three parts a thread
// are under way (8192 tokens, 32 + 8 heads of 128, bf16: one token 40.6 us, two 28.9, four 30.0 to 32.7, of the 26.0 that the copy
// bandwidth allows).
constexpr int kAhead = 3;
template <typename T, bool INTERLEAVED, int TOKENS>
__global__ void __launch_bounds__(kThreads) rotary_vec_kernel(const __grid_constant__ RotaryParams p, int64_t tokens, unsigned magic) {
    constexpr int E = Vec<T>::kElems;
    __shared__ __align__(16) float s_cos[TOKENS][kMostPairs], s_sin[TOKENS][kMostPairs];
    __shared__ int64_t s_block[TOKENS], s_at[TOKENS];  // where a token goes in the cache; block < 0: nowhere
    pdl_launch_dependents();
    pdl_wait();
    const int64_t token0 = static_cast<int64_t>(blockIdx.x) * TOKENS;
    const int here = static_cast<int>(min(static_cast<int64_t>(TOKENS), tokens - token0));
    const int turning = INTERLEAVED ? 2 * p.pairs / E : p.pairs / E;  // parts of a row that turn
    const int parts = INTERLEAVED ? p.dim / E : turning + (p.dim - 2 * p.pairs) / E;
    const int rows = p.heads + p.kv_heads * (p.cached ? 2 : 1);  // of a token
    const int all = rows * here * parts;
    // a part of a row: its token, row and vectors
    struct Spot {
        int token, row, e0, e1;
        bool turns, two;
    };
    auto spot_of = [&](int item) {
        Spot s;
        const int row = magic != 0 ? static_cast<int>(__umulhi(item, magic)) : item, part = item - row * parts;  // item / parts
        s.token = 0;
#pragma unroll
        for (int i = 1; i < TOKENS; ++i) s.token += row >= i * rows;
        s.row = row - s.token * rows;
        s.turns = part < turning;
        s.e0 = (INTERLEAVED || s.turns ? part : part + turning) * E;  // first vector
        s.e1 = s.e0 + p.pairs;                                        // second one
        s.two = !INTERLEAVED && s.turns;
        return s;
    };
    bool made = false;
    for (int item0 = threadIdx.x; !made || item0 < all; item0 += kAhead * kThreads) {
        uint4 x[kAhead], y[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            if (item0 + i * kThreads >= all) break;
            const Spot at = spot_of(item0 + i * kThreads);
            const T *src;
            T *dst;
            find_row(p, token0 + at.token, at.row, 0, 0, &src, &dst);
            x[i] = __ldg(reinterpret_cast<const uint4 *>(src + at.e0));
            if (at.two) y[i] = __ldg(reinterpret_cast<const uint4 *>(src + at.e1));
        }
        if (!made) {
            if (p.cached && threadIdx.x < here) {
                int64_t block = -1, at = 0;
                if (!find_slot(p, token0 + threadIdx.x, &block, &at)) block = -1;
                s_block[threadIdx.x] = block;
                s_at[threadIdx.x] = at;
            }
            for (int i = threadIdx.x; i < p.pairs * here; i += kThreads) {
                const int token = i / p.pairs, pair = i - token * p.pairs;
                make_turn(p, token0 + token, pair, &s_cos[token][pair], &s_sin[token][pair]);
            }
            __syncthreads();
            made = true;
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            if (item0 + i * kThreads >= all) break;
            const Spot at = spot_of(item0 + i * kThreads);
            const int64_t block = p.cached ? s_block[at.token] : 0, place = p.cached ? s_at[at.token] : 0;
            if (at.row >= p.heads && block < 0) continue;
            const T *src;
            T *dst;
            find_row(p, token0 + at.token, at.row, block, place, &src, &dst);
            if (at.turns && at.row < p.heads + p.kv_heads) {
                const float *cosine = s_cos[at.token], *sine = s_sin[at.token];
                float a[E], b[E];
                Vec<T>::unpack(x[i], a);
                if (INTERLEAVED) {
#pragma unroll
                    for (int j = 0; j < E; j += 2) {
                        const float c = cosine[(at.e0 + j) >> 1], s = sine[(at.e0 + j) >> 1];
                        b[j] = turned_first(a[j], a[j + 1], c, s);
                        b[j + 1] = turned_second(a[j], a[j + 1], c, s);
                    }
                    x[i] = Vec<T>::pack(b);
                } else {
                    Vec<T>::unpack(y[i], b);
#pragma unroll
                    for (int j = 0; j < E; ++j) {
                        const float c = cosine[at.e0 + j], s = sine[at.e0 + j], first = a[j];
                        a[j] = turned_first(first, b[j], c, s);
                        b[j] = turned_second(first, b[j], c, s);
                    }
                    x[i] = Vec<T>::pack(a);
                    y[i] = Vec<T>::pack(b);
                }
            }
            *reinterpret_cast<uint4 *>(dst + at.e0) = x[i];
            if (at.two) *reinterpret_cast<uint4 *>(dst + at.e1) = y[i];
        }
    }
}

template <typename T>
int launch_rotary(const RotaryParams &p, int64_t tokens, cudaStream_t stream) {
    constexpr int E = Vec<T>::kElems;
    const dim3 grid(static_cast<unsigned>(tokens));
    const bool vectors = p.dim % E == 0 && (p.interleaved ? 2 * p.pairs : p.pairs) % E == 0 && aligned<T>(p.q, p.q_st, p.q_sh) &&
                         aligned<T>(p.k, p.k_st, p.k_sh) && aligned<T>(p.q_out, 0, 0) && aligned<T>(p.k_out, 0, 0) &&
                         aligned<T>(p.v, p.v_st, p.v_sh) && aligned<T>(p.k_cache, p.kc_sb, p.kc_st, p.kc_sh) &&
                         aligned<T>(p.v_cache, p.vc_sb, p.vc_st, p.vc_sh);
    if (!vectors) {
        QMM_CUDA_OK(launch_pdl(rotary_kernel<T>, grid, dim3(kThreads), 0, stream, p));
        return QMM_OK;
    }
    const int parts = p.interleaved ? p.dim / E : (p.dim - p.pairs) / E;
    // item * magic >> 32 = item / parts, as long as item * parts is below 2^32; 0: parts is 1
    const unsigned magic = parts > 1 ? 0xffffffffu / parts + 1 : 0;
    // two tokens a CTA where that leaves two CTAs for every SM
    constexpr int kTokens = 2;
    const bool many = tokens >= 2ll * kTokens * sm_count();
    auto kern = p.interleaved ? (many ? rotary_vec_kernel<T, true, kTokens> : rotary_vec_kernel<T, true, 1>)
                              : (many ? rotary_vec_kernel<T, false, kTokens> : rotary_vec_kernel<T, false, 1>);
    QMM_CUDA_OK(launch_pdl(kern, many ? dim3(static_cast<unsigned>((tokens + kTokens - 1) / kTokens)) : grid, dim3(kThreads), 0, stream, p, tokens, magic));
    return QMM_OK;
}

int rotary(const char *op, RotaryParams &p, int dtype, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t dim,
           int64_t pairs, const int64_t *sections, int64_t axes, int position_dtype, cudaStream_t stream) {
    const int rc = take_sizes(op, p, tokens, heads, kv_heads, dim, pairs, sections, axes, position_dtype);
    if (rc != QMM_OK) return rc;
    if (tokens == 0 || dim == 0) return QMM_OK;
    if (dtype == QMM_DTYPE_BF16) return launch_rotary<__nv_bfloat16>(p, tokens, stream);
    if (dtype == QMM_DTYPE_F16) return launch_rotary<__half>(p, tokens, stream);
    if (dtype == QMM_DTYPE_F32) return launch_rotary<float>(p, tokens, stream);
    return fail(QMM_ERR_INVALID_ARGUMENT, std::string(op) + ": the tensors must be bf16, f16 or f32");
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
    QMM_REQUIRE(cache->pages == 0 || cache->key != cache->value,
                "qmm_rotary_axes_cache: keys and values must have places of their own, but they begin at the same address");
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
