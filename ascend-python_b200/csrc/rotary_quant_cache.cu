// Rotary positions with the write into an int8 paged key-value cache (npu_rotary_axes_quant_cache).
//
// The query is turned as npu_rotary_axes turns it.  A row (token, head) of the turned key, and of the value, is written as
//     scale = max |y| / 127, rounded to fp32;   code = y / scale, to the nearest whole number (ties to even), in int8
// (0 where the scale is 0 or not finite), without a rounding of y between.
//
// The keys' rotation, the maximum and the quotient are in 64 bits: a value next to the border of two codes then has the code of
// the definition, whichever kernel or order of operations made it, where fp32 angles alone (off by 2^-25 half turns) move a code in
// some 2^16.  Positions times frequencies are exact there up to positions of 2^29.  The quotient is a product with the
// reciprocal, corrected by its remainder, so that one that is a tie comes out as one; codes come out of its sum with 1.5 * 2^52, which has
// them in its low bits.
//
// Bound by HBM: every element is read once and written once.
#include "rotary_axes.cuh"

namespace qmm {

namespace {

struct QuantParams {
    float *k_scale, *v_scale;
    int64_t ks_sb, ks_st, ks_sh, vs_sb, vs_st, vs_sh;
};

// The cosine and sine of a token's pair in 64 bits.
__device__ __forceinline__ void make_turn_64(const RotaryParams &p, int64_t token, int pair, double *c, double *s) {
    const int64_t place = load_index(p.positions, axis_of(p, pair) * p.pos_sa + token * p.pos_st, p.wide_positions);
    sincos(static_cast<double>(place) * static_cast<double>(__ldg(p.inv_freq + pair)), s, c);
}

__device__ __forceinline__ double turned_first_64(double a, double b, double c, double s) { return fma(a, c, -(b * s)); }
__device__ __forceinline__ double turned_second_64(double a, double b, double c, double s) { return fma(b, c, a * s); }

// Magnitudes as whole numbers, which keep their order and put NaN above all.
__device__ __forceinline__ unsigned long long magnitude(double x) {
    return static_cast<unsigned long long>(__double_as_longlong(x)) & 0x7fffffffffffffffull;
}

struct RowScale {
    float scale;
    double inverse;  // 0: all codes are 0
};
// From the largest magnitudes of the lanes of a row: `lanes` of them, a power of two.
__device__ __forceinline__ RowScale make_scale(unsigned long long most, int lanes, uint32_t mask) {
    for (int o = lanes >> 1; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(mask, most, o));
    RowScale r;
    r.scale = static_cast<float>(__longlong_as_double(static_cast<long long>(most)) / 127.0);
    r.inverse = r.scale > 0.0f && r.scale <= 3.402823466e38f ? 1.0 / static_cast<double>(r.scale) : 0.0;
    return r;
}

// (a scale below fp32's full steps may be off by half of itself)
__device__ __forceinline__ int code_of(double y, const RowScale &r) {
    const double about = y * r.inverse, quotient = fma(fma(-about, static_cast<double>(r.scale), y), r.inverse, about);
    return r.inverse == 0.0 ? 0 : max(-128, min(127, __double2loint(quotient + 6755399441055744.0)));
}

// Any alignment: a CTA a token, a warp a row of keys or values, an element a lane at a time.
template <typename T>
__global__ void __launch_bounds__(kThreads) rotary_quant_kernel(const __grid_constant__ RotaryParams p, const __grid_constant__ QuantParams out) {
    __shared__ float s_cos[kMostPairs], s_sin[kMostPairs];
    __shared__ double s_cos64[kMostPairs], s_sin64[kMostPairs];
    pdl_launch_dependents();
    pdl_wait();
    const int64_t token = blockIdx.x;
    for (int i = threadIdx.x; i < p.pairs; i += kThreads) {
        make_turn(p, token, i, s_cos + i, s_sin + i);
        make_turn_64(p, token, i, s_cos64 + i, s_sin64 + i);
    }
    __syncthreads();
    for (int item = threadIdx.x; item < p.heads * p.dim; item += kThreads) {
        const int row = item / p.dim, e = item - row * p.dim;
        const T *src = static_cast<const T *>(p.q) + token * p.q_st + row * p.q_sh;
        T *dst = static_cast<T *>(p.q_out) + (token * p.heads + row) * p.dim;
        if (e >= 2 * p.pairs) {
            dst[e] = src[e];
            continue;
        }
        const int i = p.interleaved ? e >> 1 : e < p.pairs ? e : e - p.pairs;
        const bool second = p.interleaved ? (e & 1) != 0 : e >= p.pairs;
        const float a = to_float(src[p.interleaved ? 2 * i : i]), b = to_float(src[p.interleaved ? 2 * i + 1 : i + p.pairs]);
        dst[e] = from_float<T>(second ? turned_second(a, b, s_cos[i], s_sin[i]) : turned_first(a, b, s_cos[i], s_sin[i]));
    }
    int64_t block = 0, at = 0;
    if (!find_slot(p, token, &block, &at)) return;
    const int lane = threadIdx.x & 31;
    for (int row = threadIdx.x >> 5; row < 2 * p.kv_heads; row += kThreads / 32) {
        const bool key = row < p.kv_heads;
        const int head = key ? row : row - p.kv_heads;
        const T *src = key ? static_cast<const T *>(p.k) + token * p.k_st + head * p.k_sh : static_cast<const T *>(p.v) + token * p.v_st + head * p.v_sh;
        int8_t *dst = key ? static_cast<int8_t *>(p.k_cache) + block * p.kc_sb + at * p.kc_st + head * p.kc_sh
                          : static_cast<int8_t *>(p.v_cache) + block * p.vc_sb + at * p.vc_st + head * p.vc_sh;
        double y[8];
        unsigned long long most = 0;
#pragma unroll
        for (int n = 0; n < 8; ++n) {
            const int e = lane + 32 * n;
            y[n] = 0.0;
            if (e >= p.dim) continue;
            if (!key || e >= 2 * p.pairs) {
                y[n] = static_cast<double>(to_float(src[e]));
            } else {
                const int i = p.interleaved ? e >> 1 : e < p.pairs ? e : e - p.pairs;
                const bool second = p.interleaved ? (e & 1) != 0 : e >= p.pairs;
                const double a = to_float(src[p.interleaved ? 2 * i : i]), b = to_float(src[p.interleaved ? 2 * i + 1 : i + p.pairs]);
                y[n] = second ? turned_second_64(a, b, s_cos64[i], s_sin64[i]) : turned_first_64(a, b, s_cos64[i], s_sin64[i]);
            }
            most = max(most, magnitude(y[n]));
        }
        const RowScale scale = make_scale(most, 32, 0xffffffffu);
#pragma unroll
        for (int n = 0; n < 8; ++n)
            if (lane + 32 * n < p.dim) dst[lane + 32 * n] = static_cast<int8_t>(code_of(y[n], scale));
        if (lane == 0) {
            if (key)
                out.k_scale[block * out.ks_sb + at * out.ks_st + head * out.ks_sh] = scale.scale;
            else
                out.v_scale[block * out.vs_sb + at * out.vs_st + head * out.vs_sh] = scale.scale;
        }
    }
}

// Eight elements, as they are loaded and stored.
template <typename T>
struct Eight {
    uint4 w[sizeof(T) / 2];
    __device__ __forceinline__ void load(const T *src) {
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) w[i] = __ldg(reinterpret_cast<const uint4 *>(src) + i);
    }
    __device__ __forceinline__ void store(T *dst) const {
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) reinterpret_cast<uint4 *>(dst)[i] = w[i];
    }
    __device__ __forceinline__ void unpack(float (&f)[8]) const {
        const T *x = reinterpret_cast<const T *>(w);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = to_float(x[i]);
    }
    __device__ __forceinline__ void pack(const float (&f)[8]) {
        T *x = reinterpret_cast<T *>(w);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = from_float<T>(f[i]);
    }
};

__device__ __forceinline__ uint2 codes_of(const double (&y)[8], const RowScale &r) {
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i >> 2] |= static_cast<uint32_t>(code_of(y[i], r) & 255) << 8 * (i & 3);
    return make_uint2(w[0], w[1]);
}

// Vectors of eight elements.  A part of a row is, with halves, the vector of the first elements of its pairs and that of the second
// ones, or one vector behind the pairs; interleaved, one vector.  2^log_lanes lanes of a warp, as many as parts or
// more, have a row, and find its maximum together.  The first kAhead rows of a lane are under way while the sines and cosines are made.
constexpr int kAhead = 3;
template <typename T, bool INTERLEAVED, int TOKENS>
__global__ void __launch_bounds__(kThreads)
rotary_quant_vec_kernel(const __grid_constant__ RotaryParams p, const __grid_constant__ QuantParams out, int64_t tokens, int log_lanes) {
    __shared__ __align__(16) float s_cos[TOKENS][kMostPairs], s_sin[TOKENS][kMostPairs];
    __shared__ __align__(16) double s_cos64[TOKENS][kMostPairs], s_sin64[TOKENS][kMostPairs];
    __shared__ int64_t s_block[TOKENS], s_at[TOKENS];  // where a token goes in the cache; block < 0: nowhere
    pdl_launch_dependents();
    pdl_wait();
    const int64_t token0 = static_cast<int64_t>(blockIdx.x) * TOKENS;
    const int here = static_cast<int>(min(static_cast<int64_t>(TOKENS), tokens - token0));
    const int turning = INTERLEAVED ? 2 * p.pairs / 8 : p.pairs / 8;  // parts of a row that turn
    const int parts = INTERLEAVED ? p.dim / 8 : turning + (p.dim - 2 * p.pairs) / 8;
    const int rows = p.heads + 2 * p.kv_heads;  // of a token
    const int all = rows * here << log_lanes;
    const int lanes = 1 << log_lanes;
    const int part = threadIdx.x & (lanes - 1);  // the same in every row
    const bool active = part < parts, turns = part < turning, two = !INTERLEAVED && turns;
    const int e0 = (INTERLEAVED || turns ? part : part + turning) * 8, e1 = e0 + p.pairs;  // first vector, second one
    const uint32_t mask = (lanes == 32 ? 0xffffffffu : (1u << lanes) - 1) << (threadIdx.x & 31 & ~(lanes - 1));
    struct Spot {
        int token, row;
    };
    auto spot_of = [&](int item) {
        Spot s;
        const int row = item >> log_lanes;
        s.token = 0;
#pragma unroll
        for (int i = 1; i < TOKENS; ++i) s.token += row >= i * rows;
        s.row = row - s.token * rows;
        return s;
    };
    bool made = false;
    for (int item0 = threadIdx.x; !made || item0 < all; item0 += kAhead * kThreads) {
        Eight<T> x[kAhead], y[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            if (item0 + i * kThreads >= all) break;
            const Spot at = spot_of(item0 + i * kThreads);
            const int64_t token = token0 + at.token;
            const T *src = at.row < p.heads                ? static_cast<const T *>(p.q) + token * p.q_st + at.row * p.q_sh
                           : at.row < p.heads + p.kv_heads ? static_cast<const T *>(p.k) + token * p.k_st + (at.row - p.heads) * p.k_sh
                                                           : static_cast<const T *>(p.v) + token * p.v_st + (at.row - p.heads - p.kv_heads) * p.v_sh;
            if (active) x[i].load(src + e0);
            if (two) y[i].load(src + e1);
        }
        if (!made) {
            if (threadIdx.x < here) {
                int64_t block = -1, at = 0;
                if (!find_slot(p, token0 + threadIdx.x, &block, &at)) block = -1;
                s_block[threadIdx.x] = block;
                s_at[threadIdx.x] = at;
            }
            for (int i = threadIdx.x; i < p.pairs * here; i += kThreads) {
                const int token = i / p.pairs, pair = i - token * p.pairs;
                make_turn(p, token0 + token, pair, &s_cos[token][pair], &s_sin[token][pair]);
                make_turn_64(p, token0 + token, pair, &s_cos64[token][pair], &s_sin64[token][pair]);
            }
            __syncthreads();
            made = true;
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            if (item0 + i * kThreads >= all) break;
            const Spot at = spot_of(item0 + i * kThreads);
            if (at.row < p.heads) {
                if (!active) continue;
                T *dst = static_cast<T *>(p.q_out) + ((token0 + at.token) * p.heads + at.row) * p.dim;
                if (turns) {
                    const float *cosine = s_cos[at.token], *sine = s_sin[at.token];
                    float a[8], b[8];
                    x[i].unpack(a);
                    if (INTERLEAVED) {
#pragma unroll
                        for (int j = 0; j < 8; j += 2) {
                            const float c = cosine[(e0 + j) >> 1], s = sine[(e0 + j) >> 1];
                            b[j] = turned_first(a[j], a[j + 1], c, s);
                            b[j + 1] = turned_second(a[j], a[j + 1], c, s);
                        }
                        x[i].pack(b);
                    } else {
                        y[i].unpack(b);
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const float c = cosine[e0 + j], s = sine[e0 + j], first = a[j];
                            a[j] = turned_first(first, b[j], c, s);
                            b[j] = turned_second(first, b[j], c, s);
                        }
                        x[i].pack(a);
                        y[i].pack(b);
                    }
                }
                x[i].store(dst + e0);
                if (two) y[i].store(dst + e1);
                continue;
            }
            const int64_t block = s_block[at.token], place = s_at[at.token];
            if (block < 0) continue;
            const bool key = at.row < p.heads + p.kv_heads;
            const int head = at.row - p.heads - (key ? 0 : p.kv_heads);
            double a[8], b[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) a[j] = b[j] = 0.0;
            if (active) {
                float f[8];
                x[i].unpack(f);
#pragma unroll
                for (int j = 0; j < 8; ++j) a[j] = static_cast<double>(f[j]);
            }
            if (two) {
                float f[8];
                y[i].unpack(f);
#pragma unroll
                for (int j = 0; j < 8; ++j) b[j] = static_cast<double>(f[j]);
            }
            if (key && turns) {
                const double *cosine = s_cos64[at.token], *sine = s_sin64[at.token];
                if (INTERLEAVED) {
#pragma unroll
                    for (int j = 0; j < 8; j += 2) {
                        const double c = cosine[(e0 + j) >> 1], s = sine[(e0 + j) >> 1], first = a[j];
                        a[j] = turned_first_64(first, a[j + 1], c, s);
                        a[j + 1] = turned_second_64(first, a[j + 1], c, s);
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const double c = cosine[e0 + j], s = sine[e0 + j], first = a[j];
                        a[j] = turned_first_64(first, b[j], c, s);
                        b[j] = turned_second_64(first, b[j], c, s);
                    }
                }
            }
            unsigned long long most = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) most = max(most, max(magnitude(a[j]), magnitude(b[j])));
            const RowScale scale = make_scale(most, lanes, mask);
            int8_t *dst = key ? static_cast<int8_t *>(p.k_cache) + block * p.kc_sb + place * p.kc_st + head * p.kc_sh
                              : static_cast<int8_t *>(p.v_cache) + block * p.vc_sb + place * p.vc_st + head * p.vc_sh;
            if (active) *reinterpret_cast<uint2 *>(dst + e0) = codes_of(a, scale);
            if (two) *reinterpret_cast<uint2 *>(dst + e1) = codes_of(b, scale);
            if (part == 0) {
                if (key)
                    out.k_scale[block * out.ks_sb + place * out.ks_st + head * out.ks_sh] = scale.scale;
                else
                    out.v_scale[block * out.vs_sb + place * out.vs_st + head * out.vs_sh] = scale.scale;
            }
        }
    }
}

// Whether rows begin at boundaries of `bytes`, with strides in elements of `size` bytes.
bool begins_at(int bytes, int size, const void *base, int64_t a, int64_t b, int64_t c = 0) {
    return (reinterpret_cast<uintptr_t>(base) & (bytes - 1)) == 0 && ((a | b | c) & (bytes / size - 1)) == 0;
}

template <typename T>
int launch_quant(const RotaryParams &p, const QuantParams &out, int64_t tokens, cudaStream_t stream) {
    const dim3 grid(static_cast<unsigned>(tokens));
    const bool vectors = p.dim % 8 == 0 && (p.interleaved ? 2 * p.pairs : p.pairs) % 8 == 0 && begins_at(16, sizeof(T), p.q, p.q_st, p.q_sh) &&
                         begins_at(16, sizeof(T), p.k, p.k_st, p.k_sh) && begins_at(16, sizeof(T), p.v, p.v_st, p.v_sh) &&
                         begins_at(16, sizeof(T), p.q_out, 0, 0) && begins_at(8, 1, p.k_cache, p.kc_sb, p.kc_st, p.kc_sh) &&
                         begins_at(8, 1, p.v_cache, p.vc_sb, p.vc_st, p.vc_sh);
    if (!vectors) {
        QMM_CUDA_OK(launch_pdl(rotary_quant_kernel<T>, grid, dim3(kThreads), 0, stream, p, out));
        return QMM_OK;
    }
    const int parts = p.interleaved ? p.dim / 8 : (p.dim - p.pairs) / 8;
    int log_lanes = 0;
    while (1 << log_lanes < parts) ++log_lanes;
    // two tokens a CTA where that leaves two CTAs for every SM
    constexpr int kTokens = 2;
    const bool many = tokens >= 2ll * kTokens * sm_count();
    auto kern = p.interleaved ? (many ? rotary_quant_vec_kernel<T, true, kTokens> : rotary_quant_vec_kernel<T, true, 1>)
                              : (many ? rotary_quant_vec_kernel<T, false, kTokens> : rotary_quant_vec_kernel<T, false, 1>);
    QMM_CUDA_OK(launch_pdl(kern, many ? dim3(static_cast<unsigned>((tokens + kTokens - 1) / kTokens)) : grid, dim3(kThreads), 0, stream, p, out, tokens,
                           log_lanes));
    return QMM_OK;
}

}  // namespace

}  // namespace qmm

using qmm::fail;

extern "C" int qmm_rotary_axes_quant_cache(const void *query, int64_t query_stride_token, int64_t query_stride_head, const void *key,
                                           int64_t key_stride_token, int64_t key_stride_head, const void *value,
                                           int64_t value_stride_token, int64_t value_stride_head, int dtype, int64_t tokens,
                                           int64_t heads, const void *positions, int position_dtype, int64_t position_stride_axis,
                                           int64_t position_stride_token, const float *inv_freq, int64_t pairs,
                                           const int64_t *sections, int64_t axes, int interleaved, int cyclic,
                                           const qmm_kv_cache *cache, const qmm_kv_scales *scales, const void *slots, int slot_dtype,
                                           int64_t slot_stride, void *query_out, void *stream) {
    const std::string name("qmm_rotary_axes_quant_cache");
    qmm::RotaryParams p = {};
    QMM_REQUIRE(cache != nullptr && scales != nullptr, name + ": no cache or no scales given");
    QMM_REQUIRE(cache->pages >= 0 && cache->page_size >= 1 && cache->pages <= 0x7fffffff && cache->page_size <= 0x7fffffff,
                name + ": pages must be non-negative, their size positive");
    QMM_REQUIRE(cache->pages == 0 || (cache->key != cache->value && scales->key != scales->value),
                name + ": keys and values must have places of their own, but they, or their scales, begin at the same address");
    QMM_REQUIRE((reinterpret_cast<uintptr_t>(scales->key) & 3) == 0 && (reinterpret_cast<uintptr_t>(scales->value) & 3) == 0,
                name + ": scales must begin at 4-byte boundaries");
    QMM_REQUIRE(slot_dtype == QMM_DTYPE_I32 || slot_dtype == QMM_DTYPE_I64, name + ": slots must be int32 or int64");
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
    qmm::QuantParams out;
    out.k_scale = const_cast<float *>(scales->key);
    out.v_scale = const_cast<float *>(scales->value);
    out.ks_sb = scales->key_stride_page;
    out.ks_st = scales->key_stride_place;
    out.ks_sh = scales->key_stride_head;
    out.vs_sb = scales->value_stride_page;
    out.vs_st = scales->value_stride_place;
    out.vs_sh = scales->value_stride_head;
    const int rc = qmm::take_sizes(name.c_str(), p, tokens, heads, cache->kv_heads, cache->dim, pairs, sections, axes, position_dtype);
    if (rc != QMM_OK) return rc;
    if (tokens == 0 || cache->dim == 0) return QMM_OK;
    const cudaStream_t on = static_cast<cudaStream_t>(stream);
    if (dtype == QMM_DTYPE_BF16) return qmm::launch_quant<__nv_bfloat16>(p, out, tokens, on);
    if (dtype == QMM_DTYPE_F16) return qmm::launch_quant<__half>(p, out, tokens, on);
    if (dtype == QMM_DTYPE_F32) return qmm::launch_quant<float>(p, out, tokens, on);
    return fail(QMM_ERR_INVALID_ARGUMENT, name + ": the tensors must be bf16, f16 or f32");
}
