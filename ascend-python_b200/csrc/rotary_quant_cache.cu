// Rotary positions with the write into an int8 paged key-value cache (npu_rotary_axes_quant_cache).
//
// The query is turned as npu_rotary_axes turns it.  A row (token, head) of the turned key, and of the value, is written as
//     scale = max |y| / 127, rounded to fp32;   code = y / scale, to the nearest whole number (ties to even), in int8
// (0 where the scale is 0 or not finite), without a rounding of y between.
//
// The keys' rotation, the maximum and the quotient are in 64 bits: a value next to the border of two codes then has the code of
// the definition, whichever kernel or order of operations made it, where fp32 angles alone (off by 2^-25 half turns) move a code in
// some 2^16.  Positions times frequencies are exact there up to positions of 2^29.  The quotient is a product with the
// reciprocal, corrected by its remainder, which an fma gives without a rounding, so that one that is a tie comes out as one (P. Markstein, Computation of
// elementary functions on the IBM RISC System/6000 processor, 1990); reciprocals come from fp32 ones by Newton's iteration, r + r (1 - s r), whose last
// step's correction is kept beside the rounded sum.  Codes come out of the quotient's sum with 1.5 * 2^52, which has them in its low bits.
//
// HBM bounds it (28 us for 8192 tokens, 32 + 8 heads of 128) less than its instructions do: 45.8 us (two thirds of the issue slots; then the barrier between sines and rows), of which 30 without the rows that are
// quantized, each 8 lanes' work of some 400 instructions in 64 bits for keys and 250 for values.
#include "rotary_axes.cuh"

namespace qmm {

namespace {

struct QuantParams {
    float *k_scale, *v_scale;
    int64_t ks_sb, ks_st, ks_sh, vs_sb, vs_st, vs_sh;
};

// The cosine and sine of a token's pair, in 32 bits as npu_rotary_axes has them, and in 64.  For these the half turns are made of two
// numbers: the product with 1 / pi in 64 bits, and what it was rounded by (T. Dekker's exact product, 1971, with an fma) together with the next 53 bits of 1 / pi.  False: the frequency is not
// finite, and all four are NaN.
__device__ __forceinline__ bool make_turns(const RotaryParams &p, int64_t token, int pair, float *c, float *s, double *c64, double *s64) {
    const int64_t place = load_index(p.positions, axis_of(p, pair) * p.pos_sa + token * p.pos_st, p.wide_positions);
    const double angle = static_cast<double>(place) * static_cast<double>(__ldg(p.inv_freq + pair));
    const double half_turns = angle * 0.31830988618379067154, rest = half_turns - 2.0 * rint(0.5 * half_turns);
    sincospif(static_cast<float>(rest), s, c);
    sincospi(rest + fma(angle, -1.9678676675182486e-17, fma(angle, 0.31830988618379067154, -half_turns)), s64, c64);
    return rest == rest;
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
    double rest;     // of the inverse, beyond its 53 bits (of usual scales)
};
// From the largest magnitudes of the lanes of a row: `lanes` of them, a power of two.
__device__ __forceinline__ RowScale make_scale(unsigned long long most, int lanes, uint32_t mask) {
    for (int o = lanes >> 1; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(mask, most, o));
    RowScale r;
    r.scale = static_cast<float>(__longlong_as_double(static_cast<long long>(most)) / 127.0);
    r.inverse = r.scale > 0.0f && r.scale <= 3.402823466e38f ? 1.0 / static_cast<double>(r.scale) : 0.0;
    return r;
}
// From a row's largest magnitude, for scales that are neither near 0 nor very large (usual): the same by products.
__device__ __forceinline__ bool is_usual(float most) { return most >= 0x1p-90f && most <= 0x1p90f; }
__device__ __forceinline__ RowScale usual_scale(double most) {
    const double about = most * (1.0 / 127.0);
    RowScale r;
    r.scale = static_cast<float>(fma(fma(-about, 127.0, most), 1.0 / 127.0, about));
    const double scale = static_cast<double>(r.scale);
    double inverse = static_cast<double>(__frcp_rn(r.scale));
    inverse = fma(fma(-scale, inverse, 1.0), inverse, inverse);
    r.inverse = fma(fma(-scale, inverse, 1.0), inverse, inverse);
    r.rest = fma(-scale, r.inverse, 1.0) * r.inverse;
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
    for (int i = threadIdx.x; i < p.pairs; i += kThreads) make_turns(p, token, i, s_cos + i, s_sin + i, s_cos64 + i, s_sin64 + i);
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
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) w[i] = make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ void store(T *dst) const {
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) reinterpret_cast<uint4 *>(dst)[i] = w[i];
    }
    // The largest magnitude, as the bits of a float: magnitudes have the order of whole numbers.
    __device__ __forceinline__ uint32_t largest() const {
        const uint32_t *x = reinterpret_cast<const uint32_t *>(w);
        uint32_t m = 0;
        if (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < static_cast<int>(2 * sizeof(T)); ++i) m = max(m, x[i] & 0x7fffffffu);
            return m;
        }
#pragma unroll
        for (int i = 0; i < static_cast<int>(2 * sizeof(T)); ++i) m = __vmaxu2(m, x[i] & 0x7fff7fffu);
        m = max(m & 0xffffu, m >> 16);
        const unsigned short one = static_cast<unsigned short>(m);
        return __float_as_uint(to_float(*reinterpret_cast<const T *>(&one)));
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

// Vectors of eight elements.  A part of a row is, with halves, the vector of the first elements of its pairs and that of the second
// ones, or one vector behind the pairs; interleaved, one vector.  2^log_lanes lanes of a warp, as many as parts or
// more, have a row, and find its maximum together.
template <bool INTERLEAVED>
struct Parts {
    int lanes, part, e0, e1, pair0;  // lanes of a row, the lane's part, where its vectors begin, and its pairs
    bool active, turns, two;
    uint32_t mask;  // the row's lanes in the warp
    __device__ __forceinline__ Parts(const RotaryParams &p, int log_lanes) {
        const int turning = INTERLEAVED ? 2 * p.pairs / 8 : p.pairs / 8;  // parts of a row that turn
        lanes = 1 << log_lanes;
        part = threadIdx.x & (lanes - 1);
        active = part < (INTERLEAVED ? p.dim / 8 : turning + (p.dim - 2 * p.pairs) / 8);
        turns = part < turning;
        two = !INTERLEAVED && turns;
        e0 = (INTERLEAVED || turns ? part : part + turning) * 8;
        e1 = e0 + p.pairs;
        pair0 = INTERLEAVED ? e0 / 2 : e0;
        mask = (lanes == 32 ? 0xffffffffu : (1u << lanes) - 1) << (threadIdx.x & 31 & ~(lanes - 1));
    }
};
template <typename T, bool INTERLEAVED>
__device__ __forceinline__ void load_part(const Parts<INTERLEAVED> &parts, const T *src, Eight<T> &x, Eight<T> &y) {
    x.clear();
    y.clear();
    if (parts.active) x.load(src + parts.e0);
    if (parts.two) y.load(src + parts.e1);
}
// A query's part, turned (`turns`) by the cosines and sines of its pairs.
template <typename T, bool INTERLEAVED>
__device__ __forceinline__ void turn_part(const Parts<INTERLEAVED> &parts, Eight<T> &x, Eight<T> &y, const float *cosine, const float *sine, T *dst) {
    if (parts.turns) {
        float a[8], b[8];
        x.unpack(a);
        if (INTERLEAVED) {
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                b[j] = turned_first(a[j], a[j + 1], cosine[j / 2], sine[j / 2]);
                b[j + 1] = turned_second(a[j], a[j + 1], cosine[j / 2], sine[j / 2]);
            }
            x.pack(b);
        } else {
            y.unpack(b);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float one = a[j];
                a[j] = turned_first(one, b[j], cosine[j], sine[j]);
                b[j] = turned_second(one, b[j], cosine[j], sine[j]);
            }
            x.pack(a);
            y.pack(b);
        }
    }
    if (parts.active) x.store(dst + parts.e0);
    if (parts.two) y.store(dst + parts.e1);
}

__device__ __forceinline__ uint32_t low_bytes(int a, int b, int c, int d) { return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410); }
__device__ __forceinline__ uint2 codes_of(const double (&y)[8], const RowScale &r) {
    int c[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = code_of(y[i], r);
    return make_uint2(low_bytes(c[0], c[1], c[2], c[3]), low_bytes(c[4], c[5], c[6], c[7]));
}
// The same for usual scales, which no quotient passes 127 with: the inverse has 106 bits, so that a tie comes out as one here too.
__device__ __forceinline__ uint2 usual_codes_of(const double (&y)[8], const RowScale &r) {
    int c[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = __double2loint(fma(y[i], r.inverse, y[i] * r.rest) + 6755399441055744.0);
    return make_uint2(low_bytes(c[0], c[1], c[2], c[3]), low_bytes(c[4], c[5], c[6], c[7]));
}

// (fmax, which looks for NaN, is twice as many instructions)
__device__ __forceinline__ double larger(double a, double b) { return b > a ? b : a; }

// A part of a key's or a value's row, as it is written: the codes, and the scale by the first of the row's lanes.  `finite`: the sines and cosines are, so
// that NaN comes from the row's own elements alone, in whose bits it shows (`larger` passes over it).
template <typename T, bool INTERLEAVED>
__device__ __forceinline__ void quantize_part(const Eight<T> &x, const Eight<T> &y, const Parts<INTERLEAVED> &parts, bool key, bool finite, const double *cosine,
                                              const double *sine, int8_t *dst, float *scale_at) {
    float f[8], g[8];
    x.unpack(f);
    y.unpack(g);
    uint32_t bits = x.largest();  // in which NaN is above infinity
    if (!INTERLEAVED) bits = max(bits, y.largest());
    if (!finite) bits = 0x7fffffffu;
    double a[8], b[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        a[j] = static_cast<double>(f[j]);
        b[j] = INTERLEAVED ? 0.0 : static_cast<double>(g[j]);
    }
    if (key && parts.turns) {
#pragma unroll
        for (int j = 0; j < 8; j += INTERLEAVED ? 2 : 1) {
            const double c = cosine[INTERLEAVED ? j / 2 : j], s = sine[INTERLEAVED ? j / 2 : j], one = a[j], other = INTERLEAVED ? a[j + 1] : b[j];
            a[j] = turned_first_64(one, other, c, s);
            (INTERLEAVED ? a[j + 1] : b[j]) = turned_second_64(one, other, c, s);
        }
    }
    double most = __uint_as_float(bits);
    if (key) {
        most = 0.0;
#pragma unroll
        for (int j = 0; j < 8; ++j) most = larger(most, fabs(a[j]));
        if (!INTERLEAVED) {
#pragma unroll
            for (int j = 0; j < 8; ++j) most = larger(most, fabs(b[j]));
        }
    }
    for (int o = parts.lanes >> 1; o > 0; o >>= 1) {
        bits = max(bits, __shfl_xor_sync(parts.mask, bits, o));
        most = larger(most, __shfl_xor_sync(parts.mask, most, o));
    }
    RowScale scale;
    uint2 codes[2];
    if (__builtin_expect(bits < 0x7f800000u && is_usual(static_cast<float>(most)), 1)) {
        scale = usual_scale(most);
        codes[0] = usual_codes_of(a, scale);
        if (!INTERLEAVED) codes[1] = usual_codes_of(b, scale);
    } else {
        unsigned long long all = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) all = max(all, max(magnitude(a[j]), magnitude(b[j])));
        scale = make_scale(all, parts.lanes, parts.mask);
        codes[0] = codes_of(a, scale);
        if (!INTERLEAVED) codes[1] = codes_of(b, scale);
    }
    if (parts.active) *reinterpret_cast<uint2 *>(dst + parts.e0) = codes[0];
    if (parts.two) *reinterpret_cast<uint2 *>(dst + parts.e1) = codes[1];
    if (parts.part == 0) *scale_at = scale.scale;
}

// TOKENS a CTA: two where there are enough (8192 tokens, 32 + 8 heads of 128, bf16: one token 59 us, two 45.8, three 51; a warp a token, without
// a barrier, 50).  The barrier finds out whether all turns are finite (44.5 without that; the rows' lanes looking at their own cosines 46.2, CTAs
// that have others going another way 47 and more).  The first row of the query for each token and the first one that is quantized are under way while the sines and
// cosines are made.  Four CTAs an SM for two tokens (three: 47.5); few tokens need no more than one (64 registers cost 64 tokens 0.3 of 3.4 us).
template <typename T, bool INTERLEAVED, int TOKENS>
__global__ void __launch_bounds__(kThreads, TOKENS == 1 ? 1 : 4)
rotary_quant_vec_kernel(const __grid_constant__ RotaryParams p, const __grid_constant__ QuantParams out, int64_t tokens, int log_lanes) {
    __shared__ __align__(16) float s_cos[TOKENS][kMostPairs], s_sin[TOKENS][kMostPairs];
    __shared__ __align__(16) double s_cos64[TOKENS][kMostPairs], s_sin64[TOKENS][kMostPairs];
    // where a token's keys and values go in the cache (null: nowhere), and their scales
    __shared__ int8_t *s_codes[TOKENS][2];
    __shared__ float *s_scales[TOKENS][2];
    pdl_launch_dependents();
    pdl_wait();
    const int64_t token0 = static_cast<int64_t>(blockIdx.x) * TOKENS;
    const int here = static_cast<int>(min(static_cast<int64_t>(TOKENS), tokens - token0));
    const Parts<INTERLEAVED> parts(p, log_lanes);
    const int row0 = threadIdx.x >> log_lanes, step = kThreads >> log_lanes;
    Eight<T> x[TOKENS], y[TOKENS], kept_x, kept_y;
    const T *q = static_cast<const T *>(p.q) + token0 * p.q_st + row0 * p.q_sh;
#pragma unroll
    for (int i = 0; i < TOKENS; ++i)
        if (i < here && row0 < p.heads) load_part(parts, q + i * p.q_st, x[i], y[i]);
    const int kept = 2 * p.kv_heads;
    // rows that are quantized: of each token its keys, then its values
    auto kept_row = [&](int token, int head) {
        return head < p.kv_heads ? static_cast<const T *>(p.k) + (token0 + token) * p.k_st + head * p.k_sh : static_cast<const T *>(p.v) + (token0 + token) * p.v_st + (head - p.kv_heads) * p.v_sh;
    };
    auto token_of = [&](int row) {
        int token = 0;
#pragma unroll
        for (int i = 1; i < TOKENS; ++i) token += row >= i * kept;
        return token;
    };
    if (row0 < kept * here) load_part(parts, kept_row(token_of(row0), row0 - token_of(row0) * kept), kept_x, kept_y);
    if (threadIdx.x < here) {
        int64_t block = 0, at = 0;
        const bool some = find_slot(p, token0 + threadIdx.x, &block, &at);
        s_codes[threadIdx.x][0] = some ? static_cast<int8_t *>(p.k_cache) + block * p.kc_sb + at * p.kc_st : nullptr;
        s_codes[threadIdx.x][1] = static_cast<int8_t *>(p.v_cache) + block * p.vc_sb + at * p.vc_st;
        s_scales[threadIdx.x][0] = out.k_scale + block * out.ks_sb + at * out.ks_st;
        s_scales[threadIdx.x][1] = out.v_scale + block * out.vs_sb + at * out.vs_st;
    }
    bool finite = true;
    for (int i = threadIdx.x; i < p.pairs * here; i += kThreads) {
        const int token = i / p.pairs, pair = i - token * p.pairs;
        finite &= make_turns(p, token0 + token, pair, &s_cos[token][pair], &s_sin[token][pair], &s_cos64[token][pair], &s_sin64[token][pair]);
    }
    finite = __syncthreads_and(finite);
    for (int row = row0; row < p.heads; row += step) {
#pragma unroll
        for (int i = 0; i < TOKENS; ++i) {
            if (i >= here) break;
            if (row != row0) load_part(parts, q + i * p.q_st, x[i], y[i]);
        }
#pragma unroll
        for (int i = 0; i < TOKENS; ++i) {
            if (i >= here) break;
            turn_part(parts, x[i], y[i], s_cos[i] + parts.pair0, s_sin[i] + parts.pair0, static_cast<T *>(p.q_out) + ((token0 + i) * p.heads + row) * p.dim);
        }
        q += step * p.q_sh;
    }
    for (int row = row0; row < kept * here; row += step) {
        const int token = token_of(row), at = row - token * kept;
        if (row != row0) load_part(parts, kept_row(token, at), kept_x, kept_y);
        if (s_codes[token][0] == nullptr) continue;
        const bool key = at < p.kv_heads;
        const int head = key ? at : at - p.kv_heads;
        quantize_part<T, INTERLEAVED>(kept_x, kept_y, parts, key, finite, s_cos64[token] + parts.pair0, s_sin64[token] + parts.pair0,
                                      s_codes[token][!key] + head * (key ? p.kc_sh : p.vc_sh), s_scales[token][!key] + head * (key ? out.ks_sh : out.vs_sh));
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
    QMM_CUDA_OK(launch_pdl(kern, many ? dim3(static_cast<unsigned>((tokens + kTokens - 1) / kTokens)) : grid, dim3(kThreads), 0, stream, p, out, tokens, log_lanes));
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
