// Reading an int8 paged key-value cache back into pages of another type (npu_paged_cache_dequant): place j of sequence b, code times
// scale, goes to place j of the sequence in a second block table.
//
// Bound by HBM: a code is read once, its value written once; the scales are a thirty-second of that or less.  The places of all
// sequences are one list, cut into equal ranges for the CTAs, wherever sequences begin and end, so ragged lengths load the GPU
// alike (ranges for single warps: 64 sequences of 500 to 8000 places, 8 heads of 128, 213 us, this way 187; 166 at the copy rate).  A warp's lanes are dealt out to the vectors of eight codes of a row, then to the heads, then to places, so that few or
// small heads fill it too.
#include "paged_common.cuh"

namespace qmm {
namespace paged {

namespace {

constexpr int kWarps = 8;
constexpr int kCtas = 4;  // an SM (with two rows ahead a lane; that call with 3 and 4 196 us, 4 and 4 208, 6 and 2 232, 2 and 4 223)

struct Side {
    void *k, *v;
    int64_t k_sb, k_st, k_sh, v_sb, v_st, v_sh;
    const int32_t *table;
    int64_t table_st, pages;
    int page, page_shift, capacity;
};

struct Copy {
    Side from, to;
    QuantScales scales;
    const int32_t *lens, *first;
    int batch, kv_heads, dim;
};

// Places [lo, hi) of sequence b are copied; both are at most a capacity, 2^31 - 256, so that a step past them is below 2^31.
__device__ __forceinline__ void places_of(const Copy &c, int b, int *lo, int *hi) {
    const int capacity = min(c.from.capacity, c.to.capacity);
    *lo = c.first != nullptr ? min(max(0, __ldg(c.first + b)), capacity) : 0;
    *hi = max(*lo, min(__ldg(c.lens + b), capacity));
}

__device__ __forceinline__ bool find_page(const Side &s, int b, int j, int64_t *block, int *at) {
    const int i = s.page_shift >= 0 ? j >> s.page_shift : j / s.page;
    const int32_t id = __ldg(s.table + b * s.table_st + i);
    *block = id;
    *at = j - i * s.page;
    return id >= 0 && id < s.pages;
}

// Four codes as floats.
__device__ __forceinline__ void unpack4(uint32_t w, float *f) {
    w ^= 0x80808080u;  // u = code + 128; 0x4b0000uu is 2^23 + u
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440 + i)) - 8388736.0f;
}

// A vector of codes, V of them (8, or 1 for any alignment).
template <int V>
struct Codes;
template <>
struct Codes<8> {
    uint2 w;
    __device__ __forceinline__ void load(const int8_t *src) { w = __ldg(reinterpret_cast<const uint2 *>(src)); }
    template <typename T>
    __device__ __forceinline__ void store(T *dst, float scale) const {
        float f[8];
        unpack4(w.x, f);
        unpack4(w.y, f + 4);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] *= scale;
        if constexpr (sizeof(T) == 4) {
            reinterpret_cast<float4 *>(dst)[0] = make_float4(f[0], f[1], f[2], f[3]);
            reinterpret_cast<float4 *>(dst)[1] = make_float4(f[4], f[5], f[6], f[7]);
        } else {
            *reinterpret_cast<uint4 *>(dst) = make_uint4(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]), pack2<T>(f[4], f[5]), pack2<T>(f[6], f[7]));
        }
    }
};
template <>
struct Codes<1> {
    int8_t w;
    __device__ __forceinline__ void load(const int8_t *src) { w = __ldg(src); }
    template <typename T>
    __device__ __forceinline__ void store(T *dst, float scale) const { *dst = from_float<T>(static_cast<float>(w) * scale); }
};

// Rows (keys and values) that a lane has under way at once.
constexpr int kAhead = 2;

// How a warp's lanes are dealt out: 2^log_row to a row, 2^log_heads rows side by side of a place, what is left to places.
struct Lanes {
    int log_row, log_heads;
};

template <typename T, int V>
__global__ void __launch_bounds__(kWarps * 32, kCtas) dequant_kernel(const __grid_constant__ Copy c, const __grid_constant__ Lanes lanes) {
    const int warp = warp_id_uniform(), lane = threadIdx.x & 31;
    pdl_launch_dependents();
    pdl_wait();
    int64_t total = 0;
    int lo = 0, hi = 0;  // of sequence `lane`, of up to 32
    for (int b = lane; b < c.batch; b += 32) {
        places_of(c, b, &lo, &hi);
        total += hi - lo;
    }
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    const int places_at_once = 32 >> (lanes.log_row + lanes.log_heads), step = kWarps * places_at_once;
    const int64_t range = (total + gridDim.x - 1) / gridDim.x;
    const int64_t end = min(total, (blockIdx.x + 1) * range), begin = blockIdx.x * range + warp * places_at_once;
    if (begin >= end) return;
    // the sequence and place where the range begins
    int first = 0;
    int64_t before = 0;
    for (int b0 = 0;; b0 += 32) {
        if (c.batch > 32) {
            lo = hi = 0;
            if (b0 + lane < c.batch) places_of(c, b0 + lane, &lo, &hi);
        }
        const int64_t mine = hi - lo;
        int64_t sum = mine;
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t left = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += left;
        }
        const uint32_t past = __ballot_sync(0xffffffffu, before + sum > begin);
        if (past != 0) {
            const int at = __ffs(past) - 1;
            first = b0 + at;
            before += __shfl_sync(0xffffffffu, sum - mine, at);
            lo = __shfl_sync(0xffffffffu, lo, at);
            hi = __shfl_sync(0xffffffffu, hi, at);
            break;
        }
        before += __shfl_sync(0xffffffffu, sum, 31);
    }
    const int heads_at_once = 1 << lanes.log_heads;
    const int slot = lane >> lanes.log_row, head0 = slot & (heads_at_once - 1);
    int s = first, s_hi = hi;
    int64_t n = begin + (slot >> lanes.log_heads);
    int j = lo + static_cast<int>(n - before);
    for (; n < end; n += step, j += step) {
        while (j >= s_hi) {
            const int over = j - s_hi;
            places_of(c, ++s, &j, &s_hi);
            j += over;
        }
        int64_t page, out;
        int at, out_at;
        if (!find_page(c.from, s, j, &page, &at) | !find_page(c.to, s, j, &out, &out_at)) continue;
        for (int e = (lane & ((1 << lanes.log_row) - 1)) * V; e < c.dim; e += 32 * V) {
            const int8_t *k = static_cast<const int8_t *>(c.from.k) + page * c.from.k_sb + at * c.from.k_st + head0 * c.from.k_sh + e;
            const int8_t *v = static_cast<const int8_t *>(c.from.v) + page * c.from.v_sb + at * c.from.v_st + head0 * c.from.v_sh + e;
            const float *k_scale = c.scales.k + page * c.scales.k_sb + at * c.scales.k_st + head0 * c.scales.k_sh;
            const float *v_scale = c.scales.v + page * c.scales.v_sb + at * c.scales.v_st + head0 * c.scales.v_sh;
            T *k_out = static_cast<T *>(c.to.k) + out * c.to.k_sb + out_at * c.to.k_st + head0 * c.to.k_sh + e;
            T *v_out = static_cast<T *>(c.to.v) + out * c.to.v_sb + out_at * c.to.v_st + head0 * c.to.v_sh + e;
            for (int head = head0; head < c.kv_heads; head += kAhead * heads_at_once) {
                Codes<V> x[kAhead], y[kAhead];
                float x_scale[kAhead], y_scale[kAhead];
#pragma unroll
                for (int i = 0; i < kAhead; ++i) {
                    if (head + i * heads_at_once >= c.kv_heads) break;
                    x[i].load(k);
                    y[i].load(v);
                    x_scale[i] = __ldg(k_scale);
                    y_scale[i] = __ldg(v_scale);
                    k += c.from.k_sh << lanes.log_heads;
                    v += c.from.v_sh << lanes.log_heads;
                    k_scale += c.scales.k_sh << lanes.log_heads;
                    v_scale += c.scales.v_sh << lanes.log_heads;
                }
#pragma unroll
                for (int i = 0; i < kAhead; ++i) {
                    if (head + i * heads_at_once >= c.kv_heads) break;
                    x[i].store(k_out, x_scale[i]);
                    y[i].store(v_out, y_scale[i]);
                    k_out += c.to.k_sh << lanes.log_heads;
                    v_out += c.to.v_sh << lanes.log_heads;
                }
            }
        }
    }
}

template <typename T>
int launch_t(const Copy &c, bool vectors, cudaStream_t stream) {
    auto kern = vectors ? dequant_kernel<T, 8> : dequant_kernel<T, 1>;
    const int row = c.dim / (vectors ? 8 : 1);
    Lanes lanes = {0, 0};
    while (lanes.log_row < 5 && 1 << lanes.log_row < row) ++lanes.log_row;
    while (lanes.log_row + lanes.log_heads < 5 && 1 << lanes.log_heads < c.kv_heads) ++lanes.log_heads;
    QMM_CUDA_OK(launch_pdl(kern, dim3(kCtas * sm_count()), dim3(kWarps * 32), 0, stream, c, lanes));
    return QMM_OK;
}

void take_table(Side *s, const qmm_kv_cache *cache, const int32_t *table, int64_t table_stride, int64_t max_pages) {
    s->k = const_cast<void *>(cache->key);
    s->v = const_cast<void *>(cache->value);
    s->k_sb = cache->key_stride_page;
    s->k_st = cache->key_stride_place;
    s->k_sh = cache->key_stride_head;
    s->v_sb = cache->value_stride_page;
    s->v_st = cache->value_stride_place;
    s->v_sh = cache->value_stride_head;
    s->table = table;
    s->table_st = table_stride;
    s->pages = cache->pages;
    s->page = static_cast<int>(cache->page_size);
    s->page_shift = -1;
    for (int i = 0; i < 31; ++i)
        if (s->page == 1 << i) s->page_shift = i;
    const int64_t capacity = cache->pages == 0 ? 0 : max_pages * cache->page_size;
    s->capacity = static_cast<int>(capacity < 0x7fffff00 ? capacity : 0x7fffff00);
}

bool begins_at(int bytes, int size, const void *base, int64_t a, int64_t b, int64_t c) {
    return (reinterpret_cast<uintptr_t>(base) & (bytes - 1)) == 0 && ((a | b | c) & (bytes / size - 1)) == 0;
}

}  // namespace

}  // namespace paged
}  // namespace qmm

using qmm::fail;

extern "C" int qmm_paged_cache_dequant(const qmm_kv_cache *cache, const qmm_kv_scales *scales, const int32_t *block_table,
                                       int64_t table_stride, int64_t max_pages, const int32_t *seq_lens, const int32_t *first_places,
                                       int64_t batch, const qmm_kv_cache *out, int out_dtype, const int32_t *out_table,
                                       int64_t out_table_stride, int64_t out_max_pages, void *stream) {
    using namespace qmm::paged;
    const std::string name("qmm_paged_cache_dequant");
    QMM_REQUIRE(cache != nullptr && scales != nullptr && out != nullptr, name + ": no cache, no scales or no output given");
    QMM_REQUIRE(batch >= 0 && max_pages >= 0 && out_max_pages >= 0 && cache->pages >= 0 && out->pages >= 0, name + ": sizes must be non-negative");
    QMM_REQUIRE(cache->page_size >= 1 && cache->page_size <= 0x7fffffff && out->page_size >= 1 && out->page_size <= 0x7fffffff,
                name + ": the page sizes must be positive");
    QMM_REQUIRE(batch <= 0x7fffff00 && max_pages <= 0x7fffffff && out_max_pages <= 0x7fffffff && cache->pages <= 0x7fffffff && out->pages <= 0x7fffffff,
                name + ": sizes out of range");
    QMM_REQUIRE(cache->kv_heads >= 1 && cache->kv_heads <= 65535 && cache->dim >= 1 && cache->dim <= 256,
                name + ": between 1 and 65535 heads, of a dimension up to 256");
    QMM_REQUIRE(cache->kv_heads == out->kv_heads && cache->dim == out->dim, name + ": cache and output must have the same heads and dimension");
    QMM_REQUIRE(out_dtype == QMM_DTYPE_BF16 || out_dtype == QMM_DTYPE_F16 || out_dtype == QMM_DTYPE_F32, name + ": the output must be bf16, f16 or f32");
    QMM_REQUIRE(out->pages == 0 || out->key != out->value, name + ": keys and values must have places of their own, but they begin at the same address");
    const int size = out_dtype == QMM_DTYPE_F32 ? 4 : 2;
    for (const void *x : {static_cast<const void *>(scales->key), static_cast<const void *>(scales->value), static_cast<const void *>(block_table),
                          static_cast<const void *>(seq_lens), static_cast<const void *>(first_places), static_cast<const void *>(out_table)})
        QMM_REQUIRE((reinterpret_cast<uintptr_t>(x) & 3) == 0, name + ": scales, tables and lengths must begin at 4-byte boundaries");
    QMM_REQUIRE(begins_at(size, size, out->key, 0, 0, 0) && begins_at(size, size, out->value, 0, 0, 0), name + ": the output must begin at a boundary of its type");
    if (batch == 0) return QMM_OK;
    Copy c;
    take_table(&c.from, cache, block_table, table_stride, max_pages);
    take_table(&c.to, out, out_table, out_table_stride, out_max_pages);
    c.scales = {scales->key, scales->value, scales->key_stride_page, scales->key_stride_place, scales->key_stride_head,
                scales->value_stride_page, scales->value_stride_place, scales->value_stride_head};
    c.lens = seq_lens;
    c.first = first_places;
    c.batch = static_cast<int>(batch);
    c.kv_heads = static_cast<int>(cache->kv_heads);
    c.dim = static_cast<int>(cache->dim);
    const bool vectors = c.dim % 8 == 0 && begins_at(8, 1, c.from.k, c.from.k_sb, c.from.k_st, c.from.k_sh) &&
                         begins_at(8, 1, c.from.v, c.from.v_sb, c.from.v_st, c.from.v_sh) &&
                         begins_at(16, size, c.to.k, c.to.k_sb, c.to.k_st, c.to.k_sh) && begins_at(16, size, c.to.v, c.to.v_sb, c.to.v_st, c.to.v_sh);
    const cudaStream_t on = static_cast<cudaStream_t>(stream);
    if (out_dtype == QMM_DTYPE_BF16) return launch_t<__nv_bfloat16>(c, vectors, on);
    if (out_dtype == QMM_DTYPE_F16) return launch_t<__half>(c, vectors, on);
    return launch_t<float>(c, vectors, on);
}
