// Attention of one new token a sequence over an int8 paged key-value cache (npu_paged_quant_attention).
//
// A key's row is its codes times its scale, a value's likewise, so a score is a sum of query times codes, times the key's scale,
// and the output a sum of weights times the values' scales, times codes.  Codes are exact in f16, so both products are mma.sync
// m16n8k16 on f16 with fp32 sums, and the scales stay in fp32 outside of them.
//
// Bound by HBM, of which it needs about half of what a 16-bit cache does; the arithmetic on a key is the same as there plus
// the codes' way to f16.  That is five instructions for four codes: one turns the signs, two put the bytes below 0x64 (f16: 1024 + u),
// two subtract 1152.  A key's four bytes of a lane, as ldmatrix brings them, are two pairs of neighbouring dimensions; the query's
// dimensions are put in the same order, and a value's byte pairs give sums of even and of odd dimensions, so nothing is shuffled.
//
// bf16 queries become f16 by a power of two for each row, so that its largest element lies in [2^7, 2^8): an element 2^-21 of that
// or larger is exact, a smaller one is off by at most 2^-32 of it.
//
// The weights of the second product, exp(score - maximum) * value scale, are multiplied by a power of two for each row that keeps
// the largest so far below f16's largest number and above 2^8; it moves with the maximum, or when a weight would pass that.  Rounding a weight is half a
// step of f16, 2^-11 of it, or 2^-33 of the largest one for those far below it.  The sum of the softmax takes them unrounded.
//
// Ranges, rings of tiles and the joining of parts are those of the 16-bit cache (paged_decode.cuh).  Three CTAs of four warps an SM
// where the sums' columns leave room (heads of up to 128): the warps' waits for their loads and for each other's products overlap.
#include "paged_decode.cuh"

namespace qmm {
namespace paged {

namespace {

constexpr int kSlots = 3;  // of a warp's ring: keys, values, the next keys
constexpr int kTileBytes = 4096;

// DP: the head dimension rounded up to 64, 128 or 256.
template <int DP>
struct Shape {
    static constexpr int kKeys = kTileBytes / DP;  // of a tile
    static constexpr int kWarps = 4;
    static constexpr int kCtas = 2;  // an SM
    static constexpr int kQuery = kRows * DP * 2;
    static constexpr int kScales = kSlots * kKeys * 4;
    static constexpr size_t kSmem = kWarps * (kSlots * kTileBytes + kQuery + kScales);
};

Plan make_plan(int64_t batch, int64_t heads, int64_t kv_heads, int64_t dim) {
    return make_plan(batch, heads, kv_heads, dim, dim > 128 ? Shape<256>::kCtas : Shape<128>::kCtas, Shape<128>::kWarps);
}

__device__ __forceinline__ void cp_async_4(uint32_t dst, const void *src, uint32_t bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ float2 load_shared_float2(uint32_t addr) {
    float2 v;
    asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ uint2 load_shared_uint2(uint32_t addr) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void load_shared_uint4(uint32_t (&v)[4], uint32_t addr) {
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void store_shared_uint4(uint32_t addr, const uint32_t (&v)[4]) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
}

// Two of four codes (their signs turned) as f16: those that `pick` names, each above 0x64.
template <uint32_t PICK>
__device__ __forceinline__ uint32_t codes_f16(uint32_t turned) {
    const uint32_t x = __byte_perm(turned, 0x64646464u, PICK);
    uint32_t y;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(y) : "r"(x), "r"(0x64806480u));
    return y;
}

// Two elements of a query's row as f16, times a power of two for bf16.
template <typename T>
__device__ __forceinline__ uint32_t query_f16(uint32_t w, float power);
template <>
__device__ __forceinline__ uint32_t query_f16<__half>(uint32_t w, float) { return w; }
template <>
__device__ __forceinline__ uint32_t query_f16<__nv_bfloat16>(uint32_t w, float power) {
    return pack2<__half>(__uint_as_float(w << 16) * power, __uint_as_float(w & 0xffff0000u) * power);
}

// FAR: a warp may have more than kNear places.
template <typename T, int DP, bool FAR>
__global__ void __launch_bounds__(Shape<DP>::kWarps * 32, Shape<DP>::kCtas)
quant_decode_kernel(const __grid_constant__ Problem p, const __grid_constant__ QuantScales scales, const __grid_constant__ Scratch scratch) {
    using S = Shape<DP>;
    constexpr int KEYS = S::kKeys;
    constexpr int kBlocks = KEYS / 8;                  // of 8 keys
    constexpr int kChunks = DP / 16;                   // 16-byte chunks of a row of codes
    constexpr int kLooks = KEYS > 32 ? KEYS / 32 : 1;  // places of a tile that a lane looks up (16 keys: every place twice)
    constexpr bool kKept = DP < 256;  // the query in registers; 256 columns of sums leave none
    constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ Part s_parts[2 * S::kWarps];
    const int warp = warp_id_uniform(), lane = threadIdx.x & 31;
    const int worker = blockIdx.x;
    const uint32_t ring = smem_u32(smem) + warp * (kSlots * kTileBytes);
    const uint32_t query = smem_u32(smem) + S::kWarps * (kSlots * kTileBytes) + warp * S::kQuery;
    const uint32_t scale_ring = smem_u32(smem) + S::kWarps * (kSlots * kTileBytes + S::kQuery) + warp * S::kScales;
    pdl_launch_dependents();
    pdl_wait();

    const int tiles = (p.group + kRows - 1) / kRows;
    const int items = p.kv_heads * tiles;
    const int row_chunks = p.dim / 16;
    // The running maximum is one of unscaled scores, which takes a positive scale: a negative one's sign goes to the query, and
    // for a scale of 0 the query is 0.
    const float factor = p.scale * kLog2e;
    const float scale = factor == 0.0f ? 1.0f : fabsf(factor);
    const uint32_t query_and = factor == 0.0f ? 0u : 0xffffffffu, query_xor = factor < 0.0f ? 0x80008000u : 0u;

    const List list = make_list<KEYS>(p, scratch, items);
    if (!scratch.by_item && threadIdx.x == 0) scratch.cut[worker] = make_int4(-1, 0, 0, 0);

    // one round for the CTA's range; where head tiles are whole, one for each that the CTA has
    for (int64_t round = worker; round < (list.whole ? list.all_items : worker + 1); round += scratch.workers) {
        if (threadIdx.x < 2 * S::kWarps) s_parts[threadIdx.x].valid = 0;
        Piece load;
        int64_t end;
        begin_round<T, KEYS, S::kWarps>(p, scratch, list, round, tiles, load, end);
        Piece piece = load;
        bool more = load.to > load.from;
        bool working = more;
        __syncthreads();  // the parts' flags are clear

        // ---- loads: the query with a piece's first keys, then keys and values of a tile in turn, each with its scales ----
        int at = load.from;
        int at_place[kLooks], entry[kLooks];
        auto look_up = [&] {
            const int first = at < load.s.sink_tiles ? at * KEYS : (load.s.first + at - load.s.sink_tiles) * KEYS;
#pragma unroll
            for (int i = 0; i < kLooks; ++i) {
                const int j = first + 32 * i + (lane & (KEYS - 1));
                entry[i] = -1;
                if (more && j < load.s.hi && (j < load.s.sink_end || j >= load.s.lo)) {
                    const int page = page_of(p, j);
                    at_place[i] = j - page * p.page;
                    entry[i] = __ldg(p.table + load.b * p.table_st + page);
                }
            }
        };
        if (more) look_up();
        int slot = 0, value_place[kLooks], value_entry[kLooks], value_head = -1;
        uint32_t value_seen[kLooks], seen[kLooks];
        // A lane always has the same chunk, of rows kStep apart.  Rows of 16 places lie evenly apart where a page holds a
        // multiple of 16 (tiles begin at multiples of 16), and take one address; else each row its own.
        constexpr int kStep = 32 / kChunks;
        const int my_key = lane / kChunks, my_chunk = lane % kChunks;
        const bool my_part = my_chunk < row_chunks;
        const int my_offset = my_part ? my_chunk * 16 : 0;
        const bool even = p.page % 16 == 0;
        // The swizzled place of a key's chunk: chunk ^ key % 8, or where two rows make 128 bytes, chunk ^ key / 2 % 4.  The bits of
        // kStep * i + my_key are those of both parts.
        constexpr int kTurn = DP == 64 ? 1 : 0, kTurns = DP == 64 ? 3 : 7;
        const uint32_t my_dst = my_key * DP + ((my_chunk ^ ((my_key >> kTurn) & kTurns)) << 4);
        auto copy_tile = [&](const void *cache, int64_t sb, int64_t st, int64_t sh, const float *cache_scale, int64_t scale_sb, int64_t scale_st, int64_t scale_sh) {
            const uint32_t dst = ring + slot * kTileBytes + my_dst;
            int64_t offset[kLooks];
            bool full = true;
#pragma unroll
            for (int l = 0; l < kLooks; ++l) {
                const bool ok = value_seen[l] >> lane & 1;
                offset[l] = ok ? value_entry[l] * sb + value_place[l] * st + value_head * sh : 0;
                full = full && value_seen[l] == 0xffffffffu;
                if (KEYS >= 32 || lane < KEYS)
                    cp_async_4(scale_ring + (slot * KEYS + 32 * l + lane) * 4,
                               cache_scale + (ok ? value_entry[l] * scale_sb + value_place[l] * scale_st + value_head * scale_sh : 0), ok ? 4 : 0);
            }
            const int8_t *base = static_cast<const int8_t *>(cache) + my_offset;
            if (__builtin_expect(even, 1)) {
                const int8_t *row[KEYS / 16];
#pragma unroll
                for (int h = 0; h < KEYS / 16; ++h) {
                    // from the first of them that is seen
                    const uint32_t of = value_seen[h / 2] >> 16 * (h % 2) & 0xffffu;
                    const int from = of != 0 ? __ffs(of) - 1 : 0;
                    row[h] = base + __shfl_sync(0xffffffffu, offset[h / 2], 16 * (h % 2) + from) + (my_key - from) * st;
                }
                if (my_part) {
                    if (__builtin_expect(full, 1)) {
#pragma unroll
                        for (int i = 0; i < KEYS / kStep; ++i) {
                            const int first = kStep * i;
                            cp_async_16((dst ^ (((first >> kTurn) & kTurns) << 4)) + first * DP, row[first / 16], 16);
                            row[first / 16] += kStep * st;
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < KEYS / kStep; ++i) {
                            const int first = kStep * i;
                            const bool ok = value_seen[first / 32] >> ((first & 31) + my_key) & 1;
                            cp_async_16((dst ^ (((first >> kTurn) & kTurns) << 4)) + first * DP, ok ? row[first / 16] : base, ok ? 16 : 0);
                            row[first / 16] += kStep * st;
                        }
                    }
                }
                return;
            }
#pragma unroll
            for (int i = 0; i < KEYS / kStep; ++i) {
                const int first = kStep * i, key = (first & 31) + my_key;
                const int8_t *row = base + __shfl_sync(0xffffffffu, offset[first / 32], key);
                if (my_part)
                    cp_async_16((dst ^ (((first >> kTurn) & kTurns) << 4)) + first * DP, row, value_seen[first / 32] >> key & 1 ? 16 : 0);
            }
        };
        auto copy_query = [&] {
            constexpr int kQueryChunks = DP / 8, kQueryStep = 32 / kQueryChunks;  // 16-byte chunks of a row, rows a step
            const int kvh = load.item / tiles, tile = load.item - kvh * tiles;
            const int rows = min(kRows, p.group - tile * kRows);
            const int key = lane / kQueryChunks, chunk = lane % kQueryChunks;
            const T *base = static_cast<const T *>(p.q) + load.b * p.q_st + (kvh * p.group + tile * kRows) * p.q_sh + (chunk < 2 * row_chunks ? chunk * 8 : 0);
#pragma unroll
            for (int i = 0; i < kRows / kQueryStep; ++i) {
                const int row = kQueryStep * i + key;
                const bool ok = row < rows && chunk < 2 * row_chunks;
                cp_async_16(query + row * (DP * 2) + ((chunk ^ (row & 7)) << 4), base + (ok ? row * p.q_sh : 0), ok ? 16 : 0);
            }
        };
        auto load_keys = [&] {
            value_head = -1;
            if (more) {
                if (at == load.from) copy_query();
#pragma unroll
                for (int l = 0; l < kLooks; ++l) {
                    value_seen[l] = __ballot_sync(0xffffffffu, entry[l] >= 0 && entry[l] < p.pages);
                    value_place[l] = at_place[l];
                    value_entry[l] = entry[l];
                }
                value_head = load.item / tiles;
                copy_tile(p.k, p.k_sb, p.k_st, p.k_sh, scales.k, scales.k_sb, scales.k_st, scales.k_sh);
                if (__builtin_expect(++at == load.to, 0)) {
                    more = next_piece<KEYS>(p, end, items, load);
                    at = load.from;
                }
                look_up();
            }
            cp_async_commit();
            slot = slot + 1 == kSlots ? 0 : slot + 1;
        };
        auto load_values = [&] {
            if (value_head >= 0) copy_tile(p.v, p.v_sb, p.v_st, p.v_sh, scales.v, scales.v_sb, scales.v_st, scales.v_sh);
            cp_async_commit();
            slot = slot + 1 == kSlots ? 0 : slot + 1;
        };
        if (working) {
            load_keys();
            load_values();
        }

        // ---- products ----
        const int r0 = lane >> 2, c0 = (lane & 3) * 2;
        int use_slot = 0;
        uint32_t q[kKept ? DP / 16 : 1][4];
        float row_scale[2] = {scale, scale};
        // The query's rows as first operands, dimensions 16 ks + 4 (lane % 4) ... + 3 of a row a lane; where they are not kept in registers, into
        // the rows' place.
        auto take_query = [&] {
            uint32_t x[DP / 16][4];
            const uint32_t row = query + r0 * (DP * 2) + (lane & 1) * 8;
#pragma unroll
            for (int ks = 0; ks < DP / 16; ++ks) {
                const uint32_t chunk = ((2 * ks + (lane >> 1 & 1)) ^ r0) << 4;
                const uint2 a = load_shared_uint2(row + chunk), b = load_shared_uint2(row + 8 * (DP * 2) + chunk);
                x[ks][0] = a.x;
                x[ks][1] = b.x;
                x[ks][2] = a.y;
                x[ks][3] = b.y;
            }
            float power[2] = {1.0f, 1.0f};
            if (kBf16) {
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    float most = 0.0f;
#pragma unroll
                    for (int ks = 0; ks < DP / 16; ++ks) {
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const uint32_t w = x[ks][2 * i + r];
                            most = fmaxf(most, fmaxf(fabsf(__uint_as_float(w << 16)), fabsf(__uint_as_float(w & 0xffff0000u))));
                        }
                    }
                    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
                    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
                    // 2^e, e <= 127, and 2^-e
                    const int e = min(134 - static_cast<int>(__float_as_uint(most) >> 23), 127);
                    power[r] = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
                    row_scale[r] = scale * (e == 127 ? 0x1p-127f : __uint_as_float(static_cast<uint32_t>(127 - e) << 23));
                }
            }
#pragma unroll
            for (int ks = 0; ks < DP / 16; ++ks) {
#pragma unroll
                for (int i = 0; i < 4; ++i) x[ks][i] = (query_f16<T>(x[ks][i], power[i & 1]) & query_and) ^ query_xor;
                if (kKept) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) q[kKept ? ks : 0][i] = x[ks][i];
                }
            }
            if (!kKept) {
                __syncwarp();
#pragma unroll
                for (int ks = 0; ks < DP / 16; ++ks) store_shared_uint4(query + (ks * 32 + lane) * 16, x[ks]);
                __syncwarp();
            }
        };
        // ldmatrix addresses of a tile, keys and values alike: 8 keys x 16 bytes a matrix; 16 keys: of two chunks
        const int lane_key = KEYS == 16 ? (lane >> 3 & 1) * 8 + (lane & 7) : lane;
        const uint32_t lane_tile = lane_key * DP + (((((KEYS == 16 ? lane >> 4 : 0)) ^ ((lane_key >> kTurn) & kTurns))) << 4);
        constexpr int kAtOnce = KEYS == 16 ? 2 : 1;  // chunks of an ldmatrix
        while (working) {
            float o[DP / 8][4];
#pragma unroll
            for (int n = 0; n < DP / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f;
            float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.0f, 0.0f};
            // lift: the power of two of a row's weights; big: the largest of the lane's, so lifted
            float lift[2] = {1.0f, 1.0f}, big[2] = {0.0f, 0.0f};
            // A lane's sums n, n + 1 of a row, together those of dimensions 4 * (lane % 4) ... + 3 of 16.
            auto sums_of = [&](int n, int r) { return make_float4(o[n][2 * r], o[n + 1][2 * r], o[n][2 * r + 1], o[n + 1][2 * r + 1]); };
            // A long piece adds what it has to fp32 sums in its part of the workspace and begins again from 0 (back: the other way round).
            auto put_by = [&](bool first, bool back) {
                const int rows = min(kRows, p.group - piece.item % tiles * kRows);
                const int64_t part0 = ((static_cast<int64_t>(worker) * S::kWarps + warp) * 2 + (piece.from == 0)) * scratch.rows;
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const int row = r0 + r * 8;
                    float *sums = scratch.part + (part0 + row) * p.dim + 2 * c0;
                    const float down = 1.0f / lift[r], now = top[r] * row_scale[r];
                    float keep = 1.0f;
                    if (row < rows && !first && top[r] != -INFINITY) keep = exp2_fast(scratch.stat[part0 + row].x - now);
                    __syncwarp();
                    if (row < rows && (lane & 3) == 0) scratch.stat[part0 + row].x = now;
#pragma unroll
                    for (int n = 0; n < DP / 8; n += 2) {
                        float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        if (row < rows && n * 8 < p.dim) {
                            if (!first) x = *reinterpret_cast<const float4 *>(sums + n * 8);
                            const float4 y = sums_of(n, r);
                            x = make_float4(fmaf(x.x, keep, y.x * down), fmaf(x.y, keep, y.y * down), fmaf(x.z, keep, y.z * down), fmaf(x.w, keep, y.w * down));
                            if (!back) *reinterpret_cast<float4 *>(sums + n * 8) = x;
                        }
                        o[n][2 * r] = back ? x.x : 0.0f;
                        o[n + 1][2 * r] = back ? x.y : 0.0f;
                        o[n][2 * r + 1] = back ? x.z : 0.0f;
                        o[n + 1][2 * r + 1] = back ? x.w : 0.0f;
                    }
                    if (back) lift[r] = 1.0f;
                }
            };
            for (int g = piece.from; g < piece.to; ++g) {
                if (FAR && g != piece.from && (g - piece.from) % (kRun / KEYS) == 0) put_by(g - piece.from == kRun / KEYS, false);
                // scores of 16 rows x KEYS keys: accumulators of 8 keys
                float s[kBlocks][4];
#pragma unroll
                for (int n = 0; n < kBlocks; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
                cp_async_wait<kSlots - 2>();
                __syncwarp();
                bool all_seen = true;
#pragma unroll
                for (int l = 0; l < kLooks; ++l) {
                    seen[l] = value_seen[l];
                    all_seen = all_seen && seen[l] == 0xffffffffu;
                }
                if (g == piece.from) take_query();
                if (kKept) load_keys();  // into the slot of the values before
                const uint32_t keys = ring + use_slot * kTileBytes + lane_tile;
                const uint32_t key_scales = scale_ring + (use_slot * KEYS + c0) * 4;
                use_slot = use_slot + 1 == kSlots ? 0 : use_slot + 1;
#pragma unroll
                for (int ks = 0; ks < DP / 16; ks += kAtOnce) {
                    if (ks >= row_chunks) break;
                    uint32_t qk[kAtOnce][4];
#pragma unroll
                    for (int c = 0; c < kAtOnce; ++c) {
                        if (kKept) {
#pragma unroll
                            for (int i = 0; i < 4; ++i) qk[c][i] = q[kKept ? ks + c : 0][i];
                        } else {
                            load_shared_uint4(qk[c], query + ((ks + c) * 32 + lane) * 16);
                        }
                    }
#pragma unroll
                    for (int n = 0; n < kBlocks * kAtOnce; n += 4) {
                        uint32_t w[4];
                        ldmatrix_x4(w, (keys ^ (ks << 4)) + n * 8 * DP);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            w[i] ^= 0x80808080u;
                            mma_16816<__half>(s[(n + i) % kBlocks], qk[(n + i) / kBlocks], codes_f16<0x4140>(w[i]), codes_f16<0x4342>(w[i]));
                        }
                    }
                }
                if (!kKept) {
                    __syncwarp();  // the query may be overwritten
                    load_keys();
                }
#pragma unroll
                for (int n = 0; n < kBlocks; ++n) {
                    const float2 by = load_shared_float2(key_scales + n * 32);
                    s[n][0] *= by.x;
                    s[n][1] *= by.y;
                    s[n][2] *= by.x;
                    s[n][3] *= by.y;
                }
                if (__builtin_expect(!all_seen, 0)) {
#pragma unroll
                    for (int n = 0; n < kBlocks; ++n) {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (!(seen[n / 4] >> (n % 4 * 8 + c0 + (i & 1)) & 1)) s[n][i] = -INFINITY;
                    }
                }
                float most[2] = {-INFINITY, -INFINITY};
#pragma unroll
                for (int n = 0; n < kBlocks; ++n) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) most[i >> 1] = fmaxf(most[i >> 1], s[n][i]);
                }
                bool moved = false;
                float base[2], keep[2];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    most[r] = fmaxf(most[r], __shfl_xor_sync(0xffffffffu, most[r], 1));
                    most[r] = fmaxf(most[r], __shfl_xor_sync(0xffffffffu, most[r], 2));
                    const float now = fmaxf(top[r], most[r]);
                    base[r] = now == -INFINITY ? 0.0f : now * row_scale[r];
                    keep[r] = exp2_fast(fmaf(top[r], row_scale[r], -base[r]));
                    moved |= now != top[r];
                    top[r] = now;
                    sum[r] *= keep[r];
                    big[r] *= keep[r];
                }
#pragma unroll
                for (int n = 0; n < kBlocks; ++n) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        s[n][i] = exp2_fast(fmaf(s[n][i], row_scale[i >> 1], -base[i >> 1]));
                        sum[i >> 1] += s[n][i];
                    }
                }
                cp_async_wait<kSlots - 2>();
                __syncwarp();
                load_values();  // into the slot of the keys
                const uint32_t value_scales = scale_ring + (use_slot * KEYS + c0) * 4;
#pragma unroll
                for (int n = 0; n < kBlocks; ++n) {
                    const float2 by = load_shared_float2(value_scales + n * 32);
                    s[n][0] *= by.x * lift[0];
                    s[n][1] *= by.y * lift[0];
                    s[n][2] *= by.x * lift[1];
                    s[n][3] *= by.y * lift[1];
#pragma unroll
                    for (int i = 0; i < 4; ++i) big[i >> 1] = fmaxf(big[i >> 1], fabsf(s[n][i]));
                }
                moved |= fmaxf(big[0], big[1]) > 60000.0f;
                if (__builtin_expect(__any_sync(0xffffffffu, moved), 0)) {
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        big[r] = fmaxf(big[r], __shfl_xor_sync(0xffffffffu, big[r], 1));
                        big[r] = fmaxf(big[r], __shfl_xor_sync(0xffffffffu, big[r], 2));
                        float more_lift = 1.0f;
                        if (big[r] > 60000.0f || (big[r] < 256.0f && big[r] > 0.0f)) {
                            // to [2^11, 2^12), as far as lift stays finite
                            const int e = 138 - static_cast<int>(__float_as_uint(big[r]) >> 23);
                            const int has = static_cast<int>(__float_as_uint(lift[r]) >> 23) - 127;
                            more_lift = __uint_as_float(static_cast<uint32_t>(127 + max(-126 - has, min(min(e, 127), 127 - has))) << 23);
                        }
                        lift[r] *= more_lift;
                        big[r] *= more_lift;
                        keep[r] *= more_lift;
#pragma unroll
                        for (int n = 0; n < kBlocks; ++n) {
                            s[n][2 * r] *= more_lift;
                            s[n][2 * r + 1] *= more_lift;
                        }
#pragma unroll
                        for (int n = 0; n < DP / 8; ++n) {
                            o[n][2 * r] *= keep[r];
                            o[n][2 * r + 1] *= keep[r];
                        }
                    }
                }
                // the weights as they lie are the second product's first operand
                uint32_t a[KEYS / 16][4];
#pragma unroll
                for (int n = 0; n < kBlocks; ++n) {
#pragma unroll
                    for (int r = 0; r < 2; ++r) a[n >> 1][(n & 1) * 2 + r] = pack2<__half>(s[n][2 * r], s[n][2 * r + 1]);
                }
                const uint32_t values = ring + use_slot * kTileBytes + lane_tile;
                use_slot = use_slot + 1 == kSlots ? 0 : use_slot + 1;
#pragma unroll
                for (int ks = 0; ks < DP / 16; ks += kAtOnce) {
                    if (ks >= row_chunks) break;
#pragma unroll
                    for (int n = 0; n < kBlocks * kAtOnce; n += 4) {
                        uint32_t w[4];
                        ldmatrix_x4_trans(w, (values ^ (ks << 4)) + n * 8 * DP);
#pragma unroll
                        for (int i = 0; i < 4; ++i) w[i] ^= 0x80808080u;
#pragma unroll
                        for (int i = 0; i < 4; i += 2) {
                            const int to = 2 * (ks + (n + i) / kBlocks), k = (n + i) % kBlocks / 2;
                            mma_16816<__half>(o[to], a[k], codes_f16<0x4240>(w[i]), codes_f16<0x4240>(w[i + 1]));
                            mma_16816<__half>(o[to + 1], a[k], codes_f16<0x4341>(w[i]), codes_f16<0x4341>(w[i + 1]));
                        }
                    }
                }
            }

            if (FAR && piece.to - piece.from > kRun / KEYS) put_by(false, true);

            // ---- the piece's end: rows to the outputs, or sums to the workspace ----
            const int kvh = piece.item / tiles, tile = piece.item - kvh * tiles;
            const int rows = min(kRows, p.group - tile * kRows);
            const bool begins = piece.from == 0, ends = piece.to == piece.s.tiles;
            const int64_t row0 = static_cast<int64_t>(piece.b) * p.heads + kvh * p.group + tile * kRows;
            const int64_t part0 = ((static_cast<int64_t>(worker) * S::kWarps + warp) * 2 + begins) * scratch.rows;
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 1);
                sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 2);
                top[r] *= row_scale[r];
                const float down = 1.0f / lift[r];
                const int row = r0 + r * 8;
                if (row >= rows) continue;
                if (begins && ends) {
                    const float inv = sum[r] == 0.0f ? 0.0f : 1.0f / sum[r];
                    T *dst = static_cast<T *>(p.out) + (row0 + row) * p.dim + 2 * c0;
#pragma unroll
                    for (int n = 0; n < DP / 8; n += 2) {
                        const float4 x = sums_of(n, r);
                        if (n * 8 < p.dim)
                            *reinterpret_cast<uint2 *>(dst + n * 8) = make_uint2(pack2<T>(x.x * down * inv, x.y * down * inv), pack2<T>(x.z * down * inv, x.w * down * inv));
                    }
                    if ((lane & 3) == 0) p.lse[row0 + row] = sum[r] == 0.0f ? -INFINITY : top[r] * kLn2 + logf(sum[r]);
                } else {
                    float *dst = scratch.part + (part0 + row) * p.dim + 2 * c0;
#pragma unroll
                    for (int n = 0; n < DP / 8; n += 2) {
                        const float4 x = sums_of(n, r);
                        if (n * 8 < p.dim) *reinterpret_cast<float4 *>(dst + n * 8) = make_float4(x.x * down, x.y * down, x.z * down, x.w * down);
                    }
                    if ((lane & 3) == 0) scratch.stat[part0 + row] = make_float2(top[r], sum[r]);
                }
            }
            if (lane == 0) {
                if (!(begins && ends))
                    s_parts[2 * warp + begins] = {1, piece.b, piece.item, begins, ends, list.whole ? worker : static_cast<int>((piece.at - piece.from + piece.s.tiles - 1) / list.range)};
                else if (scratch.by_item && !list.whole)
                    scratch.cut[static_cast<int64_t>(piece.b) * items + piece.item] = make_int4(-1, 0, 0, 0);
            }
            working = next_piece<KEYS>(p, end, items, piece);
        }
        cp_async_wait<0>();
        __syncthreads();
        add_parts<T, S::kWarps>(p, scratch, list, s_parts, tiles);
        __syncthreads();
    }
}

template <typename T, int DP, bool FAR>
int launch_decode_kernel(const Problem &p, const QuantScales &scales, const Plan &plan, const Scratch &scratch, cudaStream_t stream) {
    QMM_CUDA_OK(cudaFuncSetAttribute(quant_decode_kernel<T, DP, FAR>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(Shape<DP>::kSmem)));
    QMM_CUDA_OK(launch_pdl(quant_decode_kernel<T, DP, FAR>, dim3(plan.workers), dim3(Shape<DP>::kWarps * 32), Shape<DP>::kSmem, stream, p, scales, scratch));
    return QMM_OK;
}

template <typename T, int DP>
int launch(const Problem &p, const QuantScales &scales, const Plan &plan, const Scratch &scratch, cudaStream_t stream) {
    const bool far = is_far(p, plan, Shape<DP>::kWarps);
    const int rc = far ? launch_decode_kernel<T, DP, true>(p, scales, plan, scratch, stream) : launch_decode_kernel<T, DP, false>(p, scales, plan, scratch, stream);
    return rc != QMM_OK ? rc : launch_join<T>(p, plan, scratch, stream);
}

template <typename T>
int launch_t(const Problem &p, const QuantScales &scales, const Plan &plan, const Scratch &scratch, cudaStream_t stream) {
    if (p.dim <= 64) return launch<T, 64>(p, scales, plan, scratch, stream);
    if (p.dim <= 128) return launch<T, 128>(p, scales, plan, scratch, stream);
    return launch<T, 256>(p, scales, plan, scratch, stream);
}

}  // namespace

size_t quant_decode_workspace(int64_t batch, int64_t heads, int64_t kv_heads, int64_t dim) {
    return batch == 0 || heads == 0 ? 0 : make_plan(batch, heads, kv_heads, dim).bytes;
}

int launch_quant_decode(const Problem &p, const QuantScales &scales, int dtype, void *workspace, size_t workspace_bytes, cudaStream_t stream) {
    const Plan plan = make_plan(p.batch, p.heads, p.kv_heads, p.dim);
    if (workspace_bytes < plan.bytes || workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 15) != 0)
        return fail(QMM_ERR_WORKSPACE, "qmm_paged_quant_attention: needs a workspace of " + std::to_string(plan.bytes) + " bytes, 16-byte aligned");
    const Scratch scratch = lay_out(plan, workspace);
    return dtype == QMM_DTYPE_BF16 ? launch_t<__nv_bfloat16>(p, scales, plan, scratch, stream) : launch_t<__half>(p, scales, plan, scratch, stream);
}

}  // namespace paged
}  // namespace qmm
