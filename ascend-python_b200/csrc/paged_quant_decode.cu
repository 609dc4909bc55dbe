// Attention of one new token a sequence over an int8 paged key-value cache (npu_paged_quant_attention).
//
// A key's row is its codes times its scale, a value's likewise, so a score is a sum of query times codes, times the key's scale,
// and the output a sum of weights times the values' scales, times codes.  Codes are exact in f16, so both products are mma.sync
// m16n8k16 on f16 with fp32 sums, and the scales stay in fp32 outside of them.
//
// Bound by HBM, of which it needs about half of what a 16-bit cache does, so that the instructions on a key count twice as much.  Keys, then
// dimensions of the values, are the 16 rows of a product and query heads its 8 columns: groups of up to 8 heads, the usual ones, need
// half of the products, sums, registers and exponentials that heads as rows would (64 sequences of 500 to 8000 places, 64/8
// heads of 128: heads as rows 125 us).  The codes' way to f16 is five instructions for four: one turns the signs, two put the bytes
// below 0x64 (f16: 1024 + u), two subtract 1152.  A key's four bytes of a lane, as ldmatrix brings them, are two pairs of neighbouring
// dimensions; the query's dimensions are put in the same order.  A value's byte pairs, transposed, are rows of even and of odd
// dimensions, so nothing is shuffled; the weights change from rows of keys to rows of heads by movmatrix.
//
// bf16 queries become f16 by a power of two for each row, so that its largest element lies in [2^7, 2^8): an element 2^-21 of that
// or larger is exact, a smaller one is off by at most 2^-32 of it.
//
// The weights of the second product, exp(score - maximum) * value scale, are multiplied by a power of two for each head that keeps
// the largest so far below f16's largest number and above 2^8; it moves with the maximum, or when a weight would pass that.  Rounding a weight is half a
// step of f16, 2^-11 of it, or 2^-33 of the largest one for those far below it.  The sum of the softmax takes them unrounded.
//
// Places that are not seen have no part in a sum: their scores are -inf and their scales 0, whatever their codes are, which are finite.
// Ranges, rings of tiles and the joining of parts are those of the 16-bit cache (paged_decode.cuh).
#include "paged_decode.cuh"

namespace qmm {
namespace paged {

namespace {

constexpr int kSlots = 3;  // of a warp's ring: keys, values, the next keys
constexpr int kTileBytes = 4096;
constexpr int kDigits = 3;    // of an element of the query, 8 bits each
constexpr float kSlack = 3.0f;  // how far, in powers of two, scores may pass their base before it follows them

// DP: the head dimension rounded up to 64, 128 or 256.  NT: 8 * NT heads are a head tile's, 1 or 2.
template <int DP, int NT>
struct Shape {
    static constexpr int kKeys = kTileBytes / DP;  // of a tile
    static constexpr int kWarps = 4;
    static constexpr int kCtas = 2;  // an SM
    static constexpr bool kKept = NT * DP < 512;  // the query in registers, else as operands in shared memory
    static constexpr int kQuery = 8 * NT * DP * (kKept ? 2 : kDigits);
    static constexpr int kScales = kSlots * kKeys * 4;
    static constexpr size_t kSmem = kWarps * (kSlots * kTileBytes + kQuery + kScales);
};

// Groups of up to 8 heads take one column tile.
bool is_narrow(int64_t heads, int64_t kv_heads) { return heads <= 8 * kv_heads; }

Plan make_plan(int64_t batch, int64_t heads, int64_t kv_heads, int64_t dim) {
    const int ctas = is_narrow(heads, kv_heads) ? (dim > 128 ? Shape<256, 1>::kCtas : Shape<128, 1>::kCtas)
                                                : (dim > 128 ? Shape<256, 2>::kCtas : Shape<128, 2>::kCtas);
    return make_plan(batch, heads, kv_heads, dim, ctas, Shape<128, 1>::kWarps);
}

__device__ __forceinline__ void cp_async_4(uint32_t dst, const void *src, uint32_t bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ float load_shared_float(uint32_t addr) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ uint2 load_shared_uint2(uint32_t addr) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void store_shared_uint2(uint32_t addr, uint2 v) {
    asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(addr), "r"(v.x), "r"(v.y) : "memory");
}
// An 8 x 8 matrix of 16-bit elements, two neighbours of a row a lane, transposed.
__device__ __forceinline__ uint32_t transposed(uint32_t w) {
    uint32_t t;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(t) : "r"(w));
    return t;
}

// Two of four codes (their signs turned) as f16: those that PICK names, each below 0x64.
template <uint32_t PICK>
__device__ __forceinline__ uint32_t codes_f16(uint32_t turned) {
    const uint32_t x = __byte_perm(turned, 0x64646464u, PICK);
    uint32_t y;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(y) : "r"(x), "r"(0x64806480u));
    return y;
}

__device__ __forceinline__ void mma_i8(int (&c)[4], const uint32_t (&a)[4], uint2 b) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b.x), "r"(b.y));
}

// Two 16-bit elements as floats.
template <typename T>
__device__ __forceinline__ float2 two_floats(uint32_t w);
template <>
__device__ __forceinline__ float2 two_floats<__half>(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2 *>(&w)); }
template <>
__device__ __forceinline__ float2 two_floats<__nv_bfloat16>(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }

// One box of a cache, and how many bytes will come, on a barrier: by one lane of a converged warp.
__device__ __forceinline__ void expect_bytes_warp(uint32_t bar, uint32_t bytes) {
    asm volatile(
        "{\n\t"
        ".reg .pred e;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "@e mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n\t"
        "}\n" ::"r"(bar),
        "r"(bytes)
        : "memory");
}

// How a cache is copied: by boxes of `rows` places of a page and a head (TMA), or where rows is 0, row by row (cp.async).
struct Boxes {
    int rows;
    uint32_t *status;  // the device status word
};

// FAR: a warp may have more than kNear places.
template <typename T, int DP, int NT, bool FAR>
__global__ void __launch_bounds__(Shape<DP, NT>::kWarps * 32, Shape<DP, NT>::kCtas)
quant_decode_kernel(const __grid_constant__ Problem p, const __grid_constant__ QuantScales scales, const __grid_constant__ Scratch scratch,
                    const __grid_constant__ Boxes boxes, const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map) {
    using S = Shape<DP, NT>;
    constexpr int KEYS = S::kKeys;
    constexpr int kSteps = DP / 16;                    // chunks of 16 dimensions, 16 bytes of codes
    constexpr int kTiles = KEYS / 16;                  // of 16 keys
    constexpr int kLooks = KEYS > 32 ? KEYS / 32 : 1;  // places of a tile that a lane looks up (16 keys: every place twice)
    constexpr bool kKept = S::kKept;
    // A tile's rows are 64 or 128 bytes, 256 columns two of those; chunk ^ key % 8, or where two rows make 128 bytes, chunk ^ key / 2 % 4.
    constexpr int kPitch = DP < 128 ? DP : 128, kRowChunks = kPitch / 16, kTurn = DP == 64 ? 1 : 0, kTurns = DP == 64 ? 3 : 7;
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ Part s_parts[2 * S::kWarps];
    __shared__ __align__(8) uint64_t s_full[S::kWarps][kSlots];
    __shared__ uint32_t s_abort;
    const int warp = warp_id_uniform(), lane = threadIdx.x & 31;
    const int worker = blockIdx.x;
    const uint32_t ring = smem_u32(smem) + warp * (kSlots * kTileBytes);
    const uint32_t query = smem_u32(smem) + S::kWarps * (kSlots * kTileBytes) + warp * S::kQuery;
    const uint32_t scale_ring = smem_u32(smem) + S::kWarps * (kSlots * kTileBytes + S::kQuery) + warp * S::kScales;
    const uint32_t full = smem_u32(&s_full[warp][0]);
    uint32_t phases = 0;  // a bit a slot
    if (threadIdx.x == 0) s_abort = 0;
    if (boxes.rows > 0 && lane < kSlots) mbar_init(full + lane * 8, 1);
    mbar_fence_init();
    pdl_launch_dependents();
    pdl_wait();

    const int tiles = (p.group + kRows - 1) / kRows;
    const int items = p.kv_heads * tiles;
    const int row_chunks = p.dim / 16;
    // The running maximum is one of unscaled scores, which takes a positive scale: a negative one's sign goes to the query, and
    // for a scale of 0 the query is 0.
    const float factor = p.scale * kLog2e;
    const float scale = factor == 0.0f ? 1.0f : fabsf(factor), sign = factor == 0.0f ? 0.0f : factor < 0.0f ? -1.0f : 1.0f;

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
        int at = load.from, load_head = load.item / tiles;
        const int box_rows = boxes.rows > 0 ? boxes.rows : 1;
        // a lane's place of the next tile: its page, if a place of its box is seen, and where it lies there; a bit a lane: whether it is seen itself
        int at_place[kLooks], entry[kLooks];
        uint32_t visible[kLooks];
        auto look_up = [&] {
            const int first = at < load.s.sink_tiles ? at * KEYS : (load.s.first + at - load.s.sink_tiles) * KEYS;
#pragma unroll
            for (int i = 0; i < kLooks; ++i) {
                const int j = first + 32 * i + (lane & (KEYS - 1)), box = j & -box_rows;
                visible[i] = __ballot_sync(0xffffffffu, j < load.s.hi && (j < load.s.sink_end || j >= load.s.lo));
                entry[i] = -1;
                const int page = page_of(p, j);
                at_place[i] = j - page * p.page;
                if (more && (box < load.s.sink_end || max(box, load.s.lo) < min(box + box_rows, load.s.hi))) entry[i] = __ldg(p.table + load.b * p.table_st + page);
            }
        };
        if (more) look_up();
        int slot = 0, value_place[kLooks], value_entry[kLooks], value_head = -1;
        uint32_t value_boxes[kLooks], value_seen[kLooks], seen[kLooks];  // a bit a place: its page is one, and it is seen
        auto copy_scales = [&](const float *of, int64_t sb, int64_t st, int64_t sh) {
#pragma unroll
            for (int l = 0; l < kLooks; ++l) {
                if (KEYS >= 32 || lane < KEYS) {
                    const bool ok = value_seen[l] >> lane & 1;
                    cp_async_4(scale_ring + (slot * KEYS + 32 * l + lane) * 4, of + (ok ? value_entry[l] * sb + value_place[l] * st + value_head * sh : 0), ok ? 4 : 0);
                }
            }
        };
        // Boxes of which a place is seen come whole.
        auto copy_boxes = [&](const CUtensorMap *map) {
            const uint32_t bar = full + slot * 8, dst = ring + slot * kTileBytes;
            int places = 0;
#pragma unroll
            for (int l = 0; l < kLooks; ++l) places += __popc(KEYS == 16 ? value_boxes[l] & 0xffffu : value_boxes[l]);
            expect_bytes_warp(bar, places * DP);
#pragma unroll
            for (int l = 0; l < kLooks; ++l) {
                for (int key = 0; key < (KEYS < 32 ? KEYS : 32); key += box_rows) {
                    if (!(value_boxes[l] >> key & 1)) continue;
                    const int page = __shfl_sync(0xffffffffu, value_entry[l], key), place = __shfl_sync(0xffffffffu, value_place[l], key);
#pragma unroll
                    for (int c = 0; c < DP / kPitch; ++c)
                        tma_load_4d_warp(dst + c * (KEYS * kPitch) + (32 * l + key) * kPitch, map, c * kPitch, place, value_head, page, bar);
                }
            }
        };
        // A lane always has the same chunk, of rows kStep apart.
        constexpr int kStep = 32 / kSteps;
        const int my_key = lane / kSteps, my_chunk = lane % kSteps;
        auto copy_rows = [&](const void *cache, int64_t sb, int64_t st, int64_t sh) {
            const uint32_t dst = ring + slot * kTileBytes + my_chunk / kRowChunks * (KEYS * kPitch);
            const int8_t *base = static_cast<const int8_t *>(cache) + value_head * sh + my_chunk * 16;
            int64_t offset[kLooks];
#pragma unroll
            for (int l = 0; l < kLooks; ++l) offset[l] = value_seen[l] >> lane & 1 ? value_entry[l] * sb + value_place[l] * st : 0;
#pragma unroll
            for (int i = 0; i < KEYS / kStep; ++i) {
                const int key = kStep * i + my_key;
                const int8_t *row = base + __shfl_sync(0xffffffffu, offset[kStep * i / 32], key & 31);
                if (my_chunk < row_chunks && (value_seen[kStep * i / 32] >> (key & 31) & 1))
                    cp_async_16(dst + key * kPitch + (((my_chunk ^ (key >> kTurn)) & kTurns) << 4), row, 16);
            }
        };
        auto copy_query = [&] {
            constexpr int kChunks = DP / 8, kHeads = 32 / kChunks;  // 16-byte chunks of a row, rows a step
            const int tile = load.item - load_head * tiles;
            const int rows = min(kRows, p.group - tile * kRows);
            const int row0 = lane / kChunks, chunk = lane % kChunks;
            const T *base = static_cast<const T *>(p.q) + load.b * p.q_st + (load_head * p.group + tile * kRows) * p.q_sh + (chunk < 2 * row_chunks ? chunk * 8 : 0);
#pragma unroll
            for (int i = 0; i < 8 * NT / kHeads; ++i) {
                const int row = kHeads * i + row0;
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
                    value_boxes[l] = __ballot_sync(0xffffffffu, entry[l] >= 0 && entry[l] < p.pages);
                    value_seen[l] = value_boxes[l] & visible[l];
                    value_place[l] = at_place[l];
                    value_entry[l] = entry[l];
                }
                value_head = load_head;
                copy_scales(scales.k, scales.k_sb, scales.k_st, scales.k_sh);
                if (boxes.rows > 0)
                    copy_boxes(&k_map);
                else
                    copy_rows(p.k, p.k_sb, p.k_st, p.k_sh);
                if (__builtin_expect(++at == load.to, 0)) {
                    more = next_piece<KEYS>(p, end, items, load);
                    at = load.from;
                    load_head = load.item / tiles;
                }
                look_up();
            }
            cp_async_commit();
            slot = slot + 1 == kSlots ? 0 : slot + 1;
        };
        auto load_values = [&] {
            if (value_head >= 0) {
                copy_scales(scales.v, scales.v_sb, scales.v_st, scales.v_sh);
                if (boxes.rows > 0)
                    copy_boxes(&v_map);
                else
                    copy_rows(p.v, p.v_sb, p.v_st, p.v_sh);
            }
            cp_async_commit();
            slot = slot + 1 == kSlots ? 0 : slot + 1;
        };
        if (working) {
            load_keys();
            load_values();
        }
        // for the next slot's tile
        int use_slot = 0;
        auto wait_tile = [&] {
            cp_async_wait<kSlots - 2>();
            if (boxes.rows > 0) mbar_wait(full + use_slot * 8, phases >> use_slot & 1, &s_abort, 0xa0);
            phases ^= 1u << use_slot;
            __syncwarp();
        };

        // ---- products ----
        // A lane's place in an operand: row (or column) lane / 4, elements 2 * (lane % 4) and the next.  Of a product's sums it has rows
        // lane / 4 and 8 more, columns c0 and c0 + 1.
        const int r0 = lane >> 2, c0 = (lane & 3) * 2;
        uint2 q[kKept ? NT : 1][kKept ? kSteps / 2 : 1][kDigits];
        float row_scale[NT][2];
        // The query's heads as second operands, a lane has dimensions 16 ks + 4 (lane % 4) ... + 3 of a head: whole numbers below 2^22, as three
        // digits from -128 to 127.
        auto take_query = [&] {
#pragma unroll
            for (int t = NT - 1; t >= 0; --t) {
                uint2 x[kSteps];
                const uint32_t row = query + (8 * t + r0) * (DP * 2) + (lane & 1) * 8;
#pragma unroll
                for (int ks = 0; ks < kSteps; ++ks) x[ks] = load_shared_uint2(row + (((2 * ks + (lane >> 1 & 1)) ^ r0) << 4));
                uint32_t pair = 0;  // the largest magnitudes, which have the order of whole numbers; those of infinity and NaN are larger than all others
#pragma unroll
                for (int ks = 0; ks < kSteps; ++ks) pair = __vmaxu2(pair, __vmaxu2(x[ks].x & 0x7fff7fffu, x[ks].y & 0x7fff7fffu));
                pair = __vmaxu2(pair, __shfl_xor_sync(0xffffffffu, pair, 1));
                pair = __vmaxu2(pair, __shfl_xor_sync(0xffffffffu, pair, 2));
                const uint32_t most = __float_as_uint(two_floats<T>(max(pair & 0xffffu, pair >> 16)).x);
                // 2^e, e <= 127, brings it to [2^21, 2^22); 2^-e
                const int e = min(148 - static_cast<int>(most >> 23), 127);
                const bool fine = most < 0x7f800000u;
                const float power = fine ? sign * __uint_as_float(static_cast<uint32_t>(127 + e) << 23) : 0.0f;
                const float back = fmaxf(scale * (e == 127 ? 0x1p-127f : __uint_as_float(static_cast<uint32_t>(127 - e) << 23)), 0x1p-126f);
#pragma unroll
                for (int i = 0; i < 2; ++i) row_scale[t][i] = __shfl_sync(0xffffffffu, fine ? back : __uint_as_float(0x7fffffffu), (c0 + i) * 4);
                if (!kKept) __syncwarp();
#pragma unroll
                for (int ks = 0; ks < kSteps; ks += 2) {
                    uint32_t digits[kDigits][2];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float2 f = two_floats<T>(x[ks + h].x), g = two_floats<T>(x[ks + h].y);
                        // 128 more in each of the lower digits, which are 0 to 255 then
                        const uint32_t v[4] = {static_cast<uint32_t>(__float2int_rn(f.x * power) + 0x8080), static_cast<uint32_t>(__float2int_rn(f.y * power) + 0x8080),
                                               static_cast<uint32_t>(__float2int_rn(g.x * power) + 0x8080), static_cast<uint32_t>(__float2int_rn(g.y * power) + 0x8080)};
                        const uint32_t low = __byte_perm(v[0], v[1], 0x5140), high = __byte_perm(v[2], v[3], 0x5140);
                        digits[0][h] = __byte_perm(low, high, 0x5410) ^ 0x80808080u;
                        digits[1][h] = __byte_perm(low, high, 0x7632) ^ 0x80808080u;
                        digits[2][h] = __byte_perm(__byte_perm(v[0], v[1], 0x0062), __byte_perm(v[2], v[3], 0x0062), 0x5410);
                    }
#pragma unroll
                    for (int d = 0; d < kDigits; ++d) {
                        if (kKept)
                            q[kKept ? t : 0][kKept ? ks / 2 : 0][d] = make_uint2(digits[d][0], digits[d][1]);
                        else  // from the last column tile on, behind the rows that are still to be taken
                            store_shared_uint2(query + (((t * (kSteps / 2) + ks / 2) * kDigits + d) * 32 + lane) * 8, make_uint2(digits[d][0], digits[d][1]));
                    }
                }
                if (!kKept) __syncwarp();
            }
        };
        auto query_part = [&](int t, int ks, int d) {
            return kKept ? q[kKept ? t : 0][kKept ? ks / 2 : 0][d] : load_shared_uint2(query + (((t * (kSteps / 2) + ks / 2) * kDigits + d) * 32 + lane) * 8);
        };
        // ldmatrix addresses of a tile, keys and values alike: 8 keys x 16 bytes a matrix, four of them; of 16 keys, two chunks
        constexpr int kAtOnce = KEYS == 16 ? 2 : 1;  // chunks of an ldmatrix
        const int lane_key = KEYS == 16 ? (lane >> 3 & 1) * 8 + (lane & 7) : lane;
        const uint32_t lane_tile = lane_key * kPitch + (((KEYS == 16 ? lane >> 4 : 0) ^ ((lane_key >> kTurn) & kTurns)) << 4);
        auto chunk_of = [&](uint32_t tile, int ks) { return (tile ^ ((ks % kRowChunks) << 4)) + ks / kRowChunks * (KEYS * kPitch); };
        while (working) {
            float o[kSteps][NT][4];  // dimensions 16 ks + 2 r0 (and the next: + 2) of heads c0, c0 + 1 (+ 1)
#pragma unroll
            for (int n = 0; n < kSteps; ++n) {
#pragma unroll
                for (int t = 0; t < NT; ++t) o[n][t][0] = o[n][t][1] = o[n][t][2] = o[n][t][3] = 0.0f;
            }
            // top: what scores are relative to, within kSlack below the largest; ceiling: a score beyond it moves that; base: top times the row's
            // scale; lift: the power of two of a head's weights; big: the largest of the lane's, so lifted
            float top[NT][2], ceiling[NT][2], base[NT][2], sum[NT][2], lift[NT][2], big[NT][2];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    top[t][i] = ceiling[t][i] = -INFINITY;
                    sum[t][i] = big[t][i] = base[t][i] = 0.0f;
                    lift[t][i] = 1.0f;
                }
            }
            // A long piece adds what it has to fp32 sums in its part of the workspace and begins again from 0 (back: the other way round).
            auto put_by = [&](bool first, bool back) {
                const int rows = min(kRows, p.group - piece.item % tiles * kRows);
                const int64_t part0 = ((static_cast<int64_t>(worker) * S::kWarps + warp) * 2 + (piece.from == 0)) * scratch.rows;
#pragma unroll
                for (int t = 0; t < NT; ++t) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int row = 8 * t + c0 + i;
                        float *sums = scratch.part + (part0 + row) * p.dim + 2 * r0;
                        const float down = 1.0f / lift[t][i], now = top[t][i] * row_scale[t][i];
                        float keep = 1.0f;
                        if (row < rows && !first && top[t][i] != -INFINITY) keep = exp2_fast(scratch.stat[part0 + row].x - now);
                        __syncwarp();
                        if (row < rows && r0 == 0) scratch.stat[part0 + row].x = now;
#pragma unroll
                        for (int n = 0; n < kSteps; ++n) {
                            float2 x = make_float2(0.0f, 0.0f);
                            if (row < rows && n < row_chunks) {
                                if (!first) x = *reinterpret_cast<const float2 *>(sums + n * 16);
                                x = make_float2(fmaf(x.x, keep, o[n][t][i] * down), fmaf(x.y, keep, o[n][t][i + 2] * down));
                                if (!back) *reinterpret_cast<float2 *>(sums + n * 16) = x;
                            }
                            o[n][t][i] = back ? x.x : 0.0f;
                            o[n][t][i + 2] = back ? x.y : 0.0f;
                        }
                        if (back) lift[t][i] = 1.0f;
                    }
                }
            };
            for (int g = piece.from; g < piece.to; ++g) {
                if (FAR && g != piece.from && (g - piece.from) % (kRun / KEYS) == 0) put_by(g - piece.from == kRun / KEYS, false);
                wait_tile();
                bool all_seen = true;
#pragma unroll
                for (int l = 0; l < kLooks; ++l) {
                    seen[l] = value_seen[l];
                    all_seen = all_seen && seen[l] == 0xffffffffu;
                }
                if (g == piece.from) take_query();
                if (kKept) load_keys();  // into the slot of the values before
                const uint32_t keys = ring + use_slot * kTileBytes + lane_tile;
                const uint32_t key_scales = scale_ring + (use_slot * KEYS + r0) * 4;
                use_slot = use_slot + 1 == kSlots ? 0 : use_slot + 1;
                // scores: keys 16 m + r0 (and + 8: + 2) of heads c0, c0 + 1 (+ 1)
                int sums[kDigits][kTiles][NT][4];
#pragma unroll
                for (int d = 0; d < kDigits; ++d) {
#pragma unroll
                    for (int m = 0; m < kTiles; ++m) {
#pragma unroll
                        for (int t = 0; t < NT; ++t) sums[d][m][t][0] = sums[d][m][t][1] = sums[d][m][t][2] = sums[d][m][t][3] = 0;
                    }
                }
#pragma unroll
                for (int ks = 0; ks < kSteps; ks += 2) {
                    if (kSteps > 8 && ks % 4 == 0 && ks >= row_chunks) break;  // (chunks behind the dimensions meet a query of 0)
#pragma unroll
                    for (int n = 0; n < kTiles; n += 2) {
                        uint32_t w[2][4];  // 16 keys: two chunks of them; else a chunk of 32 keys each
                        ldmatrix_x4(w[0], chunk_of(keys, ks) + n * 16 * kPitch);
                        if (kTiles > 1) ldmatrix_x4(w[1], chunk_of(keys, ks + 1) + n * 16 * kPitch);
#pragma unroll
                        for (int i = 0; i < (kTiles > 1 ? 2 : 1); ++i) {
                            const uint32_t a[4] = {w[0][2 * i], w[0][2 * i + 1], kTiles > 1 ? w[1][2 * i] : w[0][2], kTiles > 1 ? w[1][2 * i + 1] : w[0][3]};
#pragma unroll
                            for (int t = 0; t < NT; ++t) {
#pragma unroll
                                for (int d = 0; d < kDigits; ++d) mma_i8(sums[d][n + i][t], a, query_part(t, ks, d));
                            }
                        }
                    }
                }
                if (!kKept) {
                    __syncwarp();  // the query may be overwritten
                    load_keys();
                }
                float s[kTiles][NT][4];
#pragma unroll
                for (int m = 0; m < kTiles; ++m) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float by = load_shared_float(key_scales + (16 * m + 8 * h) * 4);
#pragma unroll
                        for (int t = 0; t < NT; ++t) {
#pragma unroll
                            for (int i = 2 * h; i < 2 * h + 2; ++i)
                                s[m][t][i] = fmaf(static_cast<float>(sums[2][m][t][i]), 65536.0f, static_cast<float>(sums[1][m][t][i] * 256 + sums[0][m][t][i])) * by;
                        }
                    }
                }
                if (__builtin_expect(!all_seen, 0)) {
#pragma unroll
                    for (int m = 0; m < kTiles; ++m) {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            if (seen[m / 2] >> (m % 2 * 16 + 8 * h + r0) & 1) continue;
#pragma unroll
                            for (int t = 0; t < NT; ++t) s[m][t][2 * h] = s[m][t][2 * h + 1] = -INFINITY;
                        }
                    }
                }
                bool moves = false;
                float most[NT][2], keep[NT][2];
#pragma unroll
                for (int t = 0; t < NT; ++t) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        most[t][i] = fmaxf(s[0][t][i], s[0][t][i + 2]);
#pragma unroll
                        for (int m = 1; m < kTiles; ++m) most[t][i] = fmaxf(most[t][i], fmaxf(s[m][t][i], s[m][t][i + 2]));
                        moves |= most[t][i] > ceiling[t][i];
                        keep[t][i] = 1.0f;
                    }
                }
                moves = __any_sync(0xffffffffu, moves);
                if (__builtin_expect(moves, 0)) {
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            float now = most[t][i];
                            now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, 4));
                            now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, 8));
                            now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, 16));
                            if (now > ceiling[t][i]) {
                                base[t][i] = now * row_scale[t][i];
                                keep[t][i] = top[t][i] == -INFINITY ? 0.0f : exp2_fast(fmaf(top[t][i], row_scale[t][i], -base[t][i]));
                                top[t][i] = now;
                                ceiling[t][i] = now + kSlack / row_scale[t][i];
                                sum[t][i] *= keep[t][i];
                                big[t][i] *= keep[t][i];
                            }
                        }
                    }
                }
#pragma unroll
                for (int m = 0; m < kTiles; ++m) {
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            s[m][t][i] = exp2_fast(fmaf(s[m][t][i], row_scale[t][i & 1], -base[t][i & 1]));
                            sum[t][i & 1] += s[m][t][i];
                        }
                    }
                }
                wait_tile();
                load_values();  // into the slot of the keys
                const uint32_t value_scales = scale_ring + (use_slot * KEYS + r0) * 4;
#pragma unroll
                for (int m = 0; m < kTiles; ++m) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float by = load_shared_float(value_scales + (16 * m + 8 * h) * 4);
#pragma unroll
                        for (int t = 0; t < NT; ++t) {
#pragma unroll
                            for (int i = 0; i < 2; ++i) {
                                float &x = s[m][t][2 * h + i];
                                x *= by * lift[t][i];
                                big[t][i] = fmaxf(big[t][i], fabsf(x));
                            }
                        }
                    }
                }
                float largest = big[0][0];
#pragma unroll
                for (int t = 0; t < NT; ++t) largest = fmaxf(largest, fmaxf(big[t][0], big[t][1]));
                if (__builtin_expect(moves || __any_sync(0xffffffffu, largest > 60000.0f), 0)) {
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            float most = big[t][i];
                            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 4));
                            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 8));
                            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 16));
                            float more_lift = 1.0f;
                            if (most > 60000.0f || (most < 256.0f && most > 0.0f)) {
                                // to [2^11, 2^12), as far as lift stays finite
                                const int e = 138 - static_cast<int>(__float_as_uint(most) >> 23);
                                const int has = static_cast<int>(__float_as_uint(lift[t][i]) >> 23) - 127;
                                more_lift = __uint_as_float(static_cast<uint32_t>(127 + max(-126 - has, min(min(e, 127), 127 - has))) << 23);
                            }
                            lift[t][i] *= more_lift;
                            big[t][i] = most * more_lift;
                            keep[t][i] *= more_lift;
#pragma unroll
                            for (int m = 0; m < kTiles; ++m) {
                                s[m][t][i] *= more_lift;
                                s[m][t][i + 2] *= more_lift;
                            }
#pragma unroll
                            for (int n = 0; n < kSteps; ++n) {
                                o[n][t][i] *= keep[t][i];
                                o[n][t][i + 2] *= keep[t][i];
                            }
                        }
                    }
                }
                uint32_t b[NT][kTiles][2];
#pragma unroll
                for (int t = 0; t < NT; ++t) {
#pragma unroll
                    for (int m = 0; m < kTiles; ++m) {
#pragma unroll
                        for (int h = 0; h < 2; ++h) b[t][m][h] = transposed(pack2<__half>(s[m][t][2 * h], s[m][t][2 * h + 1]));
                    }
                }
                const uint32_t values = ring + use_slot * kTileBytes + lane_tile;
                use_slot = use_slot + 1 == kSlots ? 0 : use_slot + 1;
#pragma unroll
                for (int ks = 0; ks < kSteps; ks += kAtOnce) {
                    if (kSteps > 8 && ks % 4 == 0 && ks >= row_chunks) break;
#pragma unroll
                    for (int n = 0; n < kTiles * kAtOnce; n += 2) {
                        uint32_t w[4];
                        ldmatrix_x4_trans(w, chunk_of(values, ks) + n * 16 * kPitch);
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const uint32_t x = w[2 * i] ^ 0x80808080u, y = w[2 * i + 1] ^ 0x80808080u;
                            const uint32_t a[4] = {codes_f16<0x4240>(x), codes_f16<0x4341>(x), codes_f16<0x4240>(y), codes_f16<0x4341>(y)};
#pragma unroll
                            for (int t = 0; t < NT; ++t) mma_16816<__half>(o[ks + (n + i) / kTiles][t], a, b[t][(n + i) % kTiles][0], b[t][(n + i) % kTiles][1]);
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
            for (int t = 0; t < NT; ++t) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float all = sum[t][i];
                    all += __shfl_xor_sync(0xffffffffu, all, 4);
                    all += __shfl_xor_sync(0xffffffffu, all, 8);
                    all += __shfl_xor_sync(0xffffffffu, all, 16);
                    const float most = top[t][i] * row_scale[t][i];
                    const float down = 1.0f / lift[t][i];
                    const int row = 8 * t + c0 + i;
                    if (row >= rows) continue;
                    if (begins && ends) {
                        const float inv = all == 0.0f ? 0.0f : 1.0f / all;
                        T *dst = static_cast<T *>(p.out) + (row0 + row) * p.dim + 2 * r0;
#pragma unroll
                        for (int n = 0; n < kSteps; ++n)
                            if (n < row_chunks) *reinterpret_cast<uint32_t *>(dst + n * 16) = pack2<T>(o[n][t][i] * down * inv, o[n][t][i + 2] * down * inv);
                        if (r0 == 0) p.lse[row0 + row] = all == 0.0f ? -INFINITY : most * kLn2 + logf(all);
                    } else {
                        float *dst = scratch.part + (part0 + row) * p.dim + 2 * r0;
#pragma unroll
                        for (int n = 0; n < kSteps; ++n)
                            if (n < row_chunks) *reinterpret_cast<float2 *>(dst + n * 16) = make_float2(o[n][t][i] * down, o[n][t][i + 2] * down);
                        if (r0 == 0) scratch.stat[part0 + row] = make_float2(most, all);
                    }
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
        if (threadIdx.x == 0 && s_abort != 0) *boxes.status = s_abort;
        add_parts<T, S::kWarps>(p, scratch, list, s_parts, tiles);
        __syncthreads();
    }
}

// A cache as TMA sees it: boxes of `rows` places of one page and head by up to 128 columns (zeros behind the head dimension).  False: its
// strides are none that TMA takes.
bool cache_map(CUtensorMap *map, const Problem &p, const void *base, int64_t sb, int64_t st, int64_t sh, int rows, int columns) {
    const int64_t sizes[4] = {p.dim, p.page, p.kv_heads, p.pages};
    int64_t strides[3] = {st, sh, sb};
    for (int i = 0; i < 3; ++i) {
        if (sizes[i + 1] == 1) strides[i] = p.dim;  // takes no step
        if (strides[i] <= 0 || strides[i] >= 1ll << 39) return false;
    }
    const int box[4] = {columns, rows, 1, 1};
    return make_tmap_4d(map, base, 1, sizes, strides, box, columns);
}

template <typename T, int DP, int NT, bool FAR>
int launch_decode_kernel(const Problem &p, const QuantScales &scales, const Plan &plan, const Scratch &scratch, cudaStream_t stream) {
    using S = Shape<DP, NT>;
    CUtensorMap k_map = {}, v_map = {};
    // as many places a box as begin together in any page and any tile
    Boxes boxes = {8, device_status_word()};
    while (2 * boxes.rows <= S::kKeys && boxes.rows < 32 && p.page % (2 * boxes.rows) == 0) boxes.rows *= 2;
    constexpr int kColumns = DP < 128 ? DP : 128;
    if (p.page % 8 != 0 || p.pages == 0 || !cache_map(&k_map, p, p.k, p.k_sb, p.k_st, p.k_sh, boxes.rows, kColumns) ||
        !cache_map(&v_map, p, p.v, p.v_sb, p.v_st, p.v_sh, boxes.rows, kColumns))
        boxes.rows = 0;
    QMM_CUDA_OK(cudaFuncSetAttribute(quant_decode_kernel<T, DP, NT, FAR>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(S::kSmem)));
    QMM_CUDA_OK(launch_pdl(quant_decode_kernel<T, DP, NT, FAR>, dim3(plan.workers), dim3(S::kWarps * 32), S::kSmem, stream, p, scales, scratch, boxes, k_map, v_map));
    return QMM_OK;
}

template <typename T, int DP, int NT>
int launch(const Problem &p, const QuantScales &scales, const Plan &plan, const Scratch &scratch, cudaStream_t stream) {
    const bool far = is_far(p, plan, Shape<DP, NT>::kWarps);
    const int rc = far ? launch_decode_kernel<T, DP, NT, true>(p, scales, plan, scratch, stream) : launch_decode_kernel<T, DP, NT, false>(p, scales, plan, scratch, stream);
    return rc != QMM_OK ? rc : launch_join<T>(p, plan, scratch, stream);
}

template <typename T, int NT>
int launch_dim(const Problem &p, const QuantScales &scales, const Plan &plan, const Scratch &scratch, cudaStream_t stream) {
    if (p.dim <= 64) return launch<T, 64, NT>(p, scales, plan, scratch, stream);
    if (p.dim <= 128) return launch<T, 128, NT>(p, scales, plan, scratch, stream);
    return launch<T, 256, NT>(p, scales, plan, scratch, stream);
}

template <typename T>
int launch_t(const Problem &p, const QuantScales &scales, const Plan &plan, const Scratch &scratch, cudaStream_t stream) {
    return is_narrow(p.heads, p.kv_heads) ? launch_dim<T, 1>(p, scales, plan, scratch, stream) : launch_dim<T, 2>(p, scales, plan, scratch, stream);
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
