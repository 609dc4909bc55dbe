// Attention of one new token a sequence over a paged key-value cache (npu_paged_attention).
//
// Bound by HBM: every visible key and value is read once, for all query heads that share it.  The heads of a group (16 at a
// time) are the rows of mma.sync m16n8k16, so a key costs the tensor pipe the same for one head as for sixteen, about a fifth of
// the time its bytes take (tcgen05 would need 64 rows at least and a hand-off through tensor memory for every few keys).
//
// A warp has a private ring of tiles of 32 keys or values in shared memory, filled by cp.async with the tiles' pages looked up
// one tile ahead, and never waits for another warp's loads.  Places that are not seen are not read but zero-filled, so what lies
// there has no part in any product.  The softmax is one pass: running maximum and sum a row, sums rescaled only when a maximum
// moved.
//
// The work of a call is the list of all (sequence, head tile, 32 places), cut into equal contiguous ranges, one for each CTA,
// wherever sequences begin and end; so a batch of ragged lengths and one long sequence load the GPU alike.  The warps of a CTA
// take the tiles of a piece (what a CTA has of one sequence's head tile) in turn and add their sums in shared memory, while the
// tiles of the next piece are under way.  A piece that is the whole is written at once; of a cut one the sums go to the
// workspace, and a second kernel joins them in the order of the CTAs.  Where every sequence is short, whole head tiles go to
// the CTAs in turn and nothing is cut.  Nothing depends on timing, and nothing has to be zero before a call.
#include "paged_common.cuh"

namespace qmm {
namespace paged {

namespace {

constexpr int kRows = 16;   // query heads of a tile
constexpr int kShort = 16;  // tiles of a sequence that is not cut while all are this short

// DP: the head dimension rounded up to 64, 128 or 256.  Shared memory of a CTA: the rings, 192 KiB, eight rows of sums of half
// the warps, and a query tile.
template <int DP>
struct Shape {
    static constexpr int kKeys = DP == 256 ? 16 : 32;  // keys of a tile: 256 columns of sums leave no registers for 32 scores
    static constexpr int kWarps = DP == 256 ? 2 : 4;
    static constexpr int kSlots = DP == 256 ? 6 : DP == 128 ? 3 : 6;  // tiles of a warp's ring, keys and values in turn
    static constexpr int kTileBytes = kKeys * DP * 2;
    static constexpr int kHalf = kWarps / 2;
    static constexpr int kPitch = DP + 8;  // floats of a row of sums: rows 8 banks apart
    static constexpr int kRing = kWarps * kSlots * kTileBytes;
    static constexpr int kSums = (kHalf * 8 * kPitch * 4 + 511) / 512 * 512;  // the query tile begins at a multiple of its rows
    static constexpr int kQuery = kRows * DP * 2;
    static constexpr int kStats = kHalf * 8 * 8;
    static constexpr size_t kSmem = kRing + kSums + kQuery + kStats;
};

// Workspace: part[CTA][2][rows][dim] sums, stat[CTA][2][rows] (maximum, sum), cut[index]: first and last CTA of a cut item, its
// sequence and head tile (first < 0: not cut); by item where there are no more items than CTAs, else by the item's first CTA.
struct Scratch {
    float *part;
    float2 *stat;
    int4 *cut;
    int rows, workers, by_item;
};

struct Plan {
    int workers, rows, tiles;
    int64_t items;
    size_t part_bytes, stat_bytes, bytes;
};

Plan make_plan(int64_t batch, int64_t heads, int64_t kv_heads, int64_t dim) {
    Plan plan;
    const int64_t group = kv_heads > 0 ? heads / kv_heads : 0;
    plan.workers = 2 * sm_count();
    plan.rows = static_cast<int>(group < kRows ? group : kRows);
    plan.tiles = static_cast<int>((group + kRows - 1) / kRows);
    plan.items = batch * kv_heads * plan.tiles;
    plan.part_bytes = static_cast<size_t>(plan.workers) * 2 * plan.rows * dim * sizeof(float);
    plan.stat_bytes = (static_cast<size_t>(plan.workers) * 2 * plan.rows * sizeof(float2) + 15) / 16 * 16;
    plan.bytes = plan.part_bytes + plan.stat_bytes + static_cast<size_t>(plan.workers) * sizeof(int4);
    return plan;
}

// What a sequence's token sees, as tiles of KEYS places: those of the sinks, then those of the window.
struct Sequence {
    int sink_end, lo, hi, sink_tiles, first, tiles;
};
template <int KEYS>
__device__ __forceinline__ Sequence sequence_of(const Problem &p, int b) {
    const int len = __ldg(p.lens + b);
    const Range r = visible_range(p, len <= 0 ? -1 : len - 1);
    Sequence s;
    s.sink_end = r.sink_end;
    s.lo = r.lo;
    s.hi = r.hi;
    s.sink_tiles = (r.sink_end + KEYS - 1) / KEYS;
    s.first = max(r.lo / KEYS, s.sink_tiles);
    const int end = r.hi / KEYS + (r.hi % KEYS != 0);
    s.tiles = s.sink_tiles + max(0, end - s.first);
    return s;
}

// A CTA's part of the list.
struct Share {
    int64_t end;    // whole: number of items; else: where the CTA's range ends
    int64_t range;  // length of a range
    int items;      // of a sequence
    bool whole;     // items are not cut, CTA c has c, c + workers, ...
};

// What a CTA has of one item: tiles [from, to) of sequence b's item.
struct Piece {
    int64_t at;  // whole: the item's number; else: where the piece begins in the list
    int b, item, from, to;
    Sequence s;
};

// Steps to the CTA's next piece; false: there is none.
template <int KEYS>
__device__ __forceinline__ bool next_piece(const Problem &p, const Share &share, int workers, Piece &piece) {
    if (share.whole) {
        piece.at += workers;
        if (piece.at >= share.end) return false;
        const int b = static_cast<int>(piece.at / share.items);
        piece.item = static_cast<int>(piece.at - static_cast<int64_t>(b) * share.items);
        piece.b = b;
        piece.s = sequence_of<KEYS>(p, b);
        piece.from = 0;
        piece.to = piece.s.tiles;
        return true;
    }
    piece.at += piece.to - piece.from;
    if (piece.at >= share.end) return false;
    if (++piece.item == share.items) {
        piece.item = 0;
        do {
            piece.s = sequence_of<KEYS>(p, ++piece.b);
        } while (piece.s.tiles == 0);
    }
    piece.from = 0;
    piece.to = static_cast<int>(min(static_cast<int64_t>(piece.s.tiles), share.end - piece.at));
    return true;
}

__device__ __forceinline__ void cp_async_16(uint32_t dst, const void *src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
template <typename T>
__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma_16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma_16816<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

template <typename T, int DP>
__global__ void __launch_bounds__(Shape<DP>::kWarps * 32, 2)
decode_kernel(const __grid_constant__ Problem p, const __grid_constant__ Scratch scratch) {
    using S = Shape<DP>;
    constexpr int KEYS = S::kKeys, kThreads = S::kWarps * 32;
    constexpr int kChunks = DP / 8;  // 16-byte chunks of a row in shared memory
    extern __shared__ __align__(512) uint8_t smem[];  // rows of up to 512 bytes, stepped through by exclusive or
    float *sums = reinterpret_cast<float *>(smem + S::kRing);
    uint8_t *query = smem + S::kRing + S::kSums;
    float2 *stats = reinterpret_cast<float2 *>(query + S::kQuery);
    const int warp = warp_id_uniform(), lane = threadIdx.x & 31;
    const int worker = blockIdx.x;
    const uint32_t ring = smem_u32(smem) + warp * (S::kSlots * S::kTileBytes);
    pdl_launch_dependents();
    pdl_wait();

    const int tiles = (p.group + kRows - 1) / kRows;
    const int ksteps = (p.dim + 15) / 16;
    const int row_chunks = p.dim / 8;
    Share share;
    share.items = p.kv_heads * tiles;

    // the list's length, and whether all sequences are short
    int64_t total = 0;
    int longest = 0;
    for (int b = lane; b < p.batch; b += 32) {
        const int n = sequence_of<KEYS>(p, b).tiles;
        total += n;
        longest = max(longest, n);
    }
    for (int o = 16; o > 0; o >>= 1) {
        total += __shfl_xor_sync(0xffffffffu, total, o);
        longest = max(longest, __shfl_xor_sync(0xffffffffu, longest, o));
    }
    total *= share.items;
    share.whole = longest <= kShort;
    Piece load;
    load.b = load.item = load.from = load.to = 0;
    if (!scratch.by_item && threadIdx.x == 0) scratch.cut[worker] = make_int4(-1, 0, 0, 0);
    if (share.whole) {
        share.end = static_cast<int64_t>(p.batch) * share.items;
        share.range = 1;
        load.at = worker - scratch.workers;
        if (!next_piece<KEYS>(p, share, scratch.workers, load)) return;
    } else {
        share.range = max(static_cast<int64_t>(S::kWarps), (total + scratch.workers - 1) / scratch.workers);
        const int64_t begin = worker * share.range;
        share.end = min(total, begin + share.range);
        int64_t before = 0;
        bool found = false;
        // sequences that see nothing, and where this CTA's range begins
        for (int b0 = 0; b0 < p.batch; b0 += 32) {
            const int b = b0 + lane;
            const int n = b < p.batch ? sequence_of<KEYS>(p, b).tiles : 1;
            if (warp == 0) {
                for (uint32_t none = __ballot_sync(0xffffffffu, n == 0); none != 0; none &= none - 1) {
                    const int e = b0 + __ffs(none) - 1;
                    if (e % scratch.workers != worker) continue;
                    for (int h = 0; h < p.heads; ++h) empty_row<T>(p, e, h);
                    if (scratch.by_item)
                        for (int i = lane; i < share.items; i += 32)
                            scratch.cut[static_cast<int64_t>(e) * share.items + i] = make_int4(-1, 0, 0, 0);
                }
            }
            if (found || begin >= share.end) continue;
            const int64_t mine = b < p.batch ? static_cast<int64_t>(n) * share.items : 0;
            int64_t sum = mine;
            for (int o = 1; o < 32; o <<= 1) {
                const int64_t left = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += left;
            }
            const uint32_t past = __ballot_sync(0xffffffffu, before + sum > begin);
            if (past == 0) {
                before += __shfl_sync(0xffffffffu, sum, 31);
                continue;
            }
            found = true;
            load.b = b0 + __ffs(past) - 1;
            before += __shfl_sync(0xffffffffu, sum - mine, __ffs(past) - 1);
        }
        if (!found) return;
        load.s = sequence_of<KEYS>(p, load.b);
        const int64_t in = begin - before;
        load.at = begin;
        load.item = static_cast<int>(in / load.s.tiles);
        load.from = static_cast<int>(in - static_cast<int64_t>(load.item) * load.s.tiles);
        load.to = static_cast<int>(min(static_cast<int64_t>(load.s.tiles), load.from + share.end - begin));
    }
    Piece piece = load;

    // ---- loads: one place of the tile a lane (16 keys: lanes 16..31 the same again), keys and values of a tile apart ----
    int at = load.from + warp;  // this warp's next tile of the piece that is being loaded
    bool more = true;
    auto settle = [&] {  // on to a piece that has a tile for this warp
        while (more && at >= load.to) {
            more = next_piece<KEYS>(p, share, scratch.workers, load);
            at = load.from + warp;
        }
    };
    settle();
    int at_place = 0, entry = -1;
    auto look_up = [&] {
        entry = -1;
        if (!more) return;
        const int first = at < load.s.sink_tiles ? at * KEYS : (load.s.first + at - load.s.sink_tiles) * KEYS;
        const int j = first + (lane & (KEYS - 1));
        if (j < load.s.hi && (j < load.s.sink_end || j >= load.s.lo)) {
            const int page = page_of(p, j);
            at_place = j - page * p.page;
            entry = __ldg(p.table + load.b * p.table_st + page);
        }
    };
    look_up();
    // every load of keys is followed by that of their values, so the lookup and the mask are kept for it
    constexpr int kMasks = S::kSlots / 2 + 1;
    uint32_t masks[kMasks];  // of the tiles under way, oldest first
#pragma unroll
    for (int i = 0; i < kMasks; ++i) masks[i] = 0;
    int under_way = 0, slot = 0, value_place = 0, value_entry = 0, value_head = 0;
    uint32_t value_seen = 0;
    // A lane always has the same chunk, of rows kStep apart.  Rows of 16 places lie evenly apart where a page holds a multiple of
    // 16 (tiles begin at multiples of 16), so a tile that is seen whole takes one address for 16 places; else each row its own.
    constexpr int kStep = 32 / kChunks;
    const int my_key = lane / kChunks, my_chunk = lane % kChunks;
    const bool my_part = my_chunk < 2 * ksteps;
    const int my_offset = my_chunk < row_chunks ? my_chunk * 8 : 0;
    const bool even = p.page % 16 == 0 && row_chunks == 2 * ksteps;
    // the swizzled place of key kStep * i + my_key: chunk ^ key % 8, where the key's parts have no bits in common
    const uint32_t my_dst = my_key * (DP * 2) + ((my_chunk ^ my_key) << 4);
    auto copy_tile = [&](const void *cache, int64_t sb, int64_t st, int64_t sh, int id, int place, int kvh, uint32_t seen) {
        const uint32_t dst = ring + slot * S::kTileBytes + my_dst;
        const bool ok = seen >> lane & 1;
        const int64_t offset = ok ? id * sb + place * st + kvh * sh : 0;
        const T *base = static_cast<const T *>(cache) + my_offset;
        if (even && seen == 0xffffffffu) {
            const T *row[KEYS / 16];
#pragma unroll
            for (int h = 0; h < KEYS / 16; ++h) row[h] = base + __shfl_sync(0xffffffffu, offset, 16 * h) + my_key * st;
            if (my_part) {
#pragma unroll
                for (int i = 0; i < KEYS / kStep; ++i) {
                    const int first = kStep * i;
                    cp_async_16((dst ^ ((first & 7) << 4)) + first * (DP * 2), row[first / 16], 16);
                    row[first / 16] += kStep * st;
                }
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < KEYS / kStep; ++i) {
            const int first = kStep * i, key = first + my_key;
            const T *row = base + __shfl_sync(0xffffffffu, offset, key);
            if (my_part)
                cp_async_16((dst ^ ((first & 7) << 4)) + first * (DP * 2), row, my_chunk < row_chunks && (seen >> key & 1) ? 16 : 0);
        }
    };
    auto load_keys = [&] {
        if (more) {
            value_seen = __ballot_sync(0xffffffffu, entry >= 0 && entry < p.pages);
            value_place = at_place;
            value_entry = entry;
            value_head = load.item / tiles;
#pragma unroll
            for (int i = 0; i < kMasks; ++i)
                if (i == under_way) masks[i] = value_seen;
            ++under_way;
            copy_tile(p.k, p.k_sb, p.k_st, p.k_sh, value_entry, value_place, value_head, value_seen);
            at += S::kWarps;
            settle();
            look_up();
        } else {
            value_head = -1;
        }
        cp_async_commit();
        slot = slot + 1 == S::kSlots ? 0 : slot + 1;
    };
    auto load_values = [&] {
        if (value_head >= 0) copy_tile(p.v, p.v_sb, p.v_st, p.v_sh, value_entry, value_place, value_head, value_seen);
        cp_async_commit();
        slot = slot + 1 == S::kSlots ? 0 : slot + 1;
    };
    static_assert(S::kSlots >= 3, "keys, values and the next keys");
#pragma unroll
    for (int i = 0; i < S::kSlots - 1; ++i) {
        if (i % 2 == 0)
            load_keys();
        else
            load_values();
    }
    // steps of one load each, in the order of the ring: the load that a step of the products makes room for
    constexpr bool kKeysNext = (S::kSlots - 1) % 2 == 0;

    // The running maximum is one of unscaled scores, which takes a positive scale: a negative one's sign goes to the query, and
    // for a scale of 0 the query is 0.
    const float factor = p.scale * kLog2e;
    const float scale = factor == 0.0f ? 1.0f : fabsf(factor);
    const uint32_t query_and = factor == 0.0f ? 0u : 0xffffffffu, query_xor = factor < 0.0f ? 0x80008000u : 0u;

    // ---- the query tile of the piece to come: loaded a piece ahead, stored when the warps meet ----
    constexpr int kQueryChunks = kRows * kChunks / kThreads > 0 ? kRows * kChunks / kThreads : 1;
    uint4 ahead[kQueryChunks];
    auto load_query = [&](const Piece &of) {
        const int kvh = of.item / tiles, tile = of.item - kvh * tiles;
        const int rows = min(kRows, p.group - tile * kRows);
        const T *base = static_cast<const T *>(p.q) + of.b * p.q_st + (kvh * p.group + tile * kRows) * p.q_sh;
#pragma unroll
        for (int i = 0; i < kQueryChunks; ++i) {
            const int idx = i * kThreads + threadIdx.x, row = idx / kChunks, chunk = idx % kChunks;
            ahead[i] = row < rows && chunk < row_chunks ? __ldg(reinterpret_cast<const uint4 *>(base + row * p.q_sh + chunk * 8))
                                                        : make_uint4(0, 0, 0, 0);
        }
    };
    auto store_query = [&] {
#pragma unroll
        for (int i = 0; i < kQueryChunks; ++i) {
            const int idx = i * kThreads + threadIdx.x, row = idx / kChunks, chunk = idx % kChunks;
            if (row < kRows)
                *reinterpret_cast<uint4 *>(query + row * (DP * 2) + ((chunk ^ (row & 7)) << 4)) =
                    make_uint4((ahead[i].x & query_and) ^ query_xor, (ahead[i].y & query_and) ^ query_xor,
                               (ahead[i].z & query_and) ^ query_xor, (ahead[i].w & query_and) ^ query_xor);
        }
    };
    load_query(piece);
    store_query();
    __syncthreads();

    // ---- products ----
    const int r0 = lane >> 2, c0 = (lane & 3) * 2;
    int use_slot = 0;
    while (true) {
        Piece next = piece;
        const bool another = next_piece<KEYS>(p, share, scratch.workers, next);
        if (another) load_query(next);
        // ldmatrix addresses: chunk 2 i + c of a row swizzled by r is (2 i) ^ (c ^ r), so a step is one exclusive or
        auto query_part = [&](uint32_t (&r)[4], int ks) {
            ldmatrix_x4(r, (smem_u32(query) + (lane & 15) * (DP * 2) + (((lane >> 4) ^ (lane & 7)) << 4)) ^ (ks << 5));
        };
        constexpr bool kKept = DP < 256;  // in registers; 256 columns of sums leave none
        uint32_t q[kKept ? DP / 16 : 1][4];
        if (kKept) {
#pragma unroll
            for (int ks = 0; ks < DP / 16; ++ks) query_part(q[kKept ? ks : 0], ks);
        }
        float o[DP / 8][4];
#pragma unroll
        for (int n = 0; n < DP / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f;
        float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.0f, 0.0f};

        for (int g = piece.from + warp; g < piece.to; g += S::kWarps) {
            // scores of 16 rows x KEYS keys: accumulators of 8 keys
            float s[KEYS / 8][4];
#pragma unroll
            for (int n = 0; n < KEYS / 8; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
            cp_async_wait<S::kSlots - 2>();
            __syncwarp();
            const uint32_t seen = masks[0];
#pragma unroll
            for (int i = 0; i + 1 < kMasks; ++i) masks[i] = masks[i + 1];
            --under_way;
            // into the slot that the step before this one used
            if (kKeysNext) load_keys(); else load_values();
            const uint32_t keys = ring + use_slot * S::kTileBytes + (((lane >> 4) << 3) + (lane & 7)) * (DP * 2) +
                                  ((((lane >> 3) & 1) ^ (lane & 7)) << 4);
            use_slot = use_slot + 1 == S::kSlots ? 0 : use_slot + 1;
#pragma unroll
            for (int ks = 0; ks < DP / 16; ++ks) {
                if (ks >= ksteps) break;
                uint32_t(&qk)[4] = q[kKept ? ks : 0];
                if (!kKept) query_part(qk, ks);
#pragma unroll
                for (int n = 0; n < KEYS / 16; ++n) {
                    uint32_t b[4];
                    ldmatrix_x4(b, (keys ^ (ks << 5)) + n * 16 * (DP * 2));
                    mma_16816<T>(s[2 * n], qk, b[0], b[1]);
                    mma_16816<T>(s[2 * n + 1], qk, b[2], b[3]);
                }
            }
            if (seen != 0xffffffffu) {
#pragma unroll
                for (int n = 0; n < KEYS / 8; ++n) {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (!(seen >> (n * 8 + c0 + (i & 1)) & 1)) s[n][i] = -INFINITY;
                }
            }
            float most[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int n = 0; n < KEYS / 8; ++n) {
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
                base[r] = now == -INFINITY ? 0.0f : now * scale;
                keep[r] = exp2_fast(fmaf(top[r], scale, -base[r]));
                moved |= now != top[r];
                top[r] = now;
            }
            if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
                for (int n = 0; n < DP / 8; ++n) {
                    o[n][0] *= keep[0];
                    o[n][1] *= keep[0];
                    o[n][2] *= keep[1];
                    o[n][3] *= keep[1];
                }
                sum[0] *= keep[0];
                sum[1] *= keep[1];
            }
            // the weights, rounded to the type of the values (the sum takes them unrounded: 2^-9 or 2^-12 of each weight,
            // independent of one another), as they lie are the second product's first operand
            uint32_t a[KEYS / 16][4];
#pragma unroll
            for (int n = 0; n < KEYS / 8; ++n) {
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const float e0 = exp2_fast(fmaf(s[n][2 * r], scale, -base[r])), e1 = exp2_fast(fmaf(s[n][2 * r + 1], scale, -base[r]));
                    sum[r] += e0 + e1;
                    a[n >> 1][(n & 1) * 2 + r] = pack2<T>(e0, e1);
                }
            }
            cp_async_wait<S::kSlots - 2>();
            __syncwarp();
            if (kKeysNext) load_values(); else load_keys();
            const uint32_t values = ring + use_slot * S::kTileBytes + ((((lane >> 3) & 1) << 3) + (lane & 7)) * (DP * 2) +
                                    (((lane >> 4) ^ (lane & 7)) << 4);
            use_slot = use_slot + 1 == S::kSlots ? 0 : use_slot + 1;
#pragma unroll
            for (int n = 0; n < DP / 16; ++n) {
                if (n >= ksteps) break;
#pragma unroll
                for (int k = 0; k < KEYS / 16; ++k) {
                    uint32_t b[4];
                    ldmatrix_x4_trans(b, (values ^ (n << 5)) + k * 16 * (DP * 2));
                    mma_16816<T>(o[2 * n], a[k], b[0], b[1]);
                    mma_16816<T>(o[2 * n + 1], a[k], b[2], b[3]);
                }
            }
        }

        // ---- the warps' sums, eight rows at a time: the upper half's to the lower half's, then what is left by all threads ----
        const int kvh = piece.item / tiles, tile = piece.item - kvh * tiles;
        const int head0 = kvh * p.group + tile * kRows;
        const int rows = min(kRows, p.group - tile * kRows);
        const bool begins = piece.from == 0, ends = piece.to == piece.s.tiles;
        const int64_t slot_row = (worker * 2 + (begins ? 1 : 0)) * static_cast<int64_t>(scratch.rows);
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            if (r * 8 >= rows) break;
            sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 1);
            sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 2);
            top[r] *= scale;
            const int buffer = warp < S::kHalf ? warp : warp - S::kHalf;
            float *mine = sums + (buffer * 8 + r0) * S::kPitch + c0;
            float2 *my_stat = stats + buffer * 8 + r0;
            auto put = [&] {
#pragma unroll
                for (int n = 0; n < DP / 8; ++n) *reinterpret_cast<float2 *>(mine + n * 8) = make_float2(o[n][2 * r], o[n][2 * r + 1]);
                if ((lane & 3) == 0) *my_stat = make_float2(top[r], sum[r]);
            };
            if (warp >= S::kHalf) put();
            __syncthreads();
            if (r == 0 && another) store_query();
            if (warp < S::kHalf) {
                const float2 other = *my_stat;
                const float now = fmaxf(top[r], other.x), base = now == -INFINITY ? 0.0f : now;
                const float keep = exp2_fast(top[r] - base), add = exp2_fast(other.x - base);
#pragma unroll
                for (int n = 0; n < DP / 8; ++n) {
                    const float2 v = *reinterpret_cast<const float2 *>(mine + n * 8);
                    o[n][2 * r] = fmaf(v.x, add, o[n][2 * r] * keep);
                    o[n][2 * r + 1] = fmaf(v.y, add, o[n][2 * r + 1] * keep);
                }
                sum[r] = fmaf(other.y, add, sum[r] * keep);
                top[r] = now;
                __syncwarp();  // a row's four lanes have read its statistics
                put();
            }
            __syncthreads();
            for (int idx = threadIdx.x; idx < min(8, rows - r * 8) * (DP / 4); idx += kThreads) {
                const int at_row = idx / (DP / 4), row = r * 8 + at_row, d = idx % (DP / 4) * 4;
                if (d >= p.dim) continue;
                float2 stat[S::kHalf];
                float now = -INFINITY;
#pragma unroll
                for (int w = 0; w < S::kHalf; ++w) {
                    stat[w] = stats[w * 8 + at_row];
                    now = fmaxf(now, stat[w].x);
                }
                const float base = now == -INFINITY ? 0.0f : now;
                float all = 0.0f;
                float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int w = 0; w < S::kHalf; ++w) {
                    const float weight = exp2_fast(stat[w].x - base);
                    const float4 x = *reinterpret_cast<const float4 *>(sums + (w * 8 + at_row) * S::kPitch + d);
                    all = fmaf(stat[w].y, weight, all);
                    v.x = fmaf(x.x, weight, v.x);
                    v.y = fmaf(x.y, weight, v.y);
                    v.z = fmaf(x.z, weight, v.z);
                    v.w = fmaf(x.w, weight, v.w);
                }
                if (begins && ends) {
                    const int64_t to = static_cast<int64_t>(piece.b) * p.heads + head0 + row;
                    const float inv = all == 0.0f ? 0.0f : 1.0f / all;
                    *reinterpret_cast<uint2 *>(static_cast<T *>(p.out) + to * p.dim + d) =
                        make_uint2(pack2<T>(v.x * inv, v.y * inv), pack2<T>(v.z * inv, v.w * inv));
                    if (d == 0) p.lse[to] = all == 0.0f ? -INFINITY : now * kLn2 + logf(all);
                } else {
                    *reinterpret_cast<float4 *>(scratch.part + (slot_row + row) * p.dim + d) = v;
                    if (d == 0) scratch.stat[slot_row + row] = make_float2(now, all);
                }
            }
            __syncthreads();  // before the buffers are written again
        }
        if (threadIdx.x == 0 && begins && (scratch.by_item || !ends)) {
            const int last = ends ? 0 : static_cast<int>((piece.at + piece.s.tiles - 1) / share.range);
            scratch.cut[scratch.by_item ? static_cast<int64_t>(piece.b) * share.items + piece.item : worker] =
                make_int4(ends ? -1 : worker, last, piece.b, piece.item);
        }
        if (!another) break;
        piece = next;
    }
    cp_async_wait<0>();
}

// Joins the parts of the cut items, in the order of the CTAs.  share_parts (few items): a CTA has one row of an item and its
// warps share the parts; else its warps share the rows.
constexpr int kJoinWarps = 8;
template <typename T>
__global__ void __launch_bounds__(kJoinWarps * 32)
join_kernel(const __grid_constant__ Problem p, const __grid_constant__ Scratch scratch, bool share_parts) {
    __shared__ float s_sum[kJoinWarps][256];
    __shared__ float2 s_stat[kJoinWarps];
    pdl_launch_dependents();
    pdl_wait();
    const int4 cut = scratch.cut[blockIdx.x];
    if (cut.x < 0) return;
    const int warp = warp_id_uniform(), lane = threadIdx.x & 31;
    const int tiles = (p.group + kRows - 1) / kRows;
    const int kvh = cut.w / tiles, tile = cut.w - kvh * tiles;
    const int rows = min(kRows, p.group - tile * kRows);
    const int parts = cut.y - cut.x + 1;
    for (int row = share_parts ? static_cast<int>(blockIdx.y) : warp; row < rows; row += share_parts ? static_cast<int>(gridDim.y) : kJoinWarps) {
        const int from = share_parts ? static_cast<int>(static_cast<int64_t>(parts) * warp / kJoinWarps) : 0;
        const int to = share_parts ? static_cast<int>(static_cast<int64_t>(parts) * (warp + 1) / kJoinWarps) : parts;
        auto place = [&](int i) { return (static_cast<int64_t>(cut.x + i) * 2 + (i == 0)) * scratch.rows + row; };
        float top = -INFINITY;
        for (int i = from + lane; i < to; i += 32) top = fmaxf(top, scratch.stat[place(i)].x);
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float base = top == -INFINITY ? 0.0f : top;
        float sum = 0.0f, acc[8] = {};
        for (int i0 = from; i0 < to; i0 += 32) {
            float weight = 0.0f;
            if (i0 + lane < to) {
                const float2 st = scratch.stat[place(i0 + lane)];
                weight = exp2_fast(st.x - base);
                sum += st.y * weight;
            }
            const int n = min(32, to - i0);
#pragma unroll 4
            for (int i = 0; i < n; ++i) {
                const float w = __shfl_sync(0xffffffffu, weight, i);
                const float *src = scratch.part + place(i0 + i) * p.dim;
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const int d = c * 128 + lane * 4;
                    if (d < p.dim) {
                        const float4 v = *reinterpret_cast<const float4 *>(src + d);
                        acc[4 * c] = fmaf(v.x, w, acc[4 * c]);
                        acc[4 * c + 1] = fmaf(v.y, w, acc[4 * c + 1]);
                        acc[4 * c + 2] = fmaf(v.z, w, acc[4 * c + 2]);
                        acc[4 * c + 3] = fmaf(v.w, w, acc[4 * c + 3]);
                    }
                }
            }
        }
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (share_parts) {
#pragma unroll
            for (int c = 0; c < 2; ++c)
                *reinterpret_cast<float4 *>(&s_sum[warp][c * 128 + lane * 4]) = make_float4(acc[4 * c], acc[4 * c + 1], acc[4 * c + 2], acc[4 * c + 3]);
            if (lane == 0) s_stat[warp] = make_float2(top, sum);
            __syncthreads();
            if (warp == 0) {
                for (int w = 0; w < kJoinWarps; ++w) top = fmaxf(top, s_stat[w].x);
                const float all = top == -INFINITY ? 0.0f : top;
                sum = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i) acc[i] = 0.0f;
                for (int w = 0; w < kJoinWarps; ++w) {
                    const float weight = exp2_fast(s_stat[w].x - all);
                    sum = fmaf(s_stat[w].y, weight, sum);
#pragma unroll
                    for (int i = 0; i < 8; ++i) acc[i] = fmaf(s_sum[w][(i >> 2) * 128 + lane * 4 + (i & 3)], weight, acc[i]);
                }
            }
        }
        if (!share_parts || warp == 0) {
            const int64_t at = static_cast<int64_t>(cut.z) * p.heads + kvh * p.group + tile * kRows + row;
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
            T *dst = static_cast<T *>(p.out) + at * p.dim;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int d = c * 128 + lane * 4;
                if (d < p.dim)
                    *reinterpret_cast<uint2 *>(dst + d) = make_uint2(pack2<T>(acc[4 * c] * inv, acc[4 * c + 1] * inv),
                                                                     pack2<T>(acc[4 * c + 2] * inv, acc[4 * c + 3] * inv));
            }
            if (lane == 0) p.lse[at] = sum == 0.0f ? -INFINITY : top * kLn2 + logf(sum);
        }
        if (share_parts) __syncthreads();
    }
}

template <typename T, int DP>
int launch(const Problem &p, const Plan &plan, Scratch scratch, cudaStream_t stream) {
    QMM_CUDA_OK(cudaFuncSetAttribute(decode_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(Shape<DP>::kSmem)));
    QMM_CUDA_OK(launch_pdl(decode_kernel<T, DP>, dim3(plan.workers), dim3(Shape<DP>::kWarps * 32), Shape<DP>::kSmem, stream, p, scratch));
    const int64_t indices = scratch.by_item ? plan.items : plan.workers;
    const bool share_parts = indices * plan.rows <= 4 * plan.workers;
    QMM_CUDA_OK(launch_pdl(join_kernel<T>, dim3(static_cast<unsigned>(indices), share_parts ? plan.rows : 1), dim3(kJoinWarps * 32), 0,
                           stream, p, scratch, share_parts));
    return QMM_OK;
}

template <typename T>
int launch_t(const Problem &p, const Plan &plan, const Scratch &scratch, cudaStream_t stream) {
    if (p.dim <= 64) return launch<T, 64>(p, plan, scratch, stream);
    if (p.dim <= 128) return launch<T, 128>(p, plan, scratch, stream);
    return launch<T, 256>(p, plan, scratch, stream);
}

}  // namespace

size_t decode_workspace(int64_t batch, int64_t heads, int64_t kv_heads, int64_t dim) {
    return batch == 0 || heads == 0 ? 0 : make_plan(batch, heads, kv_heads, dim).bytes;
}

int launch_decode(const Problem &p, int dtype, void *workspace, size_t workspace_bytes, cudaStream_t stream) {
    const Plan plan = make_plan(p.batch, p.heads, p.kv_heads, p.dim);
    if (workspace_bytes < plan.bytes || workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 15) != 0)
        return fail(QMM_ERR_WORKSPACE, "qmm_paged_attention: needs a workspace of " + std::to_string(plan.bytes) + " bytes, 16-byte aligned");
    Scratch scratch;
    uint8_t *base = static_cast<uint8_t *>(workspace);
    scratch.part = reinterpret_cast<float *>(base);
    scratch.stat = reinterpret_cast<float2 *>(base + plan.part_bytes);
    scratch.cut = reinterpret_cast<int4 *>(base + plan.part_bytes + plan.stat_bytes);
    scratch.rows = plan.rows;
    scratch.workers = plan.workers;
    scratch.by_item = plan.items <= plan.workers;
    return dtype == QMM_DTYPE_BF16 ? launch_t<__nv_bfloat16>(p, plan, scratch, stream) : launch_t<__half>(p, plan, scratch, stream);
}

}  // namespace paged
}  // namespace qmm
