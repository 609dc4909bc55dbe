// Attention of one new token a sequence over a paged key-value cache (npu_paged_attention).
//
// Bound by HBM: every visible key and value is read once, for all query heads that share it.  The heads of a group (16 at a
// time) are the rows of mma.sync m16n8k16, so a key costs the tensor pipe the same for one head as for sixteen, about a fifth of
// the time its bytes take (tcgen05 would need 64 rows at least and a hand-off through tensor memory for every few keys).
//
// A warp has a private ring of 8 KiB tiles of keys or values in shared memory, filled by cp.async with a tile's pages looked up
// one tile ahead, and never waits for another warp's loads.  Places that are not seen are not read but zero-filled, so what lies
// there has no part in any product.  The softmax is one pass: running maximum and sum a row, sums rescaled only when a maximum
// moved.
//
// The work of a call is the list of all (sequence, head tile, tile of places), cut into equal contiguous ranges, one for each
// warp, wherever sequences begin and end; so a batch of ragged lengths and one long sequence load the GPU alike, and no warp
// waits for another until its range is done.  Head tiles that a warp has whole are written from registers.  Of cut ones it
// leaves its sums in the workspace; the CTA adds those of its warps when all are done, and a second kernel those of the CTAs, in
// their order.  (The warps of a CTA taking the tiles of one sequence in turn, with a join at its end, cost about 3 us a sequence:
// 64 sequences of 500 to 8000 places, 64/8 heads of 128, 131 us.)  Where every sequence is short and head tiles are few, CTAs
// have whole ones in turn, cut for their warps alone.  Nothing depends on timing, and nothing has to be zero before a call.
#include <algorithm>
#include <type_traits>

#include "paged_common.cuh"

namespace qmm {
namespace paged {

namespace {

constexpr int kRows = 16;     // query heads of a tile
constexpr int kShort = 512;   // places that a CTA's warps share rather than several CTAs
// The tensor cores cut sums as they add, towards 0: n values of one sign lose some n * 2^-28 (f16, 2^18 places a warp: two half steps).
// So the kernel for calls that may give a warp more than kNear places puts a warp's sums by after every kRun of them.  (For all
// calls, that code cost 32 sequences through a window of 4096 places 1 of 31 us.)
constexpr int kRun = 65536;
constexpr int64_t kNear = 2 * kRun;
constexpr int kSlots = 3;     // of a warp's ring: keys, values, the next keys
constexpr int kTileBytes = 8192;

// DP: the head dimension rounded up to 64, 128 or 256.  Two CTAs an SM: 112, 112 and 96 KiB of shared memory each.
template <int DP>
struct Shape {
    static constexpr int kKeys = kTileBytes / (2 * DP);  // of a tile
    static constexpr int kWarps = DP == 256 ? 3 : 4;
    static constexpr int kQuery = kRows * DP * 2;
    static constexpr size_t kSmem = kWarps * (kSlots * kTileBytes + kQuery);
};

// Workspace.  part[2 * warp + begins][rows][dim], stat[..][rows] (maximum, sum): what a warp has of a head tile that it has not
// whole; `begins`: from its first place on.  Behind those of all warps, the same for the CTAs.  cut[index]: first and last CTA
// of a head tile that no CTA has whole, its sequence and number (first < 0: none); by head tile where there are no more of them
// than CTAs, else by the first CTA.
struct Scratch {
    float *part;
    float2 *stat;
    int4 *cut;
    int rows, workers, by_item;
    int64_t cta_parts;  // index of the first CTA's parts
};

struct Plan {
    int workers, rows, tiles;
    int64_t items, cta_parts;
    size_t part_bytes, stat_bytes, bytes;
};

Plan make_plan(int64_t batch, int64_t heads, int64_t kv_heads, int64_t dim) {
    Plan plan;
    const int64_t group = kv_heads > 0 ? heads / kv_heads : 0;
    plan.workers = 2 * sm_count();
    plan.rows = static_cast<int>(group < kRows ? group : kRows);
    plan.tiles = static_cast<int>((group + kRows - 1) / kRows);
    plan.items = batch * kv_heads * plan.tiles;
    plan.cta_parts = 2ll * plan.workers * (dim > 128 ? Shape<256>::kWarps : Shape<128>::kWarps);
    const size_t rows = static_cast<size_t>(plan.cta_parts + 2 * plan.workers) * plan.rows;
    plan.part_bytes = rows * dim * sizeof(float);
    plan.stat_bytes = (rows * sizeof(float2) + 15) / 16 * 16;
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

// What a warp has of one head tile: tiles [from, to) of sequence b's item.
struct Piece {
    int64_t at;  // where the piece begins in the list
    int b, item, from, to;
    Sequence s;
};

// Steps to the next piece of a range that ends at `end`; false: there is none.
template <int KEYS>
__device__ __forceinline__ bool next_piece(const Problem &p, int64_t end, int items, Piece &piece) {
    piece.at += piece.to - piece.from;
    if (piece.at >= end) return false;
    if (++piece.item == items) {
        piece.item = 0;
        do {
            piece.s = sequence_of<KEYS>(p, ++piece.b);
        } while (piece.s.tiles == 0);
    }
    piece.from = 0;
    piece.to = static_cast<int>(min(static_cast<int64_t>(piece.s.tiles), end - piece.at));
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

// Powers of two by which weights are larger than exp(score - maximum) until the log-sum: f16 has no full step below 2^-14 and
// nothing below 2^-25, so a weight of 1 for the largest score would lose the many keys of a long cache that lie 2^-25 and more
// below one that stands out; with 2^15 what is lost lies 2^-40 below it.  bf16 has the exponents of fp32.
template <typename T>
constexpr float kLift = std::is_same<T, __half>::value ? 15.0f : 0.0f;

// What a warp left of a head tile, for the CTA to add up.
struct Part {
    int valid, b, item, begins, ends, last;  // last: the CTA that has the head tile's last place
};

// FAR: a warp may have more than kNear places.
template <typename T, int DP, bool FAR>
__global__ void __launch_bounds__(Shape<DP>::kWarps * 32, 2)
decode_kernel(const __grid_constant__ Problem p, const __grid_constant__ Scratch scratch) {
    using S = Shape<DP>;
    constexpr int KEYS = S::kKeys, kThreads = S::kWarps * 32;
    constexpr int kChunks = DP / 8;                    // 16-byte chunks of a row in shared memory
    constexpr int kLooks = KEYS > 32 ? KEYS / 32 : 1;  // places of a tile that a lane looks up (16 keys: every place twice)
    constexpr bool kKept = DP < 256;  // the query in registers; 256 columns of sums leave none
    extern __shared__ __align__(512) uint8_t smem[];  // rows of up to 512 bytes, stepped through by exclusive or
    __shared__ Part s_parts[2 * S::kWarps];
    const int warp = warp_id_uniform(), lane = threadIdx.x & 31;
    const int worker = blockIdx.x;
    const uint32_t ring = smem_u32(smem) + warp * (kSlots * kTileBytes);
    const uint32_t query = smem_u32(smem) + S::kWarps * (kSlots * kTileBytes) + warp * S::kQuery;
    pdl_launch_dependents();
    pdl_wait();

    const int tiles = (p.group + kRows - 1) / kRows;
    const int items = p.kv_heads * tiles;
    const int ksteps = (p.dim + 15) / 16;
    const int row_chunks = p.dim / 8;
    // The running maximum is one of unscaled scores, which takes a positive scale: a negative one's sign goes to the query, and
    // for a scale of 0 the query is 0.
    const float factor = p.scale * kLog2e;
    const float scale = factor == 0.0f ? 1.0f : fabsf(factor);
    const uint32_t query_and = factor == 0.0f ? 0u : 0xffffffffu, query_xor = factor < 0.0f ? 0x80008000u : 0u;

    // the list's length, and whether all sequences are short
    int64_t total = 0;
    int longest = 0, last_n = 0;  // last_n: tiles of sequence `lane`, of up to 32
    for (int b = lane; b < p.batch; b += 32) {
        const int n = sequence_of<KEYS>(p, b).tiles;
        total += n;
        longest = max(longest, n);
        last_n = n;
    }
    for (int o = 16; o > 0; o >>= 1) {
        total += __shfl_xor_sync(0xffffffffu, total, o);
        longest = max(longest, __shfl_xor_sync(0xffffffffu, longest, o));
    }
    total *= items;
    const int64_t all_items = static_cast<int64_t>(p.batch) * items;
    const bool whole = longest <= kShort / KEYS && all_items <= 2 * scratch.workers;
    const int64_t range = total < 0x7fffffff ? (static_cast<unsigned>(total) + scratch.workers - 1) / static_cast<unsigned>(scratch.workers)
                                             : (total + scratch.workers - 1) / scratch.workers;  // of a CTA
    if (!scratch.by_item && threadIdx.x == 0) scratch.cut[worker] = make_int4(-1, 0, 0, 0);

    // one round for the CTA's range; where head tiles are whole, one for each that the CTA has
    for (int64_t round = worker; round < (whole ? all_items : worker + 1); round += scratch.workers) {
        if (threadIdx.x < 2 * S::kWarps) s_parts[threadIdx.x].valid = 0;
        Piece load;
        int64_t begin = 0, end = 0;
        load.at = 0;
        load.b = load.item = load.from = load.to = 0;
        if (whole) {
            load.b = static_cast<int>(static_cast<unsigned>(round) / static_cast<unsigned>(items));  // few
            load.item = static_cast<int>(round - static_cast<int64_t>(load.b) * items);
            load.s = sequence_of<KEYS>(p, load.b);
            load.from = load.s.tiles * warp / S::kWarps;
            load.to = load.s.tiles * (warp + 1) / S::kWarps;
            end = load.to - load.from;
            if (load.s.tiles == 0 && warp == 0) {
                const int kvh = load.item / tiles, first = (load.item - kvh * tiles) * kRows;
                for (int h = first; h < min(first + kRows, p.group); ++h) empty_row<T>(p, load.b, kvh * p.group + h);
            }
            if (scratch.by_item && threadIdx.x == 0) scratch.cut[round] = make_int4(-1, 0, 0, 0);
        } else {
            const int64_t cta_begin = min(total, worker * range), cta_end = min(total, cta_begin + range);
            begin = cta_begin + (cta_end - cta_begin) * warp / S::kWarps;
            end = cta_begin + (cta_end - cta_begin) * (warp + 1) / S::kWarps;
            int64_t before = 0;
            bool found = false;
            // sequences that see nothing, and where this warp's range begins
            for (int b0 = 0; b0 < p.batch; b0 += 32) {
                const int b = b0 + lane;
                const int n = b < p.batch ? (p.batch <= 32 ? last_n : sequence_of<KEYS>(p, b).tiles) : 1;
                if (warp == 0) {
                    for (uint32_t none = __ballot_sync(0xffffffffu, n == 0); none != 0; none &= none - 1) {
                        const int e = b0 + __ffs(none) - 1;
                        if (e % scratch.workers != worker) continue;
                        for (int h = 0; h < p.heads; ++h) empty_row<T>(p, e, h);
                        if (scratch.by_item)
                            for (int i = lane; i < items; i += 32) scratch.cut[static_cast<int64_t>(e) * items + i] = make_int4(-1, 0, 0, 0);
                    }
                }
                if (found || begin >= end) continue;
                const int64_t mine = b < p.batch ? static_cast<int64_t>(n) * items : 0;
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
            if (found) {
                load.s = sequence_of<KEYS>(p, load.b);
                const int64_t in = begin - before;
                load.at = begin;
                load.item = static_cast<int>(in / load.s.tiles);
                load.from = static_cast<int>(in - static_cast<int64_t>(load.item) * load.s.tiles);
                load.to = static_cast<int>(min(static_cast<int64_t>(load.s.tiles), load.from + end - begin));
            }
        }
        Piece piece = load;
        bool more = load.to > load.from;
        bool working = more;
        __syncthreads();  // the parts' flags are clear

        // ---- loads: the query with a piece's first keys, then keys and values of a tile in turn ----
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
        const bool my_part = my_chunk < 2 * ksteps;
        const int my_offset = my_chunk < row_chunks ? my_chunk * 8 : 0;
        const bool even = p.page % 16 == 0 && row_chunks == 2 * ksteps;
        // the swizzled place of key kStep * i + my_key: chunk ^ key % 8, where the key's parts have no bits in common
        const uint32_t my_dst = my_key * (DP * 2) + ((my_chunk ^ my_key) << 4);
        auto copy_tile = [&](const void *cache, int64_t sb, int64_t st, int64_t sh) {
            const uint32_t dst = ring + slot * kTileBytes + my_dst;
            int64_t offset[kLooks];
            bool full = true;
#pragma unroll
            for (int l = 0; l < kLooks; ++l) {
                offset[l] = value_seen[l] >> lane & 1 ? value_entry[l] * sb + value_place[l] * st + value_head * sh : 0;
                full = full && value_seen[l] == 0xffffffffu;
            }
            const T *base = static_cast<const T *>(cache) + my_offset;
            // (which way is the usual one is said throughout, so that the loop lies close together: its warps wait for
            // instructions a quarter of the time)
            if (__builtin_expect(even, 1)) {
                const T *row[KEYS / 16];
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
                            cp_async_16((dst ^ ((first & 7) << 4)) + first * (DP * 2), row[first / 16], 16);
                            row[first / 16] += kStep * st;
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < KEYS / kStep; ++i) {
                            const int first = kStep * i;
                            const bool ok = value_seen[first / 32] >> ((first & 31) + my_key) & 1;
                            cp_async_16((dst ^ ((first & 7) << 4)) + first * (DP * 2), ok ? row[first / 16] : base, ok ? 16 : 0);
                            row[first / 16] += kStep * st;
                        }
                    }
                }
                return;
            }
#pragma unroll
            for (int i = 0; i < KEYS / kStep; ++i) {
                const int first = kStep * i, key = (first & 31) + my_key;
                const T *row = base + __shfl_sync(0xffffffffu, offset[first / 32], key);
                if (my_part)
                    cp_async_16((dst ^ ((first & 7) << 4)) + first * (DP * 2), row,
                                my_chunk < row_chunks && (value_seen[first / 32] >> key & 1) ? 16 : 0);
            }
        };
        auto copy_query = [&] {
            const int kvh = load.item / tiles, tile = load.item - kvh * tiles;
            const int rows = min(kRows, p.group - tile * kRows);
            const T *base = static_cast<const T *>(p.q) + load.b * p.q_st + (kvh * p.group + tile * kRows) * p.q_sh + my_offset;
#pragma unroll
            for (int i = 0; i < kRows / kStep; ++i) {
                const int first = kStep * i, row = first + my_key;
                if (my_part)
                    cp_async_16(((query + my_dst) ^ ((first & 7) << 4)) + first * (DP * 2), base + (row < rows ? row * p.q_sh : 0),
                                row < rows && my_chunk < row_chunks ? 16 : 0);
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
                copy_tile(p.k, p.k_sb, p.k_st, p.k_sh);
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
            if (value_head >= 0) copy_tile(p.v, p.v_sb, p.v_st, p.v_sh);
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
        // ldmatrix addresses: chunk 2 i + c of a row swizzled by r is (2 i) ^ (c ^ r), so a step is one exclusive or
        auto query_part = [&](uint32_t (&r)[4], int ks) {
            ldmatrix_x4(r, (query + (lane & 15) * (DP * 2) + (((lane >> 4) ^ (lane & 7)) << 4)) ^ (ks << 5));
#pragma unroll
            for (int i = 0; i < 4; ++i) r[i] = (r[i] & query_and) ^ query_xor;
        };
        while (working) {
            float o[DP / 8][4];
#pragma unroll
            for (int n = 0; n < DP / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f;
            float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.0f, 0.0f};
            // A long piece adds what it has to fp32 sums in its part of the workspace and begins again from 0 (back: the other way round).
            auto put_by = [&](bool first, bool back) {
                const int rows = min(kRows, p.group - piece.item % tiles * kRows);
                const int64_t part0 = ((static_cast<int64_t>(worker) * S::kWarps + warp) * 2 + (piece.from == 0)) * scratch.rows;
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const int row = r0 + r * 8;
                    float *sums = scratch.part + (part0 + row) * p.dim + c0;
                    float keep = 1.0f;
                    if (row < rows && !first && top[r] != -INFINITY) keep = exp2_fast((scratch.stat[part0 + row].x - top[r]) * scale);
                    __syncwarp();
                    if (row < rows && (lane & 3) == 0) scratch.stat[part0 + row].x = top[r];
#pragma unroll
                    for (int n = 0; n < DP / 8; ++n) {
                        float2 x = make_float2(0.0f, 0.0f);
                        if (row < rows && n * 8 < p.dim) {
                            if (!first) x = *reinterpret_cast<const float2 *>(sums + n * 8);
                            x.x = fmaf(x.x, keep, o[n][2 * r]);
                            x.y = fmaf(x.y, keep, o[n][2 * r + 1]);
                            if (!back) *reinterpret_cast<float2 *>(sums + n * 8) = x;
                        }
                        o[n][2 * r] = back ? x.x : 0.0f;
                        o[n][2 * r + 1] = back ? x.y : 0.0f;
                    }
                }
            };
            for (int g = piece.from; g < piece.to; ++g) {
                if (FAR && g != piece.from && (g - piece.from) % (kRun / KEYS) == 0) put_by(g - piece.from == kRun / KEYS, false);
                // scores of 16 rows x KEYS keys: accumulators of 8 keys
                float s[KEYS / 8][4];
#pragma unroll
                for (int n = 0; n < KEYS / 8; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
                cp_async_wait<kSlots - 2>();
                __syncwarp();
                bool all_seen = true;
#pragma unroll
                for (int l = 0; l < kLooks; ++l) {
                    seen[l] = value_seen[l];
                    all_seen = all_seen && seen[l] == 0xffffffffu;
                }
                if (kKept) {
                    if (g == piece.from) {
#pragma unroll
                        for (int ks = 0; ks < DP / 16; ++ks) query_part(q[kKept ? ks : 0], ks);
                    }
                    load_keys();  // into the slot of the values before
                }
                const uint32_t keys = ring + use_slot * kTileBytes + (((lane >> 4) << 3) + (lane & 7)) * (DP * 2) +
                                      ((((lane >> 3) & 1) ^ (lane & 7)) << 4);
                use_slot = use_slot + 1 == kSlots ? 0 : use_slot + 1;
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
                if (!kKept) {
                    __syncwarp();  // the query may be overwritten
                    load_keys();
                }
                if (__builtin_expect(!all_seen, 0)) {
#pragma unroll
                    for (int n = 0; n < KEYS / 8; ++n) {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (!(seen[n / 4] >> (n % 4 * 8 + c0 + (i & 1)) & 1)) s[n][i] = -INFINITY;
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
                if (__builtin_expect(__any_sync(0xffffffffu, moved), 0)) {
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
                // the weights, rounded to the type of the values, as they lie are the second product's first operand.  That is half a
                // step, 2^-8 or 2^-11, of each weight (of f16 weights below 2^-29 of the largest: 2^-40 of that one).  The sum
                // takes them unrounded, so equal weights are all off alike.
                uint32_t a[KEYS / 16][4];
                if (kLift<T> != 0.0f) {
                    base[0] -= kLift<T>;
                    base[1] -= kLift<T>;
                }
#pragma unroll
                for (int n = 0; n < KEYS / 8; ++n) {
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const float e0 = exp2_fast(fmaf(s[n][2 * r], scale, -base[r])), e1 = exp2_fast(fmaf(s[n][2 * r + 1], scale, -base[r]));
                        sum[r] += e0 + e1;
                        a[n >> 1][(n & 1) * 2 + r] = pack2<T>(e0, e1);
                    }
                }
                cp_async_wait<kSlots - 2>();
                __syncwarp();
                load_values();  // into the slot of the keys
                const uint32_t values = ring + use_slot * kTileBytes + ((((lane >> 3) & 1) << 3) + (lane & 7)) * (DP * 2) +
                                        (((lane >> 4) ^ (lane & 7)) << 4);
                use_slot = use_slot + 1 == kSlots ? 0 : use_slot + 1;
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
                top[r] = fmaf(top[r], scale, -kLift<T>);  // the sums are 2^kLift times those of exp(score - maximum)
                const int row = r0 + r * 8;
                if (row >= rows) continue;
                if (begins && ends) {
                    const float inv = sum[r] == 0.0f ? 0.0f : 1.0f / sum[r];
                    T *dst = static_cast<T *>(p.out) + (row0 + row) * p.dim;
#pragma unroll
                    for (int n = 0; n < DP / 8; ++n)
                        if (n * 8 < p.dim)
                            *reinterpret_cast<uint32_t *>(dst + n * 8 + c0) = pack2<T>(o[n][2 * r] * inv, o[n][2 * r + 1] * inv);
                    if ((lane & 3) == 0) p.lse[row0 + row] = sum[r] == 0.0f ? -INFINITY : top[r] * kLn2 + logf(sum[r]);
                } else {
                    float *dst = scratch.part + (part0 + row) * p.dim;
#pragma unroll
                    for (int n = 0; n < DP / 8; ++n)
                        if (n * 8 < p.dim) *reinterpret_cast<float2 *>(dst + n * 8 + c0) = make_float2(o[n][2 * r], o[n][2 * r + 1]);
                    if ((lane & 3) == 0) scratch.stat[part0 + row] = make_float2(top[r], sum[r]);
                }
            }
            if (lane == 0) {
                if (!(begins && ends))
                    s_parts[2 * warp + begins] = {1, piece.b, piece.item, begins, ends, whole ? worker : static_cast<int>((piece.at - piece.from + piece.s.tiles - 1) / range)};
                else if (scratch.by_item && !whole)
                    scratch.cut[static_cast<int64_t>(piece.b) * items + piece.item] = make_int4(-1, 0, 0, 0);
            }
            working = next_piece<KEYS>(p, end, items, piece);
        }
        cp_async_wait<0>();
        __syncthreads();

        // ---- the warps' parts: neighbours of one head tile are added in their order (a warp's second part is its last) ----
        // Every thread has four columns of a row of all of them, loaded together: one after the other, a part's latency each,
        // took 10 of 133 us (64 sequences of 500 to 8000 places, 64/8 heads of 128).
        const int64_t first_part = static_cast<int64_t>(worker) * S::kWarps * 2;
        for (int idx = threadIdx.x; idx < scratch.rows * (p.dim / 4); idx += kThreads) {
            const int row = idx / (p.dim / 4), d = (idx - row * (p.dim / 4)) * 4;
            float2 stat[2 * S::kWarps];
            float4 x[2 * S::kWarps];
#pragma unroll
            for (int i = 0; i < 2 * S::kWarps; ++i) {
                if (s_parts[i].valid) {  // (rows behind the last of a head tile are never written and never used)
                    stat[i] = __ldcg(scratch.stat + (first_part + i) * scratch.rows + row);
                    x[i] = __ldcg(reinterpret_cast<const float4 *>(scratch.part + ((first_part + i) * scratch.rows + row) * p.dim + d));
                }
            }
            float now = -INFINITY, all = 0.0f;
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            bool open = false, begins = false;
            int last_part = 0;
            auto close = [&](bool ends) {
                const Part &part = s_parts[last_part];
                const int kvh = part.item / tiles, tile = part.item - kvh * tiles;
                if (row < min(kRows, p.group - tile * kRows)) {
                    if (begins && ends) {
                        const int64_t to = static_cast<int64_t>(part.b) * p.heads + kvh * p.group + tile * kRows + row;
                        const float inv = all == 0.0f ? 0.0f : 1.0f / all;
                        *reinterpret_cast<uint2 *>(static_cast<T *>(p.out) + to * p.dim + d) =
                            make_uint2(pack2<T>(v.x * inv, v.y * inv), pack2<T>(v.z * inv, v.w * inv));
                        if (d == 0) p.lse[to] = all == 0.0f ? -INFINITY : now * kLn2 + logf(all);
                    } else {
                        const int64_t to = (scratch.cta_parts + 2 * worker + begins) * scratch.rows + row;
                        *reinterpret_cast<float4 *>(scratch.part + to * p.dim + d) = v;
                        if (d == 0) scratch.stat[to] = make_float2(now, all);
                    }
                }
                if (idx == 0 && begins && !whole) {
                    const int64_t index = static_cast<int64_t>(part.b) * items + part.item;
                    if (!ends)
                        scratch.cut[scratch.by_item ? index : worker] = make_int4(worker, part.last, part.b, part.item);
                    else if (scratch.by_item)
                        scratch.cut[index] = make_int4(-1, 0, 0, 0);
                }
                open = false;
            };
#pragma unroll
            for (int i = 0; i < 2 * S::kWarps; ++i) {
                if (!s_parts[i].valid) continue;
                if (!open) {
                    open = true;
                    begins = s_parts[i].begins != 0;
                    now = stat[i].x;
                    all = stat[i].y;
                    v = x[i];
                } else {
                    const float most = fmaxf(now, stat[i].x), base = most == -INFINITY ? 0.0f : most;
                    const float keep = exp2_fast(now - base), add = exp2_fast(stat[i].x - base);
                    all = fmaf(stat[i].y, add, all * keep);
                    v.x = fmaf(x[i].x, add, v.x * keep);
                    v.y = fmaf(x[i].y, add, v.y * keep);
                    v.z = fmaf(x[i].z, add, v.z * keep);
                    v.w = fmaf(x[i].w, add, v.w * keep);
                    now = most;
                }
                last_part = i;
                if (s_parts[i].ends) close(true);
            }
            if (open) close(false);
        }
        __syncthreads();
    }
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
        auto place = [&](int i) { return (scratch.cta_parts + static_cast<int64_t>(cut.x + i) * 2 + (i == 0)) * scratch.rows + row; };
        // Four parts at a time, their statistics and sums loaded together, onto a running maximum.
        float top = -INFINITY, sum = 0.0f, acc[8] = {};
        for (int i0 = from; i0 < to; i0 += 4) {
            float2 stat[4];
            float4 v[4][2];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                stat[i] = make_float2(-INFINITY, 0.0f);
                v[i][0] = v[i][1] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (i0 + i >= to) continue;
                stat[i] = scratch.stat[place(i0 + i)];
                const float *src = scratch.part + place(i0 + i) * p.dim;
#pragma unroll
                for (int c = 0; c < 2; ++c)
                    if (c * 128 + lane * 4 < p.dim) v[i][c] = *reinterpret_cast<const float4 *>(src + c * 128 + lane * 4);
            }
            const float now = fmaxf(fmaxf(fmaxf(top, stat[0].x), fmaxf(stat[1].x, stat[2].x)), stat[3].x);
            const float base = now == -INFINITY ? 0.0f : now, keep = exp2_fast(top - base);
            sum *= keep;
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[j] *= keep;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float w = exp2_fast(stat[i].x - base);
                sum = fmaf(stat[i].y, w, sum);
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    acc[4 * c] = fmaf(v[i][c].x, w, acc[4 * c]);
                    acc[4 * c + 1] = fmaf(v[i][c].y, w, acc[4 * c + 1]);
                    acc[4 * c + 2] = fmaf(v[i][c].z, w, acc[4 * c + 2]);
                    acc[4 * c + 3] = fmaf(v[i][c].w, w, acc[4 * c + 3]);
                }
            }
            top = now;
        }
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

template <typename T, int DP, bool FAR>
int launch_decode_kernel(const Problem &p, const Plan &plan, const Scratch &scratch, cudaStream_t stream) {
    QMM_CUDA_OK(cudaFuncSetAttribute(decode_kernel<T, DP, FAR>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(Shape<DP>::kSmem)));
    QMM_CUDA_OK(launch_pdl(decode_kernel<T, DP, FAR>, dim3(plan.workers), dim3(Shape<DP>::kWarps * 32), Shape<DP>::kSmem, stream, p, scratch));
    return QMM_OK;
}

template <typename T, int DP>
int launch(const Problem &p, const Plan &plan, const Scratch &scratch, cudaStream_t stream) {
    // what a warp may have: of one head tile what a token sees, of all of them an equal share
    const int64_t seen = p.window > 0 ? std::min<int64_t>(p.capacity, static_cast<int64_t>(p.window) + p.sinks) : p.capacity;
    const bool far = seen > kNear && seen > kNear * plan.workers * Shape<DP>::kWarps / plan.items;
    const int rc = far ? launch_decode_kernel<T, DP, true>(p, plan, scratch, stream) : launch_decode_kernel<T, DP, false>(p, plan, scratch, stream);
    if (rc != QMM_OK) return rc;
    // all sequences are short whatever their lengths are, and no head tile is cut
    if (p.capacity <= kShort && plan.items <= 2 * plan.workers) return QMM_OK;
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
    scratch.cta_parts = plan.cta_parts;
    return dtype == QMM_DTYPE_BF16 ? launch_t<__nv_bfloat16>(p, plan, scratch, stream) : launch_t<__half>(p, plan, scratch, stream);
}

}  // namespace paged
}  // namespace qmm
