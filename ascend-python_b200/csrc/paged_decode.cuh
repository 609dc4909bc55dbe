// What the decode kernels over a paged cache share (paged_decode.cu: 16-bit caches, paged_quant_decode.cu: 8-bit ones): the list of
// a call's work and its ranges, the parts of head tiles that are cut, and how they are joined.
#pragma once

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

// `ctas` an SM of `warps` warps each.
inline Plan make_plan(int64_t batch, int64_t heads, int64_t kv_heads, int64_t dim, int ctas, int warps) {
    Plan plan;
    const int64_t group = kv_heads > 0 ? heads / kv_heads : 0;
    plan.workers = ctas * sm_count();
    plan.rows = static_cast<int>(group < kRows ? group : kRows);
    plan.tiles = static_cast<int>((group + kRows - 1) / kRows);
    plan.items = batch * kv_heads * plan.tiles;
    plan.cta_parts = 2ll * plan.workers * warps;
    const size_t rows = static_cast<size_t>(plan.cta_parts + 2 * plan.workers) * plan.rows;
    plan.part_bytes = rows * dim * sizeof(float);
    plan.stat_bytes = (rows * sizeof(float2) + 15) / 16 * 16;
    plan.bytes = plan.part_bytes + plan.stat_bytes + static_cast<size_t>(plan.workers) * sizeof(int4);
    return plan;
}

inline Scratch lay_out(const Plan &plan, void *workspace) {
    Scratch scratch;
    uint8_t *base = static_cast<uint8_t *>(workspace);
    scratch.part = reinterpret_cast<float *>(base);
    scratch.stat = reinterpret_cast<float2 *>(base + plan.part_bytes);
    scratch.cut = reinterpret_cast<int4 *>(base + plan.part_bytes + plan.stat_bytes);
    scratch.rows = plan.rows;
    scratch.workers = plan.workers;
    scratch.by_item = plan.items <= plan.workers;
    scratch.cta_parts = plan.cta_parts;
    return scratch;
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

// What a warp left of a head tile, for the CTA to add up.
struct Part {
    int valid, b, item, begins, ends, last;  // last: the CTA that has the head tile's last place
};

// The list of a call's work: (sequence, head tile, tile of KEYS places).
struct List {
    int items;          // head tiles of a sequence
    int last_n;         // tiles of places of sequence `lane`, of up to 32
    bool whole;         // all sequences are short and head tiles are few: CTAs have whole ones
    int64_t all_items;  // head tiles
    int64_t total, range;  // tiles of places, and those of a CTA
};

template <int KEYS>
__device__ __forceinline__ List make_list(const Problem &p, const Scratch &scratch, int items) {
    const int lane = threadIdx.x & 31;
    List list;
    list.items = items;
    list.last_n = 0;
    int64_t total = 0;
    int longest = 0;
    for (int b = lane; b < p.batch; b += 32) {
        const int n = sequence_of<KEYS>(p, b).tiles;
        total += n;
        longest = max(longest, n);
        list.last_n = n;
    }
    for (int o = 16; o > 0; o >>= 1) {
        total += __shfl_xor_sync(0xffffffffu, total, o);
        longest = max(longest, __shfl_xor_sync(0xffffffffu, longest, o));
    }
    total *= items;
    list.all_items = static_cast<int64_t>(p.batch) * items;
    list.whole = longest <= kShort / KEYS && list.all_items <= 2 * scratch.workers;
    list.total = total;
    list.range = total < 0x7fffffff ? (static_cast<unsigned>(total) + scratch.workers - 1) / static_cast<unsigned>(scratch.workers)
                                    : (total + scratch.workers - 1) / scratch.workers;
    return list;
}

// A round of a CTA: its range, or one head tile that it has whole.  Gives the first piece of the warp's part (empty: load.from ==
// load.to) and where that part ends.
template <typename T, int KEYS, int WARPS>
__device__ __forceinline__ void begin_round(const Problem &p, const Scratch &scratch, const List &list, int64_t round, int tiles, Piece &load, int64_t &end) {
    const int warp = warp_id_uniform(), lane = threadIdx.x & 31, worker = blockIdx.x, items = list.items, last_n = list.last_n;
    const int64_t total = list.total, range = list.range;
    int64_t begin = 0;
    end = 0;
    load.at = 0;
    load.b = load.item = load.from = load.to = 0;
    if (list.whole) {
        load.b = static_cast<int>(static_cast<unsigned>(round) / static_cast<unsigned>(items));  // few
        load.item = static_cast<int>(round - static_cast<int64_t>(load.b) * items);
        load.s = sequence_of<KEYS>(p, load.b);
        load.from = load.s.tiles * warp / WARPS;
        load.to = load.s.tiles * (warp + 1) / WARPS;
        end = load.to - load.from;
        if (load.s.tiles == 0 && warp == 0) {
            const int kvh = load.item / tiles, first = (load.item - kvh * tiles) * kRows;
            for (int h = first; h < min(first + kRows, p.group); ++h) empty_row<T>(p, load.b, kvh * p.group + h);
        }
        if (scratch.by_item && threadIdx.x == 0) scratch.cut[round] = make_int4(-1, 0, 0, 0);
    } else {
        const int64_t cta_begin = min(total, worker * range), cta_end = min(total, cta_begin + range);
        begin = cta_begin + (cta_end - cta_begin) * warp / WARPS;
        end = cta_begin + (cta_end - cta_begin) * (warp + 1) / WARPS;
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
}

// Adds up what the CTA's warps left of head tiles in their parts: neighbours of one head tile, in their order (a warp's second part is its
// last).  Every thread has four columns of a row of all of them, loaded together: one after the other, a part's latency each,
// took 10 of 133 us (64 sequences of 500 to 8000 places, 64/8 heads of 128).
template <typename T, int WARPS>
__device__ __forceinline__ void add_parts(const Problem &p, const Scratch &scratch, const List &list, const Part *s_parts, int tiles) {
    constexpr int kThreads = WARPS * 32;
    const int worker = blockIdx.x, items = list.items;
    const bool whole = list.whole;
    const int64_t first_part = static_cast<int64_t>(worker) * WARPS * 2;
    for (int idx = threadIdx.x; idx < scratch.rows * (p.dim / 4); idx += kThreads) {
        const int row = idx / (p.dim / 4), d = (idx - row * (p.dim / 4)) * 4;
        float2 stat[2 * WARPS];
        float4 x[2 * WARPS];
#pragma unroll
        for (int i = 0; i < 2 * WARPS; ++i) {
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
        for (int i = 0; i < 2 * WARPS; ++i) {
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

// Whether a warp may have more than kNear places: of one head tile what a token sees, of all of them an equal share.
inline bool is_far(const Problem &p, const Plan &plan, int warps) {
    const int64_t seen = p.window > 0 ? std::min<int64_t>(p.capacity, static_cast<int64_t>(p.window) + p.sinks) : p.capacity;
    return seen > kNear && seen > kNear * plan.workers * warps / plan.items;
}

template <typename T>
int launch_join(const Problem &p, const Plan &plan, const Scratch &scratch, cudaStream_t stream) {
    // all sequences are short whatever their lengths are, and no head tile is cut
    if (p.capacity <= kShort && plan.items <= 2 * plan.workers) return QMM_OK;
    const int64_t indices = scratch.by_item ? plan.items : plan.workers;
    const bool share_parts = indices * plan.rows <= 8 * sm_count();
    QMM_CUDA_OK(launch_pdl(join_kernel<T>, dim3(static_cast<unsigned>(indices), share_parts ? plan.rows : 1), dim3(kJoinWarps * 32), 0,
                           stream, p, scratch, share_parts));
    return QMM_OK;
}

}  // namespace

}  // namespace paged
}  // namespace qmm
