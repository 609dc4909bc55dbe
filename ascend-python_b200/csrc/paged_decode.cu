// Attention of one new token a sequence over a paged key-value cache (npu_paged_attention).
//
// Bound by HBM: every visible key and value is read once, for all query heads that share it.  The heads of a group (16 at a
// time) are the rows of mma.sync m16n8k16, so a key costs the tensor pipe the same for one head as for sixteen, about a fifth of
// the time its bytes take (tcgen05 would need 64 rows at least and a hand-off through tensor memory for every few keys).
//
// One warp is one worker and never waits for another: it has a private ring of stages of 16 keys and values in shared memory,
// filled by cp.async with the rows' page looked up one stage ahead.  Places that are not seen are not read but zero-filled, so
// what lies there has no part in any product.  The softmax is one pass: running maximum and sum a row, sums rescaled only
// when a maximum moved.
//
// The work of a call is the list of all (sequence, head tile, 16 keys), cut into equal contiguous ranges, one for each worker,
// wherever sequences begin and end; so a batch of ragged lengths and one long sequence load the GPU alike.  A sequence's heads
// that one worker has whole are written from registers; of a cut one each worker leaves its sums, and a second kernel joins
// them in the workers' order.  Nothing depends on timing, and nothing has to be zero before a call.
#include "paged_common.cuh"

namespace qmm {
namespace paged {

namespace {

constexpr int kKeys = 16;       // keys of a stage
constexpr int kRows = 16;       // query heads of a tile
constexpr int kMinRange = 4;    // stages of a worker at least, where there are as many

// DP: the head dimension rounded up to 64, 128 or 256.  Shared memory of a CTA: 128, 192 and 192 KiB.
template <int DP>
struct Shape {
    static constexpr int kStages = DP == 64 ? 4 : DP == 128 ? 3 : 2;
    static constexpr int kWarps = DP == 256 ? 6 : 8;
    static constexpr int kTileBytes = kKeys * DP * 2;
    static constexpr int kStageBytes = 2 * kTileBytes;
    static constexpr size_t kSmem = static_cast<size_t>(kWarps) * kStages * kStageBytes;
};

// Workspace: part[worker][2][rows][dim] sums, stat[worker][2][rows] (maximum, sum), cut[index]: the first and last worker
// of a cut item (first < 0: not cut), by item where there are no more items than workers, else by the item's first worker.
struct Scratch {
    float *part;
    float2 *stat;
    int4 *cut;
    int rows, workers, by_item;
};

struct Plan {
    int sms, warps, workers, rows, tiles;
    int64_t items;
    size_t part_bytes, stat_bytes, bytes;
};

Plan make_plan(int64_t batch, int64_t heads, int64_t kv_heads, int64_t dim) {
    Plan plan;
    const int64_t group = kv_heads > 0 ? heads / kv_heads : 0;
    plan.sms = sm_count();
    plan.warps = dim > 128 ? Shape<256>::kWarps : Shape<128>::kWarps;
    plan.workers = plan.sms * plan.warps;
    plan.rows = static_cast<int>(group < kRows ? group : kRows);
    plan.tiles = static_cast<int>((group + kRows - 1) / kRows);
    plan.items = batch * kv_heads * plan.tiles;
    plan.part_bytes = static_cast<size_t>(plan.workers) * 2 * plan.rows * dim * sizeof(float);
    plan.stat_bytes = (static_cast<size_t>(plan.workers) * 2 * plan.rows * sizeof(float2) + 15) / 16 * 16;
    plan.bytes = plan.part_bytes + plan.stat_bytes + static_cast<size_t>(plan.workers) * sizeof(int4);
    return plan;
}

// What a sequence's token sees, as stages of 16 places: those of the sinks, then those of the window.
struct Sequence {
    int sink_end, lo, hi, sink_stages, first, stages;
};
__device__ __forceinline__ Sequence sequence_of(const Problem &p, int b) {
    const int len = p.lens[b];
    const Range r = visible_range(p, len <= 0 ? -1 : len - 1);
    Sequence s;
    s.sink_end = r.sink_end;
    s.lo = r.lo;
    s.hi = r.hi;
    s.sink_stages = (r.sink_end + kKeys - 1) / kKeys;
    s.first = max(r.lo / kKeys, s.sink_stages);
    const int end = r.hi / kKeys + (r.hi % kKeys != 0);
    s.stages = s.sink_stages + max(0, end - s.first);
    return s;
}

struct Cursor {
    int b, item, at;  // sequence, head tile of it, stage of that
    Sequence s;
};

// Steps to the next stage of the list; `left`: how many there are from here on (at least 1).
__device__ __forceinline__ void step(const Problem &p, Cursor &c, int items, bool more) {
    if (++c.at < c.s.stages) return;
    c.at = 0;
    if (++c.item < items) return;
    c.item = 0;
    if (!more) return;
    do {
        c.s = sequence_of(p, ++c.b);
    } while (c.s.stages == 0);
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
__global__ void __launch_bounds__(Shape<DP>::kWarps * 32, 1)
decode_kernel(const __grid_constant__ Problem p, const __grid_constant__ Scratch scratch) {
    using S = Shape<DP>;
    extern __shared__ __align__(128) uint8_t smem[];
    constexpr int kChunks = DP / 8;  // 16-byte chunks of a row in shared memory
    const int warp = warp_id_uniform(), lane = threadIdx.x & 31;
    // neighbours of the list go to different SMs
    const int worker = warp * gridDim.x + blockIdx.x;
    const uint32_t ring = smem_u32(smem) + warp * (S::kStages * S::kStageBytes);
    pdl_launch_dependents();
    pdl_wait();

    const int tiles = (p.group + kRows - 1) / kRows;
    const int items = p.kv_heads * tiles;
    const int ksteps = (p.dim + 15) / 16;
    const int row_chunks = p.dim / 8;

    // sequences that see nothing, and the list's length
    int64_t total = 0;
    for (int b0 = 0; b0 < p.batch; b0 += 32) {
        const int b = b0 + lane;
        const int n = b < p.batch ? sequence_of(p, b).stages : 1;
        if (b < p.batch) total += n;
        for (uint32_t none = __ballot_sync(0xffffffffu, n == 0); none != 0; none &= none - 1) {
            const int e = b0 + __ffs(none) - 1;
            if (e % scratch.workers != worker) continue;
            for (int h = 0; h < p.heads; ++h) empty_row<T>(p, e, h);
            if (scratch.by_item)
                for (int i = lane; i < items; i += 32) scratch.cut[static_cast<int64_t>(e) * items + i] = make_int4(-1, 0, 0, 0);
        }
    }
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    total *= items;
    const int64_t range = max(static_cast<int64_t>(kMinRange), (total + scratch.workers - 1) / scratch.workers);
    const int64_t begin = worker * range;
    const int64_t end = min(total, begin + range);
    if (!scratch.by_item && lane == 0) scratch.cut[worker] = make_int4(-1, 0, 0, 0);
    if (begin >= end) return;

    // where this worker's range begins
    Cursor load;
    {
        int64_t before = 0;
        for (int b0 = 0;; b0 += 32) {
            const int b = b0 + lane;
            const int64_t n = b < p.batch ? static_cast<int64_t>(sequence_of(p, b).stages) * items : 0;
            int64_t sum = n;
            for (int o = 1; o < 32; o <<= 1) {
                const int64_t left = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += left;
            }
            const uint32_t past = __ballot_sync(0xffffffffu, before + sum > begin);
            if (past == 0) {
                before += __shfl_sync(0xffffffffu, sum, 31);
                continue;
            }
            const int which = __ffs(past) - 1;
            load.b = b0 + which;
            before += __shfl_sync(0xffffffffu, sum - n, which);
            break;
        }
        load.s = sequence_of(p, load.b);
        const int64_t in = begin - before;
        load.item = static_cast<int>(in / load.s.stages);
        load.at = static_cast<int>(in - static_cast<int64_t>(load.item) * load.s.stages);
    }
    Cursor use = load;

    // ---- loads: lanes 0..15 look up the stage's keys, lanes 16..31 its values ----
    int64_t loads_left = end - begin;
    int at_place = 0, entry = 0;
    bool at_seen = false;
    auto look_up = [&] {
        const int first = load.at < load.s.sink_stages ? load.at * kKeys : (load.s.first + load.at - load.s.sink_stages) * kKeys;
        const int j = first + (lane & 15);
        at_seen = j < load.s.hi && (j < load.s.sink_end || j >= load.s.lo);
        const int page = at_seen ? page_of(p, j) : 0;
        at_place = j - page * p.page;
        entry = at_seen ? __ldg(p.table + load.b * p.table_st + page) : -1;
    };
    uint64_t seen_queue = 0;  // 16 bits for each stage under way
    int under_way = 0, load_slot = 0;
    auto produce = [&] {
        if (loads_left > 0) {
            const bool ok = at_seen && entry >= 0 && entry < p.pages;
            const uint32_t seen = __ballot_sync(0xffffffffu, ok);
            seen_queue |= static_cast<uint64_t>(seen & 0xffffu) << (16 * under_way);
            const int kvh = load.item / tiles;
            const bool keys = lane < 16;
            const int64_t offset = ok ? entry * (keys ? p.k_sb : p.v_sb) + at_place * (keys ? p.k_st : p.v_st) + kvh * (keys ? p.k_sh : p.v_sh) : 0;
            const uint32_t stage = ring + load_slot * S::kStageBytes;
#pragma unroll
            for (int part = 0; part < 2; ++part) {
                const T *base = static_cast<const T *>(part == 0 ? p.k : p.v);
#pragma unroll
                for (int i = 0; i < kChunks / 2; ++i) {
                    const int idx = i * 32 + lane, key = idx / kChunks, chunk = idx % kChunks;
                    const T *row = base + __shfl_sync(0xffffffffu, offset, key + 16 * part);
                    if (chunk < 2 * ksteps)
                        cp_async_16(stage + part * S::kTileBytes + key * (DP * 2) + ((chunk ^ (key & 7)) << 4),
                                    row + (chunk < row_chunks ? chunk * 8 : 0), chunk < row_chunks && (seen >> key & 1) ? 16 : 0);
                }
            }
            --loads_left;
            step(p, load, items, loads_left > 0);
            if (loads_left > 0) look_up();
        }
        cp_async_commit();
        ++under_way;
        load_slot = load_slot + 1 == S::kStages ? 0 : load_slot + 1;
    };
    look_up();
#pragma unroll
    for (int i = 0; i < S::kStages - 1; ++i) produce();

    // ---- products ----
    const float scale = p.scale * kLog2e;
    const int r0 = lane >> 2, c0 = (lane & 3) * 2;
    uint32_t q[DP / 16][4];
    float o[DP / 8][4];
    float top[2], sum[2];
    bool fresh = true;
    int use_slot = 0;
    bool whole = use.at == 0;  // this worker has the item from its first stage on
    for (int64_t u = begin; u < end; ++u) {
        const int kvh = use.item / tiles, tile = use.item - kvh * tiles;
        const int head0 = kvh * p.group + tile * kRows;
        const int rows = min(kRows, p.group - tile * kRows);
        if (fresh) {
            fresh = false;
            const T *base = static_cast<const T *>(p.q) + use.b * p.q_st + head0 * p.q_sh;
#pragma unroll
            for (int ks = 0; ks < DP / 16; ++ks) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int row = r0 + (i & 1) * 8, col = ks * 16 + (i >> 1) * 8 + c0;
                    q[ks][i] = row < rows && col < p.dim ? __ldg(reinterpret_cast<const uint32_t *>(base + row * p.q_sh + col)) : 0;
                }
            }
#pragma unroll
            for (int n = 0; n < DP / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f;
            top[0] = top[1] = -INFINITY;
            sum[0] = sum[1] = 0.0f;
        }
        cp_async_wait<S::kStages - 2>();
        __syncwarp();
        const uint32_t seen = static_cast<uint32_t>(seen_queue) & 0xffffu;
        seen_queue >>= 16;
        --under_way;
        produce();  // into the stage that the step before this one used
        const uint32_t keys = ring + use_slot * S::kStageBytes, values = keys + S::kTileBytes;
        use_slot = use_slot + 1 == S::kStages ? 0 : use_slot + 1;

        // scores of 16 rows x 16 keys: two accumulators of 8 keys
        float s[2][4] = {};
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks) {
            if (ks >= ksteps) break;
            uint32_t b[4];
            const int key = ((lane >> 4) << 3) + (lane & 7), chunk = ks * 2 + ((lane >> 3) & 1);
            ldmatrix_x4(b, keys + key * (DP * 2) + ((chunk ^ (key & 7)) << 4));
            mma_16816<T>(s[0], q[ks], b[0], b[1]);
            mma_16816<T>(s[1], q[ks], b[2], b[3]);
        }
        float most[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int n = 0; n < 2; ++n) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int key = n * 8 + c0 + (i & 1);
                // hidden behind the scaling, whose sign and zero a hidden score must not meet
                s[n][i] = seen >> key & 1 ? s[n][i] * scale : -INFINITY;
                most[i >> 1] = fmaxf(most[i >> 1], s[n][i]);
            }
        }
        bool moved = false;
        float base[2], keep[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            most[r] = fmaxf(most[r], __shfl_xor_sync(0xffffffffu, most[r], 1));
            most[r] = fmaxf(most[r], __shfl_xor_sync(0xffffffffu, most[r], 2));
            const float now = fmaxf(top[r], most[r]);
            base[r] = now == -INFINITY ? 0.0f : now;
            keep[r] = exp2_fast(top[r] - base[r]);
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
        float e[2][4];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                e[n][i] = exp2_fast(s[n][i] - base[i >> 1]);
                sum[i >> 1] += e[n][i];
            }
        }
        // the weights, rounded to the type of the values (the sum above takes them unrounded: 2^-9 or 2^-12 of each weight,
        // independent of one another), as they lie are the second product's first operand
        const uint32_t a[4] = {pack2<T>(e[0][0], e[0][1]), pack2<T>(e[0][2], e[0][3]), pack2<T>(e[1][0], e[1][1]),
                               pack2<T>(e[1][2], e[1][3])};
#pragma unroll
        for (int n = 0; n < DP / 16; ++n) {
            if (n >= ksteps) break;
            uint32_t b[4];
            const int key = (((lane >> 3) & 1) << 3) + (lane & 7), chunk = n * 2 + (lane >> 4);
            ldmatrix_x4_trans(b, values + key * (DP * 2) + ((chunk ^ (key & 7)) << 4));
            mma_16816<T>(o[2 * n], a, b[0], b[1]);
            mma_16816<T>(o[2 * n + 1], a, b[2], b[3]);
        }

        const bool item_ends = use.at + 1 == use.s.stages;
        if (item_ends || u + 1 == end) {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 1);
                sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 2);
            }
            const int64_t index = static_cast<int64_t>(use.b) * items + use.item;
            if (whole && item_ends) {
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const int row = r0 + r * 8;
                    if (row >= rows) continue;
                    const int64_t at = static_cast<int64_t>(use.b) * p.heads + head0 + row;
                    const float inv = sum[r] == 0.0f ? 0.0f : 1.0f / sum[r];
                    T *dst = static_cast<T *>(p.out) + at * p.dim;
#pragma unroll
                    for (int n = 0; n < DP / 8; ++n)
                        if (n * 8 < p.dim)
                            *reinterpret_cast<uint32_t *>(dst + n * 8 + c0) = pack2<T>(o[n][2 * r] * inv, o[n][2 * r + 1] * inv);
                    if ((lane & 3) == 0) p.lse[at] = sum[r] == 0.0f ? -INFINITY : top[r] * kLn2 + logf(sum[r]);
                }
                if (scratch.by_item && lane == 0) scratch.cut[index] = make_int4(-1, 0, 0, 0);
            } else {
                const int64_t slot = worker * 2 + (whole ? 1 : 0);
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const int row = r0 + r * 8;
                    if (row >= rows) continue;
                    float *dst = scratch.part + (slot * scratch.rows + row) * p.dim;
#pragma unroll
                    for (int n = 0; n < DP / 8; ++n)
                        if (n * 8 < p.dim) *reinterpret_cast<float2 *>(dst + n * 8 + c0) = make_float2(o[n][2 * r], o[n][2 * r + 1]);
                    if ((lane & 3) == 0) scratch.stat[slot * scratch.rows + row] = make_float2(top[r], sum[r]);
                }
                if (whole && lane == 0) {
                    const int last = static_cast<int>((u - use.at + use.s.stages - 1) / range);
                    scratch.cut[scratch.by_item ? index : worker] = make_int4(worker, last, use.b, use.item);
                }
            }
            fresh = whole = true;
        }
        step(p, use, items, u + 1 < end);
    }
    cp_async_wait<0>();
}

// Joins the parts of the cut items, in the order of the workers.  share_parts (few items): a CTA has one row of an item and its
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
    QMM_CUDA_OK(launch_pdl(decode_kernel<T, DP>, dim3(plan.sms), dim3(Shape<DP>::kWarps * 32), Shape<DP>::kSmem, stream, p, scratch));
    const int64_t indices = scratch.by_item ? plan.items : plan.workers;
    const bool share_parts = indices * plan.rows <= 2 * plan.sms;
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
