// Attention of one new token a sequence over an int8 paged key-value cache (npu_paged_quant_attention).
//
// A key's row is its codes times its scale, a value's likewise, so a score is a sum of query times codes, times the key's scale,
// and the output a sum of weights times the values' scales, times codes; the scales stay in fp32 outside of both products.
//
// Bound by HBM, of which it needs about half of what a 16-bit cache does, so that the instructions on a key count twice as much: at
// the copy rate an SM has 350 clocks for 32 keys and values of 128.  Keys, then dimensions of the values, are the 16 rows of mma.sync and
// query heads its 8 columns: groups of up to 8 heads, the usual ones, need half of the products, sums, registers and exponentials that
// heads as rows would (64 sequences of 500 to 8000 places, 64/8 heads of 128: heads as rows 125 us).
//
// Scores: the codes are the int8 operand as they are.  The query is a whole number of at most 22 bits, in three digits of 8: an
// element is off by 2^-22 of its row's largest at most, and sums of products are exact.
// Values: codes are exact in f16, and their way there is five instructions for four: one turns the signs, two put the bytes below
// 0x64 (f16: 1024 + u), two subtract 1152.  Bytes of two keys that ldmatrix transposes together are rows of even and of odd dimensions,
// so nothing is shuffled; the weights change from rows of keys to rows of heads by movmatrix.
//
// The weights, exp(score - base) * value scale, are multiplied, as they are rounded, by a power of two for each head that keeps the largest so far below
// f16's largest number and above 2^8; it moves with the base, or when a weight would pass that, as the first one above 0 always does.  Rounding a
// weight is half a step of f16, 2^-11 of it, or 2^-33 of the largest one for those far below it.  Beside an output in bf16 (2^-9) that does not show; beside one in f16 it
// would be the larger part, so there a weight is two numbers, the second what the first leaves out: 2^-22 of it (all outputs of 131071 places 2.1e-4 off instead of 3.1e-4, in
// the same time; 32 sequences through a window of 4096, heads of 64, 19.3 -> 20.1 us, of 500 to 8000 places, 128/8 heads, 71.5 -> 77.7).  The sum of the softmax takes them unrounded.  The base
// follows the largest score only when that is 2^3 above it, so that sums are rescaled rarely.
//
// Places that are not seen have no part in a sum: their scores are -inf and their scales 0, whatever their codes are, which are finite.
//
// A CTA has four warps for products and one that copies for them, through a ring of stages: a stage has the keys and values of a tile of
// places for up to four key-value heads, a warp each (fewer heads: a warp a part of the tile's places, added up in shared memory at
// the end of a piece).  So a box of TMA, a look-up of a page and the mask of what is seen serve four warps: by each warp for itself they were 340 of
// 890 instructions on 32 keys (98 us).  The work of a call is the list of all (sequence, heads, tile of places), cut into equal contiguous ranges for
// the CTAs, wherever sequences begin and end.  Of what is cut a CTA leaves its sums in the workspace, and a second kernel adds them in
// their order.  (CTAs that have whole heads of short sequences in turn, without that kernel: one of 200 places 10.0 us, this way 7.8.)  Nothing depends
// on timing, and nothing has to be zero before a call.
//
// Measured (bf16, 64/8 heads of 128, 64 sequences of 500 to 8000 places; 364 MB, 55.6 us at the copy rate): 71.5 us, some 67 of them without the second kernel, and
// 64 for the copies with no products: memory, the start and the joining bound it.  Two CTAs an SM with three stages; three with two
// 94 us, stages of keys and of values of their own 80.  One sequence of 131071 places, 32/8 heads: 52.1 us (0.81 of the copy rate).  Groups of 9
// to 16 heads, two column tiles, wait for loads and results with two stages and three warps a scheduler (32 sequences, 128/8 heads: 72 us, 0.40), pages whose size is no multiple of 8 by
// copies row by row (5 places: 66 us, 28.6 at the copy rate).
#include "paged_decode.cuh"

namespace qmm {
namespace paged {

namespace {

constexpr int kWarps = 4;       // for products; one more copies
constexpr int kThreads = kWarps * 32 + 32;
constexpr int kMostStages = 4;    // of the ring
constexpr int kTileBytes = 4096;  // of a warp's keys, or values, in a stage
constexpr int kDigits = 3;      // of an element of the query, 8 bits each
constexpr int kControlBytes = 256;
constexpr int kSmemOfSm = 228 * 1024;
constexpr float kSlack = 3.0f;  // how far, in powers of two, scores may pass their base before it follows them

// DP: the head dimension rounded up to 64, 128 or 256.  NT: 8 * NT heads are a head tile's, 1 or 2.
template <int DP, int NT>
struct Shape {
    static constexpr int kKeys = kTileBytes / DP;  // of a warp's tile
    // The query in registers, else as operands in shared memory (32 sequences of 500 to 8000 places, 8/4 heads of 256: in registers 54 us, else 46; 128/8 of
    // 128: 117 and 71).
    static constexpr bool kKept = NT == 1 && DP < 256;
    static constexpr int kCtas = NT * DP < 512 ? 2 : 1;  // an SM
    static constexpr int kStage = kWarps * 2 * (kTileBytes + kKeys * 4);    // keys, values, and their scales
    static constexpr int kSums = 8 * NT * DP * 4 + NT * 64;                 // what a warp hands to another
    static constexpr int kOperands = kKept ? 0 : kWarps * 8 * NT * DP * kDigits;
};

// How the work is dealt out: 2^log_heads key-value heads and 2^log_parts parts of a tile's places to the four warps.  A cache comes in boxes of `rows` places of a page (TMA), or where rows is 0, row by row (cp.async).
struct Deal {
    int log_heads, log_parts, rows, stages;
    int scale_vectors;  // four places' scales lie together, at 16-byte boundaries
    uint32_t *status;  // the device status word
};

struct QuantPlan {
    Plan plan;  // workers: CTAs times heads
    Deal deal;
    int ctas;
};

// Groups of up to 8 heads take one column tile.
bool is_narrow(int64_t heads, int64_t kv_heads) { return heads <= 8 * kv_heads; }

QuantPlan make_plan(int64_t batch, int64_t heads, int64_t kv_heads, int64_t dim) {
    QuantPlan q;
    const int64_t group = kv_heads > 0 ? heads / kv_heads : 0;
    const int ctas = is_narrow(heads, kv_heads) ? (dim > 128 ? Shape<256, 1>::kCtas : Shape<128, 1>::kCtas)
                                                : (dim > 128 ? Shape<256, 2>::kCtas : Shape<128, 2>::kCtas);
    Plan &plan = q.plan;
    q.ctas = ctas * sm_count();
    plan.rows = static_cast<int>(group < kRows ? group : kRows);
    plan.tiles = static_cast<int>((group + kRows - 1) / kRows);
    plan.items = batch * kv_heads * plan.tiles;
    q.deal.log_heads = kv_heads % 2 != 0 ? 0 : kv_heads % 4 != 0 ? 1 : 2;
    q.deal.log_parts = 2 - q.deal.log_heads;
    q.deal.rows = q.deal.stages = q.deal.scale_vectors = 0;
    q.deal.status = nullptr;
    plan.workers = q.ctas << q.deal.log_heads;
    plan.cta_parts = static_cast<int64_t>(q.ctas) * kWarps;  // behind those of long pieces, a warp each
    const size_t rows = static_cast<size_t>(plan.cta_parts + 2 * plan.workers) * plan.rows;
    plan.part_bytes = rows * dim * sizeof(float);
    plan.stat_bytes = (rows * sizeof(float2) + 15) / 16 * 16;
    plan.bytes = plan.part_bytes + plan.stat_bytes + static_cast<size_t>(plan.workers) * sizeof(int4);
    return q;
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

// first: the sums begin with these products.
__device__ __forceinline__ void mma_i8(int (&c)[4], const uint32_t (&a)[4], uint2 b, bool first) {
    if (first) {
        asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
            : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b.x), "r"(b.y), "r"(0));
        return;
    }
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

// How many bytes will come, on a barrier: by one lane of a converged warp.
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

// A whole warp's wait: false for all of its lanes if one has given up.
__device__ __forceinline__ bool mbar_wait_whole_warp(uint32_t bar, uint32_t parity, volatile uint32_t *abort_flag, uint32_t where) {
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    return __all_sync(0xffffffffu, mbar_wait_slow(bar, parity, abort_flag, where));
}

// The warps for products alone.
__device__ __forceinline__ void product_warps_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kWarps * 32) : "memory"); }
// The lane's copies by cp.async so far, as one of a barrier's arrivals.
__device__ __forceinline__ void copies_arrive(uint32_t bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}

// What a sequence's token sees, as tiles of 2^log_keys places: those of the sinks, then those of the window.
__device__ __forceinline__ Sequence sequence_of(const Problem &p, int b, int log_keys) {
    const int len = __ldg(p.lens + b), more = (1 << log_keys) - 1;
    const Range r = visible_range(p, len <= 0 ? -1 : len - 1);
    Sequence s;
    s.sink_end = r.sink_end;
    s.lo = r.lo;
    s.hi = r.hi;
    s.sink_tiles = (r.sink_end + more) >> log_keys;
    s.first = max(r.lo >> log_keys, s.sink_tiles);
    s.tiles = s.sink_tiles + max(0, ((r.hi + more) >> log_keys) - s.first);  // (a capacity leaves room for a tile behind it)
    return s;
}

// A CTA's share of the list of all (sequence, item, tile): an item is a head tile of 2^log_heads key-value heads.
struct Share {
    int items, log_keys;
    int64_t end, range;
};

// Steps to the CTA's next piece; false: there is none.
__device__ __forceinline__ bool next_piece(const Problem &p, const Share &share, Piece &piece) {
    piece.at += piece.to - piece.from;
    if (piece.at >= share.end) return false;
    if (++piece.item == share.items) {
        piece.item = 0;
        do {
            piece.s = sequence_of(p, ++piece.b, share.log_keys);
        } while (piece.s.tiles == 0);
    }
    piece.from = 0;
    piece.to = static_cast<int>(min(static_cast<int64_t>(piece.s.tiles), share.end - piece.at));
    return true;
}

// The CTA's share and its first piece; false: it has none.  The warp that is told to writes the rows of sequences that see nothing.
template <typename T>
__device__ __forceinline__ bool first_piece(const Problem &p, const Scratch &scratch, const Deal &deal, int tiles, int log_keys, bool writes, Share &share, Piece &piece) {
    const int lane = threadIdx.x & 31, worker = blockIdx.x, ctas = gridDim.x;
    share.items = (p.kv_heads >> deal.log_heads) * tiles;
    share.log_keys = log_keys;
    int64_t total = 0;
    int last_n = 0;  // tiles of sequence `lane`, of up to 32
    for (int b = lane; b < p.batch; b += 32) {
        last_n = sequence_of(p, b, log_keys).tiles;
        total += last_n;
    }
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    total *= share.items;
    share.range = total < 0x7fffffff ? (static_cast<unsigned>(total) + ctas - 1) / static_cast<unsigned>(ctas) : (total + ctas - 1) / ctas;
    const int64_t begin = min(total, worker * share.range);
    share.end = min(total, begin + share.range);
    int64_t before = 0;
    bool found = false;
    for (int b0 = 0; b0 < p.batch; b0 += 32) {
        const int b = b0 + lane;
        const int n = b < p.batch ? (p.batch <= 32 ? last_n : sequence_of(p, b, log_keys).tiles) : 1;
        if (writes) {
            for (uint32_t none = __ballot_sync(0xffffffffu, n == 0); none != 0; none &= none - 1) {
                const int e = b0 + __ffs(none) - 1;
                if (e % ctas != worker) continue;
                for (int h = 0; h < p.heads; ++h) empty_row<T>(p, e, h);
                if (scratch.by_item)
                    for (int i = lane; i < p.kv_heads * tiles; i += 32) scratch.cut[static_cast<int64_t>(e) * p.kv_heads * tiles + i] = make_int4(-1, 0, 0, 0);
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
        piece.b = b0 + __ffs(past) - 1;
        before += __shfl_sync(0xffffffffu, sum - mine, __ffs(past) - 1);
    }
    if (!found) return false;
    piece.s = sequence_of(p, piece.b, log_keys);
    const int64_t in = begin - before;
    piece.at = begin;
    piece.item = static_cast<int>(in / piece.s.tiles);
    piece.from = static_cast<int>(in - static_cast<int64_t>(piece.item) * piece.s.tiles);
    piece.to = static_cast<int>(min(static_cast<int64_t>(piece.s.tiles), piece.from + share.end - begin));
    return true;
}

// FAR: a warp may have more than kNear places.
template <typename T, int DP, int NT, bool FAR>
__global__ void __launch_bounds__(kThreads, Shape<DP, NT>::kCtas)
quant_decode_kernel(const __grid_constant__ Problem p, const __grid_constant__ QuantScales scales, const __grid_constant__ Scratch scratch,
                    const __grid_constant__ Deal deal, const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map) {
    using S = Shape<DP, NT>;
    constexpr int KEYS = S::kKeys;
    constexpr int kLogKeys = KEYS == 64 ? 6 : KEYS == 32 ? 5 : 4;
    constexpr int kSteps = DP / 16;  // chunks of 16 dimensions, 16 bytes of codes
    constexpr int kTiles = KEYS / 16;  // of 16 keys
    constexpr bool kKept = S::kKept;
    constexpr int kParts = std::is_same<T, __half>::value ? 2 : 1;  // of a weight, in f16
    // A stage's rows are 64 or 128 bytes, 256 columns two of those; chunk ^ key % 8, or where two rows make 128 bytes, chunk ^ key / 2 % 4.
    // Boxes lie one behind the other, in each the rows of one head behind those of another.
    constexpr int kPitch = DP < 128 ? DP : 128, kRowChunks = kPitch / 16, kTurn = DP == 64 ? 1 : 0, kTurns = DP == 64 ? 3 : 7;
    constexpr int kHalf = kWarps * KEYS * kPitch;  // what the first 128 columns of a stage's keys take
    constexpr int kSide = kWarps * kTileBytes;     // the keys of a stage; behind them the values
    constexpr int kMostGroups = kWarps * KEYS / 32;  // of 32 places in a tile
    struct Control {
        uint64_t full[kMostStages], empty[kMostStages];
        uint32_t seen[kMostStages][kMostGroups];  // a bit a place
        uint32_t abort;
    };
    static_assert(sizeof(Control) <= kControlBytes, "the control block's place");
    extern __shared__ __align__(1024) uint8_t smem[];
    const int warp = warp_id_uniform(), lane = threadIdx.x & 31;
    const int heads = 1 << deal.log_heads;  // key-value heads of an item
    const int log_keys = kLogKeys + deal.log_parts, places = 1 << log_keys;  // of a tile
    const int groups = places < 32 ? 1 : places / 32;
    const int box_rows = deal.rows > 0 ? deal.rows : KEYS < 32 ? KEYS : 32;
    // the ring, the stages' scales, sums that warps hand on, operands of the query
    const uint32_t ring = smem_u32(smem), scale_ring = ring + deal.stages * (2 * kSide), sums_at = scale_ring + deal.stages * (kWarps * KEYS * 8);
    const uint32_t operands_at = sums_at + (deal.log_parts > 0 ? heads * S::kSums : 0);
    Control *control = reinterpret_cast<Control *>(smem + (operands_at - ring) + S::kOperands);
    if (threadIdx.x == 0) {
        for (int i = 0; i < deal.stages; ++i) {
            mbar_init(smem_u32(&control->full[i]), 32 + groups);  // the copying warp's lanes, and for 32 places each the bytes of their boxes
            mbar_init(smem_u32(&control->empty[i]), kWarps);
        }
        control->abort = 0;
        mbar_fence_init();
    }
    pdl_launch_dependents();
    pdl_wait();
    __syncthreads();

    const int tiles = (p.group + kRows - 1) / kRows;
    const int row_chunks = p.dim / 16;
    Share share;
    Piece piece;
    bool working = first_piece<T>(p, scratch, deal, tiles, log_keys, warp == 0, share, piece);
    int stage = 0;
    uint32_t phase = 0;
    auto advance = [&] {
        if (++stage == deal.stages) {
            stage = 0;
            phase ^= 1;
        }
    };

    if (warp == kWarps) {
        // ---- copies: of 32 places at a time, looked up one ahead ----
        // A lane's place: the page, if a place of its box is seen, and where it lies there; a bit a lane: whether it is seen.
        int next_place = 0, next_entry = -1;
        uint32_t next_visible = 0;
        auto look_up = [&](int g, int l) {
            const Sequence &s = piece.s;
            const int x = 32 * l + lane, j = ((g < s.sink_tiles ? g : s.first + g - s.sink_tiles) << log_keys) + x;
            const bool there = x < places, visible = there && j < s.hi && (j < s.sink_end || j >= s.lo);
            next_visible = __ballot_sync(0xffffffffu, visible);
            const int page = page_of(p, j), box = j & -box_rows;
            next_place = j - page * p.page;
            next_entry = -1;
            if (visible || (there && deal.rows > 0 && (box < s.sink_end || max(box, s.lo) < min(box + box_rows, s.hi))))
                next_entry = __ldg(p.table + piece.b * p.table_st + page);
        };
        if (working) look_up(piece.from, 0);
        const int chunk = lane % kSteps, vector_head = lane >> 3;
        while (working) {
            const int head0 = piece.item / tiles << deal.log_heads;
            for (int g = piece.from; g < piece.to;) {
                if (!mbar_wait_whole_warp(smem_u32(&control->empty[stage]), phase ^ 1, &control->abort, 0xa0)) {
                    working = false;
                    break;
                }
                const uint32_t full = smem_u32(&control->full[stage]);
#pragma unroll 1
                for (int l = 0; l < groups; ++l) {
                    const int entry = next_entry, place = next_place;
                    const uint32_t boxes = __ballot_sync(0xffffffffu, entry >= 0 && entry < p.pages), seen = boxes & next_visible;
                    // the next 32 places
                    const bool last = l + 1 == groups;
                    if (!last) {
                        look_up(g, l + 1);
                    } else if (++g < piece.to) {
                        look_up(g, 0);
                    } else {
                        working = next_piece(p, share, piece);
                        if (working) {
                            look_up(piece.from, 0);
                        }
                        g = 0x7fffffff;
                    }
                    if (lane == 0) control->seen[stage][l] = seen;
                    __syncwarp();
                    const uint32_t dst = ring + stage * (2 * kSide), x0 = 32 * l;
                    if (deal.rows > 0) {
                        expect_bytes_warp(full, __popc(boxes) * (2 * DP << deal.log_heads));
                        // boxes of which a place is seen come whole
#pragma unroll 1
                        for (int key = 0; key < 32; key += box_rows) {
                            if (!(boxes >> key & 1)) continue;
                            const int page = __shfl_sync(0xffffffffu, entry, key), at = __shfl_sync(0xffffffffu, place, key);
                            const uint32_t to = dst + ((x0 + key) << deal.log_heads) * kPitch;
#pragma unroll
                            for (int c = 0; c < DP / kPitch; ++c) {
                                tma_load_4d_warp(to + c * kHalf, &k_map, c * kPitch, at, head0, page, full);
                                tma_load_4d_warp(to + kSide + c * kHalf, &v_map, c * kPitch, at, head0, page, full);
                            }
                        }
                    } else {
                        expect_bytes_warp(full, 0);
                        // a lane has the same chunk of rows 32 / kSteps apart
                        const bool ok = boxes >> lane & 1;
                        const int64_t k_at = ok ? entry * p.k_sb + place * p.k_st + head0 * p.k_sh : 0, v_at = ok ? entry * p.v_sb + place * p.v_st + head0 * p.v_sh : 0;
                        const uint32_t column = dst + chunk / kRowChunks * kHalf;
#pragma unroll 1
                        for (int key0 = 0; key0 < min(32, places); key0 += 32 / kSteps) {
                            const int key = key0 + lane / kSteps;
                            const int8_t *k = static_cast<const int8_t *>(p.k) + __shfl_sync(0xffffffffu, k_at, key) + chunk * 16;
                            const int8_t *v = static_cast<const int8_t *>(p.v) + __shfl_sync(0xffffffffu, v_at, key) + chunk * 16;
                            if (chunk >= row_chunks || !(boxes >> key & 1)) continue;
                            const int x = x0 + key;
                            uint32_t to = column + (x / box_rows * heads * box_rows + x % box_rows) * kPitch + (((chunk ^ (key >> kTurn)) & kTurns) << 4);
                            for (int h = 0; h < heads; ++h) {
                                cp_async_16(to, k, 16);
                                cp_async_16(to + kSide, v, 16);
                                to += box_rows * kPitch;
                                k += p.k_sh;
                                v += p.v_sh;
                            }
                        }
                    }
                    const uint32_t scales_to = scale_ring + stage * (kWarps * KEYS * 8) + x0 * 4;
                    if (seen == 0xffffffffu && deal.scale_vectors) {
                        // four places a vector: lane 8 h + c has places 4 c ... + 3 of head h
                        const int page = __shfl_sync(0xffffffffu, entry, (lane & 7) * 4), at = __shfl_sync(0xffffffffu, place, (lane & 7) * 4);
                        if (vector_head < heads) {
                            const uint32_t to = scales_to + (vector_head << log_keys) * 4 + (lane & 7) * 16;
                            cp_async_16(to, scales.k + page * scales.k_sb + at + (head0 + vector_head) * scales.k_sh, 16);
                            cp_async_16(to + kWarps * KEYS * 4, scales.v + page * scales.v_sb + at + (head0 + vector_head) * scales.v_sh, 16);
                        }
                    } else if (x0 + lane < places) {
                        const bool ok = seen >> lane & 1;
                        const float *k = scales.k + (ok ? entry * scales.k_sb + place * scales.k_st + head0 * scales.k_sh : 0);
                        const float *v = scales.v + (ok ? entry * scales.v_sb + place * scales.v_st + head0 * scales.v_sh : 0);
#pragma unroll 1
                        for (int h = 0; h < heads; ++h) {
                            const uint32_t to = scales_to + ((h << log_keys) + lane) * 4;
                            cp_async_4(to, k, ok ? 4 : 0);
                            cp_async_4(to + kWarps * KEYS * 4, v, ok ? 4 : 0);
                            if (ok) {
                                k += scales.k_sh;
                                v += scales.v_sh;
                            }
                        }
                    }
                }
                copies_arrive(full);
                advance();
            }
        }
    } else {
        // ---- products ----
        const int head = warp & (heads - 1), part = warp >> deal.log_heads;  // of the item's heads, of a tile's places
        const uint32_t operands = operands_at + warp * (S::kOperands / kWarps);
        // The running maximum is one of unscaled scores, which takes a positive scale: a negative one's sign goes to the query, and
        // for a scale of 0 the query is 0.
        const float factor = p.scale * kLog2e;
        const float scale = factor == 0.0f ? 1.0f : fabsf(factor), sign = factor == 0.0f ? 0.0f : factor < 0.0f ? -1.0f : 1.0f;
        // the index of the CTA's head among all, for the parts and the cut items
        const int64_t worker = static_cast<int64_t>(head) * gridDim.x + blockIdx.x;
        if (!scratch.by_item && part == 0 && lane == 0) scratch.cut[worker] = make_int4(-1, 0, 0, 0);

        // A lane's place in an operand: row (or column) lane / 4, elements 2 * (lane % 4) and the next.  Of a product's sums it has rows
        // lane / 4 and 8 more, columns c0 and c0 + 1.
        const int r0 = lane >> 2, c0 = (lane & 3) * 2;
        uint2 q[kKept ? NT : 1][kKept ? kSteps / 2 : 1][kDigits];
        float row_scale[NT][2];
        // The query's heads as second operands, a lane has dimensions 16 ks + 4 (lane % 4) ... + 3 of a head: whole numbers below 2^22, as three
        // digits from -128 to 127.
        auto take_query = [&](int kvh, int head_tile, int rows) {
#pragma unroll
            for (int t = NT - 1; t >= 0; --t) {
                uint2 x[kSteps];
                const int row = 8 * t + r0;
                const T *src = static_cast<const T *>(p.q) + piece.b * p.q_st + (static_cast<int64_t>(kvh) * p.group + head_tile * kRows + row) * p.q_sh + (lane & 3) * 4;
#pragma unroll
                for (int ks = 0; ks < kSteps; ++ks) {
                    x[ks] = make_uint2(0, 0);
                    if (row < rows && ks < row_chunks) x[ks] = __ldg(reinterpret_cast<const uint2 *>(src + ks * 16));
                }
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
                            store_shared_uint2(operands + (((t * (kSteps / 2) + ks / 2) * kDigits + d) * 32 + lane) * 8, make_uint2(digits[d][0], digits[d][1]));
                    }
                }
                if (!kKept) __syncwarp();
            }
        };
        auto query_part = [&](int t, int ks, int d) {
            return kKept ? q[kKept ? t : 0][kKept ? ks / 2 : 0][d] : load_shared_uint2(operands + (((t * (kSteps / 2) + ks / 2) * kDigits + d) * 32 + lane) * 8);
        };
        // ldmatrix addresses of a tile, keys and values alike: 8 keys x 16 bytes a matrix, four of them; of 16 keys, two chunks
        constexpr int kAtOnce = KEYS == 16 ? 2 : 1;  // chunks of an ldmatrix
        const int lane_key = KEYS == 16 ? (lane >> 3 & 1) * 8 + (lane & 7) : lane, lane_place = part * KEYS + lane_key;
        const uint32_t lane_tile = ((lane_place / box_rows * heads + head) * box_rows + lane_place % box_rows) * kPitch +
                                   (((KEYS == 16 ? lane >> 4 : 0) ^ ((lane_key >> kTurn) & kTurns)) << 4);
        const uint32_t lane_scale = scale_ring + ((head << log_keys) + part * KEYS + r0) * 4;
        auto chunk_of = [&](uint32_t tile, int ks) { return (tile ^ ((ks % kRowChunks) << 4)) + ks / kRowChunks * kHalf; };
        auto release = [&] {
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&control->empty[stage]));
            advance();
        };
        bool ok = true;  // a warp that has given up takes no more tiles, but its part in the exchange of sums
        while (working) {
            float o[kSteps][NT][4];  // dimensions 16 ks + 2 r0 (and the next: + 2) of heads c0, c0 + 1 (+ 1)
#pragma unroll
            for (int n = 0; n < kSteps; ++n) {
#pragma unroll
                for (int t = 0; t < NT; ++t) o[n][t][0] = o[n][t][1] = o[n][t][2] = o[n][t][3] = 0.0f;
            }
            // top: what scores are relative to, within kSlack below the largest; ceiling: a score beyond it moves that; base: top times the row's
            // scale; lift: the power of two of a head's weights; big: the lane's largest, not lifted
            // sum: of the lane's weights; lost: what its additions rounded away, to be taken off (Kahan's summation: a chain of 65536 equal
            // weights is off by up to 2^-10 without)
            float top[NT][2], ceiling[NT][2], base[NT][2], sum[NT][2], lost[NT][2], lift[NT][2], big[NT][2];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    top[t][i] = ceiling[t][i] = -INFINITY;
                    sum[t][i] = lost[t][i] = big[t][i] = base[t][i] = 0.0f;
                    lift[t][i] = 1.0f;
                }
            }
            const int group0 = piece.item / tiles, head_tile = piece.item - group0 * tiles, kvh = (group0 << deal.log_heads) + head;
            const int rows = min(kRows, p.group - head_tile * kRows);
            // A long piece adds what it has to the warp's fp32 sums in the workspace and begins again from 0 (back: the other way round).
            auto put_by = [&](bool first, bool back) {
                const int64_t part0 = (static_cast<int64_t>(blockIdx.x) * kWarps + warp) * scratch.rows;
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
            take_query(kvh, head_tile, rows);
            for (int g = piece.from; g < piece.to; ++g) {
                if (FAR && g != piece.from && (g - piece.from) % (kRun / KEYS) == 0) put_by(g - piece.from == kRun / KEYS, false);
                ok = ok && mbar_wait_whole_warp(smem_u32(&control->full[stage]), phase, &control->abort, 0xa1);
                if (!ok) break;
                uint32_t tile = ring + stage * (2 * kSide) + lane_tile, scale_at = lane_scale + stage * (kWarps * KEYS * 8);
                constexpr int kLooks = KEYS > 32 ? KEYS / 32 : 1;
                uint32_t seen[kLooks];
                bool all_seen = true;
#pragma unroll
                for (int l = 0; l < kLooks; ++l) {
                    seen[l] = KEYS == 16 ? control->seen[stage][part / 2] >> 16 * (part % 2) & 0xffffu : control->seen[stage][part * kLooks + l];
                    all_seen = all_seen && seen[l] == (KEYS == 16 ? 0xffffu : 0xffffffffu);
                }
                // scores: keys 16 m + r0 (and + 8: + 2) of heads c0, c0 + 1 (+ 1)
                int sums[kDigits][kTiles][NT][4];
#pragma unroll
                for (int ks = 0; ks < kSteps; ks += 2) {
                    if (kSteps > 8 && ks % 4 == 0 && ks >= row_chunks) break;  // (chunks behind the dimensions meet a query of 0)
#pragma unroll
                    for (int n = 0; n < kTiles; n += 2) {
                        uint32_t w[2][4];  // 16 keys: two chunks of them; else a chunk of 32 keys each
                        ldmatrix_x4(w[0], chunk_of(tile, ks) + n * (16 * kPitch) * heads);
                        if (kTiles > 1) ldmatrix_x4(w[1], chunk_of(tile, ks + 1) + n * (16 * kPitch) * heads);
#pragma unroll
                        for (int i = 0; i < (kTiles > 1 ? 2 : 1); ++i) {
                            const uint32_t a[4] = {w[0][2 * i], w[0][2 * i + 1], kTiles > 1 ? w[1][2 * i] : w[0][2], kTiles > 1 ? w[1][2 * i + 1] : w[0][3]};
#pragma unroll
                            for (int t = 0; t < NT; ++t) {
#pragma unroll
                                for (int d = 0; d < kDigits; ++d) mma_i8(sums[d][n + i][t], a, query_part(t, ks, d), ks == 0);
                            }
                        }
                    }
                }
                float s[kTiles][NT][4];
#pragma unroll
                for (int m = 0; m < kTiles; ++m) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float by = load_shared_float(scale_at + (16 * m + 8 * h) * 4);
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
                                lost[t][i] *= keep[t][i];
                                big[t][i] *= keep[t][i];
                            }
                        }
                    }
                }
#pragma unroll
                for (int t = 0; t < NT; ++t) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        float all = -lost[t][i];
#pragma unroll
                        for (int m = 0; m < kTiles; ++m) {
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                float &x = s[m][t][2 * h + i];
                                x = exp2_fast(fmaf(x, row_scale[t][i], -base[t][i]));
                                all += x;
                            }
                        }
                        const float more = sum[t][i] + all;
                        lost[t][i] = (more - sum[t][i]) - all;
                        sum[t][i] = more;
                    }
                }
                tile += kSide;
                scale_at += kWarps * KEYS * 4;
#pragma unroll
                for (int m = 0; m < kTiles; ++m) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float by = load_shared_float(scale_at + (16 * m + 8 * h) * 4);
#pragma unroll
                        for (int t = 0; t < NT; ++t) {
#pragma unroll
                            for (int i = 0; i < 2; ++i) {
                                float &x = s[m][t][2 * h + i];
                                x *= by;
                                big[t][i] = fmaxf(big[t][i], fabsf(x));
                            }
                        }
                    }
                }
                float largest = 0.0f;
#pragma unroll
                for (int t = 0; t < NT; ++t) largest = fmaxf(largest, fmaxf(big[t][0] * lift[t][0], big[t][1] * lift[t][1]));
                if (__builtin_expect(moves || __any_sync(0xffffffffu, largest > 60000.0f), 0)) {
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            float most = big[t][i];
                            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 4));
                            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 8));
                            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 16));
                            big[t][i] = most;
                            const float lifted = most * lift[t][i];
                            if (lifted > 60000.0f || (lifted < 256.0f && most > 0.0f)) {
                                // to [2^11, 2^12), as far as lift and its step stay finite; sums that a step below 2^-126 leaves count no more
                                const int has = static_cast<int>(__float_as_uint(lift[t][i]) >> 23) - 127;
                                const int e = max(-126, min(min(138 - static_cast<int>(__float_as_uint(most) >> 23), 127), 127 + has));
                                lift[t][i] = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
                                keep[t][i] *= e - has < -126 ? 0.0f : __uint_as_float(static_cast<uint32_t>(127 + e - has) << 23);
                            } else if (most == 0.0f) {
                                // none above 0: the first one passes 60000 and comes here; the sums are 0, or below what fp32 has beside the new base
                                lift[t][i] = 0x1p127f;
                                keep[t][i] = 0.0f;
                            }
#pragma unroll
                            for (int n = 0; n < kSteps; ++n) {
                                o[n][t][i] *= keep[t][i];
                                o[n][t][i + 2] *= keep[t][i];
                            }
                        }
                    }
                }
                uint32_t b[kParts][NT][kTiles][2];
#pragma unroll
                for (int t = 0; t < NT; ++t) {
#pragma unroll
                    for (int m = 0; m < kTiles; ++m) {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const float x = s[m][t][2 * h] * lift[t][0], y = s[m][t][2 * h + 1] * lift[t][1];
                            const uint32_t both = pack2<__half>(x, y);
                            b[0][t][m][h] = transposed(both);
                            if constexpr (kParts == 2) {
                                const float2 first = two_floats<__half>(both);
                                // (of an infinite one the rest is NaN, and counts as 32)
                                b[1][t][m][h] = transposed(pack2<__half>(fminf(x - first.x, 32.0f), fminf(y - first.y, 32.0f)));
                            }
                        }
                    }
                }
#pragma unroll
                for (int ks = 0; ks < kSteps; ks += kAtOnce) {
                    if (kSteps > 8 && ks % 4 == 0 && ks >= row_chunks) break;
#pragma unroll
                    for (int n = 0; n < kTiles * kAtOnce; n += 2) {
                        uint32_t w[4];
                        ldmatrix_x4_trans(w, chunk_of(tile, ks) + n * (16 * kPitch) * heads);
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const uint32_t x = w[2 * i] ^ 0x80808080u, y = w[2 * i + 1] ^ 0x80808080u;
                            const uint32_t a[4] = {codes_f16<0x4240>(x), codes_f16<0x4341>(x), codes_f16<0x4240>(y), codes_f16<0x4341>(y)};
#pragma unroll
                            for (int t = 0; t < NT; ++t) {
#pragma unroll
                                for (int part = 0; part < kParts; ++part)
                                    mma_16816<__half>(o[ks + (n + i) / kTiles][t], a, b[part][t][(n + i) % kTiles][0], b[part][t][(n + i) % kTiles][1]);
                            }
                        }
                    }
                }
                release();
            }
            if (FAR && piece.to - piece.from > kRun / KEYS) put_by(false, true);

            // ---- the piece's end: rows to the outputs, or sums to the workspace ----
            float all[NT][2], most[NT][2];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    all[t][i] = sum[t][i] - lost[t][i];
                    all[t][i] += __shfl_xor_sync(0xffffffffu, all[t][i], 4);
                    all[t][i] += __shfl_xor_sync(0xffffffffu, all[t][i], 8);
                    all[t][i] += __shfl_xor_sync(0xffffffffu, all[t][i], 16);
                    most[t][i] = top[t][i] * row_scale[t][i];
                    const float down = 1.0f / lift[t][i];
#pragma unroll
                    for (int n = 0; n < kSteps; ++n) {
                        o[n][t][i] *= down;
                        o[n][t][i + 2] *= down;
                    }
                }
            }
            // the parts of a tile's places, the last one to the one before it and so on
            for (int from = (1 << deal.log_parts) - 1; from > 0; --from) {
                float *sums = reinterpret_cast<float *>(smem + (sums_at - ring) + head * S::kSums) + lane;
                float *stats = sums - lane + kSteps * NT * 128 + (lane & 3);  // the same for all lanes of a column
                if (part == from) {
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
#pragma unroll
                        for (int n = 0; n < kSteps; ++n) {
#pragma unroll
                            for (int i = 0; i < 4; ++i) sums[((n * NT + t) * 4 + i) * 32] = o[n][t][i];
                        }
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            stats[(t * 4 + i) * 4] = all[t][i];
                            stats[(t * 4 + i + 2) * 4] = most[t][i];
                        }
                    }
                }
                product_warps_sync();
                if (part == from - 1) {
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const float other = stats[(t * 4 + i + 2) * 4], now = fmaxf(most[t][i], other), to = now == -INFINITY ? 0.0f : now;
                            const float keep = exp2_fast(most[t][i] - to), add = exp2_fast(other - to);
                            all[t][i] = fmaf(stats[(t * 4 + i) * 4], add, all[t][i] * keep);
                            most[t][i] = now;
#pragma unroll
                            for (int n = 0; n < kSteps; ++n) {
                                o[n][t][i] = fmaf(sums[((n * NT + t) * 4 + i) * 32], add, o[n][t][i] * keep);
                                o[n][t][i + 2] = fmaf(sums[((n * NT + t) * 4 + i + 2) * 32], add, o[n][t][i + 2] * keep);
                            }
                        }
                    }
                }
                product_warps_sync();
            }
            const bool begins = piece.from == 0, ends = piece.to == piece.s.tiles;
            if (part == 0) {
                const int64_t row0 = static_cast<int64_t>(piece.b) * p.heads + kvh * p.group + head_tile * kRows;
                const int64_t part0 = (scratch.cta_parts + worker * 2 + begins) * scratch.rows;
#pragma unroll
                for (int t = 0; t < NT; ++t) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int row = 8 * t + c0 + i;
                        if (row >= rows) continue;
                        if (begins && ends) {
                            const float inv = all[t][i] == 0.0f ? 0.0f : 1.0f / all[t][i];
                            T *dst = static_cast<T *>(p.out) + (row0 + row) * p.dim + 2 * r0;
#pragma unroll
                            for (int n = 0; n < kSteps; ++n)
                                if (n < row_chunks) *reinterpret_cast<uint32_t *>(dst + n * 16) = pack2<T>(o[n][t][i] * inv, o[n][t][i + 2] * inv);
                            if (r0 == 0) p.lse[row0 + row] = all[t][i] == 0.0f ? -INFINITY : most[t][i] * kLn2 + logf(all[t][i]);
                        } else {
                            float *dst = scratch.part + (part0 + row) * p.dim + 2 * r0;
#pragma unroll
                            for (int n = 0; n < kSteps; ++n)
                                if (n < row_chunks) *reinterpret_cast<float2 *>(dst + n * 16) = make_float2(o[n][t][i], o[n][t][i + 2]);
                            if (r0 == 0) scratch.stat[part0 + row] = make_float2(most[t][i], all[t][i]);
                        }
                    }
                }
                if (lane == 0 && begins && (!ends || scratch.by_item)) {
                    const int item = kvh * tiles + head_tile;
                    const int64_t last = (piece.at - piece.from + piece.s.tiles - 1) / share.range;  // the CTA that has the item's last tile
                    scratch.cut[scratch.by_item ? static_cast<int64_t>(piece.b) * p.kv_heads * tiles + item : worker] =
                        ends ? make_int4(-1, 0, 0, 0)
                             : make_int4(static_cast<int>(worker), static_cast<int>(static_cast<int64_t>(head) * gridDim.x + last), piece.b, item);
                }
            }
            working = next_piece(p, share, piece);
        }
    }
    __syncthreads();
    if (control->abort != 0) {
        // what is still on its way comes before the CTA's shared memory goes
        uint32_t late = 0;
        for (int i = 0; warp == kWarps && i < deal.stages; ++i) mbar_wait(smem_u32(&control->full[i]), i < stage ? phase : phase ^ 1, &late, 0xa2);
        if (threadIdx.x == 0 && deal.status != nullptr) atomicMax(deal.status, control->abort);
    }
}

// Adds the parts of the head tiles that are cut, in the order of the CTAs: SHARE warps a row.  Statistics and sums of kAtOnce parts are under way
// together.  DP: 128 or 256.
template <int SHARE>
constexpr int kJoinWarps = SHARE < 8 ? 8 : SHARE;  // of a CTA
template <typename T, int DP, int SHARE>
__global__ void __launch_bounds__(kJoinWarps<SHARE> * 32, SHARE == 8 ? 2 : 1)
quant_join_kernel(const __grid_constant__ Problem p, const __grid_constant__ Scratch scratch, int64_t indices) {
    constexpr int kRowsOfCta = kJoinWarps<SHARE> / SHARE, kAtOnce = 1024 / DP;
    __shared__ __align__(16) float s_sums[SHARE > 1 ? kRowsOfCta : 1][SHARE][DP];
    __shared__ float2 s_stats[kRowsOfCta][SHARE];
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31, here = warp_id_uniform() / SHARE, warp = warp_id_uniform() % SHARE;
    const int64_t at = static_cast<int64_t>(blockIdx.x) * kRowsOfCta + here, index = at / scratch.rows;
    const int row = static_cast<int>(at - index * scratch.rows);
    if (index >= indices) return;
    const int4 cut = scratch.cut[index];
    if (cut.x < 0) return;
    const int tiles = (p.group + kRows - 1) / kRows;
    const int kvh = cut.w / tiles, tile = cut.w - kvh * tiles;
    if (row >= min(kRows, p.group - tile * kRows)) return;
    const int parts = cut.y - cut.x + 1;
    const int from = parts * warp / SHARE, to = parts * (warp + 1) / SHARE;
    auto place = [&](int i) { return (scratch.cta_parts + static_cast<int64_t>(cut.x + i) * 2 + (i == 0)) * scratch.rows + row; };
    float top = -INFINITY, sum = 0.0f, acc[8] = {};
    for (int i0 = from; i0 < to; i0 += kAtOnce) {
        float2 stat[kAtOnce];
        float4 v[kAtOnce][2];
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            stat[i] = make_float2(-INFINITY, 0.0f);
            v[i][0] = v[i][1] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (i0 + i >= to) continue;
            stat[i] = __ldcg(scratch.stat + place(i0 + i));
            const float *src = scratch.part + place(i0 + i) * p.dim + lane * 4;
#pragma unroll
            for (int c = 0; c < DP / 128; ++c)
                if (c * 128 + lane * 4 < p.dim) v[i][c] = __ldcg(reinterpret_cast<const float4 *>(src + c * 128));
        }
        float now = top;
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) now = fmaxf(now, stat[i].x);
        const float base = now == -INFINITY ? 0.0f : now, keep = exp2_fast(top - base);
        sum *= keep;
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j] *= keep;
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            const float w = exp2_fast(stat[i].x - base);
            sum = fmaf(stat[i].y, w, sum);
#pragma unroll
            for (int c = 0; c < DP / 128; ++c) {
                acc[4 * c] = fmaf(v[i][c].x, w, acc[4 * c]);
                acc[4 * c + 1] = fmaf(v[i][c].y, w, acc[4 * c + 1]);
                acc[4 * c + 2] = fmaf(v[i][c].z, w, acc[4 * c + 2]);
                acc[4 * c + 3] = fmaf(v[i][c].w, w, acc[4 * c + 3]);
            }
        }
        top = now;
    }
    if (SHARE > 1) {
        auto &s_sum = s_sums[here];
        auto &s_stat = s_stats[here];
#pragma unroll
        for (int c = 0; c < DP / 128; ++c)
            *reinterpret_cast<float4 *>(&s_sum[warp][c * 128 + lane * 4]) = make_float4(acc[4 * c], acc[4 * c + 1], acc[4 * c + 2], acc[4 * c + 3]);
        if (lane == 0) s_stat[warp] = make_float2(top, sum);
        asm volatile("bar.sync %0, %1;" ::"r"(here + 1), "n"(SHARE * 32) : "memory");  // the row's warps
        if (warp != 0) return;
        for (int w = 0; w < SHARE; ++w) top = fmaxf(top, s_stat[w].x);
        const float all = top == -INFINITY ? 0.0f : top;
        sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] = 0.0f;
        for (int w = 0; w < SHARE; ++w) {
            const float weight = exp2_fast(s_stat[w].x - all);
            sum = fmaf(s_stat[w].y, weight, sum);
#pragma unroll
            for (int i = 0; i < DP / 32; ++i) acc[i] = fmaf(s_sum[w][(i >> 2) * 128 + lane * 4 + (i & 3)], weight, acc[i]);
        }
    }
    const int64_t out = static_cast<int64_t>(cut.z) * p.heads + kvh * p.group + tile * kRows + row;
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    T *dst = static_cast<T *>(p.out) + out * p.dim;
#pragma unroll
    for (int c = 0; c < DP / 128; ++c) {
        const int d = c * 128 + lane * 4;
        if (d < p.dim)
            *reinterpret_cast<uint2 *>(dst + d) = make_uint2(pack2<T>(acc[4 * c] * inv, acc[4 * c + 1] * inv), pack2<T>(acc[4 * c + 2] * inv, acc[4 * c + 3] * inv));
    }
    if (lane == 0) p.lse[out] = sum == 0.0f ? -INFINITY : top * kLn2 + logf(sum);
}

// A cache as TMA sees it: boxes of `rows` places of one page and `heads` heads by up to 128 columns (zeros behind the head dimension).  False: its
// strides are none that TMA takes.
bool cache_map(CUtensorMap *map, const Problem &p, const void *base, int64_t sb, int64_t st, int64_t sh, int heads, int rows, int columns) {
    const int64_t sizes[4] = {p.dim, p.page, p.kv_heads, p.pages};
    int64_t strides[3] = {st, sh, sb};
    for (int i = 0; i < 3; ++i) {
        if (sizes[i + 1] == 1) strides[i] = p.dim;  // takes no step
        if (strides[i] <= 0 || strides[i] >= 1ll << 39) return false;
    }
    const int box[4] = {columns, rows, heads, 1};
    return make_tmap_4d(map, base, 1, sizes, strides, box, columns);
}

bool scale_vectors(const float *base, int64_t sb, int64_t st, int64_t sh) {
    return (reinterpret_cast<uintptr_t>(base) & 15) == 0 && st == 1 && ((sb | sh) & 3) == 0;
}

template <typename T, int DP, int NT, bool FAR>
int launch_decode_kernel(const Problem &p, const QuantScales &scales, const QuantPlan &plan, const Scratch &scratch, cudaStream_t stream) {
    using S = Shape<DP, NT>;
    CUtensorMap k_map = {}, v_map = {};
    Deal deal = plan.deal;
    deal.status = device_status_word();
    // as many places a box as begin together in any page and any warp's tile
    deal.rows = 8;
    while (2 * deal.rows <= S::kKeys && deal.rows < 32 && p.page % (2 * deal.rows) == 0) deal.rows *= 2;
    deal.scale_vectors = p.page % 4 == 0 && scale_vectors(scales.k, scales.k_sb, scales.k_st, scales.k_sh) && scale_vectors(scales.v, scales.v_sb, scales.v_st, scales.v_sh);
    constexpr int kColumns = DP < 128 ? DP : 128;
    const int heads = 1 << deal.log_heads;
    if (p.page % 8 != 0 || p.pages == 0 || !cache_map(&k_map, p, p.k, p.k_sb, p.k_st, p.k_sh, heads, deal.rows, kColumns) ||
        !cache_map(&v_map, p, p.v, p.v_sb, p.v_st, p.v_sh, heads, deal.rows, kColumns))
        deal.rows = 0;
    // as many stages as fit.  The kernel's limit is one for all calls, whatever each takes of it: threads that call at the same time set it to the same.
    constexpr int kMostSmem = kSmemOfSm / S::kCtas - 1024;
    const int fixed = (deal.log_parts > 0 ? heads * S::kSums : 0) + S::kOperands + kControlBytes;
    deal.stages = std::min(kMostStages, (kMostSmem - fixed) / S::kStage);
    const int smem = fixed + deal.stages * S::kStage;
    QMM_CUDA_OK(cudaFuncSetAttribute(quant_decode_kernel<T, DP, NT, FAR>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostSmem));
    QMM_CUDA_OK(launch_pdl(quant_decode_kernel<T, DP, NT, FAR>, dim3(plan.ctas), dim3(kThreads), smem, stream, p, scales, scratch, deal, k_map, v_map));
    return QMM_OK;
}

template <typename T, int DP, int NT>
int launch(const Problem &p, const QuantScales &scales, const QuantPlan &plan, const Scratch &scratch, cudaStream_t stream) {
    // what a warp may have: of one head tile's places its part, of all of them an equal share
    const int64_t seen = (p.window > 0 ? std::min<int64_t>(p.capacity, static_cast<int64_t>(p.window) + p.sinks) : p.capacity) >> plan.deal.log_parts;
    const int64_t items = plan.plan.items >> plan.deal.log_heads;
    const bool far = seen > kNear && seen > kNear * plan.ctas / items;
    const int rc = far ? launch_decode_kernel<T, DP, NT, true>(p, scales, plan, scratch, stream) : launch_decode_kernel<T, DP, NT, false>(p, scales, plan, scratch, stream);
    if (rc != QMM_OK) return rc;
    constexpr int kDims = DP < 256 ? 128 : 256;
    const int64_t indices = scratch.by_item ? plan.plan.items : plan.plan.workers, all = indices * scratch.rows;
    auto join = [&](auto kern, int warps, int share) {
        const int of_cta = warps / share;
        return launch_pdl(kern, dim3(static_cast<unsigned>((all + of_cta - 1) / of_cta)), dim3(warps * 32), 0, stream, p, scratch, indices);
    };
    // Few rows have many parts each (us, by 8, 2 and 1 warps a row: 256 rows of 4 sequences of 500 to 8000 places 14.2, -, 24.6; 1024 rows, window of 4096, heads of 64, 23.4,
    // 19.2, 20.5; 8192 rows of 128 sequences 44.2, 24.1, 19.3), a single sequence up to one of each CTA (131071 places, 148 parts: 16 warps 51.3, 8 52.3; 200 places 7.9, 7.7).
    const int64_t parts = std::min<int64_t>(plan.plan.workers / plan.plan.items, seen / Shape<DP, NT>::kKeys);
    if (all <= 2 * sm_count() && parts > 64)
        QMM_CUDA_OK(join(quant_join_kernel<T, kDims, 16>, 16, 16));
    else if (all <= 2 * sm_count())
        QMM_CUDA_OK(join(quant_join_kernel<T, kDims, 8>, 8, 8));
    else if (all <= 8 * sm_count())
        QMM_CUDA_OK(join(quant_join_kernel<T, kDims, 2>, 8, 2));
    else
        QMM_CUDA_OK(join(quant_join_kernel<T, kDims, 1>, 8, 1));
    return QMM_OK;
}

template <typename T, int NT>
int launch_dim(const Problem &p, const QuantScales &scales, const QuantPlan &plan, const Scratch &scratch, cudaStream_t stream) {
    if (p.dim <= 64) return launch<T, 64, NT>(p, scales, plan, scratch, stream);
    if (p.dim <= 128) return launch<T, 128, NT>(p, scales, plan, scratch, stream);
    return launch<T, 256, NT>(p, scales, plan, scratch, stream);
}

template <typename T>
int launch_t(const Problem &p, const QuantScales &scales, const QuantPlan &plan, const Scratch &scratch, cudaStream_t stream) {
    return is_narrow(p.heads, p.kv_heads) ? launch_dim<T, 1>(p, scales, plan, scratch, stream) : launch_dim<T, 2>(p, scales, plan, scratch, stream);
}

}  // namespace

size_t quant_decode_workspace(int64_t batch, int64_t heads, int64_t kv_heads, int64_t dim) {
    return batch == 0 || heads == 0 ? 0 : make_plan(batch, heads, kv_heads, dim).plan.bytes;
}

int launch_quant_decode(const Problem &p, const QuantScales &scales, int dtype, void *workspace, size_t workspace_bytes, cudaStream_t stream) {
    const QuantPlan plan = make_plan(p.batch, p.heads, p.kv_heads, p.dim);
    if (workspace_bytes < plan.plan.bytes || workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 15) != 0)
        return fail(QMM_ERR_WORKSPACE, "qmm_paged_quant_attention: needs a workspace of " + std::to_string(plan.plan.bytes) + " bytes, 16-byte aligned");
    const Scratch scratch = lay_out(plan.plan, workspace);
    return dtype == QMM_DTYPE_BF16 ? launch_t<__nv_bfloat16>(p, scales, plan, scratch, stream) : launch_t<__half>(p, scales, plan, scratch, stream);
}

}  // namespace paged
}  // namespace qmm
