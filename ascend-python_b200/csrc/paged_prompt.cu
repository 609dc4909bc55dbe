// Attention of the last tokens of each sequence over a paged key-value cache (npu_paged_prompt_attention).
//
// Rows: the tokens of one sequence times the query heads of one key-value head, token by token, in tiles of 128; so a few tokens
// of a wide group fill a tile as well as many of a narrow one, and every key that is read serves the whole group.
//
// For 64 keys at a time, S = Q K^T and O += P V are tcgen05 products with accumulators in tensor memory, and P, rounded to the
// values' type, is the second product's operand in tensor memory.  The softmax is one pass: a thread has a row, its running base
// (a maximum) and sum.  The base moves, and O is rescaled, only when a row's maximum has grown by more than 2^8 (f16: 2^4) since;
// until then the weights are that much larger and as exact.
//
// A CTA goes on to a further block of the grid, as long as there are blocks that have not begun (cluster launch control), so the
// hardware's order of the blocks balances the work as it does without; the next item's keys, values and query are fetched, and
// its first S made, while the softmax ends the present one.  (A CTA an item cost 7 us for each.)
//
// An item of one row tile, as a few drafted tokens are, gives both halves of the CTA its rows, every second 64 keys each; their O
// and sums are added at the end.
//
// The softmax has its scores in registers and gives S back at once: the next Q K^T runs beside it, and so does P V of the step
// before, for P has two places of its own.  Two row tiles share the keys (dimensions up to 128), and take turns at the
// exponentials.  What bounds a step (8192 tokens, 32/8 heads of 128: 1830 clocks for 64 keys, in all 488 us in a graph and 540 to
// 550 by calls one after the other, when the clock goes down; the products alone take 1280): the chain of a softmax warp, its wait (200), load and maximum (450), exponentials (700
// at least, of which the special-function unit has 512 to itself) and hand-over.  Slower or the same were: part of the
// exponentials as a polynomial on the FMA pipe, two threads a row, the row tiles half a step apart without turns, S twice with
// P in its place.
//
// The warps run different code, and evict one another's from the instruction cache where it is long (at 160 KB the same loops took
// 2250 clocks a step, and an item's end 8000): what is rare is called or looped, and each part is in the code once.
//
// Warps 0..3 and 4..7: softmax and epilogue of the two row tiles.  Warps 8 and 9: MMA, one for each row tile, so that the tensor
// pipe has the one's products while the other waits at its barriers.  Warps 10 and 11: keys; 12 and 13: values.  (In one order,
// keys would wait for the values before them, which are free two steps later.)  Warp 14: items, and the query.
//
// Where a page holds a multiple of 8 places, a tile comes by TMA, in boxes of 8 to 128 places and 64 columns (by cp.async two
// warps took 1.7 us for the 64 KiB of a block, more than its products take); the tile with the sequence's end and tiles with pages
// that are none come by cp.async, as all do with other page sizes and strides.  What no row of the CTA sees: a box is zeros; in a
// box that is seen in part it is what the page holds; by cp.async a value is zeros, and a key what shared memory held, for its
// scores are masked.  A value that some rows see and others do not is a product with 0 for those, which is only wrong where it
// is not finite; rows that come out not finite beside such a value are made again, by plain sums, at the CTA's end (remake_rows).
#include <algorithm>
#include <type_traits>

#include "paged_common.cuh"

namespace qmm {
namespace paged {

namespace {

constexpr int kSoftmax = 8;    // warps
constexpr int kLoaders = 2;    // warps, of keys and as many of values
constexpr int kThreads = 32 * (kSoftmax + 2 + 2 * kLoaders + 1);
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
// Growth of a row's maximum, in powers of two, before its base moves; and powers of two by which weights are larger than
// exp(score - base) until the log-sum.  f16 has no full step below 2^-14 and nothing below 2^-25, so with a weight of 1 at the base
// the many keys of a long cache that lie 2^-25 and more below one that stands out would be lost: the two together take its range up
// to 2^15, and what is lost lies 2^-36 below the largest.  Scores that are normal with a deviation of 1 grow by less than 2^4
// behind the first 64, but by more behind a few, as sinks are: where a row's first keys are not 64, the base begins 2^3 above them,
// and what is lost may lie 2^-33 below the largest (6 chunks of 100 to 2000 tokens, window 1024, 4 sinks: 87 to 91 us, without
// that 92 to 95).  bf16 has the exponents of fp32.
template <typename T>
constexpr float kGrowth = std::is_same<T, __half>::value ? 4.0f : 8.0f;
template <typename T>
constexpr float kSpare = std::is_same<T, __half>::value ? 3.0f : 0.0f;
template <typename T>
constexpr float kLift = std::is_same<T, __half>::value ? 15.0f - kGrowth<T> : 0.0f;

// DP: the head dimension rounded up to 64, 128 or 256.  Tensor memory, 512 columns: for each row tile S, 64, and two P, 32
// each; then O.  256 columns of O leave room for one row tile.
template <int DP>
struct Shape {
    static constexpr int kTiles = DP == 256 ? 1 : 2;
    static constexpr int kBN = DP == 256 ? 64 : 128;          // keys of a tile in shared memory
    static constexpr int kSub = kBN / 64;                     // steps of a tile
    static constexpr int kStages = DP == 64 ? 6 : 4;
    static constexpr int kBoxes = DP / 64;                    // of 64 columns: 128-byte rows
    static constexpr int kQueryBox = 128 * 128;               // bytes
    static constexpr int kQuery = kTiles * kBoxes * kQueryBox;
    static constexpr int kBox = kBN * 128;
    static constexpr int kStage = kBoxes * kBox;
    static constexpr int kO = 256;                            // first column of O
    static constexpr int kRows = kTiles * 128;
};

// A CTA's rows: `first` + i of a sequence's rows (tokens times heads of a group), and the places that any of them sees.
struct Tokens {
    int64_t first;     // a sequence's new tokens: their first row in the query, how many, and the place of the first
    int count, place;
};
struct Item {
    Tokens tokens;
    int64_t first, rows;  // this item's first row, and all of the sequence's
    int token, head;      // of the first row, from the sequence's first and the group's
    int b, kvh;
    int sink_end, lo, hi;
    int sink_blocks, first_block, blocks;  // tiles of keys that hold places that are seen
    int split, begin, end;                 // the tiles of this item
    int steps;                             // of 64 keys
    int two;                               // the second row tile has rows
    int cut;                               // its rows have parts in the workspace
    int none;                              // there is no further item
    int far;                               // where its rows' sums are put by (far_sums); -1: nowhere
};

constexpr int kValid = 8;  // tiles of keys whose masks are kept: more than may be under way
struct Tail {
    uint64_t full[6], empty[6];
    uint64_t s_full[2], s_free[2], p_full[2][2], o_done[2][2];  // [row tile], [row tile][step % 2]
    uint64_t o_free[2], q_full, q_empty, item_full[2], item_empty[2], item_loaded, next_full;
    alignas(16) uint32_t valid[kValid][4];
    alignas(16) uint32_t next[4];  // the answer to the request for a further block
    Item item[2];
    uint32_t copied[6];            // stage: by cp.async
    float sum[2][128], base[2][128];  // [group of softmax warps][row]
    uint32_t bad[2][4], going[2][4];  // [group][quarter]: rows that are not finite; the warp has an item
    uint32_t again[2][2][4];  // [item % 2][row tile][quarter]: rows to be made again when the CTA's last item is done
    uint32_t remake;          // there are such rows
    int far;                  // this CTA's place for sums that are put by; -1: none
    uint32_t loaded;          // tiles of keys that have been asked for
    uint32_t tmem_base, abort_flag;
};
template <int DP>
constexpr size_t smem_bytes() {
    return 1024 + Shape<DP>::kQuery + Shape<DP>::kStages * Shape<DP>::kStage + sizeof(Tail);
}

// O in tensor memory loses what its products are cut to as they are added, all towards 0: of n values of one sign some n * 2^-28 (so
// measured: 2^20 places, f16, 0.0029 of the sum).  Items of more than kRun steps put O by in memory every kRun steps and begin
// again from 0 (far_sums), so that this stays within 2^-11; tables of up to kNear places hold few such steps more than that, and go
// without.
constexpr int kRun = 1024;
constexpr int64_t kNear = 1 << 17;

// Workspace (splits > 1): part[split][token * heads + head][dim], stat[split][..] (base, sum), pieces; with tables of more than
// kNear places far[place][row tile][128][far_stride], a place for every SM, and which of them are taken.
struct Scratch {
    float *part;
    float2 *stat;
    int *pieces;  // of them that a call uses; 1: none
    float *far;
    int *far_taken;
    int far_places, far_stride;
    int splits, sms;
    float tile;  // microseconds
    uint32_t *status;
};

struct Plan {
    int64_t pairs;  // at most
    int splits;
    double tile;
    bool far;
    size_t part_bytes, stat_bytes, far_bytes, taken_bytes, bytes;
};
int far_stride(int64_t dim) { return static_cast<int>((dim + 15) / 16 * 16 + 4); }  // a row of O, its base, and 16-byte vectors

// The items of a call are known on the device alone; what the host knows bounds them.  Where they are few, each may be cut into
// pieces (choose_pieces), of which the host says how many at most: as many as give every SM one, or by an estimate in
// microseconds: the CTAs' mean load and half an item, or one item alone.  It takes 1.2 for a tile of 128 keys and one row tile, 2.4
// for two, 1.5 for 64 keys of more than 128 dimensions (measured, an item on every SM over 16384 and 65536 places, the difference:
// 1.08 for heads of 64 and 128, 1.75 to 1.82, 1.09; in short items, with masks and cold code, up to the figures taken), 3 for an
// item, 5 TB/s for the parts of rows, written and read, 4 for the second kernel; and, as lengths are not known, 0.6 of the longest in
// the mean, which is a guess: choose_pieces, which knows them, takes no more pieces than are good.  (Before, 4 CTAs an SM were aimed at: 1184
// tokens through a window of 1024, 32/8 heads of 128, took 111 us, twice as many tokens, whose items were not cut, 77.)
// seen: the places that an item sees at most.
Plan make_plan(int64_t tokens, int64_t batch, int64_t heads, int64_t kv_heads, int64_t dim, int64_t seen) {
    Plan plan;
    const int64_t group = kv_heads > 0 ? heads / kv_heads : 0;
    const int rows = dim > 128 ? Shape<256>::kRows : Shape<128>::kRows, keys = dim > 128 ? Shape<256>::kBN : Shape<128>::kBN;
    const int64_t sequences = batch < tokens ? batch : tokens;
    plan.pairs = tokens * group / rows + sequences;
    plan.splits = 1;
    plan.tile = dim > 128 ? 1.5 : tokens * group > 128 * sequences ? 2.4 : 1.2;
    const int64_t ctas = plan.pairs * kv_heads, sms = sm_count();
    plan.far = seen > kNear && ctas > 0;
    plan.far_bytes = plan.far ? static_cast<size_t>(sms) * rows * far_stride(dim) * sizeof(float) : 0;
    plan.taken_bytes = plan.far ? (static_cast<size_t>(sms) * sizeof(int) + 15) / 16 * 16 : 0;
    if (ctas > 0 && ctas < 2 * sms) {
        const int64_t tiles = (seen + keys - 1) / keys;
        const double tile = plan.tile;
        double best = 0.0;
        const int64_t most = std::min<int64_t>(tiles, ((256ll << 20) - static_cast<int64_t>(plan.far_bytes)) / (tokens * heads * std::max<int64_t>(dim, 1) * 4));  // 256 MiB
        for (int s = 1; s <= 64 && (s == 1 || s <= most); ++s) {
            const double item = tile * tiles / s + 3.0;
            const double load = ctas * (0.6 * tile * tiles + 3.0 * (s == 1 ? 1.0 : 0.6 * s + 0.5)) / sms + 0.5 * item;
            const double us = (load > item ? load : item) + (s > 1 ? 4.0 + tokens * heads * dim * 8.0 * s / 5e6 : 0.0);
            if (s == 1 || us < best) {
                best = us;
                plan.splits = s;
            }
        }
        if (plan.splits > 1) plan.splits = static_cast<int>(std::max<int64_t>(plan.splits, std::min({most, sms / ctas, static_cast<int64_t>(64)})));
    }
    const size_t all = plan.splits > 1 ? static_cast<size_t>(plan.splits) * tokens * heads : 0;
    plan.part_bytes = all * dim * sizeof(float);
    plan.stat_bytes = (all * sizeof(float2) + 15) / 16 * 16;
    plan.bytes = (all > 0 ? plan.part_bytes + plan.stat_bytes + 16 : 0) + plan.far_bytes + plan.taken_bytes;
    return plan;
}

// A sequence's new tokens.
__device__ __forceinline__ Tokens tokens_of(const Problem &p, int b) {
    const int64_t from = min(max(static_cast<int64_t>(__ldg(p.start + b)), static_cast<int64_t>(0)), p.tokens);
    const int64_t to = min(max(static_cast<int64_t>(__ldg(p.start + b + 1)), static_cast<int64_t>(0)), p.tokens);
    Tokens t;
    t.first = from;
    t.count = static_cast<int>(max(to - from, static_cast<int64_t>(0)));
    const int64_t place = static_cast<int64_t>(__ldg(p.lens + b)) - t.count;
    t.place = static_cast<int>(max(place, -static_cast<int64_t>(0x7fffffff)));
    return t;
}

// The token, from the sequence's first, and the group's head of an item's row; and its place.
__device__ __forceinline__ int token_of(const Problem &p, const Item &it, int row, int *head) {
    const uint32_t at = static_cast<uint32_t>(it.head + row), group = static_cast<uint32_t>(p.group), token = at / group;
    *head = static_cast<int>(at - token * group);
    return it.token + static_cast<int>(token);
}
__device__ __forceinline__ int place_of(const Problem &p, const Item &it, int row) {
    int head;
    return max(-1, it.tokens.place + token_of(p, it, row, &head));
}

template <int BN, int ROWS>
__device__ __forceinline__ void cover(const Problem &p, Item &it) {
    it.token = static_cast<int>(it.first / p.group);
    it.head = static_cast<int>(it.first - static_cast<int64_t>(it.token) * p.group);
    const int last = static_cast<int>(min(it.rows - it.first, static_cast<int64_t>(ROWS))) - 1;
    const Range a = visible_range(p, place_of(p, it, 0)), z = visible_range(p, place_of(p, it, last));
    it.sink_end = z.sink_end;
    it.lo = a.lo;
    it.hi = z.hi;
    it.sink_blocks = (z.sink_end + BN - 1) / BN;
    it.first_block = max(a.lo / BN, it.sink_blocks);
    it.blocks = it.sink_blocks + max(0, z.hi / BN + (z.hi % BN != 0) - it.first_block);
}

// The `pair`-th tile (pair) of the call, by one warp: sequences in order, a sequence's last tile, which sees most, first.
template <int BN, int ROWS>
__device__ __forceinline__ bool find_item(const Problem &p, int64_t pair, Item &it) {
    const int lane = threadIdx.x & 31;
    int64_t before = 0;
    for (int b0 = 0; b0 < p.batch; b0 += 32) {
        const int b = b0 + lane;
        int64_t n = 0;
        if (b < p.batch) n = (static_cast<int64_t>(tokens_of(p, b).count) * p.group + ROWS - 1) / ROWS;
        int64_t sum = n;
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t left = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += left;
        }
        const uint32_t past = __ballot_sync(0xffffffffu, before + sum > pair);
        if (past == 0) {
            before += __shfl_sync(0xffffffffu, sum, 31);
            continue;
        }
        const int which = __ffs(past) - 1;
        it.b = b0 + which;
        it.tokens = tokens_of(p, it.b);
        it.rows = static_cast<int64_t>(it.tokens.count) * p.group;
        const int64_t end = before + __shfl_sync(0xffffffffu, sum, which);
        it.first = (end - 1 - pair) * ROWS;
        cover<BN, ROWS>(p, it);
        return true;
    }
    return false;
}

// The tiles of keys of a sequence's item that has most, or somewhat more, and its items of one key-value head.
template <int BN, int ROWS>
__device__ __forceinline__ int most_blocks(const Problem &p, int b, int64_t *items) {
    const Tokens t = tokens_of(p, b);
    *items = (static_cast<int64_t>(t.count) * p.group + ROWS - 1) / ROWS;
    if (t.count == 0) return 0;
    const Range z = visible_range(p, max(-1, t.place + t.count - 1));
    int blocks = z.hi / BN + 1;
    if (p.window > 0) blocks = static_cast<int>(min(static_cast<int64_t>(blocks), (static_cast<int64_t>(p.window) + ROWS / p.group) / BN + 2));
    return blocks + (z.sink_end + BN - 1) / BN;
}

// How many pieces the longest sequence is cut into, and their length in tiles, which is that of all sequences' pieces, so that an
// item is as long as another; by one warp, alike in all CTAs.  The times are those of make_plan, in tiles.  (Cut into as many
// pieces whatever their length, drafts over 2000 to 16000 places took 110 us, not 104; cut at all, equal lengths of 8000 took 107,
// not 95.)
template <int BN, int ROWS>
__device__ __noinline__ int2 choose_pieces(const Problem &p, const Scratch &scratch) {
    const int lane = threadIdx.x & 31;
    int longest = 1;
    float items = 0.0f, total = 0.0f;
    for (int b = lane; b < p.batch; b += 32) {
        int64_t n;
        const int blocks = most_blocks<BN, ROWS>(p, b, &n);
        longest = max(longest, blocks);
        items += static_cast<float>(n * p.kv_heads);
        total += static_cast<float>(n * p.kv_heads) * blocks;
    }
    for (int o = 16; o > 0; o >>= 1) {
        longest = max(longest, __shfl_xor_sync(0xffffffffu, longest, o));
        items += __shfl_xor_sync(0xffffffffu, items, o);
        total += __shfl_xor_sync(0xffffffffu, total, o);
    }
    const float sms = static_cast<float>(scratch.sms), start = 3.0f / scratch.tile, join = 4.0f / scratch.tile;
    const float part = static_cast<float>(p.tokens * p.heads) * p.dim * (8.0f / 5e6f / scratch.tile);
    // as many as give every SM one, and powers of two
    int2 best = make_int2(1, longest);
    float least = INFINITY;
    for (int i = 0; i < 8; ++i) {
        const int n = i < 7 ? 1 << i : static_cast<int>(sms / fmaxf(items, 1.0f));
        if (n < 1 || n > scratch.splits || n > longest) continue;
        const int piece = (longest + n - 1) / n;
        float count = 0.0f;
        for (int b = lane; b < p.batch; b += 32) {
            int64_t m;
            const int blocks = most_blocks<BN, ROWS>(p, b, &m);
            count += static_cast<float>(m * p.kv_heads) * static_cast<float>((blocks + piece - 1) / piece);
        }
        for (int o = 16; o > 0; o >>= 1) count += __shfl_xor_sync(0xffffffffu, count, o);
        const float item = piece + start;
        const float time = (count <= sms ? item : fmaxf(item, (total + count * start) / sms + 0.5f * item)) + (n > 1 ? join + part * n : 0.0f);
        if (time < least) {
            least = time;
            best = make_int2(n, piece);
        }
    }
    return best;
}

template <int BN>
__device__ __forceinline__ int block_start(const Item &it, int i) {
    return (i < it.sink_blocks ? i : it.first_block + i - it.sink_blocks) * BN;
}

template <typename T>
__device__ __forceinline__ bool any_not_finite(const uint4 &v) {
    const uint32_t mask = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) bad |= (w[i] & mask) == mask || (w[i] >> 16 & mask) == mask;
    return bad;
}

// Whether a value of places [from, to) of the sequence is not finite, by one warp.
template <typename T>
__device__ __noinline__ bool holds_not_finite(const Problem &p, int b, int kvh, int from, int to) {
    const int lane = threadIdx.x & 31;
    bool bad = false;
    for (int j = from; j < to; ++j) {
        int64_t block;
        int at;
        if (!find_place(p, b, j, &block, &at)) continue;
        const T *row = static_cast<const T *>(p.v) + block * p.v_sb + at * p.v_st + kvh * p.v_sh;
        for (int c = lane * 8; c < p.dim; c += 256) bad |= any_not_finite<T>(__ldg(reinterpret_cast<const uint4 *>(row + c)));
    }
    return __any_sync(0xffffffffu, bad);
}

// Whether rows whose places are `low` to `high` may have met a value that is not finite at a place that they do not see but that
// is in the CTA's tiles, of the other rows or beside what they see.
template <typename T>
__device__ __forceinline__ bool met_not_finite(const Problem &p, const Item &it, int low, int high) {
    constexpr int kMost = 128;  // places of a tile
    const Range a = visible_range(p, low), z = visible_range(p, high);
    const int limit = min(p.capacity, it.tokens.place + it.tokens.count), hi = min(it.hi, limit - kMost) + kMost;
    if (holds_not_finite<T>(p, it.b, it.kvh, a.hi, hi)) return true;
    if (it.sink_end > 0 && holds_not_finite<T>(p, it.b, it.kvh, a.sink_end, min(it.sink_end, hi - kMost) + kMost)) return true;
    return holds_not_finite<T>(p, it.b, it.kvh, max(it.lo - kMost, a.sink_end), min(z.lo, hi));
}

// Rows of an item again, those that their bits say, `row0` the first, by all warps of the CTA, which share the keys.  kRemade at a
// time; `room`: shared memory for their queries and a part of each a warp.  (264 such rows of each of 8 CTAs, heads of 128: 7 ms over
// 4000 places, 266 over 131072.  One row at a time took 3.5 times as long.)
constexpr int kRemade = 4;
template <typename T>
__device__ __noinline__ void remake_rows(const Problem &p, const Item &it, int row0, uint32_t again, float *room) {
    constexpr int kWarps = kThreads / 32, kPart = 256 + 2;
    static_assert((kRemade * (kPlainDim + kWarps * kPart)) * sizeof(float) <= Shape<64>::kQuery + Shape<64>::kStages * Shape<64>::kStage, "room");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    while (again != 0) {
        int place[kRemade], head[kRemade];
        int64_t token[kRemade];
        RowPart r[kRemade];
#pragma unroll
        for (int i = 0; i < kRemade; ++i) {
            place[i] = -1;
            token[i] = head[i] = 0;
            if (again == 0) continue;
            const int row = row0 + __ffs(again) - 1;
            again &= again - 1;
            place[i] = place_of(p, it, row);
            token[i] = it.tokens.first + token_of(p, it, row, &head[i]);
            head[i] += it.kvh * p.group;
            if (warp == i) stage_query<T>(p, token[i], head[i], room + i * kPlainDim);
        }
        __syncthreads();
        rows_part<T, kRemade>(p, it.b, it.kvh, place, room, warp, kWarps, r);
        float *parts = room + kRemade * kPlainDim;
#pragma unroll
        for (int i = 0; i < kRemade; ++i) {
            float *mine = parts + (i * kWarps + warp) * kPart;
#pragma unroll
            for (int c = 0; c < 8; ++c) mine[c * 32 + lane] = r[i].acc[c];
            if (lane == 0) {
                mine[256] = r[i].top;
                mine[257] = r[i].total;
            }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kRemade; ++i) {
            if (warp != i || place[i] < 0) continue;
            RowPart all = {{}, -INFINITY, 0.0f};
            for (int w = 0; w < kWarps; ++w) {
                const float *one = parts + (i * kWarps + w) * kPart;
                const float top = fmaxf(all.top, one[256]), base = top == -INFINITY ? 0.0f : top;
                const float keep = expf(all.top - base), add = expf(one[256] - base);
                all.top = top;
                all.total = fmaf(one[257], add, all.total * keep);
#pragma unroll
                for (int c = 0; c < 8; ++c) all.acc[c] = fmaf(one[c * 32 + lane], add, all.acc[c] * keep);
            }
            write_row<T>(p, token[i], head[i], all);
        }
        __syncthreads();
    }
}

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// A place for sums that are put by, for as long as the CTA lives; by one thread.  There are as many as SMs, which have a CTA each.
__device__ __noinline__ int take_far(const Scratch &scratch) {
    const int first = static_cast<int>(blockIdx.x % static_cast<unsigned>(scratch.far_places));
    for (int i = 0; i < scratch.far_places; ++i) {
        const int at = (first + i) % scratch.far_places;
        if (atomicCAS(scratch.far_taken + at, 0, 1) == 0) {
            __threadfence();
            return at;
        }
    }
    return -1;
}
// O of a warp's 32 rows (a row a lane), relative to `base`, is added to what was put by, and begins again from 0 (back: the other way
// round).  begins: nothing has been put by.
__device__ __noinline__ void far_sums(const Scratch &scratch, int row, uint32_t o_addr, int ksteps, float base, float scale, bool begins, bool back) {
    float *far = scratch.far + static_cast<int64_t>(row) * scratch.far_stride;
    float4 *sums = reinterpret_cast<float4 *>(far);
    float &far_base = far[scratch.far_stride - 4];
    const float keep = begins || base == -INFINITY ? 1.0f : exp2_fast((far_base - base) * scale);
    for (int c = 0; c < ksteps; ++c) {
        uint32_t o[16];
        tmem_ld_32x16(o_addr + c * 16, o);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float4 x = begins ? make_float4(0.0f, 0.0f, 0.0f, 0.0f) : sums[c * 4 + j];
            x.x = fmaf(x.x, keep, __uint_as_float(o[4 * j]));
            x.y = fmaf(x.y, keep, __uint_as_float(o[4 * j + 1]));
            x.z = fmaf(x.z, keep, __uint_as_float(o[4 * j + 2]));
            x.w = fmaf(x.w, keep, __uint_as_float(o[4 * j + 3]));
            if (!back) sums[c * 4 + j] = x;
            o[4 * j] = back ? __float_as_uint(x.x) : 0u;
            o[4 * j + 1] = back ? __float_as_uint(x.y) : 0u;
            o[4 * j + 2] = back ? __float_as_uint(x.z) : 0u;
            o[4 * j + 3] = back ? __float_as_uint(x.w) : 0u;
        }
        tmem_st_32x16(o_addr + c * 16, o);
    }
    far_base = base;
    tmem_st_wait();
}
// Two warps' turns: a barrier for each, at which the one waits and the other does not.
__device__ __forceinline__ void turn_take(int bar) { asm volatile("bar.sync %0, 64;" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void turn_over(int bar) { asm volatile("bar.arrive %0, 64;" ::"r"(bar) : "memory"); }
__device__ __forceinline__ float max3(float a, float b, float c) {
    float y;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}
__device__ __forceinline__ void cp_async_16(uint32_t dst, const void *src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
// Arrives on the barrier when this thread's copies so far are done.
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
// Four K=16 MMAs under one election: both operands K-major in 128-byte rows (32 bytes, +2, a step).
__device__ __forceinline__ void mma_ss_x4(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t hi, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t"
        ".reg .pred p, e, t;\n\t"
        ".reg .b64 ad, bd;\n\t"
        ".reg .b32 al, bl;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "setp.ne.b32 p, %5, 0;\n\t"
        "setp.eq.b32 t, 0, 0;\n\t"
        "mov.b64 ad, {%1, %3};\n\t"
        "mov.b64 bd, {%2, %3};\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], ad, bd, %4, p;\n\t"
        "add.u32 al, %1, 2;\n\t"
        "add.u32 bl, %2, 2;\n\t"
        "mov.b64 ad, {al, %3};\n\t"
        "mov.b64 bd, {bl, %3};\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], ad, bd, %4, t;\n\t"
        "add.u32 al, %1, 4;\n\t"
        "add.u32 bl, %2, 4;\n\t"
        "mov.b64 ad, {al, %3};\n\t"
        "mov.b64 bd, {bl, %3};\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], ad, bd, %4, t;\n\t"
        "add.u32 al, %1, 6;\n\t"
        "add.u32 bl, %2, 6;\n\t"
        "mov.b64 ad, {al, %3};\n\t"
        "mov.b64 bd, {bl, %3};\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], ad, bd, %4, t;\n\t"
        "}\n" ::"r"(d),
        "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate)
        : "memory");
}
// Eight K=16 MMAs under one election: both operands two boxes of 128-byte rows; the first one begins the accumulator.
__device__ __forceinline__ void mma_ss_x8(uint32_t d, uint32_t a0, uint32_t a1, uint32_t b0, uint32_t b1, uint32_t hi, uint32_t idesc) {
    asm volatile(
        "{\n\t"
        ".reg .pred e, f, t;\n\t"
        ".reg .b64 ad, bd;\n\t"
        ".reg .b32 al, bl;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "setp.ne.b32 f, 0, 0;\n\t"
        "setp.eq.b32 t, 0, 0;\n\t"
        "mov.b64 ad, {%1, %5};\n\t"
        "mov.b64 bd, {%3, %5};\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], ad, bd, %6, f;\n\t"
        "add.u32 al, %1, 2;\n\t"
        "add.u32 bl, %3, 2;\n\t"
        "mov.b64 ad, {al, %5};\n\t"
        "mov.b64 bd, {bl, %5};\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], ad, bd, %6, t;\n\t"
        "add.u32 al, %1, 4;\n\t"
        "add.u32 bl, %3, 4;\n\t"
        "mov.b64 ad, {al, %5};\n\t"
        "mov.b64 bd, {bl, %5};\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], ad, bd, %6, t;\n\t"
        "add.u32 al, %1, 6;\n\t"
        "add.u32 bl, %3, 6;\n\t"
        "mov.b64 ad, {al, %5};\n\t"
        "mov.b64 bd, {bl, %5};\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], ad, bd, %6, t;\n\t"
        "mov.b64 ad, {%2, %5};\n\t"
        "mov.b64 bd, {%4, %5};\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], ad, bd, %6, t;\n\t"
        "add.u32 al, %2, 2;\n\t"
        "add.u32 bl, %4, 2;\n\t"
        "mov.b64 ad, {al, %5};\n\t"
        "mov.b64 bd, {bl, %5};\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], ad, bd, %6, t;\n\t"
        "add.u32 al, %2, 4;\n\t"
        "add.u32 bl, %4, 4;\n\t"
        "mov.b64 ad, {al, %5};\n\t"
        "mov.b64 bd, {bl, %5};\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], ad, bd, %6, t;\n\t"
        "add.u32 al, %2, 6;\n\t"
        "add.u32 bl, %4, 6;\n\t"
        "mov.b64 ad, {al, %5};\n\t"
        "mov.b64 bd, {bl, %5};\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], ad, bd, %6, t;\n\t"
        "}\n" ::"r"(d),
        "r"(a0), "r"(a1), "r"(b0), "r"(b1), "r"(hi), "r"(idesc)
        : "memory");
}
// Four K=16 MMAs under one election: A in tensor memory (eight columns a step), B MN-major (16 rows of 128 bytes, +128, a step).
__device__ __forceinline__ void mma_ts_x4(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t hi, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t"
        ".reg .pred p, e, t;\n\t"
        ".reg .b64 bd;\n\t"
        ".reg .b32 a, bl;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "setp.ne.b32 p, %5, 0;\n\t"
        "setp.eq.b32 t, 0, 0;\n\t"
        "mov.b64 bd, {%2, %3};\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], bd, %4, p;\n\t"
        "add.u32 a, %1, 8;\n\t"
        "add.u32 bl, %2, 128;\n\t"
        "mov.b64 bd, {bl, %3};\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a], bd, %4, t;\n\t"
        "add.u32 a, %1, 16;\n\t"
        "add.u32 bl, %2, 256;\n\t"
        "mov.b64 bd, {bl, %3};\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a], bd, %4, t;\n\t"
        "add.u32 a, %1, 24;\n\t"
        "add.u32 bl, %2, 384;\n\t"
        "mov.b64 bd, {bl, %3};\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a], bd, %4, t;\n\t"
        "}\n" ::"r"(d),
        "r"(a), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate)
        : "memory");
}
// 4-D tiled load global -> shared: columns, places of a page, heads, pages; by one lane of a converged warp.  (16 lanes with a box
// each took 90 clocks a box: the instruction takes uniform operands, so lanes that differ go one by one.)
__device__ __forceinline__ void tma_load_4d_warp(uint32_t dst, const CUtensorMap *m, int32_t column, int32_t place, int32_t head, int32_t page,
                                            uint32_t bar) {
    asm volatile(
        "{\n\t"
        ".reg .pred e;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "@e cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];\n\t"
        "}\n" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(m)), "r"(bar), "r"(column), "r"(place), "r"(head), "r"(page)
        : "memory");
}
// Asks for a block of the grid that has not begun, in its place; the answer, 16 bytes, is counted on the barrier.
__device__ __forceinline__ void ask_next_block(uint32_t answer, uint32_t bar) {
    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(answer), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ bool next_block(uint32_t answer, uint32_t *block) {
    uint32_t got, x;
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        ".reg .b128 a;\n\t"
        "ld.shared.b128 a, [%2];\n\t"
        "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, a;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t"
        "mov.u32 %1, 0;\n\t"
        "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, a;\n\t"
        "}\n"
        : "=r"(got), "=r"(x)
        : "r"(answer)
        : "memory");
    *block = x;
    return got != 0;
}
// Whether a barrier's phase is done, without waiting: asked some time before the answer is used, for it takes 100 clocks.
__device__ __forceinline__ uint32_t mbar_done(uint32_t bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t"
        "}\n"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    return done;
}
// mbar_wait for what takes as long as an item has keys: its limit begins anew when the tiles that have been asked for are more.
__device__ __noinline__ bool wait_while_moving(uint32_t bar, uint32_t parity, volatile uint32_t *moving, volatile uint32_t *abort_flag, uint32_t where) {
    uint64_t since = globaltimer_ns();
    uint32_t last = *moving, spins = 0;
    while (!mbar_try_wait(bar, parity)) {
        if ((++spins & 0xffu) != 0) continue;
        if (*abort_flag != 0) return false;
        const uint32_t now = *moving;
        const uint64_t time = globaltimer_ns();
        if (now != last) {
            last = now;
            since = time;
        } else if (time - since > kWaitLimitNs) {
            *abort_flag = DEV_STATUS_WAIT_TIMEOUT | where;
            return false;
        }
    }
    return true;
}
__device__ __forceinline__ void mbar_arrive_n(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
// 32 bytes to global memory, a whole sector where it begins at one.
__device__ __forceinline__ void store_32(void *dst, const uint32_t *x) {
    if ((reinterpret_cast<uintptr_t>(dst) & 31) == 0) {
        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(x[4]),
                     "r"(x[5]), "r"(x[6]), "r"(x[7])
                     : "memory");
    } else {
        static_cast<uint4 *>(dst)[0] = make_uint4(x[0], x[1], x[2], x[3]);
        static_cast<uint4 *>(dst)[1] = make_uint4(x[4], x[5], x[6], x[7]);
    }
}
// Bits [from, to) of a word, the bounds being any numbers.
__device__ __forceinline__ uint32_t bits(int from, int to) {
    const uint32_t low = to <= 0 ? 0u : to >= 32 ? 0xffffffffu : (1u << to) - 1;
    return from <= 0 ? low : from >= 32 ? 0u : low & (0xffffffffu << from);
}

// Tokens of no sequence: block `id`'s part of them.
template <typename T>
__device__ __noinline__ void clear_rest(const Problem &p, const Scratch &scratch, int64_t id, int64_t blocks) {
    const int lane = threadIdx.x & 31;
    const int64_t head = p.batch > 0 ? min(max(static_cast<int64_t>(__ldg(p.start)), static_cast<int64_t>(0)), p.tokens) : p.tokens;
    const int64_t end = p.batch > 0 ? min(max(static_cast<int64_t>(__ldg(p.start + p.batch)), head), p.tokens) : p.tokens;
    const int64_t none = head + p.tokens - end;
    for (int64_t i = id; i < none; i += blocks) {
        const int64_t token = i < head ? i : end + i - head;
        for (int h = 0; h < p.heads; ++h) empty_row<T>(p, token, h);
        if (scratch.splits > 1)
            for (int64_t h = lane; h < static_cast<int64_t>(p.heads) * scratch.splits; h += 32)
                scratch.stat[h / p.heads * p.tokens * p.heads + token * p.heads + h % p.heads] = make_float2(-INFINITY, 0.0f);
    }
}

template <typename T, int DP>
__global__ void __launch_bounds__(kThreads, 1)
prompt_kernel(const __grid_constant__ Problem p, const __grid_constant__ Scratch scratch, const __grid_constant__ CUtensorMap tmap_k,
              const __grid_constant__ CUtensorMap tmap_v, const __grid_constant__ CUtensorMap tmap_q, int box_rows, bool box_query) {
    using S = Shape<DP>;
    constexpr int BN = S::kBN;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t *smem = smem_raw + (smem_base - smem_u32(smem_raw));
    Tail *tail = reinterpret_cast<Tail *>(smem + S::kQuery + S::kStages * S::kStage);
    volatile uint32_t *abort_flag = &tail->abort_flag;
    const uint32_t ring = smem_base + S::kQuery;
    const int warp = warp_id_uniform(), lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int s = 0; s < S::kStages; ++s) {
            mbar_init(smem_u32(&tail->full[s]), kLoaders * 33);  // every lane's copies, and the lookup
            mbar_init(smem_u32(&tail->empty[s]), S::kTiles);     // every row tile's products
        }
        for (int i = 0; i < 4; ++i) {
            mbar_init(smem_u32(&tail->p_full[i >> 1][i & 1]), 4);
            mbar_init(smem_u32(&tail->o_done[i >> 1][i & 1]), 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&tail->s_full[i]), 1);
            mbar_init(smem_u32(&tail->s_free[i]), 4);
            mbar_init(smem_u32(&tail->o_free[i]), 4);
            mbar_init(smem_u32(&tail->item_full[i]), 1);
            mbar_init(smem_u32(&tail->item_empty[i]), 5 * S::kTiles + 2 * kLoaders);  // the warps that take items
        }
        mbar_init(smem_u32(&tail->q_full), 33);
        mbar_init(smem_u32(&tail->q_empty), S::kTiles);
        mbar_init(smem_u32(&tail->item_loaded), 1);
        mbar_init(smem_u32(&tail->next_full), 1);
        tail->abort_flag = 0;
        tail->remake = 0;
        tail->far = -1;
        tail->loaded = 0;
        for (int i = 0; i < 16; ++i) tail->again[i >> 3][i >> 2 & 1][i & 3] = 0;
        mbar_fence_init();
        if (box_rows > 0) {
            tma_prefetch_desc(&tmap_k);
            tma_prefetch_desc(&tmap_v);
        }
        if (box_query) tma_prefetch_desc(&tmap_q);
    }
    if (warp == kSoftmax) {
        tmem_alloc(smem_u32(&tail->tmem_base), 512);
        tmem_relinquish();
        pdl_launch_dependents();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = warp_uniform(tail->tmem_base);
    pdl_wait();

    const int ksteps = (p.dim + 15) / 16;
    const float factor = p.scale * kLog2e;
    // the `n`-th item of this CTA; and its slot free again
    auto take = [&](int n) { return mbar_wait(smem_u32(&tail->item_full[n & 1]), (n >> 1) & 1, abort_flag, 0x9d); };
    auto release = [&](int n) {
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&tail->item_empty[n & 1]));
    };

    if (warp == kSoftmax + 2 + 2 * kLoaders) {
        // ---------------- items, and the query ----------------
        uint32_t id = blockIdx.x, asked = 0, queries = 0;
        const int2 pieces = scratch.splits > 1 ? choose_pieces<BN, S::kRows>(p, scratch) : make_int2(1, 0);
        if (scratch.splits > 1 && lane == 0) *scratch.pieces = pieces.x;  // the same from all CTAs
        const uint32_t units = gridDim.x / scratch.splits;
        bool have = true, ok = true;
        int n = 0;
        while (ok && have) {
            // a block is asked for when the present item's last keys are, not earlier: what is taken cannot go to another CTA
            if (n > 0) ok = wait_while_moving(smem_u32(&tail->item_loaded), (n - 1) & 1, &tail->loaded, abort_flag, 0x9c);
            ok = ok && mbar_wait(smem_u32(&tail->item_empty[n & 1]), (n >> 1 & 1) ^ 1, abort_flag, 0x9e);
            if (!ok) break;
            Item it;
            bool found = false;
            while (true) {
                if (asked > 0) {
                    clear_rest<T>(p, scratch, id, gridDim.x);
                    // Rows are to be made again: no further item.  (What is left begins as blocks of its own.)  An item before the
                    // last two has said so by now, so that these are still in their places.
                    have = *reinterpret_cast<volatile uint32_t *>(&tail->remake) == 0;
                    have = __all_sync(0xffffffffu, have);
                    if (!have) break;
                    if (lane == 0) {
                        mbar_expect_tx(smem_u32(&tail->next_full), 16);
                        ask_next_block(smem_u32(tail->next), smem_u32(&tail->next_full));
                    }
                    __syncwarp();
                    ok = mbar_wait(smem_u32(&tail->next_full), (asked - 1) & 1, abort_flag, 0x8f);
                    if (!ok) break;
                    have = next_block(smem_u32(tail->next), &id);
                    fence_proxy_async_smem();  // read before the next answer is written
                    __syncwarp();
                    if (!have) break;
                }
                ++asked;
                it.split = id / units;
                if (it.split >= pieces.x) continue;
                it.kvh = id % units % p.kv_heads;
                found = find_item<BN, S::kRows>(p, id % units / p.kv_heads, it);
                if (!found) continue;
                it.begin = 0;
                it.end = it.blocks;
                it.cut = pieces.x > 1;
                if (!it.cut) break;
                it.begin = min(it.split * pieces.y, it.blocks);
                it.end = it.split + 1 < pieces.x ? min(it.begin + pieces.y, it.blocks) : it.blocks;
                if (it.begin < it.end) break;
                const int rows = static_cast<int>(min(it.rows - it.first, static_cast<int64_t>(S::kRows)));
                for (int r = lane; r < rows; r += 32) {
                    int head;
                    const int64_t token = it.tokens.first + token_of(p, it, r, &head);
                    scratch.stat[(it.split * p.tokens + token) * p.heads + it.kvh * p.group + head] = make_float2(-INFINITY, 0.0f);
                }
                found = false;
            }
            if (!ok) break;
            if (found) {
                it.two = S::kTiles == 2 && it.first + 128 < it.rows;
                // the last tile's second half may lie behind all that is seen (a tile of sinks may have some of the window)
                it.steps = (it.end - it.begin) * S::kSub;
                if (S::kSub == 2 && it.end > it.begin) {
                    const int last = block_start<BN>(it, it.end - 1);
                    if (last + 64 >= (it.end - 1 < it.sink_blocks && it.lo >= last + BN ? it.sink_end : it.hi)) --it.steps;
                }
                it.far = -1;
                if (scratch.far_places > 0 && it.steps > kRun) {
                    if (lane == 0 && tail->far < 0) tail->far = take_far(scratch);
                    __syncwarp();
                    it.far = tail->far;
                }
            }
            if (lane == 0) {
                it.none = 0;
                if (found)
                    tail->item[n & 1] = it;
                else
                    tail->item[n & 1].none = 1;  // the rest is that of an item whose rows may have to be made again
                mbar_arrive(smem_u32(&tail->item_full[n & 1]));
            }
            __syncwarp();
            ++n;
            if (found && it.steps > 0) {
                ok = mbar_wait(smem_u32(&tail->q_empty), (queries & 1) ^ 1, abort_flag, 0x9f);
                if (!ok) break;
                ++queries;
                const uint32_t bar = smem_u32(&tail->q_full);
                const int tiles = it.two ? 2 : 1;
                if (box_query) {
                    if (lane == 0) {
                        mbar_expect_tx(bar, tiles * S::kBoxes * S::kQueryBox);
                        mbar_arrive_n(bar, 32);
                    }
                    __syncwarp();
                    for (int tile = 0; tile < tiles; ++tile) {
                        int head;
                        const int token = static_cast<int>(it.tokens.first) + token_of(p, it, tile * 128, &head);
#pragma unroll
                        for (int column = 0; column < S::kBoxes; ++column)
                            tma_load_4d_warp(smem_base + (tile * S::kBoxes + column) * S::kQueryBox, &tmap_q, column * 64, 0, it.kvh, token, bar);
                    }
                } else {
                    // row by row: 16-byte chunks into 128-byte rows, swizzled; zeros behind the sequence's rows
                    constexpr int kChunks = DP / 8, kStep = 32 / kChunks;
                    const int chunk = lane % kChunks;
                    const bool mine = chunk < 2 * ksteps, there = chunk * 8 < p.dim;
                    const T *q = static_cast<const T *>(p.q) + it.kvh * p.group * p.q_sh + (there ? chunk * 8 : 0);
                    int head;
                    int64_t token = token_of(p, it, lane / kChunks, &head);
                    for (int r = lane / kChunks; r < tiles * 128; r += kStep) {
                        const bool row = it.first + r < it.rows;
                        if (mine)
                            cp_async_16(smem_base + ((r >> 7) * S::kBoxes + chunk / 8) * S::kQueryBox + (r & 127) * 128 + (((chunk ^ r) & 7) << 4),
                                        row ? q + (it.tokens.first + token) * p.q_st + head * p.q_sh : q, row && there ? 16 : 0);
                        for (head += kStep; head >= p.group; head -= p.group) ++token;
                    }
                    cp_async_arrive(bar);
                    if (lane == 0) mbar_arrive(bar);
                }
            }
        }
        cp_async_wait_all();
    } else if (warp >= kSoftmax + 2) {
        // ---------------- keys and values ----------------
        const int part = (warp - kSoftmax - 2) / kLoaders, loader = (warp - kSoftmax - 2) % kLoaders;  // keys 0, values 1
        constexpr int kChunks = DP / 8, kStep = 32 / kChunks;
        constexpr int kLooks = BN / 32;  // places that a lane looks up; every loader all of them
        const int my_key = lane / kChunks, my_chunk = lane % kChunks;
        const int row_chunks = p.dim / 8;
        const bool my_part = my_chunk < 2 * ksteps;
        const uint32_t my_box = (my_chunk / 8) * S::kBox;
        const int my_offset = my_chunk < row_chunks ? my_chunk * 8 : 0;
        // Boxes: a warp fetches every second (a box takes it some 100 clocks to issue).  Lane g of a warp has looked up the
        // page of a tile's g-th box a tile ahead.  A tile that is seen in part comes in boxes, too, where its boxes that are
        // seen lie before the sequence's end: what else they hold was written by earlier tokens, and is masked; a box that is
        // not seen is one behind the cache's last page, which is zeros.  (A box that is seen, once more, would give the rows that
        // see an infinite value in it 0 times that value as well.)  The rest of a page behind the end may be anything, NaN
        // as well, and comes as zeros.
        const int boxes = box_rows > 0 ? BN / box_rows : 0;
        constexpr int kMost = (BN / 8 + kLoaders - 1) / kLoaders;
        int mine = 0;
        for (int n = loader; n < boxes; n += kLoaders) ++mine;
        const uint32_t my_bytes = mine * S::kBoxes * box_rows * 128;
        const CUtensorMap *map = part == 0 ? &tmap_k : &tmap_v;
        uint32_t stage = part, phase = 0, count = 0;  // even stages: keys
        bool ok = true;
        for (int n = 0; ok; ++n) {
            ok = take(n);
            if (!ok || tail->item[n & 1].none) break;
            const Item it = tail->item[n & 1];
            release(n);
            const int limit = min(p.capacity, it.tokens.place + it.tokens.count);  // the sequence's end
            int next_id = -1, next_at = 0;
            bool next_seen = false;
            auto look_up = [&](int i) {
                if (lane >= boxes) return;
                const int j = block_start<BN>(it, i) + lane * box_rows;
                next_id = -1;
                next_seen = j < it.hi && (j < it.sink_end || j > it.lo - box_rows);
                if (next_seen && j <= limit - box_rows) {
                    const int page = page_of(p, j);
                    next_at = j - page * p.page;
                    next_id = __ldg(p.table + it.b * p.table_st + page);
                }
            };
            if (it.begin < it.end) look_up(it.begin);
            for (int i = it.begin; i < it.end && ok; ++i, ++count) {
                const int first = block_start<BN>(it, i);
                const uint32_t seen_boxes = __ballot_sync(0xffffffffu, next_seen);
                const bool whole = seen_boxes != 0 && __all_sync(0xffffffffu, !next_seen || (next_id >= 0 && next_id < p.pages));
                uint32_t mask[kLooks];
                int id[kLooks], at[kLooks], box_page[kMost], box_place[kMost];
                if (whole) {
#pragma unroll
                    for (int k = 0; k < kMost; ++k) {
                        const int box = loader + k * kLoaders;
                        box_page[k] = __shfl_sync(0xffffffffu, next_seen ? next_id : static_cast<int>(p.pages), box);
                        box_place[k] = __shfl_sync(0xffffffffu, next_at, box);
                    }
                } else {
#pragma unroll
                    for (int l = 0; l < kLooks; ++l) {
                        const int j = first + 32 * l + lane;
                        int64_t block = 0;
                        at[l] = 0;
                        const bool seen = j < it.hi && (j < it.sink_end || j >= it.lo) && find_place(p, it.b, j, &block, &at[l]);
                        id[l] = static_cast<int>(block);
                        mask[l] = __ballot_sync(0xffffffffu, seen);
                    }
                }
                if (i + 1 < it.end) look_up(i + 1);
                ok = mbar_wait(smem_u32(&tail->empty[stage]), phase ^ 1, abort_flag, 0x90);
                if (!ok) break;
                const uint32_t bar = smem_u32(&tail->full[stage]), dst = ring + stage * S::kStage;
                if (whole) {
                    if (lane == 0) {
                        if (loader == 0) {
                            if (part == 0) *reinterpret_cast<uint4 *>(tail->valid[count % kValid]) = make_uint4(~0u, ~0u, ~0u, ~0u);
                            tail->copied[stage] = 0;
                        }
                        mbar_expect_tx(bar, my_bytes);
                        mbar_arrive_n(bar, 32);
                    }
                    __syncwarp();
#pragma unroll
                    for (int k = 0; k < kMost; ++k) {
                        const int box = loader + k * kLoaders;
                        if (box >= boxes) break;
#pragma unroll
                        for (int column = 0; column < S::kBoxes; ++column)
                            tma_load_4d_warp(dst + column * S::kBox + box * box_rows * 128, map, column * 64, box_place[k], it.kvh, box_page[k], bar);
                    }
                } else {
                    if (loader == 0 && lane == 0) {
                        tail->copied[stage] = 1;
#pragma unroll
                        for (int l = 0; part == 0 && l < kLooks; ++l) tail->valid[count % kValid][l] = mask[l];
                    }
                    const T *base = static_cast<const T *>(part == 0 ? p.k : p.v) + my_offset;
                    const int64_t sb = part == 0 ? p.k_sb : p.v_sb, st = part == 0 ? p.k_st : p.v_st, head = it.kvh * (part == 0 ? p.k_sh : p.v_sh);
#pragma unroll
                    for (int l = 0; l < kLooks; ++l) {
                        static_assert(kLoaders == 2, "each takes 16 of 32 keys");
                        // keys that are not seen may be anything, for their scores are masked; values are multiplied by 0
                        if (part == 0 && (mask[l] >> loader * 16 & 0xffff) == 0) continue;
                        const int64_t offset = mask[l] >> lane & 1 ? id[l] * sb + at[l] * st + head : 0;
                        // a short loop: unrolled, these copies were 42 KB of code, and what the other warps ran was fetched
                        // again and again
#pragma unroll 2
                        for (int key = loader * 16 + my_key; key < loader * 16 + 16; key += kStep) {
                            const T *row = base + __shfl_sync(0xffffffffu, offset, key);
                            if (my_part)
                                cp_async_16(dst + my_box + (l * 32 + key) * 128 + (((my_chunk ^ key) & 7) << 4), row,
                                            my_chunk < row_chunks && (mask[l] >> key & 1) ? 16 : 0);
                        }
                    }
                    cp_async_arrive(bar);
                    if (lane == 0) mbar_arrive(bar);
                }
                if (part == 0 && loader == 0 && lane == 0) *reinterpret_cast<volatile uint32_t *>(&tail->loaded) = count + 1;
                stage += 2;
                if (stage >= S::kStages) {
                    stage -= S::kStages;
                    phase ^= 1;
                }
            }
            if (part == 0 && loader == 0 && lane == 0) mbar_arrive(smem_u32(&tail->item_loaded));
        }
        cp_async_wait_all();
    } else if (warp >= kSoftmax && warp < kSoftmax + S::kTiles) {
        // ---------------- MMA ----------------
        const uint32_t tile = warp_uniform(warp - kSoftmax);
        constexpr uint32_t kFmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
        constexpr uint32_t kHi = smem_desc_hi_sw128(1024);
        constexpr uint32_t s_desc = make_idesc(1, kFmt, kFmt, 0, 0, 128, 64);
        const uint32_t o_desc = make_idesc(1, kFmt, kFmt, 0, 1, 128, ksteps * 16);
        constexpr uint32_t kSubStep = 64 * 128 >> 4;  // 64 rows of a box
        // Counters and descriptors in a form that the compiler knows to be the same in all lanes
        const uint32_t q_lo = warp_uniform(smem_desc_lo(smem_base, 16));
        const uint32_t k_lo = warp_uniform(smem_desc_lo(ring, 16)), v_lo = warp_uniform(smem_desc_lo(ring, S::kBox));
        const uint32_t bars = warp_uniform(smem_u32(tail));
        auto bar_of = [&](const uint64_t *bar) { return bars + static_cast<uint32_t>(reinterpret_cast<const uint8_t *>(bar) - reinterpret_cast<const uint8_t *>(tail)); };
        constexpr uint32_t kStageStep = S::kStage >> 4;
        // The loaders' copies are writes of the generic proxy, which their barrier makes visible here; the fence hands them to the
        // MMA's.
        auto landed = [&](uint32_t stage, uint32_t phase, uint32_t where) {
            const bool there = mbar_wait(bar_of(tail->full) + stage * 8, phase, abort_flag, where);
            if (tail->copied[stage] != 0) fence_proxy_async_smem();
            return there;
        };
        auto product_s = [&](uint32_t a, uint32_t b) {
            const uint32_t d = tmem_base + tile * 128;
            if (S::kBoxes == 2 && ksteps == 8) {
                mma_ss_x8(d, a, a + (S::kQueryBox >> 4), b, b + (S::kBox >> 4), kHi, s_desc);
            } else {
#pragma unroll
                for (int box = 0; box < S::kBoxes; ++box)
                    if (box * 4 + 4 <= ksteps)
                        mma_ss_x4(d, a + box * (S::kQueryBox >> 4), b + box * (S::kBox >> 4), kHi, s_desc, box > 0);
#pragma unroll 1
                for (int k = ksteps & ~3; k < ksteps; ++k)
                    mma_f16_ss_warp(d, desc64(a + (k >> 2) * (S::kQueryBox >> 4) + (k & 3) * 2, kHi),
                                    desc64(b + (k >> 2) * (S::kBox >> 4) + (k & 3) * 2, kHi), s_desc, k > 0);
            }
            tc_commit_warp(bar_of(tail->s_full) + tile * 8);
        };
        // 16 keys a MMA: eight columns of P; 16 rows of 128 bytes of V, its next 64 columns a box further
        auto product_o = [&](uint32_t odd, uint32_t b, uint32_t accumulate) {
            mma_ts_x4(tmem_base + S::kO + tile * 128, tmem_base + tile * 128 + 64 + odd * 32, b, kHi, o_desc, accumulate);
            tc_commit_warp(bar_of(tail->o_done[0]) + (tile * 2 + odd) * 8);
        };
        // The tiles of keys and values that the next product takes, and its half of them: keys in the even stages, values in the
        // odd ones.  A stage is free when the products so far of both MMA warps are done.
        uint32_t k_stage = 0, k_phase = 0, k_half = 0, v_stage = 1, v_phase = 0, v_half = 0;
        bool shared = false;
        auto leave = [&](uint32_t &stage, uint32_t &phase) {
            tc_commit_warp(bar_of(tail->empty) + stage * 8);
            stage += 2;
            if (stage >= S::kStages) {
                stage -= S::kStages;
                phase ^= 1;
            }
        };
        auto advance = [&](uint32_t &stage, uint32_t &phase, uint32_t &half) {
            if (!shared) {
                if (++half < S::kSub) return;
                half = 0;
            }
            leave(stage, phase);
        };
        uint32_t done = 0, made = 0;     // steps of this warp; S made
        uint32_t queries = 0, outs = 0;  // items with a query; items that this warp had steps of
        bool ok = true;
        for (int n = 0; ok; ++n) {
            ok = take(n);
            if (!ok || tail->item[n & 1].none) break;
            const int steps = static_cast<int>(warp_uniform(tail->item[n & 1].steps));
            shared = warp_uniform(S::kTiles == 2 && !tail->item[n & 1].two) != 0;
            release(n);
            if (steps == 0) continue;
            const int all = !shared ? steps : tile == 0 ? (steps + 1) / 2 : steps / 2;
            const uint32_t a = q_lo + (shared ? 0 : tile * (S::kBoxes * S::kQueryBox >> 4));
            k_half = v_half = shared ? tile : 0;
            ok = mbar_wait(bar_of(&tail->q_full), queries & 1, abort_flag, 0x91);
            if (!box_query) fence_proxy_async_smem();
            ++queries;
            if (all == 0) tc_commit_warp(bar_of(&tail->q_empty));
            auto make_s = [&](int step) {
                if (shared || k_half == 0) ok = ok && landed(k_stage, k_phase, 0x93);
                // the softmax has taken the S before
                if (made > 0) ok = ok && mbar_wait(bar_of(tail->s_free) + tile * 8, (made - 1) & 1, abort_flag, 0x92);
                if (!ok) return;
                tc_fence_after();
                product_s(a, k_lo + k_stage * kStageStep + k_half * kSubStep);
                ++made;
                if (step + 1 == all) tc_commit_warp(bar_of(&tail->q_empty));
                advance(k_stage, k_phase, k_half);
            };
            for (int step = -1; step < all && ok; ++step) {
                if (step + 1 < all) make_s(step + 1);
                if (step < 0) continue;
                const uint32_t odd = done & 1;
                if (shared || v_half == 0) ok = ok && landed(v_stage, v_phase, 0x94);
                if (step == 0) {
                    // the softmax has read the O of the item before
                    if (outs > 0) ok = ok && mbar_wait(bar_of(tail->o_free) + tile * 8, (outs - 1) & 1, abort_flag, 0x95);
                    ++outs;
                }
                ok = ok && mbar_wait(bar_of(tail->p_full[0]) + (tile * 2 + odd) * 8, (done >> 1) & 1, abort_flag, 0x96);
                if (!ok) break;
                tc_fence_after();
                product_o(odd, v_lo + v_stage * kStageStep + v_half * kSubStep, step > 0);
                advance(v_stage, v_phase, v_half);
                ++done;
            }
            // tiles whose second half was not taken; not before they have come, lest a stage be freed twice by one warp
            if (ok && S::kSub == 2 && (steps & 1) && (!shared || tile == 1)) {
                ok = landed(k_stage, k_phase, 0x8d) && landed(v_stage, v_phase, 0x8c);
                leave(k_stage, k_phase);
                leave(v_stage, v_phase);
            }
        }
    } else if (warp < 4 * S::kTiles) {
        // ---------------- softmax and epilogue: a row a thread ----------------
        const int group = warp >> 2, quarter = warp & 3;
        const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
        const int my_lane = quarter * 32 + lane;
        // The running maximum is one of unscaled scores, which takes a positive scale: with a negative one, or 0, the scores
        // take its sign.
        const float scale = factor == 0.0f ? 1.0f : fabsf(factor), sign = factor < 0.0f ? -1.0f : 0.0f;
        // the warps of both groups that have a quarter of the rows, or two such quarters
        auto meet = [&] {
            if (S::kTiles == 2) asm volatile("bar.sync %0, 64;" ::"r"(1 + quarter) : "memory");
        };
        uint32_t done = 0, count = 0;  // steps of this warp; tiles of keys
        for (int item = 0;; ++item) {
            // A wait that gave up ends the warps that meet together; inside an item it ends the waits, not the steps.
            bool ok = take(item);
            if (lane == 0) tail->going[group][quarter] = ok && !tail->item[item & 1].none;
            __syncwarp();
            meet();
            const bool go = tail->going[0][quarter] != 0 && tail->going[S::kTiles - 1][quarter] != 0;
            meet();
            if (!go) break;
            const Item &it = tail->item[item & 1];
            // One row tile: both groups of warps have its rows, the second one the second 64 of every 128 keys.
            const bool shared = S::kTiles == 2 && !it.two;
            const int steps = !shared ? it.steps : group == 0 ? (it.steps + 1) / 2 : it.steps / 2;
            const int row0 = (shared ? 0 : group * 128) + quarter * 32;  // this warp's first one
            const int rows = static_cast<int>(min(it.rows - it.first, static_cast<int64_t>(S::kRows)));
            // Two row tiles take turns at the exponentials of a step, quarter by quarter: both at once, they would wait for the
            // special-function unit together, and leave it together.
            const bool turns = S::kTiles == 2 && !shared;
            float base = -INFINITY;  // unscaled
            float2 sum2 = make_float2(0.0f, 0.0f);
            if (steps > 0) {
                const Range range = visible_range(p, row0 + lane < rows ? place_of(p, it, row0 + lane) : -1);
                // what all rows of the warp see: places up to sink_last + 63, and from all_lo to hi_last + 63
                const Range low = visible_range(p, place_of(p, it, min(row0, rows - 1)));
                const int all_lo = visible_range(p, place_of(p, it, min(row0 + 31, rows - 1))).lo;
                const int sink_last = low.sink_end - 64, hi_last = low.hi - 64;
                // a step's first place and the masks of its places: from one tile to the next, but for the gap behind the sinks
                int start = block_start<BN>(it, it.begin) + (shared ? group * 64 : 0);
                const int stride = shared ? BN : 64, gap = (it.first_block - it.sink_blocks) * BN;
                int sink_steps = (it.sink_blocks - it.begin) * (shared ? 1 : S::kSub);  // until the gap
                const uint32_t valid_stride = shared || S::kSub == 1 ? 16 : 8;
                uint32_t valid_at = (count * 16 + (shared ? group * 8 : 0)) % (kValid * 16);
                const int far_from = it.far >= 0 ? kRun : 0x7fffffff, far_row = (it.far * S::kTiles + group) * 128 + my_lane;
                if (turns && group == 1) turn_over(5 + quarter);
                for (int n = 0; n < steps; ++n, ++done) {
                    const uint32_t odd = done & 1;
                    ok = ok && mbar_wait(smem_u32(&tail->s_full[group]), done & 1, abort_flag, 0x98);
                    tc_fence_after();
                    const uint32_t s_addr = tmem_base + lanes + group * 128, p_addr = s_addr + 64 + odd * 32;
                    uint32_t s[2][32];
                    tmem_ld_32x32(s_addr, s[0]);
                    tmem_ld_32x32(s_addr + 32, s[1]);
                    const uint2 valid = *reinterpret_cast<const uint2 *>(reinterpret_cast<const uint8_t *>(tail->valid) + valid_at);
                    // whether this step's place of P is free.  (A barrier for even and one for odd steps, each waited for in every
                    // phase, so that a phase's parity is its own.)
                    const uint32_t p_bar = smem_u32(&tail->o_done[group][odd]), p_phase = ((done - 2) >> 1) & 1;
                    const bool free = done < 2 || mbar_done(p_bar, p_phase) != 0;
                    tmem_ld_wait();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&tail->s_free[group]));
                    const bool whole = (start <= sink_last || (start >= all_lo && start <= hi_last)) && (valid.x & valid.y) == 0xffffffffu;
                    if (factor <= 0.0f) {
#pragma unroll
                        for (int j = 0; j < 64; ++j) s[j / 32][j % 32] = __float_as_uint(__uint_as_float(s[j / 32][j % 32]) * sign);
                    }
                    if (!whole) {
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            const int at = start + c * 32;
                            const uint32_t see = (c == 0 ? valid.x : valid.y) & bits(0, range.hi - at) & (bits(0, range.sink_end - at) | bits(range.lo - at, 32));
#pragma unroll
                            for (int j = 0; j < 32; ++j)
                                if (!(see >> j & 1)) s[c][j] = 0xff800000u;  // -inf
                        }
                    }
                    float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int j = 0; j < 64; j += 8) {
#pragma unroll
                        for (int c = 0; c < 4; ++c)
                            m[c] = max3(m[c], __uint_as_float(s[j / 32][j % 32 + 2 * c]), __uint_as_float(s[j / 32][j % 32 + 2 * c + 1]));
                    }
                    const float most = max3(max3(m[0], m[1], m[2]), m[3], m[3]);
                    const bool move = most > base && (most - base) * scale > kGrowth<T>;  // from -inf always
                    const bool put_by = n >= far_from && (n & (kRun - 1)) == 0;
                    if (__any_sync(0xffffffffu, move || put_by)) {
                        float now = move ? most : base;
                        if (kSpare<T> > 0.0f && move && base == -INFINITY && !whole) now += fminf(kSpare<T> / scale, 1e30f);
                        const float keep = exp2_fast(now == -INFINITY ? 0.0f : (base - now) * scale);
                        sum2 = mul2(sum2, make_float2(keep, keep));
                        if (n > 0) {
                            ok = ok && mbar_wait(smem_u32(&tail->o_done[group][odd ^ 1]), ((done - 1) >> 1) & 1, abort_flag, 0x99);
                            tc_fence_after();
                            if (put_by) far_sums(scratch, far_row, tmem_base + lanes + S::kO + group * 128, ksteps, base, scale, n == kRun, false);
                            for (int c = 0; c < ksteps && !put_by; ++c) {
                                uint32_t o[16];
                                const uint32_t addr = tmem_base + lanes + S::kO + group * 128 + c * 16;
                                tmem_ld_32x16(addr, o);
                                tmem_ld_wait();
#pragma unroll
                                for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * keep);
                                tmem_st_32x16(addr, o);
                            }
                        }
                        base = now;
                    }
                    // P in the type of the values: off by half a step, 2^-8 or 2^-11, of each weight (of f16 weights below 2^-25
                    // of the largest: up to 2^-33 of that one).  The sum takes the weights unrounded, so equal weights are all off
                    // alike.
                    float offset = base == -INFINITY ? 0.0f : fmaf(-base, scale, kLift<T>);
                    if (turns) turn_take(5 + 4 * group + quarter);
                    asm volatile("" : "+f"(offset));  // no exponential before the turn
                    const float2 scale2 = make_float2(scale, scale), offset2 = make_float2(offset, offset);
                    if (!free) ok = ok && mbar_wait(p_bar, p_phase, abort_flag, 0x9b);
                    tc_fence_after();
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        uint32_t w[16];
                        float2 e[16];
#pragma unroll
                        for (int j = 0; j < 16; ++j)
                            e[j] = fma2(make_float2(__uint_as_float(s[c][2 * j]), __uint_as_float(s[c][2 * j + 1])), scale2, offset2);
#pragma unroll
                        for (int j = 0; j < 16; ++j) e[j] = make_float2(exp2_fast(e[j].x), exp2_fast(e[j].y));
#pragma unroll
                        for (int j = 0; j < 16; ++j) w[j] = pack2<T>(e[j].x, e[j].y);
                        tmem_st_32x16(p_addr + c * 16, w);
#pragma unroll
                        for (int k = 8; k > 0; k >>= 1) {
#pragma unroll
                            for (int j = 0; j < k; ++j) e[j] = add2(e[j], e[j + k]);
                        }
                        sum2 = add2(sum2, e[0]);
                    }
                    start += stride;
                    if (--sink_steps == 0) start += gap;
                    valid_at = (valid_at + valid_stride) % (kValid * 16);
                    if (turns && (group == 0 || n + 1 < steps)) turn_over(9 - 4 * group + quarter);
                    tmem_st_wait();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&tail->p_full[group][odd]));
                }
                ok = ok && mbar_wait(smem_u32(&tail->o_done[group][(done - 1) & 1]), ((done - 1) >> 1) & 1, abort_flag, 0x9a);
                if (steps > far_from) {
                    tc_fence_after();
                    far_sums(scratch, far_row, tmem_base + lanes + S::kO + group * 128, ksteps, base, scale, false, true);
                }
            }
            float sum = sum2.x + sum2.y, keep[2] = {1.0f, 0.0f};
            const int first = shared ? 0 : group;
            const bool other = shared && it.steps > 1;  // the second group has sums, too
            if (shared) {
                tail->sum[group][my_lane] = sum;
                tail->base[group][my_lane] = base;
                tc_fence_before();
                meet();  // both groups' products are done, too
                const float base0 = tail->base[0][my_lane], base1 = tail->base[1][my_lane];
                base = fmaxf(base0, base1);
                keep[0] = exp2_fast(base == -INFINITY ? 0.0f : (base0 - base) * scale);
                if (other) keep[1] = exp2_fast(base == -INFINITY ? 0.0f : (base1 - base) * scale);
                sum = tail->sum[0][my_lane] * keep[0];
                if (other) sum = fmaf(tail->sum[1][my_lane], keep[1], sum);
            }
            tc_fence_after();
            const bool mine = row0 + lane < rows;
            const float top = fmaf(base, scale, -kLift<T>);  // the sums are 2^kLift times those of exp(score - base)
            int head;
            const int64_t token = token_of(p, it, row0 + lane, &head);
            const int64_t out_row = (it.tokens.first + token) * p.heads + it.kvh * p.group + head;
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
            float2 zeros = make_float2(0.0f, 0.0f);  // or NaN, if any of O is not finite
            // 32 columns of O at a time; two groups that share the rows take turns
            for (int c = shared ? 2 * group : 0; c < ksteps; c += shared ? 4 : 2) {
                uint32_t o[32];
                const uint32_t addr = tmem_base + lanes + S::kO + first * 128 + c * 16;
                const int halves = c + 1 < ksteps ? 2 : 1;
#pragma unroll
                for (int j = 0; j < 32; ++j) o[j] = 0;
                if (it.steps > 0) {
                    tmem_ld_32x32(addr, o);
                    tmem_ld_wait();
                    if (other) {
                        uint32_t o1[32];
                        tmem_ld_32x32(addr + 128, o1);
                        tmem_ld_wait();
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            o[j] = __float_as_uint(fmaf(__uint_as_float(o1[j]), keep[1], __uint_as_float(o[j]) * keep[0]));
                    }
                }
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    if (half == halves) break;
                    const uint32_t *x = o + 16 * half;
                    const int column = c * 16 + 16 * half;
                    if (it.cut) {
                        if (mine && it.steps > 0) {
                            float *dst = scratch.part + (static_cast<int64_t>(it.split) * p.tokens * p.heads + out_row) * p.dim + column;
                            store_32(dst, x);
                            if (column + 8 < p.dim) store_32(dst + 8, x + 8);
                        }
                    } else {
                        uint32_t w[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const float2 a = make_float2(__uint_as_float(x[2 * j]), __uint_as_float(x[2 * j + 1]));
                            zeros = fma2(a, make_float2(0.0f, 0.0f), zeros);
                            const float2 y = mul2(a, make_float2(inv, inv));
                            w[j] = pack2<T>(y.x, y.y);
                        }
                        if (mine) {
                            T *dst = static_cast<T *>(p.out) + out_row * p.dim + column;
                            if (column + 8 < p.dim)
                                store_32(dst, w);
                            else
                                *reinterpret_cast<uint4 *>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
                        }
                    }
                }
                __syncwarp();
            }
            if (mine && group == first) {
                if (it.cut)
                    scratch.stat[static_cast<int64_t>(it.split) * p.tokens * p.heads + out_row] = make_float2(top, sum);
                else
                    p.lse[out_row] = sum == 0.0f ? -INFINITY : top * kLn2 + logf(sum);
            }
            // rows that are not finite although their weights are; O may be written again when all that share it have read it
            uint32_t again = __ballot_sync(0xffffffffu, mine && zeros.x + zeros.y != 0.0f && sum == sum);
            tc_fence_before();
            if (shared) {
                if (lane == 0) tail->bad[group][quarter] = again;
                __syncwarp();
                meet();
                again = group == 0 ? tail->bad[0][quarter] | tail->bad[1][quarter] : 0;
            }
            if (steps > 0 && lane == 0) mbar_arrive(smem_u32(&tail->o_free[group]));
            // Are they so by values that they do not see, they are made again, but not here: the other warps' waits are limited, and a
            // row takes as long as its places ask for.  (This looks at some 1200 places at most.)
            if (again != 0 && !met_not_finite<T>(p, it, place_of(p, it, row0), place_of(p, it, min(row0 + 31, rows - 1)))) again = 0;
            if (lane == 0) {
                tail->again[item & 1][group][quarter] = again;
                if (again != 0) tail->remake = 1;
            }
            count += it.end - it.begin;
            release(item);
        }
    }

    tc_fence_before();
    __syncthreads();
    if (threadIdx.x == 0 && tail->abort_flag != 0 && scratch.status != nullptr) atomicMax(scratch.status, tail->abort_flag);
    if (threadIdx.x == 0 && tail->far >= 0) {
        __threadfence();
        atomicExch(scratch.far_taken + tail->far, 0);
    }
    if (warp == kSoftmax) {
        tc_fence_after();
        tmem_dealloc(tmem_base, 512);
    }
    if (tail->remake == 0 || *abort_flag != 0) return;
    // ---------------- rows that came beside values that are not finite, again, when no warp waits for another ----------------
    // The CTA's last two items (no further one is taken once one has such rows).
    for (int i = 0; i < 16; ++i) {
        const uint32_t again = tail->again[i >> 3][i >> 2 & 1][i & 3];
        if (again != 0) remake_rows<T>(p, tail->item[i >> 3], (i >> 2 & 1) * 128 + (i & 3) * 32, again, reinterpret_cast<float *>(smem));
    }
}

// Joins the splits of a row, in their order: a warp a row.
template <typename T, int BN, int ROWS>
__global__ void __launch_bounds__(256) prompt_join_kernel(const __grid_constant__ Problem p, const __grid_constant__ Scratch scratch) {
    __shared__ __align__(16) float s_query[8][kPlainDim];
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5), rows = p.tokens * p.heads;
    const int splits = *scratch.pieces;
    if (row >= rows || splits == 1) return;
    float top = -INFINITY;
    for (int i = lane; i < splits; i += 32) top = fmaxf(top, scratch.stat[i * rows + row].x);
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float base = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f, acc[8] = {};
    for (int i0 = 0; i0 < splits; i0 += 32) {
        float weight = 0.0f;
        bool any = false;
        if (i0 + lane < splits) {
            const float2 st = scratch.stat[(i0 + lane) * rows + row];
            weight = exp2_fast(st.x - base);
            sum = fmaf(st.y, weight, sum);
            any = st.y != 0.0f;  // a split without tiles has written no part
        }
        const uint32_t has = __ballot_sync(0xffffffffu, any);
#pragma unroll 4
        for (int i = 0; i < min(32, splits - i0); ++i) {
            const float w = __shfl_sync(0xffffffffu, weight, i);
            if (!(has >> i & 1)) continue;
            const float *src = scratch.part + ((i0 + i) * rows + row) * p.dim;
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
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    T *dst = static_cast<T *>(p.out) + row * p.dim;
    bool bad = false;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        const int d = c * 128 + lane * 4;
        if (d < p.dim)
            *reinterpret_cast<uint2 *>(dst + d) = make_uint2(pack2<T>(acc[4 * c] * inv, acc[4 * c + 1] * inv),
                                                             pack2<T>(acc[4 * c + 2] * inv, acc[4 * c + 3] * inv));
#pragma unroll
        for (int j = 0; j < 4; ++j) bad |= !(fabsf(acc[4 * c + j]) < INFINITY);
    }
    if (lane == 0) p.lse[row] = sum == 0.0f ? -INFINITY : top * kLn2 + logf(sum);
    if (__any_sync(0xffffffffu, bad) && sum == sum) {
        const int64_t token = row / p.heads;
        const int head = static_cast<int>(row - token * p.heads);
        Item it;
        it.kvh = head / p.group;
        for (it.b = 0; it.b < p.batch; ++it.b) {
            it.tokens = tokens_of(p, it.b);
            if (token >= it.tokens.first && token < it.tokens.first + it.tokens.count) break;
        }
        if (it.b == p.batch) return;
        it.rows = static_cast<int64_t>(it.tokens.count) * p.group;
        const int64_t at = (token - it.tokens.first) * p.group + head - it.kvh * p.group;
        it.first = at / ROWS * ROWS;
        cover<BN, ROWS>(p, it);
        const int place = place_of(p, it, static_cast<int>(at - it.first));
        if (met_not_finite<T>(p, it, place, place)) {
            RowPart r;
            stage_query<T>(p, token, head, s_query[threadIdx.x >> 5]);
            __syncwarp();
            rows_part<T, 1>(p, it.b, it.kvh, &place, s_query[threadIdx.x >> 5], 0, 1, &r);
            write_row<T>(p, token, head, r);
        }
    }
}

// A cache as TMA sees it: boxes of `rows` places of one page and head by 64 columns (zeros behind the head dimension).  False: its
// strides are none that TMA takes, cp.async loads it.
bool cache_map(CUtensorMap *map, const Problem &p, const void *base, int64_t sb, int64_t st, int64_t sh, int rows) {
    const int64_t sizes[4] = {p.dim, p.page, p.kv_heads, p.pages};
    int64_t strides[3] = {st, sh, sb};
    for (int i = 0; i < 3; ++i) {
        if (sizes[i + 1] == 1) strides[i] = p.dim;  // takes no step
        if (strides[i] <= 0 || strides[i] >= 1ll << 38) return false;
    }
    const int box[4] = {64, rows, 1, 1};
    return make_tmap_4d(map, base, sizes, strides, box);
}

// The query: columns, heads of a group, groups, tokens.
bool query_map(CUtensorMap *map, const Problem &p) {
    const int64_t sizes[4] = {p.dim, p.group, p.kv_heads, p.tokens};
    int64_t strides[3] = {p.q_sh, p.q_sh * p.group, p.q_st};
    for (int i = 0; i < 3; ++i) {
        if (sizes[i + 1] == 1) strides[i] = p.dim;  // takes no step
        if (strides[i] <= 0 || strides[i] >= 1ll << 38) return false;
    }
    const int box[4] = {64, p.group, 1, 128 / p.group};
    return make_tmap_4d(map, p.q, sizes, strides, box);
}

template <typename T, int DP>
int launch(const Problem &p, const Plan &plan, const Scratch &scratch, cudaStream_t stream) {
    const int64_t ctas = plan.pairs * p.kv_heads * plan.splits;
    if (ctas > 0x7fffffff) return fail(QMM_ERR_UNSUPPORTED, "qmm_paged_prompt_attention: too many tokens");
    QMM_CUDA_OK(cudaFuncSetAttribute(prompt_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem_bytes<DP>())));
    CUtensorMap tmap_k = {}, tmap_v = {};
    // as many places a box as begin together in any page and any tile
    int box_rows = 8;
    while (2 * box_rows <= Shape<DP>::kBN && p.page % (2 * box_rows) == 0) box_rows *= 2;
    if (p.page % 8 != 0 || p.pages == 0 || !cache_map(&tmap_k, p, p.k, p.k_sb, p.k_st, p.k_sh, box_rows) ||
        !cache_map(&tmap_v, p, p.v, p.v_sb, p.v_st, p.v_sh, box_rows))
        box_rows = 0;
    // the query's rows of a tile in one box, where the group's heads divide a tile
    CUtensorMap tmap_q = {};
    const bool box_query = 128 % p.group == 0 && query_map(&tmap_q, p);
    if (plan.far) QMM_CUDA_OK(cudaMemsetAsync(scratch.far_taken, 0, plan.taken_bytes, stream));
    QMM_CUDA_OK(launch_pdl_if(!plan.far, prompt_kernel<T, DP>, dim3(static_cast<unsigned>(ctas > 0 ? ctas : 1)), dim3(kThreads), smem_bytes<DP>(), stream, p, scratch,
                           tmap_k, tmap_v, tmap_q, box_rows, box_query));
    if (plan.splits > 1) {
        const int64_t joins = (p.tokens * p.heads + 7) / 8;
        QMM_CUDA_OK(launch_pdl(prompt_join_kernel<T, Shape<DP>::kBN, Shape<DP>::kRows>, dim3(static_cast<unsigned>(joins)), dim3(256), 0, stream, p, scratch));
    }
    return QMM_OK;
}

template <typename T>
int launch_t(const Problem &p, const Plan &plan, const Scratch &scratch, cudaStream_t stream) {
    if (p.dim <= 64) return launch<T, 64>(p, plan, scratch, stream);
    if (p.dim <= 128) return launch<T, 128>(p, plan, scratch, stream);
    return launch<T, 256>(p, plan, scratch, stream);
}

}  // namespace

size_t prompt_workspace(int64_t tokens, int64_t batch, int64_t heads, int64_t kv_heads, int64_t dim, int64_t places) {
    return tokens == 0 || heads == 0 ? 0 : make_plan(tokens, batch, heads, kv_heads, dim, places).bytes;
}

int launch_prompt(const Problem &p, int dtype, void *workspace, size_t workspace_bytes, cudaStream_t stream) {
    const int64_t places = static_cast<int64_t>(p.max_pages) * p.page;
    Plan plan = make_plan(p.tokens, p.batch, p.heads, p.kv_heads, p.dim, places);
    if (p.window > 0) {
        // an item's rows see the window of the first and a place for each further token; the workspace is for no window
        const Plan narrow = make_plan(p.tokens, p.batch, p.heads, p.kv_heads, p.dim,
                                      std::min(places, static_cast<int64_t>(p.window) + p.sinks + 256 / std::min(p.group, 256)));
        if (narrow.splits < plan.splits || (narrow.splits == plan.splits && !narrow.far)) plan = narrow;
    }
    if (plan.bytes > 0 && (workspace_bytes < plan.bytes || workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 15) != 0))
        return fail(QMM_ERR_WORKSPACE, "qmm_paged_prompt_attention: needs a workspace of " + std::to_string(plan.bytes) + " bytes, 16-byte aligned");
    Scratch scratch;
    uint8_t *base = static_cast<uint8_t *>(workspace);
    scratch.far = reinterpret_cast<float *>(base);
    scratch.far_taken = reinterpret_cast<int *>(base + plan.far_bytes);
    scratch.far_places = plan.far ? sm_count() : 0;
    scratch.far_stride = far_stride(p.dim);
    base += plan.far_bytes + plan.taken_bytes;
    scratch.part = reinterpret_cast<float *>(base);
    scratch.stat = reinterpret_cast<float2 *>(base + plan.part_bytes);
    scratch.pieces = reinterpret_cast<int *>(base + plan.part_bytes + plan.stat_bytes);
    scratch.splits = plan.splits;
    scratch.sms = sm_count();
    scratch.tile = static_cast<float>(plan.tile);
    scratch.status = device_status_word();
    return dtype == QMM_DTYPE_BF16 ? launch_t<__nv_bfloat16>(p, plan, scratch, stream) : launch_t<__half>(p, plan, scratch, stream);
}

}  // namespace paged
}  // namespace qmm
