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
#include "paged_decode.cuh"

namespace qmm {
namespace paged {

namespace {

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

Plan make_plan(int64_t batch, int64_t heads, int64_t kv_heads, int64_t dim) {
    return make_plan(batch, heads, kv_heads, dim, 2, dim > 128 ? Shape<256>::kWarps : Shape<128>::kWarps);
}

// Powers of two by which weights are larger than exp(score - maximum) until the log-sum: f16 has no full step below 2^-14 and
// nothing below 2^-25, so a weight of 1 for the largest score would lose the many keys of a long cache that lie 2^-25 and more
// below one that stands out; with 2^15 what is lost lies 2^-40 below it.  bf16 has the exponents of fp32.
template <typename T>
constexpr float kLift = std::is_same<T, __half>::value ? 15.0f : 0.0f;

// FAR: a warp may have more than kNear places.
template <typename T, int DP, bool FAR>
__global__ void __launch_bounds__(Shape<DP>::kWarps * 32, 2)
decode_kernel(const __grid_constant__ Problem p, const __grid_constant__ Scratch scratch) {
    using S = Shape<DP>;
    constexpr int KEYS = S::kKeys;
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
int launch_decode_kernel(const Problem &p, const Plan &plan, const Scratch &scratch, cudaStream_t stream) {
    QMM_CUDA_OK(cudaFuncSetAttribute(decode_kernel<T, DP, FAR>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(Shape<DP>::kSmem)));
    QMM_CUDA_OK(launch_pdl(decode_kernel<T, DP, FAR>, dim3(plan.workers), dim3(Shape<DP>::kWarps * 32), Shape<DP>::kSmem, stream, p, scratch));
    return QMM_OK;
}

template <typename T, int DP>
int launch(const Problem &p, const Plan &plan, const Scratch &scratch, cudaStream_t stream) {
    const bool far = is_far(p, plan, Shape<DP>::kWarps);
    const int rc = far ? launch_decode_kernel<T, DP, true>(p, plan, scratch, stream) : launch_decode_kernel<T, DP, false>(p, plan, scratch, stream);
    return rc != QMM_OK ? rc : launch_join<T>(p, plan, scratch, stream);
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
    const Scratch scratch = lay_out(plan, workspace);
    return dtype == QMM_DTYPE_BF16 ? launch_t<__nv_bfloat16>(p, plan, scratch, stream) : launch_t<__half>(p, plan, scratch, stream);
}

}  // namespace paged
}  // namespace qmm
