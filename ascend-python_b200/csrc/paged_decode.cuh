// What the decode kernels over a paged cache share (paged_decode.cu: 16-bit caches, paged_quant_decode.cu: 8-bit ones): what a token
// sees as tiles, where parts of head tiles that are cut lie, and instructions.
#pragma once

#include <algorithm>
#include <type_traits>

#include "paged_common.cuh"

namespace qmm {
namespace paged {

namespace {

constexpr int kRows = 16;     // query heads of a tile
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
// What a warp has of one head tile: tiles [from, to) of sequence b's item.
struct Piece {
    int64_t at;  // where the piece begins in the list
    int b, item, from, to;
    Sequence s;
};

__device__ __forceinline__ void cp_async_16(uint32_t dst, const void *src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
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

}  // namespace

}  // namespace paged
}  // namespace qmm
