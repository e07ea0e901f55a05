// Cross attention over pages: launch parameters and the work division.
//
// Every row (a sequence's token and one of the query heads of a K/V head) attends to all of the
// sequence's cached tokens:
//   s[t] = scale * q . K[t],  out = sum_t exp(s[t] - max s) V[t] / sum_t exp(s[t] - max s)
// A sequence's rows at one K/V head (token after token, query head after query head) are cut
// into blocks, a block's keys into tiles.  A block counts as `extra` units (what its
// beginning and end cost beside a tile) and one for each tile; the K/V head's units, sequence
// after sequence, block after block, are cut into equal slices, one workgroup each.  A block
// that several slices hold is joined by a second kernel, piece after piece in order.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../pool.hpp"

namespace airkv {

constexpr int kCrossBatch = 512;       // sequences per launch (the host splits larger batches)
// what a block's beginning and end cost beside a tile (many rows, 16-bit: 1, 3, 6: 279, 269, 267 us
// for int8 chunks, 93, 91, 92 for small heads; few rows: 111, 114, 113)
constexpr int cross_extra(bool few) { return few ? 1 : 3; }

struct CrossArgs {
    const void *q;                     // [total_q][q_heads][head_dim]
    void *out;
    int32_t q_dtype, out_dtype, q_heads, group;
    const int32_t *cu, *tables, *lens;
    int32_t batch, max_blocks, total_q;
    float scale_log2;
    int32_t heads, bs_log2, sg_log2, dtype;
    int64_t num_blocks;
    const void *k_pages, *v_pages;
    const float *k_scales, *v_scales;
    unsigned long long *errors;
    int32_t slices;                    // per K/V head
    // cut blocks: per (K/V head, slice) the block it begins and does not end, {sequence, block,
    // pieces}; two piece slots each, 2w for a block begun before and 2w + 1 for one that goes
    // on: [slot][row] of (base, sum, the sums' unit), and of head_dim sums
    int4 *desc;
    float4 *part_ml;
    float *part_o;
};

// One sequence of the launch.  ok: its rows lie in [0, total_q] and its length in its table.
struct CrossSeq {
    int32_t row0, rows, len;           // first of q's rows, (token, query head)s at one K/V head, cached tokens
    bool ok;
};
__device__ __forceinline__ CrossSeq cross_seq(const CrossArgs &a, int b) {
    const int32_t r0 = a.cu[b], r1 = a.cu[b + 1], len = a.lens[b];
    CrossSeq s;
    s.ok = r0 >= 0 && r1 >= r0 && r1 <= a.total_q && len >= 0 && len <= (int64_t)a.max_blocks << a.bs_log2;
    s.row0 = r0;
    s.rows = s.ok ? (r1 - r0) * a.group : 0;           // (the host bounds total_q * group)
    s.len = s.ok ? len : 0;
    return s;
}

// ROWS rows a block, TK keys a tile.
template <int TK> __device__ __forceinline__ int32_t cross_tiles(const CrossSeq &s) { return (int32_t)(((int64_t)s.len + TK - 1) / TK); }
template <int ROWS, int TK, int EXTRA> __device__ __forceinline__ int64_t cross_units(const CrossSeq &s) {
    const int64_t tiles = cross_tiles<TK>(s);
    return tiles ? ((int64_t)s.rows + ROWS - 1) / ROWS * (tiles + EXTRA) : 0;
}

// Rows of a block, workgroups that are resident on a CU, and whether a block's waves share its
// rows (asked for with `few`, and so where LDS has room for keys of each wave's own).
struct CrossBlocks {
    int rows, groups;
    bool few;
};
CrossBlocks cross_blocks_16(int head_dim, bool codes, bool few);
CrossBlocks cross_blocks_f32(int head_dim, bool wide, bool few);
hipError_t launch_cross_16(const CrossArgs &a, int head_dim, bool few, hipStream_t s);
hipError_t launch_cross_f32(const CrossArgs &a, int head_dim, bool few, hipStream_t s);

}  // namespace airkv
