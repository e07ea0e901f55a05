// Launch parameters and the work division of the differential prefill kernels.
#pragma once

#include "diff_common.hpp"
#include "diff_prefill_plan.hpp"

namespace airkv {

constexpr int kDiffPrefillBatch = 1024;    // sequences per launch (the host splits larger batches)

struct DiffPrefillArgs {
    const void *q;                 // [total_q][query heads][head_dim]
    int32_t q_dtype, pairs;        // query pairs
    const int32_t *cu, *tables, *lens;
    int32_t batch, max_blocks, total_q;
    float scale_log2;
    int32_t kv_pairs, group, heads, bs, dtype, scale_group;
    int64_t num_blocks;
    const void *k_pages, *v_pages;
    const float *k_scales, *v_scales;
    unsigned long long *errors;
    DiffOut e;
    int32_t slices;                // per K/V pair
    int32_t least;                 // units a slice holds at least
    int32_t rows, extra;           // of a block; the units it counts beside its tiles
    // cut blocks: per (pair, slice) the block it began and did not end, {sequence,
    // block (low, high), pieces}; two piece slots per (pair, slice), 2w for a block
    // begun before, 2w + 1 for one that goes on: [slot][row][map] of (max, sum), and
    // of 2 * head_dim sums
    int4 *desc;
    float *part_ml, *part_o;
};

// x, the same in every lane of the wave, in scalar registers.
__device__ __forceinline__ int64_t diff_uniform(int64_t x) {
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)x), hi = __builtin_amdgcn_readfirstlane((uint32_t)(x >> 32));
    return (int64_t)((uint64_t)hi << 32 | lo);
}

// What a row of the work list needs, for the workgroup's present block.
struct DiffItem {
    int32_t b;
    int64_t k;                     // block
    int64_t from;                  // of its units, the first
};

// Where the 16-byte chunk c of row r of a staged head of 16-bit keys lies, in chunks: 16
// rows' chunks c are read at once, and have to lie in 16 different 16-byte columns of the
// 256 bytes that the banks span.
template <int D> __device__ __forceinline__ int key_chunk(int r, int c) {
    if constexpr (D == 128) return c ^ (r & 15);
    else if constexpr (D == 64) return c ^ ((r >> 1) & 7);
    else if constexpr (D == 32) return c ^ ((r >> 2) & 3);
    else return (c + ((r >> 2) & 3)) % 12;
}

// The launch's units before each sequence (s_pre[B] in all) and each sequence's
// share of errors, in LDS.  A sequence whose rows do not lie in [0, total_q], whose
// length is outside its table or below its rows, has none; the workgroup of slice b
// % slices of pair 0 counts it and zeroes its rows.
__device__ __forceinline__ bool diff_seq(const DiffPrefillArgs &a, int b, DiffBlocks &s) {
    const int64_t r0 = a.cu[b], r1 = a.cu[b + 1], len = a.lens[b];
    s.g = a.group;
    s.rows = a.rows;
    s.extra = a.extra;
    s.q = r1 - r0;
    s.prefix = len - s.q;
    const bool ok = r0 >= 0 && r1 >= r0 && r1 <= a.total_q && len >= 0 && len <= (int64_t)a.max_blocks * a.bs && s.q <= len;
    if (!ok) s.q = s.prefix = 0;
    return ok;
}

// All THREADS threads take part.
template <int THREADS>
__device__ __forceinline__ void diff_units(const DiffPrefillArgs &a, int64_t *s_pre, int64_t (&s_sum)[THREADS / 64]) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, B = a.batch;
    const int per = (B + THREADS - 1) / THREADS, lo = tid * per, hi = lo + per < B ? lo + per : B;
    int64_t mine = 0;
    for (int b = lo; b < hi; ++b) {
        DiffBlocks s;
        diff_seq(a, b, s);
        const int64_t u = s.units();
        s_pre[b + 1] = u;
        mine += u;
    }
    int64_t incl = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int64_t y = __shfl_up(incl, o);
        if (lane >= o) incl += y;
    }
    if (lane == 63) s_sum[wave] = incl;
    if (tid == 0) s_pre[0] = 0;
    __syncthreads();
    int64_t run = incl - mine;
    for (int w = 0; w < wave; ++w) run += s_sum[w];
    for (int b = lo; b < hi; ++b) {
        run += s_pre[b + 1];
        s_pre[b + 1] = run;
    }
    __syncthreads();
}

// The block of unit u (below s_pre[B]) and its place there; the wave's lanes probe 64 blocks
// at a time.  Every wave finds the same.
__device__ __forceinline__ void diff_find(const DiffPrefillArgs &a, const int64_t *s_pre, int64_t u, DiffItem &it) {
    int lo = 0, hi = a.batch;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s_pre[mid] <= u) lo = mid;
        else hi = mid;
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    DiffBlocks s;
    diff_seq(a, lo, s);
    const int64_t at = u - diff_uniform(s_pre[lo]);
    int64_t k0 = 0, k1 = s.blocks();               // before(k0) <= at, and the block is in [k0, k1)
    const int lane = threadIdx.x & 63;
    while (k1 - k0 > 1) {
        const int64_t step = (k1 - k0 + 63) / 64;
        const int64_t k = k0 + lane * step;
        const bool le = k < k1 && s.before(k) <= at;
        const int n = __popcll(__ballot(le));      // lanes 0 .. n - 1 (before grows with k)
        k0 += (int64_t)(n - 1) * step;
        k1 = k0 + step < k1 ? k0 + step : k1;
    }
    it.b = lo;
    it.k = diff_uniform(k0);
    it.from = diff_uniform(at - s.before(it.k));
}

// The block after: of the same sequence, or the first of the next that has one.
__device__ __forceinline__ void diff_next(const DiffPrefillArgs &a, const int64_t *s_pre, const DiffBlocks &s, DiffItem &it) {
    it.from = 0;
    if (++it.k < s.blocks()) return;
    it.k = 0;
    do ++it.b;
    while (it.b < a.batch && diff_uniform(s_pre[it.b + 1]) == diff_uniform(s_pre[it.b]));
}

// Sequences that are refused: counted, and their rows (those there are) zeroed.
__device__ __forceinline__ void diff_refused(const DiffPrefillArgs &a, int cols) {
    const int pair = blockIdx.y;
    for (int b = blockIdx.x; b < a.batch; b += gridDim.x) {
        DiffBlocks s;
        if (diff_seq(a, b, s)) continue;
        if (pair == 0 && threadIdx.x == 0) atomicAdd(a.errors, 1ull);
        const int64_t r0 = a.cu[b], r1 = a.cu[b + 1];
        if (r0 < 0 || r1 > a.total_q || r1 < r0) continue;
        const int64_t n = (r1 - r0) * a.group * cols;
        for (int64_t i = threadIdx.x; i < n; i += blockDim.x) {
            const int64_t r = r0 + i / (a.group * cols), c = i % (a.group * cols);
            diff_store(a.e, (r * a.pairs + pair * a.group) * cols + c, 0.0f);
        }
    }
}

// Bytes of the largest workspace a call over this pool needs.
size_t diff_prefill_workspace(const air_kv_pool &p);
hipError_t launch_diff_prefill(const air_kv_pool &p, hipStream_t s, const void *q, int32_t q_dtype, int32_t n_q_heads,
                               const int32_t *cu, int32_t total_q, const int32_t *tables, const int32_t *lens,
                               int32_t batch, int32_t max_blocks, float scale, const DiffOut &out, void *workspace);
hipError_t launch_diff_prefill_f32(const DiffPrefillArgs &a, int head_dim, hipStream_t s);
hipError_t launch_diff_prefill_16(const DiffPrefillArgs &a, int head_dim, hipStream_t s);

}  // namespace airkv
