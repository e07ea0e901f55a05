// Differential prefill: the launch plan, and the joining of blocks that several
// slices computed (work division: diff_prefill_plan.hpp).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../pool.hpp"
#include "diff_prefill.hpp"

namespace airkv {
namespace {

// Rows of one cut block, one wave: their pieces folded by log-sum-exp, in order.  HALF:
// the 16-bit products' blocks, four rows at once (mostly of two pieces); the smaller
// launches at f32 precision take one (four prompts: 30.4 us in all, 31.8 with four).
constexpr int merge_rows(bool half) { return half ? 4 : 1; }
template <int D, bool HALF>
__global__ __launch_bounds__(256) void diff_prefill_merge_kernel(DiffPrefillArgs a) {
    constexpr int V = D / 32, N = merge_rows(HALF), kBatch = HALF ? 2 : 4;
    const int w = blockIdx.y, kp = blockIdx.z, lane = threadIdx.x & 63;
    const int row = (blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * N;
    const int64_t at = (int64_t)kp * a.slices + w;
    const int4 d = a.desc[at];
    if (d.w == 0) return;
    // rows past the sequence's last are read as they are (slots are whole) and not written
    float2 ml[N][kBatch][2];
    float po[N][kBatch][2][V];
    auto load = [&](int p0) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < N; ++j)
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                const int p = p0 + i < d.w ? p0 + i : p0;
                const int64_t slot = 2 * (at + p) + (p == 0 ? 1 : 0);
#pragma unroll
                for (int m = 0; m < 2; ++m) {
                    const int64_t r = (slot * a.rows + row + j) * 2 + m;
                    ml[j][i][m] = *reinterpret_cast<const float2 *>(a.part_ml + 2 * r);
                    diff_load<V>(a.part_o + r * (2 * D) + V * lane, po[j][i][m]);
                }
            }
    };
    load(0);                                           // before what the rows' places wait for
    const int64_t k = (int64_t)((uint64_t)(uint32_t)d.y | (uint64_t)(uint32_t)d.z << 32);
    const int64_t r0 = a.cu[d.x], f = k * a.rows + row, rows = (a.cu[d.x + 1] - r0) * a.group;
    if (f >= rows) return;
    const int n = rows - f < N ? (int)(rows - f) : N;
    const bool narrow = f >> 32 == 0;                  // (a fifth of the instructions)
    const int64_t tok = narrow ? (int64_t)((uint32_t)f / (uint32_t)a.group) : f / a.group;
    const int pair = (int)(f - tok * a.group);
    DiffTail<V> tail[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const int x = pair + j, more = x / a.group;
        tail[j].load(a.e, j < n ? r0 + tok + more : r0 + tok, kp * a.group + (j < n ? x - more * a.group : pair), lane);
    }
    DiffFold<V> c[N];
#pragma unroll
    for (int j = 0; j < N; ++j) c[j].clear();
    for (int p0 = 0; p0 < d.w; p0 += kBatch) {
        if (p0) load(p0);
#pragma unroll
        for (int j = 0; j < N; ++j)
#pragma unroll
            for (int i = 0; i < kBatch; ++i)
#pragma unroll
                for (int m = 0; m < 2; ++m) {
                    if (p0 + i < d.w) c[j].fold(m, ml[j][i][m].x, ml[j][i][m].y, po[j][i][m]);
                }
    }
#pragma unroll
    for (int j = 0; j < N; ++j)
        if (j < n) diff_finish<V>(a.e, a.pairs, c[j], tail[j], lane);
}

template <bool HALF> hipError_t launch_merge(const DiffPrefillArgs &a, int head_dim, hipStream_t s) {
    if (a.slices < 2) return hipSuccess;               // nothing is cut
    // the rows of a block run together: its slots, powers of two apart, share their memory channels
    const dim3 grid((unsigned)(a.rows / (4 * merge_rows(HALF))), (unsigned)a.slices, (unsigned)a.kv_pairs);
    if (head_dim == 128) hipLaunchKernelGGL((diff_prefill_merge_kernel<128, HALF>), grid, dim3(256), 0, s, a);
    else if (head_dim == 96) hipLaunchKernelGGL((diff_prefill_merge_kernel<96, HALF>), grid, dim3(256), 0, s, a);
    else if (head_dim == 64) hipLaunchKernelGGL((diff_prefill_merge_kernel<64, HALF>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((diff_prefill_merge_kernel<32, HALF>), grid, dim3(256), 0, s, a);
    return hipGetLastError();
}

size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }

// Slices per K/V pair: the CUs' share, rounded up; one workgroup is resident on a CU.  Where
// the pairs do not divide the CUs, the few workgroups past them start when the others end
// (8192 tokens: 466 TFLOP/s with 4 pairs, 270 to 290 with 3, 5, 6, 7 or 10).
struct Plan {
    int32_t rows, extra, slices, least;
    size_t cells, halves;          // (pair, slice)s, rows' maps in the piece slots
    size_t bytes(int d) const { return align256(cells * sizeof(int4)) + align256(halves * 2 * 4) + halves * 2 * d * 4; }
};

// half: 16-bit products (diff_prefill_16.hip), else f32 ones
Plan plan_for(const air_kv_pool &p, bool half) {
    Plan pl;
    const int kv_pairs = p.desc.n_kv_heads / 2;
    pl.rows = half ? 128 : 64;
    // what a block's beginning and end cost beside a tile (4 and 1: 399 us for eight chunks and
    // 382 us for 2048 tokens at f32 precision, 362 and 364 so), and the smallest piece of one
    // that is worth its joining (at f32 precision 6, 4, 3, 2: 44, 38, 35, 37 us for four prompts)
    pl.extra = half ? 7 : 2;
    pl.slices = std::max(1, (p.cus + kv_pairs - 1) / kv_pairs);
    pl.least = half ? 16 : 3;
    pl.cells = (size_t)kv_pairs * pl.slices;
    pl.halves = 2 * pl.cells * pl.rows * 2;
    return pl;
}

}  // namespace

size_t diff_prefill_workspace(const air_kv_pool &p) {
    return std::max(plan_for(p, false).bytes(p.desc.head_dim), plan_for(p, true).bytes(p.desc.head_dim));
}

hipError_t launch_diff_prefill(const air_kv_pool &p, hipStream_t s, const void *q, int32_t q_dtype, int32_t n_q_heads,
                               const int32_t *cu, int32_t total_q, const int32_t *tables, const int32_t *lens,
                               int32_t batch, int32_t max_blocks, float scale, const DiffOut &out, void *workspace) {
    const bool half = p.desc.dtype != AIR_KV_F32 && q_dtype == AIR_KV_BF16 && out.out_dtype == AIR_KV_BF16;
    const Plan plan = plan_for(p, half);
    const int d = p.desc.head_dim;
    DiffPrefillArgs a{};
    a.q = q;
    a.q_dtype = q_dtype;
    a.pairs = n_q_heads / 2;
    a.total_q = total_q;
    a.max_blocks = max_blocks;
    a.scale_log2 = scale * 1.4426950408889634f;
    a.kv_pairs = p.desc.n_kv_heads / 2;
    a.group = n_q_heads / p.desc.n_kv_heads;
    a.heads = p.desc.n_kv_heads;
    a.bs = p.desc.block_size;
    a.dtype = p.desc.dtype;
    a.scale_group = p.desc.scale_group;
    a.num_blocks = p.desc.num_blocks;
    a.k_pages = p.k_pages;
    a.v_pages = p.v_pages;
    a.k_scales = p.k_scales;
    a.v_scales = p.v_scales;
    a.errors = p.errors;
    a.e = out;
    a.slices = plan.slices;
    a.least = plan.least;
    a.rows = plan.rows;
    a.extra = plan.extra;
    char *ws = (char *)workspace;
    a.desc = (int4 *)ws;
    ws += align256(plan.cells * sizeof(int4));
    a.part_ml = (float *)ws;
    ws += align256(plan.halves * 2 * 4);
    a.part_o = (float *)ws;
    for (int32_t b0 = 0; b0 < batch; b0 += kDiffPrefillBatch) {
        a.batch = std::min(batch - b0, kDiffPrefillBatch);
        a.cu = cu + b0;
        a.tables = tables + (int64_t)b0 * max_blocks;
        a.lens = lens + b0;
        hipError_t e = half ? launch_diff_prefill_16(a, d, s) : launch_diff_prefill_f32(a, d, s);
        if (e == hipSuccess) e = half ? launch_merge<true>(a, d, s) : launch_merge<false>(a, d, s);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace airkv
