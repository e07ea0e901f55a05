// Cross attention over pages: the launch plan, and the joining of blocks that several slices
// computed (paged_cross.hpp).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "codecs.hpp"
#include "paged_cross.hpp"

namespace airkv {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr int kMergeThreads = 256;

// The rows of one cut block: a row's pieces folded in order, four columns a lane.
template <int LANES>
__global__ __launch_bounds__(kMergeThreads) void cross_merge_kernel(CrossArgs a, int rows, int d) {
    const int64_t cell = (int64_t)blockIdx.z * a.slices + blockIdx.y;
    const int4 it = a.desc[cell];
    if (it.z == 0) return;
    const int r = blockIdx.x * (kMergeThreads / LANES) + threadIdx.x / LANES, col = threadIdx.x % LANES * 4;
    const int32_t r0 = a.cu[it.x];
    const int32_t row = it.y * rows + r;
    if (row >= (a.cu[it.x + 1] - r0) * a.group || col >= d) return;
    // the mean of the values so far, its weight l under `base` (a mean stays within its values' range,
    // where a sum of values near the largest or the smallest floats would not)
    float base = -INFINITY, l = 0.0f;
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    constexpr int kBatch = 4;
    for (int p0 = 0; p0 < it.z; p0 += kBatch) {
        float4 ml[kBatch];
        f32x4 x[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int p = p0 + i < it.z ? p0 + i : p0;
            const int64_t at = (2 * (cell + p) + (p == 0 ? 1 : 0)) * rows + r;
            ml[i] = a.part_ml[at];
            x[i] = *reinterpret_cast<const f32x4 *>(a.part_o + at * d + col);
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            // (a piece without a key in the pool has sum 0)
            if (p0 + i >= it.z || ml[i].y == 0.0f) continue;
            const float top = fmaxf(base, ml[i].x);
            const float was = base == top ? l : l * __builtin_amdgcn_exp2f(base - top);
            const float is = ml[i].x == top ? 1.0f : __builtin_amdgcn_exp2f(ml[i].x - top);
            l = was + ml[i].y * is;
            const float k = 1.0f / l;
            o = o * (was * k) + x[i] * (is * k) * ml[i].z;
            base = top;
        }
    }
    const int64_t at = ((int64_t)(r0 + row / a.group) * a.q_heads + blockIdx.z * a.group + row % a.group) * d + col;
    if (a.out_dtype == AIR_KV_F32)
        *reinterpret_cast<f32x4 *>((float *)a.out + at) = o;
    else
        *reinterpret_cast<u32x2 *>((uint16_t *)a.out + at) = u32x2{(uint32_t)bf16_rne(o[0]) | ((uint32_t)bf16_rne(o[1]) << 16),
                                                                   (uint32_t)bf16_rne(o[2]) | ((uint32_t)bf16_rne(o[3]) << 16)};
}

hipError_t launch_merge(const CrossArgs &a, int rows, int d, hipStream_t s) {
    if (a.slices < 2) return hipSuccess;               // nothing is cut
    const int lanes = d <= 32 ? 8 : d <= 64 ? 16 : d <= 128 ? 32 : 64;
    const int per = kMergeThreads / lanes;
    const dim3 grid((unsigned)((rows + per - 1) / per), (unsigned)a.slices, (unsigned)a.heads);
    if (lanes == 8) hipLaunchKernelGGL(cross_merge_kernel<8>, grid, dim3(kMergeThreads), 0, s, a, rows, d);
    else if (lanes == 16) hipLaunchKernelGGL(cross_merge_kernel<16>, grid, dim3(kMergeThreads), 0, s, a, rows, d);
    else if (lanes == 32) hipLaunchKernelGGL(cross_merge_kernel<32>, grid, dim3(kMergeThreads), 0, s, a, rows, d);
    else hipLaunchKernelGGL(cross_merge_kernel<64>, grid, dim3(kMergeThreads), 0, s, a, rows, d);
    return hipGetLastError();
}

size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }

int rows_of(const air_kv_pool &p, bool half, bool few) {
    return half ? cross_rows_16(p.desc.head_dim, few) : cross_rows_f32(p.desc.head_dim, few, p.desc.dtype != AIR_KV_BF16);
}

// Slices per K/V head: the CUs' share; one workgroup is resident on a CU.
int slices_of(const air_kv_pool &p) { return std::max(1, p.cus / p.desc.n_kv_heads); }

size_t bytes_of(const air_kv_pool &p, int rows) {
    const size_t cells = (size_t)p.desc.n_kv_heads * slices_of(p), slots = 2 * cells * rows;
    return align256(cells * sizeof(int4)) + align256(slots * sizeof(float4)) + slots * p.desc.head_dim * 4;
}

}  // namespace

size_t cross_workspace(const air_kv_pool &p) {
    size_t most = 0;
    for (int half = 0; half < 2; ++half)
        for (int few = 0; few < 2; ++few)
            if (!half || p.desc.dtype != AIR_KV_F32) most = std::max(most, bytes_of(p, rows_of(p, half, few)));
    return most;
}

hipError_t launch_cross(const air_kv_pool &p, hipStream_t s, const void *q, int32_t q_dtype, int32_t n_q_heads, const int32_t *cu,
                        int32_t total_q, int32_t max_q_len, const int32_t *tables, const int32_t *lens, int32_t batch,
                        int32_t max_blocks, float scale, void *workspace, void *out, int32_t out_dtype) {
    const bool half = p.desc.dtype != AIR_KV_F32 && q_dtype == AIR_KV_BF16 && out_dtype == AIR_KV_BF16;
    const int d = p.desc.head_dim, group = n_q_heads / p.desc.n_kv_heads;
    const int64_t most = (int64_t)(max_q_len ? max_q_len : (total_q + batch - 1) / batch) * group;
    // rows of one wave: its keys go to the others
    const bool few = most <= 32;
    const int rows = rows_of(p, half, few);
    CrossArgs a{};
    a.q = q;
    a.out = out;
    a.q_dtype = q_dtype;
    a.out_dtype = out_dtype;
    a.q_heads = n_q_heads;
    a.group = group;
    a.max_blocks = max_blocks;
    a.total_q = total_q;
    a.scale_log2 = std::min(std::max(scale * 1.4426950408889634f, 0x1p-126f), 0x1.fffffep127f);
    a.heads = p.desc.n_kv_heads;
    a.bs_log2 = __builtin_ctz((unsigned)p.desc.block_size);
    a.sg_log2 = p.desc.scale_group > 0 ? __builtin_ctz((unsigned)p.desc.scale_group) : 0;
    a.dtype = p.desc.dtype;
    a.num_blocks = p.desc.num_blocks;
    a.k_pages = p.k_pages;
    a.v_pages = p.v_pages;
    a.k_scales = p.k_scales;
    a.v_scales = p.v_scales;
    a.errors = p.errors;
    a.slices = slices_of(p);
    a.least = 3;
    const size_t cells = (size_t)a.heads * a.slices, slots = 2 * cells * rows;
    char *ws = (char *)workspace;
    a.desc = (int4 *)ws;
    ws += align256(cells * sizeof(int4));
    a.part_ml = (float4 *)ws;
    ws += align256(slots * sizeof(float4));
    a.part_o = (float *)ws;
    for (int32_t b0 = 0; b0 < batch; b0 += kCrossBatch) {
        a.batch = std::min(batch - b0, kCrossBatch);
        a.cu = cu + b0;
        a.tables = tables + (int64_t)b0 * max_blocks;
        a.lens = lens + b0;
        hipError_t e = half ? launch_cross_16(a, d, few, s) : launch_cross_f32(a, d, few, s);
        if (e == hipSuccess) e = launch_merge(a, rows, d, s);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace airkv
