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

// A mean of values and its weight l under `base`: what a row's pieces are folded to.  (A mean stays
// within its values' range, where a sum of values near the largest or the smallest floats would not.)
struct Fold {
    float base, l;
    f32x4 o;
    __device__ __forceinline__ void add(float b, float w, f32x4 mean) {
        if (w == 0.0f) return;                         // (no key in the pool)
        const float top = fmaxf(base, b);
        const float was = base == top ? l : l * __builtin_amdgcn_exp2f(base - top);
        const float is = b == top ? w : w * __builtin_amdgcn_exp2f(b - top);
        l = was + is;
        const float k = 1.0f / l;
        o = o * (was * k) + mean * (is * k);
        base = top;
    }
};

// The rows of one cut block, rows blockIdx.x, + gridDim.x, ... : LANES lanes of four columns fold
// every GROUPS-th piece, then the groups' results, in order.
template <int LANES, int GROUPS>
__global__ __launch_bounds__(kMergeThreads) void cross_merge_kernel(CrossArgs a, int rows, int d) {
    constexpr int PER = kMergeThreads / (LANES * GROUPS);      // rows at a time
    const int64_t cell = (int64_t)blockIdx.z * a.slices + blockIdx.y;
    const int4 it = a.desc[cell];
    if (it.z == 0) return;
    __shared__ f32x4 s_o[GROUPS][kMergeThreads / GROUPS];
    __shared__ float2 s_bl[GROUPS][kMergeThreads / GROUPS];
    const int lane = threadIdx.x % LANES, g = threadIdx.x / LANES % GROUPS, pr = threadIdx.x / (LANES * GROUPS);
    const int col = lane * 4, place = pr * LANES + lane;
    const int32_t r0 = a.cu[it.x];
    const int32_t here = (a.cu[it.x + 1] - r0) * a.group - it.y * rows;        // rows of the block
    const int many = here < rows ? here : rows;
    for (int first = blockIdx.x * PER; first < many; first += gridDim.x * PER) {
        const int r = first + pr;
        const bool mine = r < many && col < d;
        Fold f = {-INFINITY, 0.0f, {0.0f, 0.0f, 0.0f, 0.0f}};
        if (mine) {
            constexpr int kBatch = 4;
            for (int p0 = g; p0 < it.z; p0 += kBatch * GROUPS) {
                float4 ml[kBatch];
                f32x4 x[kBatch];
#pragma unroll
                for (int i = 0; i < kBatch; ++i) {
                    const int p = p0 + i * GROUPS < it.z ? p0 + i * GROUPS : p0;
                    const int64_t at = (2 * (cell + p) + (p == 0 ? 1 : 0)) * rows + r;
                    ml[i] = a.part_ml[at];
                    x[i] = *reinterpret_cast<const f32x4 *>(a.part_o + at * d + col);
                }
#pragma unroll
                for (int i = 0; i < kBatch; ++i)
                    if (p0 + i * GROUPS < it.z) f.add(ml[i].x, ml[i].y, x[i] * (1.0f / ml[i].y) * ml[i].z);
            }
        }
        if constexpr (GROUPS > 1) {
            s_o[g][place] = f.o;
            s_bl[g][place] = make_float2(f.base, f.l);
            __syncthreads();
            if (g == 0) {
                f = {-INFINITY, 0.0f, {0.0f, 0.0f, 0.0f, 0.0f}};
                for (int i = 0; i < GROUPS; ++i) f.add(s_bl[i][place].x, s_bl[i][place].y, s_o[i][place]);
            }
            __syncthreads();
        }
        if (!mine || g) continue;
        const int32_t row = it.y * rows + r;
        const int64_t at = ((int64_t)(r0 + row / a.group) * a.q_heads + blockIdx.z * a.group + row % a.group) * d + col;
        if (a.out_dtype == AIR_KV_F32)
            *reinterpret_cast<f32x4 *>((float *)a.out + at) = f.o;
        else
            *reinterpret_cast<u32x2 *>((uint16_t *)a.out + at) = u32x2{(uint32_t)bf16_rne(f.o[0]) | ((uint32_t)bf16_rne(f.o[1]) << 16),
                                                                       (uint32_t)bf16_rne(f.o[2]) | ((uint32_t)bf16_rne(f.o[3]) << 16)};
    }
}

// few: blocks of at most `most` rows, of which each takes a workgroup (sequences of many pieces).
hipError_t launch_merge(const CrossArgs &a, CrossBlocks blocks, int d, bool few, int64_t most, hipStream_t s) {
    if (a.slices < 2) return hipSuccess;               // nothing is cut
    const int lanes = d <= 32 ? 8 : d <= 64 ? 16 : d <= 128 ? 32 : 64;
    const int per = few ? 1 : kMergeThreads / lanes;
    const int64_t rows = few ? std::min<int64_t>(std::max<int64_t>(most, 1), blocks.rows) : blocks.rows;
    const dim3 grid((unsigned)((rows + per - 1) / per), (unsigned)a.slices, (unsigned)a.heads), threads(kMergeThreads);
    if (few) {
        if (lanes == 8) hipLaunchKernelGGL((cross_merge_kernel<8, 32>), grid, threads, 0, s, a, blocks.rows, d);
        else if (lanes == 16) hipLaunchKernelGGL((cross_merge_kernel<16, 16>), grid, threads, 0, s, a, blocks.rows, d);
        else if (lanes == 32) hipLaunchKernelGGL((cross_merge_kernel<32, 8>), grid, threads, 0, s, a, blocks.rows, d);
        else hipLaunchKernelGGL((cross_merge_kernel<64, 4>), grid, threads, 0, s, a, blocks.rows, d);
    } else {
        if (lanes == 8) hipLaunchKernelGGL((cross_merge_kernel<8, 1>), grid, threads, 0, s, a, blocks.rows, d);
        else if (lanes == 16) hipLaunchKernelGGL((cross_merge_kernel<16, 1>), grid, threads, 0, s, a, blocks.rows, d);
        else if (lanes == 32) hipLaunchKernelGGL((cross_merge_kernel<32, 1>), grid, threads, 0, s, a, blocks.rows, d);
        else hipLaunchKernelGGL((cross_merge_kernel<64, 1>), grid, threads, 0, s, a, blocks.rows, d);
    }
    return hipGetLastError();
}

size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }

CrossBlocks blocks_of(const air_kv_pool &p, bool half, bool few) {
    return half ? cross_blocks_16(p.desc.head_dim, p.desc.dtype != AIR_KV_BF16, few)
                : cross_blocks_f32(p.desc.head_dim, p.desc.dtype != AIR_KV_BF16, few);
}

// Slices per K/V head: its share of the workgroups that are resident.
int slices_of(const air_kv_pool &p, CrossBlocks blocks) { return std::max(1, p.cus * blocks.groups / p.desc.n_kv_heads); }

struct Workspace {
    size_t ml, o, bytes;           // where the pieces' parts begin, and its end
    Workspace(const air_kv_pool &p, CrossBlocks blocks) {
        const size_t cells = (size_t)p.desc.n_kv_heads * slices_of(p, blocks), slots = 2 * cells * blocks.rows;
        ml = align256(cells * sizeof(int4));
        o = ml + align256(slots * sizeof(float4));
        bytes = o + slots * p.desc.head_dim * 4;
    }
};

}  // namespace

size_t cross_workspace(const air_kv_pool &p) {
    size_t most = 0;
    for (int half = 0; half < 2; ++half)
        for (int few = 0; few < 2; ++few)
            if (!half || p.desc.dtype != AIR_KV_F32) most = std::max(most, Workspace(p, blocks_of(p, half, few)).bytes);
    return most;
}

hipError_t launch_cross(const air_kv_pool &p, hipStream_t s, const void *q, int32_t q_dtype, int32_t n_q_heads, const int32_t *cu,
                        int32_t total_q, int32_t max_q_len, const int32_t *tables, const int32_t *lens, int32_t batch,
                        int32_t max_blocks, float scale, void *workspace, void *out, int32_t out_dtype) {
    const bool half = p.desc.dtype != AIR_KV_F32 && q_dtype == AIR_KV_BF16 && out_dtype == AIR_KV_BF16;
    const int d = p.desc.head_dim, group = n_q_heads / p.desc.n_kv_heads;
    const int64_t most = (int64_t)(max_q_len ? max_q_len : ((int64_t)total_q + batch - 1) / batch) * group;
    // Few rows: a block's waves share its 32 rows, each with keys of its own, where that makes two blocks at
    // most, one for f32 precision and large heads.  (Shared and not, us, 32 sequences of 2000 tokens, 8 heads of
    // 128: 32 rows bf16 67, 90, fp8 64, 114, f32 126, 237; 64 rows 64, 93, 73, 118, 252, 248, f32 heads of 64 99, 128,
    // of 160 478, 329; 128 rows bf16 139, 95, fp8 139, 118.)
    const bool few = most <= (half || d <= 128 ? 64 : 32);
    const CrossBlocks blocks = blocks_of(p, half, few);
    const Workspace ws(p, blocks);
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
    a.slices = slices_of(p, blocks);
    a.desc = (int4 *)workspace;
    a.part_ml = (float4 *)((char *)workspace + ws.ml);
    a.part_o = (float *)((char *)workspace + ws.o);
    for (int32_t b0 = 0; b0 < batch; b0 += kCrossBatch) {
        a.batch = std::min(batch - b0, kCrossBatch);
        a.cu = cu + b0;
        a.tables = tables + (int64_t)b0 * max_blocks;
        a.lens = lens + b0;
        hipError_t e = half ? launch_cross_16(a, d, few, s) : launch_cross_f32(a, d, few, s);
        if (e == hipSuccess) e = launch_merge(a, blocks, d, blocks.few, most, s);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace airkv
