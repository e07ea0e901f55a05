// Differential prefill at f32 precision (formulas: diff_common.hpp; work division:
// diff_prefill_plan.hpp): any page type, f32 queries or outputs.
//
// A workgroup's block is 64 rows, 16 to a wave, which keeps both maps' sums over
// the 2 * head_dim value columns in registers and walks its keys once, 32 at a
// time, with a running maximum and sum per map.  Keys and values are staged in LDS
// as f32 (dequantized as gather does).  Both products are v_mfma_f32_16x16x4_f32:
//   S   = K . Q^T      lane (n, q) holds S of keys 4q .. 4q + 3 of a 16-key half
//   O^T += V^T . P^T   step i contracts over keys {4q + i}: P stays where it is
// Bound by the f32 matrix rate (256 multiply-adds' halves a clock and CU).
#include <hip/hip_runtime.h>

#include "../pool.hpp"
#include "diff_prefill.hpp"
#include "page_io.hpp"

namespace airkv {
namespace {

typedef diff_f32x4 f32x4;

__device__ __forceinline__ f32x4 mfma_f32(float a, float b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

// 8 elements of a page row as f32.
__device__ __forceinline__ void page8(int dtype, const void *pages, const float *scales, int64_t elem, int64_t sc, float (&x)[8]) {
    pio_u32x4 raw;
    if (dtype == AIR_KV_F32) load8<AIR_KV_F32>(pages, scales, elem, sc, x, &raw);
    else if (dtype == AIR_KV_BF16) load8<AIR_KV_BF16>(pages, scales, elem, sc, x, &raw);
    else if (dtype == AIR_KV_INT8) load8<AIR_KV_INT8>(pages, scales, elem, sc, x, &raw);
    else load8<AIR_KV_FP8>(pages, scales, elem, sc, x, &raw);
}

template <int D>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) void diff_prefill_f32_kernel(DiffPrefillArgs a) {
    constexpr int R = 64, KP = D + 4, VP = 2 * D + 4, KS = D / 16, G = 2 * D / 64;
    __shared__ int64_t s_pre[kDiffPrefillBatch + 1];
    __shared__ int64_t s_sum[4];
    __shared__ __align__(16) float s_k[2 * kDiffKeys * KP];
    __shared__ __align__(16) float s_v[kDiffKeys * VP];
    // Values that are not finite, in tiles that not every row sees (a hidden key's
    // probability of 0 times such a value would be NaN): staged as 0, and each column's
    // first such key is kept here, from which on a row's column is NaN.
    __shared__ int s_bad[2 * D];
    __shared__ int s_any;
    __shared__ __align__(16) float s_w[2 * D];         // the norm's weights
    if (threadIdx.x < 2 * D) s_w[threadIdx.x] = a.e.norm && a.e.norm_w ? a.e.norm_w[threadIdx.x] : 1.0f;
    diff_refused(a, 2 * D);
    diff_units<256>(a, s_pre, s_sum);
    const int tid = threadIdx.x, lane = tid & 63, q4 = lane >> 4, r16 = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int w = blockIdx.x, kp = blockIdx.y, g = a.group;
    const int64_t units = diff_uniform(s_pre[a.batch]);
    const int64_t chunk = diff_prefill_chunk(units, a.slices, a.least);
    const int64_t cell = (int64_t)kp * a.slices + w;
    int4 begun = {0, 0, 0, 0};
    int64_t u = w * chunk;
    const int64_t end = u + chunk < units ? u + chunk : units;
    DiffItem it;
    DiffBlocks sq;
    if (u < end) diff_find(a, s_pre, u, it);
    for (; u < end; diff_next(a, s_pre, sq, it)) {
        diff_seq(a, it.b, sq);
        const int64_t nt = sq.tiles(it.k), len = sq.prefix + sq.q;
        const int64_t left = nt + a.extra - it.from, mine = end - u < left ? end - u : left;
        const int64_t t0 = diff_tile_of(it.from, a.extra), t1 = diff_tile_of(it.from + mine, a.extra);
        u += mine;
        if (t0 == t1) continue;                        // the slice ends before the block's first tile
        const bool whole = t0 == 0 && t1 == nt;
        const int64_t row0 = a.cu[it.b];
        // this lane's row, and the newest key it sees
        const int64_t f = it.k * R + 16 * wave + r16, rows = sq.q * g;
        const bool live = f < rows;
        const int64_t tok = live ? f / g : sq.q - 1;
        const int h = kp * g + (live ? (int)(f % g) : 0);
        const int64_t sees = sq.prefix + tok;
        const int64_t f0 = it.k * R + 16 * wave, f1 = f0 + 15;
        const int64_t sees0 = sq.prefix + (f0 < rows ? f0 / g : sq.q - 1);       // every row of the wave
        const int64_t sees1 = sq.prefix + (f1 < rows ? f1 / g : sq.q - 1);       // some row of it
        const int64_t seesb = sq.prefix + it.k * R / g;                          // the block's first row
        __syncthreads();
        if (tid < 2 * D) s_bad[tid] = INT32_MAX;
        if (tid == 0) s_any = 0;
        float qf[2][KS][4];
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            const int64_t at = ((row0 + tok) * 2 * a.pairs + 2 * h + m) * D + 4 * q4;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                if (a.q_dtype == AIR_KV_F32) {
                    const f32x4 x = *reinterpret_cast<const f32x4 *>((const float *)a.q + at + 16 * s);
#pragma unroll
                    for (int j = 0; j < 4; ++j) qf[m][s][j] = x[j];
                } else {
                    const diff_u32x2 x = *reinterpret_cast<const diff_u32x2 *>((const uint16_t *)a.q + at + 16 * s);
#pragma unroll
                    for (int j = 0; j < 4; ++j) qf[m][s][j] = __uint_as_float((j & 1) ? x[j / 2] & 0xFFFF0000u : x[j / 2] << 16);
                }
            }
        }
        f32x4 acc[2][G][4];
        float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.0f, 0.0f};
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int c = 0; c < G; ++c)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[m][c][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

        const int32_t *table = a.tables + (int64_t)it.b * a.max_blocks;
        for (int64_t t = t0; t < t1; ++t) {
            __syncthreads();                           // the tile before has been used
            // keys and values of both heads, 8 elements a thread and pass; what lies past the sequence is zero
            for (int i = tid; i < 2 * kDiffKeys * (D / 8); i += 256) {
                const int c = i % (D / 8), key = i / (D / 8) % kDiffKeys, m = i / (D / 8 * kDiffKeys);
                const int64_t at = t * kDiffKeys + key;
                float x[8] = {0, 0, 0, 0, 0, 0, 0, 0}, y[8] = {0, 0, 0, 0, 0, 0, 0, 0};
                if (at < len) {
                    const int32_t blk = table[at / a.bs];
                    if (blk >= 0 && blk < a.num_blocks) {
                        const int64_t row = ((int64_t)blk * a.heads + 2 * kp + m) * a.bs + at % a.bs;
                        const int64_t sc = a.k_scales ? row * (D / a.scale_group) + 8 * c / a.scale_group : 0;
                        page8(a.dtype, a.k_pages, a.k_scales, row * D + 8 * c, sc, x);
                        page8(a.dtype, a.v_pages, a.v_scales, row * D + 8 * c, sc, y);
                    } else if (c == 0 && m == 0 && kp == 0 && at % a.bs == 0) {
                        atomicAdd(a.errors, 1ull);
                    }
                }
                float *k = s_k + (m * kDiffKeys + key) * KP + 8 * c, *v = s_v + key * VP + m * D + 8 * c;
                if (t * kDiffKeys + kDiffKeys - 1 > seesb) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        if (__builtin_fabsf(y[j]) < INFINITY) continue;
                        y[j] = 0.0f;
                        s_any = 1;
                        atomicMin(&s_bad[m * D + 8 * c + j], (int)at);
                    }
                }
                *reinterpret_cast<f32x4 *>(k) = f32x4{x[0], x[1], x[2], x[3]};
                *reinterpret_cast<f32x4 *>(k + 4) = f32x4{x[4], x[5], x[6], x[7]};
                *reinterpret_cast<f32x4 *>(v) = f32x4{y[0], y[1], y[2], y[3]};
                *reinterpret_cast<f32x4 *>(v + 4) = f32x4{y[4], y[5], y[6], y[7]};
            }
            __syncthreads();
            if (t * kDiffKeys > sees1) continue;       // no row of this wave sees any of it
            f32x4 sc[2][2];
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int b = 0; b < 2; ++b) sc[m][b] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                f32x4 x[2][2];
#pragma unroll
                for (int m = 0; m < 2; ++m)
#pragma unroll
                    for (int b = 0; b < 2; ++b)
                        x[m][b] = *reinterpret_cast<const f32x4 *>(s_k + (m * kDiffKeys + 16 * b + r16) * KP + 16 * s + 4 * q4);
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int m = 0; m < 2; ++m)
#pragma unroll
                        for (int b = 0; b < 2; ++b) sc[m][b] = mfma_f32(x[m][b][j], qf[m][s][j], sc[m][b]);
            }
            const bool cut = t * kDiffKeys + kDiffKeys - 1 > sees0;
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                float top = -INFINITY;
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float v = sc[m][b][i] * a.scale_log2;
                        if (cut) v = t * kDiffKeys + 16 * b + 4 * q4 + i <= sees ? v : -INFINITY;
                        sc[m][b][i] = v;
                        top = fmaxf(top, v);
                    }
                top = max_x32(max_x16(top));
                // raised only past 2^8 times the present maximum (and on the first tile)
                if (__ballot(top > m_run[m] + 8.0f) != 0ull) {
                    const float now = top > m_run[m] + 8.0f ? top : m_run[m];
                    const float alpha = m_run[m] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m_run[m] - now);
                    l_run[m] *= alpha;
#pragma unroll
                    for (int c = 0; c < G; ++c)
#pragma unroll
                        for (int j = 0; j < 4; ++j) acc[m][c][j] *= alpha;
                    m_run[m] = now;
                }
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float v = sc[m][b][i];
                        const float p = v == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(v - m_run[m]);
                        sc[m][b][i] = p;
                        l_run[m] += p;
                    }
            }
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int c = 0; c < G; ++c) {
                        const f32x4 v = *reinterpret_cast<const f32x4 *>(s_v + (16 * b + 4 * q4 + i) * VP + 64 * c + 4 * r16);
#pragma unroll
                        for (int j = 0; j < 4; ++j)
#pragma unroll
                            for (int m = 0; m < 2; ++m) acc[m][c][j] = mfma_f32(v[j], sc[m][b][i], acc[m][c][j]);
                    }
        }

        // lane (n, q): columns 64 c + 16 q + 4 i + j of row n in acc[m][c][j][i]
        __syncthreads();
        if (s_any) {
#pragma unroll
            for (int c = 0; c < G; ++c)
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (s_bad[64 * c + 16 * q4 + 4 * i + j] <= sees) acc[0][c][j][i] = acc[1][c][j][i] = __builtin_nanf("");
        }
        float l[2];
#pragma unroll
        for (int m = 0; m < 2; ++m) l[m] = sum_x32(sum_x16(l_run[m]));
        if (whole) {
            const float lam = a.e.lam[(row0 + tok) * a.e.lam_stride + h];
            const float i0 = 1.0f / l[0], i1 = lam / l[1];
            float ss = 0.0f;
#pragma unroll
            for (int c = 0; c < G; ++c)
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float x = acc[0][c][j][i] * i0 - acc[1][c][j][i] * i1;
                        acc[0][c][j][i] = x;
                        ss += x * x;
                    }
            const float k = diff_factor(a.e, a.e.norm ? sum_x32(sum_x16(ss)) : 0.0f, 2 * D);
            if (live) {
                const int64_t at = ((row0 + tok) * a.pairs + h) * (2 * D);
#pragma unroll
                for (int c = 0; c < G; ++c)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int col = 64 * c + 16 * q4 + 4 * i;
                        const f32x4 n = *reinterpret_cast<const f32x4 *>(s_w + col) * k;
                        diff_store4(a.e, at + col, f32x4{acc[0][c][0][i] * n[0], acc[0][c][1][i] * n[1], acc[0][c][2][i] * n[2],
                                                         acc[0][c][3][i] * n[3]});
                    }
            }
        } else {
            const int64_t slot = 2 * cell + (t0 == 0 ? 1 : 0);
            const int64_t r = (slot * R + 16 * wave + r16) * 2;
#pragma unroll
            for (int m = 0; m < 2; ++m) {
#pragma unroll
                for (int c = 0; c < G; ++c)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        *reinterpret_cast<f32x4 *>(a.part_o + (r + m) * (2 * D) + 64 * c + 16 * q4 + 4 * i) =
                            f32x4{acc[m][c][0][i], acc[m][c][1][i], acc[m][c][2][i], acc[m][c][3][i]};
                if (q4 == 0) {
                    a.part_ml[2 * (r + m)] = m_run[m];
                    a.part_ml[2 * (r + m) + 1] = l[m];
                }
            }
            if (t0 == 0) {                          // begun here: its last unit's slice ends it
                const int64_t last = u - t1 + nt - 1;      // of the launch's units
                begun = int4{it.b, (int)(uint32_t)it.k, (int)(it.k >> 32), (int)(last / chunk - w + 1)};
            }
        }
    }
    if (tid == 0) a.desc[cell] = begun;
}

}  // namespace

hipError_t launch_diff_prefill_f32(const DiffPrefillArgs &a, int head_dim, hipStream_t s) {
    const dim3 grid((unsigned)a.slices, (unsigned)a.kv_pairs);
    if (head_dim == 128) hipLaunchKernelGGL((diff_prefill_f32_kernel<128>), grid, dim3(256), 0, s, a);
    else if (head_dim == 96) hipLaunchKernelGGL((diff_prefill_f32_kernel<96>), grid, dim3(256), 0, s, a);
    else if (head_dim == 64) hipLaunchKernelGGL((diff_prefill_f32_kernel<64>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((diff_prefill_f32_kernel<32>), grid, dim3(256), 0, s, a);
    return hipGetLastError();
}

}  // namespace airkv
