// Differential prefill at f32 precision (formulas: diff_common.hpp; work division:
// diff_prefill_plan.hpp): any page type, f32 queries or outputs.
//
// A workgroup's block is 64 rows.  A wave takes one map of 16 of them: its sums over
// the 2 * head_dim value columns stay in registers, and it walks the block's keys
// once, 32 at a time, with a running maximum and sum.
//
// Both products are v_mfma_f32_16x16x32_bf16 on parts: a value is the sum of three bf16
// numbers of 8 bits each, and of two values' nine products the six down to 2^-16 of the
// whole are added (the others are below 2^-23 of it); elements of bf16 pages are one
// part, exactly.  That is 6 (3) products in the time of 16 on f32 operands.
//   S   = K . Q^T      lane (n, q) holds S of keys 4q .. 4q + 3 of both 16-key halves
//   O^T += V^T . P^T   contracts over those eight: P stays where it is
// Keys and values are staged as parts in LDS (1-byte codes times their scale), in two
// buffers where they fit; while a tile is used, the next one's elements are on their
// way in registers and the one after's table entries too.
// Bound by the chain of a tile (one workgroup to a CU at head_dim 128): 2048 tokens of 16
// query pairs of 128 on f32 pages in 415 us, 83 TFLOP/s (364 on the fastest card met); four
// chunks of 500 to 1000 behind up to 4000 bf16 tokens 0.69 ms, 176.  (On f32 operands half as
// long again for the first, more than twice as long for the second; four waves of both maps,
// without tiles ahead, twice that.)
#include <hip/hip_runtime.h>

#include "../pool.hpp"
#include "diff_prefill.hpp"

namespace airkv {
namespace {

typedef diff_f32x4 f32x4;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ f32x4 mfma_bf16(diff_u32x4 a, diff_u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// The products of parts a[i] b[j], i + j < 3, the smallest first.
// Two sums in turn: a product waits for the one before it of the same sum.
template <int N>
__device__ __forceinline__ void mfma_parts(const diff_u32x4 (&a0)[N], const diff_u32x4 (&a1)[N], const diff_u32x4 (&b)[3],
                                           f32x4 &c0, f32x4 &c1) {
#pragma unroll
    for (int k = 2; k >= 0; --k)
#pragma unroll
        for (int i = N - 1 < k ? N - 1 : k; i >= 0; --i) {
            c0 = mfma_bf16(a0[i], b[k - i], c0);
            c1 = mfma_bf16(a1[i], b[k - i], c1);
        }
}

// Eight values as parts.
__device__ __forceinline__ void parts8(const float (&x)[8], diff_u32x4 (&p)[3]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        uint32_t w[3];
        split3(x[2 * j], x[2 * j + 1], w[0], w[1], w[2]);
#pragma unroll
        for (int k = 0; k < 3; ++k) p[k][j] = w[k];
    }
}

// Where the chunk c of row r of a staged head of values lies: they are read eight rows at
// a time, two chunks each.
template <int D> __device__ __forceinline__ int value_chunk8(int r, int c) {
    if constexpr (D == 128) return c ^ ((r & 7) << 1);
    else if constexpr (D == 64) return c ^ (((r >> 1) & 3) << 1);
    else return c ^ (((r >> 2) & 1) << 1);
}

// 8 elements of a page row as loaded, and as f32.
template <int DT> struct Raw8 {
    uint32_t w[DT == AIR_KV_F32 ? 8 : DT == AIR_KV_BF16 ? 4 : 2];
    float s;
};
template <int DT>
__device__ __forceinline__ void raw8(const void *pages, const float *scales, int64_t elem, int64_t sc, Raw8<DT> &r) {
    if constexpr (DT == AIR_KV_F32 || DT == AIR_KV_BF16) {
        const diff_u32x4 *p = reinterpret_cast<const diff_u32x4 *>((const char *)pages + elem * (DT == AIR_KV_F32 ? 4 : 2));
#pragma unroll
        for (int i = 0; i < (DT == AIR_KV_F32 ? 2 : 1); ++i) {
            const diff_u32x4 x = p[i];
#pragma unroll
            for (int j = 0; j < 4; ++j) r.w[4 * i + j] = x[j];
        }
    } else {
        const diff_u32x2 x = *reinterpret_cast<const diff_u32x2 *>((const char *)pages + elem);
        r.w[0] = x[0];
        r.w[1] = x[1];
        r.s = scales[sc];
    }
}
template <int DT> __device__ __forceinline__ void wide8(const Raw8<DT> &r, float (&x)[8]) {
    if constexpr (DT == AIR_KV_F32 || DT == AIR_KV_BF16) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            x[j] = __uint_as_float(DT == AIR_KV_F32 ? r.w[j] : (j & 1) ? r.w[j / 2] & 0xFFFF0000u : r.w[j / 2] << 16);
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const f32x4 v = code_values<DT>(r.w[i], r.s);
#pragma unroll
            for (int j = 0; j < 4; ++j) x[4 * i + j] = v[j];
        }
    }
}

// A tile's largest score puts the base of the probabilities 2^kLead above itself, so that they
// stay below 1 (values near the largest f32 do not overflow) and most tiles keep the base
// (with none 2048 tokens take 423 us and four chunks 718 where these take 415 and 691).
constexpr float kLead = 4.0f;

template <int D, int DT>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2, 2))) void diff_prefill_f32_kernel(DiffPrefillArgs a) {
    constexpr int R = 64, VP = 2 * D + 4, KS = D / 32, CT = 2 * D / 16, T = 512;
    constexpr bool QUANT = DT == AIR_KV_INT8 || DT == AIR_KV_FP8;
    constexpr int C8 = 2 * kDiffKeys * (D / 8), NC = (C8 + T - 1) / T;       // pieces of 8 elements of a tile; a thread's
    constexpr int NP = DT == AIR_KV_BF16 ? 1 : 3;      // parts of a cached element
    constexpr int RB = 2 * D, HB = kDiffKeys * RB;     // bytes of a staged row, of a head's part
    constexpr int BUF = NP * 4 * HB, NB = BUF > 65536 ? 1 : 2, EX = R * VP * 4;
    __shared__ int64_t s_pre[kDiffPrefillBatch + 1];
    __shared__ int64_t s_sum[8];
    // [buffer][part][keys of both heads, then values][key]; at a block's end map 1's rows of VP floats
    __shared__ __align__(16) uint8_t s_buf[NB * BUF > EX ? NB * BUF : EX];
    auto s_t = [&](int64_t t) __attribute__((always_inline)) { return s_buf + (NB == 2 && (t & 1) ? BUF : 0); };
    // Values that are not finite, in tiles that not every row sees (a hidden key's
    // probability of 0 times such a value would be NaN): staged as 0, and each column's
    // first such key is kept here, from which on a row's column is NaN.
    __shared__ int s_bad[2 * D];
    __shared__ int s_any;
    __shared__ __align__(16) float s_w[2 * D];         // the norm's weights
    if (threadIdx.x < 2 * D) s_w[threadIdx.x] = a.e.norm && a.e.norm_w ? a.e.norm_w[threadIdx.x] : 1.0f;
    diff_refused(a, 2 * D);
    diff_units<512>(a, s_pre, s_sum);
    const int tid = threadIdx.x, lane = tid & 63, q4 = lane >> 4, r16 = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int rg = wave & 3, mp = wave >> 2;           // rows 16 rg .. +16 of the block, map
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
        const int64_t f = it.k * R + 16 * rg + r16, rows = sq.q * g;
        const bool live = f < rows;
        const int64_t tok = live ? f / g : sq.q - 1;
        const int h = kp * g + (live ? (int)(f % g) : 0);
        const int64_t sees = sq.prefix + tok;
        const int64_t f0 = it.k * R + 16 * rg, f1 = f0 + 15;
        const int64_t sees0 = sq.prefix + (f0 < rows ? f0 / g : sq.q - 1);       // every row of the wave
        const int64_t sees1 = sq.prefix + (f1 < rows ? f1 / g : sq.q - 1);       // some row of it
        const int64_t seesb = sq.prefix + it.k * R / g;                          // the block's first row
        __syncthreads();
        if (tid < 2 * D) s_bad[tid] = INT32_MAX;
        if (tid == 0) s_any = 0;
        // Q^T as the B operand: lane (n, q) holds elements 32 s + 8 q .. +8 of row n, in parts
        diff_u32x4 qf[KS][3];
        {
            const int64_t at = ((row0 + tok) * 2 * a.pairs + 2 * h + mp) * D + 8 * q4;
            if (a.q_dtype == AIR_KV_F32) {
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    const f32x4 *p = reinterpret_cast<const f32x4 *>((const float *)a.q + at + 32 * s);
                    const f32x4 lo = p[0], hi = p[1];
                    const float x[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
                    parts8(x, qf[s]);
                }
            } else {
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    qf[s][0] = *reinterpret_cast<const diff_u32x4 *>((const uint16_t *)a.q + at + 32 * s);
                    qf[s][1] = qf[s][2] = diff_u32x4{0, 0, 0, 0};
                }
            }
        }
        const float lam = whole ? a.e.lam[(row0 + tok) * a.e.lam_stride + h] : 0.0f;
        f32x4 acc[CT];
        float base = -INFINITY, l_run = 0.0f;          // probabilities are 2^(score - base)
#pragma unroll
        for (int c = 0; c < CT; ++c) acc[c] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

        const int32_t *table = a.tables + (int64_t)it.b * a.max_blocks;
        int32_t blk[NC];
        Raw8<DT> rk[NC], rv[NC];
        // piece n of this thread: 8 elements c of `key` of either head
        auto place = [&](int n, int &c, int &key, int &m) __attribute__((always_inline)) {
            const int i = tid + T * n;
            c = i % (D / 8);
            key = i / (D / 8) % kDiffKeys;
            m = i / (D / 8 * kDiffKeys);
            return i < C8;
        };
        auto look = [&](int64_t t) __attribute__((always_inline)) {
            if (t >= t1) return;
#pragma unroll
            for (int n = 0; n < NC; ++n) {
                int c, key, m;
                const bool in = place(n, c, key, m);
                const int64_t at = t * kDiffKeys + key;
                blk[n] = in && at < len ? table[(uint32_t)at / (uint32_t)a.bs] : -1;
            }
        };
        auto load = [&](int64_t t) __attribute__((always_inline)) {
            if (t >= t1) return;
#pragma unroll
            for (int n = 0; n < NC; ++n) {
                int c, key, m;
                const bool in = place(n, c, key, m);
                const int64_t at = t * kDiffKeys + key;
                const uint32_t off = (uint32_t)at % (uint32_t)a.bs;
                const bool ok = blk[n] >= 0 && blk[n] < a.num_blocks;
                if (ok) {
                    const int64_t row = ((int64_t)blk[n] * a.heads + 2 * kp + m) * a.bs + off;
                    const int64_t sc = QUANT ? row * (D / a.scale_group) + 8 * c / a.scale_group : 0;
                    raw8<DT>(a.k_pages, a.k_scales, row * D + 8 * c, sc, rk[n]);
                    raw8<DT>(a.v_pages, a.v_scales, row * D + 8 * c, sc, rv[n]);
                } else {                               // past the sequence or outside the pool: zeros
                    rk[n] = Raw8<DT>{};
                    rv[n] = Raw8<DT>{};
                    if (in && at < len && c == 0 && m == 0 && kp == 0 && off == 0) atomicAdd(a.errors, 1ull);
                }
            }
        };
        auto write = [&](int64_t t) __attribute__((always_inline)) {
            if (t >= t1) return;
            uint8_t *to = s_t(t - t0);
            const bool some = t * kDiffKeys + kDiffKeys - 1 > seesb;         // hidden from some row
#pragma unroll
            for (int n = 0; n < NC; ++n) {
                int c, key, m;
                if (!place(n, c, key, m)) continue;
                float x[8], y[8];
                wide8<DT>(rk[n], x);
                wide8<DT>(rv[n], y);
                if (some) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        if (__builtin_fabsf(y[j]) < INFINITY) continue;
                        y[j] = 0.0f;
                        s_any = 1;
                        atomicMin(&s_bad[m * D + 8 * c + j], (int)(t * kDiffKeys + key));
                    }
                }
                diff_u32x4 xp[3], yp[3];
                parts8(x, xp);
                parts8(y, yp);
                uint8_t *k = to + m * HB + key * RB + 16 * key_chunk<D>(key, c);
                uint8_t *v = to + (2 + m) * HB + key * RB + 16 * value_chunk8<D>(key, c);
#pragma unroll
                for (int p = 0; p < NP; ++p) {
                    *reinterpret_cast<diff_u32x4 *>(k + p * 4 * HB) = xp[p];
                    *reinterpret_cast<diff_u32x4 *>(v + p * 4 * HB) = yp[p];
                }
            }
        };
        look(t0);
        load(t0);
        look(t0 + 1);
        __syncthreads();                               // s_bad, and the block before has used the buffers
        write(t0);
        load(t0 + 1);
        look(t0 + 2);
        __syncthreads();
        for (int64_t t = t0; t < t1; ++t) {
            const uint8_t *from = s_t(t - t0);
            if (t * kDiffKeys <= sees1) {              // else no row of this wave sees any of it
                f32x4 sc[2] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    diff_u32x4 x[2][NP];
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        const int key = 16 * b + r16;
                        const uint8_t *k = from + mp * HB + key * RB + 16 * key_chunk<D>(key, 4 * s + q4);
#pragma unroll
                        for (int p = 0; p < NP; ++p) x[b][p] = *reinterpret_cast<const diff_u32x4 *>(k + p * 4 * HB);
                    }
                    mfma_parts<NP>(x[0], x[1], qf[s], sc[0], sc[1]);
                }
                const bool cut = t * kDiffKeys + kDiffKeys - 1 > sees0;
                float top = -INFINITY;
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float v = sc[b][i] * a.scale_log2;
                        if (cut) v = t * kDiffKeys + 16 * b + 4 * q4 + i <= sees ? v : -INFINITY;
                        sc[b][i] = v;
                        top = fmaxf(top, v);
                    }
                top = max_x32(max_x16(top));
                if (__ballot(top > base) != 0ull) {
                    const float now = top > base ? top + kLead : base;
                    const float alpha = base == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(base - now);
                    l_run *= alpha;
#pragma unroll
                    for (int c = 0; c < CT; ++c) acc[c] *= alpha;
                    base = now;
                }
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float v = sc[b][i];
                        const float p = v == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(v - base);
                        sc[b][i] = p;
                        l_run += p;
                    }
                const float y[8] = {sc[0][0], sc[0][1], sc[0][2], sc[0][3], sc[1][0], sc[1][1], sc[1][2], sc[1][3]};
                diff_u32x4 pp[3];
                parts8(y, pp);
                // V^T as the A operand: lane (m, q) takes keys 4 q .. +4 of both halves of column m.
                // Within each 16-lane group, lane j of a transposing read receives element j % 4 of the
                // 8 bytes that lanes 4 k + j / 4 address, k = 0 .. 3: lane i points at key i / 4 of the
                // four and columns 4 (i % 4) of the sixteen.
                const int vr = 4 * q4 + (r16 >> 2);
#pragma unroll
                for (int c = 0; c < CT; c += 2) {
                    diff_u32x4 x[2][NP];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int hd = (c + e) / (D / 16), vc = 2 * ((c + e) % (D / 16)) + ((r16 & 3) >> 1);
                        const uint8_t *v = from + (2 + hd) * HB + 8 * (r16 & 1);
#pragma unroll
                        for (int p = 0; p < NP; ++p)
#pragma unroll
                            for (int b = 0; b < 2; ++b) {
                                typedef short s16x4 __attribute__((ext_vector_type(4)));
                                const int key = 16 * b + vr;
                                const diff_u32x2 w = __builtin_bit_cast(diff_u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                    (__attribute__((address_space(3))) s16x4 *)(v + p * 4 * HB + key * RB + 16 * value_chunk8<D>(key, vc))));
                                x[e][p][2 * b] = w[0];
                                x[e][p][2 * b + 1] = w[1];
                            }
                    }
                    mfma_parts<NP>(x[0], x[1], pp, acc[c], acc[c + 1]);
                }
            }
            if (NB == 1) __syncthreads();              // one buffer: the tile has been used
            write(t + 1);
            load(t + 2);
            look(t + 3);
            __syncthreads();
        }

        // lane (n, q): columns 16 c + 4 q + i of row n in acc[c][i]
        if (s_any) {
#pragma unroll
            for (int c = 0; c < CT; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (s_bad[16 * c + 4 * q4 + i] <= sees) acc[c][i] = __builtin_nanf("");
        }
        const float l = sum_x32(sum_x16(l_run));
        if (whole) {
            const float inv = (mp ? lam : 1.0f) / l;
            float *s_x = (float *)s_buf + (16 * rg + r16) * VP + 4 * q4;
            if (mp)
#pragma unroll
                for (int c = 0; c < CT; ++c) *reinterpret_cast<f32x4 *>(s_x + 16 * c) = acc[c] * inv;
            __syncthreads();
            if (!mp) {
                float ss = 0.0f;
#pragma unroll
                for (int c = 0; c < CT; ++c) {
                    acc[c] = acc[c] * inv - *reinterpret_cast<const f32x4 *>(s_x + 16 * c);
#pragma unroll
                    for (int i = 0; i < 4; ++i) ss += acc[c][i] * acc[c][i];
                }
                const float k = diff_factor(a.e, a.e.norm ? sum_x32(sum_x16(ss)) : 0.0f, 2 * D);
                if (live) {
                    const int64_t at = ((row0 + tok) * a.pairs + h) * (2 * D);
#pragma unroll
                    for (int c = 0; c < CT; ++c) {
                        const int col = 16 * c + 4 * q4;
                        diff_store4(a.e, at + col, acc[c] * (*reinterpret_cast<const f32x4 *>(s_w + col) * k));
                    }
                }
            }
        } else {
            const int64_t slot = 2 * cell + (t0 == 0 ? 1 : 0);
            const int64_t r = (slot * R + 16 * rg + r16) * 2 + mp;
#pragma unroll
            for (int c = 0; c < CT; ++c) *reinterpret_cast<f32x4 *>(a.part_o + r * (2 * D) + 16 * c + 4 * q4) = acc[c];
            if (q4 == 0) {
                a.part_ml[2 * r] = base;
                a.part_ml[2 * r + 1] = l;
            }
            if (t0 == 0) {                          // begun here: its last unit's slice ends it
                const int64_t last = u - t1 + nt - 1;      // of the launch's units
                begun = int4{it.b, (int)(uint32_t)it.k, (int)(it.k >> 32), (int)(last / chunk - w + 1)};
            }
        }
    }
    if (tid == 0) a.desc[cell] = begun;
}

template <int D> void launch_d(const DiffPrefillArgs &a, hipStream_t s) {
    const dim3 grid((unsigned)a.slices, (unsigned)a.kv_pairs);
    if (a.dtype == AIR_KV_F32) hipLaunchKernelGGL((diff_prefill_f32_kernel<D, AIR_KV_F32>), grid, dim3(512), 0, s, a);
    else if (a.dtype == AIR_KV_BF16) hipLaunchKernelGGL((diff_prefill_f32_kernel<D, AIR_KV_BF16>), grid, dim3(512), 0, s, a);
    else if (a.dtype == AIR_KV_INT8) hipLaunchKernelGGL((diff_prefill_f32_kernel<D, AIR_KV_INT8>), grid, dim3(512), 0, s, a);
    else hipLaunchKernelGGL((diff_prefill_f32_kernel<D, AIR_KV_FP8>), grid, dim3(512), 0, s, a);
}

}  // namespace

hipError_t launch_diff_prefill_f32(const DiffPrefillArgs &a, int head_dim, hipStream_t s) {
    if (head_dim == 128) launch_d<128>(a, s);
    else if (head_dim == 96) launch_d<96>(a, s);
    else if (head_dim == 64) launch_d<64>(a, s);
    else launch_d<32>(a, s);
    return hipGetLastError();
}

}  // namespace airkv
