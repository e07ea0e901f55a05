// Differential decode attention over the paged cache (formulas: diff_common.hpp).
//
// The batch's cached tokens are cut into 16-token tiles and these into equal
// contiguous slices per K/V pair, one wave each (decode_slices.hpp); a sequence
// that several slices hold is joined by diff_decode_merge_kernel.
//
// A wave takes eight query pairs of its K/V pair as 16 rows: row n is map n / 8 of
// query pair n % 8, so one accumulator tile holds both maps and the softmax works
// on all 64 lanes.  Per tile:
//   S  = K . Q^T  twice, with either key head; row n keeps the one of its map.
//   P  = exp2(S * scale * log2 e - m)
//   O^T += V^T . P^T over the 2 * head_dim columns of the pair's two value heads.
// No operand needs a transpose: lane (n, q) holds S of tokens 4q .. 4q + 3, and the
// second product contracts over just these, whose V rows the lane reads from the page.
//
// Products, by page type:
//   f32     v_mfma_f32_16x16x4_f32, 24 bits.
//   bf16    bf16 products of the pages as they are with queries and probabilities split
//           into parts of 8 bits, three of each (exact); bf16 queries are one part, and
//           bf16 outputs take two parts of a probability: the third is below 2^-16 of it,
//           the output's own rounding 2^-9.
//   1-byte  the same on the codes, which bf16 holds exactly; a key's scales multiply the
//           scores in f32, a value's the probabilities before they are split (so a product
//           of 16 columns has to lie in one scale group: order_v).  f32 products of
//           dequantized values took 160 and 350 us where these take 125 and 296.
//
// Bound by the reads of the pages: 64 sequences of 512 to 4096 tokens (bf16, 8 heads of
// 128) 569 MB in 102 us, 5.6 TB/s, 32 of 8192 (int8) 605 MB in 120 us, 5.0, 8 of 32K to
// 128K (fp8) 1.56 GB in 287 us, 5.4; the joining takes 7 to 10 us more.  A lone short
// sequence takes two dependent kernels of a few memory round trips, 15 us.  What carried
// it there: 16 bytes a lane of a key row (64 bytes of it at once; with 8 the fp8 case took 431 us
// where it then took 350), and the next tile's keys in flight while this one's values are used.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "../pool.hpp"
#include "decode_plan.hpp"
#include "diff_common.hpp"

namespace airkv {
namespace {

typedef diff_f32x4 f32x4;
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = kSliceThreads;
constexpr int kWaves = kThreads / 64;
constexpr int kWavesPerSimd = 2;
constexpr int kFullChunk = 4;              // tiles a slice holds at least once every SIMD has a wave

struct DiffDecodeArgs : DecodeArgs {
    DiffOut e;
    int32_t pairs;                         // query pairs
    int32_t kv_pairs, row_tiles;
};

__device__ __forceinline__ f32x4 mfma_f32(float a, float b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ f32x4 mfma_bf16(diff_u32x4 a, diff_u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma_bf16(diff_u32x2 a, diff_u32x2 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4, a), __builtin_bit_cast(s16x4, b), c, 0, 0, 0);
}

// Eight 1-byte codes as bf16, exactly.
template <int DT> __device__ __forceinline__ diff_u32x4 codes_bf16(const uint32_t (&w)[2]) {
    diff_u32x4 x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t c = w[i / 2];
        if constexpr (DT == AIR_KV_INT8) {
            const float lo = (float)(int8_t)(c >> (16 * (i & 1))), hi = (float)(int8_t)(c >> (16 * (i & 1) + 8));
            x[i] = halves<true>(__float_as_uint(lo), __float_as_uint(hi));
        } else {
            x[i] = (i & 1) ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)c, 1.0f, true))
                           : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)c, 1.0f, false));
        }
    }
    return x;
}

// x of lane l ^ 8 within each 16 lanes.
__device__ __forceinline__ float dpp_ror8(float x) {
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x128, 0xF, 0xF, false));
}

// BYTES (2, 4, 8, 16 or 32) bytes of a page at base + off.
template <int BYTES>
__device__ __forceinline__ void load_piece(const __amdgpu_buffer_rsrc_t &r, int off, int base,
                                           uint32_t (&w)[(BYTES + 3) / 4]) {
    if constexpr (BYTES == 2) {
        w[0] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(r, off, base, kDiffStream);
    } else if constexpr (BYTES == 4) {
        w[0] = __builtin_amdgcn_raw_buffer_load_b32(r, off, base, kDiffStream);
    } else if constexpr (BYTES == 8) {
        const diff_u32x2 x = __builtin_amdgcn_raw_buffer_load_b64(r, off, base, kDiffStream);
        w[0] = x[0]; w[1] = x[1];
    } else {
#pragma unroll
        for (int i = 0; i < BYTES / 16; ++i) {
            const diff_u32x4 x = __builtin_amdgcn_raw_buffer_load_b128(r, off + 16 * i, base, kDiffStream);
            w[4 * i] = x[0]; w[4 * i + 1] = x[1]; w[4 * i + 2] = x[2]; w[4 * i + 3] = x[3];
        }
    }
}

// Two 1-byte codes (the lower halves of w, or the upper) of four rows as bf16,
// exactly: x[e] holds code e of rows 0 .. 3.
template <int DT, bool HI> __device__ __forceinline__ void codes_by_row(const uint32_t (&w)[4], diff_u32x2 (&x)[2]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        // code 0 of rows 2 i and 2 i + 1, then code 1
        const uint32_t c = __builtin_amdgcn_perm(w[2 * i + 1], w[2 * i], HI ? 0x07030602u : 0x05010400u);
        if constexpr (DT == AIR_KV_INT8) {
#pragma unroll
            for (int e = 0; e < 2; ++e)
                x[e][i] = halves<true>(__float_as_uint((float)(int8_t)(c >> (16 * e))),
                                       __float_as_uint((float)(int8_t)(c >> (16 * e + 8))));
        } else {
            x[0][i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)c, 1.0f, false));
            x[1][i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)c, 1.0f, true));
        }
    }
}

template <int D, int DT, bool WIDE, bool FINE>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(kWavesPerSimd, kWavesPerSimd)))
void diff_decode_kernel(DiffDecodeArgs a) {
    static_assert(D % 32 == 0 && D <= 128, "steps of 32, two value heads of at most 256 columns");
    constexpr bool F32 = DT == AIR_KV_F32, QUANT = DT == AIR_KV_INT8 || DT == AIR_KV_FP8;
    constexpr int EB = DT == AIR_KV_F32 ? 4 : DT == AIR_KV_BF16 ? 2 : 1;
    constexpr int KS = D / 32;                         // steps of the first product
    constexpr int NS = FINE ? D / 8 : KS, SL = (16 * NS + 63) / 64;  // scales of a row at most, a lane's loads of them
    constexpr int QP = WIDE ? 3 : 1;                   // bf16 parts of a query
    // columns of a value head in a lane: CA from CA * m, then CB from 16 * CA + CB * m
    // (96 as 64 + 32: every run a power of two). 
    constexpr int CA = D == 96 ? 4 : D / 16, CB = D == 96 ? 2 : 0, C = CA + CB;
    constexpr int PW = !QUANT && D % 64 == 0 ? 4 : 2, PC = C / PW, NP = 4 * PC;      // pieces of consecutive columns of a lane
    constexpr int KW = 8 * EB / 4, VA = (CA * EB + 3) / 4, VB = CB ? (CB * EB + 3) / 4 : 1;

    __shared__ int32_t s_pre[kMaxBatch + 2];
    __shared__ int32_t s_wsum[kWaves];
    __shared__ f32x4 s_scale[QUANT ? kWaves : 1][2][2][NS][4];       // K and V; [head][group] of 16 tokens

    const int bs = a.block_size;
    tile_prefix(a, bs, s_pre, s_wsum);
    const int B = a.batch;
    const int total = s_pre[B];
    const int chunk = slice_chunk(total, a.slices, a.simd_slices, kFullChunk, s_pre[B + 1], a.max_splits);
    if (blockIdx.x == 0) {                             // for the merge: prefix, then the chunk
        for (int i = threadIdx.x; i <= B; i += kThreads) a.prefix[i] = s_pre[i];
        if (threadIdx.x == 0) a.prefix[B + 1] = chunk;
    }

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int q4 = lane >> 4, r16 = lane & 15;
    // the row tiles of a K/V pair, then the pairs, are neighbours: their pages are the same, or lie in the same blocks
    const int heads = a.kv_pairs * a.row_tiles;
    const int gw = blockIdx.x * kWaves + wave;
    const int hh = gw % heads, w = gw / heads;
    if (w >= a.slices || (int64_t)w * chunk >= total) return;
    const int kp = hh / a.row_tiles, rt = hh % a.row_tiles;
    const int lo = w * chunk;
    const int hi = total - lo < chunk ? total : lo + chunk;
    const int64_t max_len = (int64_t)a.max_blocks * bs;
    const int rows = a.group - 8 * rt < 8 ? a.group - 8 * rt : 8;       // query pairs of this wave
    const int qp = r16 & 7;                                             // this lane's row: map r16 / 8 of pair qp
    const bool map1 = r16 >= 8;
    const bool live_row = qp < rows;
    const bool wide_q = WIDE && a.q_dtype == AIR_KV_F32, wide_out = WIDE && a.e.out_dtype == AIR_KV_F32;

    // Lane k describes tile c0 + k of a window of 64: block, its first row there, sequence, valid tokens.
    int32_t tbl = 0, seq_l = 0, j_l = 0, nv_l = 0;
    uint64_t first_m = 0, last_m = 0;
    auto load_window = [&](int c0) {
        const int t = c0 + lane < hi ? c0 + lane : hi - 1;
        const int bq = seq_of_tile(s_pre, B, t);
        const int j = t - s_pre[bq];
        const int64_t len = clamp_len(a.lens[bq], max_len);
        const int per = bs / 16, in_row = j / per;     // tiles of a block; the tile's block
        tbl = a.tables[(int64_t)bq * a.max_blocks + in_row];
        seq_l = bq;
        j_l = 16 * (j - in_row * per);
        const int64_t rest = len - 16 * (int64_t)j;
        nv_l = rest < 16 ? (int)rest : 16;
        const bool valid = c0 + lane < hi;
        first_m = __ballot(valid && (t == lo || j == 0));
        last_m = __ballot(valid && (t + 1 == hi || t + 1 == s_pre[bq + 1]));
    };

    // Q^T as the B operand: lane (n, q) holds eight of row n's elements from 32 s + q_at
    // (order_k leaves the keys' elements in this order)
    const int q_at = QUANT ? 16 * (q4 & 1) + 8 * (q4 >> 1) : 8 * q4;
    // (f32 pages), or the same as bf16 parts: bf16 queries one, f32 queries three
    float qf[F32 ? KS : 1][8];
    diff_u32x4 qb[F32 || !WIDE ? 1 : 3][KS];
    auto load_q = [&](int bq) {
        const int head = 2 * (kp * a.group + 8 * rt + qp) + (map1 ? 1 : 0);
        const int64_t at = ((int64_t)bq * a.n_q_heads + (live_row ? head : 0)) * D + q_at;
        if (wide_q) {
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                const f32x4 *p = reinterpret_cast<const f32x4 *>((const float *)a.q + at + 32 * s);
                const f32x4 x = p[0], y = p[1];
                if constexpr (F32) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) qf[s][j] = j < 4 ? x[j] : y[j - 4];
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        uint32_t w[3];
                        const f32x4 z = j < 2 ? x : y;
                        split3(z[2 * (j & 1)], z[2 * (j & 1) + 1], w[0], w[1], w[2]);
#pragma unroll
                        for (int k = 0; k < (WIDE ? 3 : 1); ++k) qb[k][s][j] = w[k];
                    }
                }
            }
        } else {
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                const diff_u32x4 x = *reinterpret_cast<const diff_u32x4 *>((const uint16_t *)a.q + at + 32 * s);
                if constexpr (F32) {
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        qf[s][j] = __uint_as_float((j & 1) ? x[j / 2] & 0xFFFF0000u : x[j / 2] << 16);
                } else {
                    qb[0][s] = x;
                }
            }
        }
        // waited for here: where no sequence starts, the loads of tiles stay in flight
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            if constexpr (F32) {
#pragma unroll
                for (int j = 0; j < 8; ++j) asm volatile("" : "+v"(qf[s][j]));
            } else {
                asm volatile("" : "+v"(qb[0][s]));
            }
        }
    };

    f32x4 acc[2][C];                                   // O^T: value head, column of the lane
    float m_run = -INFINITY, l_run = 0.0f;

    const int sg = QUANT ? FINE ? __builtin_ctz(a.scale_group) : 5 : 0, nsc = D >> sg;      // scales per row
    // Piece i of a value head: its values and the first's column
    auto piece = [&](int t, int i, float (&x)[PW]) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < PW; ++e)
            x[e] = acc[t][PW * (i % PC) + e][i / PC];
        const int m = 4 * q4 + i / PC, j = PW * (i % PC);
        if constexpr (QUANT)
            return t * D + 32 * (j / 2) + (j / 2 < KS / 2 * 2 ? 16 * (q4 & 1) + 4 * (i / PC) + 2 * (q4 >> 1) : 2 * m);
        return t * D + (j < CA ? CA * m + j : 16 * CA + CB * m + j - CA);
    };

    // The piece of sequence bq that this wave holds ends.
    auto emit = [&](int bq) {
        const float l = sum_x32(sum_x16(l_run));
        const int w0 = s_pre[bq] / chunk, w1 = (s_pre[bq + 1] - 1) / chunk;
        if (w0 == w1) {                                // the whole sequence: its output rows
            const int h = kp * a.group + 8 * rt + qp;
            const float lam = live_row ? a.e.lam[bq * a.e.lam_stride + h] : 0.0f;
            const float inv = l == 0.0f ? 0.0f : (map1 ? -lam : 1.0f) / l;      // no block of it is in the pool: zeros
            float ss = 0.0f;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int j = 0; j < C; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        // row n's and row n + 8's lanes (row_ror:8)
                        const float x = acc[t][j][i] * inv;
                        const float y = x + dpp_ror8(x);
                        acc[t][j][i] = y;
                        ss += y * y;
                    }
            const float f = diff_factor(a.e, a.e.norm ? sum_x32(sum_x16(ss)) : 0.0f, 2 * D);
            if (live_row && !map1) {
                const int64_t at = ((int64_t)bq * a.pairs + h) * (2 * D);
                // no weights: an empty view, which reads as zeros
                const bool weights = a.e.norm && a.e.norm_w;
                const __amdgpu_buffer_rsrc_t rw = __builtin_amdgcn_make_buffer_rsrc(
                    (void *)a.e.norm_w, (short)0, weights ? 2 * D * 4 : 0, kDiffBufferWord3);
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int i = 0; i < NP; ++i) {
                        float x[PW];
                        const int c = piece(t, i, x);
                        uint32_t wt[PW];
                        load_piece<4 * PW>(rw, 4 * c, 0, wt);
#pragma unroll
                        for (int e = 0; e < PW; ++e) x[e] *= weights ? f * __uint_as_float(wt[e]) : f;
                        if constexpr (PW == 4) diff_store4(a.e, at + c, f32x4{x[0], x[1], x[2], x[3]});
                        else diff_store2(a.e, at + c, x[0], x[1]);
                    }
            }
        } else if (live_row) {
            const int64_t row = ((int64_t)hh * a.slots + part_row(w, bq, w == w0)) * 16 + r16;
            float *po = a.part_o + row * (2 * D);
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < NP; ++i) {
                    float x[PW];
                    const int c = piece(t, i, x);
                    if constexpr (PW == 4) *reinterpret_cast<f32x4 *>(po + c) = f32x4{x[0], x[1], x[2], x[3]};
                    else *reinterpret_cast<float2 *>(po + c) = make_float2(x[0], x[1]);
                }
            if (q4 == 0) {
                a.part_ml[row * 2] = m_run;
                a.part_ml[row * 2 + 1] = l;
            }
        }
    };

    // The next tile: its first row (of the pair's first head; the second's are bs further), its tokens and flags
    int64_t row0 = 0;
    int nv = 0, bq = 0;
    bool first = false, last = false;
    auto look = [&](int k) __attribute__((always_inline)) {
        const int idx = (k - lo) & 63;
        if (idx == 0) load_window(k);
        const int blk = __builtin_amdgcn_readlane(tbl, idx), jt = __builtin_amdgcn_readlane(j_l, idx);
        const bool ok = blk >= 0 && blk < a.num_blocks;
        row0 = ((int64_t)(ok ? blk : 0) * a.n_kv_heads + 2 * kp) * bs + jt;
        nv = ok ? __builtin_amdgcn_readlane(nv_l, idx) : 0;
        bq = __builtin_amdgcn_readlane(seq_l, idx);
        first = (first_m >> idx) & 1;
        last = (last_m >> idx) & 1;
        // an entry outside the pool is counted once, by the first pair's wave, and its tile masked
        if (!ok && lane == 0 && hh == 0) atomicAdd(a.errors, 1ull);
    };
    // The tile at `row`, `width` bytes a row, to the end of the second head's (nothing, unless `in`)
    auto view = [&](const void *p, int64_t row, int width, bool in) __attribute__((always_inline)) {
        return __builtin_amdgcn_make_buffer_rsrc((void *)((const char *)p + row * width), (short)0,
                                                 in ? (bs + 16) * width : 0, kDiffBufferWord3);
    };
    // 1-byte pages: words of two groups (order_v), the last of an odd number alone
    constexpr int VW = QUANT ? (KS + 1) / 2 : VA + (CB ? VB : 0);
    uint32_t kr[2][KS][KW], vr[2][4][VW];
    uint32_t ksc[2][SL], vsc[2][SL];                   // a tile's scales in order, either head's
    const int head1 = bs * D * EB;                     // the second head's rows, in bytes
    auto load_scales = [&](const float *p, bool in, uint32_t (&x)[2][SL]) __attribute__((always_inline)) {
        const __amdgpu_buffer_rsrc_t rs = view(p, row0, 4 * nsc, in);
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < SL; ++i)
                x[t][i] = __builtin_amdgcn_raw_buffer_load_b32(rs, lane + 64 * i < 16 * nsc ? 4 * lane + 256 * i : 0,
                                                               t ? 4 * bs * nsc : 0, kDiffStream);
    };
    auto load_k = [&](bool in) __attribute__((always_inline)) {
        const __amdgpu_buffer_rsrc_t rk = view(a.k_pages, row0, D * EB, in);
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int s = 0; s < KS; ++s)
                if (QUANT && (s | 1) < KS) {           // 64 bytes of a row at once; order_k makes steps of them
                    if (s & 1) continue;
                    uint32_t w[4];
                    load_piece<16>(rk, r16 * D + 32 * s + 16 * q4, t ? head1 : 0, w);
                    kr[t][s][0] = w[0]; kr[t][s][1] = w[1];
                    kr[t][s + 1][0] = w[2]; kr[t][s + 1][1] = w[3];
                } else {
                    load_piece<8 * EB>(rk, (r16 * D + 32 * s + q_at) * EB, t ? head1 : 0, kr[t][s]);
                }
        if constexpr (QUANT) {
            load_scales(a.k_scales, in, ksc);
        }
    };
    auto load_v = [&](bool in) __attribute__((always_inline)) {
        const __amdgpu_buffer_rsrc_t rv = view(a.v_pages, row0, D * EB, in);
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int at = (4 * q4 + i) * D;
                if constexpr (QUANT) {
#pragma unroll
                    for (int h = 0; h < VW; ++h) {
                        uint32_t w[1];
                        if (2 * h + 1 < KS) load_piece<4>(rv, at + 64 * h + 4 * r16, t ? head1 : 0, w);
                        else load_piece<2>(rv, at + 64 * h + 2 * r16, t ? head1 : 0, w);
                        vr[t][i][h] = w[0];
                    }
                } else {
                    uint32_t w[VA], z[VB];
                    load_piece<CA * EB>(rv, (at + CA * r16) * EB, t ? head1 : 0, w);
                    if constexpr (CB > 0) load_piece<CB * EB>(rv, (at + 16 * CA + CB * r16) * EB, t ? head1 : 0, z);
#pragma unroll
                    for (int j = 0; j < VW; ++j) vr[t][i][j] = j < VA ? w[j] : z[j - VA];
                }
            }
        if constexpr (QUANT) {
            load_scales(a.v_scales, in, vsc);
        }
    };

    // A tile's scales by token, [head][group][token], those of tokens from n on as zeros
    auto put_scales = [&](int kv, const uint32_t (&x)[2][SL], int n) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < SL; ++i) {
            const int at = lane + 64 * i, tok = FINE ? at / nsc : at / KS, g = at - tok * nsc;
            if (tok < 16)
#pragma unroll
                for (int t = 0; t < 2; ++t) ((uint32_t *)&s_scale[wave][kv][t][g])[tok] = tok < n ? x[t][i] : 0;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    };

    // Steps s and s + 1 are loaded 16 bytes a lane: the lower two words of lanes q = 2, 3
    // (step s + 1) change places with the upper two of lanes 0, 1 (step s).
    auto order_k = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int s = 0; s + 1 < KS; s += 2)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const auto r = __builtin_amdgcn_permlane32_swap(kr[t][s][i], kr[t][s + 1][i], false, false);
                    kr[t][s][i] = r[0];
                    kr[t][s + 1][i] = r[1];
                }
    };

    // 64 columns of a row, four to a lane: lanes m and m ^ 8 exchange halves, so that each
    // has two columns of either scale group and a product's 16 columns share a row's scale.
    auto order_v = [&]() __attribute__((always_inline)) {
        const uint32_t pick = r16 < 8 ? 0x05040100u : 0x03020706u;     // own low, other's low; other's high, own high
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int h = 0; 2 * h + 1 < KS; ++h) {
                    const uint32_t o = (uint32_t)__builtin_amdgcn_mov_dpp((int)vr[t][i][h], 0x128, 0xF, 0xF, false);
                    vr[t][i][h] = __builtin_amdgcn_perm(o, vr[t][i][h], pick);
                }
    };

    // The keys of the next tile are loaded once this one's scores are there, its
    // values after this one's product: either is in flight while the other is used.
    look(lo);
    load_k(true);
    load_v(true);
    for (int k = lo; k < hi; ++k) {
        if (first) {                                   // a sequence starts in this slice
            load_q(bq);
            m_run = -INFINITY;
            l_run = 0.0f;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int j = 0; j < C; ++j) acc[t][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        const int n = nv, seq = bq;
        const bool full = n == 16, end = last, more = k + 1 < hi;

        // S of the lane's row and tokens 4 q + i
        f32x4 sc = {0.0f, 0.0f, 0.0f, 0.0f};
        if constexpr (F32) {
            f32x4 s2[2] = {sc, sc};
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int j = 0; j < 8; ++j)
#pragma unroll
                    for (int t = 0; t < 2; ++t) s2[t] = mfma_f32(__uint_as_float(kr[t][s][j]), qf[s][j], s2[t]);
            sc = map1 ? s2[1] : s2[0];
        } else if constexpr (!QUANT) {
            f32x4 s2[2] = {sc, sc};
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const diff_u32x4 x = {kr[t][s][0], kr[t][s][1], kr[t][s][2], kr[t][s][3]};
                    s2[t] = mfma_bf16(x, qb[0][s], s2[t]);
                }
            if constexpr (WIDE)
                if (wide_q)
#pragma unroll
                for (int s = 0; s < KS; ++s)
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        const diff_u32x4 x = {kr[t][s][0], kr[t][s][1], kr[t][s][2], kr[t][s][3]};
                        s2[t] = mfma_bf16(x, qb[2][s], mfma_bf16(x, qb[1][s], s2[t]));
                    }
            sc = map1 ? s2[1] : s2[0];
        } else {
            // the codes' products, a scale group at a time, then the scales (f32)
            const f32x4 zero = sc;
            put_scales(0, ksc, 16);
            order_k();
            // groups of 8 or 16: those of a step's 32 elements one by one, the other lanes' elements as zeros
            auto pass = [&](bool rest) __attribute__((always_inline)) {
                for (int g = 0; g < (FINE ? 32 : 1); g += FINE ? 1 << sg : 1) {
                    const uint32_t mine = !FINE || (q_at >= g && q_at < g + (1 << sg)) ? ~0u : 0u;
#pragma unroll
                    for (int s = 0; s < KS; ++s) {
                        f32x4 s2[2];
                        const f32x4 ks = s_scale[wave][0][map1 ? 1 : 0][FINE ? (32 * s + g) >> sg : s][q4];
#pragma unroll
                        for (int t = 0; t < 2; ++t) {
                            const uint32_t w[2] = {kr[t][s][0] & mine, kr[t][s][1] & mine};
                            const diff_u32x4 x = codes_bf16<DT>(w);
                            s2[t] = rest ? mfma_bf16(x, qb[QP - 1][s], mfma_bf16(x, qb[QP / 2][s], zero)) : mfma_bf16(x, qb[0][s], zero);
                        }
#pragma unroll
                        for (int i = 0; i < 4; ++i) sc[i] += (map1 ? s2[1][i] : s2[0][i]) * ks[i];
                    }
                }
            };
            pass(false);
            if (wide_q) pass(true);
        }
        if (more) look(k + 1);
        load_k(more);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            sc[i] *= a.scale_log2;
            if (!full) sc[i] = 4 * q4 + i < n ? sc[i] : -INFINITY;
        }
        float mt = fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3]));
        mt = max_x32(max_x16(mt));
        // most tiles have no new maximum and skip the rescale (no slack: probabilities above 1
        // would overflow on values near the largest f32)
        if (__ballot(mt > m_run) != 0ull) {
            const float top = mt > m_run ? mt : m_run;
            const float alpha = m_run == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m_run - top);
            l_run *= alpha;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int j = 0; j < C; ++j) acc[t][j] *= alpha;
            m_run = top;
        }
        float p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = sc[i] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(sc[i] - m_run);
        l_run += (p[0] + p[1]) + (p[2] + p[3]);
        // rows past the sequence hold what was there before, non-finite values too: they become zeros
        if (!full) {
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const bool in = 4 * q4 + i < n;
#pragma unroll
                    for (int j = 0; j < VW; ++j) vr[t][i][j] = in ? vr[t][i][j] : 0;
                }
        }
        if constexpr (F32) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int j = 0; j < C; ++j) acc[t][j] = mfma_f32(__uint_as_float(vr[t][i][j]), p[i], acc[t][j]);
        } else {
            auto parts = [&](float y0, float y1, float y2, float y3, diff_u32x2 (&pb)[3]) __attribute__((always_inline)) {
                uint32_t w[2][3];
                split3(y0, y1, w[0][0], w[0][1], w[0][2]);
                split3(y2, y3, w[1][0], w[1][1], w[1][2]);
#pragma unroll
                for (int k = 0; k < 3; ++k) pb[k] = diff_u32x2{w[0][k], w[1][k]};
            };
            // rest: the third parts, for f32 outputs (two leave 2^-16 of a probability, bf16 outputs 2^-8)
            auto add = [&](bool rest, diff_u32x2 x, const diff_u32x2 (&pb)[3], f32x4 &c) __attribute__((always_inline)) {
                c = rest ? mfma_bf16(x, pb[2], c) : mfma_bf16(x, pb[1], mfma_bf16(x, pb[0], c));
            };
            diff_u32x2 pb[3];
            if constexpr (QUANT) {
                put_scales(1, vsc, n);
                order_v();
            } else {
                parts(p[0], p[1], p[2], p[3], pb);
            }
            auto pass = [&](bool rest) __attribute__((always_inline)) {
                for (int h = 0; h < (FINE ? 32 : 1); h += FINE ? 1 << sg : 1) {
#pragma unroll
                    for (int t = 0; t < 2; ++t)
#pragma unroll
                        for (int g = 0; g < VW; ++g) {
                            const uint32_t w[4] = {vr[t][0][g], vr[t][1][g], vr[t][2][g], vr[t][3][g]};
                            if constexpr (QUANT) {
#pragma unroll
                                for (int b = 0; b < 2 && 2 * g + b < KS; ++b) {
                                    // the scales, folded into the probabilities; groups of 8 or 16 as in the scores
                                    const int col = 2 * g + 1 < KS || b ? 4 * (r16 & 7) + 2 * (r16 >> 3) : 2 * r16;
                                    const uint32_t mine = !FINE || (col >= h && col < h + (1 << sg)) ? ~0u : 0u;
                                    const uint32_t wm[4] = {w[0] & mine, w[1] & mine, w[2] & mine, w[3] & mine};
                                    const f32x4 vs = s_scale[wave][1][t][FINE ? (32 * (2 * g + b) + h) >> sg : 2 * g + b][q4];
                                    diff_u32x2 x[2];
                                    if (b) codes_by_row<DT, true>(wm, x);
                                    else codes_by_row<DT, false>(wm, x);
                                    parts(p[0] * vs[0], p[1] * vs[1], p[2] * vs[2], p[3] * vs[3], pb);
#pragma unroll
                                    for (int e = 0; e < 2; ++e) add(rest, x[e], pb, acc[t][2 * (2 * g + b) + e]);
                                }
                            } else {
                                add(rest, diff_u32x2{halves<false>(w[0], w[1]), halves<false>(w[2], w[3])}, pb, acc[t][2 * g]);
                                add(rest, diff_u32x2{halves<true>(w[0], w[1]), halves<true>(w[2], w[3])}, pb, acc[t][2 * g + 1]);
                            }
                        }
                }
            };
            pass(false);
            if (wide_out) pass(true);
        }
        load_v(more);
        if (end) emit(seq);
    }
}

// One query pair of one sequence: the pieces of its two rows folded by
// log-sum-exp, WH waves sharing them, then the output row.  An empty sequence
// gives zeros; lengths outside the table are counted.
template <int D, int WH>
__global__ __launch_bounds__(64 * WH) void diff_decode_merge_kernel(DiffDecodeArgs a) {
    constexpr int V = D / 32, kBatch = 8;
    __shared__ float s_ml[WH][2][2];
    __shared__ float s_o[WH][2][V][64];
    const int b = blockIdx.x, h = blockIdx.y, lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int p0 = a.prefix[b], p1 = a.prefix[b + 1], chunk = a.prefix[a.batch + 1];
    const int len = a.lens[b];
    const int64_t max_len = (int64_t)a.max_blocks * a.block_size;
    if (threadIdx.x == 0 && h == 0 && (len < 0 || len > max_len)) atomicAdd(a.errors, 1ull);
    if (p0 == p1) {
        if (wave == 0)
            for (int i = lane; i < 2 * D; i += 64) diff_store(a.e, ((int64_t)b * a.pairs + h) * (2 * D) + i, 0.0f);
        return;
    }
    const int w0 = p0 / chunk, w1 = (p1 - 1) / chunk;
    if (w0 == w1) return;                              // written by its slice
    const int n = w1 - w0 + 1;
    DiffTail<V> tail;
    tail.load(a.e, b, h, lane);                        // along with the pieces
    const int kp = h / a.group, j = h % a.group;
    const int hh = kp * a.row_tiles + j / 8;
    DiffFold<V> c;
    c.clear();
    for (int q0 = wave; q0 < n; q0 += WH * kBatch) {
        float pm[kBatch][2], pl[kBatch][2], po[kBatch][2][V];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const bool in = q0 + WH * i < n;
            const int p = in ? q0 + WH * i : q0;
            const int64_t row = ((int64_t)hh * a.slots + part_row(w0 + p, b, p == 0)) * 16 + (j & 7);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                pm[i][k] = in ? a.part_ml[(row + 8 * k) * 2] : -INFINITY;
                pl[i][k] = in ? a.part_ml[(row + 8 * k) * 2 + 1] : 0.0f;
                diff_load<V>(a.part_o + (row + 8 * k) * (2 * D) + V * lane, po[i][k]);
            }
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i)
#pragma unroll
            for (int k = 0; k < 2; ++k) c.fold(k, pm[i][k], pl[i][k], po[i][k]);
    }
    if constexpr (WH > 1) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            if (lane == 0) {
                s_ml[wave][k][0] = c.m[k];
                s_ml[wave][k][1] = c.l[k];
            }
#pragma unroll
            for (int i = 0; i < V; ++i) s_o[wave][k][i][lane] = c.o[k][i];
        }
        __syncthreads();
        if (wave != 0) return;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            float top = -INFINITY;
#pragma unroll
            for (int w = 0; w < WH; ++w) top = fmaxf(top, s_ml[w][k][0]);
            c.m[k] = top;
            c.l[k] = 0.0f;
#pragma unroll
            for (int i = 0; i < V; ++i) c.o[k][i] = 0.0f;
#pragma unroll
            for (int w = 0; w < WH; ++w) {
                const float m = s_ml[w][k][0], f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - top);
                c.l[k] += m == -INFINITY ? s_ml[w][k][1] : s_ml[w][k][1] * f;      // a NaN of it stays
#pragma unroll
                for (int i = 0; i < V; ++i) c.o[k][i] += s_o[w][k][i][lane] * f;
            }
        }
    }
    diff_finish<V>(a.e, a.pairs, c, tail, lane);
}

template <int D, int DT>
hipError_t launch_dt(const DiffDecodeArgs &a, hipStream_t s) {
    constexpr bool QUANT = DT == AIR_KV_INT8 || DT == AIR_KV_FP8, F32 = DT == AIR_KV_F32;
    const int64_t waves = (int64_t)a.kv_pairs * a.row_tiles * a.slices;
    const dim3 blocks((unsigned)((waves + kWaves - 1) / kWaves));
    const bool wide = a.q_dtype == AIR_KV_F32 || a.e.out_dtype == AIR_KV_F32, fine = QUANT && a.scale_group != 32;
    if (fine) hipLaunchKernelGGL((diff_decode_kernel<D, DT, true, QUANT>), blocks, dim3(kThreads), 0, s, a);
    else if (F32 || wide) hipLaunchKernelGGL((diff_decode_kernel<D, DT, true, false>), blocks, dim3(kThreads), 0, s, a);
    else hipLaunchKernelGGL((diff_decode_kernel<D, DT, F32, false>), blocks, dim3(kThreads), 0, s, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const dim3 grid((unsigned)a.batch, (unsigned)a.pairs);
    // waves enough that an average sequence's pieces take each one round trip
    const int64_t tiles = ((int64_t)a.max_blocks * a.block_size + 15) / 16, pieces = std::min<int64_t>(a.slices / a.batch, tiles);
    if (pieces > 32) hipLaunchKernelGGL((diff_decode_merge_kernel<D, 16>), grid, dim3(1024), 0, s, a);
    else if (pieces > 8) hipLaunchKernelGGL((diff_decode_merge_kernel<D, 4>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((diff_decode_merge_kernel<D, 1>), grid, dim3(64), 0, s, a);
    return hipGetLastError();
}

template <int D>
hipError_t launch_d(const DiffDecodeArgs &a, int dtype, hipStream_t s) {
    return dtype == AIR_KV_F32    ? launch_dt<D, AIR_KV_F32>(a, s)
           : dtype == AIR_KV_BF16 ? launch_dt<D, AIR_KV_BF16>(a, s)
           : dtype == AIR_KV_INT8 ? launch_dt<D, AIR_KV_INT8>(a, s)
                                  : launch_dt<D, AIR_KV_FP8>(a, s);
}

size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }

}  // namespace

// A slice for every wave slot, at most batch * max_splits.  The workspace holds
// the tile prefix and the chunk, then a partial row of 16 rows for every cut
// piece there can be.
DiffDecodePlan plan_diff_decode(const air_kv_pool &p, int32_t n_q_heads, int32_t batch, int32_t max_blocks,
                                int32_t max_splits) {
    DiffDecodePlan pl;
    const int kv_pairs = p.desc.n_kv_heads / 2;
    pl.group = n_q_heads / p.desc.n_kv_heads;
    pl.row_tiles = (pl.group + 7) / 8;
    const int64_t tiles_per_seq =
        std::max<int64_t>(1, std::min<int64_t>(((int64_t)max_blocks * p.desc.block_size + 15) / 16, ((int64_t)INT32_MAX + 15) / 16));
    // tiles of a launch in 32 bits, with room for the window of 64 past the last
    const int64_t nb = std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(batch, kMaxBatch), (INT32_MAX - 65536) / tiles_per_seq));
    const int64_t per_slice = (int64_t)kv_pairs * pl.row_tiles;
    const int64_t waves = (int64_t)p.cus * 4 * kWavesPerSimd;
    const int64_t sl = std::min<int64_t>((waves + per_slice - 1) / per_slice, nb * max_splits);
    pl.batch_per_launch = (int32_t)nb;
    pl.slices = (int32_t)sl;
    pl.slots = (int32_t)part_rows(sl, nb);
    const size_t rows = (size_t)per_slice * pl.slots * 16;
    pl.ws_bytes = align256((size_t)(nb + 2) * 4) + align256(rows * 2 * 4) + rows * 2 * p.desc.head_dim * 4;
    return pl;
}

hipError_t launch_diff_decode(const air_kv_pool &p, hipStream_t s, const DiffDecodePlan &plan, const void *q,
                              int32_t q_dtype, int32_t n_q_heads, const int32_t *tables, const int32_t *lens,
                              int32_t batch, int32_t max_blocks, float scale, int32_t max_splits, const DiffOut &out,
                              void *workspace) {
    const int d = p.desc.head_dim;
    DiffDecodeArgs a{};
    a.q_dtype = q_dtype;
    a.n_q_heads = n_q_heads;
    a.pairs = n_q_heads / 2;
    a.kv_pairs = p.desc.n_kv_heads / 2;
    a.row_tiles = plan.row_tiles;
    a.group = plan.group;
    a.max_blocks = max_blocks;
    a.slices = plan.slices;
    a.slots = plan.slots;
    const int per_slice = a.kv_pairs * a.row_tiles;
    a.simd_slices = (4 * p.cus + per_slice - 1) / per_slice;
    a.max_splits = max_splits;
    a.scale_log2 = scale * 1.4426950408889634f;
    a.n_kv_heads = p.desc.n_kv_heads;
    a.block_size = p.desc.block_size;
    a.scale_group = p.desc.scale_group;
    a.head_dim = d;
    a.num_blocks = p.desc.num_blocks;
    a.k_pages = p.k_pages;
    a.v_pages = p.v_pages;
    a.k_scales = p.k_scales;
    a.v_scales = p.v_scales;
    a.errors = p.errors;
    char *ws = (char *)workspace;
    const size_t rows = (size_t)per_slice * plan.slots * 16;
    a.prefix = (int32_t *)ws;
    ws += align256((size_t)(plan.batch_per_launch + 2) * 4);
    a.part_ml = (float *)ws;
    ws += align256(rows * 2 * 4);
    a.part_o = (float *)ws;
    for (int32_t b0 = 0; b0 < batch; b0 += plan.batch_per_launch) {
        a.batch = std::min(batch - b0, plan.batch_per_launch);
        a.q = (const char *)q + (int64_t)b0 * n_q_heads * d * (q_dtype == AIR_KV_F32 ? 4 : 2);
        a.tables = tables + (int64_t)b0 * max_blocks;
        a.lens = lens + b0;
        a.e = out;
        a.e.lam = out.lam + (int64_t)b0 * out.lam_stride;
        a.e.out = (char *)out.out + (int64_t)b0 * n_q_heads * d * (out.out_dtype == AIR_KV_F32 ? 4 : 2);
        hipError_t e = d == 128 ? launch_d<128>(a, p.desc.dtype, s)
                       : d == 96 ? launch_d<96>(a, p.desc.dtype, s)
                       : d == 64 ? launch_d<64>(a, p.desc.dtype, s)
                                 : launch_d<32>(a, p.desc.dtype, s);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace airkv
