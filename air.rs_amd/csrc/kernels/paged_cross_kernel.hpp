// The kernel of cross attention over pages (formulas and work division: paged_cross.hpp), for
// paged_cross_16.hip and paged_cross_f32.hip.
//
// A wave holds 32 rows and walks keys 32 at a time, once, with a running base and sum:
//   S   = K . Q^T      v_mfma_f32_32x32x16_bf16, lane (n, h) holds 16 of the 32 keys of row n
//   O^T += V^T . P^T   the same instruction; its contraction takes the keys in the order in
//                      which the lanes hold P, so P never moves
// Operands by kind (CrossKind):
//   kBf16   bf16 queries over bf16 pages.  Probabilities of bf16's 8 bits would err about as much as the output's
//           rounding (2.3e-3 of its norm with both, 1.7e-3 with 11 bits or more): many rows round them to f16
//           and multiply values as f16 (CONVERT), few rows take them in two bf16 parts, 16 bits
//   kCodes  bf16 queries over 1-byte pages: everything as f16 (11 bits), under powers of two: of a
//           query row's, of a tile's keys (from the largest scale of those that are not all zeros,
//           known a barrier before the tile is staged) and of the values' (the smallest so far)
//   kParts  f32 precision over bf16 pages, kFloats over f32 and kWide over 1-byte ones: bf16 parts
//           that hold all 24 bits, of queries and probabilities and (not kParts) of keys and values; products with
//           i + j < 3 are formed
// Keys and values are staged in LDS as rows, padded or their 16-byte chunks placed so that neither
// the rows' reads nor the values' transposing reads meet in a bank.
//
// Many rows (16-bit products, heads up to 128) are bound by the products and the arithmetic between them,
// about as much of either: a step's exponentials run beside the next step's scores and the last one's
// values (8192 states, 4096 tokens of 32 heads of 128: 590 us, 930 TFLOP/s).
// Few rows are bound by the pages' reads (64 tokens, 512 to 4096 states, 8 heads of 128, bf16: 109 us, 5.2
// TB/s; one f32 token over each of 32 sequences 110 us, 4.8; 1-byte pages 3.4, by their conversion).
//
// Many rows: each wave has 32 rows of its own and all take the same keys; a tile is loaded two
// ahead into registers and staged one ahead where two buffers fit.  Few rows (PRIVATE): a
// workgroup's waves share 32 rows, each takes 32 keys of a tile and stages them itself, and none waits
// for another until the block ends.  SPLIT: values take the keys' place when the scores are there, half
// the LDS (all but kCodes, whose values' scales are looked through beside the keys').
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "codecs.hpp"
#include "decode_slices.hpp"
#include "paged_cross.hpp"

namespace airkv {

typedef float cross_f32x16 __attribute__((ext_vector_type(16)));
typedef float cross_f32x4 __attribute__((ext_vector_type(4)));
typedef float cross_f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 cross_bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 cross_bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 cross_f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 cross_f16x2 __attribute__((ext_vector_type(2)));
typedef uint32_t cross_u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t cross_u32x2 __attribute__((ext_vector_type(2)));

enum CrossKind { kBf16, kCodes, kParts, kFloats, kWide };

constexpr int kCrossBuffer = 0x00020000;           // a raw buffer's last word
constexpr int kCrossStream = 2;                    // non-temporal: pages are read once (64 single tokens 125 -> 111 us)
constexpr int kCrossNowhere = 0x40000000;          // an offset outside of every buffer: reads zeros

// Rows of keys and of values in LDS, bytes apart.  Keys: 16 bytes more than a whole number of
// 256, or as good.  Values are read four rows at a time, 64 bytes of each: where a row is a whole
// number of 256 bytes, the chunks of row r are placed 64 (r % 4) bytes away (exclusive or).
constexpr int cross_k_stride(int d) { return 2 * d + 16; }
constexpr bool cross_v_xor(int d) { return 2 * d % 256 == 0; }
constexpr int cross_v_stride(int d) { return cross_v_xor(d) || 2 * d / 64 % 2 ? 2 * d : 2 * d + 64; }
constexpr int cross_tile_bytes(int d, int parts, int keys) { return keys * parts * (cross_k_stride(d) + cross_v_stride(d)); }
// Waves of a workgroup, and workgroups a CU: registers leave room for two waves a SIMD, or (queries in
// three parts and their sums, the largest heads) one.  Two workgroups of four waves do not wait at each
// other's barriers, but stage every tile twice: few rows stage their own in any case (heads of 64, two in
// place of one: 104 -> 92 us; three, where registers allow them, 92), many rows gain from it at small heads.
constexpr bool cross_pipe(int d, int qp, bool few) { return !few && qp == 1 && d <= 128; }
constexpr int cross_waves(int d, int qp, bool few) { return few || (cross_pipe(d, qp, few) && d <= 64) || (qp == 3 ? d >= 96 : d >= 192) ? 4 : 8; }
constexpr int cross_groups(int d, int qp, bool few) { return few ? (d <= (qp == 3 ? 64 : 128) ? 2 : 1) : cross_pipe(d, qp, few) && d <= 64 ? 2 : 1; }
// What a workgroup's tiles may take of a CU's 160 KB.
constexpr int cross_lds(int groups) { return 160 * 1024 / groups - 7 * 1024; }
// What 32 keys, and then their values (split) or both, take of a wave that stages its own; whether
// there is room for all.  (Where registers do not suffice it pays still: f32 rows over bf16 heads of 192
// 101 us with 75 spilled, 171 with waves that share a tile.)
constexpr int cross_region(int d, int parts, bool split) {
    return !split ? cross_tile_bytes(d, parts, 32) : 32 * parts * (cross_k_stride(d) > cross_v_stride(d) ? cross_k_stride(d) : cross_v_stride(d));
}
constexpr bool cross_private(int d, int parts, int qp, bool few, bool split) {
    return few && cross_waves(d, qp, few) * cross_region(d, parts, split) <= cross_lds(1);
}
// Keys of a tile that one wave takes, in 32s.
constexpr int cross_sub(int d, int kp) { return cross_tile_bytes(d, kp, 64) <= cross_lds(1) ? 2 : 1; }

template <bool F16> __device__ __forceinline__ cross_f32x16 cross_mfma(cross_u32x4 a, cross_u32x4 b, cross_f32x16 c) {
    if constexpr (F16)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(cross_f16x8, a), __builtin_bit_cast(cross_f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(cross_bf16x8, a), __builtin_bit_cast(cross_bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ uint32_t cross_f16_pair(float x, float y) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((cross_f32x2{x, y}), cross_f16x2));
}
__device__ __forceinline__ uint32_t cross_bf16_pair(float x, float y) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((cross_f32x2{x, y}), cross_bf16x2));
}
// x, y as bf16 parts whose sum they are, 8 bits each, cut off rather than rounded (the largest
// float stays finite).
__device__ __forceinline__ void cross_split(float x, float y, uint32_t (&p)[3]) {
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        p[i] = __builtin_amdgcn_perm(__float_as_uint(y), __float_as_uint(x), 0x07060302u);
        x -= __uint_as_float(__float_as_uint(x) & 0xFFFF0000u);
        y -= __uint_as_float(__float_as_uint(y) & 0xFFFF0000u);
    }
}
// x, y as P parts: three, two bf16 ones (rounded, and what that leaves: 16 bits), or one f16 one.
template <int P> __device__ __forceinline__ void cross_parts(float x, float y, uint32_t (&p)[P]) {
    if constexpr (P == 3) cross_split(x, y, p);
    else if constexpr (P == 2) {
        p[0] = cross_bf16_pair(x, y);
        p[1] = cross_bf16_pair(x - __uint_as_float(p[0] << 16), y - __uint_as_float(p[0] & 0xFFFF0000u));
    } else p[0] = cross_f16_pair(x, y);
}
// 2^e, e clamped to the normal numbers; the exponent of a normal number.
__device__ __forceinline__ float cross_pow2(int e) { return __uint_as_float((uint32_t)(min(max(e, -126), 127) + 127) << 23); }
__device__ __forceinline__ int cross_exponent(float x) { return (int)((__float_as_uint(x) >> 23) & 0xFF) - 127; }
// The sum of a pair of f16 and c; ones: cross_ones (an inline constant would not be read as a pair).
__device__ __forceinline__ uint32_t cross_ones() {
    uint32_t x = 0x3C003C00u;
    asm("" : "+s"(x));
    return x;
}
__device__ __forceinline__ float cross_add_pair(uint32_t p, uint32_t ones, float c) {
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(cross_f16x2, p), __builtin_bit_cast(cross_f16x2, ones), c, false);
}
// The values of the four 1-byte codes in w times their scale.  SMALL: |s| is below 2^100; int8 codes
// then take two instructions each, (code + 128) s - 128 s in one step (128 s is exact, and the
// unsigned byte's conversion takes it from its place).
template <int DT, bool SMALL> __device__ __forceinline__ cross_f32x4 cross_codes(uint32_t w, float s) {
    if constexpr (DT == AIR_KV_FP8) {
        const cross_f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
        return cross_f32x4{lo[0] * s, lo[1] * s, hi[0] * s, hi[1] * s};
    } else if constexpr (SMALL) {
        const uint32_t u = w ^ 0x80808080u;
        const float off = -128.0f * s;
        return cross_f32x4{__builtin_fmaf((float)(u & 0xFFu), s, off), __builtin_fmaf((float)((u >> 8) & 0xFFu), s, off),
                           __builtin_fmaf((float)((u >> 16) & 0xFFu), s, off), __builtin_fmaf((float)(u >> 24), s, off)};
    } else return cross_f32x4{(float)(int8_t)w * s, (float)(int8_t)(w >> 8) * s, (float)(int8_t)(w >> 16) * s, (float)(int8_t)(w >> 24) * s};
}
// The largest of the wave's lanes' x >= 0.
__device__ __forceinline__ float cross_wave_max(float x) {
    return __uint_as_float(__builtin_amdgcn_readlane(wave_scan((int)__float_as_uint(x), [](int a, int b) { return a > b ? a : b; }), 63));
}
__device__ __forceinline__ int64_t cross_uniform(int64_t x) {
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)x), hi = __builtin_amdgcn_readfirstlane((uint32_t)(x >> 32));
    return (int64_t)((uint64_t)hi << 32 | lo);
}
// Four outputs of a row from element `at` on.
__device__ __forceinline__ void cross_store4(const CrossArgs &a, int64_t at, cross_f32x4 x) {
    if (a.out_dtype == AIR_KV_F32) *reinterpret_cast<cross_f32x4 *>((float *)a.out + at) = x;
    else *reinterpret_cast<cross_u32x2 *>((uint16_t *)a.out + at) = cross_u32x2{cross_bf16_pair(x[0], x[1]), cross_bf16_pair(x[2], x[3])};
}

template <int D, CrossKind KIND, bool FEW>
struct CrossShape {
    static constexpr int KP = KIND == kFloats || KIND == kWide ? 3 : 1, QP = KIND == kParts ? 3 : KP;
    static constexpr int WAVES = cross_waves(D, QP, FEW);
    static constexpr bool SPLIT = KIND != kCodes, PRIVATE = cross_private(D, KP, QP, FEW, SPLIT), PIPE = cross_pipe(D, QP, FEW);
    static constexpr int WK = PRIVATE ? WAVES : 1, SUB = PRIVATE ? 1 : cross_sub(D, KP);       // waves that share rows; 32s of a tile's keys of one
    static constexpr int ROWS = 32 * (WAVES / WK), TK = 32 * WK * SUB;
    static constexpr int REGION = cross_region(D, KP, SPLIT), TILE = PRIVATE ? WAVES * REGION : cross_tile_bytes(D, KP, TK);
    static constexpr int GROUPS = cross_groups(D, QP, FEW) == 2 && TILE <= cross_lds(2) ? 2 : 1;
    static constexpr int NB = PIPE ? 3 : !PRIVATE && 2 * TILE <= cross_lds(GROUPS) ? 2 : 1;
    static constexpr int WAVES_SIMD = WAVES / 4 * GROUPS;
    // Values of bf16 pages as f16, under a power of two, converted once for a block's rows.  (8192 states of 128: bf16
    // probabilities 560 us, f16 ones 590, in two bf16 parts with products of both 736; 2000 states, heads of 160 / 256:
    // 116 / 275, 121 / 309, 149 / 321.  Few rows, bound by the pages, lose nothing to the parts.)
    static constexpr bool CONVERT = KIND == kBf16 && !PRIVATE;
    static constexpr int PP = KIND == kBf16 && !CONVERT ? 2 : QP;      // parts of probabilities
};

template <int D, CrossKind KIND, bool FEW>
__global__ __launch_bounds__((CrossShape<D, KIND, FEW>::WAVES * 64))
__attribute__((amdgpu_waves_per_eu(CrossShape<D, KIND, FEW>::WAVES_SIMD, CrossShape<D, KIND, FEW>::WAVES_SIMD)))
void paged_cross_kernel(CrossArgs a) {
    typedef CrossShape<D, KIND, FEW> S;
    constexpr bool F16 = KIND == kCodes, CONVERT = S::CONVERT, V16 = F16 || CONVERT, PRIVATE = S::PRIVATE, SPLIT = S::SPLIT, PIPE = S::PIPE;
    constexpr int KP = S::KP, QP = S::QP, PP = S::PP, WAVES = S::WAVES, WK = S::WK, SUB = S::SUB, ROWS = S::ROWS, TK = S::TK, NB = S::NB, THREADS = 64 * WAVES;
    static_assert(!F16 || PRIVATE || NB >= 2, "tiles' scales are looked through a tile before they are staged");
    constexpr int KST = cross_k_stride(D), VST = cross_v_stride(D);
    constexpr int STAGED = PRIVATE ? 32 : TK;          // keys side by side
    constexpr int KPLANE = STAGED * KST, VPLANE = STAGED * VST, VAT = PRIVATE && SPLIT ? 0 : KP * KPLANE;      // a part's rows; where values begin
    constexpr int KS = D / 16, CT = D / 32;            // steps of the first product, 32-column tiles of the second
    // Staging: a wave takes SH of the tile's 16-key halves of keys or values, WR rows a pass, LPR lanes
    // a row (a power of two: some idle where D / 8 is none), 8 elements a lane.
    constexpr int LPR = D <= 32 ? 4 : D <= 64 ? 8 : D <= 128 ? 16 : 32, WR = 64 / LPR, NPH = 16 / WR;
    // (CONVERT with one half for each wave: eight rows of keys and eight of values instead, so that no wave has more
    // to convert than another: 610 -> 592 us for 8192 states of 128)
    constexpr int SH = 2 * TK / 16 / WAVES;
    constexpr bool EIGHT = CONVERT && SH == 1;
    constexpr int UNITS = EIGHT ? 2 : SH, UP = EIGHT ? NPH / 2 : NPH, NP = UNITS * UP;
    static_assert(UP >= 1, "whole passes");
    static_assert(SH >= 1 && SH * WAVES * 16 == 2 * TK && (SH == 1 || SH % 2 == 0), "whole halves");
    constexpr int EXTRA = cross_extra(FEW);
    constexpr int kOnce = FEW ? kCrossStream : 0;
    constexpr int JOIN = WAVES * 64 * 16 * 4;          // bytes of a column tile of every wave's sums, at a block's end
    constexpr int MEM = NB * S::TILE > JOIN || WK == 1 ? NB * S::TILE : JOIN;
    constexpr int CR = MEM / JOIN < CT ? MEM / JOIN : CT;      // column tiles joined at once (WK > 1)
    __shared__ int64_t s_pre[kCrossBatch + 1];
    __shared__ int64_t s_sum[WAVES];
    __shared__ int32_t s_ok[8][TK / 16];               // whether a tile's 16-key halves are in the pool
    __shared__ uint32_t s_top[3][2];                   // a tile's largest scale of keys and of values, as bits
    __shared__ float4 s_ml[WAVES][32];
    __shared__ __align__(16) uint8_t s_mem[MEM];

    const int tid = threadIdx.x, lane = tid & 63, hf = lane >> 5, r32 = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int rg = wave / WK, wk = wave % WK;          // 32 rows; which keys of a tile
    // workgroups of one K/V head take every heads-th place: with eight heads, one XCD's (its L2
    // then sees one head's keys and values)
    const int head = blockIdx.x % a.heads, w = blockIdx.x / a.heads;
    const int64_t cell = (int64_t)head * a.slices + w;

    // units before each sequence
    int idle = 0;                                      // whether some sequence has rows and no work
    {
        const int per = (a.batch + THREADS - 1) / THREADS, lo = min(tid * per, a.batch), hi = min(lo + per, a.batch);
        int64_t mine = 0;
        for (int b = lo; b < hi; ++b) {
            const CrossSeq s = cross_seq(a, b);
            const int64_t u = cross_units<ROWS, TK, EXTRA>(s);
            idle |= !s.ok || (s.rows && !s.len);
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
        idle = __syncthreads_or(idle);
        int64_t run = incl - mine;
        for (int i = 0; i < wave; ++i) run += s_sum[i];
        for (int b = lo; b < hi; ++b) {
            run += s_pre[b + 1];
            s_pre[b + 1] = run;
        }
        __syncthreads();
    }
    // sequences without work: rows of refused ones (counted) and of empty ones are zeros
    if (idle) {
        for (int b = w; b < a.batch; b += a.slices) {
            const CrossSeq s = cross_seq(a, b);
            if (s.ok && (s.len || !s.rows)) continue;
            if (!s.ok && head == 0 && tid == 0) atomicAdd(a.errors, 1ull);
            const int32_t r0 = a.cu[b], r1 = a.cu[b + 1];
            if (r0 < 0 || r1 > a.total_q || r1 < r0) continue;
            const int64_t n = (int64_t)(r1 - r0) * a.group * (D / 4);
            for (int64_t i = tid; i < n; i += THREADS) {
                const int64_t row = i / (D / 4), c = i % (D / 4) * 4;
                cross_store4(a, ((r0 + row / a.group) * a.q_heads + head * a.group + row % a.group) * D + c, cross_f32x4{0.0f, 0.0f, 0.0f, 0.0f});
            }
        }
    }
    const int64_t units = cross_uniform(s_pre[a.batch]);
    const int64_t chunk = (units + a.slices - 1) / a.slices;
    int64_t u = w * chunk;
    const int64_t end = u + chunk < units ? u + chunk : units;
    int4 begun = {0, 0, 0, 0};

    // this lane's place in every pass
    const int p_c = lane % LPR;
    const bool p_in = p_c < D / 8;
    constexpr bool CODES = KIND == kCodes || KIND == kWide;
    constexpr int esize = CODES ? 1 : KIND == kFloats ? 4 : 2;
    const int p_off = p_in ? (lane / LPR * D + 8 * p_c) * esize : kCrossNowhere;
    const int nsc = CODES ? D >> a.sg_log2 : 0;
    const int p_sc = p_in ? (lane / LPR * nsc + (8 * p_c >> a.sg_log2)) * 4 : kCrossNowhere;

    // half j of this wave's: of values (else keys), and which of the tile's; the first of its rows
    auto of_values = [&](int j) __attribute__((always_inline)) { return UNITS == 1 ? wave >= WAVES / 2 : j >= UNITS / 2; };
    auto half_of = [&](int j) __attribute__((always_inline)) { return EIGHT ? wave / 2 : SH == 1 ? wave % (WAVES / 2) : wave * (SH / 2) + j % (SH / 2); };
    const int row0 = EIGHT ? 8 * (wave % 2) : 0;

    const uint32_t ones = cross_ones();
    // A SIMD has waves i and i + 4 of a workgroup: the second goes first, so that the two get out of
    // phase and one's products run beside the other's arithmetic.
    if (WAVES == 8 && wave >= 4) __builtin_amdgcn_s_setprio(1);
    int b = 0;
    if (u < end) {
        int lo = 0, hi = a.batch;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (s_pre[mid] <= u) lo = mid;
            else hi = mid;
        }
        b = __builtin_amdgcn_readfirstlane(lo);
    }
    while (u < end) {
        while (cross_uniform(s_pre[b + 1]) <= u) ++b;
        CrossSeq sq = cross_seq(a, b);
        sq.row0 = __builtin_amdgcn_readfirstlane(sq.row0);
        sq.rows = __builtin_amdgcn_readfirstlane(sq.rows);
        sq.len = __builtin_amdgcn_readfirstlane(sq.len);
        const int nt = cross_tiles<TK>(sq);
        const int64_t in = u - cross_uniform(s_pre[b]);
        const int blk = (int)(in / (nt + EXTRA)), at = (int)(in - (int64_t)blk * (nt + EXTRA));
        const int64_t left = nt + EXTRA - at, mine = end - u < left ? end - u : left;
        // a block's first EXTRA units are its beginning
        const int t0 = at < EXTRA ? 0 : at - EXTRA;
        const int t1 = at + (int)mine < EXTRA ? 0 : at + (int)mine - EXTRA;
        u += mine;
        if (t0 == t1) continue;                        // the slice ends before the block's first tile
        const bool whole = t0 == 0 && t1 == nt;
        const int tiles = t1 - t0;
        const int64_t key0 = (int64_t)t0 * TK;
        const int32_t *table = a.tables + (int64_t)b * a.max_blocks;

        // rows 32 rg .. +31 of the block
        const bool any = blk * ROWS + 32 * rg < sq.rows;
        const int row = blk * ROWS + 32 * rg + r32;    // of the sequence's at this K/V head
        const bool live = row < sq.rows;
        const int row_at = live ? row : sq.rows - 1;
        const int64_t io = ((int64_t)(sq.row0 + row_at / a.group) * a.q_heads + head * a.group + row_at % a.group) * D;

        // Q^T as the B operand: lane (n, h) holds elements 16 s + 8 h .. +8 of row n
        cross_u32x4 qf[QP][KS];
        int qe = 0;                                    // (kCodes: the power of two they are under)
        if (KIND == kBf16 || KIND == kCodes || a.q_dtype == AIR_KV_BF16) {
            const uint16_t *q = (const uint16_t *)a.q + io + 8 * hf;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                qf[0][s] = *reinterpret_cast<const cross_u32x4 *>(q + 16 * s);
#pragma unroll
                for (int p = 1; p < QP; ++p) qf[p][s] = cross_u32x4{0, 0, 0, 0};
            }
        } else {
            const float *q = (const float *)a.q + io + 8 * hf;
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const cross_f32x4 x = *reinterpret_cast<const cross_f32x4 *>(q + 16 * s + 4 * i);
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        uint32_t p[QP];
                        cross_parts<QP>(x[2 * j], x[2 * j + 1], p);
#pragma unroll
                        for (int k = 0; k < QP; ++k) qf[k][s][2 * i + j] = p[k];
                    }
                }
        }
        if constexpr (F16) {
            // the row's largest element to [2^4, 2^5): bf16's 8 bits are exact in f16 down to 2^-17, 2^-21 of it
            float top = 0.0f;
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    top = fmaxf(top, fmaxf(__builtin_fabsf(__uint_as_float(qf[0][s][j] << 16)),
                                           __builtin_fabsf(__uint_as_float(qf[0][s][j] & 0xFFFF0000u))));
            const float fq = cross_pow2(4 - cross_exponent(max_x32(top)));
            qe = cross_exponent(fq);
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    qf[0][s][j] = cross_f16_pair(__uint_as_float(qf[0][s][j] << 16) * fq, __uint_as_float(qf[0][s][j] & 0xFFFF0000u) * fq);
        }
        cross_f32x16 acc[CT];
        // Probabilities are held 2^(score - base), the base kDown above every score so far: 2^24 of
        // them sum to 1 at most, so that values near the largest float do too.  (f16 ones up to
        // 2^15, so that they keep 11 bits down to 2^-25 of the largest; values are below 2^16 there.)
        // A base is taken kSlack further up, so that it seldom changes: where a score passes lim.
        constexpr float kSlack = 4.0f, kFar = 0x1p20f;
        float kDown, base, lim, l_run;
        auto clear = [&](float down) __attribute__((always_inline)) {
            kDown = down;
            base = lim = -INFINITY;
            l_run = 0.0f;
#pragma unroll
            for (int c = 0; c < CT; ++c)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[c][i] = 0.0f;
        };
        clear(V16 ? -15.0f : 24.0f);

        struct Raw {                                   // a tile on its way
            cross_u32x4 w[NP][KIND == kFloats ? 2 : 1];
            float s[CODES ? NP : 1];
        } raw, next;                                   // (next: kCodes, a tile further ahead)
        float fk = 1.0f, fk_next = 1.0f, fv = 0.0f, fv_next = 0.0f;    // kCodes: powers of two (0: no value yet); CONVERT: fv
        int counted = 0;                               // tiles whose table entries are (CONVERT comes twice)
        // lane h: the entry of a tile's half h, read a tile before it is needed, and its block
        int32_t entry = 0, window = -1;
        auto fetch = [&](int t) __attribute__((always_inline)) {
            const int64_t key = key0 + (int64_t)t * TK + 16 * lane;
            entry = lane < TK / 16 && key < sq.len ? table[key >> a.bs_log2] : 0;
        };
        auto look_up = [&](int t) __attribute__((always_inline)) {
            const int64_t key = key0 + (int64_t)t * TK + 16 * lane;
            const bool there = t < tiles && lane < TK / 16 && key < sq.len, out = there && (entry < 0 || entry >= a.num_blocks);
            window = out || !there ? -1 : entry;
            // counted once: by the first block of rows at the first head
            if (head == 0 && blk == 0 && wave == 0 && (!CONVERT || t >= counted)) {
                const int n = __popcll(__ballot(out && (key & ((1 << a.bs_log2) - 1)) == 0));
                if (n && lane == 0) atomicAdd(a.errors, (unsigned long long)n);
            }
            if (CONVERT && t >= counted) counted = t + 1;
            if (!PRIVATE && wave == 0 && lane < TK / 16) s_ok[t % 8][lane] = window >= 0;
            fetch(t + 1);
        };
        // a tile's keys and values, or one of them (SPLIT)
        constexpr std::integral_constant<int, 0> kBoth{};
        constexpr std::integral_constant<int, 1> kKeys{};
        constexpr std::integral_constant<int, 2> kValues{};
        auto skip = [&](int j, auto part) __attribute__((always_inline)) {
            return decltype(part)::value && of_values(j) != (decltype(part)::value == 2);
        };
        auto load_tile = [&](int t, Raw &raw, auto part) __attribute__((always_inline)) {
#pragma unroll
            for (int j = 0; j < UNITS; ++j) {
                if (skip(j, part)) continue;
                const int half = half_of(j);
                const bool val = of_values(j);
                const int32_t e = __builtin_amdgcn_readlane(window, half);
                const int64_t rest = sq.len - (key0 + (int64_t)t * TK + 16 * half + row0);
                const int have = e < 0 || rest <= 0 ? 0 : rest < 16 - row0 ? (int)rest : 16 - row0;
                const int64_t prow = (((int64_t)(e < 0 ? 0 : e) * a.heads + head) << a.bs_log2) + (16 * half & ((1 << a.bs_log2) - 1)) + row0;
                const uint8_t *pages = (const uint8_t *)(val ? a.v_pages : a.k_pages) + prow * (D * esize);
                // rows past the sequence's end lie outside of the buffer: zeros
                const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void *)pages, (short)0, have * D * esize, kCrossBuffer);
                const float *scales = (val ? a.v_scales : a.k_scales) + prow * nsc;
                const __amdgpu_buffer_rsrc_t ss = __builtin_amdgcn_make_buffer_rsrc((void *)scales, (short)0, have * nsc * 4, kCrossBuffer);
#pragma unroll
                for (int k = 0; k < UP; ++k) {
                    const int i = j * UP + k;
                    if constexpr (KIND == kBf16 || KIND == kParts) {
                        raw.w[i][0] = __builtin_bit_cast(cross_u32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, p_off + k * WR * D * 2, 0, kOnce));
                    } else if constexpr (CODES) {
                        const cross_u32x2 x = __builtin_bit_cast(cross_u32x2, __builtin_amdgcn_raw_buffer_load_b64(rs, p_off + k * WR * D, 0, kOnce));
                        raw.w[i][0][0] = x[0];
                        raw.w[i][0][1] = x[1];
                        raw.s[i] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(ss, p_sc + k * WR * nsc * 4, 0, 0));
                    } else {
                        raw.w[i][0] = __builtin_bit_cast(cross_u32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, p_off + k * WR * D * 4, 0, kOnce));
                        raw.w[i][1] = __builtin_bit_cast(cross_u32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, p_off + k * WR * D * 4 + 16, 0, kOnce));
                    }
                }
            }
        };
        // kCodes: the largest finite scales of tile t (PRIVATE: of this wave's part), and the powers of two
        // they ask for.  (The scale 1 that the append gives a group of zeros does not count: lanes whose
        // codes are zeros leave theirs out.)
        auto mark = [&](int t, const Raw &raw, float &k, float &v) __attribute__((always_inline)) {
            if constexpr (F16) {
                const uint32_t sign = a.dtype == AIR_KV_FP8 ? 0x7F7F7F7Fu : ~0u;
                k = v = 0.0f;
#pragma unroll
                for (int i = 0; i < NP; ++i) {
                    const float x = __builtin_fabsf(raw.s[i]);
                    const float y = x < INFINITY && ((raw.w[i][0][0] | raw.w[i][0][1]) & sign) ? x : 0.0f;
                    if (of_values(i / UP)) v = fmaxf(v, y);
                    else k = fmaxf(k, y);
                }
                if (SH > 1 || !of_values(0)) k = cross_wave_max(k);
                if (SH > 1 || of_values(0)) v = cross_wave_max(v);
                if (!PRIVATE && lane == 0) {
                    if (SH > 1 || !of_values(0)) atomicMax(&s_top[t % 3][0], __float_as_uint(k));
                    if (SH > 1 || of_values(0)) atomicMax(&s_top[t % 3][1], __float_as_uint(v));
                }
            }
        };
        // codes are at most 448 (2^9): the largest value to 2^13 at most (an int8 one, 127, to 2^10 to 2^11, f16's
        // steps of 2^-24 being 2^-34 of it; an fp8 one to 2^11.8 to 2^12.8)
        auto keys_power = [&](float k) __attribute__((always_inline)) { fk_next = k == 0.0f ? 1.0f : cross_pow2(3 - cross_exponent(k)); };
        auto values_power = [&](float v) __attribute__((always_inline)) {
            // (kept as long as the largest stays below 2^15; it never grows)
            const float want = cross_pow2(3 - cross_exponent(v));
            fv_next = v == 0.0f ? fv_next : fv_next == 0.0f || fv_next > 4.0f * want ? want : fv_next;
        };
        // CONVERT: the values' power of two, from the largest of the first 64 * 8 of the slice's, which every wave
        // reads for itself: 1 where that lies in [2^-2, 2^10), else what brings it to 2^9, and 0, no f16 values, where
        // all are zeros.  f16 holds bf16's 8 bits from 2^-17 on, in steps of 2^-24 below (2^-22 of the largest and
        // less), up to 2^16; a value beyond that is found at the block's end, which is then computed again (a call of such
        // blocks alone takes 2.1 times as long, one of zeros first 1.2).
        auto sample = [&]() __attribute__((always_inline)) {
            const int32_t e = __builtin_amdgcn_readlane(window, 0);
            const int64_t rest = sq.len - key0, prow = ((int64_t)(e < 0 ? 0 : e) * a.heads + head) << a.bs_log2;
            const int have = e < 0 ? 0 : rest < 16 ? (int)rest : 16;
            const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((uint8_t *)a.v_pages + prow * (D * esize), (short)0, have * D * esize, kCrossBuffer);
            const cross_u32x4 w = __builtin_bit_cast(cross_u32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, p_off, 0, 0));
            float x = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                x = fmaxf(x, fmaxf(__builtin_fabsf(__uint_as_float(w[j] << 16)), __builtin_fabsf(__uint_as_float(w[j] & 0xFFFF0000u))));
            x = cross_wave_max(x);
            fv = x == 0.0f ? 0.0f : !(x < INFINITY) || (x >= 0x1p-2f && x < 0x1p10f) ? 1.0f : cross_pow2(9 - cross_exponent(x));
        };
        // (exact: values of bf16 pages as they are)
        constexpr std::integral_constant<bool, !CONVERT> kFast{};
        constexpr std::true_type kExact{};
        auto write_tile = [&](int t, const Raw &raw, auto part, auto exact) __attribute__((always_inline)) {
            uint8_t *mem = PRIVATE ? s_mem + wave * S::REGION : s_mem + t % NB * S::TILE;
            if constexpr (F16 && !PRIVATE) {
                keys_power(__uint_as_float(__builtin_amdgcn_readfirstlane(s_top[t % 3][0])));
                values_power(__uint_as_float(__builtin_amdgcn_readfirstlane(s_top[t % 3][1])));
            }
            // (the type is asked for once a tile; kWide asks at each chunk: all of a tile's, twice over, do not fit the registers)
            auto rows = [&](auto type, auto scaled) __attribute__((always_inline)) {
                constexpr int DT = decltype(type)::value;
#pragma unroll
                for (int i = 0; i < NP; ++i) {
                    if (skip(i / UP, part)) continue;
                    const bool val = of_values(i / UP);
                    const int at = 16 * (PRIVATE ? i / UP % (SH > 1 ? SH / 2 : 1) : half_of(i / UP)) + row0 + i % UP * WR + lane / LPR;
                    const int chunk = val && cross_v_xor(D) ? p_c ^ ((at & 3) << 2) : p_c;
                    uint8_t *to = mem + (val ? VAT + at * VST : at * KST) + 16 * chunk;
                    const int plane = val ? VPLANE : KPLANE;
                    cross_u32x4 y[KP];
                    if constexpr (DT == AIR_KV_BF16) {
                        y[0] = raw.w[i][0];
                        if (!decltype(exact)::value && val)
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const float lo = __uint_as_float(y[0][j] << 16), hi = __uint_as_float(y[0][j] & 0xFFFF0000u);
                                y[0][j] = decltype(scaled)::value ? cross_f16_pair(lo * fv, hi * fv) : cross_f16_pair(lo, hi);
                            }
                    } else {
                        float x[8];
                        if constexpr (DT == AIR_KV_F32) {
#pragma unroll
                            for (int j = 0; j < 8; ++j) x[j] = __uint_as_float(raw.w[i][KIND == kFloats ? j / 4 : 0][j % 4]);
                        } else {
                            // (scales of groups of zeros were left out: theirs may be any size; one that is not finite
                            // leaves NaN, 0 * s, to all of its group, zero codes too)
                            const float sc = F16 ? __builtin_fmaf(raw.s[i], 0.0f, __builtin_amdgcn_fmed3f(raw.s[i] * (val ? fv_next : fk_next), -0x1p100f, 0x1p100f))
                                                 : raw.s[i];
                            uint32_t w0 = raw.w[i][0][0], w1 = raw.w[i][0][1];
                            asm volatile("" : "+v"(w0), "+v"(w1));     // (not taken apart while on its way: four registers for one)
                            cross_f32x4 lo, hi;
                            if (KIND == kWide && a.dtype == AIR_KV_INT8) {
                                lo = cross_codes<AIR_KV_INT8, F16>(w0, sc);
                                hi = cross_codes<AIR_KV_INT8, F16>(w1, sc);
                            } else {
                                lo = cross_codes<DT, F16>(w0, sc);
                                hi = cross_codes<DT, F16>(w1, sc);
                            }
#pragma unroll
                            for (int j = 0; j < 4; ++j) { x[j] = lo[j]; x[4 + j] = hi[j]; }
                        }
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            uint32_t p[KP];
                            cross_parts<KP>(x[2 * j], x[2 * j + 1], p);
#pragma unroll
                            for (int k = 0; k < KP; ++k) y[k][j] = p[k];
                        }
                    }
#pragma unroll
                    for (int k = 0; k < KP; ++k)
                        if (p_in) *reinterpret_cast<cross_u32x4 *>(to + k * plane) = y[k];
                    // (parts of several chunks at once would not fit the registers)
                    if constexpr (KP == 3) __builtin_amdgcn_sched_barrier(0);
                }
            };
            constexpr std::false_type plain{};
            if constexpr (KIND == kBf16 || KIND == kParts) {
                constexpr std::integral_constant<int, AIR_KV_BF16> bf16{};
                if (decltype(exact)::value || fv == 1.0f) rows(bf16, plain);
                else rows(bf16, std::true_type{});
            } else if constexpr (KIND == kFloats) rows(std::integral_constant<int, AIR_KV_F32>{}, plain);
            else if (KIND == kCodes && a.dtype == AIR_KV_INT8) rows(std::integral_constant<int, AIR_KV_INT8>{}, plain);
            else rows(std::integral_constant<int, AIR_KV_FP8>{}, plain);
        };
        float mk = 0.0f, mv = 0.0f;
        // Many rows: what comes between two tiles' products, t the one at hand: tile t + 1 into its
        // buffer, t + 2 on its way (kCodes: t + 2 marked, t + 3 on its way).
        auto stage = [&](int t, auto exact) __attribute__((always_inline)) {
            write_tile(t + 1, raw, kBoth, exact);
            if (t + 2 >= tiles) return;
            if constexpr (F16) {
                raw = next;
                if (t + 3 < tiles) {
                    look_up(t + 3);
                    load_tile(t + 3, next, kBoth);
                }
                mark(t + 2, raw, mk, mv);
            } else {
                look_up(t + 2);
                load_tile(t + 2, raw, kBoth);
            }
        };

        int again = 0;                                 // CONVERT: values as they are
        auto begin = [&](auto exact) __attribute__((always_inline)) {
            fetch(0);
            __syncthreads();                               // the buffers of the block before are free
            look_up(0);
            load_tile(0, raw, kBoth);
            if constexpr (!decltype(exact)::value) sample();
            if constexpr (!PRIVATE) {
                if (F16 && tid < 6) s_top[tid / 2][tid % 2] = 0;
                if (F16 && 1 < tiles) {
                    look_up(1);
                    load_tile(1, next, kBoth);
                }
                if constexpr (F16) {
                    __syncthreads();
                    mark(0, raw, mk, mv);
                    __syncthreads();
                }
                write_tile(0, raw, kBoth, exact);
                if (1 < tiles) {
                    if constexpr (F16) {
                        raw = next;
                        if (2 < tiles) {
                            look_up(2);
                            load_tile(2, next, kBoth);
                        }
                        mark(1, raw, mk, mv);
                    } else {
                        look_up(1);
                        load_tile(1, raw, kBoth);
                    }
                }
                // (a vote: whatever waves have read, all take the same way)
                if constexpr (!decltype(exact)::value) again = __syncthreads_or(fv == 0.0f);
                else __syncthreads();
            }
        };
        begin(kFast);
        // ---- a step's parts: 32 keys, those of a buffer `mem` from row k0 on

        auto scores = [&](const uint8_t *mem, int k0, cross_f32x16 &sc) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < 16; ++i) sc[i] = 0.0f;
            int ln = lane;
            asm volatile("" : "+v"(ln));
            const uint8_t *k = mem + (k0 + (ln & 31)) * KST + 16 * (ln >> 5);
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                cross_u32x4 kf[KP];
#pragma unroll
                for (int p = 0; p < KP; ++p) kf[p] = *reinterpret_cast<const cross_u32x4 *>(k + p * KPLANE + 32 * s);
#pragma unroll
                for (int i = 0; i < KP; ++i)
#pragma unroll
                    for (int j = 0; j < QP; ++j)
                        if (i + j < 3) sc = cross_mfma<F16>(kf[i], qf[j][s], sc);
            }
        };
        auto tops = [&](const cross_f32x16 &sc, float &top) __attribute__((always_inline)) {
            float x = sc[0];
#pragma unroll
            for (int i = 1; i < 16; ++i) x = fmaxf(x, sc[i]);
            top = max_x32(x);
        };
        // keys past the end (rest are left) and of blocks outside the pool (ok: a bit for each half)
        auto hide = [&](int64_t rest, int ok, cross_f32x16 &sc, float &top) __attribute__((always_inline)) {
            uint32_t mask = rest >= 32 ? ~0u : rest <= 0 ? 0u : (1u << (int)rest) - 1;
            mask &= (ok & 1 ? 0x0000FFFFu : 0u) | (ok & 2 ? 0xFFFF0000u : 0u);
            if (__builtin_expect(mask != ~0u, 0)) {
                asm volatile("");                      // (a branch: selects would cost every tile 60 instructions)
                const uint32_t m = mask >> (4 * hf);
#pragma unroll
                for (int i = 0; i < 16; ++i) sc[i] = (m >> (8 * (i / 4) + i % 4)) & 1 ? sc[i] : -INFINITY;
                tops(sc, top);
            }
        };
        // Another base for rows whose largest score passes lim; what is behind has to be multiplied by
        // alpha then (the return value: for some row).
        auto rebase = [&](cross_f32x16 &sc, float top, float &ft, float &alpha) __attribute__((always_inline)) -> bool {
            const bool past = top * ft > lim;
            if (__builtin_expect(__ballot(past) == 0ull, 1)) return false;
            asm volatile("");
            const float x = top * ft;
            const float cap = __builtin_fabsf(base) < kFar ? base - kDown : base;
            const float now = x > cap ? x + (__builtin_fabsf(x) < kFar ? kDown + kSlack : 0.0f) : base;
            alpha = base == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(base - now);
            l_run *= alpha;
            base = now;
            const bool far = !(__builtin_fabsf(now) < kFar) && now != -INFINITY;
            lim = far ? -INFINITY : now - kDown;
            // (scores past 2^20, which f32 holds in steps of an eighth and more, are each rounded as
            // the largest was, so that their distances from the base are exact)
            if (__ballot(far) != 0ull) {
                sc *= ft;
                ft = 1.0f;
            }
            return true;
        };
        auto scale_sums = [&](float by) __attribute__((always_inline)) {
#pragma unroll
            for (int c = 0; c < CT; ++c) acc[c] *= by;
        };
        // what products are multiplied by.  (Neither 0 nor infinite: a masked score, -inf, times 0 would be NaN,
        // and so would 0 times infinity.)
        auto factors = [&](float fk, float &ft) __attribute__((always_inline)) {
            ft = a.scale_log2;
            if constexpr (F16) ft = fminf(fmaxf(__builtin_amdgcn_ldexpf(ft, -(qe + cross_exponent(fk))), 0x1p-126f), 0x1.fffffep127f);
        };
        auto probabilities = [&](cross_f32x16 &sc, float ft, auto &p) __attribute__((always_inline)) {
            constexpr int P = std::extent_v<std::remove_reference_t<decltype(p)>>;
            const float from = base == -INFINITY ? 0.0f : base;
#pragma unroll
            for (int i = 0; i < 16; ++i) sc[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[i], ft, -from));
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    uint32_t x[P];
                    cross_parts<P>(sc[8 * s + 2 * j], sc[8 * s + 2 * j + 1], x);
#pragma unroll
                    for (int k = 0; k < P; ++k) p[k][s][j] = x[k];
                    // (f16 ones are summed as they were rounded)
                    if constexpr (P == 1) l_run = cross_add_pair(x[0], ones, l_run);
                    else l_run += sc[8 * s + 2 * j] + sc[8 * s + 2 * j + 1];
                }
        };
        // V^T as the A operand: lane (m, h) takes keys 16 s + 8 b + 4 h .. +4 of column m, b = 0, 1.
        // Within each 16-lane group, lane j of a transposing read receives element j % 4 of the 8
        // bytes that lanes 4 k + j / 4 address, k = 0 .. 3: lane i points at key i / 4 of the four
        // and columns 4 (i % 4) of the group's sixteen.
        auto values = [&](const uint8_t *mem, int k0, const auto &p) __attribute__((always_inline)) {
            constexpr int P = std::extent_v<std::remove_reference_t<decltype(p)>>;
            int ln = lane;                             // (its addresses are not kept in registers from step to step)
            asm volatile("" : "+v"(ln));
            const int vr = 4 * (ln >> 5) + ((ln & 15) >> 2);
            const uint8_t *v0 = mem + VAT + (k0 + vr) * VST + 32 * ((ln >> 4) & 1) + 8 * (ln & 3);
#pragma unroll
            for (int c = 0; c < CT; ++c)
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                    for (int i = 0; i < KP; ++i) {
                        typedef short s16x4 __attribute__((ext_vector_type(4)));
                        const int cc = cross_v_xor(D) ? 64 * (c ^ (vr & 3)) : 64 * c;
                        const uint8_t *v = v0 + i * VPLANE + cc + 16 * s * VST;
                        const cross_u32x2 x = __builtin_bit_cast(cross_u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                  (__attribute__((address_space(3))) s16x4 *)v));
                        const cross_u32x2 y = __builtin_bit_cast(cross_u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                  (__attribute__((address_space(3))) s16x4 *)(v + 8 * VST)));
                        const cross_u32x4 vf = {x[0], x[1], y[0], y[1]};
#pragma unroll
                        for (int j = 0; j < P; ++j)
                            if (i + j < 3) acc[c] = cross_mfma<P == 1>(vf, p[j][s], acc[c]);
                    }
        };

        // Many rows, a step after the other.
        auto walk = [&](auto exact) __attribute__((always_inline)) {
            for (int t = 0; t < tiles; ++t) {
                if constexpr (F16) {
                    fk = fk_next;
                    if (fv != fv_next) {
                        scale_sums(fv == 0.0f ? 1.0f : fv_next / fv);
                        fv = fv_next;
                    }
                    if (tid < 2) s_top[t % 3][tid] = 0;
                }
                if (NB >= 2 && t + 1 < tiles) stage(t, exact);
                if (any) {
                    const uint8_t *mem = s_mem + t % NB * S::TILE;
#pragma unroll
                    for (int sub = 0; sub < SUB; ++sub) {
                        const int64_t rest = sq.len - (key0 + (int64_t)t * TK + 32 * sub);
                        if (rest <= 0) continue;
                        cross_f32x16 sc;
                        cross_u32x4 p[CONVERT && decltype(exact)::value ? 2 : PP][2];
                        float top, ft, alpha;
                        scores(mem, 32 * sub, sc);
                        tops(sc, top);
                        hide(rest, __builtin_amdgcn_readfirstlane(s_ok[t % 8][2 * sub] + 2 * s_ok[t % 8][2 * sub + 1]), sc, top);
                        factors(fk, ft);
                        if (rebase(sc, top, ft, alpha)) scale_sums(alpha);
                        probabilities(sc, ft, p);
                        values(mem, 32 * sub, p);
                    }
                }
                __syncthreads();
                if (NB == 1 && t + 1 < tiles) {
                    stage(t, exact);
                    __syncthreads();
                }
            }
        };
        if constexpr (PIPE) {
            // A step's probabilities are computed beside the next step's scores and the one before's
            // values, so that products and arithmetic, about as much of either, run at once.  A tile is
            // two steps; the next tile is staged beside the first and there at a barrier before the second.
            static_assert(PP == 1 && KP == 1 && KS == 2 * CT && NB == 3, "16-bit parts");
            if (!again) {
                cross_f32x16 sa, sb;
                cross_u32x4 pa[2], pb[2];
                float top;
                float fv_t = fv_next;                      // kCodes: of the tile whose values come next
                // (this lane's places in a buffer: keys, values of four column tiles)
                const int k_at = r32 * KST + 16 * hf, vr = 4 * hf + ((lane & 15) >> 2);
                int v_at[4];
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    v_at[c] = VAT + vr * VST + 32 * ((lane >> 4) & 1) + 8 * (lane & 3) + 64 * (cross_v_xor(D) ? c ^ (vr & 3) : c);
                // A step from its scores in sc: p; the next step's scores, of the keys from row k0 of buffer kb, in
                // sn; the sums of the step before, its probabilities q and the values from row v0 of buffer vb.
                auto step = [&](cross_f32x16 &sc, cross_f32x16 &sn, cross_u32x4 (&p)[2], const cross_u32x4 (&q)[2], int kb, int k0, int vb,
                                int v0, int64_t rest, int ok, float fk) __attribute__((always_inline)) {
                    hide(rest, ok, sc, top);
                    float ft, alpha;
                    factors(fk, ft);
                    const bool changed = rebase(sc, top, ft, alpha);
                    // what follows is in the order in which it shall run: a product, then arithmetic that is done
                    // while it runs, fragments read three products ahead
                    constexpr int AHEAD = 3, N = KS + 2 * CT;
                    typedef const __attribute__((address_space(3))) uint8_t *lds_t;
                    const lds_t k = (lds_t)s_mem + kb * S::TILE + k0 * KST + k_at;
                    lds_t v[CT < 4 ? CT : 4];
#pragma unroll
                    for (int c = 0; c < CT && c < 4; ++c) v[c] = (lds_t)s_mem + vb * S::TILE + v0 * VST + v_at[c];
                    cross_u32x4 f[N];
                    auto read = [&](int i) __attribute__((always_inline)) {
                        typedef short s16x4 __attribute__((ext_vector_type(4)));
                        if (i < KS) {
                            f[i] = *reinterpret_cast<const __attribute__((address_space(3))) cross_u32x4 *>(k + 32 * i);
                        } else if (i < N) {
                            const int c = (i - KS) / 2, at = 256 * (c / 4) + 16 * ((i - KS) % 2) * VST;
                            const cross_u32x2 x = __builtin_bit_cast(cross_u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                      (__attribute__((address_space(3))) s16x4 *)(v[c % 4] + at)));
                            const cross_u32x2 y = __builtin_bit_cast(cross_u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                      (__attribute__((address_space(3))) s16x4 *)(v[c % 4] + at + 8 * VST)));
                            f[i] = cross_u32x4{x[0], x[1], y[0], y[1]};
                        }
                    };
                    const float from = base == -INFINITY ? 0.0f : base;
                    auto pair = [&](int i) __attribute__((always_inline)) {
                        const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[2 * i], ft, -from));
                        const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[2 * i + 1], ft, -from));
                        p[i / 4][i % 4] = cross_f16_pair(x, y);
                        l_run = cross_add_pair(p[i / 4][i % 4], ones, l_run);
                    };
#pragma unroll
                    for (int i = 0; i < 16; ++i) sn[i] = 0.0f;
#pragma unroll
                    for (int i = 0; i < AHEAD; ++i) read(i);
                    __builtin_amdgcn_sched_barrier(0);
                    int done = 0;
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        read(i + AHEAD);
                        if (i < KS) sn = cross_mfma<F16>(f[i], qf[0][i], sn);
                        else acc[(i - KS) / 2] = cross_mfma<true>(f[i], q[(i - KS) % 2], acc[(i - KS) / 2]);
#pragma unroll
                        for (; done < 8 * (i + 1) / N; ++done) pair(done);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                    tops(sn, top);
                    // (here, and not where they are used: behind a branch)
                    asm volatile("" : "+v"(p[0]), "+v"(p[1]), "+v"(l_run));
                    if (__builtin_expect(changed, 0)) {
                        asm volatile("");                  // (a branch: no products by 1)
                        scale_sums(alpha);
                    }
                };
                auto in_pool = [&](int t, int half) __attribute__((always_inline)) {
                    return __builtin_amdgcn_readfirstlane(s_ok[t % 8][half] + 2 * s_ok[t % 8][half + 1]);
                };
                // (the step before the first: probabilities of 0, of values that are there)
                pb[0] = pb[1] = cross_u32x4{0, 0, 0, 0};
                scores(s_mem, 0, sa);
                tops(sa, top);
                int before = 0, at = 0;                    // buffers of tiles t - 1 and t
                for (int t = 0; t < tiles; ++t) {
                    const int next = at == 2 ? 0 : at + 1;
                    const int64_t rest = sq.len - (key0 + (int64_t)t * TK);
                    step(sa, sb, pa, pb, at, 32, before, 32, rest, in_pool(t, 0), fk_next);
                    if constexpr (F16) {
                        fk = fk_next;
                        fv_t = fv_next;
                        if (tid < 2) s_top[t % 3][tid] = 0;
                    }
                    if (t + 1 < tiles) stage(t, kFast);
                    __syncthreads();
                    if constexpr (F16) {
                        // (a power of two that changes: the sums so far are brought under it)
                        if (__builtin_expect(fv != fv_t, 0)) {
                            scale_sums(fv == 0.0f ? 1.0f : fv_t / fv);
                            fv = fv_t;
                        }
                    }
                    step(sb, sa, pb, pa, next, 0, at, 0, rest - 32, in_pool(t, 2), fk);
                    before = at;
                    at = next;
                }
                // (the last tile's second half)
                cross_u32x4 p[PP][2] = {{pb[0], pb[1]}};
                values(s_mem + before * S::TILE, 32, p);
                __syncthreads();
            }
        } else if constexpr (PRIVATE) {
            uint8_t *mem = s_mem + wave * S::REGION;
            // (a wave's LDS accesses are in order: what was there has been read)
            auto ordered = [&]() __attribute__((always_inline)) {
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
            };
            for (int t = 0; t < tiles; ++t) {
                // whether this wave's halves are in the pool
                const int ok = (__builtin_amdgcn_readlane(window, 2 * wave) >= 0 ? 1 : 0) | (__builtin_amdgcn_readlane(window, 2 * wave + 1) >= 0 ? 2 : 0);
                const int64_t rest = sq.len - (key0 + (int64_t)t * TK + 32 * wave);
                cross_u32x4 p[PP][2];
                if constexpr (F16) {
                    mark(t, raw, mk, mv);
                    keys_power(mk);
                    values_power(mv);
                    // (a power of two that changes: the sums so far are brought under it)
                    if (fv != fv_next) {
                        scale_sums(fv == 0.0f ? 1.0f : fv_next / fv);
                        fv = fv_next;
                    }
                }
                constexpr auto kFirst = std::conditional_t<SPLIT, decltype(kKeys), decltype(kBoth)>{};
                ordered();
                write_tile(t, raw, kFirst, kFast);
                ordered();
                if (t + 1 < tiles) {
                    look_up(t + 1);
                    load_tile(t + 1, raw, kFirst);
                }
                if (rest > 0) {
                    cross_f32x16 sc;
                    float top, ft, alpha;
                    scores(mem, 0, sc);
                    tops(sc, top);
                    hide(rest, ok, sc, top);
                    factors(fk_next, ft);
                    if (rebase(sc, top, ft, alpha)) scale_sums(alpha);
                    probabilities(sc, ft, p);
                }
                if constexpr (SPLIT) {
                    ordered();
                    write_tile(t, raw, kValues, kFast);
                    ordered();
                    if (t + 1 < tiles) load_tile(t + 1, raw, kValues);
                }
                if (rest > 0) values(mem, 0, p);
            }
            __syncthreads();
        } else if (!again) {
            walk(kFast);
        }
        if constexpr (CONVERT) {
            // A row whose probabilities are finite and whose sums are not: a value was not, or beyond f16 (an
            // infinity there).
            float x = 0.0f;
#pragma unroll
            for (int c = 0; c < CT; ++c)
#pragma unroll
                for (int i = 0; i < 16; ++i) x = __builtin_fmaf(acc[c][i], 0.0f, x);
            if (!again) again = __syncthreads_or(x != 0.0f && l_run < INFINITY);
            if (__builtin_expect(again, 0)) {
                fv = 0.0f;
                clear(24.0f);
                begin(kExact);
                walk(kExact);
            }
        }

        // lane (n, h): columns 32 c + 8 (i / 4) + 4 h + i % 4 of row n in acc[c][i]
        float unit = V16 && fv != 0.0f ? 1.0f / fv : 1.0f;     // of the sums (pieces' stay under it)
        const int64_t slot = 2 * cell + (t0 == 0 ? 1 : 0);
        if constexpr (WK == 1) {
            const float l = sum_x32(l_run);
            const int64_t prow = slot * ROWS + 32 * rg + r32;
            // no key at all (every block outside the pool): zeros
            const float k = whole ? (l == 0.0f ? 0.0f : 1.0f / l) : 1.0f;
            if (whole ? live : any) {
#pragma unroll
                for (int c = 0; c < CT; ++c)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        cross_f32x4 x = cross_f32x4{acc[c][4 * i], acc[c][4 * i + 1], acc[c][4 * i + 2], acc[c][4 * i + 3]} * k;
                        if (V16 && whole) x *= unit;
                        const int col = 32 * c + 8 * i + 4 * hf;
                        if (whole) cross_store4(a, io + col, x);
                        else *reinterpret_cast<cross_f32x4 *>(a.part_o + prow * D + col) = x;
                    }
                if (!whole && hf == 0) a.part_ml[prow] = make_float4(base, l, unit, 0.0f);
            }
        } else {
            // the waves of one row group: their bases' largest, then their sums, CR column tiles at a
            // time, four columns (c, i) of all of them to one wave
            float l = sum_x32(l_run);
            const int64_t prow = slot * ROWS + 32 * rg + r32;
            if (hf == 0) s_ml[wave][r32] = make_float4(base, l, fv, 0.0f);
            __syncthreads();
            float top = -INFINITY, least = 0.0f;       // (the smallest power of two of the values': the largest unit)
#pragma unroll
            for (int i = 0; i < WK; ++i) {
                const float4 ml = s_ml[rg * WK + i][r32];
                top = fmaxf(top, ml.x);
                least = ml.z != 0.0f && (least == 0.0f || ml.z < least) ? ml.z : least;
            }
            l = 0.0f;
#pragma unroll
            for (int i = 0; i < WK; ++i) {
                const float4 ml = s_ml[rg * WK + i][r32];
                l += ml.x == -INFINITY ? ml.y : ml.y * __builtin_amdgcn_exp2f(ml.x - top);
            }
            float alpha = base == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(base - top);
            if (F16 && fv != 0.0f) alpha *= least / fv;
            if (F16) unit = least != 0.0f ? 1.0f / least : 1.0f;
            const float k = whole ? (l == 0.0f ? 0.0f : 1.0f / l) : 1.0f;
            cross_f32x4 *x = reinterpret_cast<cross_f32x4 *>(s_mem) + lane;
#pragma unroll
            for (int c0 = 0; c0 < CT; c0 += CR) {
                if (c0) __syncthreads();
#pragma unroll
                for (int c = c0; c < c0 + CR && c < CT; ++c)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        x[((wave * CR + c - c0) * 4 + i) * 64] = cross_f32x4{acc[c][4 * i], acc[c][4 * i + 1], acc[c][4 * i + 2], acc[c][4 * i + 3]} * alpha;
                __syncthreads();
                const int quads = 4 * (CT - c0 < CR ? CT - c0 : CR);
                for (int g = wk; g < quads; g += WK) {
                    cross_f32x4 y = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int i = 0; i < WK; ++i) y += x[((rg * WK + i) * CR * 4 + g) * 64];
                    y *= k;
                    if (F16 && whole) y *= unit;
                    const int col = 32 * (c0 + g / 4) + 8 * (g % 4) + 4 * hf;
                    if (whole) {
                        if (live) cross_store4(a, io + col, y);
                    } else if (any) {
                        *reinterpret_cast<cross_f32x4 *>(a.part_o + prow * D + col) = y;
                    }
                }
            }
            if (!whole && any && hf == 0 && wk == 0) a.part_ml[prow] = make_float4(top, l, unit, 0.0f);
        }
        if (!whole && t0 == 0) {                       // begun here: its last unit's slice ends it
            const int64_t last = u - mine - at + nt + EXTRA - 1;
            begun = int4{b, blk, (int)(last / chunk - w + 1), 0};
        }
    }
    if (tid == 0) a.desc[cell] = begun;
}

template <CrossKind KIND, bool FEW> hipError_t launch_cross_shape(const CrossArgs &a, int d, hipStream_t s) {
    const dim3 grid((unsigned)(a.slices * a.heads));
    switch (d) {
#define AIRKV_CROSS(D) \
    case D: { \
        constexpr bool F = FEW && CrossShape<D, KIND, true>::PRIVATE; \
        hipLaunchKernelGGL((paged_cross_kernel<D, KIND, F>), grid, dim3(CrossShape<D, KIND, F>::WAVES * 64), 0, s, a); \
        break; \
    }
        AIRKV_CROSS(32) AIRKV_CROSS(64) AIRKV_CROSS(96) AIRKV_CROSS(128)
        AIRKV_CROSS(160) AIRKV_CROSS(192) AIRKV_CROSS(224) AIRKV_CROSS(256)
#undef AIRKV_CROSS
    }
    return hipGetLastError();
}

template <CrossKind KIND, bool FEW> CrossBlocks cross_blocks_shape(int d) {
    switch (d) {
#define AIRKV_CROSS(D) \
    case D: { \
        constexpr bool F = FEW && CrossShape<D, KIND, true>::PRIVATE; \
        return {CrossShape<D, KIND, F>::ROWS, CrossShape<D, KIND, F>::GROUPS, F}; \
    }
        AIRKV_CROSS(32) AIRKV_CROSS(64) AIRKV_CROSS(96) AIRKV_CROSS(128)
        AIRKV_CROSS(160) AIRKV_CROSS(192) AIRKV_CROSS(224) AIRKV_CROSS(256)
#undef AIRKV_CROSS
    }
    return {0, 0, false};
}

}  // namespace airkv
