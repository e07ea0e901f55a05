// Differential prefill with 16-bit products (formulas: diff_common.hpp; work
// division: diff_prefill_plan.hpp): bf16 queries and outputs over bf16 or 1-byte pages.
//
// A workgroup's block is 128 rows; eight waves take 32 rows and one of the two maps
// each (a wave with both maps' sums over the 2 * head_dim value columns would need 512
// registers).  A wave walks its keys once, 32 at a time, with a running maximum and sum:
//   S   = K . Q^T      v_mfma_f32_32x32x16, lane (n, h) holds 16 of the 32 keys of row n
//   O^T += V^T . P^T   the same instruction; its contraction takes the keys in the order
//                      in which the lanes hold P, so P never moves
// and the two maps of a row meet when the block ends.  Keys and values are staged in LDS
// as rows, in three buffers (two tiles ahead, loaded three ahead, one barrier a tile), with
// 16-byte chunks placed so that neither the rows' reads nor the values' transposing reads
// meet in a bank.
//
// The second product takes f16 operands: values (exact when they come from bf16 pages
// and lie in f16's normal range, else rounded to 11 bits) and probabilities rounded to 11
// bits, an error below the bf16 output's own rounding, where bf16 probabilities would add as
// much again (measured against 64 bits: 1.7e-3 and 2.6e-3 of the result's norm).  The
// first product takes bf16 operands as they are from bf16 pages, f16 ones (dequantized,
// 11 bits) from 1-byte pages.  Powers of two bring f16's operands into its range: a running
// one for keys and one for values, by the largest so far, one per row for queries, a constant
// for probabilities.  What lies far below the largest keeps f16's absolute step, 2^-21 of it
// (kLeast) at the coarsest.
//
// Bound by vector issue and the tile's chain: per tile and SIMD 1540 of 4300 clocks are
// products, 2000 arithmetic (exponentials, the values' rounding, staging), which overlap
// in part.  8192 tokens of 16 query pairs of 128 in 1.08 ms: 510 TFLOP/s of 8 d a (query
// pair, key), 765 of the 12 d that two running maps take; eight chunks of 200 to 512
// behind up to 6000 tokens 361 us, 437 TFLOP/s; int8 pages, 32 query pairs, 621 us, 438
// (2 to 3% less or more from card to card).
#include <hip/hip_runtime.h>

#include "../pool.hpp"
#include "diff_prefill.hpp"

namespace airkv {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef diff_u32x4 u32x4;
typedef diff_u32x2 u32x2;
typedef diff_f32x4 f32x4;

template <bool F16> __device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
    if constexpr (F16)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

__device__ __forceinline__ uint32_t bf16_pair(float x, float y) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{x, y}), bf16x2));
}

// Two values rounded to f16, x in the low half.
__device__ __forceinline__ uint32_t f16_pair(float x, float y) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{x, y}), f16x2));
}

// Lanes (n, 0) and (n, 1) hold columns 0 .. 3 and 4 .. 7 of a row's eight in x, and of the
// next eight in y: the eight of x to lane (n, 0), those of y to (n, 1).
__device__ __forceinline__ u32x4 eight(u32x2 x, u32x2 y) {
    const auto a = __builtin_amdgcn_permlane32_swap(x[0], y[0], false, false), b = __builtin_amdgcn_permlane32_swap(x[1], y[1], false, false);
    return u32x4{a[0], b[0], a[1], b[1]};
}

// 2^(e - exponent of x) for a finite x >= 0, from 2^-126 to 2^112 (subnormal x, and normal
// ones below 2^(e - 112), get the largest), else 1.
__device__ __forceinline__ float pow2_to(float x, int e) {
    const int f = (int)((__float_as_uint(x) >> 23) & 0xFF), k = 127 + e - (f - 127);
    return f == 255 ? 1.0f : __uint_as_float((uint32_t)(k < 1 ? 1 : k > 239 ? 239 : k) << 23);
}

// The exponent of a power of two (a normal number).
__device__ __forceinline__ int exponent(float x) { return (int)(__float_as_uint(x) >> 23) - 127; }

// The schedule of N matrix products that take READS LDS reads each: the reads of the
// first AHEAD, then a product and the reads of the next in turn.
template <int N, int AHEAD, int READS> __device__ __forceinline__ void read_ahead() {
    constexpr int kMfma = 0x008, kLdsRead = 0x100;
    __builtin_amdgcn_sched_group_barrier(kLdsRead, READS * AHEAD, 0);
#pragma unroll
    for (int i = 0; i < N - AHEAD; ++i) {
        __builtin_amdgcn_sched_group_barrier(kMfma, 1, 0);
        __builtin_amdgcn_sched_group_barrier(kLdsRead, READS, 0);
    }
    __builtin_amdgcn_sched_group_barrier(kMfma, AHEAD, 0);
}

// Probabilities are held 2^kUp times their size, so that f16 has 11 bits of those down to
// 2^-25 of the running maximum's, and an absolute step of 2^-35 of it below: of a key among a
// million that none of them stands out from, too.  kSlack: how far the running maximum may lag
// (f16 ends at 2^16; a score's rounding is a factor of at most 2^(1/2) where it is below 2^22).
constexpr float kUp = 11.0f, kSlack = 4.0f;

constexpr int kRows = 128;
constexpr int kThreads16 = 512;

// Where the 16-byte chunk c of row r of a staged head of values lies, in chunks: they
// are read eight rows at a time, 64 bytes each: four rows in a row, in different quarters.
template <int D> __device__ __forceinline__ int value_chunk(int r, int c) {
    if constexpr (D == 128) return c ^ ((r & 3) << 2);
    else if constexpr (D == 64) return c ^ (((r >> 1) & 1) << 2);
    else return c;
}

template <int D, int DT>
__global__ __launch_bounds__(kThreads16) __attribute__((amdgpu_waves_per_eu(2, 2)))
void diff_prefill_16_kernel(DiffPrefillArgs a) {
    constexpr bool QUANT = DT != AIR_KV_BF16;
    constexpr int EB = QUANT ? 1 : 2;
    constexpr int RB = 2 * D;                          // bytes of a staged row
    constexpr int HB = kDiffKeys * RB;                 // of a staged head; keys of both heads, then values
    constexpr int KS = D / 16, CT = D / 16;            // steps of the first product, 32-column tiles of the second
    // Staging: a wave's pass covers WR rows of one 16-key half of one head of keys or
    // values, CP 8-element pieces a row (head_dim 96: 12 of 16 lanes), so its addresses
    // differ between lanes by a constant only and its bounds are a buffer's.
    constexpr int CP = D == 96 ? 16 : D / 8, WR = 64 / CP, NP = 4 * kDiffKeys / (8 * WR);
    __shared__ int64_t s_pre[kDiffPrefillBatch + 1];
    __shared__ int64_t s_sum[kThreads16 / 64];
    // the three buffers; in them, at a block's end, CR column tiles of every wave's half
    constexpr int CH = CT / 2, CR = D == 128 ? 2 : 1, XB = 8 * CR * 4 * 64 * 16;
    __shared__ __align__(16) uint8_t s_mem[12 * HB > XB ? 12 * HB : XB];
    auto s_t = [&](int t) __attribute__((always_inline)) { return s_mem + t % 3 * (4 * HB); };
    // Per tile (mod 3), keys' scale and values' (scale): the bits of the largest of those that
    // leave f16's range under the present power of two (of all, as long as a block had zeros only)
    __shared__ uint32_t s_top[3][2];
    __shared__ __align__(16) float s_w[2 * D];         // the norm's weights
    __shared__ float s_ss[2][4][32];                   // the halves' sums of squares
    // Values that are not finite, in tiles that not every row sees (a hidden key's
    // probability of 0 times such a value would be NaN): staged as 0, and each column's
    // first such key is kept here, from which on a row's column is NaN.
    __shared__ int s_bad[2 * D];
    __shared__ int s_any;
    if (threadIdx.x < 2 * D) s_w[threadIdx.x] = a.e.norm && a.e.norm_w ? a.e.norm_w[threadIdx.x] : 1.0f;
    diff_refused(a, 2 * D);
    diff_units<kThreads16>(a, s_pre, s_sum);
    const int tid = threadIdx.x, lane = tid & 63, hf = lane >> 5, r32 = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int rg = wave & 3, mp = wave >> 2;           // 32 rows, one map
    const int w = blockIdx.x, kp = blockIdx.y, g = a.group;
    const int64_t units = diff_uniform(s_pre[a.batch]);
    const int64_t chunk = diff_prefill_chunk(units, a.slices, a.least);
    const int64_t cell = (int64_t)kp * a.slices + w;
    int4 begun = {0, 0, 0, 0};
    // A SIMD has one wave of either map: map 1's goes first, so that the two stay out of phase
    // and one's products run beside the other's arithmetic (8192 tokens 1.08 -> 1.04 ms).
    if (mp) __builtin_amdgcn_s_setprio(1);

    // This lane's piece of every pass: row (of its 16-key half) and 16-byte chunk
    const int nsc = QUANT ? D / a.scale_group : 0;
    const int p_c = lane % CP, p_row0 = wave * WR;     // the wave's first row of pass 0, of the 128 staged
    const int p_key = (p_row0 + lane / CP) % kDiffKeys;
    const bool p_in = D != 96 || p_c < D / 8;
    const int p_off = p_in ? ((p_key % 16) * D + 8 * p_c) * EB : 0x40000000;
    const int p_sc = p_in && QUANT ? ((p_key % 16) * nsc + 8 * p_c / a.scale_group) * 4 : 0x40000000;
    const int p_klds = p_key * RB + 16 * key_chunk<D>(p_key, p_c), p_vlds = p_key * RB + 16 * value_chunk<D>(p_key, p_c);
    const int p_half = p_row0 % kDiffKeys / 16;        // of every pass: 8 WR rows are a multiple of 32

    // The powers of two under which keys and values are staged, kept from block to block.
    // The largest scale (a 2^9th of a value), or value, under it: below f16's largest; at
    // least where values 2^-11 of it keep their bits; and where a new one puts it.
    constexpr float kMost = QUANT ? 64.0f : 32768.0f, kLeast = QUANT ? 0.5f : 0.125f;
    constexpr int kAim = QUANT ? 3 : 8;
    float fk = 1.0f, fv = 1.0f;
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
        const int64_t rows = sq.q * g;
        // this lane's row: token and query pair (of the last token, if there is none)
        auto my_row = [&](int r, bool &live, int &tok, int &h) __attribute__((always_inline)) {
            const int64_t f = it.k * kRows + 32 * rg + r;
            live = f < rows;
            tok = (int)(live ? f / g : sq.q - 1);
            h = kp * g + (live ? (int)(f % g) : 0);
        };
        const int64_t f0 = it.k * kRows + 32 * rg, f1 = f0 + 31;
        // the newest key, counted from the item's first tile: of this row, of the wave's first
        // and last row, of the block's first, and the sequence's end (32-bit: at most 2^31 keys)
        const int64_t key0 = t0 * kDiffKeys;
        const int sees0 = (int)(sq.prefix + (f0 < rows ? f0 / g : sq.q - 1) - key0);
        const int sees1 = (int)(sq.prefix + (f1 < rows ? f1 / g : sq.q - 1) - key0);
        const int seesb = (int)(sq.prefix + it.k * kRows / g - key0);
        const int rest = (int)(len - key0), tiles = (int)(t1 - t0);

        // Q^T as the B operand: lane (n, h) holds elements 16 s + 8 h .. +8 of row n
        u32x4 qf[KS];
        int qe = 0;                                    // (the power of two they are under)
        int sees;
        {
            bool live;
            int tok, h;
            my_row(r32, live, tok, h);
            sees = (int)(sq.prefix + tok - key0);
            const uint16_t *q = (const uint16_t *)a.q + ((row0 + tok) * 2 * a.pairs + 2 * h + mp) * D + 8 * hf;
#pragma unroll
            for (int s = 0; s < KS; ++s) qf[s] = *reinterpret_cast<const u32x4 *>(q + 16 * s);
        }
        if constexpr (QUANT) {
            float top = 0.0f;
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    top = fmaxf(top, fmaxf(__builtin_fabsf(__uint_as_float(qf[s][j] << 16)),
                                           __builtin_fabsf(__uint_as_float(qf[s][j] & 0xFFFF0000u))));
            const float fq = pow2_to(max_x32(top), 4);          // the row's largest element in [2^4, 2^5)
            qe = exponent(fq);
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    qf[s][j] = f16_pair(__uint_as_float(qf[s][j] << 16) * fq, __uint_as_float(qf[s][j] & 0xFFFF0000u) * fq);
        }
        f32x16 acc[CT];
        // probabilities are 2^(score - base); a row's scores past `lim` ask for another base
        float base = -INFINITY, lim = -INFINITY, l_run = 0.0f;
        // what the sums have to be multiplied by to be under the present tile's power of two,
        // and for the next tile's
        float owed = 1.0f, owed_next = 1.0f;
#pragma unroll
        for (int c = 0; c < CT; ++c)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[c][i] = 0.0f;

        const int32_t *table = a.tables + (int64_t)it.b * a.max_blocks + key0 / a.bs;
        struct Raw {                                   // a tile on its way
            uint32_t w[NP][2 * EB];
            float s[NP];
        };
        // Lane k: the entry of the half that this wave stages of tile t + k, for a window of
        // 64 tiles (an entry a tile would be waited for behind that tile's loads); entries
        // outside the pool are counted once per block of tokens, and read nothing.
        const int shift = a.bs == 32 ? 5 : 4;
        int32_t window = 0;
        auto look_up = [&](int t) __attribute__((always_inline)) {
            const int key = (t + lane < tiles ? t + lane : tiles - 1) * kDiffKeys + 16 * p_half;
            window = key < rest ? table[key >> shift] : 0;
            const bool out = t + lane < tiles && (window < 0 || window >= a.num_blocks);
            window = out || key >= rest ? -1 : window;
            if (kp == 0 && p_row0 % 16 == 0 && p_row0 < kDiffKeys && (p_half == 0 || a.bs == 16)) {
                const int n = __popcll(__ballot(out));
                if (n && lane == 0) atomicAdd(a.errors, (unsigned long long)n);
            }
        };
        // A head's rows of a block lie bs rows behind the head's before: one buffer holds both
        // heads', and a lane whose key is not there reads outside of it: zeros.
        const int head_step = a.bs * D * EB, head_sc = a.bs * nsc * 4;
        auto load_rows = [&](int t, int32_t blk, Raw &r) __attribute__((always_inline)) {
            const int left = blk < 0 ? 0 : rest - t * kDiffKeys - 16 * p_half;
            const int off = (p_key & 15) < left ? p_off : 0x40000000;
            const int64_t row = (((int64_t)(blk < 0 ? 0 : blk) * a.heads + 2 * kp) << shift) + (16 * p_half & (a.bs - 1));
            const __amdgpu_buffer_rsrc_t rk = __builtin_amdgcn_make_buffer_rsrc(
                (void *)((const uint8_t *)a.k_pages + row * (D * EB)), (short)0, head_step + 16 * D * EB, kDiffBufferWord3);
            const __amdgpu_buffer_rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc(
                (void *)((const uint8_t *)a.v_pages + row * (D * EB)), (short)0, head_step + 16 * D * EB, kDiffBufferWord3);
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                const int part = (p_row0 + 8 * WR * i) / kDiffKeys;          // keys of head 0, 1, values of head 0, 1
                const int step = (part & 1) * head_step;
                if constexpr (QUANT) {
                    const u32x2 x = part < 2 ? __builtin_amdgcn_raw_buffer_load_b64(rk, off, step, 0)
                                             : __builtin_amdgcn_raw_buffer_load_b64(rv, off, step, 0);
                    r.w[i][0] = x[0]; r.w[i][1] = x[1];
                } else {
                    const u32x4 x = part < 2 ? __builtin_amdgcn_raw_buffer_load_b128(rk, off, step, 0)
                                             : __builtin_amdgcn_raw_buffer_load_b128(rv, off, step, 0);
#pragma unroll
                    for (int j = 0; j < 4; ++j) r.w[i][j] = x[j];
                }
            }
            if constexpr (QUANT) {
                const int osc = (p_key & 15) < left ? p_sc : 0x40000000;
                const __amdgpu_buffer_rsrc_t sk = __builtin_amdgcn_make_buffer_rsrc((void *)(a.k_scales + row * nsc), (short)0,
                                                                                    head_sc + 16 * nsc * 4, kDiffBufferWord3);
                const __amdgpu_buffer_rsrc_t sv = __builtin_amdgcn_make_buffer_rsrc((void *)(a.v_scales + row * nsc), (short)0,
                                                                                    head_sc + 16 * nsc * 4, kDiffBufferWord3);
#pragma unroll
                for (int i = 0; i < NP; ++i) {
                    const int part = (p_row0 + 8 * WR * i) / kDiffKeys, step = (part & 1) * head_sc;
                    r.s[i] = __uint_as_float(part < 2 ? __builtin_amdgcn_raw_buffer_load_b32(sk, osc, step, 0)
                                                      : __builtin_amdgcn_raw_buffer_load_b32(sv, osc, step, 0));
                }
            }
        };
        // The next tile, and the blocks of the last two: a tile that is staged again is loaded
        // from its block here, not from the window, which may have gone on past it.
        int32_t blk_at = -1, blk_before = -1;
        auto load_tile = [&](int t, Raw &r) __attribute__((always_inline)) {
            if (t % 64 == 0) look_up(t);
            blk_before = blk_at;
            blk_at = __builtin_amdgcn_readlane(window, t % 64);
            load_rows(t, blk_at, r);
        };
        // Scales and values of the tile in registers that leave f16's range are marked for all
        // waves; behind the barrier the tile is staged again under another power of two.  Until a
        // tile has something that is not zero the power of two is another block's, and too small
        // ones count too.  (The scale 1 that the append gives a group of zeros does not count.)
        uint32_t lim_k = 1, lim_v = 1;                 // the bits from which on one is marked
        auto mark = [&](int t, const Raw &r) __attribute__((always_inline)) {
            uint32_t k = 0, v = 0;                     // this lane's largest finite ones, as bits
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                const bool val = (p_row0 + 8 * WR * i) / kDiffKeys >= 2;
                if constexpr (QUANT) {
                    const uint32_t y = __float_as_uint(r.s[i]) & 0x7FFFFFFFu;
                    const bool zeros = ((r.w[i][0] | r.w[i][1]) & (DT == AIR_KV_FP8 ? 0x7F7F7F7Fu : ~0u)) == 0 && y <= 0x3F800000u;
                    const uint32_t x = y < 0x7F800000u && !zeros ? y : 0;
                    if (val) v = x > v ? x : v;
                    else k = x > k ? x : k;
                } else if (val) {
                    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
                    u16x2 top = {0, 0};
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, r.w[i][j] & 0x7FFF7FFFu));
                    uint32_t b = top[0] > top[1] ? top[0] : top[1];
                    if (b >= 0x7F80u) {
                        b = 0;
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const uint32_t x = r.w[i][j / 2] >> (16 * (j & 1)) & 0x7FFFu;
                            b = x < 0x7F80u && x > b ? x : b;
                        }
                    }
                    v = b << 16 > v ? b << 16 : v;
                }
            }
            if (t == 0) {                              // of all lanes: one atomic a wave
                auto most = [](int x, int y) { return x > y ? x : y; };
                if (QUANT) k = __builtin_amdgcn_readlane(wave_scan((int)k, most), 63);
                v = __builtin_amdgcn_readlane(wave_scan((int)v, most), 63);
                if (lane == 0) {
                    if (QUANT) atomicMax(&s_top[0][0], k);
                    atomicMax(&s_top[0][1], v);
                }
            } else {
                if (QUANT && k >= lim_k) atomicMax(&s_top[t % 3][0], k);
                if (v >= lim_v) atomicMax(&s_top[t % 3][1], v);
            }
        };
        // the tile in registers into its buffer
        auto write_tile = [&](int t, const Raw &r) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                const int part = (p_row0 + 8 * WR * i) / kDiffKeys;
                const bool val = part >= 2;
                u32x4 x;
                if constexpr (QUANT) {
                    const float s = r.s[i] * (val ? fv : fk);
                    const f32x4 lo = code_values<DT>(r.w[i][0], s), hi = code_values<DT>(r.w[i][1], s);
                    x = u32x4{f16_pair(lo[0], lo[1]), f16_pair(lo[2], lo[3]), f16_pair(hi[0], hi[1]), f16_pair(hi[2], hi[3])};
                } else {
                    x = u32x4{r.w[i][0], r.w[i][1], r.w[i][2], r.w[i][3]};
                    if (val) {
                        if (fv == 1.0f) {
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                x[j] = f16_pair(__uint_as_float(x[j] << 16), __uint_as_float(x[j] & 0xFFFF0000u));
                        } else {
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                x[j] = f16_pair(__uint_as_float(x[j] << 16) * fv, __uint_as_float(x[j] & 0xFFFF0000u) * fv);
                        }
                    }
                }
                if (val && t * kDiffKeys + kDiffKeys - 1 > seesb && p_in) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const int sh = 16 * (j & 1);
                        if ((x[j / 2] >> sh & 0x7C00u) != 0x7C00u) continue;
                        x[j / 2] &= ~(0xFFFFu << sh);
                        // a finite value that left the range: the tile is staged again
                        if constexpr (QUANT) {
                            const float y = __builtin_fabsf(r.s[i]);
                            if (y < INFINITY && y * fv >= kMost) continue;
                        } else if ((r.w[i][j / 2] >> sh & 0x7F80u) != 0x7F80u) {
                            continue;
                        }
                        s_any = 1;
                        atomicMin(&s_bad[(part & 1) * D + 8 * p_c + j], t * kDiffKeys + p_key);
                    }
                }
                if (p_in) *reinterpret_cast<u32x4 *>(s_t(t) + part * HB + (val ? p_vlds : p_klds)) = x;
            }
        };

        float fk_now = fk;                             // the keys' power of two of the present tile
        // Behind the barrier after tile j was staged: whether its marks (largest key scale kt,
        // value vt) ask for another power of two; then it has to be staged again.
        auto settle = [&](uint32_t kt, uint32_t vt) __attribute__((always_inline)) -> bool {
            const float kx = __uint_as_float(kt) * fk, vx = __uint_as_float(vt) * fv;
            const bool newk = QUANT && kt && !(kx >= kLeast && kx < kMost), newv = vt && !(vx >= kLeast && vx < kMost);
            if (newk) fk = pow2_to(__uint_as_float(kt), kAim);
            if (newv) {
                const float now = pow2_to(__uint_as_float(vt), kAim);
                if (lim_v != 1) owed_next *= now / fv; // (else the sums are zeros)
                fv = now;
            }
            // where kMost lies without the power of two (past the largest float: nothing is marked)
            auto limit = [&](float f) __attribute__((always_inline)) {
                const int e = exponent(kMost) - exponent(f);
                return e > 127 ? 0x7F800000u : (uint32_t)(e + 127) << 23;
            };
            if (kt) lim_k = limit(fk);
            if (vt) lim_v = limit(fv);
            return newk || newv;
        };
        Raw raw;
        {
            Raw r0;
            load_tile(0, r0);
            if (1 < tiles) load_tile(1, raw);
            __syncthreads();                           // the buffers of the block before are free
            if (tid < 2 * D) s_bad[tid] = INT32_MAX;
            if (tid == 0) s_any = 0;
            if (tid < 6) s_top[tid / 2][tid % 2] = 0;
            __syncthreads();
            mark(0, r0);
            write_tile(0, r0);
            __syncthreads();
            if (settle(__builtin_amdgcn_readfirstlane(s_top[0][0]), __builtin_amdgcn_readfirstlane(s_top[0][1]))) {
                write_tile(0, r0);
                __syncthreads();
            }
            if (1 < tiles) {
                mark(1, raw);
                write_tile(1, raw);
                if (2 < tiles) load_tile(2, raw);
            }
        }
        fk_now = fk;
        f32x16 sc;
        // A tile is staged two ahead, with one barrier a tile.  Map 0's waves pass it before
        // a tile's first product, map 1's between that product and the softmax, so that on
        // each SIMD one wave's products meet the other's arithmetic.
        for (int t = 0; t < tiles; ++t) {
            const bool some = t * kDiffKeys <= sees1;  // some row of this wave sees some of it
            auto scores = [&]() __attribute__((always_inline)) {
                const uint8_t *sk = s_t(t) + mp * HB;
#pragma unroll
                for (int i = 0; i < 16; ++i) sc[i] = 0.0f;
                {
                    // a fragment is read while the products of those before it run
                    constexpr int AHEAD = KS < 3 ? KS : 3;
                    int at = r32;                      // (the chunks' places are not kept in registers from tile to tile)
                    asm volatile("" : "+v"(at));
                    u32x4 kf[KS];
#pragma unroll
                    for (int s = 0; s < KS; ++s)
                        kf[s] = *reinterpret_cast<const u32x4 *>(sk + at * RB + 16 * key_chunk<D>(at, 2 * s + hf));
#pragma unroll
                    for (int s = 0; s < KS; ++s) sc = mfma<QUANT>(kf[s], qf[s], sc);
                    read_ahead<KS, AHEAD, 1>();
                }
            };
            if (mp && some) scores();
            __syncthreads();                           // tile t + 1 is staged, tile t - 1 used
            const uint32_t kt = s_top[(t + 1) % 3][0], vt = s_top[(t + 1) % 3][1];
            if (tid < 2) s_top[t % 3][tid] = 0;
            if (!mp && some) scores();
            if (__builtin_amdgcn_readfirstlane(kt | vt)) {
                if (settle(__builtin_amdgcn_readfirstlane(kt), __builtin_amdgcn_readfirstlane(vt))) {       // rare
                    const bool ahead = t + 2 < tiles;  // (it is in the registers)
                    load_rows(t + 1, ahead ? blk_before : blk_at, raw);
                    write_tile(t + 1, raw);
                    __syncthreads();
                    if (ahead) load_rows(t + 2, blk_at, raw);
                }
            }
            if (some) {
                // what the products have to be multiplied by.  Neither 0 nor infinite: a masked
                // score, -inf, times 0 would be NaN, and so would 0 times infinity.  (Products are
                // below 2^32: under the least factor here their scores are 0 all the same.)
                float ft = a.scale_log2;
                if constexpr (QUANT) ft = __builtin_amdgcn_ldexpf(ft, -(qe + exponent(fk_now)));
                ft = fminf(fmaxf(ft, 0x1p-126f), 0x1.fffffep127f);
                const uint8_t *sv = s_t(t) + 2 * HB;
                const bool cut = t * kDiffKeys + kDiffKeys - 1 > sees0;
                if (cut) {
                    const int lim = sees - t * kDiffKeys;
#pragma unroll
                    for (int i = 0; i < 16; ++i) sc[i] = 8 * (i / 4) + 4 * hf + i % 4 <= lim ? sc[i] : -INFINITY;
                }
                float top = sc[0];
#pragma unroll
                for (int i = 1; i < 16; ++i) top = fmaxf(top, sc[i]);
                top = max_x32(top) * ft;
                // another base where a probability would pass 2^(kUp + kSlack), and on the first tile.
                // Scores past 2^22 are whole numbers or nearly: kUp would be lost in their rounding, and
                // each is rounded as the largest was, so that its distance from the base is exact.
                if (__ballot(top > lim) != 0ull) {
                    const float now = top - base > kUp + kSlack ? top - (__builtin_fabsf(top) < 0x1p22f ? kUp : 0.0f) : base;
                    float alpha = base == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(base - now);
                    l_run *= alpha;
                    alpha *= owed;
                    owed = 1.0f;
#pragma unroll
                    for (int c = 0; c < CT; ++c) acc[c] *= alpha;
                    base = now;
                    const bool far = !(__builtin_fabsf(base) < 0x1p22f);
                    lim = far ? -INFINITY : base + (kUp + kSlack);
                    if (__ballot(far) != 0ull) {
#pragma unroll
                        for (int i = 0; i < 16; ++i) sc[i] *= ft;
                        ft = 1.0f;
                    }
                }
                const float from = base == -INFINITY ? 0.0f : base;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    sc[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[i], ft, -from));
                    l_run += sc[i];
                }
                u32x4 p[2];
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                    for (int j = 0; j < 4; ++j) p[s][j] = f16_pair(sc[8 * s + 2 * j], sc[8 * s + 2 * j + 1]);
                // V^T as the A operand: lane (m, h) takes keys 16 s + 8 b + 4 h .. +4 of column m, b = 0, 1.
                // Within each 16-lane group, lane j of a transposing read receives element j % 4 of the 8
                // bytes that lanes 4 k + j / 4 address, k = 0 .. 3: lane i points at key i / 4 of the four
                // and columns 4 (i % 4) of the group's sixteen.
                int ln = lane;
                asm volatile("" : "+v"(ln));
                const int vr = 4 * (ln >> 5) + ((ln & 15) >> 2);
                u32x4 vf[CT][2];
#pragma unroll
                for (int c = 0; c < CT; ++c) {
                    const int hd = c / (D / 32), cl = c % (D / 32);
                    const int vc = 4 * cl + 2 * ((ln >> 4) & 1) + ((ln & 3) >> 1);
                    const uint8_t *v = sv + hd * HB + vr * RB + 16 * value_chunk<D>(vr, vc) + 8 * (ln & 1);
#pragma unroll
                    for (int s = 0; s < 2; ++s) {
                        typedef short s16x4 __attribute__((ext_vector_type(4)));
                        const u32x2 x = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                            (__attribute__((address_space(3))) s16x4 *)(v + 16 * s * RB)));
                        const u32x2 y = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                            (__attribute__((address_space(3))) s16x4 *)(v + (16 * s + 8) * RB)));
                        vf[c][s] = u32x4{x[0], x[1], y[0], y[1]};
                    }
                }
#pragma unroll
                for (int c = 0; c < CT; ++c)
#pragma unroll
                    for (int s = 0; s < 2; ++s) acc[c] = mfma<true>(vf[c][s], p[s], acc[c]);
                read_ahead<2 * CT, 3, 2>();
            }
            if (t + 2 < tiles) {
                mark(t + 2, raw);
                write_tile(t + 2, raw);
                if (t + 3 < tiles) load_tile(t + 3, raw);
            }
            fk_now = fk;
            if (owed_next != 1.0f) {                   // rare; paid with the next change of base, at once
                owed *= owed_next;
                owed_next = 1.0f;
                lim = -INFINITY;
            }
        }

        // lane (n, h): columns 32 c + 8 (i / 4) + 4 h + i % 4 of row n in acc[c][i]
        const float l = sum_x32(l_run);
        // the row again (its place in the output is not kept in registers through the tiles)
        bool live;
        int tok, h, r_end = r32;
        asm volatile("" : "+v"(r_end));
        my_row(r_end, live, tok, h);
        __syncthreads();
        if (s_any) {
#pragma unroll
            for (int c = 0; c < CT; ++c)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (s_bad[32 * c + 8 * (i / 4) + 4 * hf + i % 4] <= sees) acc[c][i] = __builtin_nanf("");
        }
        const float back = owed / fv;
        if (whole) {
            // the row's other map comes through the buffers: map 0's waves end the first half
            // of the columns, map 1's the second, CR tiles of those at a time
            const float lam = a.e.lam[(row0 + tok) * a.e.lam_stride + h];
            const float inv = back * (mp ? -lam : 1.0f) / l;
            float ss = 0.0f;
            f32x4 *x = reinterpret_cast<f32x4 *>(s_mem) + lane;
#pragma unroll
            for (int c0 = 0; c0 < CH; c0 += CR) {
                __syncthreads();
#pragma unroll
                for (int c = c0; c < c0 + CR && c < CH; ++c)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        f32x4 o;
#pragma unroll
                        for (int j = 0; j < 4; ++j) o[j] = (mp ? acc[c][4 * i + j] : acc[CH + c][4 * i + j]) * inv;
                        x[(((4 * mp + rg) * CR + c - c0) * 4 + i) * 64] = o;
                    }
                __syncthreads();
#pragma unroll
                for (int c = c0; c < c0 + CR && c < CH; ++c)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const f32x4 y = x[(((4 * (1 - mp) + rg) * CR + c - c0) * 4 + i) * 64];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const float z = (mp ? acc[CH + c][4 * i + j] : acc[c][4 * i + j]) * inv + y[j];
                            acc[c][4 * i + j] = z;
                            ss += z * z;
                        }
                    }
            }
            float k = a.e.scale;
            if (a.e.norm) {
                ss = sum_x32(ss);
                if (hf == 0) s_ss[mp][rg][r32] = ss;
                __syncthreads();
                k = diff_factor(a.e, ss + s_ss[1 - mp][rg][r32], 2 * D);
            }
            if (live) {
                uint16_t *o = (uint16_t *)a.e.out + ((row0 + tok) * a.pairs + h) * (2 * D) + mp * D + 8 * hf;
#pragma unroll
                for (int c = 0; c < CH; ++c)
#pragma unroll
                    for (int i = 0; i < 4; i += 2) {
                        u32x2 x[2];
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const f32x4 n = *reinterpret_cast<const f32x4 *>(s_w + mp * D + 32 * c + 8 * (i + e) + 4 * hf) * k;
                            x[e] = u32x2{bf16_pair(acc[c][4 * (i + e)] * n[0], acc[c][4 * (i + e) + 1] * n[1]),
                                         bf16_pair(acc[c][4 * (i + e) + 2] * n[2], acc[c][4 * (i + e) + 3] * n[3])};
                        }
                        *reinterpret_cast<u32x4 *>(o + 32 * c + 8 * i) = eight(x[0], x[1]);
                    }
            }
        } else {
            const int64_t slot = 2 * cell + (t0 == 0 ? 1 : 0);
            const int64_t r = (slot * kRows + 32 * rg + r32) * 2 + mp;
            // the piece's sums, without the probabilities' and the values' powers of two (f16 means
            // in their place would err by 2^-12 of a map, which the difference of two alike does not keep)
            // and under 2^-24, so that sums over a million keys of values near the largest f32 are finite
            const float down = __builtin_amdgcn_exp2f(-kUp - 24.0f);
            float *o = a.part_o + r * (2 * D) + 4 * hf;
#pragma unroll
            for (int c = 0; c < CT; ++c)
#pragma unroll
                for (int i = 0; i < 16; i += 4)
                    *reinterpret_cast<f32x4 *>(o + 32 * c + 2 * i) =
                        f32x4{acc[c][i] * down * back, acc[c][i + 1] * down * back, acc[c][i + 2] * down * back, acc[c][i + 3] * down * back};
            if (hf == 0) {
                a.part_ml[2 * r] = base;
                a.part_ml[2 * r + 1] = l * down;
            }
            if (t0 == 0) {                          // begun here: its last unit's slice ends it
                const int64_t last = u - t1 + nt - 1;      // of the launch's units
                begun = int4{it.b, (int)(uint32_t)it.k, (int)(it.k >> 32), (int)(last / chunk - w + 1)};
            }
        }
    }
    if (tid == 0) a.desc[cell] = begun;
}

template <int D>
hipError_t launch_d(const DiffPrefillArgs &a, hipStream_t s) {
    const dim3 grid((unsigned)a.slices, (unsigned)a.kv_pairs);
    if (a.dtype == AIR_KV_BF16) hipLaunchKernelGGL((diff_prefill_16_kernel<D, AIR_KV_BF16>), grid, dim3(kThreads16), 0, s, a);
    else if (a.dtype == AIR_KV_INT8) hipLaunchKernelGGL((diff_prefill_16_kernel<D, AIR_KV_INT8>), grid, dim3(kThreads16), 0, s, a);
    else hipLaunchKernelGGL((diff_prefill_16_kernel<D, AIR_KV_FP8>), grid, dim3(kThreads16), 0, s, a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_diff_prefill_16(const DiffPrefillArgs &a, int head_dim, hipStream_t s) {
    return head_dim == 128 ? launch_d<128>(a, s) : head_dim == 96 ? launch_d<96>(a, s) : head_dim == 64 ? launch_d<64>(a, s) : launch_d<32>(a, s);
}

}  // namespace airkv
