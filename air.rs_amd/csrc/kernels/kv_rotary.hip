// Rotary positions on the way into the pages (append) and inside them (rotate); angles and
// pairs: rotary.hpp.
//
// A lane owns 8 consecutive elements of a row, as kv_append.hip's: the codes and scales of
// 1-byte pages are then made by the same lanes and code.  Rows take a power of two of lanes,
// so that a row lies in one wave: its lanes load what they turn, their own elements and the
// partners', before any of them stores, and a row may be written where it was read.
//
// Both move bytes: an append reads and writes each row once (8192 tokens of 32 + 16 heads of 128, bf16:
// 44.8 us, 4.5 TB/s; int8 pages 47.8), a rotation reads and writes the keys alone (4 sequences of 16000
// tokens, 8 heads of 128, bf16 50.7 us, f32 79 us; a copy of 2 GiB reaches 4.9 TB/s read and written).
// A position costs rot_dim / 2 angles in 64 bits, computed once a token, in a workgroup's LDS, while the
// first rows are on their way.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../pool.hpp"
#include "codecs.hpp"
#include "page_io.hpp"
#include "rotary.hpp"

namespace airkv {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr int kThreads = 256;
constexpr int kMaxPairs = 128;         // head_dim up to 256

struct RotaryPool {
    void *k_pages, *v_pages;
    float *k_scales, *v_scales;
    int64_t num_blocks;
    int32_t heads, head_dim, bs_log2, sg_log2;      // K/V heads; block size and scale group are powers of two
    int32_t lanes_log2;                             // of a row
    unsigned long long *errors;
};

struct Rotary {
    const float *inv_freq;
    int32_t rot;
    bool pairs;
    float magnitude;
};

// Four elements as they lie in memory (bf16 or f32), and as f32.
template <bool HALF> struct Four;
template <> struct Four<true> {
    u32x2 w;
    __device__ __forceinline__ void load(const void *p, int64_t at) { w = __builtin_nontemporal_load(reinterpret_cast<const u32x2 *>((const uint16_t *)p + at)); }
    __device__ __forceinline__ void get(float *x) const {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            x[2 * j] = __uint_as_float(w[j] << 16);
            x[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
        }
    }
};
template <> struct Four<false> {
    f32x4 w;
    __device__ __forceinline__ void load(const void *p, int64_t at) { w = *reinterpret_cast<const f32x4 *>((const float *)p + at); }
    __device__ __forceinline__ void get(float *x) const {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = w[j];
    }
};

// 8 f32 to a page or an output of type DT, as store_row_chunk; bf16 by the hardware's rounding (to
// nearest even, a NaN stays one), where bf16_rne's branches cost more than all else.
template <int DT>
__device__ __forceinline__ void store8(const float (&x)[8], void *pages, float *scales, int64_t elem, int64_t scale_idx, bool lead, int lanes) {
    if constexpr (DT == AIR_KV_BF16) {
        typedef float f32x2 __attribute__((ext_vector_type(2)));
        typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
        u32x4 w;
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{x[2 * j], x[2 * j + 1]}), bf16x2));
        *reinterpret_cast<u32x4 *>((uint16_t *)pages + elem) = w;
    } else {
        store_row_chunk<DT>(x, pages, scales, elem, scale_idx, lead, lanes, true);
    }
}

// A row's lanes have loaded what they turn before any of them stores: a wave runs in step, and neither the
// compiler nor the memory moves an access over this.  (No instruction.)
__device__ __forceinline__ void row_loaded() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// The 8 elements x from element e on of a row, turned; y their partners (half layout).
__device__ __forceinline__ void turn8(float (&x)[8], const float (&y)[2][4], const Rotary &r, const float2 *cs, int e) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if (e + 4 * i >= r.rot) continue;
        float z[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) z[j] = x[4 * i + j];
        if (r.pairs) rotary_pairs4(z, cs, e + 4 * i);
        else rotary_half4(z, y[i], cs, e + 4 * i, r.rot / 2);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[4 * i + j] = z[j];
    }
}

struct AppendArgs {
    RotaryPool p;
    Rotary r;
    const void *q, *k, *v;
    int64_t q_stride, k_stride, v_stride;           // elements from one token's row to the next
    int32_t q_heads;
    void *q_out;
    const int64_t *slots;
    const int32_t *positions;
    int32_t per_part;                               // rows (heads of q, k and v) of a workgroup
};

// One token and per_part of its rows (query heads, then key heads, then value heads).  A row is
// read before the one before it is stored; the angles are computed while the first is on its way.
template <int DT, bool IN16, bool OUT16>
__global__ __launch_bounds__(kThreads) void append_rotary_kernel(AppendArgs a) {
    __shared__ float2 s_cs[kMaxPairs];
    const int64_t t = blockIdx.x;
    const int tid = threadIdx.x, d = a.p.head_dim;
    const int e = (tid & ((1 << a.p.lanes_log2) - 1)) * 8, step = kThreads >> a.p.lanes_log2;
    const int all = a.q_heads + 2 * a.p.heads;
    const int end = min(all, (int)(blockIdx.y + 1) * a.per_part);
    struct Row {
        Four<IN16> own[2], partner[2];
    };
    auto load = [&](int row, Row &x) __attribute__((always_inline)) {
        if (row >= end || e >= d) return;
        const bool q = row < a.q_heads, k = !q && row < a.q_heads + a.p.heads;
        const void *src = q ? a.q : k ? a.k : a.v;
        const int h = q ? row : k ? row - a.q_heads : row - a.q_heads - a.p.heads;
        const int64_t from = t * (q ? a.q_stride : k ? a.k_stride : a.v_stride) + (int64_t)h * d;
#pragma unroll
        for (int i = 0; i < 2; ++i) x.own[i].load(src, from + e + 4 * i);
        if ((q || k) && !a.r.pairs) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if (e + 4 * i < a.r.rot) x.partner[i].load(src, from + rotary_partner(e + 4 * i, a.r.rot / 2));
        }
    };
    int row = blockIdx.y * a.per_part + (tid >> a.p.lanes_log2);
    const int64_t slot = a.slots[t];
    const int position = a.positions[t];
    Row now, next;
    load(row, now);
    const bool kept = slot >= 0 && slot < a.p.num_blocks << a.p.bs_log2;
    if (blockIdx.y == 0 && tid == 0 && slot >= a.p.num_blocks << a.p.bs_log2) atomicAdd(a.p.errors, 1ull);
    if (tid < a.r.rot / 2) s_cs[tid] = rotary_turn(position, a.r.inv_freq[tid], a.r.magnitude);
    __syncthreads();
    if (e >= d) return;
    constexpr bool QUANT = DT == AIR_KV_INT8 || DT == AIR_KV_FP8;      // (their codes need the registers)
    for (; row < end; row += step) {
        if (!QUANT) load(row + step, next);
        const int kind = row < a.q_heads ? 0 : row < a.q_heads + a.p.heads ? 1 : 2;
        if (kind == 0 || kept) {
            float x[8], y[2][4];
            now.own[0].get(x);
            now.own[1].get(x + 4);
            if (kind < 2) {
                if (!a.r.pairs) {
                    now.partner[0].get(y[0]);
                    now.partner[1].get(y[1]);
                }
                turn8(x, y, a.r, s_cs, e);
            }
            row_loaded();                              // (q_out may be q)
            if (kind == 0) {
                const int64_t to = (t * a.q_heads + row) * d + e;
                if constexpr (OUT16) store8<AIR_KV_BF16>(x, a.q_out, nullptr, to, 0, false, 1);
                else store8<AIR_KV_F32>(x, a.q_out, nullptr, to, 0, false, 1);
            } else {
                const int h = kind == 1 ? row - a.q_heads : row - a.q_heads - a.p.heads;
                const int64_t dst = (((slot >> a.p.bs_log2) * a.p.heads + h) << a.p.bs_log2) + (slot & ((1 << a.p.bs_log2) - 1));
                int lanes = 1;
                int64_t sc = 0;
                bool lead = false;
                if constexpr (DT == AIR_KV_INT8 || DT == AIR_KV_FP8) {
                    lanes = 1 << (a.p.sg_log2 - 3);
                    sc = dst * (d >> a.p.sg_log2) + (e >> a.p.sg_log2);
                    lead = ((e >> 3) & (lanes - 1)) == 0;
                }
                store8<DT>(x, kind == 1 ? a.p.k_pages : a.p.v_pages, kind == 1 ? a.p.k_scales : a.p.v_scales, dst * d + e, sc, lead, lanes);
            }
        }
        if (QUANT) load(row + step, now);
        else now = next;
    }
}

// Four cached elements of a row of a scale group's or wider.
template <int DT>
__device__ __forceinline__ void cached4(const void *pages, const float *scales, int64_t row, int d, int sg_log2, int e, float (&x)[4]) {
    const int64_t at = row * d + e;
    if constexpr (DT == AIR_KV_F32) {
        Four<false> f;
        f.load(pages, at);
        f.get(x);
    } else if constexpr (DT == AIR_KV_BF16) {
        Four<true> f;
        f.load(pages, at);
        f.get(x);
    } else {
        const uint32_t w = *reinterpret_cast<const uint32_t *>((const uint8_t *)pages + at);
        const float s = scales[row * (d >> sg_log2) + (e >> sg_log2)];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t byte = (w >> (8 * j)) & 0xFFu;
            const float val = DT == AIR_KV_INT8 ? (float)(int32_t)(int8_t)byte : fp8_decode(byte);
            {
#pragma clang fp contract(off)
                x[j] = val * s;
            }
        }
    }
}

struct RotateArgs {
    RotaryPool p;
    Rotary r;
    const int32_t *tables, *from, *to, *cu;         // to NULL: a token's place in its sequence
    int32_t max_blocks, total;
};

constexpr int kRun = 16;               // tokens at a time: they share a block

// A sequence's runs of kRun tokens, run y, y + gridDim.y, ...: its angles first, then the
// heads' rows, which of one head lie side by side.
template <int DT>
__global__ __launch_bounds__(kThreads) void rotate_kernel(RotateArgs a) {
    constexpr bool QUANT = DT == AIR_KV_INT8 || DT == AIR_KV_FP8;
    __shared__ float2 s_cs[kRun * kMaxPairs];
    __shared__ int64_t s_by[kRun];
    const int b = blockIdx.x, tid = threadIdx.x, d = a.p.head_dim, half = a.r.rot / 2;
    const int c0 = a.cu[b], c1 = a.cu[b + 1];
    if (c0 < 0 || c1 > a.total || c1 < c0) {
        if (blockIdx.y == 0 && tid == 0) atomicAdd(a.p.errors, 1ull);
        return;
    }
    const int n = c1 - c0;
    const int e = (tid & ((1 << a.p.lanes_log2) - 1)) * 8;
    const int row0 = tid >> a.p.lanes_log2, rows = kThreads >> a.p.lanes_log2;
    for (int64_t at = (int64_t)blockIdx.y * kRun; at < n; at += (int64_t)gridDim.y * kRun) {
        const int64_t index = at >> a.p.bs_log2;
        const int32_t block = index < a.max_blocks ? a.tables[(int64_t)b * a.max_blocks + index] : -1;
        const int here = n - at < kRun ? (int)(n - at) : kRun;
        if (block < 0 || block >= a.p.num_blocks) {
            if (tid == 0) atomicAdd(a.p.errors, (unsigned long long)here);
            continue;
        }
        int64_t by = 0;
        if (tid < here) {
            const int64_t i = c0 + at + tid;
            by = (a.to ? (int64_t)a.to[i] : at + tid) - a.from[i];
        }
        if (tid < kRun) s_by[tid] = by;
        if (!__syncthreads_or(by != 0)) continue;      // (also: the rows of the run before are done)
#pragma unroll 1
        for (int i = tid; i < here * half; i += kThreads) {
            const int k = i / half;
            s_cs[i] = rotary_turn(s_by[k], a.r.inv_freq[i - k * half], 1.0f);
        }
        __syncthreads();
        const int64_t first = ((int64_t)block * a.p.heads << a.p.bs_log2) + (at & ((1 << a.p.bs_log2) - 1));
        if (e < d) {
            for (int i = row0; i < kRun * a.p.heads; i += rows) {
                const int k = i % kRun, h = i / kRun;
                if (k >= here || s_by[k] == 0) continue;
                const int64_t row = first + ((int64_t)h << a.p.bs_log2) + k;
                const int lanes = QUANT ? 1 << (a.p.sg_log2 - 3) : 1;
                // 1-byte pages: whole scale groups, as far as one holds a turned element
                const int end = QUANT ? (((a.r.rot - 1) >> a.p.sg_log2) + 1) << a.p.sg_log2 : a.r.rot;
                if (e >= end) continue;
                float x[8];
                auto four = [&](int e4, float (&y)[4]) { cached4<DT>(a.p.k_pages, a.p.k_scales, row, d, a.p.sg_log2, e4, y); };
                float lo[4], hi[4];
                four(e, lo);
                four(e + 4, hi);
#pragma unroll
                for (int j = 0; j < 4; ++j) { x[j] = lo[j]; x[4 + j] = hi[j]; }
                float y[2][4];
                if (!a.r.pairs) {
#pragma unroll
                    for (int p = 0; p < 2; ++p)
                        if (e + 4 * p < a.r.rot) four(rotary_partner(e + 4 * p, half), y[p]);
                }
                turn8(x, y, a.r, s_cs + k * half, e);
                row_loaded();
                const int64_t sc = QUANT ? row * (d >> a.p.sg_log2) + (e >> a.p.sg_log2) : 0;
                store8<DT>(x, a.p.k_pages, a.p.k_scales, row * d + e, sc, ((e >> 3) & (lanes - 1)) == 0, lanes);
            }
        }
        __syncthreads();
    }
}

// The same where a row is floats and rot a multiple of 16: a lane owns 8 elements and their 8
// partners (or 16 neighbours) of one token's rows, so nothing is read twice, and the pairs' c and s
// stay in its registers from head to head.  (4 sequences of 16000 tokens: bf16 50.7 us, with the kernel
// above 86; f32 79 and 86.)  ROWS rows are on their way before the first is stored, as many as leave four
// waves a SIMD (bf16 / f32: 1 and 1 rows 55.7 / 80, 2 and 1 51.9 / 79, 4 and 2 48.5 / 81 but 131 in place of
// 129 us for sequences whose keys no cache holds, and one f32 sequence 23.7 in place of 21.2).
template <bool HALF, bool PAIRS>
__global__ __launch_bounds__(kThreads, 4) void rotate_floats_kernel(RotateArgs a) {
    __shared__ float2 s_cs[kRun * kMaxPairs];
    const int b = blockIdx.x, tid = threadIdx.x, d = a.p.head_dim, half = a.r.rot / 2;
    const int c0 = a.cu[b], c1 = a.cu[b + 1];
    if (c0 < 0 || c1 > a.total || c1 < c0) {
        if (blockIdx.y == 0 && tid == 0) atomicAdd(a.p.errors, 1ull);
        return;
    }
    const int n = c1 - c0;
    int lanes_log2 = 0;                                // of a row, 16 elements each
    while (16 << lanes_log2 < a.r.rot) ++lanes_log2;
    const int part = tid & ((1 << lanes_log2) - 1), k = (tid >> lanes_log2) % kRun;
    const int group = tid >> lanes_log2 >> 4, groups = kThreads >> lanes_log2 >> 4;        // of heads
    const int e0 = PAIRS ? 16 * part : 8 * part, e1 = PAIRS ? e0 + 8 : e0 + half;
    constexpr int ROWS = HALF ? 2 : 1;                 // on their way
    const int stride = (int)gridDim.y * kRun;
    for (int64_t at = (int64_t)blockIdx.y * kRun; at < n; at += stride) {
        const int64_t index = at >> a.p.bs_log2;
        const int32_t block = index < a.max_blocks ? a.tables[(int64_t)b * a.max_blocks + index] : -1;
        const int here = n - at < kRun ? (int)(n - at) : kRun;
        auto turn = [&](int i) __attribute__((always_inline)) -> int64_t {     // of token i of the run
            const int64_t j = c0 + at + i;
            return i < here ? (a.to ? (int64_t)a.to[j] : at + i) - a.from[j] : 0;
        };
        const int64_t by = turn(k);
        if (block < 0 || block >= a.p.num_blocks) {
            if (tid == 0) atomicAdd(a.p.errors, (unsigned long long)here);
            continue;
        }
        const bool mine = by != 0 && 16 * part < a.r.rot;
        const int64_t row = (((int64_t)block * a.p.heads << a.p.bs_log2) + (at & ((1 << a.p.bs_log2) - 1)) + k) * d;
        Four<HALF> x[ROWS][4];
        auto load = [&](int h, Four<HALF> (&x)[4]) __attribute__((always_inline)) {
            if (!mine || h >= a.p.heads) return;
            const int64_t from = row + ((int64_t)h << a.p.bs_log2) * d;
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i].load(a.p.k_pages, from + (i < 2 ? e0 + 4 * i : e1 + 4 * (i - 2)));
        };
#pragma unroll
        for (int r = 0; r < ROWS; ++r) load(group + r * groups, x[r]);
        if (!__syncthreads_or(by != 0)) continue;      // (also: the angles of the run before are used)
        // (lanes a row hold 8 pairs each)
#pragma unroll 1                                       // (unrolled, it takes the registers of the rows on their way)
        for (int i = tid; i < kRun << (lanes_log2 + 3); i += kThreads) {
            const int token = i >> (lanes_log2 + 3), pair = i & ((8 << lanes_log2) - 1);
            if (pair < half) s_cs[token * half + pair] = rotary_turn(turn(token), a.r.inv_freq[pair], 1.0f);
        }
        __syncthreads();
        if (!mine) continue;
        float2 cs[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) cs[j] = s_cs[k * half + 8 * part + j];
#pragma unroll 1
        for (int h0 = group; h0 < a.p.heads; h0 += ROWS * groups) {
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
                const int h = h0 + r * groups;
                if (h >= a.p.heads) break;
                float y[2][8];
#pragma unroll
                for (int i = 0; i < 4; ++i) x[r][i].get(y[i / 2] + 4 * (i % 2));
                load(h + ROWS * groups, x[r]);
#pragma unroll
                for (int j = 0; j < 8; ++j) {          // pair j: elements j of both halves, or neighbours
                    if constexpr (PAIRS) rotary_pair(y[j / 4][2 * (j % 4)], y[j / 4][2 * (j % 4) + 1], cs[j]);
                    else rotary_pair(y[0][j], y[1][j], cs[j]);
                }
                const int64_t to = row + ((int64_t)h << a.p.bs_log2) * d;
                store8<HALF ? AIR_KV_BF16 : AIR_KV_F32>(y[0], a.p.k_pages, nullptr, to + e0, 0, false, 1);
                store8<HALF ? AIR_KV_BF16 : AIR_KV_F32>(y[1], a.p.k_pages, nullptr, to + e1, 0, false, 1);
            }
        }
    }
}

RotaryPool pool_args(const air_kv_pool &p) {
    RotaryPool a;
    a.k_pages = p.k_pages;
    a.v_pages = p.v_pages;
    a.k_scales = p.k_scales;
    a.v_scales = p.v_scales;
    a.num_blocks = p.desc.num_blocks;
    a.heads = p.desc.n_kv_heads;
    a.head_dim = p.desc.head_dim;
    a.bs_log2 = __builtin_ctz((unsigned)p.desc.block_size);
    a.sg_log2 = p.desc.scale_group > 0 ? __builtin_ctz((unsigned)p.desc.scale_group) : 0;
    a.lanes_log2 = 2;                               // 8 elements a lane
    while (8 << a.lanes_log2 < p.desc.head_dim) ++a.lanes_log2;
    a.errors = p.errors;
    return a;
}

template <bool IN16, bool OUT16>
hipError_t launch_append_io(const AppendArgs &a, int dtype, dim3 grid, hipStream_t s) {
    switch (dtype) {
    case AIR_KV_F32: hipLaunchKernelGGL((append_rotary_kernel<AIR_KV_F32, IN16, OUT16>), grid, dim3(kThreads), 0, s, a); break;
    case AIR_KV_BF16: hipLaunchKernelGGL((append_rotary_kernel<AIR_KV_BF16, IN16, OUT16>), grid, dim3(kThreads), 0, s, a); break;
    case AIR_KV_INT8: hipLaunchKernelGGL((append_rotary_kernel<AIR_KV_INT8, IN16, OUT16>), grid, dim3(kThreads), 0, s, a); break;
    default: hipLaunchKernelGGL((append_rotary_kernel<AIR_KV_FP8, IN16, OUT16>), grid, dim3(kThreads), 0, s, a); break;
    }
    return hipGetLastError();
}

}  // namespace

hipError_t launch_append_rotary(const air_kv_pool &p, hipStream_t s, const void *q, int64_t q_stride, int32_t n_q_heads,
                                const void *k, int64_t k_stride, const void *v, int64_t v_stride, int32_t in_dtype,
                                const int64_t *slots, const int32_t *positions, int32_t n_tokens, const float *inv_freq,
                                int32_t rot_dim, int32_t layout, float magnitude, void *q_out, int32_t q_out_dtype) {
    AppendArgs a;
    a.p = pool_args(p);
    a.r = {inv_freq, rot_dim, layout == AIR_ROTARY_PAIRS, magnitude};
    a.q_stride = q_stride; a.k_stride = k_stride; a.v_stride = v_stride;
    a.q_heads = n_q_heads;
    const int all = n_q_heads + 2 * p.desc.n_kv_heads, pass = kThreads >> a.p.lanes_log2;
    // few tokens: a pass of rows per workgroup, until the CUs have two each (bf16, us, split and whole: 64
    // tokens 3.0, 4.4; 512: 4.9, 5.7; 1024: 7.9, 8.1; 4096: 26.7, 25.3; int8, 1024: 9.1, 8.7)
    int parts = (all + pass - 1) / pass;
    if (n_tokens > 2 * p.cus) parts = 1;
    a.per_part = (all + parts - 1) / parts;
    const bool in16 = in_dtype == AIR_KV_BF16, out16 = q_out_dtype == AIR_KV_BF16;
    const int64_t in = in16 ? 2 : 4, out = out16 ? 2 : 4;
    // (a dispatch counts its work-items in 32 bits)
    constexpr int32_t kMost = 1 << 22;
    for (int64_t t0 = 0; t0 < n_tokens; t0 += kMost) {
        a.q = (const uint8_t *)q + t0 * q_stride * in;
        a.k = (const uint8_t *)k + t0 * k_stride * in;
        a.v = (const uint8_t *)v + t0 * v_stride * in;
        a.q_out = (uint8_t *)q_out + t0 * n_q_heads * p.desc.head_dim * out;
        a.slots = slots + t0;
        a.positions = positions + t0;
        const dim3 grid((unsigned)std::min<int64_t>(kMost, n_tokens - t0), (unsigned)parts);
        const hipError_t e = in16 ? out16 ? launch_append_io<true, true>(a, p.desc.dtype, grid, s)
                                          : launch_append_io<true, false>(a, p.desc.dtype, grid, s)
                             : out16 ? launch_append_io<false, true>(a, p.desc.dtype, grid, s)
                                     : launch_append_io<false, false>(a, p.desc.dtype, grid, s);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

hipError_t launch_rotate(const air_kv_pool &p, hipStream_t s, const int32_t *tables, int32_t batch, int32_t max_blocks,
                         const int32_t *from, const int32_t *to, const int32_t *cu, int32_t total, const float *inv_freq,
                         int32_t rot_dim, int32_t layout) {
    RotateArgs a;
    a.p = pool_args(p);
    a.r = {inv_freq, rot_dim, layout == AIR_ROTARY_PAIRS, 1.0f};
    a.tables = tables;
    a.from = from;
    a.to = to;
    a.cu = cu;
    a.max_blocks = max_blocks;
    a.total = total;
    // runs are dealt to workgroups, 16 a CU (bf16, us: one sequence of 16000 tokens 16.1 with 8, 15.4 with 16
    // and 64; 4 of 16000: 51.9, 50.7, 50.7; four a CU are resident)
    const int64_t runs = ((int64_t)total + kRun - 1) / kRun, most = std::max<int64_t>(1, (16LL * p.cus + batch - 1) / batch);
    const dim3 grid((unsigned)batch, (unsigned)std::max<int64_t>(1, std::min(runs, most)));
    if (rot_dim % 16 == 0 && !dtype_quantized(p.desc.dtype)) {
        const bool bf16 = p.desc.dtype == AIR_KV_BF16;
        if (a.r.pairs) {
            if (bf16) hipLaunchKernelGGL((rotate_floats_kernel<true, true>), grid, dim3(kThreads), 0, s, a);
            else hipLaunchKernelGGL((rotate_floats_kernel<false, true>), grid, dim3(kThreads), 0, s, a);
        } else {
            if (bf16) hipLaunchKernelGGL((rotate_floats_kernel<true, false>), grid, dim3(kThreads), 0, s, a);
            else hipLaunchKernelGGL((rotate_floats_kernel<false, false>), grid, dim3(kThreads), 0, s, a);
        }
        return hipGetLastError();
    }
    switch (p.desc.dtype) {
    case AIR_KV_F32: hipLaunchKernelGGL(rotate_kernel<AIR_KV_F32>, grid, dim3(kThreads), 0, s, a); break;
    case AIR_KV_BF16: hipLaunchKernelGGL(rotate_kernel<AIR_KV_BF16>, grid, dim3(kThreads), 0, s, a); break;
    case AIR_KV_INT8: hipLaunchKernelGGL(rotate_kernel<AIR_KV_INT8>, grid, dim3(kThreads), 0, s, a); break;
    default: hipLaunchKernelGGL(rotate_kernel<AIR_KV_FP8>, grid, dim3(kThreads), 0, s, a); break;
    }
    return hipGetLastError();
}

}  // namespace airkv
