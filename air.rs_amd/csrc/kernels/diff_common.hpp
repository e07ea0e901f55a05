// Shared parts of the differential attention kernels.
//
// K/V heads 2p and 2p + 1 of a pool are pair p.  Query pair h (query heads 2h
// and 2h + 1) reads K/V pair p = h / group:
//   s_m[t] = scale * q[2h + m] . K[2p + m][t]                   m = 0, 1
//   P_m    = softmax of s_m over the tokens the row sees
//   x      = sum_t (P_0[t] - lambda P_1[t]) (V[2p][t] | V[2p + 1][t])
//   out    = out_scale * (x, or x / sqrt(mean(x^2) + eps) * w)
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "air_kv.h"
#include "codecs.hpp"
#include "decode_slices.hpp"

namespace airkv {

// What turns the two maps' sums into an output row.
struct DiffOut {
    const float *lam;              // lambda of query pair h of row r: lam[r * lam_stride + h]
    int64_t lam_stride;            // 0: one per query pair
    const float *norm_w;           // [2 * head_dim], or NULL: ones
    float eps;                     // of the norm
    bool norm;
    float scale;
    void *out;                     // [rows][query pairs][2 * head_dim]
    int32_t out_dtype;
};

typedef float diff_f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t diff_u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t diff_u32x2 __attribute__((ext_vector_type(2)));

constexpr int kDiffBufferWord3 = 0x00020000;       // raw buffer access
constexpr int kDiffStream = 2;                     // non-temporal: pages are read once

// The values of the four 1-byte codes in w times their scale, each rounded once:
// int8 as (code + 128) * s - 128 s in one fused step, fp8 by the hardware's
// conversion (exact) and a product.  The pools' E4M3 and the hardware's differ
// in codes that the append never writes only (zero exponents are +-0, no 0xFF);
// they read as the hardware's here, as in the other matrix-core kernels.
template <int DT>
__device__ __forceinline__ diff_f32x4 code_values(uint32_t w, float s) {
    if constexpr (DT == AIR_KV_INT8) {
        const uint32_t u = w ^ 0x80808080u;
        const float off = -128.0f * s;
        return diff_f32x4{__builtin_fmaf((float)(u & 0xFFu), s, off), __builtin_fmaf((float)((u >> 8) & 0xFFu), s, off),
                          __builtin_fmaf((float)((u >> 16) & 0xFFu), s, off), __builtin_fmaf((float)(u >> 24), s, off)};
    } else {
        typedef float f32x2 __attribute__((ext_vector_type(2)));
        const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
        return diff_f32x4{lo[0] * s, lo[1] * s, hi[0] * s, hi[1] * s};
    }
}

// The upper (HI) or lower halves of two words, a's in the low half.
template <bool HI> __device__ __forceinline__ uint32_t halves(uint32_t a, uint32_t b) {
    return __builtin_amdgcn_perm(b, a, HI ? 0x07060302u : 0x05040100u);
}

// x, y = the sum of three bf16 pairs, each holding the next eight bits: exact,
// and every part has its value's sign.
__device__ __forceinline__ void split3(float x, float y, uint32_t &p0, uint32_t &p1, uint32_t &p2) {
    p0 = halves<true>(__float_as_uint(x), __float_as_uint(y));
    x -= __uint_as_float(__float_as_uint(x) & 0xFFFF0000u);
    y -= __uint_as_float(__float_as_uint(y) & 0xFFFF0000u);
    p1 = halves<true>(__float_as_uint(x), __float_as_uint(y));
    x -= __uint_as_float(__float_as_uint(x) & 0xFFFF0000u);
    y -= __uint_as_float(__float_as_uint(y) & 0xFFFF0000u);
    p2 = halves<true>(__float_as_uint(x), __float_as_uint(y));
}

// Four consecutive outputs (idx a multiple of 4).
__device__ __forceinline__ void diff_store4(const DiffOut &e, int64_t idx, diff_f32x4 v) {
    if (e.out_dtype == AIR_KV_F32) {
        *reinterpret_cast<diff_f32x4 *>((float *)e.out + idx) = v;
    } else {
        *reinterpret_cast<diff_u32x2 *>((uint16_t *)e.out + idx) =
            diff_u32x2{(uint32_t)bf16_rne(v[0]) | ((uint32_t)bf16_rne(v[1]) << 16),
                       (uint32_t)bf16_rne(v[2]) | ((uint32_t)bf16_rne(v[3]) << 16)};
    }
}
// Two (idx even).
__device__ __forceinline__ void diff_store2(const DiffOut &e, int64_t idx, float x, float y) {
    if (e.out_dtype == AIR_KV_F32) *reinterpret_cast<float2 *>((float *)e.out + idx) = make_float2(x, y);
    else *reinterpret_cast<uint32_t *>((uint16_t *)e.out + idx) = (uint32_t)bf16_rne(x) | ((uint32_t)bf16_rne(y) << 16);
}
__device__ __forceinline__ void diff_store(const DiffOut &e, int64_t idx, float v) {
    if (e.out_dtype == AIR_KV_F32) ((float *)e.out)[idx] = v;
    else ((uint16_t *)e.out)[idx] = bf16_rne(v);
}

// x's factor before the weight: out_scale, divided by the root mean square of
// the row's `cols` columns (sum of squares ss) under the norm.
__device__ __forceinline__ float diff_factor(const DiffOut &e, float ss, int cols) {
    return e.norm ? e.scale / sqrtf(ss / (float)cols + e.eps) : e.scale;
}

// Folding the pieces of a row that several waves computed: piece i's maximum
// (log2 units), sum and values, by log-sum-exp, two maps at a time.  A lane
// holds V columns of each.
template <int V> struct DiffFold {
    float m[2], l[2], o[2][V];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            m[k] = -INFINITY;
            l[k] = 0.0f;
#pragma unroll
            for (int i = 0; i < V; ++i) o[k][i] = 0.0f;
        }
    }
    __device__ __forceinline__ void fold(int k, float pm, float pl, const float (&po)[V]) {
        if (pm == -INFINITY && pl == 0.0f) return;       // past the last piece, or all of it masked
        const float top = fmaxf(m[k], pm);
        const float sa = __builtin_amdgcn_exp2f(m[k] - top), sb = __builtin_amdgcn_exp2f(pm - top);
        l[k] = l[k] * sa + pl * sb;
#pragma unroll
        for (int i = 0; i < V; ++i) o[k][i] = o[k][i] * sa + po[i] * sb;
        m[k] = top;
    }
};

template <int V> __device__ __forceinline__ void diff_load(const float *p, float (&x)[V]) {
    if constexpr (V == 4) {
        const diff_f32x4 w = *reinterpret_cast<const diff_f32x4 *>(p);
        x[0] = w[0]; x[1] = w[1]; x[2] = w[2]; x[3] = w[3];
    } else if constexpr (V == 2) {
        const float2 w = *reinterpret_cast<const float2 *>(p);
        x[0] = w.x; x[1] = w.y;
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = p[i];
    }
}

// The sum over a wave's lanes, in every lane.
__device__ __forceinline__ float diff_wave_sum(float x) {
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) x += __shfl_xor(x, o);
    return sum_x32(sum_x16(x));
}

// What the output row of (row, query pair h) needs beside its sums: lane l holds
// the weights of columns V l .. +V of 64 V.
template <int V> struct DiffTail {
    int64_t row;
    int h;
    float lam, w[V];
    __device__ __forceinline__ void load(const DiffOut &e, int64_t row_, int h_, int lane) {
        row = row_;
        h = h_;
        lam = e.lam[row * e.lam_stride + h];
#pragma unroll
        for (int i = 0; i < V; ++i) w[i] = 1.0f;
        if (e.norm && e.norm_w) diff_load<V>(e.norm_w + V * lane, w);
    }
};

template <int V>
__device__ __forceinline__ void diff_finish(const DiffOut &e, int pairs, const DiffFold<V> &c, const DiffTail<V> &tail, int lane) {
    // no key at all (every block of the sequence outside the pool): zeros
    const float i0 = c.l[0] == 0.0f ? 0.0f : 1.0f / c.l[0], i1 = c.l[1] == 0.0f ? 0.0f : tail.lam / c.l[1];
    float x[V], ss = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        x[i] = c.o[0][i] * i0 - c.o[1][i] * i1;
        ss += x[i] * x[i];
    }
    const float f = diff_factor(e, e.norm ? diff_wave_sum(ss) : 0.0f, 64 * V);
    const int64_t at = (tail.row * pairs + tail.h) * (64 * V) + V * lane;
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] *= f * tail.w[i];
    if constexpr (V == 4) {
        diff_store4(e, at, diff_f32x4{x[0], x[1], x[2], x[3]});
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) diff_store(e, at + i, x[i]);
    }
}

// ---- launches (shape checks are the entry points') ----

struct DiffDecodePlan {
    int32_t group, row_tiles;      // query pairs per K/V pair; 8 of them to a wave
    int32_t slices, batch_per_launch, slots;
    size_t ws_bytes;
};
DiffDecodePlan plan_diff_decode(const air_kv_pool &p, int32_t n_q_heads, int32_t batch, int32_t max_blocks,
                                int32_t max_splits);
hipError_t launch_diff_decode(const air_kv_pool &p, hipStream_t s, const DiffDecodePlan &plan, const void *q,
                              int32_t q_dtype, int32_t n_q_heads, const int32_t *tables, const int32_t *lens,
                              int32_t batch, int32_t max_blocks, float scale, int32_t max_splits, const DiffOut &out,
                              void *workspace);

}  // namespace airkv
