// extern "C" entry points of rotary positions (air_kv.h).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "host/span.hpp"
#include "host/status.hpp"
#include "on_device.hpp"
#include "pool.hpp"

using airkv::fail;
using airkv::OnDevice;
using airkv::Span;

namespace {

int hip_fail(hipError_t e, const char *what) {
    return fail(AIR_KV_E_HIP, "%s: %s", what, hipGetErrorString(e));
}

int check_rotary(const air_kv_pool *p, const float *inv_freq, int32_t rot_dim, int32_t layout) {
    if (!inv_freq) return fail(AIR_KV_E_INVALID_ARG, "inv_freq is NULL");
    if (rot_dim < 8 || rot_dim % 8 || rot_dim > p->desc.head_dim)
        return fail(AIR_KV_E_INVALID_ARG, "rot_dim %d is not a multiple of 8 up to head_dim %d", rot_dim, p->desc.head_dim);
    if (layout != AIR_ROTARY_HALF && layout != AIR_ROTARY_PAIRS)
        return fail(AIR_KV_E_INVALID_ARG, "unknown rotary layout %d", layout);
    return AIR_KV_OK;
}

}  // namespace

extern "C" {

int air_rotary_frequencies(int32_t rot_dim, double base, int32_t scaling, double factor, double trained_len, double low,
                           double high, float *inv_freq, float *magnitude) {
    if (!inv_freq || !magnitude) return fail(AIR_KV_E_INVALID_ARG, "inv_freq or magnitude is NULL");
    if (rot_dim < 2 || rot_dim % 2) return fail(AIR_KV_E_INVALID_ARG, "rot_dim %d is not even and positive", rot_dim);
    if (!(base > 1.0 && base < INFINITY)) return fail(AIR_KV_E_INVALID_ARG, "base must be finite and > 1");
    if (scaling < AIR_ROTARY_PLAIN || scaling > AIR_ROTARY_RAMP) return fail(AIR_KV_E_INVALID_ARG, "unknown scaling %d", scaling);
    if (scaling != AIR_ROTARY_PLAIN && !(factor >= 1.0 && factor < INFINITY))
        return fail(AIR_KV_E_INVALID_ARG, "factor must be finite and >= 1");
    const bool bands = scaling == AIR_ROTARY_BANDS || scaling == AIR_ROTARY_RAMP;
    if (bands && !(trained_len > 0.0 && trained_len < INFINITY && low > 0.0 && high > low && high < INFINITY))
        return fail(AIR_KV_E_INVALID_ARG, "trained_len must be > 0 and 0 < low < high");
    if (scaling == AIR_ROTARY_BASE) {
        if (rot_dim == 2) return fail(AIR_KV_E_INVALID_ARG, "another base changes nothing at rot_dim 2");
        base *= std::pow(factor, rot_dim / (rot_dim - 2.0));
        if (!(base < INFINITY)) return fail(AIR_KV_E_INVALID_ARG, "the base times a power of factor %g is not finite", factor);
    }
    const double two_pi = 6.283185307179586;
    auto turns = [&](double n) { return rot_dim * std::log(trained_len / (two_pi * n)) / (2.0 * std::log(base)); };
    double a = 0.0, b = 0.0;
    if (scaling == AIR_ROTARY_RAMP) {
        a = std::max(0.0, std::floor(turns(high)));
        b = std::min(rot_dim - 1.0, std::ceil(turns(low)));
        if (b <= a) b = a + 0.001;
    }
    for (int32_t i = 0; i < rot_dim / 2; ++i) {
        double f = std::pow(base, -2.0 * i / rot_dim);
        if (scaling == AIR_ROTARY_LINEAR) {
            f /= factor;
        } else if (scaling == AIR_ROTARY_BANDS) {
            const double over = trained_len * f / two_pi;              // L / w
            const double t = std::min(1.0, std::max(0.0, (over - low) / (high - low)));
            f = (1.0 - t) * f / factor + t * f;
        } else if (scaling == AIR_ROTARY_RAMP) {
            const double t = std::min(1.0, std::max(0.0, (i - a) / (b - a)));
            f = (1.0 - t) * f + t * f / factor;
        }
        inv_freq[i] = (float)f;
    }
    *magnitude = scaling == AIR_ROTARY_RAMP ? (float)(0.1 * std::log(factor) + 1.0) : 1.0f;
    return AIR_KV_OK;
}

int air_kv_append_rotary(air_kv_pool *p, void *stream, const void *q, int64_t q_stride, int32_t n_q_heads, const void *k,
                         int64_t k_stride, const void *v, int64_t v_stride, int32_t in_dtype, const int64_t *slot_mapping,
                         const int32_t *positions, int32_t n_tokens, const float *inv_freq, int32_t rot_dim, int32_t layout,
                         float magnitude, void *q_out, int32_t q_out_dtype) {
    if (!p) return fail(AIR_KV_E_INVALID_ARG, "pool is NULL");
    if (n_tokens < 0) return fail(AIR_KV_E_INVALID_ARG, "n_tokens < 0");
    if (n_q_heads < 0 || n_q_heads > 65535) return fail(AIR_KV_E_INVALID_ARG, "n_q_heads %d out of range", n_q_heads);
    if (in_dtype != AIR_KV_F32 && in_dtype != AIR_KV_BF16) return fail(AIR_KV_E_INVALID_ARG, "in_dtype must be F32 or BF16");
    if (q_out_dtype != AIR_KV_F32 && q_out_dtype != AIR_KV_BF16) return fail(AIR_KV_E_INVALID_ARG, "q_out_dtype must be F32 or BF16");
    if (!std::isfinite(magnitude)) return fail(AIR_KV_E_INVALID_ARG, "magnitude must be finite");
    if (n_tokens == 0) return AIR_KV_OK;
    if (int rc = check_rotary(p, inv_freq, rot_dim, layout)) return rc;
    if (!k || !v || !slot_mapping || !positions || (n_q_heads && (!q || !q_out)))
        return fail(AIR_KV_E_INVALID_ARG, "NULL q, k, v, slot_mapping, positions or q_out");
    const int64_t d = p->desc.head_dim, kv = p->desc.n_kv_heads * d, width = n_q_heads * d;
    const int64_t in = in_dtype == AIR_KV_BF16 ? 2 : 4, out = q_out_dtype == AIR_KV_BF16 ? 2 : 4;
    constexpr int64_t kMost = (int64_t)1 << 31;
    if ((n_q_heads && (q_stride < width || q_stride > kMost)) || k_stride < kv || v_stride < kv || k_stride > kMost || v_stride > kMost)
        return fail(AIR_KV_E_INVALID_ARG, "a row stride is smaller than its row, or beyond 2^31");
    if ((uintptr_t)k % 16 || (uintptr_t)v % 16 || k_stride * in % 16 || v_stride * in % 16 ||
        (n_q_heads && ((uintptr_t)q % 16 || q_stride * in % 16 || (uintptr_t)q_out % 16)))
        return fail(AIR_KV_E_INVALID_ARG, "q, k, v, q_out and the row strides must be multiples of 16 bytes");
    if (n_q_heads) {
        const Span o(q_out, n_tokens, width, width, out);
        const bool same = q_out == q && q_stride == width && in_dtype == q_out_dtype;
        if ((!same && o.meets(Span(q, n_tokens, q_stride, width, in))) || o.meets(Span(k, n_tokens, k_stride, kv, in)) ||
            o.meets(Span(v, n_tokens, v_stride, kv, in)))
            return fail(AIR_KV_E_INVALID_ARG, "q_out overlaps an input (it may be q itself where q is dense and of its type)");
    }
    const OnDevice on(p->device);
    if (on.status() != hipSuccess) return hip_fail(on.status(), "hipSetDevice");
    const hipError_t e = airkv::launch_append_rotary(*p, (hipStream_t)stream, q, q_stride, n_q_heads, k, k_stride, v, v_stride,
                                                     in_dtype, slot_mapping, positions, n_tokens, inv_freq, rot_dim, layout,
                                                     magnitude, q_out, q_out_dtype);
    return e == hipSuccess ? AIR_KV_OK : hip_fail(e, "air_kv_append_rotary launch");
}

int air_kv_rotate(air_kv_pool *p, void *stream, const int32_t *block_tables, int32_t batch, int32_t max_blocks,
                  const int32_t *from, const int32_t *to, const int32_t *cu, int32_t total, const float *inv_freq,
                  int32_t rot_dim, int32_t layout) {
    if (!p) return fail(AIR_KV_E_INVALID_ARG, "pool is NULL");
    if (batch < 0 || max_blocks <= 0 || total < 0) return fail(AIR_KV_E_INVALID_ARG, "bad batch, max_blocks or total");
    if (batch == 0 || total == 0) return AIR_KV_OK;
    if (int rc = check_rotary(p, inv_freq, rot_dim, layout)) return rc;
    if (batch > 1 << 20) return fail(AIR_KV_E_INVALID_ARG, "batch %d out of range", batch);
    if (!block_tables || !from || !cu) return fail(AIR_KV_E_INVALID_ARG, "NULL rotation buffer");
    const OnDevice on(p->device);
    if (on.status() != hipSuccess) return hip_fail(on.status(), "hipSetDevice");
    const hipError_t e = airkv::launch_rotate(*p, (hipStream_t)stream, block_tables, batch, max_blocks, from, to, cu, total,
                                              inv_freq, rot_dim, layout);
    return e == hipSuccess ? AIR_KV_OK : hip_fail(e, "air_kv_rotate launch");
}

}  // extern "C"
