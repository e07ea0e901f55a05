// extern "C" entry points of cross attention (air_kv.h).
#include <hip/hip_runtime.h>

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

int check_shape(const air_kv_pool *p, int32_t n_q_heads, int32_t batch, int32_t max_q_len) {
    if (!p) return fail(AIR_KV_E_INVALID_ARG, "pool is NULL");
    if (n_q_heads <= 0 || n_q_heads % p->desc.n_kv_heads)
        return fail(AIR_KV_E_INVALID_ARG, "n_q_heads %d is not a multiple of n_kv_heads %d", n_q_heads, p->desc.n_kv_heads);
    if (batch < 0 || max_q_len < 0) return fail(AIR_KV_E_INVALID_ARG, "negative batch or max_q_len");
    return AIR_KV_OK;
}

}  // namespace

extern "C" {

int air_paged_cross_workspace_size(const air_kv_pool *p, int32_t n_q_heads, int32_t batch, int32_t max_q_len, size_t *bytes) {
    if (int rc = check_shape(p, n_q_heads, batch, max_q_len)) return rc;
    if (!bytes) return fail(AIR_KV_E_INVALID_ARG, "bytes is NULL");
    *bytes = airkv::cross_workspace(*p);
    return AIR_KV_OK;
}

int air_paged_cross(air_kv_pool *p, void *stream, const void *q, int32_t q_dtype, int32_t n_q_heads, const int32_t *cu_q,
                    int32_t total_q, int32_t max_q_len, const int32_t *block_tables, const int32_t *seq_lens, int32_t batch,
                    int32_t max_blocks, float scale, void *workspace, size_t ws_bytes, void *out, int32_t out_dtype) {
    if (int rc = check_shape(p, n_q_heads, batch, max_q_len)) return rc;
    if (total_q < 0 || max_blocks < 0) return fail(AIR_KV_E_INVALID_ARG, "negative total_q or max_blocks");
    if (batch == 0 || total_q == 0) return AIR_KV_OK;
    if (!q || !cu_q || !block_tables || !seq_lens || !workspace || !out)
        return fail(AIR_KV_E_INVALID_ARG, "NULL q, cu_q, block_tables, seq_lens, workspace or out");
    if ((uintptr_t)q % 16 || (uintptr_t)out % 16 || (uintptr_t)workspace % 16)
        return fail(AIR_KV_E_INVALID_ARG, "q, out and workspace must be 16-byte aligned");
    if (q_dtype != AIR_KV_F32 && q_dtype != AIR_KV_BF16) return fail(AIR_KV_E_INVALID_ARG, "q_dtype must be F32 or BF16");
    if (out_dtype != AIR_KV_F32 && out_dtype != AIR_KV_BF16) return fail(AIR_KV_E_INVALID_ARG, "out_dtype must be F32 or BF16");
    if (!(scale > 0.0f && scale < INFINITY)) return fail(AIR_KV_E_INVALID_ARG, "scale must be finite and > 0");
    if ((int64_t)total_q * (n_q_heads / p->desc.n_kv_heads) > INT32_MAX - 65536)
        return fail(AIR_KV_E_INVALID_ARG, "total_q times the query heads of a K/V head exceeds int32");
    if ((int64_t)max_blocks * p->desc.block_size > INT32_MAX)
        return fail(AIR_KV_E_INVALID_ARG, "max_blocks * block_size exceeds int32");
    const int64_t width = (int64_t)n_q_heads * p->desc.head_dim, in = q_dtype == AIR_KV_BF16 ? 2 : 4, res = out_dtype == AIR_KV_BF16 ? 2 : 4;
    if (!(out == q && q_dtype == out_dtype) && Span(out, total_q, width, width, res).meets(Span(q, total_q, width, width, in)))
        return fail(AIR_KV_E_INVALID_ARG, "out overlaps q (it may be q itself where both have one type)");
    const size_t needed = airkv::cross_workspace(*p);
    if (ws_bytes < needed) return fail(AIR_KV_E_INVALID_ARG, "workspace %zu bytes < %zu needed", ws_bytes, needed);
    const OnDevice on(p->device);
    if (on.status() != hipSuccess) return hip_fail(on.status(), "hipSetDevice");
    const hipError_t e = airkv::launch_cross(*p, (hipStream_t)stream, q, q_dtype, n_q_heads, cu_q, total_q, max_q_len, block_tables,
                                             seq_lens, batch, max_blocks, scale, workspace, out, out_dtype);
    return e == hipSuccess ? AIR_KV_OK : hip_fail(e, "air_paged_cross launch");
}

}  // extern "C"
