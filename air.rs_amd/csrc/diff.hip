// extern "C" entry points of differential attention and compaction (air_kv.h).
#include <hip/hip_runtime.h>

#include <cmath>

#include "host/status.hpp"
#include "kernels/diff_common.hpp"
#include "kernels/diff_prefill.hpp"
#include "pool.hpp"

using airkv::fail;

namespace {

int hip_fail(hipError_t e, const char *what) {
    return fail(AIR_KV_E_HIP, "%s: %s", what, hipGetErrorString(e));
}

// The pool's device is the current one while this lives.
class OnDevice {
public:
    explicit OnDevice(int device) {
        status_ = hipGetDevice(&before_);
        if (status_ == hipSuccess && before_ != device) {
            status_ = hipSetDevice(device);
            changed_ = status_ == hipSuccess;
        }
    }
    ~OnDevice() {
        if (changed_) (void)hipSetDevice(before_);
    }
    hipError_t status() const { return status_; }

private:
    int before_ = 0;
    bool changed_ = false;
    hipError_t status_;
};

// The pool and the heads of a differential call.
int check_shape(const air_kv_pool *p, int32_t n_q_heads) {
    if (!p) return fail(AIR_KV_E_INVALID_ARG, "pool is NULL");
    const air_kv_pool_desc &d = p->desc;
    if (d.n_kv_heads % 2) return fail(AIR_KV_E_INVALID_ARG, "differential attention pairs K/V heads: n_kv_heads %d is odd", d.n_kv_heads);
    if (d.head_dim > 128) return fail(AIR_KV_E_INVALID_ARG, "differential attention supports head_dim up to 128 (pool has %d)", d.head_dim);
    if (n_q_heads <= 0 || n_q_heads % d.n_kv_heads)
        return fail(AIR_KV_E_INVALID_ARG, "n_q_heads %d is not a multiple of n_kv_heads %d", n_q_heads, d.n_kv_heads);
    if (n_q_heads / 2 > 65535) return fail(AIR_KV_E_INVALID_ARG, "n_q_heads %d out of range", n_q_heads);
    return AIR_KV_OK;
}

int check_io(const void *q, int32_t q_dtype, const void *lambda, const void *out, int32_t out_dtype, const float *norm_weight,
             float norm_eps, float out_scale, const void *workspace, size_t ws_bytes, size_t needed) {
    if (!q || !lambda || !out || !workspace) return fail(AIR_KV_E_INVALID_ARG, "NULL q, lambda, out or workspace");
    if ((uintptr_t)q % 16 || (uintptr_t)out % 16 || (uintptr_t)workspace % 16)
        return fail(AIR_KV_E_INVALID_ARG, "q, out and workspace must be 16-byte aligned");
    if (q_dtype != AIR_KV_F32 && q_dtype != AIR_KV_BF16) return fail(AIR_KV_E_INVALID_ARG, "q_dtype must be F32 or BF16");
    if (out_dtype != AIR_KV_F32 && out_dtype != AIR_KV_BF16)
        return fail(AIR_KV_E_INVALID_ARG, "out_dtype must be F32 or BF16");
    if (!(norm_eps >= 0.0f && norm_eps < INFINITY)) return fail(AIR_KV_E_INVALID_ARG, "norm_eps must be 0 (no norm) or finite and > 0");
    if (norm_eps == 0.0f && norm_weight) return fail(AIR_KV_E_INVALID_ARG, "norm_weight without norm_eps");
    if (!(out_scale == out_scale)) return fail(AIR_KV_E_INVALID_ARG, "out_scale is NaN");
    if (ws_bytes < needed) return fail(AIR_KV_E_INVALID_ARG, "workspace %zu bytes < %zu needed", ws_bytes, needed);
    return AIR_KV_OK;
}

airkv::DiffOut diff_out(int32_t pairs, const float *lambda, int32_t per_row, const float *norm_weight, float norm_eps,
                        float out_scale, void *out, int32_t out_dtype) {
    airkv::DiffOut e;
    e.lam = lambda;
    e.lam_stride = per_row ? pairs : 0;
    e.norm_w = norm_weight;
    e.eps = norm_eps;
    e.norm = norm_eps > 0.0f;
    e.scale = out_scale;
    e.out = out;
    e.out_dtype = out_dtype;
    return e;
}

int check_decode(const air_kv_pool *p, int32_t n_q_heads, int32_t batch, int32_t max_blocks, int32_t max_splits) {
    if (int rc = check_shape(p, n_q_heads)) return rc;
    if (batch < 0 || batch > 65535) return fail(AIR_KV_E_INVALID_ARG, "batch %d out of range", batch);
    if (max_blocks <= 0) return fail(AIR_KV_E_INVALID_ARG, "max_blocks must be positive");
    if (max_splits < 1 || max_splits > 256) return fail(AIR_KV_E_INVALID_ARG, "max_splits %d outside 1..256", max_splits);
    return AIR_KV_OK;
}

int check_prefill(const air_kv_pool *p, int32_t n_q_heads, int32_t batch, int32_t max_q_len) {
    if (int rc = check_shape(p, n_q_heads)) return rc;
    if (batch < 0 || max_q_len < 0) return fail(AIR_KV_E_INVALID_ARG, "negative batch or max_q_len");
    return AIR_KV_OK;
}

}  // namespace

extern "C" {

int air_paged_diff_decode_workspace_size(const air_kv_pool *p, int32_t n_q_heads, int32_t batch, int32_t max_blocks,
                                         int32_t max_splits, size_t *bytes) {
    if (int rc = check_decode(p, n_q_heads, batch, max_blocks, max_splits)) return rc;
    if (!bytes) return fail(AIR_KV_E_INVALID_ARG, "bytes is NULL");
    *bytes = airkv::plan_diff_decode(*p, n_q_heads, batch, max_blocks, max_splits).ws_bytes;
    return AIR_KV_OK;
}

int air_paged_diff_decode(air_kv_pool *p, void *stream, const void *q, int32_t q_dtype, int32_t n_q_heads,
                          const float *lambda, int32_t lambda_per_row, const int32_t *block_tables,
                          const int32_t *seq_lens, int32_t batch, int32_t max_blocks, float scale, int32_t max_splits,
                          const float *norm_weight, float norm_eps, float out_scale, void *workspace, size_t ws_bytes,
                          void *out, int32_t out_dtype) {
    if (int rc = check_decode(p, n_q_heads, batch, max_blocks, max_splits)) return rc;
    if (batch == 0) return AIR_KV_OK;
    const airkv::DiffDecodePlan plan = airkv::plan_diff_decode(*p, n_q_heads, batch, max_blocks, max_splits);
    if (int rc = check_io(q, q_dtype, lambda, out, out_dtype, norm_weight, norm_eps, out_scale, workspace, ws_bytes, plan.ws_bytes))
        return rc;
    if (!block_tables || !seq_lens) return fail(AIR_KV_E_INVALID_ARG, "NULL decode buffer");
    if (!(scale == scale)) return fail(AIR_KV_E_INVALID_ARG, "scale is NaN");
    const OnDevice on(p->device);
    if (on.status() != hipSuccess) return hip_fail(on.status(), "hipSetDevice");
    const hipError_t e = airkv::launch_diff_decode(
        *p, (hipStream_t)stream, plan, q, q_dtype, n_q_heads, block_tables, seq_lens, batch, max_blocks, scale, max_splits,
        diff_out(n_q_heads / 2, lambda, lambda_per_row, norm_weight, norm_eps, out_scale, out, out_dtype), workspace);
    return e == hipSuccess ? AIR_KV_OK : hip_fail(e, "air_paged_diff_decode launch");
}

int air_paged_diff_prefill_workspace_size(const air_kv_pool *p, int32_t n_q_heads, int32_t batch, int32_t max_q_len,
                                          size_t *bytes) {
    if (int rc = check_prefill(p, n_q_heads, batch, max_q_len)) return rc;
    if (!bytes) return fail(AIR_KV_E_INVALID_ARG, "bytes is NULL");
    *bytes = airkv::diff_prefill_workspace(*p);
    return AIR_KV_OK;
}

int air_paged_diff_prefill(air_kv_pool *p, void *stream, const void *q, int32_t q_dtype, int32_t n_q_heads,
                           const float *lambda, int32_t lambda_per_row, const int32_t *cu_q, int32_t total_q,
                           int32_t max_q_len, const int32_t *block_tables, const int32_t *seq_lens, int32_t batch,
                           int32_t max_blocks, float scale, const float *norm_weight, float norm_eps, float out_scale,
                           void *workspace, size_t ws_bytes, void *out, int32_t out_dtype) {
    if (int rc = check_prefill(p, n_q_heads, batch, max_q_len)) return rc;
    if (total_q < 0 || max_blocks < 0) return fail(AIR_KV_E_INVALID_ARG, "negative total_q or max_blocks");
    if (batch == 0 || total_q == 0) return AIR_KV_OK;
    if (int rc = check_io(q, q_dtype, lambda, out, out_dtype, norm_weight, norm_eps, out_scale, workspace, ws_bytes,
                          airkv::diff_prefill_workspace(*p)))
        return rc;
    if (!cu_q || !block_tables || !seq_lens) return fail(AIR_KV_E_INVALID_ARG, "NULL prefill buffer");
    if (!(scale > 0.0f && scale < INFINITY)) return fail(AIR_KV_E_INVALID_ARG, "prefill scale must be finite and > 0");
    if ((int64_t)max_blocks * p->desc.block_size > INT32_MAX)
        return fail(AIR_KV_E_INVALID_ARG, "max_blocks * block_size exceeds int32");
    const OnDevice on(p->device);
    if (on.status() != hipSuccess) return hip_fail(on.status(), "hipSetDevice");
    const hipError_t e = airkv::launch_diff_prefill(
        *p, (hipStream_t)stream, q, q_dtype, n_q_heads, cu_q, total_q, block_tables, seq_lens, batch, max_blocks, scale,
        diff_out(n_q_heads / 2, lambda, lambda_per_row, norm_weight, norm_eps, out_scale, out, out_dtype), workspace);
    return e == hipSuccess ? AIR_KV_OK : hip_fail(e, "air_paged_diff_prefill launch");
}

int air_kv_compact(air_kv_pool *p, void *stream, const int32_t *block_tables, const int32_t *seq_lens, int32_t batch,
                   int32_t max_blocks, const int32_t *keep, const int32_t *cu_keep, int32_t total_keep) {
    if (!p) return fail(AIR_KV_E_INVALID_ARG, "pool is NULL");
    if (batch < 0 || max_blocks <= 0 || total_keep < 0)
        return fail(AIR_KV_E_INVALID_ARG, "bad batch, max_blocks or total_keep");
    if (batch == 0 || total_keep == 0) return AIR_KV_OK;
    if (!block_tables || !seq_lens || !keep || !cu_keep) return fail(AIR_KV_E_INVALID_ARG, "NULL compaction buffer");
    const OnDevice on(p->device);
    if (on.status() != hipSuccess) return hip_fail(on.status(), "hipSetDevice");
    const hipError_t e = airkv::launch_compact(*p, (hipStream_t)stream, block_tables, seq_lens, batch, max_blocks, keep,
                                               cu_keep, total_keep);
    return e == hipSuccess ? AIR_KV_OK : hip_fail(e, "air_kv_compact launch");
}

}  // extern "C"
