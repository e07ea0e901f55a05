"""The 16-bit products of differential prefill where the operands' sizes are far from 1
or far from each other, against 64 bits."""
import numpy as np
import pytest

import airkv
from diff_ref import attend, check, pool_values, sequence
from gpu_helpers import log, torch_mod
from test_gpu_diff_attention import Cache, _p_step, _refill

pytestmark = pytest.mark.gpu


def _prefill(c, qlens, q, lam, p_step, floor=0.0, tables=None, **more):
    """bf16 rows through the kernels, held to 64 bits; (output, share of the bound used)."""
    torch = torch_mod()
    cu = np.concatenate([[0], np.cumsum(qlens)]).astype(np.int32)
    total, pairs, d = int(cu[-1]), q.shape[1] // 2, c.d
    tables = c.tables if tables is None else tables
    q64 = q.float().cpu().numpy().astype(np.float64)
    lam64 = np.broadcast_to(lam.cpu().numpy().astype(np.float64), (total, pairs))
    kv, vv = pool_values(c.pool)
    want, bound = np.zeros((total, pairs, 2 * d)), np.zeros((total, pairs, 2 * d))
    scale = float(np.float32(1.0) / np.sqrt(np.float32(d)))
    for i, (m, ql) in enumerate(zip(c.lens, qlens)):
        k, v = (sequence(x, tables[i], int(m), c.bs) for x in (kv, vv))
        s = slice(cu[i], cu[i + 1])
        want[s], bound[s] = attend(q64[s], k, v, lam64[s], scale, m - ql + np.arange(ql), p_step=p_step, **more)
        bound[s] += floor * (1 + np.abs(lam64[s]).max(initial=0)) * np.abs(v).max(initial=0)
    out = torch.full((total, pairs, 2 * d), float("nan"), device="cuda", dtype=torch.bfloat16)
    c.pool.paged_diff_prefill(q, lam, torch.from_numpy(cu).cuda(), torch.from_numpy(tables).cuda(), torch.from_numpy(c.lens).cuda(), out,
                              max_q_len=max(qlens), **more)
    got = out.float().cpu().numpy()
    return got, check(got, want, bound, airkv.BF16, "prefill", p_step)


@pytest.mark.parametrize("dtype,q_mul,k_mul", [(airkv.INT8, 2.0 ** -40, 2.0 ** -100), (airkv.INT8, 2.0 ** -120, 2.0 ** -20),
                                               (airkv.FP8, 2.0 ** -118, 2.0 ** -24), (airkv.BF16, 2.0 ** -100, 2.0 ** -100)])
def test_scores_below_the_smallest_float(dtype, q_mul, k_mul):
    """Queries and keys so small that every score is 0: each row attends to what it sees
    alike, and to nothing that is hidden."""
    torch = torch_mod()
    c = Cache(dtype, 64, 2, 16, [100, 33, 7], seed=50)
    _refill(c, lambda t: k_mul, lambda t: 1.0)
    q, lam, _, _, _, _ = c.rows(60, 2, False, False, False)
    q = (q.float() * q_mul).to(torch.bfloat16)
    _, used = _prefill(c, [50, 3, 7], q, lam, _p_step(c))
    log(f"scores below the smallest float dtype={dtype}: {used:.3f} of the bound")


@pytest.mark.parametrize("dtype", [airkv.INT8, airkv.FP8])
def test_a_factor_past_the_largest_float(dtype):
    """Large queries and keys that share no element: every score is 0."""
    torch = torch_mod()
    c = Cache(dtype, 64, 2, 16, [100, 33, 7], seed=51)
    c.k[:, :, 1:] = 0
    _refill(c, lambda t: 2.0 ** 40, lambda t: 1.0)
    q, lam, _, _, _, _ = c.rows(60, 2, False, False, False)
    q = (q.float() * 2.0 ** 118).to(torch.bfloat16)
    q[:, :, 0] = 0
    _, used = _prefill(c, [50, 3, 7], q, lam, _p_step(c))
    log(f"a factor past the largest float dtype={dtype}: {used:.3f} of the bound")


@pytest.mark.parametrize("dtype,v_mul,k_mul", [(airkv.BF16, 2.0 ** -122, 1.0), (airkv.INT8, 2.0 ** -118, 1.0),
                                               (airkv.INT8, 1.0, 2.0 ** -118)])
def test_values_and_keys_near_the_smallest_normal_float(dtype, v_mul, k_mul):
    """Nothing is lost of values, keys or queries that the largest power of two brings into
    f16's range."""
    torch = torch_mod()
    c = Cache(dtype, 64, 2, 16, [100, 33, 7], seed=55)
    _refill(c, lambda t: k_mul, lambda t: v_mul)
    q, lam, _, _, _, _ = c.rows(60, 2, False, False, False)
    q = (q.float() / k_mul).to(torch.bfloat16)
    # outputs of this size are scaled up before they are rounded
    _, used = _prefill(c, [50, 3, 7], q, lam, _p_step(c), out_scale=1 / v_mul)
    log(f"near the smallest normal float dtype={dtype} v_mul={v_mul:.2g} k_mul={k_mul:.2g}: {used:.3f} of the bound")


def test_small_queries_and_large_keys():
    torch = torch_mod()
    c = Cache(airkv.INT8, 64, 2, 16, [100, 33, 7], seed=56)
    _refill(c, lambda t: 2.0 ** 118, lambda t: 1.0)
    q, lam, _, _, _, _ = c.rows(60, 2, False, False, False)
    q = (q.float() * 2.0 ** -118).to(torch.bfloat16)
    _, used = _prefill(c, [50, 3, 7], q, lam, _p_step(c))
    log(f"small queries, large keys: {used:.3f} of the bound")
