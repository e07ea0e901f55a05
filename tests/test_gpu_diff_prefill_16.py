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


def _two(dtype, v_mul, k_mul=lambda t: 1.0, q_mul=1.0, out=False, seed=52):
    """A short sequence and a long one behind it, which share a workgroup (128 pairs, two
    workgroups a pair: the first has the short one and the long one's first nine tiles).
    v_mul, k_mul: factors of the long one's tokens; the short one's values are 1e20 times
    those of normal rows.  out: the long one's first 64 tokens lie outside the pool."""
    torch = torch_mod()
    c = Cache(dtype, 32, 256, 16, [20, 1000], seed=seed)
    t = np.arange(1000)
    f = np.concatenate([np.full(20, 1e20), v_mul(t) * np.ones(1000)]).astype(np.float32)[:, None, None]
    g = np.concatenate([np.ones(20), k_mul(t) * np.ones(1000)]).astype(np.float32)[:, None, None]
    slots = np.concatenate([c.tables[i, np.arange(n) // 16].astype(np.int64) * 16 + np.arange(n) % 16 for i, n in enumerate(c.lens)])
    c.pool.append(torch.from_numpy(c.k * g).cuda(), torch.from_numpy(c.v * f).cuda(), torch.from_numpy(slots).cuda())
    tables = c.tables.copy()
    if out:
        tables[1, :4] = -1
    q, lam, _, _, _, _ = c.rows(5, 1, False, False, False)
    q[1:] = (q[1:].float() * q_mul).to(torch.bfloat16)
    return _prefill(c, [1, 4], q, lam, _p_step(c), tables=tables)[1]


@pytest.mark.parametrize("dtype", [airkv.BF16, airkv.INT8, airkv.FP8])
def test_a_sequence_that_begins_with_zeros_behind_a_large_one(dtype):
    """What a sequence's values are rounded to does not come from the one before it: zeros
    (or, on 1-byte pages, tokens outside the pool, which are zeros with a scale of 0) say
    nothing about the power of two."""
    used = _two(dtype, lambda t: np.where(t < 64, 0.0, 1.0))
    more = _two(dtype, lambda t: 1.0, out=True)
    log(f"zeros first dtype={dtype}: {used:.3f}, outside the pool {more:.3f} of the bound")


@pytest.mark.parametrize("dtype,size", [(airkv.BF16, 1e-30), (airkv.INT8, 1e-30), (airkv.FP8, 1e-7)])
def test_zeros_first_then_small_values(dtype, size):
    used = _two(dtype, lambda t: np.where(t < 64, 0.0, size), seed=53)
    log(f"zeros, then {size} dtype={dtype}: {used:.3f} of the bound")


@pytest.mark.parametrize("dtype,size", [(airkv.INT8, 1e-30), (airkv.FP8, 1e-7)])
def test_zero_keys_first_then_small_ones(dtype, size):
    """Queries as large as the keys are small: scores of normal rows."""
    used = _two(dtype, lambda t: 1.0, lambda t: np.where(t < 64, 0.0, size), 1 / size, seed=54)
    log(f"zero keys, then {size} dtype={dtype}: {used:.3f} of the bound")


@pytest.mark.parametrize("dtype", [airkv.INT8, airkv.FP8])
def test_zeros_among_small_values(dtype):
    """Groups of zeros (their scale is 1) between values that are all small."""
    size = 1e-34 if dtype == airkv.INT8 else 1e-7
    used = _two(dtype, lambda t: np.where(t % 3 == 1, 0.0, size), seed=57)
    log(f"zeros among {size} dtype={dtype}: {used:.3f} of the bound")


@pytest.mark.parametrize("dtype", [airkv.BF16, airkv.INT8, airkv.FP8])
@pytest.mark.parametrize("bits,n", [(12.0, 5000), (20.0, 131072), (22.7, 131072), (25.5, 131072)])
def test_many_small_probabilities(dtype, bits, n):
    """One key that takes nearly all of a row's attention and whose values are 0, and many
    behind it, each 2^-bits as probable: the result is what those sum to.  A probability
    is off by 2^-11 of itself or, below f16's normal numbers, 2^-36 of the largest.  256
    sequences over the same blocks: a workgroup each, which walks all of its keys."""
    torch = torch_mod()
    c = Cache(dtype, 32, 2, 16, [n], seed=58)
    c.k[:] = 0
    c.k[0] = bits * np.log(2.0) / np.sqrt(32.0)         # against queries of ones
    c.v[:] = 1 + 0.1 * c.v
    c.v[0] = 0
    _refill(c, lambda t: 1.0, lambda t: 1.0)
    k, v = (sequence(x, c.tables[0], n, 16) for x in pool_values(c.pool))
    # values (of 1-byte pages) and pieces round to 11 bits; the scores of 1-byte keys err by
    # 2^-11 of themselves, `bits` at most, and move a probability by twice that
    p_step = 2.0 ** -11 * (2 if dtype == airkv.BF16 else 3 + 2 * bits)
    want, bound = attend(np.ones((1, 2, 32)), k, v, np.full((1, 1), 0.25), 32 ** -0.5, [n - 1], p_step=p_step)
    bound += 2.0 ** -36 * n * 1.25 * np.abs(v).max()
    many = 256
    q = torch.ones(many, 2, 32, device="cuda", dtype=torch.bfloat16)
    tables, lens = (torch.from_numpy(np.repeat(x, many, 0)).cuda() for x in (c.tables, c.lens))
    out = torch.full((many, 1, 64), float("nan"), device="cuda", dtype=torch.bfloat16)
    c.pool.paged_diff_prefill(q, torch.full((1,), 0.25, device="cuda"), torch.arange(many + 1, dtype=torch.int32, device="cuda"),
                              tables, lens, out, max_q_len=1)
    used = check(out.float().cpu().numpy(), np.repeat(want, many, 0), np.repeat(bound, many, 0), airkv.BF16, "small", p_step)
    log(f"small probabilities dtype={dtype} 2^-{bits}: {used:.3f} of the bound")


@pytest.mark.parametrize("d", [32, 64, 96, 128])
def test_two_maps_that_nearly_cancel(d):
    """Two maps whose means differ by 2^-12 of themselves, over a block that several
    workgroups share.  Map 0 sees every key alike, map 1 every second one; values are
    1 + j 2^-7 and lambda 1: probabilities are 0 or 1, every sum of them and of their
    products is a number of 24 bits, and what is left to round is the two quotients and
    their difference, 8 half steps of 2^-24 of values below 2 together, and the output."""
    torch = torch_mod()
    n, new, scale = 2000, 8, float(np.float32(1.0) / np.sqrt(np.float32(d)))
    c = Cache(airkv.BF16, d, 4, 16, [n], seed=59)
    c.k[:] = 0
    c.k[1::2, 1::2] = -1000.0                           # map 1's keys at odd tokens
    c.v[:] = 1 + c.r.integers(0, 4, c.v.shape) * 2.0 ** -7
    _refill(c, lambda t: 1.0, lambda t: 1.0)
    q = torch.zeros(new, 8, d, device="cuda", dtype=torch.bfloat16)
    q[:, 1::2] = 1.0
    assert 1000.0 * d * scale > 200                     # 2^-200 and less: 0 beside 1
    out = torch.full((new, 4, 2 * d), float("nan"), device="cuda", dtype=torch.bfloat16)
    tables, lens = c.device()
    c.pool.paged_diff_prefill(q, torch.ones(4, device="cuda"), torch.tensor([0, new], dtype=torch.int32, device="cuda"), tables, lens,
                              out, max_q_len=new)
    got = out.float().cpu().numpy()
    v = c.v.astype(np.float64)                          # exact in bf16
    for r in range(new):
        m = n - new + r + 1
        for h in range(4):
            x = np.concatenate([v[:m, 2 * (h // 2)], v[:m, 2 * (h // 2) + 1]], -1)
            want = x.mean(0) - x[::2].mean(0)
            bad = np.abs(got[r, h] - want) > 8 * 2.0 ** -24 * 2 + 2.0 ** -8 * np.abs(want)
            assert not bad.any(), (r, h, int(bad.sum()), got[r, h][bad][:4], want[bad][:4])


@pytest.mark.parametrize("d,group,scale_group", [(128, 4, 32), (64, 1, 32), (96, 3, 32), (32, 8, 8)])
@pytest.mark.parametrize("dtype", [airkv.BF16, airkv.INT8, airkv.FP8])
def test_the_error_of_normal_rows(dtype, d, group, scale_group):
    """The whole result's error: roundings of random sign add up by squares.  The output's
    is 2^-9 of a value at most; probability, value and key (of 1-byte pages) err by 2^-12
    of themselves at most, independently from key to key, as the result's own terms are."""
    torch = torch_mod()
    n, new = [1500, 700, 40], [300, 700, 40]
    c = Cache(dtype, d, 4, 16, n, seed=60, scale_group=scale_group)
    q, lam, _, q64, lam64, _ = c.rows(sum(new), group, False, True, False)
    cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    tables, lens = c.device()
    out = torch.empty(sum(new), lam64.shape[1], 2 * d, device="cuda", dtype=torch.bfloat16)
    c.pool.paged_diff_prefill(q, lam, torch.from_numpy(cu).cuda(), tables, lens, out, max_q_len=max(new))
    got = out.float().cpu().numpy()
    kv, vv = pool_values(c.pool)
    scale = float(np.float32(1.0) / np.sqrt(np.float32(d)))
    limit = ((2.0 ** -9) ** 2 + 3 * (2.0 ** -12) ** 2) ** 0.5
    for i in range(3):
        k, v = (sequence(x, c.tables[i], n[i], 16) for x in (kv, vv))
        s = slice(cu[i], cu[i + 1])
        want, _ = attend(q64[s], k, v, lam64[s], scale, n[i] - new[i] + np.arange(new[i]))
        rel = np.linalg.norm(got[s] - want) / np.linalg.norm(want)
        log(f"normal rows dtype={dtype} d={d} sequence {i}: {rel:.3g} of {limit:.3g}")
        assert rel <= limit
