"""Differential attention, decode and prefill, over values near either end of f32, against
64 bits."""
import numpy as np
import pytest

import airkv
from diff_ref import attend, check, pool_values, sequence
from gpu_helpers import log, torch_mod
from test_gpu_diff_attention import Cache, _p_step, _refill

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [airkv.F32, airkv.BF16, airkv.INT8, airkv.FP8])
@pytest.mark.parametrize("f32", [True, False])
@pytest.mark.parametrize("case", ["huge", "small", "tiny"])
def test_values_near_the_ends_of_f32(dtype, f32, case):
    """Values of 1e36 under scores that grow by a nat a tile, so that every tile's
    probabilities are the largest so far; values of 1e-28 and 1e-36 (outputs times 2^80
    and 2^100).  Products on bf16 parts cut a value of an f32 page off below bf16's least
    number, 2^-133: so much of it may be missing."""
    torch = torch_mod()
    if case != "huge" and dtype == airkv.FP8:
        pytest.skip("the pool's own rule: groups below 1e-8 are zeros")
    if case == "tiny" and dtype == airkv.INT8:
        pytest.skip("decode: a scale times a probability is cut off below 2^-133 and met by codes up to 127: outside its range")
    d, n, new = 64, [1100, 130, 33], [60, 1, 33]
    c = Cache(dtype, d, 2, 16, n, seed=80)
    if case == "huge":
        t = np.concatenate([np.arange(m) for m in n]).astype(np.float32)[:, None]
        c.k[:, :, 0] = t / 16 * np.sqrt(d)
        c.v[:] = c.v * np.float32(1e35) + np.float32(1e36)
        _refill(c, lambda t: 1.0, lambda t: 1.0)
    else:
        _refill(c, lambda t: 1.0, lambda t: 1e-36 if case == "tiny" else 1e-28)
    out_scale = {"huge": 0.5, "small": 2.0 ** 80, "tiny": 2.0 ** 100}[case]
    floor = 2.0 ** -133 * out_scale if dtype == airkv.F32 else 0.0
    kv, vv = pool_values(c.pool)
    scale = float(np.float32(1.0) / np.sqrt(np.float32(d)))
    tables, lens = c.device()
    # scores up to 70: those of 1-byte keys err by 2^-11 of themselves under 16-bit products
    p_step = 0.0 if f32 or dtype == airkv.F32 else _p_step(c) + (0.0 if dtype == airkv.BF16 else 2.0 ** -11 * 2 * 70)
    for name, rows in (("decode", [1, 1, 1]), ("prefill", new)):
        cu = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        q, lam, _, _, lam64, _ = c.rows(int(cu[-1]), 2, f32, True, False)
        if case == "huge":
            q[:, :, 0] = 1.0
        q64 = q.float().cpu().numpy().astype(np.float64)
        step = p_step if name == "prefill" else 0.0
        want, bound = np.zeros((int(cu[-1]), 2, 2 * d)), np.zeros((int(cu[-1]), 2, 2 * d))
        for i, (m, r) in enumerate(zip(n, rows)):
            k, v = (sequence(x, c.tables[i], m, 16) for x in (kv, vv))
            s = slice(cu[i], cu[i + 1])
            want[s], bound[s] = attend(q64[s], k, v, lam64[s], scale, m - r + np.arange(r), out_scale=out_scale, p_step=step)
            bound[s] += floor * (1 + np.abs(lam64[s, :, None]))
        odt = airkv.F32 if f32 else airkv.BF16
        out = torch.full(want.shape, float("nan"), device="cuda", dtype=q.dtype)
        if name == "decode":
            for splits in (256, 3, 1):
                c.pool.paged_diff_decode(q, lam, tables, lens, out.fill_(float("nan")), out_scale=out_scale, max_splits=splits)
                used = check(out.float().cpu().numpy(), want, bound, odt, f"decode, splits {splits}", step)
        else:
            c.pool.paged_diff_prefill(q, lam, torch.from_numpy(cu).cuda(), tables, lens, out, max_q_len=max(rows), out_scale=out_scale)
            # (the whole result's error is held to 1e-5 where nothing is cut off: 2^-133 is 9e-5 of 1e-36)
            used = check(out.float().cpu().numpy(), want, bound, odt, "prefill", step or (floor if case == "tiny" else 0.0))
        log(f"{case} {name} dtype={dtype} f32={f32}: {used:.3f} of the bound")
    assert c.pool.error_count() == 0


@pytest.mark.parametrize("dtype", [airkv.BF16, airkv.INT8, airkv.FP8])
def test_sums_of_a_long_block_near_the_largest_float(dtype):
    """Pieces of a block under 16-bit products: sums of a thousand values of 1e36."""
    torch = torch_mod()
    c = Cache(dtype, 32, 2, 16, [40000], seed=81)
    c.v[:] = c.v * np.float32(1e35) + np.float32(1e36)
    _refill(c, lambda t: 1.0, lambda t: 1.0)
    q, lam, _, q64, lam64, _ = c.rows(4, 2, False, True, False)
    tables, lens = c.device()
    kv, vv = (sequence(x, c.tables[0], 40000, 16) for x in pool_values(c.pool))
    p_step = _p_step(c)
    want, bound = attend(q64, kv, vv, lam64, float(np.float32(1.0) / np.sqrt(np.float32(32))), 39996 + np.arange(4), p_step=p_step)
    out = torch.full((4, 2, 64), float("nan"), device="cuda", dtype=torch.bfloat16)
    c.pool.paged_diff_prefill(q, lam, torch.tensor([0, 4], dtype=torch.int32, device="cuda"), tables, lens, out, max_q_len=4)
    used = check(out.float().cpu().numpy(), want, bound, airkv.BF16, "prefill", p_step)
    log(f"long sums dtype={dtype}: {used:.3f} of the bound")


@pytest.mark.parametrize("dtype", [airkv.F32, airkv.BF16, airkv.INT8, airkv.FP8])
@pytest.mark.parametrize("f32", [True, False])
def test_scores_that_f32_rounds_by_whole_numbers(dtype, f32):
    """Scores of 2^20 to 2^36, whose roundings are a probability's factor of up to 2^12.  The
    largest of a row lies so far above the others that the row is its values."""
    torch = torch_mod()
    d, n, new = 64, [500, 90, 33], [100, 90, 33]
    odt = airkv.F32 if f32 else airkv.BF16
    for e in range(10, 20, 2):
        c = Cache(dtype, d, 2, 16, n, seed=82 + e)
        _refill(c, lambda t: 2.0 ** e, lambda t: 1.0)
        kv, vv = pool_values(c.pool)
        cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        q, lam, _, _, lam64, _ = c.rows(int(cu[-1]), 2, f32, True, False)
        q = (q.float() * 2.0 ** e).to(q.dtype)
        q64 = q.float().cpu().numpy().astype(np.float64)
        tables, lens = c.device()
        out = torch.full((int(cu[-1]), 2, 2 * d), float("nan"), device="cuda", dtype=q.dtype)
        c.pool.paged_diff_prefill(q, lam, torch.from_numpy(cu).cuda(), tables, lens, out, max_q_len=max(new))
        got = out.float().cpu().numpy()
        assert np.isfinite(got).all(), e
        last = torch.from_numpy(cu[1:].astype(np.int64) - 1).cuda()
        dec = torch.full((3, 2, 2 * d), float("nan"), device="cuda", dtype=q.dtype)
        c.pool.paged_diff_decode(q[last].contiguous(), lam[last].contiguous(), tables, lens, dec)
        dec = dec.float().cpu().numpy()
        assert np.isfinite(dec).all(), e
        seen = 0
        for i in range(3):
            k, v = (sequence(x, c.tables[i], n[i], 16) for x in (kv, vv))
            for r in range(new[i]):
                row, m = cu[i] + r, n[i] - new[i] + r + 1
                for h in range(2):
                    want, sure = 0.0, True
                    for a in range(2):
                        s = k[a, :m] @ q64[row, 2 * h + a]
                        top = np.sort(s)[::-1]
                        # scores in 32 bits, from keys of 1-byte pages in 11: apart by more than they can err
                        size = (np.abs(k[a, :m]) @ np.abs(q64[row, 2 * h + a])).max()
                        sure &= m == 1 or (top[0] - top[1]) > size * (2.0 ** -9 if dtype in (airkv.INT8, airkv.FP8) else 2.0 ** -16) + 800
                        best = int(s.argmax())
                        want = want + (1.0 if a == 0 else -lam64[row, h]) * np.concatenate([v[0, best], v[1, best]])
                    if not sure:
                        continue
                    seen += 1
                    # values in 11 bits under the 16-bit products, two maps' errors and the output's
                    tol = (2.0 ** -10 if not f32 else 2.0 ** -20) * (1 + abs(lam64[row, h])) * np.abs(v).max() + \
                        (2.0 ** -8 if not f32 else 0.0) * np.abs(want)
                    assert (np.abs(got[row, h] - want) <= tol).all(), (e, i, r, h)
                    if r == new[i] - 1:
                        assert (np.abs(dec[i, h] - want) <= tol).all(), (e, i, h, "decode")
        assert seen > 200, seen
    assert c.pool.error_count() == 0
