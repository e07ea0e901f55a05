"""1-byte pages: what lies far below its neighbours, in queries, keys and values, to the steps the header names."""
import numpy as np
import pytest

import airkv
from gpu_helpers import torch_mod
from test_gpu_cross import Case

pytestmark = pytest.mark.gpu

STEP = {airkv.INT8: 2.0 ** -34, airkv.FP8: 2.0 ** -35.8}


@pytest.mark.parametrize("rows", [1, 200])
@pytest.mark.parametrize("dtype", sorted(STEP))
def test_small_values_beside_large_ones(dtype, rows):
    """One key: the output is its value, whatever the probability.  A group of 2^-20 to 2^-40 beside one of 1."""
    torch = torch_mod()
    d = 64
    for e in (-10, -20, -26, -30, -33, -40):
        c = Case(dtype, d, 1, 1, 16, [1], [rows], seed=rows)
        v = torch.ones(16, 1, d, device="cuda")
        v[:, :, 32:] = 1.5 * 2.0 ** e
        c.pool.append(torch.randn(16, 1, d, device="cuda"), v, torch.arange(16, device="cuda") + 16 * int(c.tables[0, 0]))
        got = c.call(max_q_len=rows).double().cpu()
        want, _ = c.want()
        # f16's 11 bits, or its step, half of it off; the output's rounding to bf16, f32's of the two
        bound = want.abs() * (2.0 ** -8 + 2.0 ** -11 + 2.0 ** -20) + STEP[dtype] / 2
        near = bool(((got - want).abs() <= bound).all())
        assert near, e


@pytest.mark.parametrize("rows", [1, 200])
@pytest.mark.parametrize("dtype", sorted(STEP))
def test_small_queries_beside_large_ones(dtype, rows):
    """Element 0 of a query is 1 and meets keys of 0; element 40 is 2^e and meets keys that differ by 2^-e: which of two
    keys wins depends on it alone.  Exact down to 2^-21, to half a step of 2^-28 below."""
    torch = torch_mod()
    d = 64
    for e in (-8, -15, -21, -24, -27):
        c = Case(dtype, d, 1, 1, 16, [2], [rows], seed=rows)
        k, v = torch.zeros(16, 1, d, device="cuda"), torch.zeros(16, 1, d, device="cuda")
        k[0, 0, 40], k[1, 0, 40] = 2.0 ** -e, -(2.0 ** -e)
        v[0], v[1] = 1.0, -1.0
        c.pool.append(k, v, torch.arange(16, device="cuda") + 16 * int(c.tables[0, 0]))
        c.q.zero_()
        c.q[:, :, 0] = 1.0
        c.q[:, :, 40] = 1.0078125 * 2.0 ** e           # (all of bf16's 8 bits)
        got = c.call(scale=0.5, max_q_len=rows).double().cpu()
        off = 0.0 if e >= -21 else 2.0 ** (-29 - e)    # of the small element, relative to it
        # the difference of the scores is 1.0078 times a key's 2 * 0.5 (11 bits); the output is tanh of half of it
        lo, hi = (np.tanh(0.5 * 1.0078125 * (1 + s * (off + 2.0 ** -11))) + s * (2.0 ** -8 + 2.0 ** -10) for s in (-1, 1))
        near = bool(((got >= lo) & (got <= hi)).all())
        assert near, (e, got.flatten()[:2].tolist())
