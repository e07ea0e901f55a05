"""Cross attention over 1-byte pages that hold rows which were not finite when they were appended."""
import math

import numpy as np
import pytest

import airkv
from gpu_helpers import torch_mod
from test_gpu_cross import Case, _dev

pytestmark = pytest.mark.gpu


def _appended(c, seq, token, key=None, value=None):
    """Token `token` of sequence `seq` again, its element 5 at head 0 the given key or value."""
    torch = torch_mod()
    rows = [torch.randn(1, c.pool.n_kv_heads, c.pool.head_dim, device="cuda") for _ in range(2)]
    for x, y in zip(rows, (key, value)):
        if y is not None:
            x[0, 0, 5] = y
    slot = int(c.tables[seq, token // c.bs]) * c.bs + token % c.bs
    c.pool.append(*rows, torch.tensor([slot], device="cuda"))


@pytest.mark.parametrize("what", ["key", "value"])
@pytest.mark.parametrize("size", [math.inf, -math.inf])
@pytest.mark.parametrize("rows", ["few", "many"])
@pytest.mark.parametrize("dtype,d", [(airkv.INT8, 64), (airkv.FP8, 64), (airkv.INT8, 192), (airkv.FP8, 128)])
def test_infinite_rows(dtype, d, rows, size, what):
    """An infinite element leaves its group an infinite scale: 0 * inf = NaN for each of its elements, in whatever type
    the output is.  A key's reach every column of the rows that see it, a value's its group's columns."""
    for out in ("bf16", "f32"):
        c = Case(dtype, d, 2, 2, 16, [300, 90], [3, 2] if rows == "few" else [150, 70], out=out, seed=d)
        for token in (0, 77):
            _appended(c, 0, token, **{what: size})
        got = c.call(max_q_len=int(c.rows.max())).double().cpu()
        with np.errstate(invalid="ignore"):
            want, bound = c.want()
        n = int(c.rows[0])
        # (heads 0 and 1 read head 0's pages; a scale group is 32 elements)
        hit = torch_mod().zeros(want.shape, dtype=bool)
        hit[:n, :2, :d if what == "key" else 32] = True
        expected, same = bool((want.isnan() == hit).all()), bool((got.isnan() == hit).all())
        assert expected and same, (out, int(got.isnan().sum()), int(hit.sum()))
        near = bool(((got - want).abs() <= bound)[~hit].all())
        assert near


@pytest.mark.parametrize("dtype", [airkv.INT8, airkv.FP8])
def test_groups_of_zeros(dtype):
    """Finite scales of any size are none of that: tokens of zeros (whose scale is 1) beside tiny and large ones."""
    torch = torch_mod()
    for size in (1e-34, 1e34):
        c = Case(dtype, 64, 1, 2, 16, [300, 90], [150, 3], seed=3, out="f32" if size > 1 else "bf16")
        n = c.pool.num_blocks * 16
        k, v = torch.randn(n, 1, 64, device="cuda"), torch.randn(n, 1, 64, device="cuda") * size
        v[::3] = 0.0
        k[1::3] = 0.0
        c.pool.append(k, v, torch.arange(n, device="cuda"))
        c.out = c.out.bfloat16()
        c.out_io, c.precise = "bf16", False
        got = c.call(max_q_len=150).double().cpu()
        want, bound = c.want()
        near = bool(((got - want).abs() <= bound).all())
        assert near
