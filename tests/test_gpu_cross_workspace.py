"""Cross attention's workspace: one serves every call of a pool."""
import pytest

import airkv
from gpu_helpers import torch_mod
from test_gpu_cross import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,io", [(airkv.BF16, "bf16"), (airkv.F32, "f32"), (airkv.INT8, "f32")])
def test_one_workspace_for_every_shape(dtype, io):
    torch = torch_mod()
    one = Case(dtype, 64, 2, 4, 16, [9000, 5], [1, 1], io=io, seed=1)
    many = Case(dtype, 64, 2, 4, 16, [9000, 700], [300, 77], io=io, seed=2)
    size = one.pool.cross_workspace_size(8, 2, 1)
    assert size == many.pool.cross_workspace_size(2, 600, 0) == many.pool.cross_workspace_size(16, 1, 4096)
    ws = torch.full((size,), 255, dtype=torch.uint8, device="cuda")    # (every f32 of it a NaN)
    for c, most in ((one, 1), (many, 300), (one, 0), (many, 0), (one, 1)):
        c.out.fill_(7.0)
        c.check(max_q_len=most, workspace=ws)
