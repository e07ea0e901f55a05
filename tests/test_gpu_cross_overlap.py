"""Cross attention's output over its queries: in place, and otherwise refused."""
import pytest

import airkv
from gpu_helpers import torch_mod
from test_gpu_cross import Case

pytestmark = pytest.mark.gpu


def test_out_over_q():
    torch = torch_mod()
    c = Case(airkv.BF16, 64, 2, 2, 16, [100, 30], [5, 40])
    want = c.call(max_q_len=40).clone()
    flat = torch.zeros(2 * c.q.numel(), dtype=torch.bfloat16, device="cuda")
    n, shape = c.q.numel(), c.q.shape
    rows = flat[:n].view(shape).copy_(c.q)
    c.q = rows
    # a row later, the last element alone, the same memory as another type
    for out in (flat[256:256 + n].view(shape), flat[n - 8:2 * n - 8].view(shape), flat.view(torch.float32).view(shape)):
        c.out = out
        with pytest.raises(airkv.AirKvError, match="overlaps"):
            c.call(max_q_len=40)
    torch.cuda.synchronize()
    assert torch.equal(flat[:n].view(shape), rows) and not flat[n:].any()
    # side by side, and in place
    c.out = flat[n:].view(shape)
    assert torch.equal(c.call(max_q_len=40), want)
    c.out = rows
    assert torch.equal(c.call(max_q_len=40), want)
