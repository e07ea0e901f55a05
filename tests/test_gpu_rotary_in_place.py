"""Rows that are written where they are read: every head size and layout, against another output's bits."""
import pytest

import airkv
import rotary_ref as ref
from gpu_helpers import torch_mod

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("io", ["bf16", "f32"])
@pytest.mark.parametrize("d,rot", [(32, 8), (64, 64), (96, 40), (128, 128), (160, 160), (224, 112), (256, 256), (256, 24)])
def test_queries_in_place(d, rot, io, pairs):
    torch = torch_mod()
    f = torch.from_numpy(ref.frequencies(rot)).cuda()
    for n, heads in ((1, 1), (3, 40), (700, 6)):
        gen = torch.Generator(device="cuda").manual_seed(n + d)
        q, k, v = (torch.randn(n, h, d, generator=gen, device="cuda").to(torch.bfloat16 if io == "bf16" else torch.float32) for h in (heads, 2, 2))
        pool = airkv.KvPool(-(-n // 16), 16, 2, d, airkv.BF16)
        slots, at = torch.arange(n, device="cuda"), torch.arange(n, dtype=torch.int32, device="cuda") * 37 + 5
        want = pool.append_rotary(q, k, v, slots, at, f, interleaved=pairs)
        own = q.clone()
        assert pool.append_rotary(own, k, v, slots, at, f, q_out=own, interleaved=pairs) is own
        same = torch.equal(own.view(torch.uint8), want.view(torch.uint8))
        assert same, (n, heads)
