"""Cross attention counts every key once: all keys weigh the same and a column's output is the share of the keys that
it marks, so that one key left out, or taken twice, changes a column by far more than any rounding."""
import numpy as np
import pytest

import airkv
from gpu_helpers import torch_mod
from test_gpu_cross import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("io", ["bf16", "f32"])
@pytest.mark.parametrize("dtype", [airkv.BF16, airkv.F32, airkv.INT8, airkv.FP8])
@pytest.mark.parametrize("d", [64, 96, 128, 256])
def test_every_key_counts_once(d, dtype, io):
    torch = torch_mod()
    # lengths around tiles of 16 to 128 keys, and one that many slices share
    lens = [1, 15, 16, 17, 31, 33, 63, 65, 127, 129, 40 * d + 5]
    for rows in ([1] * len(lens), [2] * len(lens), [150, 1, 40, 3, 70, 1, 33, 2, 65, 300, 90]):
        c = Case(dtype, d, 1, 2, 16, lens, rows, io=io, seed=d)
        n = c.pool.num_blocks * 16
        k, v = torch.randn(n, 1, d, device="cuda"), torch.zeros(n, 1, d, device="cuda")
        want = np.zeros((len(lens), d))
        for i, m in enumerate(lens):
            at = np.arange(m)
            slots = c.tables[i].astype(np.int64)[at // 16] * 16 + at % 16
            # neighbours, keys a tile apart and a tile of keys all mark different columns
            v[torch.from_numpy(slots).cuda(), 0, torch.from_numpy(at % d).cuda()] = 1.0
            want[i] = np.bincount(at % d, minlength=d) / m
        c.pool.append(k, v, torch.arange(n, device="cuda"))
        c.q.zero_()
        for hint in (1, max(rows)):
            c.out.fill_(7.0)
            out = c.call(max_q_len=hint).double().cpu().numpy()
            for i in range(len(lens)):
                got = out[c.cu[i]:c.cu[i + 1]]
                # at most 41 keys of a column: one is 1 in 41 of it.  Half a step of bf16 (2^-8) for the output, and f32
                # sums of at most 2^14 terms (fp8 marks 1 as 448 / 448, int8 as 127 / 127: each within 2^-23)
                bound = want[i] * ((2.0 ** -8 if io == "bf16" else 0.0) + 2.0 ** -9)
                near = bool((np.abs(got - want[i]) <= bound).all())
                assert near, (lens[i], rows[i], hint)
