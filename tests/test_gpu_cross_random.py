"""Cross attention at random shapes, types, lengths and hints, against 64 bits."""
import numpy as np
import pytest

import airkv
from test_gpu_cross import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seed", range(64))
def test_random(seed):
    r = np.random.default_rng(1000 + seed)
    dtype = [airkv.F32, airkv.BF16, airkv.INT8, airkv.FP8][seed % 4]
    d = 32 * int(r.integers(1, 9))
    groups = [g for g in (8, 16, 32, 64) if d % g == 0]
    batch = int(r.integers(1, 9))
    lens = r.integers(0, [40, 200, 900, 3000][int(r.integers(4))], batch)
    rows = r.integers(0, [2, 5, 30, 150][int(r.integers(4))], batch)
    rows[int(r.integers(batch))] += 1
    io, out = (["bf16", "f32"][int(x)] for x in r.integers(0, 2, 2))
    hint = [None, 0, int(rows.max()), 1, 4096][int(r.integers(5))]
    c = Case(dtype, d, int(r.integers(1, 5)), int(r.choice([1, 2, 3, 4, 7, 8])), int(r.choice([16, 32])), lens, rows, io, out,
             int(r.choice(groups)), seed, float(r.choice([0.1, 1.0, 3.0])))
    c.check(f"dtype {dtype}, d {d}, lens {lens.tolist()}, rows {rows.tolist()}", max_q_len=hint)
