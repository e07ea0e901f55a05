"""A session's keys to their new places after its compaction: air_kv_rotate over each layer's pool."""
import numpy as np
import pytest

import airkv
import rotary_ref as ref
from gpu_helpers import torch_mod

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [airkv.F32, airkv.BF16])
def test_rotate_after_a_sessions_compaction(dtype):
    torch = torch_mod()
    r = np.random.default_rng(8)
    f = ref.frequencies(64)
    mgr = airkv.SequenceManager(40, 16)
    pools = [airkv.KvPool(40, 16, 2, 64, dtype) for _ in range(2)]
    s = airkv.PagedSessionCache(mgr, pools)
    raw = r.standard_normal((2, 2, 150, 2, 64)).astype(np.float32)
    for layer in range(2):
        s.append(layer, torch.from_numpy(ref.turned(raw[layer, 0], np.arange(150), f, False)).cuda(), torch.from_numpy(raw[layer, 1]).cuda())
    child = s.fork()                                   # shares every block
    before = [[x.clone() for x in child.load(layer)] for layer in range(2)]
    keep = np.concatenate([np.arange(20), np.sort(r.permutation(np.arange(20, 150))[:60])])
    s.compact(keep)
    tables, lens = mgr.export_tables([s.seq_id], 5)
    assert lens[0] == 80
    at = [torch.from_numpy(np.ascontiguousarray(x, np.int32)).cuda() for x in (tables, keep, [0, 80])]
    for layer, pool in enumerate(pools):
        pool.rotate(*at, torch.from_numpy(f).cuda())
        k, v = (x.double().cpu().numpy().reshape(80, 2, 64) for x in s.load(layer))
        want = ref.exact(raw[layer, 0][keep], np.arange(80), f, False)
        a, b = ref._parts(64, False)
        size = np.tile(np.hypot(raw[layer, 0][keep][..., a], raw[layer, 0][keep][..., b]), 2)
        # stored twice (half a step of the page each time), turned twice (f32: 3 * 2^-24 * sqrt(2) of a pair's size)
        half = 2.0 ** -24 if dtype == airkv.F32 else 2.0 ** -8
        near = bool((np.abs(k - want) <= size * (2 * half * 2 ** 0.5 + 6 * 2.0 ** -24 * 2 ** 0.5)).all())
        assert near
        assert np.array_equal(v.astype(np.float32), before[layer][1].float().cpu().numpy().reshape(150, 2, 64)[keep])
        for x, y in zip(child.load(layer), before[layer]):
            assert torch.equal(x, y)
