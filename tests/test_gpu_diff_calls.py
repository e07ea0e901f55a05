"""Calls of differential attention whose workspace is their own: on a stream that is busy
while the current one takes and fills memory."""
import numpy as np
import pytest

import airkv
from gpu_helpers import torch_mod
from test_gpu_diff_attention import Cache

pytestmark = pytest.mark.gpu


def test_a_call_on_a_busy_stream_keeps_its_workspace():
    torch = torch_mod()
    c = Cache(airkv.BF16, 64, 4, 16, [700, 30, 2000], seed=70)
    q, lam, _, _, _, _ = c.rows(3, 4, False, False, False)
    tables, lens = c.device()
    cu = torch.arange(4, dtype=torch.int32, device="cuda")
    plain = torch.zeros(3, 16, 64, device="cuda", dtype=torch.bfloat16)
    calls = [lambda out, s: c.pool.paged_diff_decode(q, lam, tables, lens, out, stream=s),
             lambda out, s: c.pool.paged_diff_prefill(q, lam, cu, tables, lens, out, max_q_len=1, stream=s)]
    sizes = [c.pool.diff_decode_workspace_size(16, 3, tables.shape[1]), c.pool.diff_prefill_workspace_size(16, 3, 1)]
    calls.append(lambda out, s: c.pool.paged_decode(q, tables, lens, plain, stream=s) if s else c.pool.paged_decode(q, tables, lens, plain))
    sizes.append(c.pool.decode_workspace_size(16, 3, tables.shape[1]))
    busy = torch.randn(4096, 4096, device="cuda")
    for call, size in zip(calls, sizes):
        want = torch.zeros(3, 8, 128, device="cuda", dtype=torch.bfloat16)
        out = want.clone()
        call(want, None)
        torch.cuda.synchronize()
        want_plain = plain.clone()
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            for _ in range(20):
                torch.mm(busy, busy)
        call(out, side)
        held = [torch.empty(size, dtype=torch.uint8, device="cuda").fill_(0xFF) for _ in range(4)]
        torch.cuda.synchronize()
        same = torch.equal(out, want), torch.equal(plain, want_plain)
        assert all(same) and len(held) == 4
    assert c.pool.error_count() == 0


def test_a_captured_prefill_without_max_q_len():
    """Captured with nothing but the tensors it needs, replayed with other queries."""
    torch = torch_mod()
    c = Cache(airkv.BF16, 64, 4, 16, [300, 90], seed=71)
    q, lam, _, _, _, _ = c.rows(40, 2, False, False, False)
    tables, lens = c.device()
    cu = torch.tensor([0, 30, 40], dtype=torch.int32, device="cuda")
    ws = c.pool.new_diff_prefill_workspace(8, 2, 30)
    out = torch.zeros(40, 4, 128, device="cuda", dtype=torch.bfloat16)
    want = torch.zeros_like(out)
    c.pool.paged_diff_prefill(q, lam, cu, tables, lens, out, workspace=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.pool.paged_diff_prefill(q, lam, cu, tables, lens, out, workspace=ws)
    for i in range(3):
        q.copy_(torch.from_numpy(np.random.default_rng(i).standard_normal(tuple(q.shape)).astype(np.float32)))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        c.pool.paged_diff_prefill(q, lam, cu, tables, lens, want, max_q_len=30)
        torch.cuda.synchronize()
        assert bool((out == want).all()), i
