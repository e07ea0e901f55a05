"""What KvPool's methods do in front of a launch, without a GPU: the library's calls, the
tensors' checks and torch's streams are stood in for."""
import contextlib
import types

import pytest
import torch

import airkv
from airkv import pool as pool_module

HERE = 4096                                             # an address


class _Stream:
    cuda_stream = 77


@pytest.fixture
def call(monkeypatch):
    """A pool whose launches are recorded, with the stream of every allocation."""
    now, log = [None], types.SimpleNamespace(allocated=[], launched=[])

    @contextlib.contextmanager
    def on(stream):
        before, now[0] = now[0], stream.cuda_stream
        yield
        now[0] = before

    real = torch.empty

    def empty(n, dtype=None, device=None):
        assert device == "cuda"
        log.allocated.append(now[0])
        return real(n, dtype=dtype)

    class Lib:
        def __getattr__(self, name):
            def fn(*args):
                log.launched.append((name, args))
                return 0
            return fn

    lib = Lib()
    monkeypatch.setattr(pool_module._lib, "load", lambda: lib)
    monkeypatch.setattr(pool_module, "_dev", lambda t, dtype, what, shape=None: HERE)
    monkeypatch.setattr(pool_module, "_stream_ptr", lambda s: 0 if s is None else s.cuda_stream)
    monkeypatch.setattr(torch, "empty", empty)
    monkeypatch.setattr(torch.cuda, "stream", on)
    monkeypatch.setattr(torch.cuda, "ExternalStream", lambda p: types.SimpleNamespace(cuda_stream=p))
    p = airkv.KvPool.__new__(airkv.KvPool)
    p.handle, p.n_kv_heads, p.head_dim, p.block_size, p._scale, p.dtype = None, 2, 32, 16, 0.1, airkv.BF16
    for name in ("decode", "prefill", "diff_decode", "diff_prefill"):
        monkeypatch.setattr(p, name + "_workspace_size", lambda *a: 64, raising=False)
    q = torch.zeros(3, 4, 32)
    tables, lens = torch.zeros(3, 2, dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    cu = torch.arange(4, dtype=torch.int32)
    lam, rows, wide = torch.zeros(2), torch.zeros(3, 2, 32), torch.zeros(3, 2, 64)
    log.pool, log.args = p, dict(q=q, tables=tables, lens=lens, cu=cu, lam=lam, wide=wide)
    log.calls = {
        "paged_decode": lambda s, **k: p.paged_decode(q, tables, lens, q, stream=s, **k),
        "paged_decode_append": lambda s, **k: p.paged_decode_append(q, rows, rows, tables, lens, q, stream=s, **k),
        "bind_decode": lambda s, **k: p.bind_decode(q, tables, lens, q, None, stream=s, **k),
        "bind_decode_append": lambda s, **k: p.bind_decode_append(q, rows, rows, tables, lens, q, None, stream=s, **k),
        "paged_prefill": lambda s, **k: p.paged_prefill(q, cu, tables, lens, q, max_q_len=1, stream=s, **k),
        "bind_prefill": lambda s, **k: p.bind_prefill(q, cu, tables, lens, q, max_q_len=1, stream=s, **k),
        "paged_diff_decode": lambda s, **k: p.paged_diff_decode(q, lam, tables, lens, wide, stream=s, **k),
        "bind_diff_decode": lambda s, **k: p.bind_diff_decode(q, lam, tables, lens, wide, stream=s, **k),
        "paged_diff_prefill": lambda s, **k: p.paged_diff_prefill(q, lam, cu, tables, lens, wide, stream=s, **k),
        "bind_diff_prefill": lambda s, **k: p.bind_diff_prefill(q, lam, cu, tables, lens, wide, stream=s, **k)}
    return log


@pytest.mark.parametrize("name", ["paged_decode", "paged_decode_append", "bind_decode", "bind_decode_append", "paged_prefill",
                                  "bind_prefill", "paged_diff_decode", "bind_diff_decode", "paged_diff_prefill", "bind_diff_prefill"])
def test_a_calls_own_workspace_is_its_streams(call, name):
    """A workspace that a call makes is memory of the stream the call runs on."""
    call.calls[name](_Stream())
    assert call.allocated == [77] and call.launched
    call.calls[name](None)
    assert call.allocated == [77, None]


@pytest.mark.parametrize("name", ["paged_diff_decode", "bind_diff_decode", "paged_diff_prefill", "bind_diff_prefill"])
def test_a_norm_eps_that_is_no_float32_is_refused(call, name):
    """What float32 holds as 0 would be a call without the norm."""
    for eps in (1e-50, 0.0, -1e-5, float("nan")):
        with pytest.raises(ValueError, match="norm_eps"):
            call.calls[name](None, norm_eps=eps)
    assert not call.launched
    call.calls[name](None, norm_eps=1e-40)              # a subnormal float32
    assert call.launched


@pytest.mark.parametrize("name", ["paged_diff_prefill", "bind_diff_prefill"])
def test_differential_prefill_reads_nothing_back(call, name, monkeypatch):
    """Without max_q_len too: no wait for the device, so the call can be captured."""
    def waits(*a, **k):
        raise AssertionError("read back")
    for f in ("item", "cpu", "tolist", "__int__", "__bool__"):
        monkeypatch.setattr(torch.Tensor, f, waits)
    call.calls[name](None)
    assert call.launched and call.launched[-1][1][9] == 3                # the rows there are


def test_a_sessions_compaction_takes_positions_only(monkeypatch):
    """A mask is no list of positions, and a fraction none of them."""
    import numpy as np
    from airkv import session as session_module
    got = []

    class Lib:
        @staticmethod
        def air_kv_session_compact(h, stream, keep, n):
            got.append(n)
            return 0

    monkeypatch.setattr(session_module._lib, "load", lambda: Lib)
    monkeypatch.setattr(session_module, "_stream_ptr", lambda s: 0)
    s = airkv.PagedSessionCache.__new__(airkv.PagedSessionCache)
    s._h = None
    for bad in (np.array([False, True]), [True, False, True], [0.0, 1.5], np.array([0.0])):
        with pytest.raises(TypeError, match="integers"):
            s.compact(bad)
    with pytest.raises(ValueError):
        s.compact([[0, 1]])
    assert not got
    for good in ([], [0, 2], np.arange(3, dtype=np.int32), np.arange(4, dtype=np.uint8), (1, 2)):
        s.compact(good)
    assert got == [0, 2, 3, 4, 2]
